"""The paged 8-bit cache, attention over it and norm_rope_axes against their definitions in 64 bits
(oracle/attention.py, whose bounds say how far a correct implementation may be off)."""

from __future__ import annotations

import pytest
import torch

from oracle import attention as oracle
from oracle.linear import expected_norm_rope
from tests.test_attention_cpu import request

pytestmark = pytest.mark.gpu

DIM = 128
EPS = 1e-6
SCALE = DIM**-0.5
CACHE = ("pages", "cu", "lengths", "k_cache", "v_cache", "k_scale", "v_scale")
HEADS = [(16, 2), (4, 4), (5, 1), (12, 4), (32, 2), (40, 1)]


def announce(**what):
    print("case:", " ".join(f"{k}={v}" for k, v in what.items()), flush=True)


def case_of(lengths, new, page, heads, seed, device, *, gated=False, front=0, behind=0):
    """A cache of `lengths` tokens a request and the call's activations, as column slices of one
    buffer; `front` and `behind` rows outside every request."""
    cache, _ = request(lengths, new, page, heads[1], seed, device)
    cache["cu"] += front
    tokens = front + sum(new) + behind
    gen = torch.Generator(device=device).manual_seed(seed)
    q_heads, kv_heads = heads
    rows = torch.randn(tokens, (2 * q_heads + 2 * kv_heads) * DIM, generator=gen,
                       device=device).bfloat16()
    q, k, v, gate = (x.view(tokens, -1, DIM) for x in
                     rows.split([n * DIM for n in (q_heads, kv_heads, kv_heads, q_heads)], 1))
    return dict(cache, q=q, k=k, v=v, gate=gate if gated else None,
                out=torch.full((tokens, q_heads, DIM), 7.0, dtype=torch.bfloat16, device=device))


def within(actual, expected, bound, label):
    """Inside the bound where the definition is finite, NaN where it is not."""
    actual, expected, bound = (x.cpu().double() for x in (actual, expected, bound))
    fine = expected.isfinite()
    assert actual[~fine].isnan().all(), f"{label}: finite where the definition is not"
    error = (actual - expected).abs()[fine]
    worst = (error - bound[fine]).max().item() if error.numel() else -1.0
    assert not torch.isnan(error).any() and worst <= 0, (
        f"{label}: {worst:.3e} over the bound, {int((error > bound[fine]).sum())} elements of "
        f"{error.numel()}")


def attend(case, width=None, scale=SCALE):
    args = [case["q"], *(case[x] for x in CACHE), case["gate"], case["out"]]
    if width is None:
        torch.ops.lightdelta.attention_prefill(*args, scale)
    else:
        torch.ops.lightdelta.attention_decode(*args, width, scale)


def check_attention(case, width=None, scale=SCALE):
    want, bound = oracle.expected_attention(case["q"], *(case[x] for x in CACHE), case["gate"],
                                            case["out"], scale, width)
    attend(case, width, scale)
    torch.cuda.synchronize()
    within(case["out"], want, bound, "out")


def check_write(case):
    want = oracle.expected_write(case["k"], case["v"], *(case[x] for x in CACHE))
    torch.ops.lightdelta.cache_write(case["k"], case["v"], *(case[x] for x in CACHE))
    torch.cuda.synchronize()
    for name, expected in zip(("k_cache", "v_cache", "k_scale", "v_scale"), want):
        got = case[name].view(torch.uint8).cpu()
        if name.endswith("cache"):
            got, expected = oracle.canonical(got), oracle.canonical(expected)
        assert torch.equal(got, expected), (name, int((got != expected).sum()))


def check_read(case):
    k, v = (torch.full_like(case[x].contiguous(), 7.0) for x in "kv")
    want = oracle.expected_read(*(case[x] for x in CACHE), k, v)
    torch.ops.lightdelta.cache_read(*(case[x] for x in CACHE), k, v)
    torch.cuda.synchronize()
    for got, expected in zip((k, v), want):
        torch.testing.assert_close(got.double().cpu(), expected, rtol=0, atol=0, equal_nan=True)


# ---- the cache -----------------------------------------------------------------------------


SPANS = [([1], [1]), ([300], [300]), ([5, 64, 129, 1, 40], [5, 64, 129, 1, 40]),
         ([17, 64, 65, 200, 33], [1, 1, 1, 1, 1]), ([100, 31, 250], [37, 16, 130]),
         ([0, 90, 0], [0, 3, 2]), ([130, 4], [4, 4])]


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("span", range(len(SPANS)))
@pytest.mark.parametrize("kv_heads", [1, 3])
def test_write_and_read(gpu, page, span, kv_heads):
    lengths, new = SPANS[span]
    announce(test="cache", page=page, lengths=lengths, new=new, kv_heads=kv_heads)
    case = case_of(lengths, new, page, (kv_heads, kv_heads), seed=span, device=gpu, front=2,
                   behind=3)
    check_write(case)
    check_read(case)


def test_write_grows_scales(gpu):
    """Louder tokens make what a page holds be rounded anew, by up to more powers than e4m3 has;
    quieter ones leave its scale."""
    announce(test="cache_grow")
    for page in (16, 128):
        for power in (-30, -3, 0, 1, 2, 5, 9, 14, 30, 100):
            case = case_of([page + 9, 7], [2, 3], page, (2, 2), seed=3, device=gpu)
            case["k"] *= 2.0**power
            case["v"] *= 2.0**(power / 2)
            check_write(case)


def test_every_value(gpu):
    """Every bf16 there is, in pages with a scale of their own and in one with all of them."""
    announce(test="cache_values")
    every = torch.arange(2**16, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    n = 2**16 // DIM
    for page in (16, 64):
        case = case_of([n], [n], page, (1, 1), seed=4, device=gpu)
        case["k"] = every.view(n, 1, DIM).to(gpu)
        case["v"] = every.flip(0).view(DIM, n).t().reshape(n, 1, DIM).contiguous().to(gpu)
        check_write(case)
        check_read(case)


@pytest.mark.parametrize("value", [float("nan"), float("inf"), 3.3e38, 1e-40, 0.0])
def test_write_far_values(gpu, value):
    announce(test="cache_far", value=value)
    case = case_of([70, 20], [30, 20], 64, (2, 2), seed=5, device=gpu)
    case["k"][3, 0, 5] = value
    case["k"][4, 0, 100] = -value
    case["v"][:, 1] = value
    check_write(case)
    check_read(case)


def test_scales_out_of_range(gpu):
    """Scales that no write made stand for the nearest of their range."""
    announce(test="cache_scales")
    for byte in (0, 26, 27, 246, 247, 255):
        case = case_of([40], [4], 16, (1, 1), seed=6, device=gpu)
        for x in ("k_scale", "v_scale"):
            case[x].view(torch.uint8).fill_(byte)
        check_read(case)
        check_write(case)


@pytest.mark.parametrize("page", [16, 64])
def test_pages_without_a_place(gpu, page):
    """Page ids outside the pool, positions before the first token and past the table."""
    announce(test="cache_places", page=page)
    case = case_of([90, 200, 40, 5], [90, 60, 40, 9], page, (2, 1), seed=7, device=gpu)
    case["pages"][0, 1] = 0
    case["pages"][1, -2] = 10**6
    case["pages"][2, 0] = -3
    case["lengths"][1] += 3 * page
    check_write(case)
    check_read(case)
    check_attention(case)
    check_attention(case, width=4)


# ---- attention -----------------------------------------------------------------------------


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("width", [1, 4])
def test_decode(gpu, heads, page, width):
    lengths = [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 300, 0, 1000]
    new = [min(n, 1 + i % width) if n else 1 for i, n in enumerate(lengths)]
    announce(test="decode", heads=heads, page=page, width=width)
    check_attention(case_of(lengths, new, page, heads, seed=page + width, device=gpu,
                            gated=width == 4, front=1, behind=2), width)


@pytest.mark.parametrize("lengths", [[5000], [3, 9000, 40], [257] * 40, [33] * 150 + [2000],
                                     [1] * 300, [0] * 5])
def test_decode_long_and_many(gpu, lengths):
    """Long contexts beside short ones, more requests than workgroups, and none that has a token."""
    announce(test="decode_many", requests=len(lengths), longest=max(lengths))
    new = [1] * len(lengths)
    check_attention(case_of(lengths, new, 64, (8, 1), seed=8, device=gpu), 1)
    check_attention(case_of(lengths, new, 16, (4, 2), seed=9, device=gpu), 3)


@pytest.mark.parametrize("requests", [90, 200, 260])
@pytest.mark.parametrize("width", [1, 3])
def test_decode_of_many_short(gpu, requests, width):
    """About one, two or three tiles of 64 tokens a workgroup, of one head and the next."""
    announce(test="decode_short", requests=requests, width=width)
    lengths = [7 * i % 200 for i in range(requests)]
    new = [min(n, 1 + i % width) if n else 1 for i, n in enumerate(lengths)]
    check_attention(case_of(lengths, new, 64, (6, 3), seed=11, device=gpu), width)


def test_decode_of_more_rows_than_its_width(gpu):
    announce(test="decode_wide")
    check_attention(case_of([40, 50, 9], [2, 3, 9], 32, (4, 2), seed=10, device=gpu), 2)


PROMPTS = [([1], [1]), ([17], [17]), ([300], [300]), ([1000], [1000]),
           ([5, 64, 129, 1, 40, 257], [5, 64, 129, 1, 40, 257]),
           ([500, 90, 700, 4], [37, 90, 1, 4]), ([3000, 0, 200], [5, 2, 33]), ([5, 90], [9, 3])]


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("prompt", range(len(PROMPTS)))
def test_prefill(gpu, heads, prompt):
    lengths, new = PROMPTS[prompt]
    page = (16, 32, 64, 128)[prompt % 4]
    announce(test="prefill", heads=heads, page=page, lengths=lengths, new=new)
    check_attention(case_of(lengths, new, page, heads, seed=prompt, device=gpu,
                            gated=prompt % 2 == 0, front=2, behind=3))


@pytest.mark.parametrize("width", [None, 2])
@pytest.mark.parametrize("what", ["k", "v", "q"])
def test_values_that_are_not_finite(gpu, what, width):
    """A NaN in the last token's key or value reaches the rows at or behind it, one in a query its
    row and head; what lies behind a request's last token in its page reaches none."""
    announce(test="not_finite", what=what, width=width)
    new = [40, 3] if width is None else [2, 2]
    case = case_of([70, 50], new, 32, (4, 2), seed=11, device=gpu)
    stale = oracle.INDEX
    for name in ("k", "v"):
        codes = case[name + "_cache"].view(torch.uint8).flatten(2)
        for r, n in enumerate((70, 50)):
            last = case["pages"][r, n // 32]
            for t in range(n % 32, 32):  # behind the last token
                codes[last, :, stale[name](32, t).to(gpu)] = 0x7F
        if what == name:
            codes[case["pages"][0, 69 // 32], 1, stale[name](32, 69 % 32)[:5].to(gpu)] = 0xFF
            codes[case["pages"][0, 35 // 32], 0, stale[name](32, 35 % 32)[77].to(gpu)] = 0x7F
    if what == "q":
        case["q"][0, 1, 3] = float("nan")
        case["q"][1, 2, 100] = float("inf")
    check_attention(case, width)
    assert case["out"].isnan().any() and not case["out"].isnan().all()


@pytest.mark.parametrize("width", [None, 2])
def test_not_finite_beside_a_page_that_there_is_not(gpu, width):
    """A NaN in a value that every row sees, in a tile with a page of no place."""
    announce(test="not_finite_beside", width=width)
    for first in (0, 1):
        case = case_of([200, 150], [2, 2], 16, (4, 2), seed=14, device=gpu)
        case["pages"][0, first] = 0
        codes = case["v_cache"].view(torch.uint8).flatten(2)
        codes[case["pages"][0, 2], 1, oracle.INDEX["v"](16, 3)[50].to(gpu)] = 0x7F
        check_attention(case, width)
        assert int(case["out"].isnan().sum()) == 2 * 2  # the rows, and the kv head's two q heads


def test_decode_of_rows_before_the_first_token(gpu):
    """More rows than tokens: those without a position see nothing."""
    announce(test="decode_before")
    check_attention(case_of([2, 0, 1, 70], [4, 2, 3, 4], 16, (6, 2), seed=15, device=gpu, gated=True),
                    4)


def test_one_token_takes_all(gpu):
    """Scores of thousands: weights of one and of zero, the largest first, last and in between."""
    announce(test="attention_peaks")
    for at in (0, 130, 299):
        case = case_of([300, 20], [200, 1], 64, (2, 1), seed=12, device=gpu)
        codes = case["k_cache"].view(torch.uint8).flatten(2)
        codes[case["pages"][0, at // 64], 0, oracle.INDEX["k"](64, at % 64).to(gpu)] = 0x7E
        case["q"].abs_()
        check_attention(case, scale=4.0)


def test_equal_scores(gpu):
    """Queries of zero: the mean of the values seen, whatever the keys' magnitude."""
    announce(test="attention_mean")
    case = case_of([500, 31], [500, 31], 16, (4, 2), seed=13, device=gpu)
    case["q"].zero_()
    check_attention(case)


# ---- norm_rope_axes ------------------------------------------------------------------------


def rope_case(tokens, q_heads, k_heads, rotary, axes, seed, device, dtype=torch.int64):
    gen = torch.Generator(device=device).manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=device)

    half = torch.arange(rotary // 2, device=device, dtype=torch.int32)
    return dict(qkv=normal(tokens, (q_heads + k_heads + 1) * DIM).bfloat16(),
                q_weight=1 + 0.1 * normal(DIM), k_weight=(1 + 0.1 * normal(DIM)).bfloat16(),
                positions=torch.randint(0, 10**5, (axes, tokens), generator=gen, device=device)
                .to(dtype), axes=half % axes,
                inv_freq=10000.0 ** (-torch.arange(0, rotary, 2, device=device) / max(1, rotary)),
                q_heads=q_heads, k_heads=k_heads)


def check_axes(case, interleaved):
    """Sines and cosines of the hardware are good to 2^-20 of a unit vector (tests of norm_rope
    hold that), the norm's sums of 128 squares and its root to 2^-20, and the result is rounded to
    bf16."""
    want = oracle.expected_norm_rope_axes(*case.values(), EPS, interleaved)
    rotary = 2 * case["inv_freq"].numel()
    pair = torch.zeros_like(want)
    heads = case["q_heads"] + case["k_heads"]
    for h in range(heads):
        x = want[:, h * DIM:h * DIM + rotary]
        a, b = ((x[:, 0::2], x[:, 1::2]) if interleaved
                else (x[:, :rotary // 2], x[:, rotary // 2:]))
        size = torch.hypot(a, b)
        size = torch.stack([size, size], -1).flatten(1) if interleaved else size.repeat(1, 2)
        pair[:, h * DIM:h * DIM + rotary] = size
    bound = 2.0**-18 * (pair + want.abs()) + 2.0**-8 * want.abs() + 1e-30
    bound[:, heads * DIM:] = 0
    torch.ops.lightdelta.norm_rope_axes(*case.values(), EPS, interleaved)
    torch.cuda.synchronize()
    within(case["qkv"], want, bound, "norm_rope_axes")


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rotary", [0, 16, 32, 64, 96, 128])
@pytest.mark.parametrize("tokens", [1, 37, 5000])
def test_norm_rope_axes(gpu, tokens, rotary, interleaved):
    announce(test="norm_rope_axes", tokens=tokens, rotary=rotary, interleaved=interleaved)
    case = rope_case(tokens, 5, 2, rotary, 3, seed=rotary, device=gpu,
                     dtype=torch.int32 if rotary == 64 else torch.int64)
    check_axes(case, interleaved)


def test_axes_that_there_are_not(gpu):
    """Pairs whose axis is outside the positions' are only normalised; positions may be rows of a
    wider buffer."""
    announce(test="axes_outside")
    case = rope_case(9, 2, 2, 128, 4, seed=1, device=gpu)
    case["axes"] = torch.tensor([-1, 0, 1, 2, 3, 4, 2**31 - 1, -2**31] * 8, dtype=torch.int32,
                                device=gpu)
    wide = torch.randint(0, 1000, (4, 40), device=gpu)
    case["positions"] = wide[:, 11:20]
    check_axes(case, False)


def test_one_axis_is_norm_rope(gpu):
    """One axis for all frequencies gives norm_rope's bits."""
    announce(test="one_axis")
    for interleaved in (False, True):
        case = rope_case(33, 3, 2, 64, 1, seed=2, device=gpu)
        other = case["qkv"].clone()
        torch.ops.lightdelta.norm_rope(other, case["q_weight"], case["k_weight"],
                                       case["positions"][0], case["inv_freq"], 3, 2, EPS,
                                       interleaved)
        want, bound = expected_norm_rope(case["qkv"], case["q_weight"], case["k_weight"],
                                         case["positions"][0], case["inv_freq"], 3, 2, EPS,
                                         interleaved)
        torch.ops.lightdelta.norm_rope_axes(*case.values(), EPS, interleaved)
        torch.cuda.synchronize()
        assert torch.equal(case["qkv"], other)
        within(case["qkv"], want, bound, "norm_rope")
