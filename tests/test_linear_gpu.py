"""linear_decode, linear_prefill and norm_rope against their definitions in 64 bits
(oracle/linear.py, whose bounds say how far a correct implementation may be off)."""

from __future__ import annotations

import pytest
import torch

from lightdelta_amd import ops
from lightdelta_amd.workloads import HEAD_DIM as DIM
from oracle.linear import expected_linear_decode, expected_linear_prefill, expected_norm_rope

pytestmark = pytest.mark.gpu

EPS = 1e-6
SCALE = DIM**-0.5
DECODE = ("qkv", "log_decay", "indices", "cu", "accepted", "pool", "gate", "weight", "out")
PREFILL = ("qkv", "log_decay", "slots", "has_initial", "cu", "pool", "gate", "weight", "out")


def announce(**what):
    print("case:", " ".join(f"{k}={v}" for k, v in what.items()), flush=True)


def layer(tokens, heads, v_heads, slots, seed, device, *, gated=True, per_token=True,
          weight_dtype=torch.float32, decay=1.0):
    """Activations as column slices of one buffer, decays, parameters and a pool."""
    gen = torch.Generator(device=device).manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=device)

    cols = (2 * heads + v_heads) * DIM
    rows = normal(tokens, cols + v_heads * DIM).bfloat16()
    g = -decay * torch.rand((tokens, v_heads) if per_token else (v_heads,), generator=gen,
                            device=device)
    return dict(
        qkv=rows[:, :cols], log_decay=g,
        gate=rows[:, cols:].view(tokens, v_heads, DIM) if gated else None,
        weight=(1 + 0.1 * normal(DIM)).to(weight_dtype) if gated else None,
        pool=normal(slots, v_heads, DIM, DIM),
        out=torch.full((tokens, v_heads, DIM), 7.0, dtype=torch.bfloat16, device=device))


def prefill_case(lengths, heads, v_heads, seed, device, *, front=0, behind=0, **kw):
    """Prompts of these lengths, `front` and `behind` rows outside them, one slot each."""
    n = len(lengths)
    case = layer(front + sum(lengths) + behind, heads, v_heads, n + 2, seed, device, **kw)
    gen = torch.Generator().manual_seed(seed + 1)
    cu = front + torch.tensor([0] + lengths).cumsum(0)
    case.update(cu=cu.to(torch.int32).to(device),
                slots=(torch.randperm(n + 1, generator=gen)[:n] + 1).to(torch.int32).to(device),
                has_initial=(torch.rand(n, generator=gen) < 0.6).to(device))
    return case


def decode_case(batch, width, heads, v_heads, seed, device, **kw):
    gen = torch.Generator().manual_seed(seed)
    lengths = torch.randint(1, width + 1, (batch,), generator=gen)
    case = layer(batch * width, heads, v_heads, batch * width + 1, seed, device, **kw)
    cu = torch.zeros(batch + 1, dtype=torch.int32)
    cu[1:] = lengths.cumsum(0)
    case.update(
        cu=cu.to(device),
        indices=(torch.randperm(batch * width, generator=gen) + 1).to(torch.int32)
        .view(batch, width).to(device),
        accepted=torch.randint(1, width + 1, (batch,), generator=gen).to(torch.int32).to(device))
    return case


def within(actual, expected, bound, label):
    error = (actual.double() - expected).abs()
    worst = (error - bound).max().item() if error.numel() else -1.0
    assert not torch.isnan(error).any() and worst <= 0, (
        f"{label}: {worst:.3e} over the bound, {int((error > bound).sum())} elements of "
        f"{error.numel()}")


def run_decode(case, eps=EPS, scale=SCALE):
    torch.ops.lightdelta.linear_decode(*[case[k] for k in DECODE], scale, eps)


def run_prefill(case, eps=EPS, scale=SCALE):
    torch.ops.lightdelta.linear_prefill(*[case[k] for k in PREFILL], scale, eps)


def check(case, run, expected, order, eps=EPS, scale=SCALE):
    want = expected(*[case[k] for k in order], scale, eps)
    run(case, eps, scale)
    torch.cuda.synchronize()
    within(case["out"], want[0], want[1], "out")
    within(case["pool"], want[2], want[3], "pool")
    # roundings of 2^-24 on an entry's path, some hundreds of them, add as their root
    written = want[3].flatten(1).amax(1) > 0
    if written.any():
        got, ref = case["pool"].double()[written], want[2][written]
        assert (got - ref).norm() <= 2.0**-19 * ref.norm()


def check_prefill(case, **kw):
    check(case, run_prefill, expected_linear_prefill, PREFILL, **kw)


def check_decode(case, **kw):
    check(case, run_decode, expected_linear_decode, DECODE, **kw)


@pytest.fixture(params=["keep", "stream"])
def policy(request):
    saved = ops.state_cache_policy()
    ops.set_state_cache_policy(request.param)
    yield request.param
    ops.set_state_cache_policy(saved)


# ---- linear_decode -------------------------------------------------------------------------


@pytest.mark.parametrize("heads", [(4, 8), (2, 6), (1, 1), (3, 3)])
@pytest.mark.parametrize("width", [1, 2, 3, 4])
@pytest.mark.parametrize("gated", [False, True])
def test_decode(gpu, policy, heads, width, gated):
    announce(test="linear_decode", heads=heads, width=width, gated=gated, policy=policy)
    check_decode(decode_case(5, width, *heads, seed=width, device=gpu, gated=gated,
                             per_token=width % 2 == 0))


def test_decode_invalid_requests(gpu, policy):
    """Padding sources, slots past the pool, accepted out of range, too many tokens, no tokens, a
    discarded state, rows behind the last request."""
    announce(test="linear_decode_invalid", policy=policy)
    case = decode_case(9, 2, 2, 4, seed=3, device=gpu)
    case["cu"].copy_(torch.tensor([0, 2, 4, 6, 8, 8, 9, 12, 13, 14]))
    case["accepted"].copy_(torch.tensor([1, 3, 2, 0, 1, 2, 1, 1, 1]))
    case["indices"].copy_(torch.tensor([[0, 3], [1, 2], [4, -1], [5, 6], [7, 8], [9, 10], [11, 12],
                                        [19, 13], [14, 19]]))
    before = case["pool"].clone()
    check_decode(case)
    assert case["out"][:2].abs().sum() == 0 and (case["out"][14:] == 7).all()
    assert torch.equal(case["pool"][0], before[0])


@pytest.mark.parametrize("value", [0.0, -200.0, float("-inf"), -1e-30])
def test_decode_extreme_decays(gpu, value):
    announce(test="linear_decode_decays", value=value)
    case = decode_case(3, 2, 2, 4, seed=8, device=gpu)
    case["log_decay"].fill_(value)
    check_decode(case)


def test_decode_strides_and_types(gpu):
    """Rows that start at odd elements, a strided pool, bf16 weight, an expanded decay, a scale
    and an epsilon of their own."""
    announce(test="linear_decode_strides")
    case = decode_case(4, 3, 2, 4, seed=5, device=gpu, weight_dtype=torch.bfloat16,
                       per_token=False)
    wide = torch.zeros(12, case["qkv"].shape[1] + 7, dtype=torch.bfloat16, device=gpu)
    wide[:, 3:-4] = case["qkv"]
    case["qkv"] = wide[:, 3:-4]
    pool = torch.randn(13, 6, DIM, DIM, device=gpu)
    case["pool"] = pool[:, 1:5]
    untouched = pool[:, [0, 5]].clone()
    case["log_decay"] = case["log_decay"][None].expand(12, 4)
    check_decode(case, eps=1e-2, scale=0.3)
    assert torch.equal(pool[:, [0, 5]], untouched)


def test_decode_empty(gpu):
    case = decode_case(2, 1, 2, 4, seed=5, device=gpu)
    case["indices"], case["accepted"] = case["indices"][:0], case["accepted"][:0]
    case["cu"] = case["cu"][:1]
    before = case["out"].clone()
    run_decode(case)
    assert torch.equal(case["out"], before)


# ---- linear_prefill ------------------------------------------------------------------------


@pytest.mark.parametrize("lengths", [[1], [2, 0, 3], [31, 32, 33], [63, 64, 65], [127, 1, 130],
                                     [0, 0, 5], [16] * 9])
@pytest.mark.parametrize("heads", [(2, 4), (1, 3), (2, 2)])
@pytest.mark.parametrize("gated", [False, True])
def test_prefill(gpu, lengths, heads, gated):
    announce(test="linear_prefill", lengths=lengths, heads=heads, gated=gated)
    check_prefill(prefill_case(lengths, *heads, seed=len(lengths), device=gpu, gated=gated,
                               per_token=heads[1] != 3))


@pytest.mark.parametrize("lengths,heads", [([700], (1, 2)), ([1300, 3, 257], (1, 1)),
                                           ([513, 511, 512, 2], (1, 2)), ([5] * 70 + [600], (1, 1)),
                                           ([2100], (1, 1))])
@pytest.mark.parametrize("decay", [0.01, 2.0])
def test_prefill_long(gpu, lengths, heads, decay):
    announce(test="linear_prefill_long", lengths=lengths[-3:], heads=heads, decay=decay)
    check_prefill(prefill_case(lengths, *heads, seed=7, device=gpu, decay=decay))


def test_prefill_padding_and_outside_rows(gpu):
    """Padding slots (0, -1, past the pool), rows ahead of the first and behind the last
    sequence, NaN in rows outside every sequence."""
    announce(test="linear_prefill_padding")
    case = prefill_case([40, 70, 3, 20], 2, 4, seed=4, device=gpu, front=5, behind=9)
    case["slots"].copy_(torch.tensor([0, 2, -1, 6]))
    case["qkv"][:5] = float("nan")
    case["qkv"][-9:] = float("inf")
    case["gate"][-9:] = float("nan")
    before = case["pool"].clone()
    check_prefill(case)
    assert (case["out"][:5] == 7).all() and (case["out"][-9:] == 7).all()
    assert torch.equal(case["pool"][[0, 1, 3, 4, 5]], before[[0, 1, 3, 4, 5]])


@pytest.mark.parametrize("value", [0.0, -200.0, float("-inf"), -1e-30])
def test_prefill_extreme_decays(gpu, value):
    """Also mixed among ordinary ones: -inf empties the state at its token."""
    announce(test="linear_prefill_decays", value=value)
    case = prefill_case([100, 65], 1, 2, seed=6, device=gpu)
    case["log_decay"][::7] = value
    check_prefill(case)
    case = prefill_case([100, 65], 1, 2, seed=6, device=gpu)
    case["log_decay"].fill_(value)
    check_prefill(case)


def test_prefill_nonfinite_stays_in_its_sequence(gpu):
    announce(test="linear_prefill_nonfinite")
    clean = prefill_case([50, 90, 30], 2, 4, seed=12, device=gpu)
    case = {k: v.clone() for k, v in clean.items()}
    case["qkv"][60] = float("nan")
    run_prefill(clean)
    run_prefill(case)
    torch.cuda.synchronize()
    keep = torch.ones(170, dtype=torch.bool, device=gpu)
    keep[50:140] = False
    assert torch.equal(case["out"][keep], clean["out"][keep])
    slots = case["slots"][[0, 2]].long()
    assert torch.equal(case["pool"][slots], clean["pool"][slots])


def test_prefill_strides_and_types(gpu):
    announce(test="linear_prefill_strides")
    case = prefill_case([70, 130], 2, 4, seed=5, device=gpu, weight_dtype=torch.bfloat16,
                        per_token=False)
    n = case["qkv"].shape[0]
    wide = torch.zeros(n, case["qkv"].shape[1] + 7, dtype=torch.bfloat16, device=gpu)
    wide[:, 3:-4] = case["qkv"]
    case["qkv"] = wide[:, 3:-4]
    gate = torch.zeros(n, 4 * DIM + 1, dtype=torch.bfloat16, device=gpu)
    gate[:, 1:] = case["gate"].flatten(1)
    case["gate"] = gate[:, 1:].unflatten(1, (4, DIM))
    pool = torch.randn(4, 6, DIM, DIM, device=gpu)
    case["pool"] = pool[:, 1:5]
    untouched = pool[:, [0, 5]].clone()
    case["log_decay"] = case["log_decay"][None].expand(n, 4)
    check_prefill(case, eps=1e-2, scale=0.3)
    assert torch.equal(pool[:, [0, 5]], untouched)


def test_prefill_shared_row(gpu):
    """One row of activations expanded over the tokens (a row stride of 0)."""
    announce(test="linear_prefill_shared_row")
    case = prefill_case([150], 1, 2, seed=9, device=gpu)
    case["qkv"] = case["qkv"][:1].expand(150, -1)
    check_prefill(case)


def test_prefill_then_decode_equals_longer_prefill(gpu):
    """The two forms of one recurrence: a prompt and then single tokens give what the whole
    prompt gives, within both bounds."""
    announce(test="linear_forms")
    whole = prefill_case([90, 70], 2, 4, seed=15, device=gpu, gated=False)
    whole["cu"] = torch.tensor([0, 90, 160], dtype=torch.int32, device=gpu)
    want = expected_linear_prefill(*[whole[k] for k in PREFILL], SCALE, EPS)
    rows = torch.cat([torch.arange(0, 80), torch.arange(90, 150)]).to(gpu)
    part = dict(whole, qkv=whole["qkv"][rows].contiguous(),
                log_decay=whole["log_decay"][rows].contiguous(),
                cu=torch.tensor([0, 80, 140], dtype=torch.int32, device=gpu),
                out=whole["out"][rows].contiguous())
    run_prefill(part)
    for t in range(10):
        rows = torch.tensor([80 + t, 150 + t], device=gpu)
        step = dict(qkv=whole["qkv"][rows].contiguous(),
                    log_decay=whole["log_decay"][rows].contiguous(),
                    indices=whole["slots"][:, None].contiguous(),
                    cu=torch.tensor([0, 1, 2], dtype=torch.int32, device=gpu),
                    accepted=torch.ones(2, dtype=torch.int32, device=gpu), pool=whole["pool"],
                    gate=None, weight=None, out=whole["out"][:2].clone())
        run_decode(step)
        torch.cuda.synchronize()
        within(step["out"], want[0][rows], 2 * want[1][rows], f"token {t}")
    within(whole["pool"], want[2], 2 * want[3], "pool")


# ---- norm_rope -----------------------------------------------------------------------------


def rope_case(tokens, q_heads, k_heads, rotary, seed, device, *, extra=2, weights=torch.float32,
              positions=torch.int64, far=100):
    gen = torch.Generator(device=device).manual_seed(seed)
    width = (q_heads + k_heads + extra) * DIM
    return dict(
        qkv=(3 * torch.randn(tokens, width, generator=gen, device=device)).bfloat16(),
        q_weight=(1 + 0.1 * torch.randn(DIM, generator=gen, device=device)).to(weights),
        k_weight=(1 + 0.1 * torch.randn(DIM, generator=gen, device=device)).to(weights),
        positions=torch.randint(0, far, (tokens,), generator=gen, device=device).to(positions),
        inv_freq=10000.0 ** (-torch.arange(0, rotary, 2, device=device) / max(rotary, 1)),
        q_heads=q_heads, k_heads=k_heads)


def check_rope(case, interleaved, eps=EPS):
    want, bound = expected_norm_rope(*case.values(), eps, interleaved)
    torch.ops.lightdelta.norm_rope(*case.values(), eps, interleaved)
    torch.cuda.synchronize()
    within(case["qkv"], want, bound, "qkv")


@pytest.mark.parametrize("tokens", [1, 3, 130])
@pytest.mark.parametrize("heads", [(4, 4), (5, 1), (1, 0), (0, 2), (32, 8)])
@pytest.mark.parametrize("rotary", [0, 16, 64, 96, 128])
@pytest.mark.parametrize("interleaved", [False, True])
def test_norm_rope(gpu, tokens, heads, rotary, interleaved):
    announce(test="norm_rope", tokens=tokens, heads=heads, rotary=rotary, interleaved=interleaved)
    check_rope(rope_case(tokens, *heads, rotary, seed=rotary + tokens, device=gpu), interleaved)


@pytest.mark.parametrize("rotary", [2, 6, 50])
def test_norm_rope_interleaved_odd_widths(gpu, rotary):
    check_rope(rope_case(9, 3, 2, rotary, seed=2, device=gpu), True)


@pytest.mark.parametrize("positions", [torch.int32, torch.int64])
@pytest.mark.parametrize("weights", [torch.float32, torch.bfloat16])
def test_norm_rope_types_and_far_positions(gpu, positions, weights):
    case = rope_case(77, 4, 2, 128, seed=3, device=gpu, weights=weights, positions=positions,
                     far=2**31 - 1)
    case["positions"][::5] *= -1
    check_rope(case, False, eps=1e-3)


def test_norm_rope_zero_rows_and_strides(gpu):
    """A row of zeros stays zeros; rows at odd elements; a NaN in one head stays there."""
    case = rope_case(6, 3, 2, 64, seed=4, device=gpu, extra=0)
    wide = torch.zeros(6, case["qkv"].shape[1] + 9, dtype=torch.bfloat16, device=gpu)
    wide[:, 5:-4] = case["qkv"]
    case["qkv"] = wide[:, 5:-4]
    case["qkv"][2] = 0
    check_rope(case, False)
    assert case["qkv"][2].abs().sum() == 0 and wide[:, :5].abs().sum() == 0
    case["qkv"][4, DIM + 3] = float("nan")
    others = [h for h in range(5) if h != 1]
    torch.ops.lightdelta.norm_rope(*case.values(), EPS, False)
    torch.cuda.synchronize()
    assert torch.isfinite(case["qkv"].view(6, 5, DIM)[:, others]).all()
    assert torch.isnan(case["qkv"][4, DIM:2 * DIM]).all()


def test_norm_rope_empty(gpu):
    case = rope_case(4, 2, 2, 64, seed=4, device=gpu)
    case.update(qkv=case["qkv"][:0], positions=case["positions"][:0])
    torch.ops.lightdelta.norm_rope(*case.values(), EPS, False)
