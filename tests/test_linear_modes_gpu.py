"""linear_prefill where a mode or a value is what matters: outputs whose every bit is known, values
that are not finite, and every mode of a call on sequences that are cut into segments."""

from __future__ import annotations

import pytest
import torch

from tests.test_linear_gpu import DIM, announce, check_prefill, prefill_case, run_prefill

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("has_initial", [False, True])
def test_prefill_of_one_far_row(gpu, has_initial):
    """The last tokens of buffers whose rows are further apart than several rows may be: with one
    row there is no distance to keep."""
    announce(test="linear_prefill_one_row", has_initial=has_initial)
    case = prefill_case([1], 1, 2, seed=8, device=gpu)
    case["has_initial"].fill_(has_initial)
    for name, rows in (("qkv", 2**14 + 1), ("gate", 2**15 + 1), ("log_decay", 2**22 + 1)):
        x = case[name]
        wide = torch.zeros(1, rows, *x.shape[1:], dtype=x.dtype, device=gpu)
        wide[:, -1] = x
        case[name] = wide[:, -1]
        assert case[name].stride(0) > 2**23
    check_prefill(case)


def near_ties(shape, seed, device):
    """fp32 values 1 to 16 units in the last place to either side of the middle between two bf16
    neighbours: 16 bits of them are the middle itself, which rounds to even."""
    gen = torch.Generator().manual_seed(seed)
    bits = torch.randn(shape, generator=gen).bfloat16().view(torch.int16).int() << 16
    away = torch.randint(1, 17, shape, generator=gen) * (2 * torch.randint(0, 2, shape, generator=gen) - 1)
    return (bits + 0x8000 + away.int()).view(torch.float32).to(device)


def bare_case(lengths, v_heads, device):
    """No decay, gate or activations; every prompt starts from its slot."""
    case = prefill_case(lengths, 1, v_heads, seed=1, device=device, gated=False, per_token=False)
    case["qkv"] = torch.zeros_like(case["qkv"]).contiguous()
    case["log_decay"].zero_()
    case["has_initial"].fill_(True)
    return case


@pytest.mark.parametrize("lengths", [[70], [600], [3, 64, 65], [1300, 40]])
def test_prefill_reads_every_bit_of_the_state(gpu, lengths):
    """With unit vectors as q and no update, o is an entry of S: exact in fp32, rounded once."""
    announce(test="linear_prefill_state_bits", lengths=lengths)
    case = bare_case(lengths, 2, gpu)
    case["pool"].copy_(near_ties(case["pool"].shape, 2, gpu))
    tokens = sum(lengths)
    key = (torch.arange(tokens, device=gpu) * 37) % DIM
    case["qkv"][torch.arange(tokens, device=gpu), key] = 1.0
    slot = case["slots"].long().repeat_interleave(torch.tensor(lengths, device=gpu))
    want = case["pool"][slot[:, None], torch.arange(2, device=gpu)[None], :, key[:, None]].bfloat16()
    start = case["pool"].clone()
    run_prefill(case, scale=1.0)
    torch.cuda.synchronize()
    assert torch.equal(case["out"], want)
    assert torch.equal(case["pool"], start)


@pytest.mark.parametrize("lengths", [[64], [37, 64], [100]])
@pytest.mark.parametrize("scale", [1 + 2.0**-8 + 2.0**-20, 1 + 3 * 2.0**-8 - 2.0**-19, 1 / 3])
def test_prefill_reads_every_bit_of_the_scores(gpu, lengths, scale):
    """A chunk's keys are different unit vectors, q is the key of a token up to its own, v powers
    of two: o is scale * v of that token, exact in fp32."""
    announce(test="linear_prefill_score_bits", lengths=lengths, scale=scale)
    scale = torch.tensor(scale, dtype=torch.float32).item()
    case = bare_case(lengths, 2, gpu)
    case["pool"].zero_()
    gen = torch.Generator().manual_seed(3)
    tokens = sum(lengths)
    within = torch.cat([torch.arange(n) for n in lengths])           # its token of the prompt
    first = torch.arange(tokens) - within % 64                       # its chunk's first row
    source = first + (torch.rand(tokens, generator=gen) * (within % 64 + 1)).long()
    rows = torch.arange(tokens)
    case["qkv"][rows.to(gpu), (within[source] % DIM).to(gpu)] = 1.0
    case["qkv"][rows.to(gpu), (DIM + within % DIM).to(gpu)] = 1.0
    v = torch.randint(-3, 4, (tokens, 2, DIM), generator=gen).float().exp2()
    v *= 2 * torch.randint(0, 2, v.shape, generator=gen) - 1
    case["qkv"][:, 2 * DIM:] = v.flatten(1).bfloat16().to(gpu)
    run_prefill(case, scale=scale)
    torch.cuda.synchronize()
    assert torch.equal(case["out"], (v[source] * scale).bfloat16().to(gpu))


@pytest.mark.parametrize("lengths,token", [([130], t) for t in (0, 17, 31, 32, 45, 63, 64, 100, 129)] +
                         [([700, 20], t) for t in (100, 128, 383, 390, 699)])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_prefill_nonfinite_v_goes_forward(gpu, lengths, token, gated, value):
    """One v that is not finite: its column of the outputs from its token on (every column where
    they are normed), its row of the state, and nothing else."""
    announce(test="linear_prefill_nonfinite_v", lengths=lengths, token=token, gated=gated, value=value)
    clean = prefill_case(lengths, 1, 2, seed=21, device=gpu, gated=gated)
    case = {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in clean.items()}
    case["qkv"][token, 2 * DIM + 77] = value
    run_prefill(clean)
    run_prefill(case)
    torch.cuda.synchronize()
    bad = torch.zeros_like(clean["out"], dtype=torch.bool)
    bad[token:lengths[0], 0, slice(None) if gated else 77] = True
    assert not torch.isfinite(case["out"][bad]).any()
    assert torch.equal(case["out"][~bad], clean["out"][~bad])
    bad = torch.zeros_like(clean["pool"], dtype=torch.bool)
    bad[int(clean["slots"][0]), 0, 77] = True
    assert not torch.isfinite(case["pool"][bad]).any()
    assert torch.equal(case["pool"][~bad], clean["pool"][~bad])


@pytest.mark.parametrize("column", [5, DIM + 5, 2 * DIM + 5], ids=["q", "k", "v"])
@pytest.mark.parametrize("tokens", [[20], [40, 50, 41], [3, 3, 70, 129]])
def test_prefill_nonfinite_rows_go_forward(gpu, column, tokens):
    """Several of them in one column, and in all heads at once: earlier tokens keep their bits, and
    behind a q all but its own do."""
    announce(test="linear_prefill_nonfinite_rows", column=column, tokens=tokens)
    clean = prefill_case([130], 1, 2, seed=22, device=gpu, gated=False)
    case = {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in clean.items()}
    for i, token in enumerate(tokens):
        case["qkv"][token, column] = float("-inf" if i % 2 else "nan")
    run_prefill(clean)
    run_prefill(case)
    torch.cuda.synchronize()
    keep = torch.ones(130, dtype=torch.bool, device=gpu)
    if column < DIM:
        keep[tokens] = False
        assert torch.equal(case["pool"], clean["pool"])
    else:
        keep[min(tokens):] = False
    assert torch.equal(case["out"][keep], clean["out"][keep])
    assert not torch.isfinite(case["out"][~keep][:, 0, 5]).any()


@pytest.mark.parametrize("lengths,token", [([130], 45), ([700], 300)])
@pytest.mark.parametrize("odd", [False, True])
def test_prefill_nonfinite_token_goes_forward(gpu, lengths, token, odd):
    """A token of which nothing is finite, also in rows at odd elements."""
    announce(test="linear_prefill_nonfinite_token", lengths=lengths, token=token, odd=odd)
    clean = prefill_case(lengths, 2, 4, seed=23, device=gpu)
    if odd:
        clean["qkv"] = odd_rows(clean["qkv"], gpu)
    case = {k: v.clone() if k in ("pool", "out") else v for k, v in clean.items()}
    run_prefill(clean)
    clean["qkv"][token] = float("nan")
    run_prefill(case)
    torch.cuda.synchronize()
    assert torch.equal(case["out"][:token], clean["out"][:token])
    assert not torch.isfinite(case["out"][token:]).any()
    assert not torch.isfinite(case["pool"][case["slots"].long()]).any()


# ---- segments ------------------------------------------------------------------------------

# Of these the first prompts are cut: into 11 segments of 128 tokens, 6 of 256 (and the last prompt
# into two of 192), 18 of 256 behind a join.
CUT = [([1300], (1, 2)), ([1300, 3, 257], (1, 2)), ([4400], (1, 1))]


def odd_rows(x, device):
    """The same rows at odd elements of wider ones."""
    flat = x.flatten(1)
    wide = torch.zeros(flat.shape[0], flat.shape[1] + 7, dtype=x.dtype, device=device)
    wide[:, 3:-4] = flat
    return wide[:, 3:-4].unflatten(1, x.shape[1:]) if x.dim() == 3 else wide[:, 3:-4]


def cut_case(lengths, heads, device, **kw):
    case = prefill_case(lengths, *heads, seed=31, device=device, decay=0.05, **kw)
    case["has_initial"][0] = True
    return case


@pytest.mark.parametrize("lengths,heads", CUT)
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("odd", [False, True])
def test_cut_prompts_layouts(gpu, lengths, heads, gated, odd):
    """With and without the norm, one constant decay a head, bf16 weight, rows at odd elements."""
    announce(test="linear_prefill_cut_layouts", lengths=lengths, gated=gated, odd=odd)
    case = cut_case(lengths, heads, gpu, gated=gated, per_token=False, weight_dtype=torch.bfloat16)
    if odd:
        case["qkv"] = odd_rows(case["qkv"], gpu)
        if gated:
            case["gate"] = odd_rows(case["gate"], gpu)
    check_prefill(case, eps=1e-3, scale=0.3)


@pytest.mark.parametrize("lengths,heads", CUT)
@pytest.mark.parametrize("slot", [0, -1, 5])
def test_cut_prompts_padding_and_outside_rows(gpu, lengths, heads, slot):
    """A cut prompt whose slot is padding; rows that are not finite ahead of and behind all."""
    announce(test="linear_prefill_cut_padding", lengths=lengths, slot=slot)
    case = cut_case(lengths, heads, gpu, front=7, behind=70)
    case["slots"][0] = slot if slot < 1 else case["pool"].shape[0]
    case["qkv"][:7] = float("nan")
    case["qkv"][-70:] = float("-inf")
    case["gate"][-70:] = float("nan")
    case["log_decay"][:7] = float("nan")
    case["log_decay"][-70:] = float("nan")
    check_prefill(case)
    assert (case["out"][:7] == 7).all() and (case["out"][-70:] == 7).all()


@pytest.mark.parametrize("lengths,heads", CUT)
@pytest.mark.parametrize("value", [float("-inf"), -200.0])
@pytest.mark.parametrize("tokens", [[0, 128, 256, 512], [127, 255, 511], [192, 300], [1299]])
def test_cut_prompts_extreme_decays(gpu, lengths, heads, value, tokens):
    """Tokens that empty the state: a segment's first, its last, one inside, a prompt's last."""
    announce(test="linear_prefill_cut_decays", lengths=lengths, value=value, tokens=tokens)
    case = cut_case(lengths, heads, gpu)
    case["log_decay"][tokens] = value
    case["log_decay"][[t - lengths[-1] for t in tokens if t < lengths[-1]]] = value   # (the last prompt's)
    check_prefill(case)


def test_cut_prompt_far_rows(gpu):
    """One prompt in five segments over rows 16 MiB apart: all but the first start past 2 GiB, the
    last two past 4 GiB."""
    announce(test="linear_prefill_cut_far")
    tokens, apart = 600, 2**23
    case = cut_case([tokens], (1, 2), gpu)
    flat = torch.zeros((tokens - 1) * apart + 6 * DIM, dtype=torch.bfloat16, device=gpu)
    far = flat.as_strided((tokens, 4 * DIM), (apart, 1))
    gate = flat[4 * DIM:].as_strided((tokens, 2, DIM), (apart, DIM, 1))
    far.copy_(case["qkv"])
    gate.copy_(case["gate"])
    case.update(qkv=far, gate=gate)
    check_prefill(case)
