"""linear_prefill where a mode or a value is what matters: outputs whose every bit is known."""

from __future__ import annotations

import pytest
import torch

from tests.test_linear_gpu import DIM, announce, prefill_case, run_prefill

pytestmark = pytest.mark.gpu


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
