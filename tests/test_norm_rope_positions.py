"""norm_rope's angles at any position, int64 ones far past what a double's product holds, and their
sines and cosines."""

from __future__ import annotations

import pytest
import torch

from oracle.linear import exact_angles, expected_norm_rope
from tests.test_linear_gpu import EPS, check_rope, rope_case, within

FAR = [2**31 - 1, -(2**31), 2**32, 2**35 + 3, 2**40 + 12345, -(2**45) - 1, 2**53 + 1,
       2**62 + 987654321, 2**63 - 1, -(2**63)]


def test_angles_are_exact():
    """At positions whose products doubles hold the two forms agree; far angles add up."""
    gen = torch.Generator().manual_seed(1)
    inv_freq = 10000.0 ** (-torch.arange(0, 128, 2) / 128)
    near = torch.randint(-(2**29) + 1, 2**29, (20,), generator=gen)
    simple = exact_angles(near, inv_freq)
    whole = exact_angles(torch.cat([near, torch.tensor([2**40])]), inv_freq)[:-1]
    for of in (torch.sin, torch.cos):
        # (the products are exact, an angle below a turn is rounded by 2^-51)
        torch.testing.assert_close(of(simple), of(whole), rtol=0, atol=2.0**-49)
    far = torch.tensor(FAR[2:-3])
    one, two = exact_angles(far, inv_freq), exact_angles(2 * far, inv_freq)
    torch.testing.assert_close(torch.sin(2 * one), torch.sin(two), rtol=0, atol=2.0**-48)


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rotary", [16, 96, 128])
def test_far_positions(gpu, interleaved, rotary):
    case = rope_case(len(FAR), 3, 2, rotary, seed=6, device=gpu)
    case["positions"] = torch.tensor(FAR, device=gpu)
    check_rope(case, interleaved)


@pytest.mark.gpu
@pytest.mark.parametrize("frequency", [1.0, 0.7310585975646973, 2.0**-20, 100.0, -0.3])
def test_far_positions_of_one_frequency(gpu, frequency):
    """Also above 1, where the error of the reduction grows with the frequency to 2^-37 of a turn."""
    case = rope_case(400, 1, 1, 128, seed=7, device=gpu, far=2**62)
    case["inv_freq"].fill_(frequency)
    case["positions"][::2] *= -1
    check_rope(case, False)


@pytest.mark.gpu
def test_far_positions_int32(gpu):
    case = rope_case(400, 1, 1, 64, seed=8, device=gpu, far=2**31 - 1)
    case["positions"][::2] *= -1
    check_rope(dict(case, positions=case["positions"].int()), True)


@pytest.mark.gpu
@pytest.mark.parametrize("zeros", ["first", "second"])
def test_small_sines_and_cosines(gpu, zeros):
    """Where one element of a pair is 0 the other's sine or cosine alone is what an output holds, and
    a small one shows its error: that of an fp32 fraction of a turn (2^-26 of one, 2^-23.3 of the
    element), and some roundings of the value itself, far below bf16's."""
    case = rope_case(32768, 1, 1, 128, seed=9, device=gpu, extra=0, far=2**20)
    x = case["qkv"].view(-1, 2, 2, 64)
    x.copy_(torch.where(x < 0, -1.0, 1.0))
    x[:, :, 0 if zeros == "first" else 1] = 0
    case["q_weight"].fill_(1.0)
    case["k_weight"].fill_(1.0)
    want, _ = expected_norm_rope(*case.values(), EPS, False)
    torch.ops.lightdelta.norm_rope(*case.values(), EPS, False)
    torch.cuda.synchronize()
    assert (want.abs() < 2.0**-13).sum() > 100
    within(case["qkv"], want, want.abs() * (2.0**-8 + 2.0**-20) + 2**0.5 * 2.0**-23, "qkv")
