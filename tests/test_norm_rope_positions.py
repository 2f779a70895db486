"""norm_rope's angles at any position: int64 ones far past what a double's product holds."""

from __future__ import annotations

import pytest
import torch

from oracle.linear import exact_angles
from tests.test_linear_gpu import check_rope, rope_case

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
