"""attention_decode and attention_prefill on scores, scales and values over all of fp32's range, with
inputs whose scores are exact in 32 bits, so that the softmax is known far more closely than a bound
on the scores' own errors would say."""

from __future__ import annotations

import pytest
import torch

from oracle import attention as oracle
from tests.test_attention_gpu import CACHE, DIM, announce, attend, case_of, within

pytestmark = pytest.mark.gpu

PAGE = 32


def call_case(device, width, *, seed=21):
    """Requests of several tiles, tokens in one or split over workgroups; page scales of 1."""
    lengths, new = ([700, 70, 1], [200, 5, 1]) if width is None else ([700, 70, 1], [2, 2, 1])
    case = case_of(lengths, new, PAGE, (4, 2), seed=seed, device=device, front=1, behind=1)
    for x in ("k_scale", "v_scale"):
        case[x].view(torch.uint8).fill_(127)
    return case


def long_case(device, seed=22):
    """A few rows behind a long context, whose tokens prefill too splits over workgroups."""
    case = case_of([3000], [3], PAGE, (4, 2), seed=seed, device=device)
    for x in ("k_scale", "v_scale"):
        case[x].view(torch.uint8).fill_(127)
    return case


def cases(device, width):
    return [call_case(device, width), long_case(device)]


def set_keys(case, element, values):
    """Element `element` of every key of the cache, to values that e4m3 holds; `values` takes a count
    and gives as many."""
    k = case["k_cache"].view(torch.uint8)
    count, heads, _, page, _ = k.shape
    x = values(count * heads * page).view(count, heads, page)
    code = x.to(torch.float8_e4m3fn)
    assert torch.equal(code.float(), x)
    k[:, :, element // 16, :, element % 16] = code.to(k.device).view(torch.uint8)


def check_exact_scores(case, width, scale, label):
    """The definition's outputs, with scores that are exact: weights are then good to 2^-12 (exponents
    moved by a maximum of up to 2^10 in them, rounded at 2^-14, twice; exp2 far below), rounded to bf16
    (2^-8), as is the output; the sums of n weights and of n products, in 32 bits, are off by n 2^-24."""
    args = (case["q"], *(case[x] for x in CACHE), case["gate"], case["out"], scale, width)
    want, _ = oracle.expected_attention(*args)
    values = case["v_cache"]
    magnitudes = dict(case, v_cache=(values.view(torch.uint8) & 127).view(torch.float8_e4m3fn))
    big, _ = oracle.expected_attention(case["q"], *(magnitudes[x] for x in CACHE), None,
                                       torch.zeros_like(case["out"]), scale, width)
    attend(case, width, scale)
    torch.cuda.synchronize()
    tokens = int(case["lengths"].max())
    error = big * (2.0**-8 + 2.0**-12 + 2 * tokens * 2.0**-24)
    within(case["out"], want, error + 2.0**-8 * (want.abs() + error), label)


@pytest.mark.parametrize("width", [None, 4])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("power", [0, 8, 11, 16, 20])
def test_small_differences_of_large_scores(gpu, power, sign, width):
    """All scores about sign * 2^power, a few units apart."""
    announce(test="score_differences", power=power, sign=sign, width=width)
    gen = torch.Generator().manual_seed(power)
    for case in cases(gpu, width):
        case["q"] = torch.zeros_like(case["q"])
        case["q"][..., 0], case["q"][..., 17] = sign * 2.0**power, 1.0
        set_keys(case, 0, torch.ones)
        set_keys(case, 17, lambda n: torch.randint(-8, 9, (n,), generator=gen) / 2)
        check_exact_scores(case, width, 1.0, f"scores of 2^{power}")


@pytest.mark.parametrize("width", [None, 4])
@pytest.mark.parametrize("power,scale", [(6, 1.0), (24, 1.0), (33, 1.0), (60, 0.125), (117, 1.0),
                                         (117, 2.0**20), (0, 2.0**90), (-60, 2.0**100)])
def test_largest_score_takes_all(gpu, power, scale, width):
    """Scores far apart: the mean of the values whose keys tie for the largest that the row sees."""
    announce(test="score_range", power=power, scale=scale, width=width)
    gen = torch.Generator().manual_seed(3)
    for case in cases(gpu, width):
        case["q"] = torch.zeros_like(case["q"])
        case["q"][..., 5] = 2.0**power
        case["q"][:, 1::2, 5] *= -1
        set_keys(case, 5, lambda n: (torch.randint(-14, 15, (n,), generator=gen) * 32.0))
        check_exact_scores(case, width, scale, f"scores of 2^{power}")


@pytest.mark.parametrize("width", [None, 4])
def test_largest_scale(gpu, width):
    """Scales up to 2.3e38: equal scores give the mean of the values, others the largest's."""
    announce(test="score_scale", width=width)
    gen = torch.Generator().manual_seed(4)
    for case in cases(gpu, width):
        for power in (None, -8, -60):
            case["q"] = torch.zeros_like(case["q"])
            if power is not None:
                case["q"][..., 5] = 2.0**power
            set_keys(case, 5, lambda n: torch.randint(-14, 15, (n,), generator=gen) * 32.0)
            check_exact_scores(case, width, 2.3e38, f"scores of 2^{power}")


@pytest.mark.parametrize("width", [None, 4])
@pytest.mark.parametrize("exponent", [119, 100, 0, -60, -100])
@pytest.mark.parametrize("power", [None, 0, 20])
def test_values_of_any_size(gpu, power, exponent, width):
    """Values up to the largest that the cache holds, whose mean is finite and whose sum is not, and
    down to the smallest; queries of zero, scores a few units apart, and the largest last."""
    announce(test="value_range", power=power, exponent=exponent, width=width)
    gen = torch.Generator().manual_seed(5)
    for case in cases(gpu, width):
        case["v_scale"].view(torch.uint8).fill_(127 + exponent)
        values = case["v_cache"].view(torch.uint8)
        values[:, :, :, 40:60] = 0x7E
        values[:, :, :, 60:80] = 0xFE
        case["q"] = torch.zeros_like(case["q"])
        if power is not None:
            case["q"][..., 0], case["q"][..., 17] = 2.0**power, 1.0
        set_keys(case, 0, torch.ones)
        set_keys(case, 17, lambda n: torch.randint(-8, 9, (n,), generator=gen) / 2)
        check_exact_scores(case, width, 1.0, f"values of 2^{exponent}")


def test_weights_of_decode(gpu):
    """Decode's weights are two bf16 each: about equal ones times 1 and -1, whose sum is small beside
    them.  A weight is off by 2^-17 as it is held, by 2^-18 from its exponent (near 24, rounded twice
    at 2^-20) and by 2^-21 from exp2; two sums of 129 at the most by 2^-16: together below 2^-15 of
    the sum of weights."""
    announce(test="decode_weights")
    gen = torch.Generator().manual_seed(6)
    case = case_of([2, 18, 70, 129], [1, 2, 2, 2], PAGE, (4, 2), seed=23, device=gpu)
    for x in ("k_scale", "v_scale"):
        case[x].view(torch.uint8).fill_(127)
    values = case["v_cache"].view(torch.uint8)
    values[..., 0::2], values[..., 1::2] = 0x38, 0xB8
    case["q"] = torch.zeros_like(case["q"])
    case["q"][..., 17] = 2.0**-6
    set_keys(case, 17, lambda n: torch.randint(-8, 9, (n,), generator=gen) / 2)
    want, _ = oracle.expected_attention(case["q"], *(case[x] for x in CACHE), None, case["out"], 1.0, 2)
    attend(case, 2, 1.0)
    torch.cuda.synchronize()
    within(case["out"], want, 2.0**-15 + 2.0**-8 * (want.abs() + 2.0**-15), "out")
