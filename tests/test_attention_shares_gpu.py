"""attention_prefill where tokens are split over workgroups: the join by single groups of threads (more than
64 blocks of columns and kv heads), and plans of more than 64 requests."""

from __future__ import annotations

import pytest

from tests.test_attention_gpu import (
    announce,
    case_of,
    check_attention,
    check_read,
    check_write,
)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("new,heads", [(512, (16, 2)), (600, (20, 5))])
def test_many_blocks_of_one_request(gpu, new, heads, gated):
    """66 and 95 blocks and kv heads, of 7 and 6 shares each."""
    announce(test="shares_blocks", new=new, heads=heads, gated=gated)
    check_attention(case_of([3300], [new], 64, heads, seed=31, device=gpu, gated=gated, front=1,
                            behind=2))


@pytest.mark.parametrize("requests,heads", [(100, (4, 1)), (100, (2, 2)), (200, (1, 1))])
def test_shares_of_many_requests(gpu, requests, heads):
    """Split requests in the first 64, at both sides of its end and in later ones, between short ones
    and empty ones.  The first blocks of request 64 see fewer tiles than it has shares for: some are
    empty."""
    announce(test="shares_requests", requests=requests, heads=heads)
    lengths = [40 + 7 * i % 90 if i % 7 else 0 for i in range(requests)]
    new = [min(n, 1 + i % 3 if i % 5 else 0) for i, n in enumerate(lengths)]
    split = {3: (3000, 30), 63: (2500, 40), 64: (3000, 1900), 70: (5000, 7),
             requests - 1: (2100, 9)}
    for i, (length, rows) in split.items():
        lengths[i], new[i] = length, rows
    check_attention(case_of(lengths, new, 64, heads, seed=32, device=gpu))


def test_thousands_of_requests(gpu):
    """Requests are found by a search of three levels past 4,096 of them."""
    announce(test="thousands")
    lengths = [i % 23 if i % 3 else 0 for i in range(4400)]
    new = [min(n, 1 + i % 2) for i, n in enumerate(lengths)]
    lengths[4200], new[4200] = 70, 40
    case = case_of(lengths, new, 16, (2, 1), seed=33, device=gpu, front=1, behind=3)
    check_write(case)
    check_read(case)
    check_attention(case)
    check_attention(case, width=2)
