"""The largest sizes and numbers that the softmax-attention operators take: what is past them is refused
ahead of any launch (nothing here has memory behind its pointers)."""

from __future__ import annotations

import pytest
import torch

from lightdelta_amd import _lib, ops
from tests.test_attention_cpu import GOOD, attention_args, decode_args, meta, refused  # noqa: F401


@pytest.mark.parametrize("scale", [2.37e38, 3.4e38])
def test_scale_whose_logarithm_is_not_finite(meta, scale):  # noqa: F811
    """log2(e) * scale is what multiplies scores."""
    lib = _lib.load()
    for call in (lib.ld_attention_decode, lib.ld_attention_prefill):
        refused("log2(e) times it finite", call, _lib.PagedCache(**GOOD),
                _lib.AttentionArgs(q=16, out=16, num_q_heads=4, width=1, scale=scale))
    for make, check in ((decode_args, ops.check_attention_decode),
                        (attention_args, ops.check_attention_prefill)):
        check(**dict(make(meta), scale=2.35e38))
        with pytest.raises(RuntimeError, match="log2.e. times it finite"):
            check(**dict(make(meta), scale=scale))


def test_launches_of_too_many_threads():
    """2^32 threads in all of a launch are refused, those of a call's second launch ahead of its first."""
    lib = _lib.load()
    rows = _lib.CacheRows(k=16, v=16, k_row_stride=2**12, v_row_stride=2**12)
    many = _lib.PagedCache(**dict(GOOD, num_tokens=2**25, num_kv_heads=8))  # 2^25 blocks of 128
    for call in (lib.ld_cache_write, lib.ld_cache_read):
        refused("too many pages and heads", call, many, rows)
    args = _lib.AttentionArgs(q=16, out=16, num_q_heads=16, width=1, scale=0.1, workspace=16,
                              workspace_bytes=2**60)
    refused("too many rows and heads", lib.ld_attention_prefill,
            _lib.PagedCache(**dict(GOOD, num_tokens=2**27, num_kv_heads=8)), args)
    # (a join of four columns a workgroup of 512 threads: 2 kv heads of two each)
    refused("too many requests and heads", lib.ld_attention_decode,
            _lib.PagedCache(**dict(GOOD, num_tokens=2**21, num_requests=2**21)), args)


def test_more_requests_than_their_units_are_counted_for():
    """The cache's pages are found by a count of rows / page + 2 * requests, which is held in 32 bits."""
    lib = _lib.load()
    rows = _lib.CacheRows(k=16, v=16, k_row_stride=256, v_row_stride=256)
    many = _lib.PagedCache(**dict(GOOD, num_tokens=1000, num_requests=2**30))
    for call in (lib.ld_cache_write, lib.ld_cache_read):
        refused("too many requests", call, many, rows)
