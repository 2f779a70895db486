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
