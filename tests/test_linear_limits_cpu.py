"""Limits of sizes and strides that the linear-attention ops' checks state, on the meta device."""

from __future__ import annotations

import pytest
import torch

from lightdelta_amd import ops
from tests.test_linear_cpu import DIM, decode_args, f32, i32, meta, prefill_args, rope_args  # noqa: F401


def rows_apart(device, shape, apart, dtype=torch.bfloat16):
    """[tokens, ...] with rows this many elements apart."""
    dense = torch.empty(shape, dtype=dtype, device=device)
    return torch.empty_strided(shape, (apart, *dense.stride()[1:]), dtype=dtype, device=device)


@pytest.mark.parametrize("name,shape,dtype", [
    ("qkv", (8 * DIM,), torch.bfloat16), ("gate", (4, DIM), torch.bfloat16),
    ("log_decay", (4,), torch.float32)])
def test_prefill_row_distance(meta, name, shape, dtype):  # noqa: F811
    for tokens, apart, good in [(2, 2**23, True), (2, 2**23 + 8, False), (1, 2**23 + 8, True)]:
        args = prefill_args(meta, n=tokens)
        args[name] = rows_apart(meta, (tokens, *shape), apart, dtype)
        if good:
            ops.check_linear_prefill(**args)
        else:
            with pytest.raises(RuntimeError, match="at most 2.23 elements apart"):
                ops.check_linear_prefill(**args)


def test_prefill_tokens(meta):  # noqa: F811
    args = prefill_args(meta, n=2**31)
    with pytest.raises(RuntimeError, match="too many tokens"):
        ops.check_linear_prefill(**args)


@pytest.mark.parametrize("make,check", [(decode_args, ops.check_linear_decode),
                                        (prefill_args, ops.check_linear_prefill)])
def test_pool_size(meta, make, check):  # noqa: F811
    args = make(meta)
    check(**dict(args, state=f32(meta, 2**31 - 1, 4, DIM, DIM)))
    with pytest.raises(RuntimeError, match="state pool too large"):
        check(**dict(args, state=f32(meta, 2**31, 4, DIM, DIM)))
    heads = 2**24 + 4
    args = make(meta, h=heads // 4, hv=heads)
    with pytest.raises(RuntimeError, match="state pool too large"):
        check(**args)


def test_metadata_sizes(meta):  # noqa: F811
    many = 2**31
    args = dict(decode_args(meta), indices=i32(meta, many, 1), cu=i32(meta, many + 1),
                accepted=i32(meta, many))
    with pytest.raises(RuntimeError, match="invalid request metadata shapes"):
        ops.check_linear_decode(**args)
    args = prefill_args(meta, sequences=many)
    with pytest.raises(RuntimeError, match="invalid sequence metadata shapes"):
        ops.check_linear_prefill(**args)


def test_rope_heads(meta):  # noqa: F811
    heads = 2**24
    args = dict(rope_args(meta), qkv=torch.empty(5, heads * DIM, dtype=torch.bfloat16, device=meta),
                q_heads=heads, k_heads=0)
    with pytest.raises(RuntimeError, match="qkv must be"):
        ops.check_norm_rope(**args)
