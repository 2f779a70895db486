"""The linear-attention operators without a GPU: the oracle against closed forms, the ops' checks
of arguments (on the meta device), and the C ABI's declarations and refusals."""

from __future__ import annotations

import ctypes
import re
from pathlib import Path

import pytest
import torch

from lightdelta_amd import _lib, ops
from oracle.linear import expected_linear_decode, expected_linear_prefill, expected_norm_rope

DIM = 128
HEADER = Path(__file__).resolve().parents[1] / "include" / "lightdelta_linear_hip.h"


# ---- the oracle ----------------------------------------------------------------------------


def tiny(tokens, heads, v_heads, slots, seed):
    gen = torch.Generator().manual_seed(seed)
    cols = (2 * heads + v_heads) * DIM
    return dict(qkv=torch.randn(tokens, cols, generator=gen).bfloat16(),
                log_decay=-torch.rand(tokens, v_heads, generator=gen),
                pool=torch.randn(slots, v_heads, DIM, DIM, generator=gen),
                out=torch.zeros(tokens, v_heads, DIM, dtype=torch.bfloat16))


def test_oracle_prefill_is_the_sum_over_pairs():
    """o_t = scale * (e^(c_t) S0 q_t + sum over s <= t of e^(c_t - c_s) (k_s . q_t) v_s)."""
    c = tiny(7, 1, 2, 3, 0)
    out, _, pool, _ = expected_linear_prefill(
        c["qkv"], c["log_decay"], torch.tensor([2]), torch.tensor([True]), torch.tensor([0, 7]),
        c["pool"], None, None, c["out"], 0.5, 1e-6)
    x = c["qkv"].double().view(7, 4, DIM)
    total = c["log_decay"].double().cumsum(0)
    for h in range(2):
        s0 = c["pool"][2, h].double()
        between = (total[:, None, h] - total[None, :, h]).exp().tril()
        o = ((x[:, 0] @ x[:, 1].T) * between) @ x[:, 2 + h]
        o = 0.5 * (o + total[:, h, None].exp() * (x[:, 0] @ s0.T))
        torch.testing.assert_close(out[:, h], o, rtol=1e-12, atol=1e-12)
        left = (total[-1, h] - total[:, h]).exp()
        s = total[-1, h].exp() * s0 + (x[:, 2 + h] * left[:, None]).T @ x[:, 1]
        torch.testing.assert_close(pool[2, h], s, rtol=1e-12, atol=1e-12)


def test_oracle_decode_steps_are_a_prefill():
    c = tiny(3, 1, 1, 5, 1)
    one = expected_linear_prefill(c["qkv"], c["log_decay"], torch.tensor([4]), torch.tensor([True]),
                                  torch.tensor([0, 3]), c["pool"], None, None, c["out"], 1.0, 1e-6)
    step = expected_linear_decode(c["qkv"], c["log_decay"], torch.tensor([[4, 1, 2]]),
                                  torch.tensor([0, 3]), torch.tensor([1]), c["pool"], None, None,
                                  c["out"], 1.0, 1e-6)
    assert torch.equal(one[0], step[0]) and torch.equal(one[2][4], step[2][2])


def test_oracle_rotation_keeps_lengths_and_differences():
    """Rotations keep a head's length, and q . k depends on the positions' difference alone."""
    gen = torch.Generator().manual_seed(2)
    row = torch.randn(1, 2 * DIM, generator=gen).bfloat16().expand(4, -1).contiguous()
    inv_freq = 10000.0 ** (-torch.arange(0, DIM, 2) / DIM)
    ones = torch.ones(DIM)
    for interleaved in (False, True):
        near, _ = expected_norm_rope(row, ones, ones, torch.tensor([0, 3, 7, 9]), inv_freq, 1, 1,
                                     1e-6, interleaved)
        far, _ = expected_norm_rope(row, ones, ones, torch.tensor([0, 3, 7, 9]) + 10**6, inv_freq,
                                    1, 1, 1e-6, interleaved)
        length = near[:, :DIM].square().sum(1)
        torch.testing.assert_close(length, length[:1].expand(4), rtol=1e-12, atol=0)
        products = [x[:, :DIM] @ x[:, DIM:].T for x in (near, far)]
        torch.testing.assert_close(*products, rtol=1e-8, atol=1e-8)


# ---- argument checks -----------------------------------------------------------------------


@pytest.fixture
def meta(monkeypatch):
    monkeypatch.setattr(ops, "_is_gpu", lambda t: t.device.type == "meta")
    return torch.device("meta")


def base(device, n, h, hv):
    def t(*shape, dtype=torch.bfloat16):
        return torch.empty(*shape, dtype=dtype, device=device)

    return t, dict(qkv=t(n, (2 * h + hv) * DIM), log_decay=t(hv, dtype=torch.float32),
                   state=t(10, hv, DIM, DIM, dtype=torch.float32), gate=t(n, hv, DIM),
                   weight=t(DIM), out=t(n, hv, DIM), scale=0.1, eps=1e-6)


def decode_args(device, n=4, h=2, hv=4, width=1):
    t, a = base(device, n, h, hv)
    a.update(indices=t(n // width, width, dtype=torch.int32),
             cu=t(n // width + 1, dtype=torch.int32), accepted=t(n // width, dtype=torch.int32))
    return a


def prefill_args(device, n=9, h=2, hv=4, sequences=3):
    t, a = base(device, n, h, hv)
    a.update(slots=t(sequences, dtype=torch.int32), has_initial=t(sequences, dtype=torch.bool),
             cu_seqlens=t(sequences + 1, dtype=torch.int32))
    return a


def rope_args(device, n=5, q_heads=4, k_heads=2):
    def t(*shape, dtype=torch.bfloat16):
        return torch.empty(*shape, dtype=dtype, device=device)

    return dict(qkv=t(n, (q_heads + k_heads + 1) * DIM), q_weight=t(DIM), k_weight=t(DIM),
                positions=t(n, dtype=torch.int64), inv_freq=t(32, dtype=torch.float32),
                q_heads=q_heads, k_heads=k_heads, eps=1e-6, interleaved=False)


def f32(m, *shape):
    return torch.empty(*shape, device=m)


def bf16(m, *shape):
    return torch.empty(*shape, dtype=torch.bfloat16, device=m)


def i32(m, *shape):
    return torch.empty(*shape, dtype=torch.int32, device=m)


SHARED = [
    (dict(qkv=lambda m: f32(m, 4, 8 * DIM)), "qkv must be CUDA BF16"),
    (dict(qkv=lambda m: bf16(m, 4, 8 * DIM + 1)), r"qkv must be \[tokens"),
    (dict(qkv=lambda m: bf16(m, 4, 7 * DIM)), r"qkv must be \[tokens"),
    (dict(qkv=lambda m: bf16(m, 8 * DIM, 4).T), r"qkv must be \[tokens"),
    (dict(state=lambda m: bf16(m, 10, 4, DIM, DIM)), "state must be CUDA FP32"),
    (dict(state=lambda m: f32(m, 10, 4, 64, DIM)), "state must be CUDA FP32"),
    (dict(state=lambda m: f32(m, 10, 4, DIM, DIM).transpose(2, 3)), "state must be CUDA FP32"),
    (dict(log_decay=lambda m: f32(m, 3)), "log_decay must be CUDA FP32"),
    (dict(log_decay=lambda m: bf16(m, 4)), "log_decay must be CUDA FP32"),
    (dict(log_decay=lambda m: f32(m, 4, 1)), "log_decay must be CUDA FP32"),
    (dict(log_decay=lambda m: f32(m, 8)[::2]), "log_decay must be CUDA FP32"),
    (dict(out=lambda m: f32(m, 4, 4, DIM)), "out must be contiguous CUDA BF16"),
    (dict(out=lambda m: bf16(m, 4, 4, 2 * DIM)[..., :DIM]), "out must be contiguous CUDA BF16"),
    (dict(gate=lambda m: None), "gate and weight must be given together"),
    (dict(weight=lambda m: None), "gate and weight must be given together"),
    (dict(gate=lambda m: bf16(m, 4, 4, 64)), "gate must be CUDA BF16"),
    (dict(weight=lambda m: bf16(m, 64)), "weight must be contiguous"),
    (dict(state=lambda m: torch.zeros(10, 4, DIM, DIM)), "state must be CUDA FP32"),
    (dict(log_decay=lambda m: torch.zeros(4)), "log_decay must be CUDA FP32"),
    (dict(out=lambda m: torch.zeros(4, 4, DIM, dtype=torch.bfloat16)), "out must be contiguous CUDA"),
    (dict(weight=lambda m: torch.zeros(DIM)), "weight must be contiguous CUDA"),
    (dict(scale=lambda m: float("nan")), "scale must be finite"),
    (dict(scale=lambda m: 1e39), "scale must be finite"),
    (dict(eps=lambda m: 0.0), "epsilon must be positive"),
]
DECODE_ONLY = [
    (dict(indices=lambda m: i32(m, 4, 5)), "1 through 4 tokens"),
    (dict(indices=lambda m: torch.empty(4, 1, dtype=torch.int64, device=m)), "metadata must be"),
    (dict(cu=lambda m: i32(m, 4)), "invalid request metadata shapes"),
    (dict(accepted=lambda m: i32(m, 8)[::2]), "metadata must be"),
    (dict(indices=lambda m: torch.zeros(4, 1, dtype=torch.int32)), "metadata must be"),
]
PREFILL_ONLY = [
    (dict(slots=lambda m: i32(m, 3, 1)), "metadata must be"),
    (dict(has_initial=lambda m: i32(m, 3)), "has_initial must be"),
    (dict(cu_seqlens=lambda m: i32(m, 3)), "invalid sequence metadata shapes"),
    (dict(slots=lambda m: torch.zeros(3, dtype=torch.int32)), "metadata must be"),
]
ROPE = [
    (dict(qkv=lambda m: f32(m, 5, 7 * DIM)), "qkv must be CUDA BF16"),
    (dict(qkv=lambda m: bf16(m, 5, 5 * DIM)), r"qkv must be \[tokens"),
    (dict(qkv=lambda m: bf16(m, 1, 7 * DIM).expand(5, -1)), "rows must not overlap"),
    (dict(q_heads=lambda m: -1), r"qkv must be \[tokens"),
    (dict(q_weight=lambda m: bf16(m, 64)), "weights must be contiguous"),
    (dict(positions=lambda m: f32(m, 5)), "positions must be"),
    (dict(positions=lambda m: i32(m, 4)), "positions must be"),
    (dict(inv_freq=lambda m: f32(m, 65)), "inv_freq must be"),
    (dict(inv_freq=lambda m: f32(m, 12)), "inv_freq must be"),
    (dict(eps=lambda m: -1.0), "epsilon must be positive"),
    (dict(positions=lambda m: torch.zeros(5, dtype=torch.int64)), "positions must be"),
    (dict(inv_freq=lambda m: torch.zeros(32)), "inv_freq must be"),
]
KINDS = {
    "linear_decode": (decode_args, ops.check_linear_decode, SHARED + DECODE_ONLY),
    "linear_prefill": (lambda m: prefill_args(m, n=4), ops.check_linear_prefill,
                       SHARED + PREFILL_ONLY),
    "norm_rope": (rope_args, ops.check_norm_rope, ROPE),
}
CASES = [(name, i) for name, (_, _, cases) in KINDS.items() for i in range(len(cases))]


@pytest.mark.parametrize("name", KINDS)
def test_accepts(meta, name):
    make, check, _ = KINDS[name]
    args = make(meta)
    check(**args)
    if name != "norm_rope":
        n, hv = args["out"].shape[:2]
        check(**dict(args, gate=None, weight=None, log_decay=f32(meta, n, hv)))
        check(**dict(args, log_decay=f32(meta, hv).expand(n, hv)))
    else:
        check(**dict(args, inv_freq=f32(meta, 0)))
        check(**dict(args, inv_freq=f32(meta, 5), interleaved=True))


@pytest.mark.parametrize("name,i", CASES)
def test_refusals(meta, name, i):
    make, check, cases = KINDS[name]
    change, message = cases[i]
    with pytest.raises(RuntimeError, match=message):
        check(**dict(make(meta), **{k: f(meta) for k, f in change.items()}))


@pytest.mark.gpu
@pytest.mark.parametrize("name,i", CASES)
def test_kernel_refusals(gpu, name, i):
    """The same by the ops' own kernels; zeros as metadata, so that nothing is launched that
    reads or writes a state."""
    make, _, cases = KINDS[name]
    change, message = cases[i]
    args = {k: torch.zeros_like(v) if isinstance(v, torch.Tensor) else v
            for k, v in make(gpu).items()}
    for k, f in change.items():
        v = f(gpu)
        args[k] = v.zero_() if isinstance(v, torch.Tensor) and v.stride(0) != 0 else v
    with pytest.raises(RuntimeError, match=message):
        order = re.findall(r"(\w+)[,)]", ops.SCHEMAS[name])
        getattr(torch.ops.lightdelta, name)(*[args[k] for k in order])


# ---- the C ABI -----------------------------------------------------------------------------


def test_header_and_binding_agree():
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    declared = set(re.findall(r"^\s*(?:const\s+)?\w+\s*\*?\s*(ld_\w+)\s*\(", text, flags=re.M))
    assert declared == set(_lib.LINEAR_SIGNATURES)
    for struct, mirror in (("ld_linear_decode_args", _lib.LinearDecodeArgs),
                           ("ld_linear_prefill_args", _lib.LinearPrefillArgs),
                           ("ld_norm_rope_args", _lib.NormRopeArgs)):
        body = re.search(r"typedef struct " + struct + r" \{(.*?)\}", text, flags=re.S).group(1)
        assert re.findall(r"(\w+);", body) == [name for name, _ in mirror._fields_]


def refused(call, args, message):
    assert call(ctypes.byref(args), None) == 1
    assert message in _lib.load().ld_last_error().decode()


def test_c_abi_refuses_without_launching():
    lib = _lib.load()
    for call in (lib.ld_linear_decode, lib.ld_linear_prefill, lib.ld_norm_rope):
        assert call(None, None) == 1 and b"args is NULL" in lib.ld_last_error()
    d = _lib.LinearDecodeArgs(num_requests=1, width=5, num_k_heads=2, num_v_heads=4, eps=1e-6)
    refused(lib.ld_linear_decode, d, "1 through 4 tokens")
    d.width, d.num_v_heads = 1, 5
    refused(lib.ld_linear_decode, d, "multiple of num_k_heads")
    d.num_v_heads, d.eps = 4, 0.0
    refused(lib.ld_linear_decode, d, "epsilon must be positive")
    d.eps, d.gate = 1e-6, 16
    refused(lib.ld_linear_decode, d, "given together")
    d.gate, d.state = None, 8
    refused(lib.ld_linear_decode, d, "16-byte aligned")
    d.state = 16
    refused(lib.ld_linear_decode, d, "NULL tensor pointer")
    d.cache_policy = 3
    refused(lib.ld_linear_decode, d, "cache_policy")
    d.cache_policy, d.num_requests = 0, -1
    refused(lib.ld_linear_decode, d, "num_requests")
    d.num_requests = 0
    assert lib.ld_linear_decode(ctypes.byref(d), None) == 0

    p = _lib.LinearPrefillArgs(num_sequences=1, num_k_heads=2, num_v_heads=3, eps=1e-6)
    refused(lib.ld_linear_prefill, p, "multiple of num_k_heads")
    p.num_v_heads = 4
    refused(lib.ld_linear_prefill, p, "NULL tensor pointer")
    p.num_tokens = -1
    refused(lib.ld_linear_prefill, p, "num_tokens")
    p.num_tokens, p.num_sequences = 0, 0
    assert lib.ld_linear_prefill(ctypes.byref(p), None) == 0

    r = _lib.NormRopeArgs(num_tokens=1, q_heads=1, k_heads=1, eps=1e-6, rotary=24)
    refused(lib.ld_norm_rope, r, "multiple of 16")
    r.interleaved, r.rotary = 1, 130
    refused(lib.ld_norm_rope, r, "at most 128")
    r.rotary = 24
    refused(lib.ld_norm_rope, r, "NULL tensor pointer")
    r.q_heads = 1 << 21
    refused(lib.ld_norm_rope, r, "too many heads")
    r.q_heads, r.k_heads = 0, 0
    assert lib.ld_norm_rope(ctypes.byref(r), None) == 0


def test_c_abi_prefill_limits():
    """A prefill's own refusals, all ahead of any launch: row strides past what a chunk's offsets
    hold, tokens and tiles past what a grid does, and a missing, short or misaligned workspace."""
    lib = _lib.load()
    good = dict(qkv=16, qkv_row_stride=1024, log_decay=16, slots=16, has_initial=16, cu_seqlens=16,
                state=16, out=16, num_tokens=4096, num_slots=4, num_sequences=1, num_k_heads=2,
                num_v_heads=4, eps=1e-6, workspace=16, workspace_bytes=1 << 40)
    for change, message in [
            (dict(qkv_row_stride=2**23 + 1), "2^23 elements"),
            (dict(qkv_row_stride=-1), "2^23 elements"),
            (dict(log_decay_row_stride=2**23 + 1), "2^23 elements"),
            (dict(gate=16, norm_weight=16, gate_row_stride=2**23 + 1), "2^23 elements"),
            (dict(num_v_heads=2**16 + 2), "2^23 elements"),
            (dict(num_tokens=2**31), "too many tokens"),
            (dict(num_sequences=2**30), "too many (sequence, head) tiles"),
            (dict(workspace=None), "workspace missing or too small"),
            (dict(workspace=8), "workspace missing or too small"),
            (dict(workspace_bytes=lib.ld_linear_prefill_workspace_bytes(4096, 1, 4) - 1),
             "workspace missing or too small"),
            (dict(state_slot_stride=2), "16-byte aligned")]:
        refused(lib.ld_linear_prefill, _lib.LinearPrefillArgs(**dict(good, **change)), message)


@pytest.mark.parametrize("tokens,sequences,heads,segment", [
    (128, 1, 4, 128), (129, 1, 4, 128), (1024, 1, 33, 192), (2048, 1, 32, 256), (3000, 1, 4, 192),
    (256, 2, 4, 512), (512, 2, 4, 512), (513, 2, 4, 256), (4096, 3, 32, 256), (2176, 1, 1, 128),
    (4097, 1, 32, 320), (5000, 3, 32, 320), (2**17, 3, 32, 2**13), (10**6, 9, 48, 93760),
    (2**31 - 1, 1, 1, 2**22)])
def test_prefill_workspace(tokens, sequences, heads, segment):
    """Two states and a decay for each segment of a head but the first: a segment has a 512th of all
    heads' tokens in whole chunks of 64, at least 256 (several sequences of 512 in all are whole,
    one alone may have segments of 128), so that it is 64 MiB and little more at the most."""
    got = _lib.load().ld_linear_prefill_workspace_bytes(tokens, sequences, heads)
    assert got == (tokens - 1) // segment * heads * (2 * DIM * DIM + 4) * 4
    assert got <= 512 * (2 * DIM * DIM + 4) * 4


def test_prefill_workspace_of_nothing():
    call = _lib.load().ld_linear_prefill_workspace_bytes
    assert [call(*a) for a in [(0, 1, 4), (-1, 1, 4), (10, 0, 4), (10, 1, 0), (128, 1, 4),
                                 (2**31, 1, 4)]] == [0] * 6
