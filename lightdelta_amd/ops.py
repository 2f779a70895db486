"""`torch.ops.lightdelta.*` on PyTorch-ROCm, backed by the gfx950 HIP library.

The three reference ops keep their schema strings verbatim (reference csrc/register.cpp:5-9)
and are registered for the CUDA dispatch key, under which HIP tensors dispatch on ROCm; the
fake (meta) impls return None like the reference's (python/lightdelta/ops/__init__.py:10-22).
Argument validation raises RuntimeError with the reference's messages
(csrc/gdn_decode.cu:367-403, csrc/state_io.cu:29-49), generalised from the hard-coded
16 k-heads / 48 v-heads / qkv width 10240 to any H, HV with HV % H == 0 (dk = dv = 128).

Additive ops (no reference counterpart):
  copy_state(pool, src, dst)            slot -> slot copy inside one pool (MTP commit,
                                        slot reuse), any dtype, padding slot <= 0 skipped;
                                        a pair that overlaps another (its source another's
                                        destination, its destination another's source or
                                        destination) is rejected and writes nothing
  copy_state_checked(pool, src, dst, rejected)
                                        copy_state that also writes, per pair, 1 to
                                        rejected (int32 [pairs]) if it was rejected for
                                        overlap, else 0 (every entry on every call, so no
                                        clearing is needed; graph-safe)
  zero_slots(pool, slots)               zero whole slots in place (a slot reused by a new
                                        sequence), any dtype, padding slot <= 0 skipped
  decode_conv(mixed_qkv, conv_state, conv_weight, conv_bias, <decode args without qkv>)
                                        causal conv1d (width 4, SiLU, bf16 output) of the
                                        pre-conv activations fused into the decode step;
                                        conv_state [slots, conv_dim, state_len] (any strides,
                                        so vLLM's transposed dim-last view works); 1 to 4
                                        tokens per request, speculative verify with vLLM's
                                        num_accepted_tokens semantics (accepted)
  prefill(qkv, a, b, a_log, dt_bias, slots, has_initial, cu_seqlens, state, gate, weight,
          out, eps)                     the layer's prefill (post-conv activations of several
                                        sequences, cu_seqlens rows each) in one launch: state
                                        from slots[n] if has_initial[n] else zeros, the
                                        decode recurrence token by token, gated RMSNorm
                                        outputs, final state to slots[n]
  gather_slots / scatter_slots          dtype-generic gather_state / scatter_state, for the
                                        bf16 conv-state pool and any dense-inner pool
  packed_plan(slots, cu, accepted, source, valid, indices, destinations)
                                        the packed path's bookkeeping (GDNBackend,
                                        state_io = "packed") in one launch: each request's
                                        source slot and validity, its scratch rows, and the
                                        slots its per-token states go back to
  linear_decode(qkv, log_decay, indices, cu, accepted, state, gate, weight, out, scale, eps)
                                        linear attention with a decay for each head, S <-
                                        exp(g) S + v k^T, o = scale S q, on the same pool and
                                        request metadata as decode (1 to 4 tokens a request);
                                        log_decay fp32 [HV] or [tokens, HV]; with gate and
                                        weight the gated RMSNorm of o, with both None o itself
  linear_prefill(qkv, log_decay, slots, has_initial, cu_seqlens, state, gate, weight, out,
                 scale, eps)            the same for prompts, metadata as prefill's
  norm_rope(qkv, q_weight, k_weight, positions, inv_freq, q_heads, k_heads, eps, interleaved)
                                        RMSNorm of every q and k head with its weight and the
                                        rotation of its first 2 * len(inv_freq) elements by
                                        positions * inv_freq, in place on qkv's first
                                        (q_heads + k_heads) * 128 columns
  norm_rope_axes(qkv, q_weight, k_weight, positions, axes, inv_freq, q_heads, k_heads, eps,
                 interleaved)           the same with positions [axes, tokens] of several axes
                                        (time, height, width); axes int32 [rotary/2] names each
                                        frequency's
  cache_write(k, v, pages, cu, lengths, k_cache, v_cache, k_scale, v_scale)
                                        keys and values of the last tokens of each request into a
                                        paged cache in e4m3, a power of two as the scale of each
                                        page and head (attention_cache allocates one)
  cache_read(pages, cu, lengths, k_cache, v_cache, k_scale, v_scale, k, v)
                                        the values at the same places back in bf16
  attention_decode(q, pages, cu, lengths, k_cache, v_cache, k_scale, v_scale, gate, out, width,
                   scale)               softmax attention of up to `width` (1 to 4) new tokens a
                                        request to all tokens up to their own, over that cache;
                                        gate None, or out times sigmoid(gate)
  attention_prefill(q, pages, cu, lengths, k_cache, v_cache, k_scale, v_scale, gate, out, scale)
                                        the same for any number of new tokens

Every kernel launches on the caller's current stream and reads no device memory on the host,
so it can be captured in a HIP graph.  None allocates, except prefill's chunked form, which
keeps one workspace per device and stream for later eager calls (release_prefill_workspaces
frees them) and gives a call under graph capture a workspace the graph keeps, and
linear_prefill, attention_decode and attention_prefill, which take what workspace they need (for
linear_prefill 64 MiB and little more at most) from torch's allocator for the call.  The kernels of every op but prefill are C++ (csrc/torch_ops.cpp,
liblightdelta_torch.so); the check_* functions below restate their argument checks so they
can run without a GPU.
"""

from __future__ import annotations

import ctypes
import math
import os
from pathlib import Path

import torch

from . import _lib

SCHEMAS = {
    "decode": (
        "decode(Tensor qkv, Tensor a, Tensor b, Tensor a_log, Tensor dt_bias, "
        "Tensor indices, Tensor cu, Tensor accepted, Tensor(s!) state, Tensor gate, "
        "Tensor weight, Tensor(o!) out, float eps) -> ()"
    ),
    "gather_state": "gather_state(Tensor pool, Tensor slots, Tensor valid, Tensor(o!) out) -> ()",
    "scatter_state": "scatter_state(Tensor packed, Tensor slots, Tensor(p!) pool) -> ()",
    "copy_state": "copy_state(Tensor(p!) pool, Tensor src, Tensor dst) -> ()",
    "copy_state_checked": (
        "copy_state_checked(Tensor(p!) pool, Tensor src, Tensor dst, Tensor(r!) rejected) -> ()"
    ),
    "zero_slots": "zero_slots(Tensor(p!) pool, Tensor slots) -> ()",
    "prefill": (
        "prefill(Tensor qkv, Tensor a, Tensor b, Tensor a_log, Tensor dt_bias, Tensor slots, "
        "Tensor has_initial, Tensor cu_seqlens, Tensor(s!) state, Tensor gate, Tensor weight, "
        "Tensor(o!) out, float eps) -> ()"
    ),
    "decode_conv": (
        "decode_conv(Tensor mixed_qkv, Tensor(c!) conv_state, Tensor conv_weight, "
        "Tensor? conv_bias, Tensor a, Tensor b, Tensor a_log, Tensor dt_bias, Tensor indices, "
        "Tensor cu, Tensor accepted, Tensor(s!) state, Tensor gate, Tensor weight, "
        "Tensor(o!) out, float eps) -> ()"
    ),
    "gather_slots": "gather_slots(Tensor pool, Tensor slots, Tensor valid, Tensor(o!) out) -> ()",
    "packed_plan": (
        "packed_plan(Tensor slots, Tensor cu, Tensor accepted, Tensor(s!) source, "
        "Tensor(v!) valid, Tensor(i!) indices, Tensor(d!) destinations) -> ()"
    ),
    "scatter_slots": "scatter_slots(Tensor packed, Tensor slots, Tensor(p!) pool) -> ()",
    "linear_decode": (
        "linear_decode(Tensor qkv, Tensor log_decay, Tensor indices, Tensor cu, Tensor accepted, "
        "Tensor(s!) state, Tensor? gate, Tensor? weight, Tensor(o!) out, float scale, float eps) "
        "-> ()"
    ),
    "linear_prefill": (
        "linear_prefill(Tensor qkv, Tensor log_decay, Tensor slots, Tensor has_initial, "
        "Tensor cu_seqlens, Tensor(s!) state, Tensor? gate, Tensor? weight, Tensor(o!) out, "
        "float scale, float eps) -> ()"
    ),
    "norm_rope": (
        "norm_rope(Tensor(q!) qkv, Tensor q_weight, Tensor k_weight, Tensor positions, "
        "Tensor inv_freq, int q_heads, int k_heads, float eps, bool interleaved) -> ()"
    ),
    "norm_rope_axes": (
        "norm_rope_axes(Tensor(q!) qkv, Tensor q_weight, Tensor k_weight, Tensor positions, "
        "Tensor axes, Tensor inv_freq, int q_heads, int k_heads, float eps, bool interleaved) "
        "-> ()"
    ),
    "cache_write": (
        "cache_write(Tensor k, Tensor v, Tensor pages, Tensor cu, Tensor lengths, "
        "Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor(c!) k_scale, Tensor(d!) v_scale) -> ()"
    ),
    "cache_read": (
        "cache_read(Tensor pages, Tensor cu, Tensor lengths, Tensor k_cache, Tensor v_cache, "
        "Tensor k_scale, Tensor v_scale, Tensor(k!) k, Tensor(v!) v) -> ()"
    ),
    "attention_decode": (
        "attention_decode(Tensor q, Tensor pages, Tensor cu, Tensor lengths, Tensor k_cache, "
        "Tensor v_cache, Tensor k_scale, Tensor v_scale, Tensor? gate, Tensor(o!) out, int width, "
        "float scale) -> ()"
    ),
    "attention_prefill": (
        "attention_prefill(Tensor q, Tensor pages, Tensor cu, Tensor lengths, Tensor k_cache, "
        "Tensor v_cache, Tensor k_scale, Tensor v_scale, Tensor? gate, Tensor(o!) out, "
        "float scale) -> ()"
    ),
}

HEAD_DIM = _lib.HEAD_DIM
_INT32_MAX = 2**31 - 1
QK_SCALE = HEAD_DIM**-0.5  # reference csrc/gdn_decode.cu:417

# State cache policy of the decode kernel (never changes results, only which kernel shape and
# cache hints move the state): "stream" is tuned for working sets far beyond the 256 MB
# Infinity Cache -- a model's many layers between two steps of one layer, the serving regime
# -- and is the default; "keep" for one layer's working set stepped again while it is still
# cached (a single-layer benchmark), where it is ~4% faster and "stream" ~17% slower cold.
# Set with set_state_cache_policy() or the LIGHTDELTA_STATE_CACHE environment variable.
_POLICIES = {"keep": _lib.CACHE_KEEP, "stream": _lib.CACHE_STREAM}


def _policy_from_env() -> int:
    name = os.environ.get("LIGHTDELTA_STATE_CACHE", "stream")
    if name not in _POLICIES:
        raise ValueError(f"LIGHTDELTA_STATE_CACHE={name!r}: the state cache policy must be one of "
                         f"{sorted(_POLICIES)}")
    return _POLICIES[name]


_cache_policy = _policy_from_env()


def set_state_cache_policy(policy: str) -> None:
    global _cache_policy
    if policy not in _POLICIES:
        raise ValueError(f"state cache policy must be one of {sorted(_POLICIES)}")
    _cache_policy = _POLICIES[policy]
    if _TORCH_KERNELS is not None:
        _TORCH_KERNELS.ld_torch_set_cache_policy(_cache_policy)


def state_cache_policy() -> str:
    return next(name for name, code in _POLICIES.items() if code == _cache_policy)

_FLOATS = (torch.float32, torch.bfloat16)


def _require(condition: bool, message: str) -> None:
    if not condition:
        raise RuntimeError(message)


def _is_gpu(t: torch.Tensor) -> bool:
    return t.is_cuda


_BF16, _F32, _I32 = torch.bfloat16, torch.float32, torch.int32

# The calling thread's current device and a device's current stream as plain integers:
# torch's raw accessors where this build has them (torch.cuda.current_stream() builds a Stream
# object, ~2 us per call), the public API otherwise.
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream(device) -> int:
    index = device if isinstance(device, int) else device.index
    if index is None:
        index = _current_device()
    if _raw_stream is not None:
        return _raw_stream(index)
    return torch.cuda.current_stream(index).cuda_stream


class _DeviceGuard:
    """Makes `device` current for the duration of a launch (the reference's CUDAGuard)."""

    __slots__ = ("index", "previous")

    def __init__(self, device):
        index = device if isinstance(device, int) else device.index
        self.index = index if index is not None else _current_device()
        self.previous = None

    def __enter__(self):
        current = _current_device()
        if current != self.index:
            self.previous = current
            torch.cuda.set_device(self.index)

    def __exit__(self, *exc):
        if self.previous is not None:
            torch.cuda.set_device(self.previous)


# ---------------------------------------------------------------------------------------
# decode
# ---------------------------------------------------------------------------------------


def decode_geometry(qkv: torch.Tensor, state: torch.Tensor) -> tuple[int, int]:
    """(H, HV) implied by qkv's width (2*H + HV)*128 and the state's head count."""
    hv = state.shape[1] if state.dim() == 4 else 0
    cols = qkv.shape[1] if qkv.dim() == 2 else 0
    h2 = cols // HEAD_DIM - hv
    h = h2 // 2
    valid = (
        hv > 0
        and cols % HEAD_DIM == 0
        and h2 > 0
        and h2 % 2 == 0
        and hv % h == 0
    )
    return (h, hv) if valid else (0, hv)


def _decode_layout(qkv, a, b, a_log, dt_bias, indices, cu, accepted, state, gate, weight, out,
                   eps):
    """Validation of lightdelta::decode (reference csrc/gdn_decode.cu:366-403), reading each
    tensor property once: returns (H, HV, device index, requests, width) and the row strides
    of qkv, a, b, state and gate, which the launch needs."""
    if not (_is_gpu(qkv) and qkv.dtype is _BF16):
        raise RuntimeError("qkv must be CUDA BF16")
    dev = qkv.get_device()
    for t in (a, b, gate, out):
        if not (t.get_device() == dev and t.dtype is _BF16 and t.dim() > 0 and t.stride(-1) == 1):
            raise RuntimeError("activations must be BF16 with dense rows")
    for t in (a_log, state):
        if not (t.get_device() == dev and t.dtype is _F32 and t.dim() > 0 and t.stride(-1) == 1):
            raise RuntimeError("state and A_log must be CUDA FP32 with dense rows")
    for t in (indices, cu, accepted):
        if not (t.get_device() == dev and t.dtype is _I32 and t.is_contiguous()):
            raise RuntimeError("metadata must be contiguous CUDA int32")
    for t in (dt_bias, weight):
        if not (t.get_device() == dev and t.is_contiguous() and t.dtype in _FLOATS):
            raise RuntimeError("weights must be contiguous FP32/BF16")
    qkv_shape, qkv_stride = qkv.shape, qkv.stride()
    state_shape, state_stride = state.shape, state.stride()
    h, hv = decode_geometry(qkv, state)
    if not (len(qkv_shape) == 2 and h > 0 and qkv_stride[1] == 1):
        raise RuntimeError("qkv must be [tokens,(2*H+HV)*128] with HV a multiple of H")
    if not (len(state_shape) == 4 and state_shape[2] == HEAD_DIM and state_shape[3] == HEAD_DIM
            and state_stride[2] == HEAD_DIM and state_stride[1] == HEAD_DIM * HEAD_DIM):
        raise RuntimeError("state must be [slots,HV,128,128]")
    indices_shape = indices.shape
    if not (len(indices_shape) == 2 and 1 <= indices_shape[1] <= _lib.MAX_TOKENS):
        raise RuntimeError("decode/MTP supports 1 through 4 tokens per request")
    n = qkv_shape[0]
    gate_stride = gate.stride()
    if not (a.shape == (n, hv) and b.shape == (n, hv) and gate.shape == (n, hv, HEAD_DIM)
            and out.shape == (n, hv, HEAD_DIM) and out.is_contiguous()
            and gate_stride[1] == HEAD_DIM):
        raise RuntimeError("invalid activation shape or output layout")
    if not (a_log.numel() == hv and dt_bias.numel() == hv and weight.numel() == HEAD_DIM):
        raise RuntimeError("invalid weight shapes")
    requests = indices_shape[0]
    if not (cu.dim() == 1 and cu.numel() == requests + 1 and accepted.dim() == 1
            and accepted.numel() == requests):
        raise RuntimeError("invalid request metadata shapes")
    if not eps > 0:
        raise RuntimeError("norm epsilon must be positive")
    return (h, hv, dev, requests, indices_shape[1], qkv_stride[0], a.stride(0), b.stride(0),
            state_stride[0], gate_stride[0])


def check_decode(qkv, a, b, a_log, dt_bias, indices, cu, accepted, state, gate, weight, out, eps):
    """Validation of lightdelta::decode (reference csrc/gdn_decode.cu:366-403); returns
    (H, HV)."""
    return _decode_layout(qkv, a, b, a_log, dt_bias, indices, cu, accepted, state, gate, weight,
                          out, eps)[:2]


def check_prefill(qkv, a, b, a_log, dt_bias, slots, has_initial, cu_seqlens, state, gate,
                  weight, out, eps):
    """Validation of prefill: decode's activation, weight and state rules, with per-sequence
    metadata slots [N] int32, has_initial [N] bool and cu_seqlens [N+1] int32."""
    for t in (slots, cu_seqlens):
        _require(
            t.device == qkv.device and t.dtype == torch.int32 and t.dim() == 1
            and t.is_contiguous(),
            "metadata must be contiguous CUDA int32",
        )
    _require(
        has_initial.device == qkv.device and has_initial.dtype == torch.bool
        and has_initial.dim() == 1 and has_initial.is_contiguous(),
        "has_initial must be a contiguous CUDA bool vector",
    )
    _require(
        cu_seqlens.numel() == slots.numel() + 1 and has_initial.numel() == slots.numel(),
        "invalid sequence metadata shapes",
    )
    return check_decode(qkv, a, b, a_log, dt_bias, slots.view(-1, 1), cu_seqlens, slots, state,
                        gate, weight, out, eps)


# Prefill algorithm: "auto" runs chunks in the WY form, of 64 or 32 tokens, for the shapes
# where they are faster (ld_gdn_prefill_auto_chunked gives the chunk length, 0 for none),
# else the token-serial recurrence; "token_serial", "chunked" (64-token chunks) and
# "chunked_32" force one.  Results agree within rounding; the token-serial form reproduces
# the decode kernel bit for bit.
_PREFILL_ALGORITHMS = {"auto": _lib.PREFILL_AUTO, "token_serial": _lib.PREFILL_TOKEN_SERIAL,
                       "chunked": _lib.PREFILL_CHUNKED, "chunked_32": _lib.PREFILL_CHUNKED_32}
_prefill_algorithm = _lib.PREFILL_AUTO


def set_prefill_algorithm(name: str) -> None:
    global _prefill_algorithm
    if name not in _PREFILL_ALGORITHMS:
        raise ValueError(f"prefill algorithm must be one of {sorted(_PREFILL_ALGORITHMS)}")
    _prefill_algorithm = _PREFILL_ALGORITHMS[name]


def prefill_algorithm() -> str:
    return next(k for k, v in _PREFILL_ALGORITHMS.items() if v == _prefill_algorithm)


# Chunked-prefill workspaces of eager calls, one per (device, stream), kept and grown to the
# largest prefill seen (ld_gdn_prefill_workspace_bytes: 115,712 bytes per 64-token chunk and
# v-head, e.g. 2.0 GB for 32 x 1024 tokens at 32 v-heads).  Eager calls on one stream run in
# order, so they can share one; the buffer comes from torch's allocator once instead of on
# every call.  release_prefill_workspaces() drops them.
#
# A call under HIP-graph capture never touches this cache: the graph records the raw pointer
# and writes through it on every replay, so its workspace must stay the graph's for the
# graph's lifetime.  It gets a buffer of its own, allocated during the capture, which torch
# takes from the graph's private memory pool; that memory stays reserved for the graph's
# replays after the tensor is dropped (later allocations of the same capture may reuse it,
# which is stream-ordered after this call), and no eager call, cache growth or release can
# hand it to other tensors while the graph exists.
_workspaces: dict = {}


def _prefill_workspace(device: torch.device, nbytes: int) -> torch.Tensor:
    if torch.cuda.is_current_stream_capturing():
        return torch.empty(nbytes, dtype=torch.uint8, device=device)
    key = (device.index, _stream(device))
    buffer = _workspaces.get(key)
    if buffer is None or buffer.numel() < nbytes:
        _workspaces.pop(key, None)
        buffer = torch.empty(nbytes, dtype=torch.uint8, device=device)
        _workspaces[key] = buffer
    return buffer


def release_prefill_workspaces() -> None:
    """Frees the cached chunked-prefill workspaces of eager calls (the next chunked prefill
    allocates again).  Captured graphs hold workspaces of their own and are unaffected."""
    _workspaces.clear()


def _prefill_impl(qkv, a, b, a_log, dt_bias, slots, has_initial, cu_seqlens, state, gate,
                  weight, out, eps):
    h, hv = check_prefill(qkv, a, b, a_log, dt_bias, slots, has_initial, cu_seqlens, state,
                          gate, weight, out, eps)
    if slots.numel() == 0:
        return
    lib = _lib.load()
    algorithm = _prefill_algorithm
    chunked = algorithm in (_lib.PREFILL_CHUNKED, _lib.PREFILL_CHUNKED_32) or (
        algorithm == _lib.PREFILL_AUTO
        and lib.ld_gdn_prefill_auto_chunked(qkv.shape[0], slots.numel(), hv) != 0)
    workspace = None
    if chunked:
        nbytes = lib.ld_gdn_prefill_workspace_bytes(qkv.shape[0], slots.numel(), hv)
        workspace = _prefill_workspace(qkv.device, nbytes)
    args = _lib.PrefillArgs(
        qkv.data_ptr(), qkv.stride(0), a.data_ptr(), a.stride(0), b.data_ptr(), b.stride(0),
        a_log.data_ptr(), dt_bias.data_ptr(), _dtype_code(dt_bias), _dtype_code(weight),
        slots.data_ptr(), has_initial.data_ptr(), cu_seqlens.data_ptr(), state.data_ptr(),
        state.stride(0), gate.data_ptr(), gate.stride(0), weight.data_ptr(), out.data_ptr(),
        qkv.shape[0], slots.numel(), h, hv, QK_SCALE, eps, algorithm,
        0 if workspace is None else workspace.data_ptr(),
        0 if workspace is None else workspace.numel(),
    )
    with _DeviceGuard(qkv.device):
        _lib.check(lib.ld_gdn_prefill(args, _stream(qkv.device)))


def _dtype_code(t: torch.Tensor) -> int:
    return _lib.DTYPE_BF16 if t.dtype == torch.bfloat16 else _lib.DTYPE_F32


def check_decode_conv(mixed_qkv, conv_state, conv_weight, conv_bias, a, b, a_log, dt_bias,
                      indices, cu, accepted, state, gate, weight, out, eps):
    """Validation of decode_conv: decode's checks on the pre-conv activations, plus the conv
    pool, weight and bias."""
    h, hv = check_decode(mixed_qkv, a, b, a_log, dt_bias, indices, cu, accepted, state, gate,
                         weight, out, eps)
    conv_dim = mixed_qkv.shape[1]
    _require(
        conv_state.device == mixed_qkv.device
        and conv_state.dtype == torch.bfloat16
        and conv_state.dim() == 3
        and conv_state.shape[1] == conv_dim
        and 3 <= conv_state.shape[2] <= 8,
        "conv_state must be CUDA BF16 [slots, conv_dim, 3..8]",
    )
    _require(
        conv_weight.device == mixed_qkv.device
        and conv_weight.dtype == torch.bfloat16
        and tuple(conv_weight.shape) == (conv_dim, 4)
        and conv_weight.is_contiguous()
        and conv_weight.data_ptr() % 8 == 0,
        "conv_weight must be contiguous CUDA BF16 [conv_dim, 4]",
    )
    if conv_bias is not None:
        _require(
            conv_bias.device == mixed_qkv.device
            and conv_bias.dtype == torch.bfloat16
            and conv_bias.numel() == conv_dim
            and conv_bias.is_contiguous(),
            "conv_bias must be contiguous CUDA BF16 [conv_dim]",
        )
    return h, hv


# ---------------------------------------------------------------------------------------
# state-pool copies: the checks of the C++ kernels (csrc/torch_ops.cpp), restated
# ---------------------------------------------------------------------------------------


def _dense_inner(t: torch.Tensor) -> bool:
    """Every dimension after the first is densely packed (row-major)."""
    expected = 1
    for size, stride in zip(reversed(t.shape[1:]), reversed(t.stride()[1:])):
        if size != 1 and stride != expected:
            return False
        expected *= size
    return True


def check_state_layout(pool, slots, packed, *, fp32_4d: bool):
    """The reference's `check` (csrc/state_io.cu:29-41); `fp32_4d=False` drops the fp32 /
    4-D requirement for the dtype-generic ops."""
    if fp32_4d:
        _require(
            _is_gpu(pool)
            and pool.dtype == torch.float32
            and pool.dim() == 4
            and pool.stride(3) == 1
            and pool.stride(2) == pool.shape[3]
            and pool.stride(1) == pool.shape[2] * pool.shape[3],
            "pool must be CUDA FP32 with dense inner dimensions",
        )
    else:
        _require(
            _is_gpu(pool) and pool.dim() >= 1 and _dense_inner(pool),
            "pool must be a CUDA tensor with dense inner dimensions",
        )
    _require(
        slots.device == pool.device and slots.dtype == torch.int32 and slots.dim() == 1,
        "slots must be a CUDA int32 vector",
    )
    _require(
        packed.device == pool.device
        and packed.dtype == pool.dtype
        and packed.dim() == pool.dim()
        and packed.shape[0] == slots.numel()
        and tuple(packed.shape[1:]) == tuple(pool.shape[1:])
        and _dense_inner(packed),
        "invalid packed layout",
    )


def _check_valid(valid, slots, pool):
    _require(
        valid.device == pool.device
        and valid.dtype == torch.bool
        and tuple(valid.shape) == tuple(slots.shape)
        and valid.is_contiguous(),
        "valid must be a CUDA bool vector",
    )


def check_copy(pool, src, dst):
    _require(
        _is_gpu(pool) and pool.dim() >= 1 and _dense_inner(pool),
        "pool must be a CUDA tensor with dense inner dimensions",
    )
    for t in (src, dst):
        _require(
            t.device == pool.device and t.dtype == torch.int32 and t.dim() == 1 and t.is_contiguous(),
            "src and dst must be contiguous CUDA int32 vectors",
        )
    _require(src.numel() == dst.numel(), "src and dst must have the same length")


def check_copy_checked(pool, src, dst, rejected):
    check_copy(pool, src, dst)
    _require(
        rejected.device == pool.device and rejected.dtype == torch.int32 and rejected.dim() == 1
        and rejected.is_contiguous() and rejected.numel() == src.numel(),
        "rejected must be a contiguous CUDA int32 vector with one entry per pair",
    )


def check_packed_plan(slots, cu, accepted, source, valid, indices, destinations):
    """Validation of packed_plan: int32 metadata [B, W] / [B + 1] / [B], outputs source [B]
    int32, valid [B] bool, indices [B, W] int32, destinations [B * W] int32, all contiguous
    on one device."""
    _require(
        _is_gpu(slots) and slots.dtype == torch.int32 and slots.dim() == 2
        and slots.is_contiguous() and 1 <= slots.shape[1] <= _lib.MAX_TOKENS,
        "slots must be a contiguous CUDA int32 [batch, 1..4] tensor",
    )
    batch, width = slots.shape
    for t, shape in ((cu, (batch + 1,)), (accepted, (batch,)), (source, (batch,)),
                     (indices, (batch, width)), (destinations, (batch * width,))):
        _require(
            t.device == slots.device and t.dtype == torch.int32 and tuple(t.shape) == shape
            and t.is_contiguous(),
            "packed_plan tensors must be contiguous CUDA int32 of the batch's shapes",
        )
    _require(
        valid.device == slots.device and valid.dtype == torch.bool
        and tuple(valid.shape) == (batch,) and valid.is_contiguous(),
        "valid must be a contiguous CUDA bool vector",
    )


def check_zero(pool, slots):
    _require(
        _is_gpu(pool) and pool.dim() >= 1 and _dense_inner(pool),
        "pool must be a CUDA tensor with dense inner dimensions",
    )
    _require(
        slots.device == pool.device and slots.dtype == torch.int32 and slots.dim() == 1
        and slots.is_contiguous(),
        "slots must be a contiguous CUDA int32 vector",
    )


# ---------------------------------------------------------------------------------------
# linear attention: the checks of the C++ kernels (csrc/torch_ops.cpp), restated
# ---------------------------------------------------------------------------------------


def _linear_layout(qkv, log_decay, state, gate, weight, out, scale, eps):
    """What linear_decode and linear_prefill share; returns (H, HV)."""
    _require(_is_gpu(qkv) and qkv.dtype == torch.bfloat16, "qkv must be CUDA BF16")
    _require(
        state.device == qkv.device and state.dtype == torch.float32 and state.dim() == 4
        and tuple(state.shape[2:]) == (HEAD_DIM, HEAD_DIM)
        and tuple(state.stride()[1:]) == (HEAD_DIM * HEAD_DIM, HEAD_DIM, 1),
        "state must be CUDA FP32 [slots,HV,128,128] with dense heads",
    )
    h, hv = decode_geometry(qkv, state)
    _require(qkv.dim() == 2 and h > 0 and qkv.stride(1) == 1,
             "qkv must be [tokens,(2*H+HV)*128] with HV a multiple of H")
    n = qkv.shape[0]
    _require(
        log_decay.device == qkv.device and log_decay.dtype == torch.float32
        and tuple(log_decay.shape) in ((hv,), (n, hv)) and log_decay.stride(-1) == 1,
        "log_decay must be CUDA FP32 [HV] or [tokens,HV] with dense rows",
    )
    _require(
        out.device == qkv.device and out.dtype == torch.bfloat16
        and tuple(out.shape) == (n, hv, HEAD_DIM) and out.is_contiguous(),
        "out must be contiguous CUDA BF16 [tokens,HV,128]",
    )
    _require((gate is None) == (weight is None), "gate and weight must be given together")
    if gate is not None:
        _require(
            gate.device == qkv.device and gate.dtype == torch.bfloat16
            and tuple(gate.shape) == (n, hv, HEAD_DIM)
            and tuple(gate.stride()[1:]) == (HEAD_DIM, 1),
            "gate must be CUDA BF16 [tokens,HV,128] with dense rows",
        )
        _require(
            weight.device == qkv.device and weight.is_contiguous() and weight.dtype in _FLOATS
            and weight.numel() == HEAD_DIM,
            "weight must be contiguous CUDA FP32/BF16 [128]",
        )
    _require(abs(scale) <= torch.finfo(torch.float32).max, "scale must be finite")
    _require(eps > 0, "norm epsilon must be positive")
    _require(state.shape[0] <= _INT32_MAX and hv <= _INT32_MAX // HEAD_DIM, "state pool too large")
    return h, hv


def check_linear_decode(qkv, log_decay, indices, cu, accepted, state, gate, weight, out, scale,
                        eps):
    """Validation of linear_decode; returns (H, HV)."""
    heads = _linear_layout(qkv, log_decay, state, gate, weight, out, scale, eps)
    for t in (indices, cu, accepted):
        _require(t.device == qkv.device and t.dtype == torch.int32 and t.is_contiguous(),
                 "metadata must be contiguous CUDA int32")
    _require(indices.dim() == 2 and 1 <= indices.shape[1] <= _lib.MAX_TOKENS,
             "decode/MTP supports 1 through 4 tokens per request")
    requests = indices.shape[0]
    _require(tuple(cu.shape) == (requests + 1,) and tuple(accepted.shape) == (requests,)
             and requests <= _INT32_MAX, "invalid request metadata shapes")
    return heads


# Elements between rows, at most, and tokens of ld_linear_prefill (include/lightdelta_linear_hip.h).
LINEAR_PREFILL_MAX_ROW = 1 << 23
LINEAR_PREFILL_MAX_TOKENS = _INT32_MAX


def check_linear_prefill(qkv, log_decay, slots, has_initial, cu_seqlens, state, gate, weight, out,
                         scale, eps):
    """Validation of linear_prefill; returns (H, HV)."""
    heads = _linear_layout(qkv, log_decay, state, gate, weight, out, scale, eps)
    for t in (slots, cu_seqlens):
        _require(t.device == qkv.device and t.dtype == torch.int32 and t.dim() == 1
                 and t.is_contiguous(), "metadata must be contiguous CUDA int32")
    _require(has_initial.device == qkv.device and has_initial.dtype == torch.bool
             and has_initial.dim() == 1 and has_initial.is_contiguous(),
             "has_initial must be a contiguous CUDA bool vector")
    _require(cu_seqlens.numel() == slots.numel() + 1 and has_initial.numel() == slots.numel()
             and slots.numel() <= _INT32_MAX, "invalid sequence metadata shapes")
    if slots.numel() == 0:
        return heads
    rows = [x for x in (qkv, gate, log_decay if log_decay.dim() == 2 else None) if x is not None]
    _require(
        heads[1] <= LINEAR_PREFILL_MAX_ROW // HEAD_DIM
        and (qkv.shape[0] <= 1 or all(x.stride(0) <= LINEAR_PREFILL_MAX_ROW for x in rows)),
        "qkv, log_decay, gate and out rows must be at most 2^23 elements apart",
    )
    _require(qkv.shape[0] <= LINEAR_PREFILL_MAX_TOKENS, "too many tokens")
    return heads


def check_norm_rope(qkv, q_weight, k_weight, positions, inv_freq, q_heads, k_heads, eps,
                    interleaved):
    """Validation of norm_rope."""
    n = _rope_layout(qkv, q_weight, k_weight, inv_freq, q_heads, k_heads, eps, interleaved)
    _require(positions.device == qkv.device and positions.dtype in (torch.int32, torch.int64)
             and tuple(positions.shape) == (n,) and positions.is_contiguous(),
             "positions must be contiguous CUDA int32/int64 [tokens]")


def check_norm_rope_axes(qkv, q_weight, k_weight, positions, axes, inv_freq, q_heads, k_heads, eps,
                         interleaved):
    """Validation of norm_rope_axes."""
    n = _rope_layout(qkv, q_weight, k_weight, inv_freq, q_heads, k_heads, eps, interleaved)
    _require(positions.device == qkv.device and positions.dtype in (torch.int32, torch.int64)
             and positions.dim() == 2 and 1 <= positions.shape[0] <= _INT32_MAX
             and positions.shape[1] == n and (n <= 1 or positions.stride(1) == 1),
             "positions must be CUDA int32/int64 [axes,tokens] with dense rows")
    _require(axes.device == qkv.device and axes.dtype == torch.int32
             and tuple(axes.shape) == tuple(inv_freq.shape) and axes.is_contiguous(),
             "axes must be contiguous CUDA int32 [rotary/2]")


def _rope_layout(qkv, q_weight, k_weight, inv_freq, q_heads, k_heads, eps, interleaved):
    """What norm_rope and norm_rope_axes share; returns the tokens."""
    _require(_is_gpu(qkv) and qkv.dtype == torch.bfloat16, "qkv must be CUDA BF16")
    columns = (q_heads + k_heads) * HEAD_DIM
    _require(q_heads >= 0 and k_heads >= 0 and max(q_heads, k_heads) <= _INT32_MAX // HEAD_DIM
             and qkv.dim() == 2 and qkv.shape[1] >= columns and qkv.stride(1) == 1,
             "qkv must be [tokens,>=(q_heads+k_heads)*128] with dense rows")
    n = qkv.shape[0]
    _require(n <= 1 or qkv.stride(0) >= columns, "qkv rows must not overlap")
    for t in (q_weight, k_weight):
        _require(t.device == qkv.device and t.is_contiguous() and t.dtype in _FLOATS
                 and t.numel() == HEAD_DIM, "weights must be contiguous CUDA FP32/BF16 [128]")
    rotary = 2 * inv_freq.numel()
    _require(inv_freq.device == qkv.device and inv_freq.dtype == torch.float32
             and inv_freq.dim() == 1 and inv_freq.is_contiguous() and rotary <= HEAD_DIM
             and (interleaved or rotary % 16 == 0),
             "inv_freq must be contiguous CUDA FP32 [rotary/2], rotary at most 128 and a "
             "multiple of 16 unless interleaved")
    _require(eps > 0, "norm epsilon must be positive")
    return n


# ---------------------------------------------------------------------------------------
# softmax attention over a paged cache in 8 bits: the checks of the C++ kernels, restated
# ---------------------------------------------------------------------------------------

PAGE_SIZES = (16, 32, 64, 128)
ATTENTION_MAX_HEADS = 1 << 16


def attention_cache(num_pages: int, kv_heads: int, page_size: int = 64, device="cuda"):
    """(k_cache, v_cache, k_scale, v_scale) of a paged cache, all zeros: e4m3
    [pages, kv_heads, 8, page, 16] and [pages, kv_heads, page / 16, 128, 16] (element d of token t
    of a page at [d / 16, t, d % 16], and at [t / 16, d, t % 16]), scales e8m0 [pages, kv_heads].
    Page 0 is padding."""
    _require(page_size in PAGE_SIZES, "page size must be 16, 32, 64 or 128")
    k = torch.zeros(num_pages, kv_heads, 8, page_size, 16, dtype=torch.uint8, device=device)
    v = torch.zeros(num_pages, kv_heads, page_size // 16, HEAD_DIM, 16, dtype=torch.uint8,
                    device=device)
    scales = torch.full((2, num_pages, kv_heads), 127, dtype=torch.uint8, device=device)
    return (k.view(torch.float8_e4m3fn), v.view(torch.float8_e4m3fn),
            *scales.view(torch.float8_e8m0fnu).unbind(0))


def _cache_layout(rows, pages, cu, lengths, k_cache, v_cache, k_scale, v_scale):
    """The cache and its requests, for activations like `rows`; returns the kv heads."""
    device = rows.device
    for t in (k_cache, v_cache):
        _require(t.device == device and t.dtype == torch.float8_e4m3fn and t.dim() == 5
                 and _dense_inner(t) and t.data_ptr() % 16 == 0
                 and (t.shape[0] <= 1 or (t.stride(0) % 16 == 0
                                          and t.stride(0) >= t.shape[1:].numel())),
                 "caches must be CUDA float8_e4m3fn with dense pages, 16-byte aligned")
    count, heads, _, page, _ = k_cache.shape
    _require(page in PAGE_SIZES and tuple(k_cache.shape[2:]) == (8, page, 16)
             and 1 <= heads <= ATTENTION_MAX_HEADS,
             "k_cache must be [pages,kv_heads,8,page,16], page 16, 32, 64 or 128")
    _require(tuple(v_cache.shape) == (count, heads, page // 16, HEAD_DIM, 16),
             "v_cache must be [pages,kv_heads,page/16,128,16]")
    for t in (k_scale, v_scale):
        _require(t.device == device and t.dtype == torch.float8_e8m0fnu
                 and tuple(t.shape) == (count, heads) and _dense_inner(t)
                 and (count <= 1 or t.stride(0) >= heads),
                 "scales must be CUDA float8_e8m0fnu [pages,kv_heads] with dense rows")
    for t in (pages, cu, lengths):
        _require(t.device == device and t.dtype == torch.int32, "metadata must be CUDA int32")
    requests = lengths.numel()
    _require(lengths.dim() == 1 and lengths.is_contiguous() and cu.dim() == 1
             and cu.numel() == requests + 1 and cu.is_contiguous()
             and pages.dim() == 2 and pages.shape[0] == requests
             and (pages.shape[1] <= 1 or pages.stride(1) == 1)
             and max(requests, pages.shape[1], count) <= _INT32_MAX,
             "invalid request metadata shapes")
    return heads


def _cache_rows(k, v, heads):
    for t in (k, v):
        _require(t.device == k.device and t.dtype == torch.bfloat16 and t.dim() == 3
                 and tuple(t.shape) == (k.shape[0], heads, HEAD_DIM) and _dense_inner(t),
                 "k and v must be CUDA BF16 [tokens,kv_heads,128] with dense rows")
    _require(k.shape[0] <= _INT32_MAX, "too many tokens")


def check_cache_write(k, v, pages, cu, lengths, k_cache, v_cache, k_scale, v_scale):
    """Validation of cache_write; returns the kv heads."""
    _require(_is_gpu(k), "k and v must be CUDA BF16 [tokens,kv_heads,128] with dense rows")
    heads = _cache_layout(k, pages, cu, lengths, k_cache, v_cache, k_scale, v_scale)
    _cache_rows(k, v, heads)
    return heads


def check_cache_read(pages, cu, lengths, k_cache, v_cache, k_scale, v_scale, k, v):
    """Validation of cache_read; returns the kv heads."""
    heads = check_cache_write(k, v, pages, cu, lengths, k_cache, v_cache, k_scale, v_scale)
    _require(k.shape[0] <= 1 or min(k.stride(0), v.stride(0)) >= heads * HEAD_DIM,
             "rows of k and v must not overlap")
    return heads


def check_attention_prefill(q, pages, cu, lengths, k_cache, v_cache, k_scale, v_scale, gate, out,
                            scale):
    """Validation of attention_prefill; returns (q heads, kv heads)."""
    _require(_is_gpu(q) and q.dtype == torch.bfloat16 and q.dim() == 3 and q.shape[2] == HEAD_DIM
             and _dense_inner(q), "q must be CUDA BF16 [tokens,q_heads,128] with dense rows")
    heads = _cache_layout(q, pages, cu, lengths, k_cache, v_cache, k_scale, v_scale)
    q_heads = q.shape[1]
    _require(0 < q_heads <= ATTENTION_MAX_HEADS and q_heads % heads == 0,
             "q_heads must be a positive multiple of kv_heads")
    _require(gate is None or (gate.device == q.device and gate.dtype == torch.bfloat16
                              and tuple(gate.shape) == tuple(q.shape) and _dense_inner(gate)),
             "gate must be CUDA BF16 [tokens,q_heads,128] with dense rows")
    _require(out.device == q.device and out.dtype == torch.bfloat16
             and tuple(out.shape) == tuple(q.shape) and out.is_contiguous(),
             "out must be contiguous CUDA BF16 [tokens,q_heads,128]")
    _require(scale > 0 and scale * math.log2(math.e) <= torch.finfo(torch.float32).max,
             "scale must be positive, log2(e) times it finite")
    _require(q.shape[0] <= _INT32_MAX, "too many tokens")
    return q_heads, heads


def check_attention_decode(q, pages, cu, lengths, k_cache, v_cache, k_scale, v_scale, gate, out,
                           width, scale):
    """Validation of attention_decode; returns (q heads, kv heads)."""
    _require(1 <= width <= _lib.MAX_TOKENS, "decode/MTP supports 1 through 4 tokens per request")
    return check_attention_prefill(q, pages, cu, lengths, k_cache, v_cache, k_scale, v_scale, gate,
                                   out, scale)


# ---------------------------------------------------------------------------------------
# registration
# ---------------------------------------------------------------------------------------

# The per-step ops have C++ kernels (csrc/torch_ops.cpp, liblightdelta_torch.so): their host
# path is on every decode step.  prefill's kernel is the Python function below (it keeps the
# chunked form's workspace cache and the algorithm choice).
_CXX_KERNELS = ("decode", "decode_conv", "gather_state", "scatter_state", "gather_slots",
                "scatter_slots", "copy_state", "copy_state_checked", "zero_slots", "packed_plan",
                "linear_decode", "linear_prefill", "norm_rope", "norm_rope_axes", "cache_write",
                "cache_read", "attention_decode", "attention_prefill")
_IMPLS = {
    "prefill": _prefill_impl,
}


def _fake(*args, **kwargs):
    return None


TORCH_KERNELS_PATH = Path(__file__).resolve().with_name("liblightdelta_torch.so")


def _not_built(*args, **kwargs):
    raise RuntimeError(f"{TORCH_KERNELS_PATH.name} is not built; run `python -m "
                       "lightdelta_amd.build` (hipcc, gfx950, and g++ against torch) before "
                       "using the lightdelta ops")


def _register():
    """Defines the ops, registers their fakes and their CUDA-key kernels: the C++ ones by
    loading liblightdelta_torch.so (with its liblightdelta_hip.so), the others from _IMPLS.
    Without the C++ library, decode and decode_conv raise."""
    library = torch.library.Library("lightdelta", "DEF")
    for name, schema in SCHEMAS.items():
        library.define(schema)
        torch.library.register_fake(f"lightdelta::{name}", _fake, lib=library)
        if name in _IMPLS:
            library.impl(name, _IMPLS[name], "CUDA")
    kernels = None
    if TORCH_KERNELS_PATH.exists():
        torch.ops.load_library(str(TORCH_KERNELS_PATH))
        kernels = ctypes.CDLL(str(TORCH_KERNELS_PATH))
        kernels.ld_torch_set_cache_policy.argtypes = [ctypes.c_int]
        kernels.ld_torch_set_cache_policy.restype = ctypes.c_int
        kernels.ld_torch_set_cache_policy(_cache_policy)
    else:
        for name in _CXX_KERNELS:
            library.impl(name, _not_built, "CUDA")
    return library, kernels


_LIBRARY, _TORCH_KERNELS = _register()
