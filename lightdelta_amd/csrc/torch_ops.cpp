// Dispatcher kernels of the lightdelta ops (CUDA key, under which HIP tensors dispatch on
// PyTorch-ROCm): decode and decode_conv with the argument checks of the reference's launcher
// (csrc/gdn_decode.cu:366-403), generalised to any H, HV with HV % H == 0, with its
// messages; the state-pool ops with the checks of the reference's state_io
// (csrc/state_io.cu:29-49) and of the additive ones; the linear-attention ops (linear_decode,
// linear_prefill, norm_rope) and the softmax-attention ones (norm_rope_axes, cache_write,
// cache_read, attention_decode, attention_prefill); then the C ABI of liblightdelta_hip.so on the
// current HIP stream of the tensors' device.  The schemas are defined by lightdelta_amd/ops.py, which
// loads this library (prefill keeps a Python kernel).
// Host-only C++ (no device code): one eager call costs a few microseconds of host time, as
// the reference's C++ launcher does, where a Python kernel costs about twelve.
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/library.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <limits>
#include <optional>

#include "lightdelta_attention_hip.h"
#include "lightdelta_hip.h"
#include "lightdelta_linear_hip.h"

namespace {

constexpr int64_t kDim = LD_HEAD_DIM;

std::atomic<int> g_cache_policy{LD_CACHE_STREAM};

bool floats(const at::Tensor& t) {
  return t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16;
}

int32_t dtype_code(const at::Tensor& t) {
  return t.scalar_type() == at::kBFloat16 ? LD_DTYPE_BF16 : LD_DTYPE_F32;
}

// The decode step's checks (ops.py _decode_layout has the same ones for the Python-side
// callers); returns H, HV.
std::pair<int64_t, int64_t> check_decode(const at::Tensor& qkv, const at::Tensor& a,
                                         const at::Tensor& b, const at::Tensor& a_log,
                                         const at::Tensor& dt_bias, const at::Tensor& indices,
                                         const at::Tensor& cu, const at::Tensor& accepted,
                                         const at::Tensor& state, const at::Tensor& gate,
                                         const at::Tensor& weight, const at::Tensor& out,
                                         double eps) {
  TORCH_CHECK(qkv.is_cuda() && qkv.scalar_type() == at::kBFloat16, "qkv must be CUDA BF16");
  const c10::Device device = qkv.device();
  for (const at::Tensor* t : {&a, &b, &gate, &out})
    TORCH_CHECK(t->device() == device && t->scalar_type() == at::kBFloat16 && t->dim() > 0 &&
                    t->stride(-1) == 1,
                "activations must be BF16 with dense rows");
  for (const at::Tensor* t : {&a_log, &state})
    TORCH_CHECK(t->device() == device && t->scalar_type() == at::kFloat && t->dim() > 0 &&
                    t->stride(-1) == 1,
                "state and A_log must be CUDA FP32 with dense rows");
  for (const at::Tensor* t : {&indices, &cu, &accepted})
    TORCH_CHECK(t->device() == device && t->scalar_type() == at::kInt && t->is_contiguous(),
                "metadata must be contiguous CUDA int32");
  for (const at::Tensor* t : {&dt_bias, &weight})
    TORCH_CHECK(t->device() == device && t->is_contiguous() && floats(*t),
                "weights must be contiguous FP32/BF16");
  // H and HV from qkv's width (2H + HV) * 128 and the state's head count
  const int64_t hv = state.dim() == 4 ? state.size(1) : 0;
  const int64_t cols = qkv.dim() == 2 ? qkv.size(1) : 0;
  const int64_t h2 = cols / kDim - hv;
  const int64_t h = h2 / 2;
  const bool geometry = hv > 0 && cols % kDim == 0 && h2 > 0 && h2 % 2 == 0 && hv % h == 0;
  TORCH_CHECK(qkv.dim() == 2 && geometry && qkv.stride(1) == 1,
              "qkv must be [tokens,(2*H+HV)*128] with HV a multiple of H");
  TORCH_CHECK(state.dim() == 4 && state.size(2) == kDim && state.size(3) == kDim &&
                  state.stride(2) == kDim && state.stride(1) == kDim * kDim,
              "state must be [slots,HV,128,128]");
  TORCH_CHECK(indices.dim() == 2 && indices.size(1) >= 1 && indices.size(1) <= LD_MAX_TOKENS,
              "decode/MTP supports 1 through 4 tokens per request");
  const int64_t n = qkv.size(0);
  TORCH_CHECK(a.dim() == 2 && a.size(0) == n && a.size(1) == hv && b.dim() == 2 &&
                  b.size(0) == n && b.size(1) == hv && gate.dim() == 3 && gate.size(0) == n &&
                  gate.size(1) == hv && gate.size(2) == kDim && out.dim() == 3 &&
                  out.size(0) == n && out.size(1) == hv && out.size(2) == kDim &&
                  out.is_contiguous() && gate.stride(1) == kDim,
              "invalid activation shape or output layout");
  TORCH_CHECK(a_log.numel() == hv && dt_bias.numel() == hv && weight.numel() == kDim,
              "invalid weight shapes");
  const int64_t requests = indices.size(0);
  TORCH_CHECK(cu.dim() == 1 && cu.numel() == requests + 1 && accepted.dim() == 1 &&
                  accepted.numel() == requests,
              "invalid request metadata shapes");
  TORCH_CHECK(eps > 0, "norm epsilon must be positive");
  return {h, hv};
}

ld_gdn_decode_args decode_args(const at::Tensor& qkv, const at::Tensor& a,
                               const at::Tensor& b, const at::Tensor& a_log,
                               const at::Tensor& dt_bias, const at::Tensor& indices,
                               const at::Tensor& cu, const at::Tensor& accepted,
                               const at::Tensor& state, const at::Tensor& gate,
                               const at::Tensor& weight, const at::Tensor& out, double eps,
                               std::pair<int64_t, int64_t> heads) {
  ld_gdn_decode_args args{};
  args.qkv = qkv.data_ptr();
  args.qkv_row_stride = qkv.stride(0);
  args.a = a.data_ptr();
  args.a_row_stride = a.stride(0);
  args.b = b.data_ptr();
  args.b_row_stride = b.stride(0);
  args.a_log = static_cast<const float*>(a_log.data_ptr());
  args.dt_bias = dt_bias.data_ptr();
  args.dt_bias_dtype = dtype_code(dt_bias);
  args.norm_weight_dtype = dtype_code(weight);
  args.indices = static_cast<const int32_t*>(indices.data_ptr());
  args.cu = static_cast<const int32_t*>(cu.data_ptr());
  args.accepted = static_cast<const int32_t*>(accepted.data_ptr());
  args.state = static_cast<float*>(state.data_ptr());
  args.state_slot_stride = state.stride(0);
  args.gate = gate.data_ptr();
  args.gate_row_stride = gate.stride(0);
  args.norm_weight = weight.data_ptr();
  args.out = out.data_ptr();
  args.num_requests = static_cast<int32_t>(indices.size(0));
  args.width = static_cast<int32_t>(indices.size(1));
  args.num_k_heads = static_cast<int32_t>(heads.first);
  args.num_v_heads = static_cast<int32_t>(heads.second);
  args.scale = static_cast<float>(0.08838834764831845);  // 128^-0.5 (reference csrc/gdn_decode.cu:417)
  args.eps = static_cast<float>(eps);
  args.cache_policy = g_cache_policy.load(std::memory_order_relaxed);
  return args;
}

void decode(const at::Tensor& qkv, const at::Tensor& a, const at::Tensor& b,
            const at::Tensor& a_log, const at::Tensor& dt_bias, const at::Tensor& indices,
            const at::Tensor& cu, const at::Tensor& accepted, at::Tensor state,
            const at::Tensor& gate, const at::Tensor& weight, at::Tensor out, double eps) {
  const auto heads = check_decode(qkv, a, b, a_log, dt_bias, indices, cu, accepted, state, gate,
                                  weight, out, eps);
  if (indices.size(0) == 0) return;
  const ld_gdn_decode_args args = decode_args(qkv, a, b, a_log, dt_bias, indices, cu, accepted,
                                              state, gate, weight, out, eps, heads);
  const c10::DeviceGuard guard(qkv.device());
  const int rc = ld_gdn_decode(&args, c10::hip::getCurrentHIPStream(qkv.get_device()).stream());
  TORCH_CHECK(rc == LD_OK, ld_last_error());
}

void decode_conv(const at::Tensor& mixed_qkv, at::Tensor conv_state, const at::Tensor& conv_weight,
                 const std::optional<at::Tensor>& conv_bias, const at::Tensor& a,
                 const at::Tensor& b, const at::Tensor& a_log, const at::Tensor& dt_bias,
                 const at::Tensor& indices, const at::Tensor& cu, const at::Tensor& accepted,
                 at::Tensor state, const at::Tensor& gate, const at::Tensor& weight,
                 at::Tensor out, double eps) {
  const auto heads = check_decode(mixed_qkv, a, b, a_log, dt_bias, indices, cu, accepted, state,
                                  gate, weight, out, eps);
  const int64_t conv_dim = mixed_qkv.size(1);
  TORCH_CHECK(conv_state.device() == mixed_qkv.device() &&
                  conv_state.scalar_type() == at::kBFloat16 && conv_state.dim() == 3 &&
                  conv_state.size(1) == conv_dim && conv_state.size(2) >= 3 &&
                  conv_state.size(2) <= 8,
              "conv_state must be CUDA BF16 [slots, conv_dim, 3..8]");
  TORCH_CHECK(conv_weight.device() == mixed_qkv.device() &&
                  conv_weight.scalar_type() == at::kBFloat16 && conv_weight.dim() == 2 &&
                  conv_weight.size(0) == conv_dim && conv_weight.size(1) == 4 &&
                  conv_weight.is_contiguous() &&
                  reinterpret_cast<uintptr_t>(conv_weight.data_ptr()) % 8 == 0,
              "conv_weight must be contiguous CUDA BF16 [conv_dim, 4]");
  const at::Tensor* bias = conv_bias.has_value() ? &*conv_bias : nullptr;
  if (bias != nullptr)
    TORCH_CHECK(bias->device() == mixed_qkv.device() && bias->scalar_type() == at::kBFloat16 &&
                    bias->numel() == conv_dim && bias->is_contiguous(),
                "conv_bias must be contiguous CUDA BF16 [conv_dim]");
  ld_gdn_decode_args args = decode_args(mixed_qkv, a, b, a_log, dt_bias, indices, cu, accepted,
                                        state, gate, weight, out, eps, heads);
  args.qkv = nullptr;  // the post-conv activations are the kernel's own
  args.qkv_row_stride = 0;
  ld_conv_args conv{};
  conv.x = mixed_qkv.data_ptr();
  conv.x_row_stride = mixed_qkv.stride(0);
  conv.state = conv_state.data_ptr();
  conv.state_slots = conv_state.size(0);
  conv.state_slot_stride = conv_state.stride(0);
  conv.state_dim_stride = conv_state.stride(1);
  conv.state_len_stride = conv_state.stride(2);
  conv.state_len = static_cast<int32_t>(conv_state.size(2));
  conv.width = 4;
  conv.weight = conv_weight.data_ptr();
  conv.weight_dtype = LD_DTYPE_BF16;
  conv.bias_dtype = LD_DTYPE_BF16;
  conv.bias = bias != nullptr ? bias->data_ptr() : nullptr;
  const c10::DeviceGuard guard(mixed_qkv.device());
  const int rc = ld_gdn_decode_conv(
      &args, &conv, c10::hip::getCurrentHIPStream(mixed_qkv.get_device()).stream());
  TORCH_CHECK(rc == LD_OK, ld_last_error());
}

// ---- state-pool ops ----------------------------------------------------------------------

// Every dimension after the first densely packed (row-major).
bool dense_inner(const at::Tensor& t) {
  int64_t expected = 1;
  for (int64_t d = t.dim() - 1; d >= 1; --d) {
    if (t.size(d) != 1 && t.stride(d) != expected) return false;
    expected *= t.size(d);
  }
  return true;
}

int64_t row_bytes(const at::Tensor& t) {
  int64_t count = 1;
  for (int64_t d = 1; d < t.dim(); ++d) count *= t.size(d);
  return count * static_cast<int64_t>(t.element_size());
}

bool same_row_shape(const at::Tensor& a, const at::Tensor& b) {
  if (a.dim() != b.dim()) return false;
  for (int64_t d = 1; d < a.dim(); ++d)
    if (a.size(d) != b.size(d)) return false;
  return true;
}

// The reference's `check` (csrc/state_io.cu:29-41); fp32_4d = false drops the fp32 / 4-D
// requirement for the dtype-generic ops.
void check_state_layout(const at::Tensor& pool, const at::Tensor& slots, const at::Tensor& packed,
                        bool fp32_4d) {
  if (fp32_4d) {
    TORCH_CHECK(pool.is_cuda() && pool.scalar_type() == at::kFloat && pool.dim() == 4 &&
                    pool.stride(3) == 1 && pool.stride(2) == pool.size(3) &&
                    pool.stride(1) == pool.size(2) * pool.size(3),
                "pool must be CUDA FP32 with dense inner dimensions");
  } else {
    TORCH_CHECK(pool.is_cuda() && pool.dim() >= 1 && dense_inner(pool),
                "pool must be a CUDA tensor with dense inner dimensions");
  }
  TORCH_CHECK(slots.device() == pool.device() && slots.scalar_type() == at::kInt &&
                  slots.dim() == 1,
              "slots must be a CUDA int32 vector");
  TORCH_CHECK(packed.device() == pool.device() && packed.scalar_type() == pool.scalar_type() &&
                  packed.dim() == pool.dim() && packed.size(0) == slots.numel() &&
                  same_row_shape(packed, pool) && dense_inner(packed),
              "invalid packed layout");
}

void check_valid(const at::Tensor& valid, const at::Tensor& slots, const at::Tensor& pool) {
  TORCH_CHECK(valid.device() == pool.device() && valid.scalar_type() == at::kBool &&
                  valid.sizes() == slots.sizes() && valid.is_contiguous(),
              "valid must be a CUDA bool vector");
}

hipStream_t stream_of(const at::Tensor& t) {
  return c10::hip::getCurrentHIPStream(t.get_device()).stream();
}

void gather(const at::Tensor& pool, const at::Tensor& slots, const at::Tensor& valid,
            at::Tensor out) {
  if (slots.numel() == 0) return;
  const int64_t size = static_cast<int64_t>(pool.element_size());
  const c10::DeviceGuard guard(pool.device());
  const int rc = ld_state_gather(pool.data_ptr(), pool.stride(0) * size,
                                 static_cast<const int32_t*>(slots.data_ptr()), slots.stride(0),
                                 static_cast<const uint8_t*>(valid.data_ptr()), out.data_ptr(),
                                 out.stride(0) * size, row_bytes(pool), slots.numel(),
                                 stream_of(pool));
  TORCH_CHECK(rc == LD_OK, ld_last_error());
}

void scatter(const at::Tensor& packed, const at::Tensor& slots, at::Tensor pool) {
  if (slots.numel() == 0) return;
  const int64_t size = static_cast<int64_t>(pool.element_size());
  const c10::DeviceGuard guard(pool.device());
  const int rc = ld_state_scatter(packed.data_ptr(), packed.stride(0) * size,
                                  static_cast<const int32_t*>(slots.data_ptr()), slots.stride(0),
                                  pool.data_ptr(), pool.stride(0) * size, row_bytes(pool),
                                  slots.numel(), stream_of(pool));
  TORCH_CHECK(rc == LD_OK, ld_last_error());
}

void gather_state(const at::Tensor& pool, const at::Tensor& slots, const at::Tensor& valid,
                  at::Tensor out) {
  check_state_layout(pool, slots, out, true);
  check_valid(valid, slots, pool);
  gather(pool, slots, valid, out);
}

void scatter_state(const at::Tensor& packed, const at::Tensor& slots, at::Tensor pool) {
  check_state_layout(pool, slots, packed, true);
  scatter(packed, slots, pool);
}

void gather_slots(const at::Tensor& pool, const at::Tensor& slots, const at::Tensor& valid,
                  at::Tensor out) {
  check_state_layout(pool, slots, out, false);
  check_valid(valid, slots, pool);
  gather(pool, slots, valid, out);
}

void scatter_slots(const at::Tensor& packed, const at::Tensor& slots, at::Tensor pool) {
  check_state_layout(pool, slots, packed, false);
  scatter(packed, slots, pool);
}

void check_copy(const at::Tensor& pool, const at::Tensor& src, const at::Tensor& dst) {
  TORCH_CHECK(pool.is_cuda() && pool.dim() >= 1 && dense_inner(pool),
              "pool must be a CUDA tensor with dense inner dimensions");
  for (const at::Tensor* t : {&src, &dst})
    TORCH_CHECK(t->device() == pool.device() && t->scalar_type() == at::kInt && t->dim() == 1 &&
                    t->is_contiguous(),
                "src and dst must be contiguous CUDA int32 vectors");
  TORCH_CHECK(src.numel() == dst.numel(), "src and dst must have the same length");
}

void copy_state(at::Tensor pool, const at::Tensor& src, const at::Tensor& dst) {
  check_copy(pool, src, dst);
  if (src.numel() == 0) return;
  const c10::DeviceGuard guard(pool.device());
  const int rc = ld_state_copy(pool.data_ptr(),
                               pool.stride(0) * static_cast<int64_t>(pool.element_size()),
                               static_cast<const int32_t*>(src.data_ptr()),
                               static_cast<const int32_t*>(dst.data_ptr()), src.numel(),
                               row_bytes(pool), stream_of(pool));
  TORCH_CHECK(rc == LD_OK, ld_last_error());
}

void copy_state_checked(at::Tensor pool, const at::Tensor& src, const at::Tensor& dst,
                        at::Tensor rejected) {
  check_copy(pool, src, dst);
  TORCH_CHECK(rejected.device() == pool.device() && rejected.scalar_type() == at::kInt &&
                  rejected.dim() == 1 && rejected.is_contiguous() &&
                  rejected.numel() == src.numel(),
              "rejected must be a contiguous CUDA int32 vector with one entry per pair");
  if (src.numel() == 0) return;
  TORCH_CHECK(row_bytes(pool) > 0, "pool slots must not be empty");
  const c10::DeviceGuard guard(pool.device());
  const int rc = ld_state_copy_checked(
      pool.data_ptr(), pool.stride(0) * static_cast<int64_t>(pool.element_size()),
      static_cast<const int32_t*>(src.data_ptr()), static_cast<const int32_t*>(dst.data_ptr()),
      src.numel(), row_bytes(pool), static_cast<int32_t*>(rejected.data_ptr()), stream_of(pool));
  TORCH_CHECK(rc == LD_OK, ld_last_error());
}

void zero_slots(at::Tensor pool, const at::Tensor& slots) {
  TORCH_CHECK(pool.is_cuda() && pool.dim() >= 1 && dense_inner(pool),
              "pool must be a CUDA tensor with dense inner dimensions");
  TORCH_CHECK(slots.device() == pool.device() && slots.scalar_type() == at::kInt &&
                  slots.dim() == 1 && slots.is_contiguous(),
              "slots must be a contiguous CUDA int32 vector");
  if (slots.numel() == 0) return;
  const c10::DeviceGuard guard(pool.device());
  const int rc = ld_state_zero(pool.data_ptr(),
                               pool.stride(0) * static_cast<int64_t>(pool.element_size()),
                               static_cast<const int32_t*>(slots.data_ptr()), slots.numel(),
                               row_bytes(pool), stream_of(pool));
  TORCH_CHECK(rc == LD_OK, ld_last_error());
}

void packed_plan(const at::Tensor& slots, const at::Tensor& cu, const at::Tensor& accepted,
                 at::Tensor source, at::Tensor valid, at::Tensor indices,
                 at::Tensor destinations) {
  TORCH_CHECK(slots.is_cuda() && slots.scalar_type() == at::kInt && slots.dim() == 2 &&
                  slots.is_contiguous() && slots.size(1) >= 1 && slots.size(1) <= LD_MAX_TOKENS,
              "slots must be a contiguous CUDA int32 [batch, 1..4] tensor");
  const int64_t batch = slots.size(0);
  const int64_t width = slots.size(1);
  const std::pair<const at::Tensor*, std::vector<int64_t>> ints[] = {
      {&cu, {batch + 1}}, {&accepted, {batch}}, {&source, {batch}},
      {&indices, {batch, width}}, {&destinations, {batch * width}}};
  for (const auto& [t, shape] : ints)
    TORCH_CHECK(t->device() == slots.device() && t->scalar_type() == at::kInt &&
                    t->sizes() == at::IntArrayRef(shape) && t->is_contiguous(),
                "packed_plan tensors must be contiguous CUDA int32 of the batch's shapes");
  TORCH_CHECK(valid.device() == slots.device() && valid.scalar_type() == at::kBool &&
                  valid.dim() == 1 && valid.size(0) == batch && valid.is_contiguous(),
              "valid must be a contiguous CUDA bool vector");
  TORCH_CHECK(batch <= INT32_MAX, "batch too large");
  if (batch == 0) return;
  const c10::DeviceGuard guard(slots.device());
  const int rc = ld_packed_plan(
      static_cast<const int32_t*>(slots.data_ptr()), static_cast<const int32_t*>(cu.data_ptr()),
      static_cast<const int32_t*>(accepted.data_ptr()), static_cast<int32_t>(batch),
      static_cast<int32_t>(width), static_cast<int32_t*>(source.data_ptr()),
      static_cast<uint8_t*>(valid.data_ptr()), static_cast<int32_t*>(indices.data_ptr()),
      static_cast<int32_t*>(destinations.data_ptr()), stream_of(slots));
  TORCH_CHECK(rc == LD_OK, ld_last_error());
}

// ---- linear attention with a decay for each head -------------------------------------------

// The checks that linear_decode and linear_prefill share (ops.py _linear_layout restates them);
// returns H, HV.
std::pair<int64_t, int64_t> check_linear(const at::Tensor& qkv, const at::Tensor& log_decay,
                                         const at::Tensor& state,
                                         const std::optional<at::Tensor>& gate,
                                         const std::optional<at::Tensor>& weight,
                                         const at::Tensor& out, double scale, double eps) {
  TORCH_CHECK(qkv.is_cuda() && qkv.scalar_type() == at::kBFloat16, "qkv must be CUDA BF16");
  const c10::Device device = qkv.device();
  TORCH_CHECK(state.device() == device && state.scalar_type() == at::kFloat && state.dim() == 4 &&
                  state.size(2) == kDim && state.size(3) == kDim && state.stride(3) == 1 &&
                  state.stride(2) == kDim && state.stride(1) == kDim * kDim,
              "state must be CUDA FP32 [slots,HV,128,128] with dense heads");
  const int64_t hv = state.size(1);
  const int64_t cols = qkv.dim() == 2 ? qkv.size(1) : 0;
  const int64_t h2 = cols / kDim - hv;
  const int64_t h = h2 / 2;
  TORCH_CHECK(qkv.dim() == 2 && hv > 0 && cols % kDim == 0 && h2 > 0 && h2 % 2 == 0 &&
                  hv % h == 0 && qkv.stride(1) == 1,
              "qkv must be [tokens,(2*H+HV)*128] with HV a multiple of H");
  const int64_t n = qkv.size(0);
  const int64_t ld = log_decay.dim();
  TORCH_CHECK(log_decay.device() == device && log_decay.scalar_type() == at::kFloat &&
                  ((ld == 1 && log_decay.size(0) == hv) ||
                   (ld == 2 && log_decay.size(0) == n && log_decay.size(1) == hv)) &&
                  log_decay.stride(-1) == 1,
              "log_decay must be CUDA FP32 [HV] or [tokens,HV] with dense rows");
  TORCH_CHECK(out.device() == device && out.scalar_type() == at::kBFloat16 && out.dim() == 3 &&
                  out.size(0) == n && out.size(1) == hv && out.size(2) == kDim &&
                  out.is_contiguous(),
              "out must be contiguous CUDA BF16 [tokens,HV,128]");
  TORCH_CHECK(gate.has_value() == weight.has_value(), "gate and weight must be given together");
  if (gate.has_value()) {
    TORCH_CHECK(gate->device() == device && gate->scalar_type() == at::kBFloat16 &&
                    gate->dim() == 3 && gate->size(0) == n && gate->size(1) == hv &&
                    gate->size(2) == kDim && gate->stride(2) == 1 && gate->stride(1) == kDim,
                "gate must be CUDA BF16 [tokens,HV,128] with dense rows");
    TORCH_CHECK(weight->device() == device && weight->is_contiguous() && floats(*weight) &&
                    weight->numel() == kDim,
                "weight must be contiguous CUDA FP32/BF16 [128]");
  }
  TORCH_CHECK(std::abs(scale) <= std::numeric_limits<float>::max(), "scale must be finite");
  TORCH_CHECK(eps > 0, "norm epsilon must be positive");
  TORCH_CHECK(state.size(0) <= INT32_MAX && hv <= INT32_MAX / kDim, "state pool too large");
  return {h, hv};
}

// The arguments that both entry points' structs have.
template <typename Args>
Args linear_args(const at::Tensor& qkv, const at::Tensor& log_decay, const at::Tensor& state,
                 const std::optional<at::Tensor>& gate, const std::optional<at::Tensor>& weight,
                 const at::Tensor& out, double scale, double eps,
                 std::pair<int64_t, int64_t> heads) {
  Args args{};
  args.qkv = qkv.data_ptr();
  args.qkv_row_stride = qkv.stride(0);
  args.log_decay = static_cast<const float*>(log_decay.data_ptr());
  args.log_decay_row_stride = log_decay.dim() == 2 ? log_decay.stride(0) : 0;
  args.state = static_cast<float*>(state.data_ptr());
  args.state_slot_stride = state.stride(0);
  if (gate.has_value() && gate->size(0) > 0) {   // (without tokens its pointer is NULL)
    args.gate = gate->data_ptr();
    args.gate_row_stride = gate->stride(0);
    args.norm_weight = weight->data_ptr();
    args.norm_weight_dtype = dtype_code(*weight);
  }
  args.out = out.data_ptr();
  args.num_tokens = qkv.size(0);
  args.num_slots = static_cast<int32_t>(state.size(0));
  args.num_k_heads = static_cast<int32_t>(heads.first);
  args.num_v_heads = static_cast<int32_t>(heads.second);
  args.scale = static_cast<float>(scale);
  args.eps = static_cast<float>(eps);
  return args;
}

void linear_decode(const at::Tensor& qkv, const at::Tensor& log_decay, const at::Tensor& indices,
                   const at::Tensor& cu, const at::Tensor& accepted, at::Tensor state,
                   const std::optional<at::Tensor>& gate, const std::optional<at::Tensor>& weight,
                   at::Tensor out, double scale, double eps) {
  const auto heads = check_linear(qkv, log_decay, state, gate, weight, out, scale, eps);
  for (const at::Tensor* t : {&indices, &cu, &accepted})
    TORCH_CHECK(t->device() == qkv.device() && t->scalar_type() == at::kInt && t->is_contiguous(),
                "metadata must be contiguous CUDA int32");
  TORCH_CHECK(indices.dim() == 2 && indices.size(1) >= 1 && indices.size(1) <= LD_MAX_TOKENS,
              "decode/MTP supports 1 through 4 tokens per request");
  const int64_t requests = indices.size(0);
  TORCH_CHECK(cu.dim() == 1 && cu.numel() == requests + 1 && accepted.dim() == 1 &&
                  accepted.numel() == requests && requests <= INT32_MAX,
              "invalid request metadata shapes");
  if (requests == 0 || qkv.size(0) == 0) return;
  auto args = linear_args<ld_linear_decode_args>(qkv, log_decay, state, gate, weight, out, scale,
                                                 eps, heads);
  args.indices = static_cast<const int32_t*>(indices.data_ptr());
  args.cu = static_cast<const int32_t*>(cu.data_ptr());
  args.accepted = static_cast<const int32_t*>(accepted.data_ptr());
  args.num_requests = static_cast<int32_t>(requests);
  args.width = static_cast<int32_t>(indices.size(1));
  args.cache_policy = g_cache_policy.load(std::memory_order_relaxed);
  const c10::DeviceGuard guard(qkv.device());
  const int rc = ld_linear_decode(&args, stream_of(qkv));
  TORCH_CHECK(rc == LD_OK, ld_last_error());
}

void linear_prefill(const at::Tensor& qkv, const at::Tensor& log_decay, const at::Tensor& slots,
                    const at::Tensor& has_initial, const at::Tensor& cu_seqlens, at::Tensor state,
                    const std::optional<at::Tensor>& gate, const std::optional<at::Tensor>& weight,
                    at::Tensor out, double scale, double eps) {
  const auto heads = check_linear(qkv, log_decay, state, gate, weight, out, scale, eps);
  for (const at::Tensor* t : {&slots, &cu_seqlens})
    TORCH_CHECK(t->device() == qkv.device() && t->scalar_type() == at::kInt && t->dim() == 1 &&
                    t->is_contiguous(),
                "metadata must be contiguous CUDA int32");
  TORCH_CHECK(has_initial.device() == qkv.device() && has_initial.scalar_type() == at::kBool &&
                  has_initial.dim() == 1 && has_initial.is_contiguous(),
              "has_initial must be a contiguous CUDA bool vector");
  const int64_t sequences = slots.numel();
  TORCH_CHECK(cu_seqlens.numel() == sequences + 1 && has_initial.numel() == sequences &&
                  sequences <= INT32_MAX,
              "invalid sequence metadata shapes");
  if (sequences == 0) return;
  auto args = linear_args<ld_linear_prefill_args>(qkv, log_decay, state, gate, weight, out, scale,
                                                  eps, heads);
  args.slots = static_cast<const int32_t*>(slots.data_ptr());
  args.has_initial = static_cast<const uint8_t*>(has_initial.data_ptr());
  args.cu_seqlens = static_cast<const int32_t*>(cu_seqlens.data_ptr());
  args.num_sequences = static_cast<int32_t>(sequences);
  const c10::DeviceGuard guard(qkv.device());
  // From torch's caching allocator for this call alone: on one stream the next call may take the
  // same memory, in order; under capture it is the graph's own.
  at::Tensor workspace;
  const int64_t bytes = ld_linear_prefill_workspace_bytes(args.num_tokens, args.num_sequences,
                                                          args.num_v_heads);
  if (bytes > 0) {
    workspace = at::empty({bytes}, qkv.options().dtype(at::kByte));
    args.workspace = workspace.data_ptr();
    args.workspace_bytes = bytes;
  }
  const int rc = ld_linear_prefill(&args, stream_of(qkv));
  TORCH_CHECK(rc == LD_OK, ld_last_error());
}

// What norm_rope and norm_rope_axes share (ops.py _rope_layout restates the checks): the C ABI's
// arguments but for the positions.
ld_norm_rope_args rope_args(const at::Tensor& qkv, const at::Tensor& q_weight,
                            const at::Tensor& k_weight, const at::Tensor& inv_freq,
                            int64_t q_heads, int64_t k_heads, double eps, bool interleaved) {
  TORCH_CHECK(qkv.is_cuda() && qkv.scalar_type() == at::kBFloat16, "qkv must be CUDA BF16");
  TORCH_CHECK(q_heads >= 0 && k_heads >= 0 && q_heads <= INT32_MAX / kDim &&
                  k_heads <= INT32_MAX / kDim && qkv.dim() == 2 &&
                  qkv.size(1) >= (q_heads + k_heads) * kDim && qkv.stride(1) == 1,
              "qkv must be [tokens,>=(q_heads+k_heads)*128] with dense rows");
  const int64_t n = qkv.size(0);
  TORCH_CHECK(n <= 1 || qkv.stride(0) >= (q_heads + k_heads) * kDim, "qkv rows must not overlap");
  for (const at::Tensor* t : {&q_weight, &k_weight})
    TORCH_CHECK(t->device() == qkv.device() && t->is_contiguous() && floats(*t) &&
                    t->numel() == kDim,
                "weights must be contiguous CUDA FP32/BF16 [128]");
  const int64_t rotary = 2 * inv_freq.numel();
  TORCH_CHECK(inv_freq.device() == qkv.device() && inv_freq.scalar_type() == at::kFloat &&
                  inv_freq.dim() == 1 && inv_freq.is_contiguous() && rotary <= kDim &&
                  (interleaved || rotary % 16 == 0),
              "inv_freq must be contiguous CUDA FP32 [rotary/2], rotary at most 128 and a multiple "
              "of 16 unless interleaved");
  TORCH_CHECK(eps > 0, "norm epsilon must be positive");
  ld_norm_rope_args args{};
  args.qkv = qkv.data_ptr();
  args.qkv_row_stride = qkv.stride(0);
  args.q_weight = q_weight.data_ptr();
  args.k_weight = k_weight.data_ptr();
  args.q_weight_dtype = dtype_code(q_weight);
  args.k_weight_dtype = dtype_code(k_weight);
  args.rotary = static_cast<int32_t>(rotary);
  args.inv_freq = static_cast<const float*>(inv_freq.data_ptr());
  args.num_tokens = n;
  args.q_heads = static_cast<int32_t>(q_heads);
  args.k_heads = static_cast<int32_t>(k_heads);
  args.interleaved = interleaved;
  args.eps = static_cast<float>(eps);
  return args;
}

bool is_index(const at::Tensor& t) {
  return t.scalar_type() == at::kInt || t.scalar_type() == at::kLong;
}

void norm_rope(at::Tensor qkv, const at::Tensor& q_weight, const at::Tensor& k_weight,
               const at::Tensor& positions, const at::Tensor& inv_freq, int64_t q_heads,
               int64_t k_heads, double eps, bool interleaved) {
  auto args = rope_args(qkv, q_weight, k_weight, inv_freq, q_heads, k_heads, eps, interleaved);
  TORCH_CHECK(positions.device() == qkv.device() && is_index(positions) && positions.dim() == 1 &&
                  positions.size(0) == args.num_tokens && positions.is_contiguous(),
              "positions must be contiguous CUDA int32/int64 [tokens]");
  if (args.num_tokens == 0 || q_heads + k_heads == 0) return;
  args.positions = positions.data_ptr();
  args.positions_int64 = positions.scalar_type() == at::kLong;
  const c10::DeviceGuard guard(qkv.device());
  const int rc = ld_norm_rope(&args, stream_of(qkv));
  TORCH_CHECK(rc == LD_OK, ld_last_error());
}

// ---- softmax attention over a paged cache in 8 bits ----------------------------------------

void norm_rope_axes(at::Tensor qkv, const at::Tensor& q_weight, const at::Tensor& k_weight,
                    const at::Tensor& positions, const at::Tensor& axes,
                    const at::Tensor& inv_freq, int64_t q_heads, int64_t k_heads, double eps,
                    bool interleaved) {
  auto args = rope_args(qkv, q_weight, k_weight, inv_freq, q_heads, k_heads, eps, interleaved);
  const int64_t n = args.num_tokens;
  TORCH_CHECK(positions.device() == qkv.device() && is_index(positions) && positions.dim() == 2 &&
                  positions.size(0) >= 1 && positions.size(0) <= INT32_MAX &&
                  positions.size(1) == n && (n <= 1 || positions.stride(1) == 1),
              "positions must be CUDA int32/int64 [axes,tokens] with dense rows");
  TORCH_CHECK(axes.device() == qkv.device() && axes.scalar_type() == at::kInt && axes.dim() == 1 &&
                  axes.size(0) == inv_freq.size(0) && axes.is_contiguous(),
              "axes must be contiguous CUDA int32 [rotary/2]");
  if (n == 0 || q_heads + k_heads == 0) return;
  args.positions = positions.data_ptr();
  args.positions_int64 = positions.scalar_type() == at::kLong;
  ld_rope_axes several{};
  several.axes = static_cast<const int32_t*>(axes.data_ptr());
  several.position_axis_stride = positions.stride(0);
  several.num_axes = static_cast<int32_t>(positions.size(0));
  const c10::DeviceGuard guard(qkv.device());
  const int rc = ld_norm_rope_axes(&args, &several, stream_of(qkv));
  TORCH_CHECK(rc == LD_OK, ld_last_error());
}

// The cache and its requests, for activations like `rows` (ops.py _cache_layout restates the
// checks).
ld_paged_cache paged_cache(const at::Tensor& rows, const at::Tensor& pages, const at::Tensor& cu,
                           const at::Tensor& lengths, const at::Tensor& k_cache,
                           const at::Tensor& v_cache, const at::Tensor& k_scale,
                           const at::Tensor& v_scale) {
  const c10::Device device = rows.device();
  for (const at::Tensor* t : {&k_cache, &v_cache})
    TORCH_CHECK(t->device() == device && t->scalar_type() == at::kFloat8_e4m3fn &&
                    t->dim() == 5 && dense_inner(*t) &&
                    reinterpret_cast<uintptr_t>(t->data_ptr()) % 16 == 0 &&
                    (t->size(0) <= 1 || (t->stride(0) % 16 == 0 && t->stride(0) >= row_bytes(*t))),
                "caches must be CUDA float8_e4m3fn with dense pages, 16-byte aligned");
  const int64_t count = k_cache.size(0), heads = k_cache.size(1), page = k_cache.size(3);
  TORCH_CHECK((page == 16 || page == 32 || page == 64 || page == 128) && k_cache.size(2) == 8 &&
                  k_cache.size(4) == 16 && heads >= 1 && heads <= 1 << 16,
              "k_cache must be [pages,kv_heads,8,page,16], page 16, 32, 64 or 128");
  TORCH_CHECK(v_cache.size(0) == count && v_cache.size(1) == heads &&
                  v_cache.size(2) == page / 16 && v_cache.size(3) == kDim && v_cache.size(4) == 16,
              "v_cache must be [pages,kv_heads,page/16,128,16]");
  for (const at::Tensor* t : {&k_scale, &v_scale})
    TORCH_CHECK(t->device() == device && t->scalar_type() == at::kFloat8_e8m0fnu &&
                    t->dim() == 2 && t->size(0) == count && t->size(1) == heads &&
                    dense_inner(*t) && (count <= 1 || t->stride(0) >= heads),
                "scales must be CUDA float8_e8m0fnu [pages,kv_heads] with dense rows");
  for (const at::Tensor* t : {&pages, &cu, &lengths})
    TORCH_CHECK(t->device() == device && t->scalar_type() == at::kInt,
                "metadata must be CUDA int32");
  const int64_t requests = lengths.numel();
  TORCH_CHECK(lengths.dim() == 1 && lengths.is_contiguous() && cu.dim() == 1 &&
                  cu.numel() == requests + 1 && cu.is_contiguous() && pages.dim() == 2 &&
                  pages.size(0) == requests && (pages.size(1) <= 1 || pages.stride(1) == 1) &&
                  std::max({requests, pages.size(1), count}) <= INT32_MAX,
              "invalid request metadata shapes");
  ld_paged_cache cache{};
  cache.k = k_cache.data_ptr();
  cache.v = v_cache.data_ptr();
  cache.k_scale = static_cast<uint8_t*>(k_scale.data_ptr());
  cache.v_scale = static_cast<uint8_t*>(v_scale.data_ptr());
  cache.k_page_stride = count > 1 ? k_cache.stride(0) : 0;
  cache.v_page_stride = count > 1 ? v_cache.stride(0) : 0;
  cache.k_scale_stride = count > 1 ? k_scale.stride(0) : 0;
  cache.v_scale_stride = count > 1 ? v_scale.stride(0) : 0;
  cache.pages = static_cast<const int32_t*>(pages.data_ptr());
  cache.pages_row_stride = pages.stride(0);
  cache.cu = static_cast<const int32_t*>(cu.data_ptr());
  cache.lengths = static_cast<const int32_t*>(lengths.data_ptr());
  cache.num_tokens = rows.dim() > 0 ? rows.size(0) : 0;
  cache.table_width = static_cast<int32_t>(pages.size(1));
  cache.num_pages = static_cast<int32_t>(count);
  cache.page_size = static_cast<int32_t>(page);
  cache.num_kv_heads = static_cast<int32_t>(heads);
  cache.num_requests = static_cast<int32_t>(requests);
  return cache;
}

ld_cache_rows cache_rows(const at::Tensor& k, const at::Tensor& v, int64_t heads) {
  for (const at::Tensor* t : {&k, &v})
    TORCH_CHECK(t->device() == k.device() && t->scalar_type() == at::kBFloat16 && t->dim() == 3 &&
                    t->size(0) == k.size(0) && t->size(1) == heads && t->size(2) == kDim &&
                    dense_inner(*t),
                "k and v must be CUDA BF16 [tokens,kv_heads,128] with dense rows");
  TORCH_CHECK(k.size(0) <= INT32_MAX, "too many tokens");
  return ld_cache_rows{k.data_ptr(), v.data_ptr(), k.stride(0), v.stride(0)};
}

bool nothing(const ld_paged_cache& cache) {
  return cache.num_requests == 0 || cache.num_tokens == 0;
}

void cache_write(const at::Tensor& k, const at::Tensor& v, const at::Tensor& pages,
                 const at::Tensor& cu, const at::Tensor& lengths, at::Tensor k_cache,
                 at::Tensor v_cache, at::Tensor k_scale, at::Tensor v_scale) {
  TORCH_CHECK(k.is_cuda(), "k and v must be CUDA BF16 [tokens,kv_heads,128] with dense rows");
  auto cache = paged_cache(k, pages, cu, lengths, k_cache, v_cache, k_scale, v_scale);
  const auto rows = cache_rows(k, v, cache.num_kv_heads);
  if (nothing(cache)) return;
  const c10::DeviceGuard guard(k.device());
  const int rc = ld_cache_write(&cache, &rows, stream_of(k));
  TORCH_CHECK(rc == LD_OK, ld_last_error());
}

void cache_read(const at::Tensor& pages, const at::Tensor& cu, const at::Tensor& lengths,
                const at::Tensor& k_cache, const at::Tensor& v_cache, const at::Tensor& k_scale,
                const at::Tensor& v_scale, at::Tensor k, at::Tensor v) {
  TORCH_CHECK(k.is_cuda(), "k and v must be CUDA BF16 [tokens,kv_heads,128] with dense rows");
  auto cache = paged_cache(k, pages, cu, lengths, k_cache, v_cache, k_scale, v_scale);
  const auto rows = cache_rows(k, v, cache.num_kv_heads);
  TORCH_CHECK(k.size(0) <= 1 || std::min(k.stride(0), v.stride(0)) >= cache.num_kv_heads * kDim,
              "rows of k and v must not overlap");
  if (nothing(cache)) return;
  const c10::DeviceGuard guard(k.device());
  const int rc = ld_cache_read(&cache, &rows, stream_of(k));
  TORCH_CHECK(rc == LD_OK, ld_last_error());
}

// attention_decode (a width) and attention_prefill (none).
void attend(const at::Tensor& q, const at::Tensor& pages, const at::Tensor& cu,
            const at::Tensor& lengths, const at::Tensor& k_cache, const at::Tensor& v_cache,
            const at::Tensor& k_scale, const at::Tensor& v_scale,
            const std::optional<at::Tensor>& gate, const at::Tensor& out,
            std::optional<int64_t> width, double scale) {
  TORCH_CHECK(!width || (*width >= 1 && *width <= LD_MAX_TOKENS),
              "decode/MTP supports 1 through 4 tokens per request");
  TORCH_CHECK(q.is_cuda() && q.scalar_type() == at::kBFloat16 && q.dim() == 3 &&
                  q.size(2) == kDim && dense_inner(q),
              "q must be CUDA BF16 [tokens,q_heads,128] with dense rows");
  auto cache = paged_cache(q, pages, cu, lengths, k_cache, v_cache, k_scale, v_scale);
  const int64_t heads = q.size(1);
  TORCH_CHECK(heads > 0 && heads <= 1 << 16 && heads % cache.num_kv_heads == 0,
              "q_heads must be a positive multiple of kv_heads");
  TORCH_CHECK(!gate.has_value() ||
                  (gate->device() == q.device() && gate->scalar_type() == at::kBFloat16 &&
                   gate->sizes() == q.sizes() && dense_inner(*gate)),
              "gate must be CUDA BF16 [tokens,q_heads,128] with dense rows");
  TORCH_CHECK(out.device() == q.device() && out.scalar_type() == at::kBFloat16 &&
                  out.sizes() == q.sizes() && out.is_contiguous(),
              "out must be contiguous CUDA BF16 [tokens,q_heads,128]");
  TORCH_CHECK(scale > 0 && scale * 1.44269504088896340736 <= std::numeric_limits<float>::max(),
              "scale must be positive, log2(e) times it finite");
  TORCH_CHECK(q.size(0) <= INT32_MAX, "too many tokens");
  if (nothing(cache)) return;
  ld_attention_args args{};
  args.q = q.data_ptr();
  args.q_row_stride = q.stride(0);
  if (gate.has_value()) {
    args.gate = gate->data_ptr();
    args.gate_row_stride = gate->stride(0);
  }
  args.out = out.data_ptr();
  args.num_q_heads = static_cast<int32_t>(heads);
  args.width = static_cast<int32_t>(width.value_or(0));
  args.scale = static_cast<float>(scale);
  const c10::DeviceGuard guard(q.device());
  // (a workspace as linear_prefill's: from torch's allocator for this call alone)
  at::Tensor workspace;
  const int64_t bytes = width ? ld_attention_decode_workspace_bytes(&cache, &args)
                              : ld_attention_prefill_workspace_bytes(&cache, &args);
  if (bytes > 0) {
    workspace = at::empty({bytes}, q.options().dtype(at::kByte));
    args.workspace = workspace.data_ptr();
    args.workspace_bytes = bytes;
  }
  const int rc = width ? ld_attention_decode(&cache, &args, stream_of(q))
                       : ld_attention_prefill(&cache, &args, stream_of(q));
  TORCH_CHECK(rc == LD_OK, ld_last_error());
}

void attention_decode(const at::Tensor& q, const at::Tensor& pages, const at::Tensor& cu,
                      const at::Tensor& lengths, const at::Tensor& k_cache,
                      const at::Tensor& v_cache, const at::Tensor& k_scale,
                      const at::Tensor& v_scale, const std::optional<at::Tensor>& gate,
                      at::Tensor out, int64_t width, double scale) {
  attend(q, pages, cu, lengths, k_cache, v_cache, k_scale, v_scale, gate, out, width, scale);
}

void attention_prefill(const at::Tensor& q, const at::Tensor& pages, const at::Tensor& cu,
                       const at::Tensor& lengths, const at::Tensor& k_cache,
                       const at::Tensor& v_cache, const at::Tensor& k_scale,
                       const at::Tensor& v_scale, const std::optional<at::Tensor>& gate,
                       at::Tensor out, double scale) {
  attend(q, pages, cu, lengths, k_cache, v_cache, k_scale, v_scale, gate, out, std::nullopt,
         scale);
}

}  // namespace

TORCH_LIBRARY_IMPL(lightdelta, CUDA, m) {
  m.impl("decode", &decode);
  m.impl("decode_conv", &decode_conv);
  m.impl("gather_state", &gather_state);
  m.impl("scatter_state", &scatter_state);
  m.impl("gather_slots", &gather_slots);
  m.impl("scatter_slots", &scatter_slots);
  m.impl("copy_state", &copy_state);
  m.impl("copy_state_checked", &copy_state_checked);
  m.impl("zero_slots", &zero_slots);
  m.impl("packed_plan", &packed_plan);
  m.impl("linear_decode", &linear_decode);
  m.impl("linear_prefill", &linear_prefill);
  m.impl("norm_rope", &norm_rope);
  m.impl("norm_rope_axes", &norm_rope_axes);
  m.impl("cache_write", &cache_write);
  m.impl("cache_read", &cache_read);
  m.impl("attention_decode", &attention_decode);
  m.impl("attention_prefill", &attention_prefill);
}

// The state cache policy these kernels pass (LD_CACHE_KEEP / LD_CACHE_STREAM), set from
// lightdelta_amd.ops.set_state_cache_policy.
extern "C" int ld_torch_set_cache_policy(int policy) {
  if (policy != LD_CACHE_KEEP && policy != LD_CACHE_STREAM) return LD_ERR_INVALID_ARGUMENT;
  g_cache_policy.store(policy, std::memory_order_relaxed);
  return LD_OK;
}
