// torch.library registration of the W8A16 GEMM (rla::w8a16_gemm), of the 8-bit
// activation path and of the mixture-of-experts layer.
//
// A thin C++ layer over the C ABI of include/rla_w8a16.h (rla_w8a16_gemm):
// it checks the tensors, allocates the fp16 output with torch's caching
// allocator on the input's device, picks the current torch CUDA stream and a
// per-(device, stream) split-K workspace, and calls the library.  No
// arithmetic happens here.  It replaces the launcher of rotalabs-accel's
// Triton path (src/rotalabs_accel/kernels/gemm.py:140-186, called from
// int8_gemm at :232) for 2-D fp16 activations; the Python int8_gemm keeps the
// reference's shape handling around it.
//
//   rla::w8a16_gemm(Tensor x, Tensor weight_int8, Tensor scale, Tensor? bias=None) -> Tensor
//     x       fp16 [M, K], unit inner stride (any row stride)
//     weight  int8 [N, K], unit inner stride
//     scale   fp32 or fp16 [N], contiguous
//     bias    fp16 or fp32 [N], contiguous, or None
//     -> fp16 [M, N], contiguous
//
// The Meta kernel gives the output's shape and dtype without computing, so
// the op traces under FakeTensor / torch.compile as an opaque call.
//
// The same file is also a Python extension module (_rla_torch_ops) whose
// w8a16_gemm calls the CUDA kernel function directly: the per-token hot path
// (Int8Linear.forward) takes it to skip the dispatcher's schema parsing and
// dispatch, a few microseconds of host time per call.  Same checks, same
// launch, same result as the op.
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/extension.h>
#include <torch/library.h>

#include <algorithm>
#include <map>
#include <mutex>
#include <tuple>
#include <utility>

#include "../../include/rla_w8a16.h"

namespace {

// Split-K workspaces, one per (device, stream), zero-filled when made and
// grown on demand.  Calls on one stream are ordered, so they share it.
at::Tensor workspace_for(const at::Device& dev, cudaStream_t stream, size_t bytes) {
  static std::mutex mu;
  static std::map<std::pair<int, cudaStream_t>, at::Tensor> cache;
  std::lock_guard<std::mutex> lock(mu);
  auto& ws = cache[{dev.index(), stream}];
  if (!ws.defined() || static_cast<size_t>(ws.numel()) < bytes) {
    const int64_t n = static_cast<int64_t>(bytes < (size_t(1) << 20) ? (size_t(1) << 20) : bytes);
    ws = at::zeros({n}, at::TensorOptions().dtype(at::kByte).device(dev));
  }
  return ws;
}

void check_args(const at::Tensor& x, const at::Tensor& w, const at::Tensor& scale,
                const std::optional<at::Tensor>& bias) {
  TORCH_CHECK(x.dim() == 2 && x.scalar_type() == at::kHalf, "rla::w8a16_gemm: x must be a 2-D float16 tensor");
  TORCH_CHECK(w.dim() == 2 && w.scalar_type() == at::kChar, "Weight must be INT8");
  TORCH_CHECK(w.size(1) == x.size(1), "Weight shape mismatch: ", w.sizes(), " vs (", w.size(0), ", ", x.size(1), ")");
  TORCH_CHECK(scale.dim() == 1 && scale.size(0) == w.size(0), "Scale shape mismatch: ", scale.sizes(), " vs (",
              w.size(0), ",)");
  TORCH_CHECK(scale.scalar_type() == at::kFloat || scale.scalar_type() == at::kHalf,
              "rla::w8a16_gemm: scale must be float32 or float16");
  if (bias.has_value()) {
    TORCH_CHECK(bias->dim() == 1 && bias->size(0) == w.size(0), "rla::w8a16_gemm: bias must be [N]");
    TORCH_CHECK(bias->scalar_type() == at::kHalf || bias->scalar_type() == at::kFloat,
                "rla::w8a16_gemm: bias must be float16 or float32");
  }
}

at::Tensor w8a16_gemm_cuda(const at::Tensor& x, const at::Tensor& w, const at::Tensor& scale,
                           const std::optional<at::Tensor>& bias) {
  check_args(x, w, scale, bias);
  const at::Device dev = x.device();
  TORCH_CHECK(dev.is_cuda() && w.device() == dev && scale.device() == dev &&
                  (!bias.has_value() || bias->device() == dev),
              "rla::w8a16_gemm: all tensors must be on the same CUDA device");
  const int64_t M = x.size(0), K = x.size(1), N = w.size(0);
  TORCH_CHECK(M == 0 || K == 0 || x.stride(1) == 1, "rla::w8a16_gemm: x needs a unit inner stride");
  TORCH_CHECK(N == 0 || K == 0 || w.stride(1) == 1, "rla::w8a16_gemm: weight_int8 needs a unit inner stride");
  TORCH_CHECK(scale.is_contiguous(), "rla::w8a16_gemm: scale must be contiguous");
  TORCH_CHECK(!bias.has_value() || bias->is_contiguous(), "rla::w8a16_gemm: bias must be contiguous");
  c10::cuda::CUDAGuard guard(dev);
  at::Tensor y = at::empty({M, N}, x.options());
  if (M == 0 || N == 0) return y;
  cudaStream_t stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
  const size_t need = rla_w8a16_workspace_size(M, N, K);
  void* ws_ptr = nullptr;
  size_t ws_bytes = 0;
  if (need) {
    at::Tensor ws = workspace_for(dev, stream, need);
    ws_ptr = ws.data_ptr();
    ws_bytes = static_cast<size_t>(ws.numel());
  }
  const int sdt = scale.scalar_type() == at::kFloat ? RLA_DTYPE_F32 : RLA_DTYPE_F16;
  const int bdt = !bias.has_value() ? RLA_DTYPE_NONE : bias->scalar_type() == at::kFloat ? RLA_DTYPE_F32 : RLA_DTYPE_F16;
  const int st = rla_w8a16_gemm(x.data_ptr(), K > 0 ? x.stride(0) : 0, static_cast<const int8_t*>(w.data_ptr()),
                                K > 0 ? w.stride(0) : 0, scale.data_ptr(), sdt,
                                bias.has_value() ? bias->data_ptr() : nullptr, bdt, y.data_ptr(), N, M, N, K,
                                ws_ptr, ws_bytes, stream);
  TORCH_CHECK(st == RLA_OK, "rla_w8a16_gemm failed with status ", st, ": ", rla_last_error());
  return y;
}

at::Tensor w8a16_gemm_meta(const at::Tensor& x, const at::Tensor& w, const at::Tensor& scale,
                           const std::optional<at::Tensor>& bias) {
  check_args(x, w, scale, bias);
  return at::empty({x.size(0), w.size(0)}, x.options());
}

// ---------------------------------------------------------------------------
// The 8-bit activation path and the mixture-of-experts layer: checks, outputs
// and per-call scratch from torch's allocator (a captured graph then owns its
// own scratch), the current stream, one call of the library.
// ---------------------------------------------------------------------------
cudaStream_t stream_of(const at::Device& dev) { return c10::cuda::getCurrentCUDAStream(dev.index()).stream(); }

// An output or scratch tensor from torch's allocator, without the dispatcher
// (a call of the norm makes three).
at::Tensor empty_on(const at::Device& dev, at::IntArrayRef sizes, at::ScalarType dtype) {
  return at::detail::empty_cuda(sizes, dtype, dev, std::nullopt);
}

int act_dtype(const at::Tensor& t, const char* what) {
  TORCH_CHECK_TYPE(t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16, what,
                   " must be float16 or bfloat16, got ", t.scalar_type());
  return t.scalar_type() == at::kHalf ? RLA_DTYPE_F16 : RLA_DTYPE_BF16;
}

int scale_dtype_of(const at::Tensor& t, const char* what) {
  TORCH_CHECK_TYPE(t.scalar_type() == at::kFloat || t.scalar_type() == at::kHalf, what,
                   " must be float32 or float16, got ", t.scalar_type());
  return t.scalar_type() == at::kFloat ? RLA_DTYPE_F32 : RLA_DTYPE_F16;
}

// Rows with a unit inner stride (a copy only where they have none) that do not
// overlap: a broadcast row stride is materialized.
at::Tensor rows_of(const at::Tensor& t) {
  return t.size(1) == 0 || ((t.size(1) == 1 || t.stride(1) == 1) && (t.size(0) <= 1 || t.stride(0) >= t.size(1)))
             ? t
             : t.contiguous();
}
int64_t row_stride(const at::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

void check_status(int st, const char* what) {
  TORCH_CHECK(st == RLA_OK, what, " failed with status ", st, ": ", rla_last_error());
}

void check_norm_args(const at::Tensor& x, const std::optional<at::Tensor>& residual, const at::Tensor& weight) {
  TORCH_CHECK(x.dim() == 2, "add_rmsnorm: x must be 2-D");
  act_dtype(x, "add_rmsnorm: x");
  TORCH_CHECK(weight.dim() == 1 && weight.size(0) == x.size(1), "Hidden dim mismatch: ", x.size(1), " vs ",
              weight.sizes());
  TORCH_CHECK_TYPE(weight.scalar_type() == at::kFloat || weight.scalar_type() == at::kHalf ||
                       weight.scalar_type() == at::kBFloat16,
                   "add_rmsnorm: unsupported weight dtype ", weight.scalar_type());
  if (residual.has_value()) {
    TORCH_CHECK(residual->sizes() == x.sizes(), "Residual shape mismatch: ", residual->sizes(), " vs ", x.sizes());
    TORCH_CHECK_TYPE(residual->scalar_type() == x.scalar_type(), "add_rmsnorm: residual must have x's dtype, got ",
                     residual->scalar_type(), " and ", x.scalar_type());
  }
}

// (q or y, scale or undefined, h)
std::tuple<at::Tensor, at::Tensor, at::Tensor> norm_cuda(const at::Tensor& x_in,
                                                         const std::optional<at::Tensor>& residual,
                                                         const at::Tensor& weight_in, double eps, bool int8) {
  check_norm_args(x_in, residual, weight_in);
  const at::Device dev = x_in.device();
  TORCH_CHECK(dev.is_cuda() && weight_in.device() == dev && (!residual.has_value() || residual->device() == dev),
              "add_rmsnorm: all tensors must be on the same CUDA device");
  c10::cuda::CUDAGuard guard(dev);
  const at::Tensor x = rows_of(x_in), weight = weight_in.contiguous();
  at::Tensor r, h = x_in;
  if (residual.has_value()) {
    r = rows_of(*residual);
    h = empty_on(dev, x.sizes(), x.scalar_type());
  }
  const int64_t M = x.size(0), K = x.size(1);
  at::Tensor y = empty_on(dev, {M, K}, int8 ? at::kChar : x.scalar_type());
  at::Tensor scale;
  if (int8) scale = empty_on(dev, {M}, at::kFloat);
  const int dt = act_dtype(x, "x");
  const int wdt = weight.scalar_type() == at::kFloat  ? RLA_DTYPE_F32
                  : weight.scalar_type() == at::kHalf ? RLA_DTYPE_F16
                                                      : RLA_DTYPE_BF16;
  const void* rp = residual.has_value() ? r.data_ptr() : nullptr;
  void* hp = residual.has_value() ? h.data_ptr() : nullptr;
  const int64_t ldr = residual.has_value() ? row_stride(r) : 0;
  if (int8)
    check_status(rla_add_rmsnorm_int8(x.data_ptr(), row_stride(x), rp, ldr, dt, weight.data_ptr(), wdt,
                                      static_cast<float>(eps), hp, K, static_cast<int8_t*>(y.data_ptr()), K,
                                      static_cast<float*>(scale.data_ptr()), M, K, stream_of(dev)),
                 "rla_add_rmsnorm_int8");
  else
    check_status(rla_add_rmsnorm(x.data_ptr(), row_stride(x), rp, ldr, dt, weight.data_ptr(), wdt,
                                 static_cast<float>(eps), hp, K, y.data_ptr(), K, M, K, stream_of(dev)),
                 "rla_add_rmsnorm");
  return {y, scale, h};
}

std::tuple<at::Tensor, at::Tensor> add_rmsnorm(const at::Tensor& x, const std::optional<at::Tensor>& residual,
                                               const at::Tensor& weight, double eps) {
  auto [y, s, h] = norm_cuda(x, residual, weight, eps, false);
  return {y, h};
}
std::tuple<at::Tensor, at::Tensor, at::Tensor> add_rmsnorm_int8(const at::Tensor& x,
                                                                const std::optional<at::Tensor>& residual,
                                                                const at::Tensor& weight, double eps) {
  return norm_cuda(x, residual, weight, eps, true);
}
// The ops take a residual always: an op's outputs must not alias its inputs.
std::tuple<at::Tensor, at::Tensor> add_rmsnorm_op(const at::Tensor& x, const at::Tensor& residual,
                                                  const at::Tensor& weight, double eps) {
  return add_rmsnorm(x, residual, weight, eps);
}
std::tuple<at::Tensor, at::Tensor, at::Tensor> add_rmsnorm_int8_op(const at::Tensor& x, const at::Tensor& residual,
                                                                   const at::Tensor& weight, double eps) {
  return add_rmsnorm_int8(x, residual, weight, eps);
}
std::tuple<at::Tensor, at::Tensor> add_rmsnorm_meta(const at::Tensor& x, const at::Tensor& residual,
                                                    const at::Tensor& weight, double) {
  check_norm_args(x, residual, weight);
  return {at::empty(x.sizes(), x.options()), at::empty(x.sizes(), x.options())};
}
std::tuple<at::Tensor, at::Tensor, at::Tensor> add_rmsnorm_int8_meta(const at::Tensor& x, const at::Tensor& residual,
                                                                     const at::Tensor& weight, double) {
  check_norm_args(x, residual, weight);
  return {at::empty(x.sizes(), x.options().dtype(at::kChar)), at::empty({x.size(0)}, x.options().dtype(at::kFloat)),
          at::empty(x.sizes(), x.options())};
}

void check_swiglu_args(const at::Tensor& gate, const at::Tensor& up) {
  TORCH_CHECK(gate.dim() == 2 && up.sizes() == gate.sizes(), "Gate and up shape mismatch: ", gate.sizes(), " vs ",
              up.sizes());
  act_dtype(gate, "swiglu_int8: gate");
  TORCH_CHECK_TYPE(up.scalar_type() == gate.scalar_type(), "swiglu_int8: up must have gate's dtype, got ",
                   up.scalar_type(), " and ", gate.scalar_type());
}
std::tuple<at::Tensor, at::Tensor> swiglu_int8_meta(const at::Tensor& gate, const at::Tensor& up) {
  check_swiglu_args(gate, up);
  return {at::empty(gate.sizes(), gate.options().dtype(at::kChar)),
          at::empty({gate.size(0)}, gate.options().dtype(at::kFloat))};
}
std::tuple<at::Tensor, at::Tensor> swiglu_int8_cuda(const at::Tensor& gate_in, const at::Tensor& up_in) {
  check_swiglu_args(gate_in, up_in);
  const at::Device dev = gate_in.device();
  TORCH_CHECK(dev.is_cuda() && up_in.device() == dev, "swiglu_int8: all tensors must be on the same CUDA device");
  c10::cuda::CUDAGuard guard(dev);
  const at::Tensor gate = rows_of(gate_in), up = rows_of(up_in);
  const int64_t M = gate.size(0), N = gate.size(1);
  at::Tensor q = empty_on(dev, {M, N}, at::kChar);
  at::Tensor scale = empty_on(dev, {M}, at::kFloat);
  check_status(rla_swiglu_int8(gate.data_ptr(), row_stride(gate), up.data_ptr(), row_stride(up),
                               act_dtype(gate, "gate"), static_cast<int8_t*>(q.data_ptr()), N,
                               static_cast<float*>(scale.data_ptr()), M, N, stream_of(dev)),
               "rla_swiglu_int8");
  return {q, scale};
}

void check_w8a8_args(const at::Tensor& x, const at::Tensor& x_scale, const at::Tensor& w, const at::Tensor& scale,
                     const std::optional<at::Tensor>& bias) {
  TORCH_CHECK(x.dim() == 2 && x.scalar_type() == at::kChar, "rla::w8a8_gemm: x must be a 2-D int8 tensor");
  TORCH_CHECK(w.dim() == 2 && w.scalar_type() == at::kChar, "Weight must be INT8");
  TORCH_CHECK(w.size(1) == x.size(1), "Weight shape mismatch: ", w.sizes(), " vs (", w.size(0), ", ", x.size(1), ")");
  TORCH_CHECK(x_scale.dim() == 1 && x_scale.size(0) == x.size(0), "Activation scale shape mismatch: ",
              x_scale.sizes(), " vs (", x.size(0), ",)");
  TORCH_CHECK_TYPE(x_scale.scalar_type() == at::kFloat, "rla::w8a8_gemm: x_scale must be float32");
  TORCH_CHECK(scale.dim() == 1 && scale.size(0) == w.size(0), "Scale shape mismatch: ", scale.sizes(), " vs (",
              w.size(0), ",)");
  scale_dtype_of(scale, "rla::w8a8_gemm: scale");
  if (bias.has_value()) {
    TORCH_CHECK(bias->dim() == 1 && bias->size(0) == w.size(0), "rla::w8a8_gemm: bias must be [N]");
    scale_dtype_of(*bias, "rla::w8a8_gemm: bias");
  }
}
at::Tensor w8a8_gemm_meta(const at::Tensor& x, const at::Tensor& x_scale, const at::Tensor& w, const at::Tensor& scale,
                          const std::optional<at::Tensor>& bias) {
  check_w8a8_args(x, x_scale, w, scale, bias);
  return at::empty({x.size(0), w.size(0)}, x.options().dtype(at::kHalf));
}
bool rows_aligned(const at::Tensor& t) {
  return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) == 0 && (t.size(0) <= 1 || t.stride(0) % 16 == 0);
}
at::Tensor w8a8_gemm_cuda(const at::Tensor& x_in, const at::Tensor& x_scale_in, const at::Tensor& w_in,
                          const at::Tensor& scale_in, const std::optional<at::Tensor>& bias_in) {
  check_w8a8_args(x_in, x_scale_in, w_in, scale_in, bias_in);
  const at::Device dev = x_in.device();
  TORCH_CHECK(dev.is_cuda() && w_in.device() == dev && scale_in.device() == dev && x_scale_in.device() == dev &&
                  (!bias_in.has_value() || bias_in->device() == dev),
              "rla::w8a8_gemm: all tensors must be on the same CUDA device");
  c10::cuda::CUDAGuard guard(dev);
  const at::Tensor x = rows_of(x_in), w = rows_of(w_in), x_scale = x_scale_in.contiguous(),
                   scale = scale_in.contiguous();
  at::Tensor bias;
  if (bias_in.has_value()) bias = bias_in->contiguous();
  const int64_t M = x.size(0), K = x.size(1), N = w.size(0);
  at::Tensor y = empty_on(dev, {M, N}, at::kHalf);
  if (M == 0 || N == 0) return y;
  at::Tensor ws;
  if (K > 0 && (!rows_aligned(x) || !rows_aligned(w)))
    ws = empty_on(dev, {static_cast<int64_t>(rla_w8a8_workspace_size(M, N, K))}, at::kByte);
  check_status(
      rla_w8a8_gemm(static_cast<const int8_t*>(x.data_ptr()), row_stride(x), static_cast<const float*>(x_scale.data_ptr()),
                    static_cast<const int8_t*>(w.data_ptr()), row_stride(w), scale.data_ptr(),
                    scale_dtype_of(scale, "scale"), bias.defined() ? bias.data_ptr() : nullptr,
                    bias.defined() ? scale_dtype_of(bias, "bias") : RLA_DTYPE_NONE, y.data_ptr(), N, M, N, K,
                    ws.defined() ? ws.data_ptr() : nullptr, ws.defined() ? static_cast<size_t>(ws.numel()) : 0,
                    stream_of(dev)),
      "rla_w8a8_gemm");
  return y;
}

void check_moe_args(const at::Tensor& x, const at::Tensor& router, const at::Tensor& w_gate, const at::Tensor& s_gate,
                    const at::Tensor& w_up, const at::Tensor& s_up, const at::Tensor& w_down, const at::Tensor& s_down,
                    int64_t top_k) {
  TORCH_CHECK(x.dim() == 2 && x.scalar_type() == at::kHalf, "rla::moe: x must be a 2-D float16 tensor");
  TORCH_CHECK_TYPE(router.dim() == 2 && router.scalar_type() == at::kHalf,
                   "rla::moe: router_weight must be a 2-D float16 tensor");
  TORCH_CHECK(w_gate.scalar_type() == at::kChar && w_up.scalar_type() == at::kChar && w_down.scalar_type() == at::kChar,
              "Weight must be INT8");
  const int64_t E = router.size(0), H = x.size(1);
  TORCH_CHECK(router.size(1) == H, "Router shape mismatch: ", router.sizes(), " vs (", E, ", ", H, ")");
  TORCH_CHECK(w_gate.dim() == 3 && w_gate.size(0) == E && w_gate.size(2) == H && w_up.sizes() == w_gate.sizes(),
              "Weight shape mismatch: ", w_gate.sizes(), " / ", w_up.sizes(), " vs (", E, ", intermediate, ", H, ")");
  const int64_t I = w_gate.size(1);
  TORCH_CHECK(w_down.dim() == 3 && w_down.size(0) == E && w_down.size(1) == H && w_down.size(2) == I,
              "Weight shape mismatch: ", w_down.sizes(), " vs (", E, ", ", H, ", ", I, ")");
  TORCH_CHECK(s_gate.dim() == 2 && s_gate.size(0) == E && s_gate.size(1) == I && s_up.sizes() == s_gate.sizes() &&
                  s_down.dim() == 2 && s_down.size(0) == E && s_down.size(1) == H,
              "Scale shape mismatch: ", s_gate.sizes(), " / ", s_up.sizes(), " / ", s_down.sizes());
  scale_dtype_of(s_gate, "rla::moe: scales");
  TORCH_CHECK_TYPE(s_up.scalar_type() == s_gate.scalar_type() && s_down.scalar_type() == s_gate.scalar_type(),
                   "rla::moe: the three scales must have one dtype");
  TORCH_CHECK(w_gate.is_contiguous() && w_up.is_contiguous() && w_down.is_contiguous(),
              "rla::moe: expert weights must be contiguous");
  TORCH_CHECK(top_k >= 1 && top_k <= E, "rla::moe: top_k must be in [1, ", E, "], got ", top_k);
}
at::Tensor moe_meta(const at::Tensor& x, const at::Tensor& router, const at::Tensor& w_gate, const at::Tensor& s_gate,
                    const at::Tensor& w_up, const at::Tensor& s_up, const at::Tensor& w_down, const at::Tensor& s_down,
                    int64_t top_k, bool) {
  check_moe_args(x, router, w_gate, s_gate, w_up, s_up, w_down, s_down, top_k);
  return at::empty(x.sizes(), x.options());
}
at::Tensor moe_cuda(const at::Tensor& x_in, const at::Tensor& router_in, const at::Tensor& w_gate,
                    const at::Tensor& s_gate_in, const at::Tensor& w_up, const at::Tensor& s_up_in,
                    const at::Tensor& w_down, const at::Tensor& s_down_in, int64_t top_k, bool renormalize) {
  check_moe_args(x_in, router_in, w_gate, s_gate_in, w_up, s_up_in, w_down, s_down_in, top_k);
  const at::Device dev = x_in.device();
  TORCH_CHECK(dev.is_cuda() && router_in.device() == dev && w_gate.device() == dev && w_up.device() == dev &&
                  w_down.device() == dev && s_gate_in.device() == dev && s_up_in.device() == dev &&
                  s_down_in.device() == dev,
              "rla::moe: all tensors must be on the same CUDA device");
  c10::cuda::CUDAGuard guard(dev);
  // small operands may come in any layout; the kernel reads them in 16-byte pieces
  auto aligned = [](const at::Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) == 0; };
  at::Tensor x = rows_of(x_in), router = router_in.contiguous();
  if (!aligned(x) || (x.size(0) > 1 && x.stride(0) % 8 != 0)) x = x.clone(at::MemoryFormat::Contiguous);
  if (!aligned(router)) router = router.clone();
  const at::Tensor s_gate = s_gate_in.contiguous(), s_up = s_up_in.contiguous(), s_down = s_down_in.contiguous();
  const int64_t T = x.size(0), H = x.size(1), I = w_gate.size(1), E = router.size(0);
  at::Tensor y = empty_on(dev, {T, H}, at::kHalf);
  const int64_t most = std::min<int64_t>(T, RLA_MOE_MAX_TOKENS);
  const size_t need = rla_moe_workspace_size(most, I, top_k);
  at::Tensor ws = empty_on(dev, {static_cast<int64_t>(need)}, at::kByte);
  // longer batches RLA_MOE_MAX_TOKENS rows at a time, in stream order on one scratch
  for (int64_t t0 = 0; t0 < T || t0 == 0; t0 += RLA_MOE_MAX_TOKENS) {
    const int64_t rows = std::min<int64_t>(T - t0, RLA_MOE_MAX_TOKENS);
    check_status(rla_moe(static_cast<const at::Half*>(x.data_ptr()) + t0 * row_stride(x), row_stride(x),
                         router.data_ptr(), static_cast<const int8_t*>(w_gate.data_ptr()), s_gate.data_ptr(),
                         static_cast<const int8_t*>(w_up.data_ptr()), s_up.data_ptr(),
                         static_cast<const int8_t*>(w_down.data_ptr()), s_down.data_ptr(),
                         scale_dtype_of(s_gate, "scales"), renormalize ? 1 : 0,
                         static_cast<at::Half*>(y.data_ptr()) + t0 * H, H, rows, H, I, E, top_k,
                         need ? ws.data_ptr() : nullptr, need, stream_of(dev)),
                 "rla_moe");
  }
  return y;
}

}  // namespace

PYBIND11_MODULE(_rla_torch_ops, m) {
  m.def("w8a16_gemm", &w8a16_gemm_cuda, "rla::w8a16_gemm's CUDA kernel function, called without the dispatcher",
        pybind11::arg("x"), pybind11::arg("weight_int8"), pybind11::arg("scale"),
        pybind11::arg("bias") = pybind11::none());
  m.def("add_rmsnorm", &add_rmsnorm, "RMSNorm of x + residual: (y, h)");
  m.def("add_rmsnorm_int8", &add_rmsnorm_int8, "RMSNorm of x + residual in int8: (q, scale, h)");
  m.def("swiglu_int8", &swiglu_int8_cuda, "silu(gate) * up in int8: (q, scale)");
  m.def("w8a8_gemm", &w8a8_gemm_cuda, "int8 rows times int8 weights: fp16 [M, N]");
  m.def("moe", &moe_cuda, "mixture-of-experts layer with int8 experts: fp16 [T, H]");
}

TORCH_LIBRARY(rla, m) {
  m.def("w8a16_gemm(Tensor x, Tensor weight_int8, Tensor scale, Tensor? bias=None) -> Tensor");
  m.def("add_rmsnorm(Tensor x, Tensor residual, Tensor weight, float eps=1e-06) -> (Tensor, Tensor)");
  m.def("add_rmsnorm_int8(Tensor x, Tensor residual, Tensor weight, float eps=1e-06) -> (Tensor, Tensor, Tensor)");
  m.def("swiglu_int8(Tensor gate, Tensor up) -> (Tensor, Tensor)");
  m.def("w8a8_gemm(Tensor x_int8, Tensor x_scale, Tensor weight_int8, Tensor scale, Tensor? bias=None) -> Tensor");
  m.def("moe(Tensor x, Tensor router_weight, Tensor w_gate, Tensor scale_gate, Tensor w_up, Tensor scale_up, "
        "Tensor w_down, Tensor scale_down, int top_k, bool renormalize=True) -> Tensor");
}
TORCH_LIBRARY_IMPL(rla, CUDA, m) {
  m.impl("w8a16_gemm", &w8a16_gemm_cuda);
  m.impl("add_rmsnorm", &add_rmsnorm_op);
  m.impl("add_rmsnorm_int8", &add_rmsnorm_int8_op);
  m.impl("swiglu_int8", &swiglu_int8_cuda);
  m.impl("w8a8_gemm", &w8a8_gemm_cuda);
  m.impl("moe", &moe_cuda);
}
TORCH_LIBRARY_IMPL(rla, Meta, m) {
  m.impl("w8a16_gemm", &w8a16_gemm_meta);
  m.impl("add_rmsnorm", &add_rmsnorm_meta);
  m.impl("add_rmsnorm_int8", &add_rmsnorm_int8_meta);
  m.impl("swiglu_int8", &swiglu_int8_meta);
  m.impl("w8a8_gemm", &w8a8_gemm_meta);
  m.impl("moe", &moe_meta);
}
