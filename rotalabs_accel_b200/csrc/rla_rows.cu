// Row-wise kernels of the 8-bit activation path: RMSNorm with the residual's
// addition (16-bit or 8-bit output) and SwiGLU with an 8-bit output.
//
// Mathematics.  For a row of length K, in fp32 from 16-bit inputs:
//   norm    h = T(x + residual),  r = rsqrt(mean(h^2) + eps),  v = h * r * w
//   SwiGLU  v = silu(gate) * up
// 16-bit output: T(v).  8-bit output: s = max|v| / 127 (1 for a zero row),
// q = rint(v / s).  In the norm's 8-bit form r is a common factor of the row,
// so q = rint(p * 127 / max|p|) with p = h * w: the maximum does not have to
// wait for the mean, both statistics come out of ONE pass and one reduction,
// and r only enters the scale.  A row that holds an infinity or NaN gets the
// scale NaN and q = 0 (the maximum propagates NaN), so the row dequantizes to
// NaN instead of to a plausible number.
//
// Bound by memory: every input is read once and every output written once.
// A row is held in registers (EPT elements a thread) between the reduction
// and the output, so nothing is read twice up to 1024 * 32 = 32768 columns;
// longer rows are read a second time.
#include <cuda_bf16.h>

#include <algorithm>

#include "rla_common.cuh"
#include "rla_internal.h"

namespace rla {

enum RowsOp { kRowsNorm = 0, kRowsNormInt8 = 1, kRowsSwiGLUInt8 = 2 };

struct RowsArgs {
  const void* a;  // x, or gate
  int64_t lda;
  const void* b;  // residual (may be null), or up
  int64_t ldb;
  const void* weight;  // norm only
  int weight_dtype;
  float eps;
  void* h;  // norm with a residual: the sum
  int64_t ldh;
  void* y;  // 16-bit output, or int8
  int64_t ldy;
  float* scale;  // 8-bit output only
  int64_t M;
  int K;
};

template <typename T, int V>
struct alignas(sizeof(T) * V) RowVec {
  T v[V];
};

RLA_DEVFN float rows_to_f(__half v) { return __half2float(v); }
RLA_DEVFN float rows_to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
RLA_DEVFN T rows_from_f(float v);
template <>
RLA_DEVFN __half rows_from_f<__half>(float v) { return __float2half_rn(v); }
template <>
RLA_DEVFN __nv_bfloat16 rows_from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// max that keeps a NaN (fmaxf drops it)
RLA_DEVFN float rows_max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

template <int V>
RLA_DEVFN void rows_load_weight(const void* w, int dtype, int k, float (&out)[V]) {
  if (dtype == RLA_DTYPE_F32) {
    const float* p = static_cast<const float*>(w) + k;
    if constexpr (V >= 4) {
#pragma unroll
      for (int i = 0; i < V; i += 4) {
        const float4 f = *reinterpret_cast<const float4*>(p + i);
        out[i] = f.x, out[i + 1] = f.y, out[i + 2] = f.z, out[i + 3] = f.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) out[i] = p[i];
    }
  } else if (dtype == RLA_DTYPE_F16) {
    const RowVec<__half, V> p = *reinterpret_cast<const RowVec<__half, V>*>(static_cast<const __half*>(w) + k);
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = __half2float(p.v[i]);
  } else {
    const RowVec<__nv_bfloat16, V> p =
        *reinterpret_cast<const RowVec<__nv_bfloat16, V>*>(static_cast<const __nv_bfloat16*>(w) + k);
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = __bfloat162float(p.v[i]);
  }
}

// One vector of a row: p (norm: h * w, SwiGLU: v), and for the norm the sum of
// h^2 added to ss and h stored when `store` says so.
template <typename T, int V, int OP>
RLA_DEVFN void rows_vector(const RowsArgs& g, int64_t row, int k, bool store, float (&p)[V], float& ss) {
  using Vec = RowVec<T, V>;
  const Vec a = *reinterpret_cast<const Vec*>(static_cast<const T*>(g.a) + row * g.lda + k);
  if constexpr (OP == kRowsSwiGLUInt8) {
    const Vec b = *reinterpret_cast<const Vec*>(static_cast<const T*>(g.b) + row * g.ldb + k);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float f = rows_to_f(a.v[i]);
      // silu = f / (1 + e^-f); the intrinsics' few ulp are far below the
      // 8-bit step, and move the scale by less than 1e-6 of itself
      p[i] = __fdividef(f, 1.0f + __expf(-f)) * rows_to_f(b.v[i]);
    }
  } else {
    Vec h = a;
    if (g.b) {
      const Vec b = *reinterpret_cast<const Vec*>(static_cast<const T*>(g.b) + row * g.ldb + k);
      // the residual stream has the activations' type: one rounding, and the
      // norm is taken of the rounded sum, which is what later layers read
#pragma unroll
      for (int i = 0; i < V; ++i) h.v[i] = rows_from_f<T>(rows_to_f(a.v[i]) + rows_to_f(b.v[i]));
      if (store) *reinterpret_cast<Vec*>(static_cast<T*>(g.h) + row * g.ldh + k) = h;
    }
    float w[V];
    rows_load_weight<V>(g.weight, g.weight_dtype, k, w);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float f = rows_to_f(h.v[i]);
      ss = fmaf(f, f, ss);
      p[i] = f * w[i];
    }
  }
}

// blockDim = (threads of a row, rows of a CTA); rows of one warp need no
// barrier.  T: fp16 or bf16.  V: elements of a load.  EPT: elements a thread
// holds.
template <typename T, int V, int EPT, int OP>
__global__ void __launch_bounds__(1024) rows_kernel(const RowsArgs g) {
  constexpr int NV = EPT / V;
  rla_griddep_launch_dependents();
  rla_griddep_wait();  // nothing is read or written before the previous kernel has finished
  const int64_t row = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y;
  const bool live = row < g.M;
  const int chunk = blockDim.x * EPT;
  const bool held = g.K <= chunk;  // the whole row stays in registers

  float p[NV][V];
  float ss = 0.f, top = 0.f;
  if (live) {
    for (int c0 = 0; c0 < g.K; c0 += chunk) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int k = c0 + (j * blockDim.x + threadIdx.x) * V;
        if (k < g.K) {
          rows_vector<T, V, OP>(g, row, k, true, p[j], ss);
          if constexpr (OP != kRowsNorm) {
#pragma unroll
            for (int i = 0; i < V; ++i) top = rows_max_nan(top, fabsf(p[j][i]));
          }
        }
      }
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    if constexpr (OP != kRowsSwiGLUInt8) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if constexpr (OP != kRowsNorm) top = rows_max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
  }
  if (blockDim.x > 32) {  // one row a CTA
    __shared__ float2 red[32];
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = make_float2(ss, top);
    __syncthreads();
    const int warps = blockDim.x >> 5;
    const float2 v = (threadIdx.x & 31) < warps ? red[threadIdx.x & 31] : make_float2(0.f, 0.f);
    ss = v.x;
    top = v.y;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      if constexpr (OP != kRowsSwiGLUInt8) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      if constexpr (OP != kRowsNorm) top = rows_max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
    }
  }
  if (!live) return;

  float r = 1.f;
  if constexpr (OP != kRowsSwiGLUInt8) r = g.K > 0 ? rsqrtf(ss / static_cast<float>(g.K) + g.eps) : 1.f;
  float inv = 0.f;
  bool divide = false;
  if constexpr (OP != kRowsNorm) {
    const float vmax = top * r;
    float s = vmax / 127.f;
    if (!(vmax < INFINITY)) {
      s = NAN;  // q = 0: inv stays 0 and the products below are not used
    } else if (s == 0.f) {
      s = 1.f;
    } else {
      // 127 / max overflows below 4e-37: such rows divide element by element
      divide = top < 1e-30f;
      inv = divide ? 1.f : 127.f / top;
    }
    if (threadIdx.x == 0) g.scale[row] = s;
  }

  for (int c0 = 0; c0 < g.K; c0 += chunk) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int k = c0 + (j * blockDim.x + threadIdx.x) * V;
      if (k >= g.K) continue;
      float unused = 0.f;
      if (!held) rows_vector<T, V, OP>(g, row, k, false, p[j], unused);
      if constexpr (OP == kRowsNorm) {
        RowVec<T, V> o;
#pragma unroll
        for (int i = 0; i < V; ++i) o.v[i] = rows_from_f<T>(p[j][i] * r);
        *reinterpret_cast<RowVec<T, V>*>(static_cast<T*>(g.y) + row * g.ldy + k) = o;
      } else {
        RowVec<int8_t, V> o;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float t = divide ? __fdiv_rn(p[j][i], top) * 127.f : p[j][i] * inv;
          o.v[i] = inv == 0.f ? int8_t(0) : static_cast<int8_t>(__float2int_rn(fminf(fmaxf(t, -127.f), 127.f)));
        }
        *reinterpret_cast<RowVec<int8_t, V>*>(static_cast<int8_t*>(g.y) + row * g.ldy + k) = o;
      }
    }
  }
}

template <typename T, int V, int EPT>
static cudaError_t launch_rows_cfg(const RowsArgs& g, int op, cudaStream_t s) {
  const int tx = std::min(1024, std::max(32, (g.K / EPT + (g.K % EPT != 0) + 31) / 32 * 32));
  const int ty = tx == 32 ? 4 : 1;
  const int64_t blocks = (g.M + ty - 1) / ty;
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(tx, ty);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  switch (op) {
    case kRowsNorm: return cudaLaunchKernelEx(&cfg, rows_kernel<T, V, EPT, kRowsNorm>, g);
    case kRowsNormInt8: return cudaLaunchKernelEx(&cfg, rows_kernel<T, V, EPT, kRowsNormInt8>, g);
    default: return cudaLaunchKernelEx(&cfg, rows_kernel<T, V, EPT, kRowsSwiGLUInt8>, g);
  }
}

// Elements of a load: the most that every row of every operand is aligned to.
static int rows_vector_width(const RowsArgs& g, int op) {
  auto fits = [&](int v) {
    auto ok = [&](const void* p, int64_t ld, int64_t size) {
      return p == nullptr || (reinterpret_cast<uintptr_t>(p) % (v * size) == 0 && (g.M == 1 || ld % v == 0));
    };
    bool w = true;
    if (op != kRowsSwiGLUInt8) {
      const int64_t ws = g.weight_dtype == RLA_DTYPE_F32 ? 4 : 2;
      const int64_t bytes = ws == 4 && v >= 4 ? 16 : v * ws;  // fp32 weights: 16-byte loads at most
      w = reinterpret_cast<uintptr_t>(g.weight) % bytes == 0;
    }
    return g.K % v == 0 && w && ok(g.a, g.lda, 2) && ok(g.b, g.ldb, 2) && ok(g.h, g.ldh, 2) &&
           ok(g.y, g.ldy, op == kRowsNorm ? 2 : 1);
  };
  return fits(8) ? 8 : fits(4) ? 4 : 1;
}

template <typename T>
static cudaError_t launch_rows(const RowsArgs& g, int op, cudaStream_t s) {
  const bool small = g.K <= 8 * 1024;
  switch (rows_vector_width(g, op)) {
    case 8: return small ? launch_rows_cfg<T, 8, 8>(g, op, s) : launch_rows_cfg<T, 8, 32>(g, op, s);
    case 4: return small ? launch_rows_cfg<T, 4, 8>(g, op, s) : launch_rows_cfg<T, 4, 32>(g, op, s);
    default: return small ? launch_rows_cfg<T, 1, 8>(g, op, s) : launch_rows_cfg<T, 1, 32>(g, op, s);
  }
}

static int rows_fail(int code, const char* what, const char* msg) {
  set_error("%s: %s", what, msg);
  return code;
}

static int run_rows(const char* what, const RowsArgs& g, int op, int dtype, int64_t K, void* stream) {
  const bool norm = op != kRowsSwiGLUInt8;
  if (g.M < 0 || K < 0 || g.M > INT32_MAX || K > (int64_t(1) << 30))  // column indices are 32 bits, a chunk beyond K
    return rows_fail(RLA_ERR_INVALID_ARGUMENT, what, "rows must be in [0, 2^31), columns in [0, 2^30]");
  if (dtype != RLA_DTYPE_F16 && dtype != RLA_DTYPE_BF16)
    return rows_fail(RLA_ERR_INVALID_ARGUMENT, what, "dtype must be F16 or BF16");
  if (norm && g.weight_dtype != RLA_DTYPE_F32 && g.weight_dtype != RLA_DTYPE_F16 && g.weight_dtype != RLA_DTYPE_BF16)
    return rows_fail(RLA_ERR_INVALID_ARGUMENT, what, "weight_dtype must be F32, F16 or BF16");
  if (norm && !(g.eps >= 0.f)) return rows_fail(RLA_ERR_INVALID_ARGUMENT, what, "eps must be >= 0");
  if (g.M == 0) return RLA_OK;
  if (op != kRowsNorm && !g.scale) return rows_fail(RLA_ERR_INVALID_ARGUMENT, what, "null scale");
  if (K > 0) {
    if (!g.a || !g.y || (norm && !g.weight) || (!norm && !g.b) || (norm && g.b && !g.h))
      return rows_fail(RLA_ERR_INVALID_ARGUMENT, what, "null pointer");
    if (g.lda < K || (g.b && g.ldb < K) || (norm && g.b && g.ldh < K) || g.ldy < K)
      return rows_fail(RLA_ERR_INVALID_ARGUMENT, what, "leading dimensions must be >= the row length");
  } else if (op == kRowsNorm) {
    return RLA_OK;  // no element to write
  }
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = dtype == RLA_DTYPE_F16 ? launch_rows<__half>(g, op, s) : launch_rows<__nv_bfloat16>(g, op, s);
  if (e != cudaSuccess) {
    set_error("%s: %s", what, cudaGetErrorString(e));
    return RLA_ERR_CUDA;
  }
  note_launch();
  return RLA_OK;
}

}  // namespace rla

extern "C" {

int rla_add_rmsnorm(const void* x, int64_t ldx, const void* residual, int64_t ldr, int dtype, const void* weight,
                    int weight_dtype, float eps, void* h, int64_t ldh, void* y, int64_t ldy, int64_t M, int64_t K,
                    void* stream) {
  const rla::RowsArgs g{x, ldx, residual, ldr, weight, weight_dtype, eps, residual ? h : nullptr, ldh, y, ldy, nullptr,
                        M, static_cast<int>(K)};
  return rla::run_rows("rla_add_rmsnorm", g, rla::kRowsNorm, dtype, K, stream);
}

int rla_add_rmsnorm_int8(const void* x, int64_t ldx, const void* residual, int64_t ldr, int dtype, const void* weight,
                         int weight_dtype, float eps, void* h, int64_t ldh, int8_t* q, int64_t ldq, float* scale,
                         int64_t M, int64_t K, void* stream) {
  const rla::RowsArgs g{x, ldx, residual, ldr, weight, weight_dtype, eps, residual ? h : nullptr, ldh, q, ldq, scale,
                        M, static_cast<int>(K)};
  return rla::run_rows("rla_add_rmsnorm_int8", g, rla::kRowsNormInt8, dtype, K, stream);
}

int rla_swiglu_int8(const void* gate, int64_t ldg, const void* up, int64_t ldu, int dtype, int8_t* q, int64_t ldq,
                    float* scale, int64_t M, int64_t N, void* stream) {
  const rla::RowsArgs g{gate, ldg, up, ldu, nullptr, RLA_DTYPE_NONE, 0.f, nullptr, 0, q, ldq, scale,
                        M, static_cast<int>(N)};
  return rla::run_rows("rla_swiglu_int8", g, rla::kRowsSwiGLUInt8, dtype, N, stream);
}

}  // extern "C"
