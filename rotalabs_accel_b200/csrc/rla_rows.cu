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
// longer rows are read a second time.  Many rows run through persistent CTAs
// that have the next rows on their way while one is reduced (below).  SwiGLU has
// some 11 instructions an element, two of them on the special-function unit, so
// the quantization is one FMA: p * (127 / max) + 1.5 * 2^23 rounds to nearest
// even in the last bit of the sum, whose low byte is q.
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

// silu(f) = f / (1 + e^-f) for f > -87 (so that nothing is flushed: e^87 < 2^126; saving
// the instructions that scale subnormals).  Its relative error is at most 2^-20, and for
// negative f also |f| 2^-23.7 from the rounding of f log2(e) and of log2(e): far below
// the 8-bit step, and up to 6e-6 of a scale that comes from a gate of -87.
RLA_DEVFN float rows_silu(float f) {
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(f * -1.44269504f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
  return f * r;
}
// v = silu(a) * b; `low`: the lowest a so far, in two 16-bit halves.
template <typename T>
struct RowsPair {
  using type = __half2;
};
template <>
struct RowsPair<__nv_bfloat16> {
  using type = __nv_bfloat162;
};
template <typename T, int V>
RLA_DEVFN void rows_swiglu(const RowVec<T, V>& a, const RowVec<T, V>& b, float (&p)[V], typename RowsPair<T>::type& low) {
  using Pair = typename RowsPair<T>::type;
#pragma unroll
  for (int i = 0; i < V; ++i) p[i] = rows_silu(rows_to_f(a.v[i])) * rows_to_f(b.v[i]);
#pragma unroll
  for (int i = 0; i < V; i += 2) low = __hmin2(low, Pair{a.v[i], a.v[V > 1 ? i + 1 : i]});
}
// Gates below -87 are rare, and v there is 0 so far: the callers look once at the
// lowest and set those v (a test at each took 1.7 us of 26 at 2048 x 11008).
template <typename Pair>
RLA_DEVFN bool rows_far(const Pair& low) {
  return __builtin_expect(fminf(rows_to_f(low.x), rows_to_f(low.y)) < -87.f, 0);
}
template <typename T, int V>
RLA_DEVFN void rows_swiglu_far(const RowVec<T, V>& a, const RowVec<T, V>& b, float (&p)[V], float& top) {
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const float f = rows_to_f(a.v[i]);
    if (f < -87.f) p[i] = rla_silu_mul(f, rows_to_f(b.v[i]));
    top = rows_max_nan(top, fabsf(p[i]));
  }
}
// The residual stream has the activations' type: one rounding, and the norm is
// taken of the rounded sum, which is what later layers read.
template <typename T, int V>
RLA_DEVFN RowVec<T, V> rows_add(const RowVec<T, V>& a, const RowVec<T, V>& b) {
  RowVec<T, V> h;
#pragma unroll
  for (int i = 0; i < V; ++i) h.v[i] = rows_from_f<T>(rows_to_f(a.v[i]) + rows_to_f(b.v[i]));
  return h;
}
template <typename T, int V>
RLA_DEVFN void rows_weigh(const RowVec<T, V>& h, const float (&w)[V], float (&p)[V], float& ss) {
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const float f = rows_to_f(h.v[i]);
    ss = fmaf(f, f, ss);
    p[i] = f * w[i];
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
    typename RowsPair<T>::type low{rows_from_f<T>(0.f), rows_from_f<T>(0.f)};
    rows_swiglu(a, b, p, low);
    float unused = 0.f;
    if (rows_far(low)) rows_swiglu_far(a, b, p, unused);
  } else {
    Vec h = a;
    if (g.b) {
      h = rows_add(a, *reinterpret_cast<const Vec*>(static_cast<const T*>(g.b) + row * g.ldb + k));
      if (store) *reinterpret_cast<Vec*>(static_cast<T*>(g.h) + row * g.ldh + k) = h;
    }
    float w[V];
    rows_load_weight<V>(g.weight, g.weight_dtype, k, w);
    rows_weigh(h, w, p, ss);
  }
}

// What the statistics of a row make of its values.
struct RowsScale {
  float r = 1.f;        // 1 / rms (norm)
  float top;            // max |p|
  float inv = 0.f;      // q = rint(p * inv); 0: the row's q are 0
  bool divide = false;  // q = rint(p / top * inv)
  float scale = 0.f;
};
template <int OP>
RLA_DEVFN RowsScale rows_scale(const RowsArgs& g, float ss, float top) {
  RowsScale c;
  c.top = top;
  if constexpr (OP != kRowsSwiGLUInt8) c.r = g.K > 0 ? rsqrtf(ss / static_cast<float>(g.K) + g.eps) : 1.f;
  if constexpr (OP != kRowsNorm) {
    const float vmax = top * c.r;
    c.scale = vmax / 127.f;
    if (!(vmax < INFINITY)) {
      c.scale = NAN;
    } else if (c.scale == 0.f) {
      c.scale = 1.f;
    } else {
      // 127 / max overflows below 4e-37: such rows divide element by element
      c.divide = top < 1e-30f;
      c.inv = c.divide ? 127.f : 127.f / top;
    }
  }
  return c;
}
template <typename T, int V, int OP>
RLA_DEVFN void rows_store(const RowsArgs& g, int64_t row, int k, const RowsScale& c, float (&p)[V]) {
  if constexpr (OP == kRowsNorm) {
    RowVec<T, V> o;
#pragma unroll
    for (int i = 0; i < V; ++i) o.v[i] = rows_from_f<T>(p[i] * c.r);
    *reinterpret_cast<RowVec<T, V>*>(static_cast<T*>(g.y) + row * g.ldy + k) = o;
  } else {
    if (c.divide) {
#pragma unroll
      for (int i = 0; i < V; ++i) p[i] = __fdiv_rn(p[i], c.top);
    }
    uint32_t q[V];
#pragma unroll
    for (int i = 0; i < V; ++i) q[i] = c.inv == 0.f ? 0u : __float_as_uint(fmaf(p[i], c.inv, 12582912.f));
    int8_t* to = static_cast<int8_t*>(g.y) + row * g.ldy + k;
    if constexpr (V == 1) {
      *to = static_cast<int8_t>(q[0]);
    } else {
      uint32_t o[V / 4];
#pragma unroll
      for (int i = 0; i < V; i += 4)
        o[i / 4] = __byte_perm(__byte_perm(q[i], q[i + 1], 0x0040), __byte_perm(q[i + 2], q[i + 3], 0x0040), 0x5410);
      if constexpr (V == 4)
        *reinterpret_cast<uint32_t*>(to) = o[0];
      else
        *reinterpret_cast<uint2*>(to) = make_uint2(o[0], o[1]);
    }
  }
}
// Sum of ss and maximum of top over a warp.
template <int OP>
RLA_DEVFN void rows_reduce_warp(float& ss, float& top) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    if constexpr (OP != kRowsSwiGLUInt8) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if constexpr (OP != kRowsNorm) top = rows_max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
  }
}

// blockDim = (threads of a row, rows of a CTA); rows of one warp need no
// barrier.  T: fp16 or bf16.  V: elements of a load.  EPT: elements a thread
// holds.
template <typename T, int V, int EPT, int MAXT, int OP>
__global__ void __launch_bounds__(MAXT, EPT == 8 ? 2 : 1) rows_kernel(const RowsArgs g) {
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
  rows_reduce_warp<OP>(ss, top);
  if (blockDim.x > 32) {  // one row a CTA
    __shared__ float2 red[32];
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = make_float2(ss, top);
    __syncthreads();
    const int warps = blockDim.x >> 5;
    const float2 v = (threadIdx.x & 31) < warps ? red[threadIdx.x & 31] : make_float2(0.f, 0.f);
    ss = v.x;
    top = v.y;
    rows_reduce_warp<OP>(ss, top);
  }
  if (!live) return;

  const RowsScale c = rows_scale<OP>(g, ss, top);
  if (OP != kRowsNorm && threadIdx.x == 0) g.scale[row] = c.scale;
  for (int c0 = 0; c0 < g.K; c0 += chunk) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int k = c0 + (j * blockDim.x + threadIdx.x) * V;
      if (k >= g.K) continue;
      float unused = 0.f;
      if (!held) rows_vector<T, V, OP>(g, row, k, false, p[j], unused);
      rows_store<T, V, OP>(g, row, k, c, p[j]);
    }
  }
}

// ---------------------------------------------------------------------------
// Many rows, 16-byte aligned.  A CTA of the kernel above waits for its row,
// then for its reduction, and only other CTAs fill that time: 0.60 of the
// memory's rate (2048 x 4096, 14.9 us).  Here a persistent CTA takes every
// gridDim.x-th row from a ring in shared memory that bulk copies fill: the next
// rows are on their way through every wait, and a row costs one barrier.  The
// norm's weight stays in registers (HOLDW) where there is room.
// ---------------------------------------------------------------------------
constexpr int kRowsMaxStages = 4;
// `bytes` contiguous bytes (a multiple of 16, both ends 16-byte aligned) into this CTA's shared memory.
RLA_DEVFN void rows_bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   rla_smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(rla_smem_u32(bar))
               : "memory");
}

template <typename T, int NV, int MAXT, int CTAS, bool HOLDW, int OP>
__global__ void __launch_bounds__(MAXT, CTAS) rows_stream_kernel(const RowsArgs g, int stages, int row_bytes) {
  using Vec = RowVec<T, 8>;
  extern __shared__ __align__(128) uint8_t rows_ring[];  // [stages][a row, b row]
  __shared__ uint64_t full[kRowsMaxStages];
  __shared__ float2 red[2][32];
  __shared__ int abort_word;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
  const bool two = g.b != nullptr;
  if (tid == 0) {
    for (int s = 0; s < stages; ++s) rla_mbar_init(&full[s], 1);
    abort_word = 0;
    rla_fence_barrier_init();
  }
  __syncthreads();
  rla_griddep_launch_dependents();
  rla_griddep_wait();  // nothing is read or written before the previous kernel has finished

  auto issue = [&](int64_t row, int s) {  // thread 0
    uint8_t* to = rows_ring + (size_t)s * 2 * row_bytes;
    rla_mbar_arrive_expect_tx(&full[s], two ? 2 * row_bytes : row_bytes);
    rows_bulk_load(to, static_cast<const T*>(g.a) + row * g.lda, row_bytes, &full[s]);
    if (two) rows_bulk_load(to + row_bytes, static_cast<const T*>(g.b) + row * g.ldb, row_bytes, &full[s]);
  };
  if (tid == 0)
    for (int s = 0; s < stages; ++s)
      if (blockIdx.x + (int64_t)s * gridDim.x < g.M) issue(blockIdx.x + (int64_t)s * gridDim.x, s);

  float w[HOLDW ? NV : 1][8];
  if constexpr (HOLDW) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int k = (j * blockDim.x + tid) * 8;
      if (k < g.K) rows_load_weight<8>(g.weight, g.weight_dtype, k, w[j]);
    }
  }

  int s = 0, phase = 0, odd = 0;
  int64_t row = blockIdx.x;
  for (; row < g.M; row += gridDim.x) {
    if (!rla_mbar_wait(&full[s], phase, RLA_DEVERR_TIMEOUT_TMA_FULL, &abort_word)) break;
    const uint8_t* from = rows_ring + (size_t)s * 2 * row_bytes;
    float p[NV][8];
    float ss = 0.f, top = 0.f;
    typename RowsPair<T>::type low{rows_from_f<T>(0.f), rows_from_f<T>(0.f)};
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int k = (j * blockDim.x + tid) * 8;
      if (k >= g.K) continue;
      const Vec a = *reinterpret_cast<const Vec*>(from + k * 2);
      if constexpr (OP == kRowsSwiGLUInt8) {
        rows_swiglu(a, *reinterpret_cast<const Vec*>(from + row_bytes + k * 2), p[j], low);
      } else {
        Vec h = a;
        if (two) {
          h = rows_add(a, *reinterpret_cast<const Vec*>(from + row_bytes + k * 2));
          *reinterpret_cast<Vec*>(static_cast<T*>(g.h) + row * g.ldh + k) = h;
        }
        if constexpr (!HOLDW) rows_load_weight<8>(g.weight, g.weight_dtype, k, w[0]);
        rows_weigh(h, w[HOLDW ? j : 0], p[j], ss);
      }
      if constexpr (OP != kRowsNorm) {
#pragma unroll
        for (int i = 0; i < 8; ++i) top = rows_max_nan(top, fabsf(p[j][i]));
      }
    }
    if constexpr (OP == kRowsSwiGLUInt8) {
      if (rows_far(low)) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          const int k = (j * blockDim.x + tid) * 8;
          if (k < g.K)
            rows_swiglu_far(*reinterpret_cast<const Vec*>(from + k * 2),
                            *reinterpret_cast<const Vec*>(from + row_bytes + k * 2), p[j], top);
        }
      }
    }
    rows_reduce_warp<OP>(ss, top);
    if (lane == 0) red[odd][warp] = make_float2(ss, top);
    __syncthreads();  // the sums are there, and the ring's slot has been read
    if (tid == 0 && row + (int64_t)stages * gridDim.x < g.M) issue(row + (int64_t)stages * gridDim.x, s);
    const float2 v = lane < warps ? red[odd][lane] : make_float2(0.f, 0.f);
    ss = v.x;
    top = v.y;
    rows_reduce_warp<OP>(ss, top);
    const RowsScale c = rows_scale<OP>(g, ss, top);
    if (OP != kRowsNorm && tid == 0) g.scale[row] = c.scale;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int k = (j * blockDim.x + tid) * 8;
      if (k < g.K) rows_store<T, 8, OP>(g, row, k, c, p[j]);
    }
    odd ^= 1;  // (the other sums may still be read)
    if (++s == stages) s = 0, phase ^= 1;
  }
  // after a wait that gave up: the copies in flight land before the CTA leaves
  if (tid == 0 && abort_word)
    for (int i = 0; i < stages && row + (int64_t)i * gridDim.x < g.M; ++i) {
      rla_mbar_wait(&full[s], phase, RLA_DEVERR_TIMEOUT_TMA_FULL, nullptr);
      if (++s == stages) s = 0, phase ^= 1;
    }
}

template <typename T, int NV, int MAXT, int CTAS, bool HOLDW>
static cudaError_t launch_rows_stream_cfg(const RowsArgs& g, int op, cudaStream_t s) {
  const int row_bytes = g.K * 2;
  const int budget = 216 * 1024 / CTAS;  // of a CTA's shared memory
  const int stages = std::min(kRowsMaxStages, budget / (2 * row_bytes));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(std::min<int64_t>(g.M, (int64_t)CTAS * device_sm_count())));
  cfg.blockDim = dim3((g.K / 8 + NV - 1) / NV <= 32 ? 32 : ((g.K / 8 + NV - 1) / NV + 31) / 32 * 32);
  cfg.dynamicSmemBytes = (size_t)stages * 2 * row_bytes;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  static std::atomic<uint64_t> done[3];
  auto run = [&](auto kern) {
    const cudaError_t e = allow_smem(kern, budget, done[op]);
    return e != cudaSuccess ? e : cudaLaunchKernelEx(&cfg, kern, g, stages, row_bytes);
  };
  switch (op) {
    case kRowsNorm: return run(rows_stream_kernel<T, NV, MAXT, CTAS, HOLDW, kRowsNorm>);
    case kRowsNormInt8: return run(rows_stream_kernel<T, NV, MAXT, CTAS, HOLDW, kRowsNormInt8>);
    default: return run(rows_stream_kernel<T, NV, MAXT, CTAS, false, kRowsSwiGLUInt8>);
  }
}

template <typename T, int V, int EPT, int MAXT>
static cudaError_t launch_rows_cfg(const RowsArgs& g, int op, cudaStream_t s) {
  const int tx = std::min(MAXT, std::max(32, (g.K / EPT + (g.K % EPT != 0) + 31) / 32 * 32));
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
    case kRowsNorm: return cudaLaunchKernelEx(&cfg, rows_kernel<T, V, EPT, MAXT, kRowsNorm>, g);
    case kRowsNormInt8: return cudaLaunchKernelEx(&cfg, rows_kernel<T, V, EPT, MAXT, kRowsNormInt8>, g);
    default: return cudaLaunchKernelEx(&cfg, rows_kernel<T, V, EPT, MAXT, kRowsSwiGLUInt8>, g);
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

// Threads of a row and elements of a thread.  Few rows (fewer than four for
// each SM) wait for one round of loads: as many threads as there are, up to
// 1024 (333 x 4100 in bf16: 4.5 us, 9.6 with 32 elements a thread).  Many rows
// that the stream cannot take: 256 threads or fewer with up to 32 elements
// each, so that several rows are on their way in an SM while others reduce.
template <typename T, int V>
static cudaError_t launch_rows_width(const RowsArgs& g, int op, cudaStream_t s) {
  const bool many = g.M >= 4 * device_sm_count();
  if constexpr (V == 8) {
    // CTAs an SM, threads and stages by measurement: 2048 x 4096 int8 14.0 us
    // with three CTAs, 16.6 with two; 4096 x 8192 bf16 to int8 60 us without the
    // stream, 40.7 with it (0.88 of the memory's rate); 4096 x 16384 119 and
    // 79 us (0.91); with a bf16 output 50.3 and 97.5 us.  Not below 2048: 4096 x 1024 9.1 us without, 10.0 with it.
    if (many && g.K >= 2048) {
      if (g.K <= 4096) return launch_rows_stream_cfg<T, 2, 256, 3, true>(g, op, s);
      if (g.K <= 8192) return launch_rows_stream_cfg<T, 4, 256, 2, true>(g, op, s);
      if (g.K <= 13824) return launch_rows_stream_cfg<T, 4, 512, 2, false>(g, op, s);  // two stages of up to 54 KB
      if (g.K <= 16384) return launch_rows_stream_cfg<T, 4, 512, 1, true>(g, op, s);   // three of up to 64 KB
    }
  }
  const int threads = many && V > 1 ? 256 : 1024;
  if (g.K <= 8 * threads) return launch_rows_cfg<T, V, 8, 1024>(g, op, s);
  if constexpr (V > 1) {  // (single elements: the two ends only)
    if (g.K <= 16 * threads) return launch_rows_cfg<T, V, 16, 1024>(g, op, s);
    if (g.K <= 32 * 512) return launch_rows_cfg<T, V, 32, 512>(g, op, s);
  }
  return launch_rows_cfg<T, V, 32, 1024>(g, op, s);
}

template <typename T>
static cudaError_t launch_rows(const RowsArgs& g, int op, cudaStream_t s) {
  switch (rows_vector_width(g, op)) {
    case 8: return launch_rows_width<T, 8>(g, op, s);
    case 4: return launch_rows_width<T, 4>(g, op, s);
    default: return launch_rows_width<T, 1>(g, op, s);
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
