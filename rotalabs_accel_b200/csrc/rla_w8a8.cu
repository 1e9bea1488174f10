// W8A8 product: int8 rows (one scale a token) times the framework's int8
// weights (one scale an output channel),
//     y[m, n] = fp16( sx[m] * sw[n] * sum_k x[m, k] * w[n, k]  (+ bias[n]) ),
// on the 5th-generation tensor cores (tcgen05.mma.kind::i8, int32
// accumulators in Tensor Memory).  The sum is exact in int32 (|sum| <= K * 2^14,
// so K < 2^17), whatever order it is taken in: results do not depend on the
// tile, the split of K or the number of CTAs.
//
// Orientation: a tile is 128 output channels (the MMA's M, the 128 TMEM
// lanes) x BT tokens (the MMA's N), so the channel's scale and bias are two
// registers of an epilogue thread, and one token costs BT = 16 columns, not
// 128 rows.
//
// Work split.  The K axis of a tile is split over the CTAs of a thread-block
// cluster where there are fewer tiles than SMs: every rank leaves its int32
// partial tile in shared memory, and each rank adds up every splits-th token
// column from all ranks through distributed shared memory.  No workspace, no
// atomics.
//
// Warp roles (192 threads): warp 0 TMA producer (a ring of 128-byte-wide k
// blocks, 128-byte swizzle), warp 1 TMEM allocation and MMA issue, warps 2-5
// epilogue (one TMEM lane quarter each).  All waits are bounded.
#include <algorithm>

#include "rla_common.cuh"
#include "rla_internal.h"
#include "rla_tmap.cuh"

namespace rla {

namespace w8 {
constexpr int BR = 128;       // output channels of a tile
constexpr int BK = 128;       // k (bytes) of a stage: one 128-byte swizzle row
constexpr int THREADS = 192;
constexpr int MAX_STAGES = 12;
constexpr int MAX_SPLITS = 8;  // portable cluster size
constexpr int MAX_K = 131071;  // K * 128 * 128 < 2^31
__host__ __device__ constexpr int stage_bytes(int bt) { return (BR + bt) * BK; }
}  // namespace w8

// D[tmem] (+)= A[smem] * B[smem]^T, kind::i8 (signed 8-bit inputs, int32 accumulate).
RLA_DEVFN void rla_umma_ss_i8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Instruction descriptor, kind::i8: signed 8-bit A and B (K-major), int32 D.
__host__ __device__ constexpr uint32_t rla_idesc_i8_s32(int M, int N) {
  return (2u << 4)                                   // D format: s32
         | (1u << 7) | (1u << 10)                    // A, B format: signed 8 bits
         | (static_cast<uint32_t>(N >> 3) << 17)     // N / 8
         | (static_cast<uint32_t>(M >> 4) << 24);    // M / 16
}
RLA_DEVFN void rla_tmem_ld_32x32b_x16(uint32_t taddr, uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
        "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(taddr));
}
RLA_DEVFN uint32_t rla_ld_dsmem_u32(uint32_t addr, uint32_t rank) {
  uint32_t remote, v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(addr), "r"(rank));
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(remote) : "memory");
  return v;
}

struct W8Out {
  const float* sx;  // [M]
  const void* sw;   // [N]
  int sw_f32;
  const void* bias;  // [N] or null
  int bias_kind;     // 0 none, 1 fp16, 2 fp32
  __half* y;
  int64_t ldy;
  int M, N;
};

template <int BT>
__global__ void __launch_bounds__(w8::THREADS)
    w8a8_split_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x,
                      const W8Out out, int num_kb, int stages) {
  constexpr int COLS = BT < 32 ? 32 : BT;  // TMEM columns (a power of two, at least 32)
  constexpr int LD = BT < 32 ? 16 : 32;    // token columns of one TMEM load
  constexpr uint32_t STAGE = w8::stage_bytes(BT);

  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t full[w8::MAX_STAGES], empty[w8::MAX_STAGES], dfull;
  __shared__ uint32_t tmem_base;
  __shared__ int abort_word;
  __shared__ float sx_s[BT];

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int n0 = blockIdx.x * w8::BR;
  const int m0 = blockIdx.y * BT;
  const int splits = gridDim.z;
  const int rank = blockIdx.z;  // == cluster rank: the cluster spans z
  const int kb0 = static_cast<int>((int64_t)num_kb * rank / splits);
  const int nkb = static_cast<int>((int64_t)num_kb * (rank + 1) / splits) - kb0;
  volatile int* abort_flag = &abort_word;

  rla_griddep_launch_dependents();
  if (threadIdx.x == 0) {
    rla_tma_prefetch_desc(&tmap_w);
    rla_tma_prefetch_desc(&tmap_x);
    for (int s = 0; s < stages; ++s) {
      rla_mbar_init(&full[s], 1);
      rla_mbar_init(&empty[s], 1);
    }
    rla_mbar_init(&dfull, 1);
    abort_word = 0;
    rla_fence_barrier_init();
    // the first weight tiles into L2 while the previous kernel finishes
    for (int i = 0; i < min(stages, nkb); ++i) rla_tma_prefetch_l2_2d(&tmap_w, (kb0 + i) * w8::BK, n0);
  }
  if (warp == 1) {
    rla_tmem_alloc(&tmem_base, COLS);
    rla_tmem_relinquish();
  }
  rla_tc_fence_before();
  __syncthreads();
  rla_tc_fence_after();
  const uint32_t tmem = tmem_base;
  rla_griddep_wait();  // before any read of what an earlier kernel may have written

  bool ok = true;
  if (warp == 0) {
    if (lane == 0) {
      int issued = 0;
      for (int i = 0; i < nkb; ++i) {
        const int s = i % stages;
        if (i >= stages &&
            !rla_mbar_wait(&empty[s], ((i / stages) - 1) & 1, RLA_DEVERR_TIMEOUT_SLOT_EMPTY, abort_flag))
          break;
        uint8_t* slot = ring + (uint32_t)s * STAGE;
        rla_mbar_arrive_expect_tx(&full[s], STAGE);
        rla_tma_load_2d(slot, &tmap_w, &full[s], (kb0 + i) * w8::BK, n0);
        rla_tma_load_2d(slot + w8::BR * w8::BK, &tmap_x, &full[s], (kb0 + i) * w8::BK, m0);
        issued = i + 1;
      }
      if (*abort_flag)  // do not leave while copies may still land in shared memory
        for (int i = max(0, issued - stages); i < issued; ++i)
          rla_mbar_wait(&full[i % stages], (i / stages) & 1, RLA_DEVERR_TIMEOUT_TMA_FULL, nullptr);
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = rla_idesc_i8_s32(w8::BR, BT);
      for (int i = 0; i < nkb && ok; ++i) {
        const int s = i % stages;
        ok = rla_mbar_wait(&full[s], (i / stages) & 1, RLA_DEVERR_TIMEOUT_TMA_FULL, abort_flag);
        if (!ok) break;
        rla_tc_fence_after();
        const uint32_t wbase = rla_smem_u32(ring) + (uint32_t)s * STAGE;
        const uint32_t xbase = wbase + w8::BR * w8::BK;
#pragma unroll
        for (int ks = 0; ks < w8::BK / 32; ++ks)
          rla_umma_ss_i8(tmem, rla_smem_desc_sw128(wbase + ks * 32), rla_smem_desc_sw128(xbase + ks * 32), idesc,
                         (i | ks) != 0 ? 1u : 0u);
        rla_umma_commit(&empty[s]);
      }
      rla_umma_commit(&dfull);
      if (!ok) rla_mbar_wait(&dfull, 0, RLA_DEVERR_TIMEOUT_ACCUM, nullptr);  // no MMA writes TMEM after its release
    }
    __syncwarp();
  } else {
    const int quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const uint32_t lane_addr = static_cast<uint32_t>(quarter * 32) << 16;
    const int n = n0 + row;
    for (int c = threadIdx.x - 64; c < BT; c += 128) sx_s[c] = m0 + c < out.M ? out.sx[m0 + c] : 0.f;
    float sw = 0.f, bias = 0.f;
    if (n < out.N) {
      sw = out.sw_f32 ? static_cast<const float*>(out.sw)[n] : __half2float(static_cast<const __half*>(out.sw)[n]);
      bias = out.bias_kind == 0 ? 0.f
             : out.bias_kind == 1 ? __half2float(static_cast<const __half*>(out.bias)[n])
                                  : static_cast<const float*>(out.bias)[n];
    }
    asm volatile("bar.sync 1, 128;" ::: "memory");  // the epilogue warps: sx_s is complete
    ok = rla_mbar_wait(&dfull, 0, RLA_DEVERR_TIMEOUT_ACCUM, abort_flag);
    ok = __all_sync(0xffffffffu, ok);
    rla_tc_fence_after();
    int* part = reinterpret_cast<int*>(ring);  // [BT][128]: every copy and MMA of the ring is done
    if (ok) {
      const int cols = min(BT, out.M - m0);
#pragma unroll 1
      for (int j = 0; j < cols; j += LD) {
        uint32_t d[LD];
        if constexpr (LD == 16)
          rla_tmem_ld_32x32b_x16(tmem + lane_addr + j, d);
        else
          rla_tmem_ld_32x32b_x32(tmem + lane_addr + j, d);
        rla_tmem_wait_ld();
        if (splits > 1) {
#pragma unroll
          for (int i = 0; i < LD; ++i) part[(j + i) * w8::BR + row] = static_cast<int>(d[i]);
        } else if (n < out.N) {
          __half* yp = out.y + (int64_t)(m0 + j) * out.ldy + n;
#pragma unroll
          for (int i = 0; i < LD; ++i)
            if (j + i < cols)
              yp[i * out.ldy] = __float2half_rn(fmaf(static_cast<float>(static_cast<int>(d[i])) * sw, sx_s[j + i], bias));
        }
      }
    }
    if (splits > 1) {
      __syncwarp();
      rla_cluster_sync();
      if (ok && n < out.N) {
        const int cols = min(BT, out.M - m0);
        const uint32_t mine = rla_smem_u32(part) + row * 4;
        for (int c = rank; c < cols; c += splits) {
          int sum = 0;
          for (int r = 0; r < splits; ++r)
            sum += static_cast<int>(rla_ld_dsmem_u32(mine + c * (w8::BR * 4), r));
          out.y[(int64_t)(m0 + c) * out.ldy + n] = __float2half_rn(fmaf(static_cast<float>(sum) * sw, sx_s[c], bias));
        }
      }
      __syncwarp();
      rla_cluster_sync();  // nobody leaves while its shared memory may still be read
    }
  }
  if (warp < 2 && splits > 1) {
    rla_cluster_sync();
    rla_cluster_sync();
  }
  rla_tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    rla_tc_fence_after();
    rla_tmem_dealloc(tmem, COLS);
  }
}

// Rows of K bytes (any alignment, any stride) into rows of `ldd` bytes, zero
// behind K: what TMA's 16-byte rules need where K or a row stride is odd.
__global__ void w8a8_align_rows_kernel(const int8_t* __restrict__ src, int64_t lds, int8_t* __restrict__ dst, int ldd,
                                       int64_t rows, int K) {
  const int per_row = ldd / 16;
  const int64_t total = rows * per_row;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int64_t r = i / per_row;
    const int k = static_cast<int>(i - r * per_row) * 16;
    const int8_t* p = src + r * lds + k;
    alignas(16) int8_t v[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = k + j < K ? p[j] : int8_t(0);
    *reinterpret_cast<uint4*>(dst + r * ldd + k) = *reinterpret_cast<const uint4*>(v);
  }
}

struct W8Plan {
  int bt = 0, splits = 1, per_sm = 1, stages = 0;
  int grid_x = 0, grid_y = 0;
  size_t smem = 0;
};

// Token columns: the smallest MMA shape that holds the batch (256 above 128).
// K slices and CTAs per SM: the pair with the shortest estimated time, in k
// blocks of one SM's share of the memory system -- rounds of resident CTAs x
// the k blocks a CTA streams, plus a fixed cost a round.
static W8Plan w8a8_plan(int64_t M, int64_t N, int64_t K) {
  W8Plan p;
  p.bt = M <= 16 ? 16 : M <= 32 ? 32 : M <= 64 ? 64 : M <= 128 ? 128 : 256;
  p.grid_x = static_cast<int>((N + w8::BR - 1) / w8::BR);
  p.grid_y = static_cast<int>((M + p.bt - 1) / p.bt);
  const int64_t tiles = (int64_t)p.grid_x * p.grid_y;
  const int kb = static_cast<int>((K + w8::BK - 1) / w8::BK);
  const int sms = device_sm_count();
  const int stage = w8::stage_bytes(p.bt);
  double best = 0;
  for (int c = 1; c <= (p.bt <= 32 ? 4 : p.bt <= 64 ? 2 : 1); ++c) {
    const int ring = (c == 1 ? 220 : c == 2 ? 108 : c == 3 ? 70 : 52) * 1024;
    int stages = ring / stage;
    if (stages > w8::MAX_STAGES) stages = w8::MAX_STAGES;
    for (int s = 1; s <= w8::MAX_SPLITS && s <= kb; ++s) {
      const int64_t rounds = (tiles * s + (int64_t)sms * c - 1) / ((int64_t)sms * c);
      const double cost = static_cast<double>(rounds) * c * ((kb + s - 1) / s + 1) + (s > 1 ? 1.0 : 0.0);
      if (best == 0 || cost < best) {
        best = cost;
        p.splits = s;
        p.per_sm = c;
        p.stages = stages;
      }
    }
  }
  p.smem = (size_t)p.stages * stage + 1024;
  return p;
}

template <int BT>
static cudaError_t launch_w8a8_cfg(const W8Plan& p, const CUtensorMap& tw, const CUtensorMap& tx, const W8Out& out,
                                   int num_kb, cudaStream_t s) {
  auto kern = w8a8_split_kernel<BT>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)p.smem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.grid_x, p.grid_y, p.splits);
  cfg.blockDim = dim3(w8::THREADS);
  cfg.dynamicSmemBytes = p.smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (p.splits > 1) {
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = 1;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = static_cast<unsigned>(p.splits);
    cfg.numAttrs = 2;
  }
  return cudaLaunchKernelEx(&cfg, kern, tw, tx, out, num_kb, p.stages);
}

static cudaError_t launch_w8a8(const int8_t* x, int64_t ldx, const int8_t* w, int64_t ldw, const W8Out& out, int64_t K,
                               cudaStream_t s) {
  const W8Plan p = w8a8_plan(out.M, out.N, K);
  CUtensorMap tw, tx;
  if (!make_tmap_2d(&tw, CU_TENSOR_MAP_DATA_TYPE_UINT8, w, (uint64_t)K, (uint64_t)out.N, (uint64_t)ldw, w8::BK, w8::BR,
                    CU_TENSOR_MAP_SWIZZLE_128B) ||
      !make_tmap_2d(&tx, CU_TENSOR_MAP_DATA_TYPE_UINT8, x, (uint64_t)K, (uint64_t)out.M, (uint64_t)ldx, w8::BK, p.bt,
                    CU_TENSOR_MAP_SWIZZLE_128B))
    return cudaErrorInvalidValue;
  const int num_kb = static_cast<int>((K + w8::BK - 1) / w8::BK);
  switch (p.bt) {
    case 16: return launch_w8a8_cfg<16>(p, tw, tx, out, num_kb, s);
    case 32: return launch_w8a8_cfg<32>(p, tw, tx, out, num_kb, s);
    case 64: return launch_w8a8_cfg<64>(p, tw, tx, out, num_kb, s);
    case 128: return launch_w8a8_cfg<128>(p, tw, tx, out, num_kb, s);
    default: return launch_w8a8_cfg<256>(p, tw, tx, out, num_kb, s);
  }
}

static bool w8a8_rows_aligned(const void* p, int64_t ld, int64_t rows) {
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && (rows == 1 || ld % 16 == 0);
}

static int w8a8_fail(int code, const char* msg) {
  set_error("rla_w8a8_gemm: %s", msg);
  return code;
}

}  // namespace rla

extern "C" {

size_t rla_w8a8_workspace_size(int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  const size_t ld = ((size_t)K + 15) & ~size_t(15);
  return ((size_t)M + (size_t)N) * ld;
}

int rla_w8a8_gemm(const int8_t* x, int64_t ldx, const float* x_scale, const int8_t* w, int64_t ldw, const void* scale,
                  int scale_dtype, const void* bias, int bias_dtype, void* y, int64_t ldy, int64_t M, int64_t N,
                  int64_t K, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace rla;
  if (M < 0 || N < 0 || K < 0 || M > INT32_MAX - 256 || N > INT32_MAX - 256)
    return w8a8_fail(RLA_ERR_INVALID_ARGUMENT, "M, N must be in [0, 2^31 - 256)");
  if (K > w8::MAX_K) return w8a8_fail(RLA_ERR_UNSUPPORTED, "K must be below 131072 (the int32 sum could overflow)");
  if (scale_dtype != RLA_DTYPE_F16 && scale_dtype != RLA_DTYPE_F32)
    return w8a8_fail(RLA_ERR_INVALID_ARGUMENT, "scale_dtype must be F16 or F32");
  if (bias_dtype != RLA_DTYPE_NONE && bias_dtype != RLA_DTYPE_F16 && bias_dtype != RLA_DTYPE_F32)
    return w8a8_fail(RLA_ERR_INVALID_ARGUMENT, "bias_dtype must be NONE, F16 or F32");
  if (M == 0 || N == 0) return RLA_OK;
  if (bias_dtype != RLA_DTYPE_NONE && !bias) return w8a8_fail(RLA_ERR_INVALID_ARGUMENT, "bias is NULL but bias_dtype is set");
  if (!y || !scale || !x_scale || (K > 0 && (!x || !w)))
    return w8a8_fail(RLA_ERR_INVALID_ARGUMENT, "null x, x_scale, w, scale or y");
  if (ldy < N || (K > 0 && (ldx < K || ldw < K)))
    return w8a8_fail(RLA_ERR_INVALID_ARGUMENT, "leading dimensions must be >= the row length");
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int bias_kind = bias_dtype == RLA_DTYPE_NONE ? 0 : bias_dtype == RLA_DTYPE_F16 ? 1 : 2;
  cudaError_t e = cudaSuccess;
  if (K == 0) {
    GemmArgs a{};
    a.bias = bias, a.bias_kind = bias_kind, a.y = y, a.ldy = ldy, a.M = (int)M, a.N = (int)N;
    e = launch_fill(a, s);
  } else {
    const bool xok = w8a8_rows_aligned(x, ldx, M), wok = w8a8_rows_aligned(w, ldw, N);
    const int64_t ld = (K + 15) / 16 * 16;
    if (!xok || !wok) {
      const size_t need = (xok ? 0 : (size_t)(M * ld)) + (wok ? 0 : (size_t)(N * ld));
      if (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15u)) {
        set_error("rla_w8a8_gemm: rows that are not 16-byte aligned need %zu bytes of 16-byte aligned workspace "
                  "(rla_w8a8_workspace_size), got %zu", need, workspace ? workspace_bytes : size_t(0));
        return RLA_ERR_WORKSPACE;
      }
      int8_t* to = static_cast<int8_t*>(workspace);
      auto align = [&](const int8_t*& p, int64_t& lds, int64_t rows) {
        const int64_t blocks = std::min<int64_t>((rows * (ld / 16) + 255) / 256, 148 * 16);
        rla_clear_stale_launch_error();
        w8a8_align_rows_kernel<<<(unsigned)blocks, 256, 0, s>>>(p, lds, to, (int)ld, rows, (int)K);
        p = to;
        lds = ld;
        to += rows * ld;
        note_launch();
        return cudaGetLastError();
      };
      if (!xok) e = align(x, ldx, M);
      if (e == cudaSuccess && !wok) e = align(w, ldw, N);
    }
    const W8Out out{x_scale, scale, scale_dtype == RLA_DTYPE_F32 ? 1 : 0, bias, bias_kind, static_cast<__half*>(y), ldy,
                    (int)M, (int)N};
    if (e == cudaSuccess) e = launch_w8a8(x, M == 1 ? (ldx + 15) / 16 * 16 : ldx, w, N == 1 ? (ldw + 15) / 16 * 16 : ldw, out, K, s);
  }
  if (e != cudaSuccess) {
    set_error("rla_w8a8_gemm: %s", cudaGetErrorString(e));
    return RLA_ERR_CUDA;
  }
  note_launch();
  return RLA_OK;
}

}  // extern "C"
