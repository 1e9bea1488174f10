// W8A8 product: int8 rows (one scale a token) times the framework's int8
// weights (one scale an output channel),
//     y[m, n] = fp16( sx[m] * sw[n] * sum_k x[m, k] * w[n, k]  (+ bias[n]) ),
// on the 5th-generation tensor cores (tcgen05.mma.kind::i8, int32
// accumulators in Tensor Memory).  The sum is exact in int32 (|sum| <= K * 2^14,
// so K < 2^17), whatever order it is taken in: results do not depend on the
// tile, the split of K or the number of CTAs.
//
// Orientation: a tile is 128 (or, of a CTA pair, 256) output channels (the
// MMA's M, the TMEM lanes) x up to 128 (256) tokens (the MMA's N), so the channel's
// scale and bias are two registers of an epilogue thread, and one token costs
// 16 columns, not 128 rows.
//
// Two kernels:
//   split  one tile a cluster.  Where there are fewer tiles than SMs, the K
//          axis is split over the CTAs of the cluster: every rank leaves its
//          int32 partial tile in shared memory, and each rank adds up every
//          splits-th token column from all ranks through distributed shared
//          memory.  No workspace, no atomics.
//   pair   persistent CTA pairs (cta_group::2), 256 x 256 tiles, for problems
//          of many tiles.  Each CTA of a pair loads 128 channels and 128
//          tokens of a k block and the MMA reads both CTAs' shared memory, so
//          an SM takes 32 KB from L2 for each 512 clocks of MMA; a 128 x 256
//          tile of one CTA would take 48 KB, more than L2 gives an SM.  Two
//          accumulators: the epilogue of a tile runs under the next tile's MMAs.
//
// Warp roles: warp 0 TMA producer (a ring of 128-byte-wide k blocks, 128-byte
// swizzle), warp 1 TMEM allocation and MMA issue, then the epilogue's warps, one
// (of a pair's CTA two) for each TMEM lane quarter.
//
// Waits.  Every mbarrier wait is bounded; after one that gave up, the CTAs still
// see all their copies land and their MMAs end before they leave.  The cluster's
// barriers and tcgen05.alloc have no limit.  A barrier is reached by every
// warp whatever its waits returned.  An allocation waits for other CTAs of its
// SM to hand Tensor Memory back, and none of those waits for this one in turn:
// a split CTA holds Tensor Memory only while it waits for its own copies and MMAs,
// not for its cluster, and a CTA pair is alone on its SMs (kW8PairSmem).  Not
// excluded: a kernel of another library, earlier in the stream, that lets
// dependent kernels start before it has allocated its own.
#include <algorithm>
#include <atomic>

#include "rla_common.cuh"
#include "rla_internal.h"
#include "rla_tmap.cuh"

namespace rla {

namespace w8 {
constexpr int BR = 128;       // output channels of a tile
constexpr int BK = 128;       // k (bytes) of a stage: one 128-byte swizzle row
constexpr int THREADS = 192;
constexpr int MAX_STAGES = 4;
constexpr int MAX_BT = 128;    // token columns of a split tile
constexpr int MAX_SPLITS = 8;  // portable cluster size
constexpr int MAX_K = 131071;  // K * 128 * 128 < 2^31
__host__ __device__ constexpr int stage_bytes(int bt) { return (BR + bt) * BK; }
constexpr int PAIR_ROWS = 256;   // tile of a CTA pair: channels, and tokens
constexpr int PAIR_STAGES = 6;   // 32 KB each
constexpr int PAIR_THREADS = 320;
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
// Counted at the named barrier without waiting there.
RLA_DEVFN void rla_named_bar_arrive(int id, int nthreads) {
  asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(nthreads) : "memory");
}
RLA_DEVFN uint32_t rla_mapa(uint32_t addr, uint32_t rank) {
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(addr), "r"(rank));
  return remote;
}
RLA_DEVFN int4 rla_ld_cluster_int4(uint32_t remote) {
  int4 v;
  asm volatile("ld.shared::cluster.v4.s32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(remote)
               : "memory");
  return v;
}

RLA_DEVFN void rla_st_cluster_u32(uint32_t remote, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(remote), "r"(v) : "memory");
}
// As if `bytes` of a copy that counts on the barrier had arrived.
RLA_DEVFN void rla_mbar_complete_tx(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.complete_tx.relaxed.cluster.shared::cta.b64 [%0], %1;" ::"r"(rla_smem_u32(bar)), "r"(bytes) : "memory");
}

// ---- CTA pairs (cta_group::2): the even CTA of the cluster leads ----
RLA_DEVFN void rla_umma2_ss_i8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Arrive on the barrier at this offset in both CTAs once the MMAs issued so far are done.
RLA_DEVFN void rla_umma2_commit(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          rla_smem_u32(bar)),
      "h"(static_cast<uint16_t>(3))
      : "memory");
}
RLA_DEVFN void rla_tmem2_alloc(uint32_t* smem_result, uint32_t ncols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(rla_smem_u32(smem_result)),
               "r"(ncols)
               : "memory");
}
RLA_DEVFN void rla_tmem2_relinquish() {
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
RLA_DEVFN void rla_tmem2_dealloc(uint32_t taddr, uint32_t ncols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}
// Tile copy into this CTA's shared memory that counts on a barrier of either CTA of the pair.
RLA_DEVFN void rla_tma2_load_2d(void* smem_dst, const void* desc, uint32_t bar, int32_t c0, int32_t c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4}], [%2];" ::"r"(rla_smem_u32(smem_dst)),
      "l"(desc), "r"(bar), "r"(c0), "r"(c1)
      : "memory");
}
// Relaxed: it says that Tensor Memory has been read (tcgen05.wait::ld came before
// it), and a release would wait for the tile's stores to global memory as well.
RLA_DEVFN void rla_mbar_arrive_cluster(uint32_t remote) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(remote) : "memory");
}
RLA_DEVFN bool rla_mbar_try_wait_cluster(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, 1000;\n\t"
      "selp.b32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(rla_smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
// rla_mbar_wait for a barrier that the other CTA of the pair arrives on too.
RLA_DEVFN bool rla_mbar_wait_cluster(uint64_t* bar, uint32_t parity, unsigned int err, volatile int* abort_flag) {
  if (rla_mbar_try_wait_cluster(bar, parity)) return true;
  const uint64_t t0 = rla_globaltimer();
  uint32_t spins = 0;
  while (true) {
    if (rla_mbar_try_wait_cluster(bar, parity)) return true;
    if ((++spins & 15u) == 0) {
      if (abort_flag && *abort_flag) return false;
      if (rla_globaltimer() - t0 > RLA_WAIT_LIMIT_NS) {
        rla_record_error(err);
        if (abort_flag) *abort_flag = 1;
        return false;
      }
    }
  }
}

struct W8Out {
  const float* sx;  // [M]
  const void* sw;   // [N]
  int sw_f32;
  const void* bias;  // [N] or null
  int bias_kind;     // 0 none, 1 fp16, 2 fp32
  __half* y;
  int64_t ldy;
  int vec;  // channels of a store: 8, 4 or fewer, as y and its rows are aligned
  int M, N;
};

RLA_DEVFN float w8a8_channel(const void* p, int kind, int n) {  // kind: 0 none, 1 fp16, 2 fp32
  return kind == 0 ? 0.f : kind == 1 ? __half2float(static_cast<const __half*>(p)[n]) : static_cast<const float*>(p)[n];
}
RLA_DEVFN __half w8a8_value(int sum, float sw, float sx, float bias) {
  return __float2half_rn(fmaf(static_cast<float>(sum) * sw, sx, bias));
}

// Two tokens of a channel (the same roundings, one conversion for both).
RLA_DEVFN __half2 w8a8_values(int sum0, int sum1, float sw, float sx0, float sx1, float bias) {
  return __floats2half2_rn(fmaf(static_cast<float>(sum0) * sw, sx0, bias), fmaf(static_cast<float>(sum1) * sw, sx1, bias));
}

// 32 rows of 32 channels, out of `buf`, to y: V channels a lane, V rows a store.
template <int V, typename Word>
RLA_DEVFN void w8a8_store_rows(const __half* buf, __half* y, int64_t ldy, int rows, int channels) {
  static_assert(sizeof(Word) == V * sizeof(__half), "");
  const int lane = threadIdx.x & 31;
  const int c = lane % (32 / V) * V;
  const int left = channels - c;
#pragma unroll 4
  for (int h = 0; h < 32; h += V) {
    const int r = h + lane / (32 / V);
    if (r >= rows) continue;
    const Word v = *reinterpret_cast<const Word*>(buf + r * 32 + c);
    __half* to = y + r * ldy + c;
    if (left >= V) {
      *reinterpret_cast<Word*>(to) = v;
    } else {
      const __half* e = reinterpret_cast<const __half*>(&v);
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (i < left) to[i] = e[i];
    }
  }
}
// One epilogue warp's 32 channels (TMEM lanes) into y: of `cols` token columns
// 32 from `first` on, and 32 after every `step` (both multiples of 32).
// A lane holds one channel, a row of y many: 32 tokens at a time pass through
// 2 KB of shared memory (`buf`, the warp's own), so that a store instruction is
// 8 rows of 64 bytes (4 where y's rows are 8-byte aligned), where the lanes' own
// values would be 32 of one row.  Measured against those stores: 2048x4096x1024
// 26.7 us to 12.5, 256x8192x128 7.3 to 4.8.  Rows of lesser alignment are stored
// by the lanes: through the buffer 300x2001x64 took 11.8 us where this takes 8.1.
RLA_DEVFN void w8a8_store_warp(const W8Out& out, uint32_t taddr, int first, int step, int cols, int m0, int n_warp,
                               float sw, float bias, const float* sx, __half* buf) {
  const int lane = threadIdx.x & 31;
  const int channels = out.N - n_warp;
  __half* yp = out.y + (int64_t)(m0 + first) * out.ldy + n_warp;
  if (out.vec < 4) {
#pragma unroll 1
    for (int j = first; j < cols; j = (j & 16) ? j + step - 16 : j + 16) {
      uint32_t d[16];
      rla_tmem_ld_32x32b_x16(taddr + j, d);
      rla_tmem_wait_ld();
      if (lane < channels) {
        __half* to = out.y + (int64_t)(m0 + j) * out.ldy + n_warp + lane;
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (j + i < cols) to[i * out.ldy] = w8a8_value(static_cast<int>(d[i]), sw, sx[j + i], bias);
      }
    }
    return;
  }
#pragma unroll 1
  for (int j = first; j < cols; j += step, yp += step * out.ldy) {
    uint32_t d[2][16];
    rla_tmem_ld_32x32b_x16(taddr + j, d[0]);
    rla_tmem_ld_32x32b_x16(taddr + j + 16, d[1]);  // (may lie behind `cols`, never behind the allocation)
    rla_tmem_wait_ld();
    const int rows = cols - j;
    __syncwarp();  // the last 32 tokens have left the buffer
#pragma unroll
    for (int i = 0; i < 32; i += 4) {
      const uint32_t* di = d[i >> 4] + (i & 15);
      const float4 s4 = *reinterpret_cast<const float4*>(sx + j + i);
      const __half2 lo = w8a8_values(static_cast<int>(di[0]), static_cast<int>(di[1]), sw, s4.x, s4.y, bias);
      const __half2 hi = w8a8_values(static_cast<int>(di[2]), static_cast<int>(di[3]), sw, s4.z, s4.w, bias);
      buf[(i + 0) * 32 + lane] = __low2half(lo);
      buf[(i + 1) * 32 + lane] = __high2half(lo);
      buf[(i + 2) * 32 + lane] = __low2half(hi);
      buf[(i + 3) * 32 + lane] = __high2half(hi);
    }
    __syncwarp();
    if (out.vec == 8)
      w8a8_store_rows<8, uint4>(buf, yp, out.ldy, rows, channels);
    else
      w8a8_store_rows<4, uint2>(buf, yp, out.ldy, rows, channels);
  }
}

// bt: token columns of a tile, a multiple of 16 up to MAX_BT.
__global__ void __launch_bounds__(w8::THREADS, 5)
    w8a8_split_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x,
                      const W8Out out, int num_kb, int stages, int bt, int tmem_cols) {
  const uint32_t stage = w8::stage_bytes(bt);

  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t full[w8::MAX_STAGES], empty[w8::MAX_STAGES], dfull;
  __shared__ uint32_t tmem_base;
  __shared__ int abort_word;
  __shared__ __align__(16) float sx_s[w8::MAX_BT + 16];
  __shared__ __align__(16) float sw_s[w8::BR], bias_s[w8::BR];

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int n0 = blockIdx.x * w8::BR;
  const int m0 = blockIdx.y * bt;
  const int splits = gridDim.z;
  const int rank = blockIdx.z;  // == cluster rank: the cluster spans z
  const int kb0 = static_cast<int>((int64_t)num_kb * rank / splits);
  const int nkb = static_cast<int>((int64_t)num_kb * (rank + 1) / splits) - kb0;
  volatile int* abort_flag = &abort_word;

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
    rla_tmem_alloc(&tmem_base, tmem_cols);
    rla_tmem_relinquish();
  }
  rla_tc_fence_before();
  __syncthreads();
  rla_tc_fence_after();
  const uint32_t tmem = tmem_base;
  // (only now, so that a dependent launch cannot take the TMEM columns first)
  rla_griddep_launch_dependents();
  rla_griddep_wait();  // before any read of what an earlier kernel may have written

  bool ok = true;
  int* part = reinterpret_cast<int*>(ring);  // [bt][128], once every copy and MMA of the ring is done
  const int cols = min(bt, out.M - m0);
  const int t = threadIdx.x - 64;
  if (warp == 0) {
    if (lane == 0) {
      int issued = 0;
      for (int i = 0; i < nkb; ++i) {
        const int s = i % stages;
        if (i >= stages &&
            !rla_mbar_wait(&empty[s], ((i / stages) - 1) & 1, RLA_DEVERR_TIMEOUT_SLOT_EMPTY, abort_flag))
          break;
        uint8_t* slot = ring + (uint32_t)s * stage;
        rla_mbar_arrive_expect_tx(&full[s], stage);
        rla_tma_load_2d(slot, &tmap_w, &full[s], (kb0 + i) * w8::BK, n0);
        rla_tma_load_2d(slot + w8::BR * w8::BK, &tmap_x, &full[s], (kb0 + i) * w8::BK, m0);
        issued = i + 1;
      }
      // do not leave while copies may still land in shared memory: the MMA warp
      // waits for them too, but may give up after this warp has issued its last
      for (int i = max(0, issued - stages); i < issued; ++i)
        rla_mbar_wait(&full[i % stages], (i / stages) & 1, RLA_DEVERR_TIMEOUT_TMA_FULL, nullptr);
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc = rla_idesc_i8_s32(w8::BR, bt);
      for (int i = 0; i < nkb && ok; ++i) {
        const int s = i % stages;
        ok = rla_mbar_wait(&full[s], (i / stages) & 1, RLA_DEVERR_TIMEOUT_TMA_FULL, abort_flag);
        if (!ok) break;
        rla_tc_fence_after();
        const uint32_t wbase = rla_smem_u32(ring) + (uint32_t)s * stage;
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
    for (int c = t; c < cols; c += 128) sx_s[c] = out.sx[m0 + c];
    const float sw = n < out.N ? w8a8_channel(out.sw, out.sw_f32 ? 2 : 1, n) : 0.f;
    const float bias = n < out.N ? w8a8_channel(out.bias, out.bias_kind, n) : 0.f;
    sw_s[row] = sw;
    bias_s[row] = bias;
    rla_named_bar_sync(1, 128);  // the epilogue warps
    ok = rla_mbar_wait(&dfull, 0, RLA_DEVERR_TIMEOUT_ACCUM, abort_flag);
    ok = __all_sync(0xffffffffu, ok);
    rla_tc_fence_after();
    if (ok && splits == 1) {
      w8a8_store_warp(out, tmem + lane_addr, 0, 32, cols, m0, n0 + quarter * 32, sw, bias, sx_s,
                      reinterpret_cast<__half*>(ring) + quarter * (32 * 32));
    } else if (ok) {
#pragma unroll 1
      for (int j = 0; j < cols; j += 16) {
        uint32_t d[16];
        rla_tmem_ld_32x32b_x16(tmem + lane_addr + j, d);
        rla_tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 16; ++i) part[(j + i) * w8::BR + row] = static_cast<int>(d[i]);
      }
    }
  }
  rla_tc_fence_before();
  if (splits == 1) {
    __syncthreads();
    if (warp == 1) {
      rla_tc_fence_after();
      rla_tmem_dealloc(tmem, tmem_cols);
    }
  } else {
    // Tensor Memory goes back before the CTA waits for its cluster: holding it
    // meanwhile, it could be what the cluster's other CTAs wait for (their
    // allocation behind one of a third kernel that is stuck on these columns).
    rla_cluster_arrive();
    if (warp == 1) {
      rla_named_bar_sync(2, 160);  // the epilogue warps have read it
      rla_tc_fence_after();
      rla_tmem_dealloc(tmem, tmem_cols);
    } else if (warp >= 2) {
      rla_named_bar_arrive(2, 160);
    }
    rla_cluster_wait();
    // thread t: four channels (16 bytes) of the columns rank + splits * (t / 32 + 4 i);
    // all ranks' loads are issued before the first is used
    if (warp >= 2 && ok) {
      const int r4 = lane * 4;
      const uint32_t mine = rla_smem_u32(part) + r4 * 4;
      for (int c = rank + splits * (t >> 5); c < cols; c += splits * 4) {
        int4 v[w8::MAX_SPLITS];
#pragma unroll
        for (int r = 0; r < w8::MAX_SPLITS; ++r)
          if (r < splits) v[r] = rla_ld_cluster_int4(rla_mapa(mine + c * (w8::BR * 4), r));
        int4 sum = v[0];
#pragma unroll
        for (int r = 1; r < w8::MAX_SPLITS; ++r)
          if (r < splits) sum.x += v[r].x, sum.y += v[r].y, sum.z += v[r].z, sum.w += v[r].w;
        const float sx = sx_s[c];
        const float4 w4 = *reinterpret_cast<const float4*>(sw_s + r4), b4 = *reinterpret_cast<const float4*>(bias_s + r4);
        __half* yp = out.y + (int64_t)(m0 + c) * out.ldy + n0 + r4;
        alignas(8) const __half h[4] = {w8a8_value(sum.x, w4.x, sx, b4.x), w8a8_value(sum.y, w4.y, sx, b4.y),
                                        w8a8_value(sum.z, w4.z, sx, b4.z), w8a8_value(sum.w, w4.w, sx, b4.w)};
        if (out.vec >= 4 && n0 + r4 + 4 <= out.N) {
          *reinterpret_cast<uint2*>(yp) = *reinterpret_cast<const uint2*>(h);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (n0 + r4 + i < out.N) yp[i] = h[i];
        }
      }
    }
    __syncwarp();
    rla_cluster_sync();  // nobody leaves while its shared memory may still be read
  }
}

// Tile number -> (channel tile, token tile): token tiles in groups that stay
// in L2 while all channel tiles pass over them.
struct W8Order {
  int tiles_n, tiles_m, group;
  RLA_DEVFN void at(int tile, int& tn, int& tm) const {
    const int per = group * tiles_n;
    const int g = tile / per, in = tile - g * per;
    const int rows = min(group, tiles_m - g * group);
    tn = in / rows;
    tm = g * group + in - tn * rows;
  }
};

struct W8PairShared {
  alignas(1024) uint8_t ring[w8::PAIR_STAGES][2 * 128 * w8::BK];  // 128 channels, then 128 tokens
  alignas(16) float sx[2][w8::PAIR_ROWS];
  alignas(16) __half buf[8][32 * 32];  // one an epilogue warp
  uint64_t full[w8::PAIR_STAGES], empty[w8::PAIR_STAGES], dfull[2], dempty[2], drain;
  uint32_t tmem_base;
  int abort_flag, issued;            // issued: k blocks that this CTA's copies were issued for
  int peer_abort_flag, peer_issued;  // the other CTA's, at the end
};
// After a wait that gave up, by the leader when both CTAs are through: all
// copies in flight land.  Both CTAs' bytes count on the leader's barriers, which
// expect them for the blocks that the leader issued (n0); the other CTA may have
// stopped before it (n1 < n0), and its bytes are taken as arrived, or after it, and
// they are expected now.  (It is at most a ring ahead: it waits for the leader's commits.)
RLA_DEVFN void w8a8_pair_drain(W8PairShared& sm, uint32_t half) {
  constexpr int STAGES = w8::PAIR_STAGES;
  const int n0 = sm.issued, n1 = sm.peer_issued, last = max(n0, n1);
  for (int i = max(0, last - STAGES); i < last; ++i) {
    uint64_t* bar = &sm.full[i % STAGES];
    if (i >= n0) rla_mbar_arrive_expect_tx(bar, 2 * half);
    if (i >= n1) rla_mbar_complete_tx(bar, 2 * half);
  }
  for (int i = max(0, last - STAGES); i < last; ++i)
    rla_mbar_wait_cluster(&sm.full[i % STAGES], (i / STAGES) & 1, RLA_DEVERR_TIMEOUT_TMA_FULL, nullptr);
}

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(w8::PAIR_THREADS, 1)
    w8a8_pair_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x,
                     const W8Out out, int num_kb, const W8Order order) {
  extern __shared__ uint8_t smem_raw[];
  W8PairShared& sm =
      *reinterpret_cast<W8PairShared*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  constexpr int STAGES = w8::PAIR_STAGES;
  constexpr uint32_t HALF = 128 * w8::BK;  // bytes of one operand's part in one CTA
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = rla_cluster_ctarank();
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int tiles = order.tiles_n * order.tiles_m;
  volatile int* abort_flag = &sm.abort_flag;

  if (threadIdx.x == 0) {
    rla_tma_prefetch_desc(&tmap_w);
    rla_tma_prefetch_desc(&tmap_x);
    for (int s = 0; s < STAGES; ++s) {
      rla_mbar_init(&sm.full[s], 1);   // the leader's expect_tx; both CTAs' bytes count on the leader's barrier
      rla_mbar_init(&sm.empty[s], 1);  // the leader's commit, to both
    }
    for (int a = 0; a < 2; ++a) {
      rla_mbar_init(&sm.dfull[a], 1);
      rla_mbar_init(&sm.dempty[a], 16);  // (leader's) eight epilogue warps of each CTA
    }
    rla_mbar_init(&sm.drain, 1);
    sm.abort_flag = 0;
    sm.issued = 0;
    rla_fence_barrier_init();
  }
  if (warp == 1) {
    rla_tmem2_alloc(&sm.tmem_base, 512);
    rla_tmem2_relinquish();
  }
  rla_tc_fence_before();
  __syncthreads();
  rla_cluster_sync();  // the other CTA's barriers are ready
  rla_tc_fence_after();
  const uint32_t tmem = sm.tmem_base;
  rla_griddep_launch_dependents();
  rla_griddep_wait();

  if (warp == 0) {
    if (lane == 0) {
      int it = 0;  // k blocks since the start, over all tiles
      bool ok = true;
      for (int tile = pair; tile < tiles && ok; tile += pairs) {
        int tn, tm;
        order.at(tile, tn, tm);
        const int n0 = tn * w8::PAIR_ROWS + static_cast<int>(rank) * 128;
        const int m0 = tm * w8::PAIR_ROWS + static_cast<int>(rank) * 128;
        for (int kb = 0; kb < num_kb; ++kb, ++it) {
          const int s = it % STAGES;
          if (it >= STAGES) {
            ok = rla_mbar_wait_cluster(&sm.empty[s], ((it / STAGES) - 1) & 1, RLA_DEVERR_TIMEOUT_SLOT_EMPTY, abort_flag);
            if (!ok) break;
          }
          if (rank == 0) rla_mbar_arrive_expect_tx(&sm.full[s], 4 * HALF);
          const uint32_t bar = rla_mapa(rla_smem_u32(&sm.full[s]), 0);
          rla_tma2_load_2d(sm.ring[s], &tmap_w, bar, kb * w8::BK, n0);
          rla_tma2_load_2d(sm.ring[s] + HALF, &tmap_x, bar, kb * w8::BK, m0);
        }
      }
      sm.issued = it;
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      constexpr uint32_t idesc = rla_idesc_i8_s32(w8::PAIR_ROWS, w8::PAIR_ROWS);
      int it = 0, n = 0;
      bool ok = true;
      for (int tile = pair; tile < tiles && ok; tile += pairs, ++n) {
        const int a = n & 1;
        if (n >= 2) {
          ok = rla_mbar_wait_cluster(&sm.dempty[a], ((n >> 1) - 1) & 1, RLA_DEVERR_TIMEOUT_ACCUM, abort_flag);
          if (!ok) break;
          rla_tc_fence_after();
        }
        for (int kb = 0; kb < num_kb; ++kb, ++it) {
          const int s = it % STAGES;
          ok = rla_mbar_wait_cluster(&sm.full[s], (it / STAGES) & 1, RLA_DEVERR_TIMEOUT_TMA_FULL, abort_flag);
          if (!ok) break;
          rla_tc_fence_after();
          const uint32_t wbase = rla_smem_u32(sm.ring[s]);
#pragma unroll
          for (int ks = 0; ks < w8::BK / 32; ++ks)
            rla_umma2_ss_i8(tmem + a * 256, rla_smem_desc_sw128(wbase + ks * 32),
                            rla_smem_desc_sw128(wbase + HALF + ks * 32), idesc, (kb | ks) != 0 ? 1u : 0u);
          rla_umma2_commit(&sm.empty[s]);
        }
        rla_umma2_commit(&sm.dfull[a]);
      }
      if (!ok) {  // no MMA writes TMEM after its release
        rla_umma2_commit(&sm.drain);
        rla_mbar_wait_cluster(&sm.drain, 0, RLA_DEVERR_TIMEOUT_ACCUM, nullptr);
      }
    }
    __syncwarp();
  } else {
    const int quarter = warp & 3, half = (warp - 2) >> 2;
    const uint32_t lane_addr = static_cast<uint32_t>(quarter * 32) << 16;
    const int t = threadIdx.x - 64;
    int n_tile = 0;
    // a thread's channel, and the scale of one of the tokens, for the tile to come
    // (read while the tile before is stored)
    float sw = 0.f, bias = 0.f, sx = 0.f;
    auto fetch = [&](int tile) {
      if (tile >= tiles) return;
      int tn, tm;
      order.at(tile, tn, tm);
      const int n = tn * w8::PAIR_ROWS + static_cast<int>(rank) * 128 + quarter * 32 + lane;
      const int m = tm * w8::PAIR_ROWS + t;
      sw = n < out.N ? w8a8_channel(out.sw, out.sw_f32 ? 2 : 1, n) : 0.f;
      bias = n < out.N ? w8a8_channel(out.bias, out.bias_kind, n) : 0.f;
      sx = m < out.M ? out.sx[m] : 0.f;
    };
    fetch(pair);
    for (int tile = pair; tile < tiles; tile += pairs, ++n_tile) {
      const int a = n_tile & 1;
      int tn, tm;
      order.at(tile, tn, tm);
      const int n_warp = tn * w8::PAIR_ROWS + static_cast<int>(rank) * 128 + quarter * 32;
      const int m0 = tm * w8::PAIR_ROWS;
      const int cols = min(w8::PAIR_ROWS, out.M - m0);
      const float sw_now = sw, bias_now = bias;
      sm.sx[a][t] = sx;
      rla_named_bar_sync(1, 256);  // (nobody still reads what tile - 2 had here)
      fetch(tile + pairs);
      bool ok = rla_mbar_wait_cluster(&sm.dfull[a], (n_tile >> 1) & 1, RLA_DEVERR_TIMEOUT_ACCUM, abort_flag);
      ok = __all_sync(0xffffffffu, ok);
      // (a warp that gave up still meets the others at the barrier above)
      if (!ok) continue;
      rla_tc_fence_after();
      w8a8_store_warp(out, tmem + lane_addr + a * 256, half * 32, 64, cols, m0, n_warp, sw_now, bias_now, sm.sx[a], sm.buf[warp - 2]);
      rla_tc_fence_before();
      __syncwarp();
      if (lane == 0) rla_mbar_arrive_cluster(rla_mapa(rla_smem_u32(&sm.dempty[a]), 0));
    }
  }
  rla_tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0) {
    rla_st_cluster_u32(rla_mapa(rla_smem_u32(&sm.peer_abort_flag), rank ^ 1u), static_cast<uint32_t>(*abort_flag));
    rla_st_cluster_u32(rla_mapa(rla_smem_u32(&sm.peer_issued), rank ^ 1u), static_cast<uint32_t>(sm.issued));
  }
  __syncwarp();
  // both CTAs are through: without a wait that gave up, nothing reads or writes
  // the other's shared memory or TMEM any more
  rla_cluster_sync();
  if (*abort_flag || sm.peer_abort_flag) {  // (the same in all threads of both)
    if (rank == 0 && threadIdx.x == 0) w8a8_pair_drain(sm, HALF);
    __syncwarp();
    rla_cluster_sync();
  }
  if (warp == 1) {
    rla_tc_fence_after();
    rla_tmem2_dealloc(tmem, 512);
  }
}

// Rows of K bytes (any alignment, any stride) into rows of `ldd` bytes, zero
// behind K: what TMA's 16-byte rules need where K or a row stride is odd.  A
// thread makes 16 bytes of five aligned words; at the ends of a row, where those
// would reach beyond it, of single bytes.
__global__ void w8a8_align_rows_kernel(const int8_t* __restrict__ src, int64_t lds, int8_t* __restrict__ dst, int ldd,
                                       int64_t rows, int K) {
  const int per_row = ldd / 16;
  const int64_t total = rows * per_row;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int64_t r = i / per_row;
    const int k = static_cast<int>(i - r * per_row) * 16;
    const int8_t* p = src + r * lds + k;
    const uint32_t off = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p)) & 3u;
    alignas(16) uint32_t v[4];
    if (k >= static_cast<int>(off) && k + 20 - static_cast<int>(off) <= K) {
      const uint32_t* a = reinterpret_cast<const uint32_t*>(p - off);  // five aligned words, all of this row
      uint32_t lo = a[0];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t hi = a[j + 1];
        v[j] = __funnelshift_r(lo, hi, off * 8);
        lo = hi;
      }
    } else {
      int8_t* b = reinterpret_cast<int8_t*>(v);
#pragma unroll
      for (int j = 0; j < 16; ++j) b[j] = k + j < K ? p[j] : int8_t(0);
    }
    *reinterpret_cast<uint4*>(dst + r * ldd + k) = *reinterpret_cast<const uint4*>(v);
  }
}

struct W8Plan {
  bool pair = false;
  int bt = 0, splits = 1, stages = 0;
  int grid_x = 0, grid_y = 0;
  size_t smem = 0;
};

// A pair CTA takes all of its SM's shared memory, although it needs less, so
// that no other CTA with Tensor Memory sits beside it: a pair holds all 512
// columns of one SM while it waits for those of the other.
constexpr int kW8PairSmem = 227 * 1024;
static_assert(sizeof(W8PairShared) + 1024 <= kW8PairSmem, "the ring fits");

// Dynamic shared memory of the split kernel, at most.
constexpr int kW8SplitSmem = w8::MAX_STAGES * w8::stage_bytes(w8::MAX_BT) + 1024;
static cudaError_t w8a8_allow_split_smem() {
  static std::atomic<uint64_t> done{0};
  return allow_smem(w8a8_split_kernel, kW8SplitSmem, done);
}

// CTAs that run at once, one an SM, when `splits` of them form a cluster (whole
// clusters: all CTAs of one sit in one GPC).  Per device.
static int w8a8_cluster_ctas(int splits) {
  static std::atomic<int> cache[64][w8::MAX_SPLITS + 1];
  const int sms = device_sm_count();
  int dev = -1;
  if (splits == 1 || cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return sms / splits * splits;
  int n = cache[dev][splits].load(std::memory_order_relaxed);
  if (n > 0) return n;
  cudaError_t e = w8a8_allow_split_smem();
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(1, 1, splits);
  cfg.blockDim = dim3(w8::THREADS);
  cfg.dynamicSmemBytes = kW8SplitSmem;  // more than half an SM's
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 1;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = static_cast<unsigned>(splits);
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (e == cudaSuccess) e = cudaOccupancyMaxActiveClusters(&n, w8a8_split_kernel, &cfg);
  if (e != cudaSuccess || n < 1) {
    (void)cudaGetLastError();
    return sms / splits * splits;  // (no device: planning only)
  }
  cache[dev][splits].store(n * splits, std::memory_order_relaxed);
  return n * splits;
}
// Split CTAs that an SM holds with this ring: the dynamic shared memory, the
// static and the system's.  (The occupancy query counts one an SM for a kernel
// that allocates Tensor Memory; as many run as fit.)
static int w8a8_per_sm(int bt, int stages) { return 228 * 1024 / (stages * w8::stage_bytes(bt) + 4 * 1024); }

// Which kernel, tile, split of K and ring, by estimated time.  Measured on
// B200 (CUDA graphs, inputs beyond L2), over token tiles of 64 to 256, 1 to 8
// slices and rings of 2 to 12 stages:
//  - Several CTAs an SM with short rings, whose starts and ends overlap one
//    another's streams (and the next launch's start), beat one CTA with the
//    whole shared memory: 8x28672x8192 38 us against 83, 16x14336x4096 13.5
//    against 16.6, 1x4096x4096 6.4 against 7.9.  So token tiles of at most
//    128 columns and two or three stages.
//  - A round of n CTAs an SM takes about 0.31 + 0.16 n us a k block (256x4096,
//    512x4096, 512x11008, K = 4096), a seventh more with two stages.
//  - Joining the slices takes about 2.4 us for a tile of 128 tokens, in
//    proportion for narrower ones, and longer where several CTAs of an SM do
//    it: 3000x512x512 8.9 us unsplit, 13.7 as two slices.
//  - A round starts and ends in about 1.5 us: 1x28672x1024 8.3 us as 3 slices
//    in one round, 16.4 as 8 in three.
//  - Slices whose clusters do not all fit at once cost a second round
//    (300x4096x4096: 21.8 us as 3, 16.1 as 2).
//  - Pairs (256 x 256 tiles) take 2.7 us and, a round, 0.38 us a k block, or
//    the 3.85 us of an epilogue where that is longer.  Split clusters take 2.6
//    us, 0.88 of the sum of the above, and 1.1 us a tile of 128 tokens that an
//    SM stores.  Fitted to 238 sizes (M 144..4096, N 256..28672, K 128..8192)
//    that both ran, it picks the faster one or one less than 16 % slower:
//    272x28672x128 pairs 16.5 us, split 9.9; 512x11008x4096 25.6 and 27.3;
//    2048x4096x1024 12.7 and 18.5; 272x28672x4096 44 and 84.
static W8Plan w8a8_plan(int64_t M, int64_t N, int64_t K) {
  W8Plan p;
  const int sms = device_sm_count();
  const int kb = static_cast<int>((K + w8::BK - 1) / w8::BK);
  // token tiles of equal width, a multiple of 16 columns
  p.grid_y = static_cast<int>((M + 127) / 128);
  p.bt = static_cast<int>(((M + p.grid_y - 1) / p.grid_y + 15) / 16 * 16);
  p.grid_x = static_cast<int>((N + w8::BR - 1) / w8::BR);
  const int64_t tiles = (int64_t)p.grid_x * p.grid_y;
  const int stage = w8::stage_bytes(p.bt);
  double best = -1;
  for (int s = 1; s <= w8::MAX_SPLITS && s <= kb; ++s) {
    for (int st = 3; st >= 2; --st) {
      if (s > 1 && st * stage < p.bt * w8::BR * 4) continue;  // no room for the partial tile
      const int c = w8a8_per_sm(p.bt, st);
      const int64_t slots = (int64_t)c * w8a8_cluster_ctas(s), rounds = (tiles * s + slots - 1) / slots;
      const int64_t n = rounds > 1 ? c : std::min<int64_t>(c, (tiles * s + sms - 1) / sms);
      double us = static_cast<double>(rounds) * ((kb + s - 1) / s) * (0.31 + 0.16 * n) * (st == 2 ? 1.15 : 1.0);
      us += 1.5 * rounds;
      if (s > 1) us += 2.4 * p.bt / 128 * (1 + 0.5 * (n - 1));
      if (best < 0 || us < best) {
        best = us;
        p.splits = s;
        p.stages = st;
      }
    }
  }
  if (tiles * p.splits <= w8a8_cluster_ctas(p.splits)) p.stages = w8::MAX_STAGES;  // one CTA an SM: room for more
  // (no more stages than k blocks, but room for the partial tile)
  p.stages = std::max(std::min(p.stages, (kb + p.splits - 1) / p.splits),
                      p.splits > 1 ? (p.bt * w8::BR * 4 + stage - 1) / stage : 1);
  p.smem = (size_t)p.stages * stage + 1024;
  if (M > 128) {
    const int64_t pair_tiles = ((N + 255) / 256) * ((M + 255) / 256), pairs = std::max(1, sms / 2);
    const double rounds = static_cast<double>((pair_tiles + pairs - 1) / pairs);
    const double stores = static_cast<double>(tiles) * p.bt / 128 / sms;
    p.pair = 2.7 + rounds * std::max(0.38 * kb, 3.85) < 2.6 + 0.88 * best + 1.1 * stores || p.grid_y > 65535;
  }
  return p;
}

static cudaError_t launch_w8a8(const int8_t* x, int64_t ldx, const int8_t* w, int64_t ldw, const W8Out& out, int64_t K,
                               cudaStream_t s) {
  const W8Plan p = w8a8_plan(out.M, out.N, K);
  CUtensorMap tw, tx;
  if (!make_tmap_2d(&tw, CU_TENSOR_MAP_DATA_TYPE_UINT8, w, (uint64_t)K, (uint64_t)out.N, (uint64_t)ldw, w8::BK, w8::BR,
                    CU_TENSOR_MAP_SWIZZLE_128B) ||
      !make_tmap_2d(&tx, CU_TENSOR_MAP_DATA_TYPE_UINT8, x, (uint64_t)K, (uint64_t)out.M, (uint64_t)ldx, w8::BK,
                    p.pair ? 128 : p.bt, CU_TENSOR_MAP_SWIZZLE_128B))
    return cudaErrorInvalidValue;
  const int num_kb = static_cast<int>((K + w8::BK - 1) / w8::BK);
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(w8::THREADS);
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (p.pair) {
    W8Order order;
    order.tiles_n = (out.N + w8::PAIR_ROWS - 1) / w8::PAIR_ROWS;
    order.tiles_m = (out.M + w8::PAIR_ROWS - 1) / w8::PAIR_ROWS;
    // a group of token tiles takes at most 32 MB of L2
    order.group = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(order.tiles_m, (32 << 20) / (w8::PAIR_ROWS * K))));
    const int64_t tiles = (int64_t)order.tiles_n * order.tiles_m;
    if (tiles > INT32_MAX / 2) return cudaErrorInvalidConfiguration;
    const int pairs = static_cast<int>(std::min<int64_t>(tiles, device_sm_count() / 2));
    cfg.gridDim = dim3(2 * pairs);
    cfg.blockDim = dim3(w8::PAIR_THREADS);
    cfg.dynamicSmemBytes = kW8PairSmem;
    static std::atomic<uint64_t> done{0};
    const cudaError_t e = allow_smem(w8a8_pair_kernel, (int)cfg.dynamicSmemBytes, done);
    if (e != cudaSuccess) return e;
    return cudaLaunchKernelEx(&cfg, w8a8_pair_kernel, tw, tx, out, num_kb, order);
  }
  const cudaError_t e = w8a8_allow_split_smem();
  if (e != cudaSuccess) return e;
  cfg.gridDim = dim3(p.grid_x, p.grid_y, p.splits);
  cfg.dynamicSmemBytes = p.smem;
  if (p.splits > 1) {
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = 1;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = static_cast<unsigned>(p.splits);
    cfg.numAttrs = 2;
  }
  int cols = 32;  // TMEM columns: a power of two
  while (cols < p.bt) cols *= 2;
  return cudaLaunchKernelEx(&cfg, w8a8_split_kernel, tw, tx, out, num_kb, p.stages, p.bt, cols);
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
    int vec = 8;  // (y may have any stride: a slice of a wider tensor)
    while (vec > 1 && ((reinterpret_cast<uintptr_t>(y) & (2u * vec - 1)) != 0 || (M > 1 && ldy % vec != 0))) vec /= 2;
    const W8Out out{x_scale, scale, scale_dtype == RLA_DTYPE_F32 ? 1 : 0, bias, bias_kind, static_cast<__half*>(y), ldy,
                    vec, (int)M, (int)N};
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
