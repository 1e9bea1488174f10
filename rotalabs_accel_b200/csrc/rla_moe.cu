// A whole mixture-of-experts layer for up to 32 tokens with int8 expert
// weights (one scale an output channel), in two kernels:
//   1. route + gate/up:  p = softmax(x router^T), the top_k largest per token;
//      a = fp16( silu(sg * (Wg x)) * su * (Wu x) ) for every chosen expert
//   2. down + combine:   y = fp16( sum over the chosen experts of
//                                  c * sd * (Wd a) ),  c = p or p / sum p
//
// Bound by the weights of the experts that some token chose: each byte is
// read once, by one warp, and meets all tokens that chose its expert.  The
// products are "swap-AB" tensor-core products like the decode GEMM's: 16
// weight rows are the rows of an m16n8k16 MMA, tokens its columns, int8 ->
// fp16 in registers, fp32 sums.  Column = token index, so no gather: a lane
// whose token did not choose the expert loads nothing and multiplies zeros,
// and 8-token tiles without any such token are skipped.
//
// Routing.  Which weights to read is not known before the logits are, so
// the whole GPU waits for them.  Each cluster of 8 CTAs computes all logits by
// itself (K split over its CTAs, joined through distributed shared memory):
// no grid-wide barrier, one kernel launch less, and 1/8 of the router's bytes
// an SM.  A choice between two experts is a border, so the partial logits
// (fp32 sums over 1/8 of K or less) are added in 64 bits.  Ties go to the
// lower index.
//
// Every sum has a fixed order: results are bit-reproducible.
#include <algorithm>

#include "rla_common.cuh"
#include "rla_internal.h"

namespace rla {

namespace moe {
constexpr int THREADS = 256;
constexpr int WARPS = THREADS / 32;
constexpr int CLUSTER = 8;
constexpr int MAX_T = 32;
constexpr int MAX_E = 256;
constexpr int MAX_K = 32;  // top_k
constexpr int MAX_SPLITS = 8;
}  // namespace moe

struct MoeArgs {
  const __half* x;  // [T, H], row stride ldx
  int64_t ldx;
  const __half* router;  // [E, H]
  const int8_t* w_gate;  // [E, I, H]
  const int8_t* w_up;
  const int8_t* w_down;  // [E, H, I]
  const void* s_gate;    // [E, I]
  const void* s_up;
  const void* s_down;  // [E, H]
  int scale_f32;
  __half* y;  // [T, H], row stride ldy
  int64_t ldy;
  __half* a;    // workspace: [T * top_k, I]
  int* ids;     // workspace: [T * top_k]
  float* coef;  // workspace: [T * top_k]
  int T, H, I, E, top_k, renorm;
};

RLA_DEVFN float moe_scale(const void* p, int f32, int64_t i) {
  return f32 ? static_cast<const float*>(p)[i] : __half2float(static_cast<const __half*>(p)[i]);
}
// Store into CTA `rank`'s copy of the shared variable at `p`.
RLA_DEVFN void rla_st_dsmem_u32(const void* p, uint32_t rank, uint32_t v) {
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(remote), "r"(v) : "memory");
}

// What every CTA of both kernels knows of the routing.
struct MoeRoute {
  int ids[moe::MAX_T * moe::MAX_K];
  float coef[moe::MAX_T * moe::MAX_K];
  uint32_t mask[moe::MAX_E];                // tokens that chose expert e
  uint8_t slot[moe::MAX_E][moe::MAX_T];     // at which of their top_k places
  short active[moe::MAX_E];                 // experts that some token chose, in order
  int warp_count[moe::WARPS];
  int num_active;
};

// ids / coef -> mask, slot, active.  All threads of the CTA.
RLA_DEVFN void moe_build_lists(MoeRoute& r, int T, int E, int top_k) {
  const int tid = threadIdx.x;
  static_assert(moe::THREADS >= moe::MAX_E, "one thread an expert");
  if (tid < E) r.mask[tid] = 0;
  __syncthreads();
  for (int p = tid; p < T * top_k; p += moe::THREADS) {
    const int t = p / top_k;
    atomicOr(&r.mask[r.ids[p]], 1u << t);
    r.slot[r.ids[p]][t] = static_cast<uint8_t>(p - t * top_k);
  }
  __syncthreads();
  const bool on = tid < E && r.mask[tid] != 0;
  const uint32_t votes = __ballot_sync(0xffffffffu, on);
  if ((tid & 31) == 0) r.warp_count[tid >> 5] = __popc(votes);
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < moe::WARPS; ++w) {
    before += w < (tid >> 5) ? r.warp_count[w] : 0;
    all += r.warp_count[w];
  }
  if (on) r.active[before + __popc(votes & ((1u << (tid & 31)) - 1))] = static_cast<short>(tid);
  if (tid == 0) r.num_active = all;
  __syncthreads();
}

// One 64-wide k chunk: 16 weight rows (rows g and g + 8 in wa) times NT tiles
// of 8 tokens.  The k order inside the fragments follows the 16-byte loads
// (rla_skinny.cu); `tiles` has a bit for each 8-token tile with a token.
template <int NT>
RLA_DEVFN void moe_chunk_mma(float (&acc)[NT][4], const uint4 (&wa)[2], const uint4 (&xb)[NT][2], uint32_t tiles) {
  const uint32_t* w0 = reinterpret_cast<const uint32_t*>(&wa[0]);
  const uint32_t* w1 = reinterpret_cast<const uint32_t*>(&wa[1]);
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    uint32_t a0, a1, a2, a3;
    rla_i8x4_to_h2x2(w0[s], a0, a2);
    rla_i8x4_to_h2x2(w1[s], a1, a3);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      if (NT > 1 && !(tiles >> t & 1)) continue;
      const uint32_t* xw = reinterpret_cast<const uint32_t*>(&xb[t][0]);
      rla_mma_16816(acc[t], a0, a1, a2, a3, xw[2 * s], xw[2 * s + 1]);
    }
  }
}

RLA_DEVFN uint32_t moe_tiles(uint32_t mask) {
  return (mask & 0xffu ? 1u : 0u) | (mask & 0xff00u ? 2u : 0u) | (mask & 0xff0000u ? 4u : 0u) |
         (mask & 0xff000000u ? 8u : 0u);
}

// Partial logits of this CTA's K slice: part[t][e], fp32.  Warps take 16
// experts each; a lane's fragment columns are its 8-token tile's tokens.
template <int NT>
RLA_DEVFN void moe_logits(const MoeArgs& g, int rank, float* part) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int gr = lane >> 2, q = lane & 3;
  const int blocks = (g.H + 31) / 32;  // 32 halves = one 8-half load of each of 4 lanes
  const int b0 = blocks * rank / moe::CLUSTER, b1 = blocks * (rank + 1) / moe::CLUSTER;
  for (int e0 = warp * 16; e0 < g.E; e0 += moe::WARPS * 16) {
    const int r0 = min(e0 + gr, g.E - 1), r1 = min(e0 + gr + 8, g.E - 1);
    const __half* w0 = g.router + (int64_t)r0 * g.H + q * 8;
    const __half* w1 = g.router + (int64_t)r1 * g.H + q * 8;
    float acc[NT][4] = {};
#pragma unroll 4
    for (int b = b0; b < b1; ++b) {
      const uint4 zero = make_uint4(0, 0, 0, 0);
      const bool in = b * 32 + q * 8 < g.H;
      const uint4 a = in ? rla_ldg_keep(w0 + b * 32) : zero;
      const uint4 c = in ? rla_ldg_keep(w1 + b * 32) : zero;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const int tok = t * 8 + gr;
        const uint4 x = in && tok < g.T ? rla_ldg_keep(g.x + (int64_t)tok * g.ldx + q * 8 + b * 32) : zero;
        rla_mma_16816(acc[t], a.x, c.x, a.y, c.y, x.x, x.y);
        rla_mma_16816(acc[t], a.z, c.z, a.w, c.w, x.z, x.w);
      }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int e = e0 + gr + 8 * (i >> 1), tok = t * 8 + 2 * q + (i & 1);
        if (e < g.E && tok < g.T) part[tok * g.E + e] = acc[t][i];
      }
  }
}

// Top-k and softmax of the tokens t = rank, rank + 8, ... (one a warp), from
// all ranks' partial logits; ids and coef go into every CTA of the cluster.
RLA_DEVFN void moe_choose(const MoeArgs& g, int rank, const float* part, MoeRoute& r) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  constexpr int PER = moe::MAX_E / 32;
  for (int t = rank + moe::CLUSTER * warp; t < g.T; t += moe::CLUSTER * moe::WARPS) {
    double v[PER];
    double top = -INFINITY;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int e = lane + 32 * i;
      v[i] = -INFINITY;
      if (e < g.E) {
        double sum = 0;
        const uint32_t at = rla_smem_u32(part + t * g.E + e);
#pragma unroll
        for (int c = 0; c < moe::CLUSTER; ++c) {
          uint32_t remote;
          float f;
          asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(at), "r"(c));
          asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(f) : "r"(remote) : "memory");
          sum += static_cast<double>(f);
        }
        v[i] = sum;
        top = fmax(top, sum);  // (drops NaN)
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmax(top, __shfl_xor_sync(0xffffffffu, top, o));
    // softmax relative to the largest; a NaN logit makes the sum NaN
    float total = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (lane + 32 * i < g.E) total += expf(static_cast<float>(v[i] - top));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    // k rounds of "largest not yet taken, the lower index on a tie"; NaN
    // counts as the smallest, so that every round finds an expert
    uint32_t taken = 0;
    float chosen = 0.f;  // sum of the chosen, in the order of choice
    int my_id = 0;
    float my_p = 0.f;
    for (int j = 0; j < g.top_k; ++j) {
      double bv = -INFINITY;
      int bi = INT32_MAX;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int e = lane + 32 * i;
        const double c = isnan(v[i]) ? -INFINITY : v[i];
        if (e < g.E && !(taken >> i & 1) && (bi == INT32_MAX || c > bv)) bv = c, bi = e;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const double ov = __shfl_xor_sync(0xffffffffu, bv, o);
        const int oi = __shfl_xor_sync(0xffffffffu, bi, o);
        if (oi != INT32_MAX && (bi == INT32_MAX || ov > bv || (ov == bv && oi < bi))) bv = ov, bi = oi;
      }
      const float p = expf(static_cast<float>(bv - top)) / total;
      if (lane == (bi & 31)) taken |= 1u << (bi >> 5);
      chosen += p;
      if (lane == j) my_id = bi, my_p = p;
    }
    if (lane < g.top_k) {
      const float c = g.renorm ? my_p / chosen : my_p;
      for (int d = 0; d < moe::CLUSTER; ++d) {
        rla_st_dsmem_u32(&r.ids[t * g.top_k + lane], d, static_cast<uint32_t>(my_id));
        rla_st_dsmem_u32(&r.coef[t * g.top_k + lane], d, __float_as_uint(c));
      }
    }
  }
}

template <int NT>
__global__ void __cluster_dims__(moe::CLUSTER, 1, 1) __launch_bounds__(moe::THREADS, 2)
    moe_gate_up_kernel(const MoeArgs g) {
  extern __shared__ __align__(16) uint8_t moe_smem[];
  MoeRoute& r = *reinterpret_cast<MoeRoute*>(moe_smem);
  float* part = reinterpret_cast<float*>(moe_smem + sizeof(MoeRoute));  // [T][E]
  __shared__ float red[moe::WARPS - 1][NT * 4][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int gr = lane >> 2, q = lane & 3;
  const int rank = static_cast<int>(rla_cluster_ctarank());

  rla_griddep_launch_dependents();
  rla_griddep_wait();
  moe_logits<NT>(g, rank, part);
  rla_cluster_sync();
  moe_choose(g, rank, part, r);
  rla_cluster_sync();
  if (blockIdx.x == 0)
    for (int p = threadIdx.x; p < g.T * g.top_k; p += moe::THREADS) {
      g.ids[p] = r.ids[p];
      g.coef[p] = r.coef[p];
    }
  moe_build_lists(r, g.T, g.E, g.top_k);

  // Units of 8 gate rows and the same 8 up rows; the warps split K.
  const int groups = (g.I + 7) / 8;
  const int units = r.num_active * groups;
  const int chunks = (g.H + 63) / 64;
  constexpr int U = NT >= 4 ? 2 : 4;
  const uint4 zero = make_uint4(0, 0, 0, 0);
  for (int u = blockIdx.x; u < units; u += gridDim.x) {
    const int e = r.active[u / groups];
    const int i0 = (u % groups) * 8;
    const uint32_t mask = r.mask[e];
    const uint32_t tiles = moe_tiles(mask);
    const int64_t row = (int64_t)e * g.I + min(i0 + gr, g.I - 1);
    const int8_t* wg = g.w_gate + row * g.H + q * 16;
    const int8_t* wu = g.w_up + row * g.H + q * 16;
    float acc[NT][4] = {};
    for (int c = warp; c < chunks; c += moe::WARPS * U) {
      uint4 wa[U][2], xb[U][NT][2];
#pragma unroll
      for (int v = 0; v < U; ++v) {
        const int k = (c + v * moe::WARPS) * 64;
        const bool in = k + q * 16 < g.H;
        wa[v][0] = in ? rla_ldg_stream(wg + k) : zero;
        wa[v][1] = in ? rla_ldg_stream(wu + k) : zero;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const int tok = t * 8 + gr;
          const bool has = in && (mask >> tok & 1);
          const __half* xp = g.x + (int64_t)tok * g.ldx + q * 16 + k;
          xb[v][t][0] = has ? rla_ldg_keep(xp) : zero;
          xb[v][t][1] = has ? rla_ldg_keep(xp + 8) : zero;
        }
      }
#pragma unroll
      for (int v = 0; v < U; ++v) moe_chunk_mma<NT>(acc, wa[v], xb[v], tiles);
    }
    __syncthreads();  // the previous unit's sums have been read
    if (warp > 0) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) red[warp - 1][t * 4 + i][lane] = acc[t][i];
    }
    __syncthreads();
    if (warp == 0) {
      const int i = i0 + gr;
      const float sg = i < g.I ? moe_scale(g.s_gate, g.scale_f32, (int64_t)e * g.I + i) : 0.f;
      const float su = i < g.I ? moe_scale(g.s_up, g.scale_f32, (int64_t)e * g.I + i) : 0.f;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        if (!(tiles >> t & 1)) continue;
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int w = 0; w < moe::WARPS - 1; ++w) acc[t][j] += red[w][t * 4 + j][lane];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int tok = t * 8 + 2 * q + j;
          if ((mask >> tok & 1) && i < g.I) {
            const float gate = acc[t][j] * sg, up = acc[t][2 + j] * su;
            // the down product's tensor-core operand is fp16: one rounding
            g.a[((int64_t)tok * g.top_k + r.slot[e][tok]) * g.I + i] =
                __float2half_rn(__fdividef(gate, 1.0f + __expf(-gate)) * up);
          }
        }
      }
    }
  }
}

// One CTA: 16 output rows, and of the (active expert, 64-wide chunk of I)
// list the `splits`-th part, of which each warp takes a contiguous run.
template <int NT>
__global__ void __launch_bounds__(moe::THREADS, 2) moe_down_kernel(const MoeArgs g) {
  extern __shared__ __align__(16) uint8_t moe_smem[];
  MoeRoute& r = *reinterpret_cast<MoeRoute*>(moe_smem);
  __shared__ __align__(16) float red[moe::WARPS][NT * 4][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int gr = lane >> 2, q = lane & 3;
  const int splits = gridDim.y, split = blockIdx.y;  // == cluster rank

  rla_griddep_launch_dependents();
  rla_griddep_wait();
  for (int p = threadIdx.x; p < g.T * g.top_k; p += moe::THREADS) {
    r.ids[p] = g.ids[p];
    r.coef[p] = g.coef[p];
  }
  __syncthreads();
  moe_build_lists(r, g.T, g.E, g.top_k);

  const int n0 = blockIdx.x * 16;
  const int na = min(n0 + gr, g.H - 1), nb = min(n0 + gr + 8, g.H - 1);
  const int chunks = (g.I + 63) / 64;
  const int64_t items = (int64_t)r.num_active * chunks;
  const int parts = splits * moe::WARPS, mine = split * moe::WARPS + warp;
  int64_t c0 = items * mine / parts;
  const int64_t c1 = items * (mine + 1) / parts;
  constexpr int U = NT >= 4 ? 2 : 4;
  const uint4 zero = make_uint4(0, 0, 0, 0);
  float sum[NT][4] = {};
  while (c0 < c1) {
    const int ai = static_cast<int>(c0 / chunks);
    const int e = r.active[ai];
    const int kc0 = static_cast<int>(c0 - (int64_t)ai * chunks);
    const int kc1 = static_cast<int>(min((int64_t)chunks, c1 - (int64_t)ai * chunks));
    const uint32_t mask = r.mask[e];
    const uint32_t tiles = moe_tiles(mask);
    const int8_t* w0 = g.w_down + ((int64_t)e * g.H + na) * g.I + q * 16;
    const int8_t* w1 = g.w_down + ((int64_t)e * g.H + nb) * g.I + q * 16;
    const __half* ap[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int tok = t * 8 + gr;
      const int64_t arow = (mask >> tok & 1) ? (int64_t)tok * g.top_k + r.slot[e][tok] : 0;
      ap[t] = g.a + arow * g.I + q * 16;
    }
    float acc[NT][4] = {};
    for (int c = kc0; c < kc1; c += U) {
      uint4 wa[U][2], xb[U][NT][2];
#pragma unroll
      for (int v = 0; v < U; ++v) {
        const int k = (c + v) * 64;
        const bool in = c + v < kc1 && k + q * 16 < g.I;
        wa[v][0] = in ? rla_ldg_stream(w0 + k) : zero;
        wa[v][1] = in ? rla_ldg_stream(w1 + k) : zero;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const bool has = in && (mask >> (t * 8 + gr) & 1);
          xb[v][t][0] = has ? rla_ldg_keep(ap[t] + k) : zero;
          xb[v][t][1] = has ? rla_ldg_keep(ap[t] + k + 8) : zero;
        }
      }
#pragma unroll
      for (int v = 0; v < U; ++v) moe_chunk_mma<NT>(acc, wa[v], xb[v], tiles);
    }
    // this expert's part: x channel scale x token coefficient
    const float s0 = moe_scale(g.s_down, g.scale_f32, (int64_t)e * g.H + na);
    const float s1 = moe_scale(g.s_down, g.scale_f32, (int64_t)e * g.H + nb);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int tok = t * 8 + 2 * q + j;
        if (mask >> tok & 1) {
          const float c = r.coef[tok * g.top_k + r.slot[e][tok]];
          sum[t][j] = fmaf(acc[t][j] * s0, c, sum[t][j]);
          sum[t][2 + j] = fmaf(acc[t][2 + j] * s1, c, sum[t][2 + j]);
        }
      }
    }
    c0 = (int64_t)ai * chunks + kc1;
  }

#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) red[warp][t * 4 + i][lane] = sum[t][i];
  __syncthreads();
  // the CTA's sum into red[0] (each thread its own entries), then the ranks'
  for (int p = threadIdx.x; p < NT * 4 * 32; p += moe::THREADS) {
    float v = red[0][p / 32][p % 32];
#pragma unroll
    for (int w = 1; w < moe::WARPS; ++w) v += red[w][p / 32][p % 32];
    red[0][p / 32][p % 32] = v;
  }
  if (splits > 1)
    rla_cluster_sync();
  else
    __syncthreads();
  if (split == 0) {
    for (int p = threadIdx.x; p < NT * 4 * 32; p += moe::THREADS) {
      const int l = p % 32, ti = p / 32, t = ti / 4, i = ti % 4;
      float v = red[0][ti][l];
      const uint32_t at = rla_smem_u32(&red[0][ti][l]);
      for (int c = 1; c < splits; ++c) {
        uint32_t remote;
        float f;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(at), "r"(c));
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(f) : "r"(remote) : "memory");
        v += f;
      }
      const int n = n0 + (l >> 2) + 8 * (i >> 1), tok = t * 8 + 2 * (l & 3) + (i & 1);
      if (n < g.H && tok < g.T) g.y[(int64_t)tok * g.ldy + n] = __float2half_rn(v);
    }
  }
  if (splits > 1) rla_cluster_sync();  // no CTA leaves while rank 0 may still read it
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
template <int NT>
static cudaError_t launch_moe(const MoeArgs& g, cudaStream_t s) {
  const int sms = device_sm_count();
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(moe::THREADS);
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;

  cfg.dynamicSmemBytes = sizeof(MoeRoute) + (size_t)g.T * g.E * 4;
  cudaError_t e = cudaFuncSetAttribute(moe_gate_up_kernel<NT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       (int)cfg.dynamicSmemBytes);
  if (e != cudaSuccess) return e;
  const int64_t most = (int64_t)std::min(g.E, g.T * g.top_k) * ((g.I + 7) / 8);
  int64_t ctas = std::min<int64_t>(2 * sms, most);
  ctas = (ctas + moe::CLUSTER - 1) / moe::CLUSTER * moe::CLUSTER;
  cfg.gridDim = dim3((unsigned)ctas);
  e = cudaLaunchKernelEx(&cfg, moe_gate_up_kernel<NT>, g);
  if (e != cudaSuccess) return e;

  cfg.dynamicSmemBytes = sizeof(MoeRoute);
  const int rows = (g.H + 15) / 16;
  int splits = std::max(1, std::min(moe::MAX_SPLITS, 2 * sms / rows));
  cfg.gridDim = dim3(rows, splits);
  if (splits > 1) {
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = 1;
    attr[1].val.clusterDim.y = static_cast<unsigned>(splits);
    attr[1].val.clusterDim.z = 1;
    cfg.numAttrs = 2;
  }
  return cudaLaunchKernelEx(&cfg, moe_down_kernel<NT>, g);
}

static int moe_fail(int code, const char* msg) {
  set_error("rla_moe: %s", msg);
  return code;
}

static size_t moe_up256(size_t n) { return (n + 255) & ~size_t(255); }

}  // namespace rla

extern "C" {

size_t rla_moe_workspace_size(int64_t T, int64_t I, int64_t top_k) {
  if (T <= 0 || I <= 0 || top_k <= 0 || T > RLA_MOE_MAX_TOKENS || top_k > RLA_MOE_MAX_TOP_K) return 0;
  const size_t n = (size_t)T * (size_t)top_k;
  return rla::moe_up256(n * (size_t)I * 2) + 2 * rla::moe_up256(n * 4);
}

int rla_moe(const void* x, int64_t ldx, const void* router, const int8_t* w_gate, const void* scale_gate,
            const int8_t* w_up, const void* scale_up, const int8_t* w_down, const void* scale_down, int scale_dtype,
            int renormalize, void* y, int64_t ldy, int64_t T, int64_t H, int64_t I, int64_t E, int64_t top_k,
            void* workspace, size_t workspace_bytes, void* stream) {
  using namespace rla;
  static_assert(moe::MAX_T == RLA_MOE_MAX_TOKENS && moe::MAX_E == RLA_MOE_MAX_EXPERTS && moe::MAX_K == RLA_MOE_MAX_TOP_K,
                "limits of the header");
  if (T < 0 || H < 1 || I < 1 || E < 1 || H > (1 << 24) || I > (1 << 24))
    return moe_fail(RLA_ERR_INVALID_ARGUMENT, "T must be >= 0, H and I in [1, 2^24], E >= 1");
  if (top_k < 1 || top_k > E) return moe_fail(RLA_ERR_INVALID_ARGUMENT, "top_k must be in [1, E]");
  if (T > moe::MAX_T || E > moe::MAX_E || top_k > moe::MAX_K)
    return moe_fail(RLA_ERR_UNSUPPORTED, "at most 32 tokens, 256 experts and top_k 32");
  if (H % 16 != 0 || I % 16 != 0) return moe_fail(RLA_ERR_UNSUPPORTED, "H and I must be multiples of 16");
  if (scale_dtype != RLA_DTYPE_F16 && scale_dtype != RLA_DTYPE_F32)
    return moe_fail(RLA_ERR_INVALID_ARGUMENT, "scale_dtype must be F16 or F32");
  if (T == 0) return RLA_OK;
  if (!x || !router || !w_gate || !scale_gate || !w_up || !scale_up || !w_down || !scale_down || !y)
    return moe_fail(RLA_ERR_INVALID_ARGUMENT, "null pointer");
  if (ldx < H || ldy < H) return moe_fail(RLA_ERR_INVALID_ARGUMENT, "leading dimensions must be >= H");
  auto odd = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) != 0; };
  if (odd(x) || odd(router) || odd(w_gate) || odd(w_up) || odd(w_down) || (T > 1 && ldx % 8 != 0))
    return moe_fail(RLA_ERR_UNSUPPORTED, "x (its rows too), router and weights must be 16-byte aligned");
  const size_t need = rla_moe_workspace_size(T, I, top_k);
  if (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 255u)) {
    set_error("rla_moe: needs %zu bytes of 256-byte aligned workspace (rla_moe_workspace_size), got %zu", need,
              workspace ? workspace_bytes : size_t(0));
    return RLA_ERR_WORKSPACE;
  }
  char* ws = static_cast<char*>(workspace);
  const size_t n = (size_t)T * (size_t)top_k;
  const size_t a_bytes = moe_up256(n * (size_t)I * 2);
  const MoeArgs g{static_cast<const __half*>(x), ldx, static_cast<const __half*>(router), w_gate, w_up, w_down,
                  scale_gate, scale_up, scale_down, scale_dtype == RLA_DTYPE_F32 ? 1 : 0, static_cast<__half*>(y), ldy,
                  reinterpret_cast<__half*>(ws), reinterpret_cast<int*>(ws + a_bytes),
                  reinterpret_cast<float*>(ws + a_bytes + moe_up256(n * 4)), (int)T, (int)H, (int)I, (int)E, (int)top_k,
                  renormalize ? 1 : 0};
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = T <= 8 ? launch_moe<1>(g, s) : T <= 16 ? launch_moe<2>(g, s) : launch_moe<4>(g, s);
  if (e != cudaSuccess) {
    set_error("rla_moe: %s", cudaGetErrorString(e));
    return RLA_ERR_CUDA;
  }
  note_launch();
  note_launch();
  return RLA_OK;
}

}  // extern "C"
