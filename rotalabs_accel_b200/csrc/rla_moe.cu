// A whole mixture-of-experts layer for up to 32 tokens with int8 expert
// weights (one scale an output channel), in two kernels:
//   1. route + gate/up:  p = softmax(x router^T), the top_k largest per token;
//      a = silu(sg * (Wg x)) * su * (Wu x) for every chosen expert
//   2. down + combine:   y = fp16( sum over the chosen experts of
//                                  c * sd * (Wd a) ),  c = p or p / sum p
// a is the sum of two bf16 terms, a = hi + lo with hi = a cut off to bf16, lo =
// bf16(a - hi): 2^-16 of a at most is lost and fp32's range is kept (a may be far above
// fp16's 65504 and the scales bring y back).  Tensor-core operands hold no more
// bits, so the down product is Wd hi + Wd lo in one fp32 sum.
//
// Bound by the weights of the experts that some token chose: each byte is
// read once, by one warp, and meets all tokens that chose its expert.
//
// Stream.  Every warp has a ring of its own in shared memory, filled by bulk
// tile copies that it issues itself: a stage is 128 bytes of 32 weight rows, in
// one or two copies.  One CTA of 12 or 16 warps an SM keeps warps x stages x
// 4 KB on their way (latency x bandwidth needs about 50 KB), through every
// reduction and change of expert, and no warp waits for another one's data.
// The work is cut into stages, and every CTA, and every warp of it, gets an
// equal, contiguous run; a block of rows that spans warps is added up in shared
// memory.  Measured for one token, 2 of 8 experts of 4096 x 14336 (54 us at the
// memory's rate): 69 us, the gate/up stream at 6.4 TB/s.  Loads into
// registers with the warps of a CTA splitting K and meeting after every 16 rows
// took 119 us; copies of single rows, which a warp issues one by one, 93.
//
// Products are "swap-AB" tensor-core products like the decode GEMM's: 16
// weight rows are the rows of an m16n8k16 MMA, the tokens that chose the
// expert its columns (1, 2 or 4 tiles of 8), int8 -> fp16 (bf16 in the down
// product) in registers, fp32 sums.  The down product of up to 4 tokens has hi
// and lo as columns of their own, two of the 8 for each token, and one term
// would cost as many products; of more tokens, every tile has an MMA for each.
// What the two terms cost against one of fp16 (of smaller range): 1 token, 2 of
// 8 experts 67.5 -> 69.4 us, 16 tokens, 8 of 64 71.7 -> 76.0, 32 tokens, 4 of 8
// (4096 x 2048) 75 -> 84.
// A column with no token repeats another one's activations and is
// dropped: columns of a product do not mix, and loads without conditions
// keep the instructions of a 1 KB piece near those of its conversion (40, and
// 56 to bf16).
//
// Routing.  Which weights to read is not known before the logits are, so
// the whole GPU waits for them.  Each cluster of 4 CTAs computes all logits by
// itself (K split over its CTAs, joined through distributed shared memory):
// no grid-wide barrier, one kernel launch less, and 1/4 of the router's bytes
// an SM.  A choice between two experts is a border, so the fp32 sums of the
// tensor cores, which truncate, are 128 products long (8 instructions), a
// warp's are added with what their additions lose, and the warps' in 64 bits.
// Ties go to the lower index.
//
// Every sum has a fixed order: results are bit-reproducible.
#include <cuda_bf16.h>
#include <limits.h>

#include <algorithm>
#include <atomic>

#include "rla_common.cuh"
#include "rla_internal.h"
#include "rla_tmap.cuh"

namespace rla {

namespace moe {
// By the tiles of 8 tokens (NT = 1, 2, 4): more accumulators, fewer warps, so
// that nothing spills (a spilled register comes back from an L2 that is busy
// with weights, microseconds later).
__host__ __device__ constexpr int warps(int nt) { return nt == 4 ? 12 : 16; }
constexpr int MAX_WARPS = 16;
constexpr int CLUSTER = 4;
constexpr int MAX_T = 32;
constexpr int MAX_E = 256;
constexpr int MAX_K = 32;  // top_k
constexpr int MAX_SPLITS = 8;
// A stage: 128 bytes of 32 weight rows (two 64-wide chunks), 128-byte swizzled
// by the copy (16-byte piece c of row r lies at piece c ^ (r % 8)).
constexpr int KB = 128;
constexpr int ROWS = 32;
constexpr int SLOT = ROWS * KB;
constexpr int MAX_STAGES = 3;
constexpr size_t SMEM = 227 * 1024;  // of a CTA
}  // namespace moe

// What every CTA of both kernels knows of the routing.  A pair p = token *
// top_k + place stands for (token, one of its experts); entry[] lists the
// pairs by expert, the tokens of an expert in order, and token[] their tokens.
struct MoeTables {
  float coef[moe::MAX_T * moe::MAX_K];  // by pair
  uint32_t mask[moe::MAX_E];            // tokens that chose expert e
  short begin[moe::MAX_E];              // first entry of expert e
  short active[moe::MAX_E];             // experts that some token chose, in order
  short entry[moe::MAX_T * moe::MAX_K];
  uint8_t token[moe::MAX_T * moe::MAX_K];
  int num_active, unused[3];  // (a multiple of 16 bytes)
};

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
  __nv_bfloat16* a;     // workspace: [T * top_k][hi, lo][I], see moe_place
  MoeTables* tables;    // workspace: the routing, for the second kernel
  int T, H, I, E, top_k, renorm;
};

RLA_DEVFN float moe_scale(const void* p, int f32, int64_t i) {
  return f32 ? static_cast<const float*>(p)[i] : __half2float(static_cast<const __half*>(p)[i]);
}
RLA_DEVFN uint32_t rla_and_or(uint32_t a, uint32_t b, uint32_t c) {  // a & b | c
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
// int8 -> bf16, four values of a word: bytes 0 and 2 into `even`, 1 and 3 into
// `odd`.  A byte b >= 0 is (128 + b) - 128, b < 0 is (256 + b) - 256 with
// 256 + b = 128 + (its low seven bits): both terms are exponent 0x43 with some of the
// byte's bits in the mantissa, and the difference is exact.
// (The second is made negative and added: with `sub` of this type the down
// product of one token issues a third more instructions, 35 us against 30.)
RLA_DEVFN void rla_i8x4_to_bf2x2(uint32_t w, uint32_t& even, uint32_t& odd) {
  const uint32_t v = w >> 8;
  asm("add.rn.bf16x2 %0, %1, %2;"
      : "=r"(even)
      : "r"(rla_and_or(w, 0x007f007fu, 0x43004300u)), "r"(rla_and_or(w, 0x00800080u, 0xc300c300u)));
  asm("add.rn.bf16x2 %0, %1, %2;"
      : "=r"(odd)
      : "r"(rla_and_or(v, 0x007f007fu, 0x43004300u)), "r"(rla_and_or(v, 0x00800080u, 0xc300c300u)));
}
RLA_DEVFN void rla_mma_16816_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                  uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Where channel i lies in a row of `a`: the order of the conversion above.
RLA_DEVFN int moe_place(int i) { return (i & ~3) | (i & 1) << 1 | (i >> 1 & 1); }
// v = hi + lo; hi is v cut off (the largest finite values would round up to
// infinity), lo is 0 where v is infinite or NaN.
RLA_DEVFN void moe_split(float v, __nv_bfloat16& hi, __nv_bfloat16& lo) {
  hi = __float2bfloat16_rz(v);
  const float h = __bfloat162float(hi);
  lo = __float2bfloat16_rn(fabsf(h) < INFINITY ? v - h : 0.f);
}
// Store into, and or with, CTA `rank`'s copy of the shared variable at `p`.
RLA_DEVFN void rla_st_dsmem_u32(const void* p, uint32_t rank, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(rla_mapa(rla_smem_u32(p), rank)), "r"(v) : "memory");
}
RLA_DEVFN void rla_or_dsmem_u32(const void* p, uint32_t rank, uint32_t v) {
  asm volatile("red.relaxed.cluster.shared::cluster.or.b32 [%0], %1;" ::"r"(rla_mapa(rla_smem_u32(p), rank)), "r"(v)
               : "memory");
}
RLA_DEVFN double rla_ld_dsmem_f64(const void* p, uint32_t rank) {
  double v;
  asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(rla_mapa(rla_smem_u32(p), rank)) : "memory");
  return v;
}
RLA_DEVFN float rla_ld_dsmem_f32(const void* p, uint32_t rank) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(rla_mapa(rla_smem_u32(p), rank)) : "memory");
  return v;
}
RLA_DEVFN uint4 rla_lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}

struct MoeRoute : MoeTables {
  int ids[moe::MAX_T * moe::MAX_K];
  int abort_flag;
};

// Shared memory of both kernels: routing, barriers, a buffer for partial sums
// (warps x 32 values for each column of the 8-token tiles), the warps' rings.
struct MoeShared {
  MoeRoute r;
  uint64_t full[moe::MAX_WARPS][moe::MAX_STAGES];
};
__host__ __device__ constexpr size_t moe_sums_offset() { return (sizeof(MoeShared) + 1023) & ~size_t(1023); }
__host__ __device__ constexpr int moe_tiles(int T) { return T <= 8 ? 1 : T <= 16 ? 2 : 4; }
__host__ __device__ constexpr size_t moe_ring_offset(int T) { return moe_sums_offset() + (size_t)moe_tiles(T) * moe::warps(moe_tiles(T)) * 1024; }
__host__ __device__ constexpr size_t moe_smem_bytes(int T, int stages) {
  return 1024 + moe_ring_offset(T) + (size_t)moe::warps(moe_tiles(T)) * stages * moe::SLOT;
}

// A warp's ring: issue() starts the copy of the next stage, wait() waits for
// the oldest; the caller keeps at most `stages` in flight.
struct MoeRing {
  uint32_t base;
  uint64_t* full;
  int stages, flying = 0;          // copies issued and not waited for
  int put_slot = 0, get_slot = 0, phase = 0;
  RLA_DEVFN MoeRing(uint8_t* ring, MoeShared& sm, int warp, int lane, int n) : stages(n) {
    base = rla_smem_u32(ring + (size_t)warp * n * moe::SLOT);
    full = sm.full[warp];
    if (lane < n) rla_mbar_init(&full[lane], 1);
  }
  // The next stage: columns [k, k + 128) of rows r0.. of map0 (all 32, or 16
  // of them and the same 16 rows of map1).
  template <int MAPS>
  RLA_DEVFN void issue(const CUtensorMap* map0, const CUtensorMap* map1, int k, int r0, int lane) {
    if (lane == 0) {
      uint64_t* bar = &full[put_slot];
      const uint32_t to = base + put_slot * moe::SLOT;
      rla_mbar_arrive_expect_tx(bar, moe::SLOT);
      tile(to, map0, bar, k, r0);
      if (MAPS == 2) tile(to + moe::SLOT / 2, map1, bar, k, r0);
    }
    put_slot = put_slot + 1 == stages ? 0 : put_slot + 1;
    ++flying;
  }
  RLA_DEVFN void tile(uint32_t to, const CUtensorMap* map, uint64_t* bar, int c0, int c1) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cta.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4}], [%2];" ::"r"(to),
        "l"(map), "r"(rla_smem_u32(bar)), "r"(c0), "r"(c1)
        : "memory");
  }
  RLA_DEVFN bool landed(volatile int* abort_flag) {
    const bool ok = rla_mbar_wait(&full[get_slot], phase, RLA_DEVERR_TIMEOUT_TMA_FULL, abort_flag);
    if (!__all_sync(0xffffffffu, ok)) return false;
    if (++get_slot == stages) get_slot = 0, phase ^= 1;
    --flying;
    return true;
  }
  // `at`: the stage's address; false: gave up
  RLA_DEVFN bool wait(volatile int* abort_flag, uint32_t& at) {
    at = base + get_slot * moe::SLOT;
    return landed(abort_flag);
  }
  // after a wait that gave up: the copies in flight land before the CTA leaves
  RLA_DEVFN void drain() {
    while (flying > 0 && landed(nullptr)) {
    }
  }
};

// ids, mask -> begin, active, entry, token.  All threads of the CTA.
RLA_DEVFN void moe_build_lists(MoeRoute& r, int T, int E, int top_k) {
  const int tid = threadIdx.x, lane = tid & 31;
  __syncthreads();
  if (tid < 32) {  // a lane takes PER experts in a row
    constexpr int PER = moe::MAX_E / 32;
    int count[PER], own = 0;  // entries in the low half, experts in the high half
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int e = lane * PER + i;
      count[i] = e < E ? __popc(r.mask[e]) : 0;
      own += count[i] + (count[i] ? 1 << 16 : 0);
    }
    int upto = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    if (lane == 31) r.num_active = upto >> 16;
    int at = upto - own;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int e = lane * PER + i;
      if (e < E) r.begin[e] = static_cast<short>(at & 0xffff);
      if (count[i]) {
        r.active[at >> 16] = static_cast<short>(e);
        at += count[i] + (1 << 16);
      }
    }
  }
  __syncthreads();
  for (int p = tid; p < T * top_k; p += blockDim.x) {
    const int t = p / top_k, e = r.ids[p];
    const int at = r.begin[e] + __popc(r.mask[e] & ((1u << t) - 1));
    r.entry[at] = static_cast<short>(p);
    r.token[at] = static_cast<uint8_t>(t);
  }
  __syncthreads();
}

// Start of part i of n, parts of equal length or one more.
RLA_DEVFN int moe_part(int total, int i, int n) {
  const int each = total / n;
  return each * i + min(i, total - each * n);
}

// The weight row of a stage that is row g of the MMA (and row 8 + this, of
// its row 8 + g).  In a phase of a 128-bit load eight lanes read 64 bytes of
// the rows of g and g + 1, g even: four rows apart, the swizzle puts them into
// different halves of the 32 banks.
RLA_DEVFN int moe_row(int g) { return (g >> 1) | ((g & 1) << 2); }

// 16-bit activations of a stage.  xp[t]: this lane's of column 8 t + lane / 4
// at the stage's first k + 16 * (lane % 4); a second term (PARTS = 2) lies
// `part` elements behind the first.  load(c) reads those of the 64-wide chunk
// c.  The k order inside the fragments follows the 16-byte pieces
// (rla_skinny.cu).  `bytes`: the k that are left; behind them zeros meet zeros.
RLA_DEVFN const uint16_t* moe_at(const uint16_t*, const uint16_t* p) { return p; }
RLA_DEVFN const uint16_t* moe_at(const uint16_t* base, int i) { return base + i; }
template <int NT, int PARTS>
struct MoeActs {
  static constexpr int LT = NT * PARTS;
  static constexpr int HELD = LT <= 2 ? 2 : 1;  // chunks in registers
  uint4 v[HELD][LT][2];
  template <bool FULL, class P>
  RLA_DEVFN void load(int c, const uint16_t* base, const P (&xp)[NT], int part, int bytes, int q) {
#pragma unroll
    for (int t = 0; t < LT; ++t) {
      if (FULL || c * 64 + q * 16 < bytes) {
        const uint16_t* p = moe_at(base, xp[t / PARTS]) + (t % PARTS ? part : 0) + c * 64;
        v[c % HELD][t][0] = rla_ldg_keep(p);
        v[c % HELD][t][1] = rla_ldg_keep(p + 8);
      } else {
        v[c % HELD][t][0] = v[c % HELD][t][1] = make_uint4(0, 0, 0, 0);
      }
    }
  }
  template <class P>
  RLA_DEVFN void load_first(const uint16_t* base, const P (&xp)[NT], int part, int bytes, int q) {
    if (bytes >= moe::KB) {
#pragma unroll
      for (int c = 0; c < HELD; ++c) load<true>(c, base, xp, part, bytes, q);
    } else {
#pragma unroll
      for (int c = 0; c < HELD; ++c) load<false>(c, base, xp, part, bytes, q);
    }
  }
};

// Two row tiles of 16 x NTM column tiles of 8 (those of all tokens), fp32.
template <int NTM>
using MoeAcc = float[2][NTM][4];

// One stage in shared memory at `w`: 32 weight rows x 128 k times NT tiles of
// 8 columns.  Row g of row tile m is at row m * STEP / 128 + moe_row(g) of the
// stage, row 8 + g UPPER bytes behind it.  The first chunks of x are loaded.
template <int NT, int PARTS, bool BF16, int STEP, int UPPER, int NTM, class P>
RLA_DEVFN void moe_stage(float (&acc)[2][NTM][4], uint32_t w, MoeActs<NT, PARTS>& x, const uint16_t* base, const P (&xp)[NT],
                         int part, int bytes, int lane) {
  const int q = lane & 3;
  const int row = moe_row(lane >> 2);
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const uint32_t at = w + row * 128 + (((c * 4 + q) ^ row) << 4);
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      const uint4 wa = rla_lds128(at + m * STEP), wb = rla_lds128(at + m * STEP + UPPER);
      const uint32_t* w0 = reinterpret_cast<const uint32_t*>(&wa);
      const uint32_t* w1 = reinterpret_cast<const uint32_t*>(&wb);
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        uint32_t a0, a1, a2, a3;
        if constexpr (BF16) {
          rla_i8x4_to_bf2x2(w0[s], a0, a2);
          rla_i8x4_to_bf2x2(w1[s], a1, a3);
        } else {
          rla_i8x4_to_h2x2(w0[s], a0, a2);
          rla_i8x4_to_h2x2(w1[s], a1, a3);
        }
#pragma unroll
        for (int t = 0; t < x.LT; ++t) {
          const uint32_t* xw = reinterpret_cast<const uint32_t*>(&x.v[c % x.HELD][t][0]);
          if constexpr (BF16)
            rla_mma_16816_bf16(acc[m][t / PARTS], a0, a1, a2, a3, xw[2 * s], xw[2 * s + 1]);
          else
            rla_mma_16816(acc[m][t / PARTS], a0, a1, a2, a3, xw[2 * s], xw[2 * s + 1]);
        }
      }
    }
    if (c == 0 && x.HELD == 1) {
      if (bytes >= moe::KB)
        x.template load<true>(1, base, xp, part, bytes, q);
      else
        x.template load<false>(1, base, xp, part, bytes, q);
    }
  }
}

// `n` stages of one expert from the ring, from k = k0 of `width` on.  The
// columns behind the first `count` repeat column 0 and are not used.  row(i):
// the activations' row of column i.
//
// The activations come from L2, whose latency a warp would meet at every
// stage: up to 8 tokens they are loaded a stage ahead.  32 rows share them
// (16 rows of 256 bytes a stage needed twice the loads, and too many
// registers to load them ahead: 85 us for 8-of-64 at 16 tokens, of which the
// loads took 14).
template <int NT, int PARTS, bool BF16, int STEP, int UPPER, int NTM, class Row, class Put>
RLA_DEVFN bool moe_run_tiles(float (&acc)[2][NTM][4], MoeRing& ring, int n, int k0, int width, int part, int count,
                             int lane, volatile int* abort_flag, const uint16_t* base, const Row& row, const Put& put) {
  constexpr bool AHEAD = NT * PARTS == 1;
  const int q = lane & 3;
  using P = decltype(row(0));
  P xp[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int col = t * 8 + (lane >> 2);
    xp[t] = row(col < count ? col : 0) + k0 + q * 16;
  }
  int bytes = width - k0;  // from this stage's k on
  MoeActs<NT, PARTS> x;
  if constexpr (AHEAD) x.load_first(base, xp, part, bytes, q);
#pragma unroll 1
  for (int i = 0; i < n; ++i) {
    MoeActs<NT, PARTS> ahead;
    if constexpr (AHEAD) {
      const P next[1] = {xp[0] + moe::KB};
      if (i + 1 < n) ahead.load_first(base, next, part, bytes - moe::KB, q);
    } else {
      x.load_first(base, xp, part, bytes, q);
    }
    uint32_t w;
    if (!ring.wait(abort_flag, w)) return false;
    moe_stage<NT, PARTS, BF16, STEP, UPPER>(acc, w, x, base, xp, part, bytes, lane);
    __syncwarp();
    put();
#pragma unroll
    for (int t = 0; t < NT; ++t) xp[t] += moe::KB;
    bytes -= moe::KB;
    if constexpr (AHEAD) x = ahead;
  }
  return true;
}
// The tiles that `count` columns need, of PARTS terms each.
template <int PARTS, bool BF16, int STEP, int UPPER, int NTM, class Row, class Put>
RLA_DEVFN bool moe_run(float (&acc)[2][NTM][4], MoeRing& ring, int n, int k0, int width, int part, int count, int lane,
                       volatile int* abort_flag, const uint16_t* base, const Row& row, const Put& put) {
  if constexpr (NTM == 4)
    if (count > 16)
      return moe_run_tiles<4, PARTS, BF16, STEP, UPPER>(acc, ring, n, k0, width, part, count, lane, abort_flag, base, row, put);
  if constexpr (NTM >= 2)
    if (count > 8)
      return moe_run_tiles<2, PARTS, BF16, STEP, UPPER>(acc, ring, n, k0, width, part, count, lane, abort_flag, base, row, put);
  return moe_run_tiles<1, PARTS, BF16, STEP, UPPER>(acc, ring, n, k0, width, part, count, lane, abort_flag, base, row, put);
}
template <int NTM>
RLA_DEVFN void moe_zero(float (&acc)[2][NTM][4]) {
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int t = 0; t < NTM; ++t) acc[m][t][0] = acc[m][t][1] = acc[m][t][2] = acc[m][t][3] = 0.f;
}

// Logits of this CTA's K slice, v[t][e] in 64 bits.  A warp takes 16 experts
// and, where there are fewer 16-expert tiles than warps, a part of the slice;
// the parts [parts][T][E] lie behind v.  A lane's fragment columns are its
// 8-token tile's tokens.  Every CHUNK blocks the fp32 sums go into pairs of
// fp32: a sum and what its roundings lost, which the two-sum (Knuth) gives
// exactly.  One fp32 sum of 1024 products lost up to 1e-5 of a logit; the pairs
// cost no time that shows (4 tokens, 256 experts of 4096: 58.9 us, 58.0 before).
__host__ __device__ constexpr int moe_logit_parts(int E, int warps) {
  return (E + 15) / 16 > warps / 2 ? 1 : warps / ((E + 15) / 16);
}
__host__ __device__ constexpr size_t moe_logit_bytes(int T, int E, int warps) {
  return (size_t)T * E * 8 * (moe_logit_parts(E, warps) > 1 ? 1 + moe_logit_parts(E, warps) : 1);
}
__host__ __device__ constexpr size_t moe_logit_most(int T, int warps) {
  size_t most = 0;
  for (int E = 1; E <= moe::MAX_E; ++E) most = moe_logit_bytes(T, E, warps) > most ? moe_logit_bytes(T, E, warps) : most;
  return most;
}
template <int NT>
RLA_DEVFN void moe_logits(const MoeArgs& g, int rank, double* v) {
  constexpr int WARPS = moe::warps(NT), CHUNK = 4;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int gr = lane >> 2, q = lane & 3;
  const int etiles = (g.E + 15) / 16;
  const int parts = moe_logit_parts(g.E, WARPS);
  double* part = parts > 1 ? v + g.T * g.E : v;
  const int blocks = (g.H + 31) / 32;  // 32 halves = one 8-half load of each of 4 lanes
  for (int item = warp; item < etiles * parts; item += WARPS) {
    const int e0 = item % etiles * 16, sub = item / etiles;
    const int slices = moe::CLUSTER * parts, slice = rank * parts + sub;
    const int b0 = moe_part(blocks, slice, slices), b1 = moe_part(blocks, slice + 1, slices);
    const int r0 = min(e0 + gr, g.E - 1), r1 = min(e0 + gr + 8, g.E - 1);
    const __half* w0 = g.router + (int64_t)r0 * g.H + q * 8;
    const __half* w1 = g.router + (int64_t)r1 * g.H + q * 8;
    const __half* xp[NT];  // (a column without a token repeats the last one and is not stored)
#pragma unroll
    for (int t = 0; t < NT; ++t) xp[t] = g.x + (int64_t)min(t * 8 + gr, g.T - 1) * g.ldx + q * 8;
    float sum[NT][4] = {}, lost[NT][4] = {}, acc[NT][4];
    auto block = [&](int b, bool in) {
      const uint4 zero = make_uint4(0, 0, 0, 0);
      const uint4 a = in ? rla_ldg_keep(w0 + b * 32) : zero;
      const uint4 d = in ? rla_ldg_keep(w1 + b * 32) : zero;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const uint4 x = in ? rla_ldg_keep(xp[t] + b * 32) : zero;
        rla_mma_16816(acc[t], a.x, d.x, a.y, d.y, x.x, x.y);
        rla_mma_16816(acc[t], a.z, d.z, a.w, d.w, x.z, x.w);
      }
    };
    for (int c = b0; c < b1; c += CHUNK) {
#pragma unroll
      for (int t = 0; t < NT; ++t) acc[t][0] = acc[t][1] = acc[t][2] = acc[t][3] = 0.f;
      if (c + CHUNK <= b1 && (c + CHUNK) * 32 <= g.H) {  // loads without conditions: all in flight at once
#pragma unroll
        for (int i = 0; i < CHUNK; ++i) block(c + i, true);
      } else {
#pragma unroll 1
        for (int b = c; b < b1; ++b) block(b, b * 32 + q * 8 < g.H);
      }
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float old = sum[t][i], v = acc[t][i], s = old + v, from_v = s - old;
          lost[t][i] += (old - (s - from_v)) + (v - from_v);
          sum[t][i] = s;
        }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int e = e0 + gr + 8 * (i >> 1), tok = t * 8 + 2 * q + (i & 1);
        if (e < g.E && tok < g.T)
          part[(sub * g.T + tok) * g.E + e] =
              static_cast<double>(sum[t][i]) + (fabsf(sum[t][i]) < INFINITY ? static_cast<double>(lost[t][i]) : 0.0);
      }
  }
  __syncthreads();
  if (parts == 1) return;
  for (int p = threadIdx.x; p < g.T * g.E; p += 32 * WARPS) {
    double sum = 0;
#pragma unroll 4
    for (int j = 0; j < parts; ++j) sum += part[j * g.T * g.E + p];
    v[p] = sum;
  }
}

// A logit as an integer of the same order; a NaN counts as the smallest.
RLA_DEVFN long long moe_key(double v) {  // (never -0: sums start from +0)
  const long long b = __double_as_longlong(v);
  return isnan(v) ? LLONG_MIN : b >= 0 ? b : b ^ LLONG_MAX;
}
RLA_DEVFN double moe_logit(long long key) {
  return key == LLONG_MIN ? __longlong_as_double(LLONG_MAX) : __longlong_as_double(key >= 0 ? key : key ^ LLONG_MAX);
}

// Softmax and choice from all ranks' partial logits: a warp a token.  Every
// CTA of the cluster chooses for itself where its warps hold all tokens;
// otherwise (share) each takes every CLUSTER-th token and tells the others.
// top_k rounds of "the largest that is left, the lowest index of equals";
// every round finds an expert, NaN or not.
template <int PER>  // experts of a lane, at least E / 32
RLA_DEVFN void moe_choose_of(const MoeArgs& g, int rank, bool share, const double* mine, MoeRoute& r) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  for (int t = share ? rank + moe::CLUSTER * warp : warp; t < g.T; t += share ? moe::CLUSTER * warps : warps) {
    double part[PER][moe::CLUSTER];
#pragma unroll
    for (int i = 0; i < PER; ++i)
#pragma unroll
      for (int d = 0; d < moe::CLUSTER; ++d)  // (a lane without an expert repeats the last one)
        part[i][d] = rla_ld_dsmem_f64(mine + t * g.E + min(i * 32 + lane, g.E - 1), d);
    long long key[PER];
    uint32_t left = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      double sum = 0;
#pragma unroll
      for (int d = 0; d < moe::CLUSTER; ++d) sum += part[i][d];
      key[i] = moe_key(sum);
      left |= i * 32 + lane < g.E ? 1u << i : 0u;
    }
    int my_id = 0;
    long long my_key = 0;
    double top = 0;
    uint32_t taken = 0;
    for (int j = 0; j < g.top_k; ++j) {
      long long best = LLONG_MIN;
      unsigned at = 0xffffffffu;  // none left in this lane
#pragma unroll
      for (int i = PER - 1; i >= 0; --i)
        if ((left & ~taken) >> i & 1 && key[i] >= best) best = key[i], at = i * 32 + lane;
      const int hi = static_cast<int>(best >> 32);
      const int hi_max = __reduce_max_sync(0xffffffffu, hi);
      const unsigned lo = hi == hi_max ? static_cast<unsigned>(best) : 0u;
      const unsigned lo_max = __reduce_max_sync(0xffffffffu, lo);
      const unsigned e = __reduce_min_sync(0xffffffffu, hi == hi_max && lo == lo_max ? at : 0xffffffffu);
      if (lane == (e & 31)) taken |= 1u << (e >> 5);
      const long long k = static_cast<long long>(static_cast<unsigned long long>(static_cast<unsigned>(hi_max)) << 32 | lo_max);
      if (j == 0) top = moe_logit(k);
      if (lane == j) my_id = static_cast<int>(e), my_key = k;
    }
    // softmax relative to the largest; a NaN logit makes the sum NaN.  (The
    // intrinsics are a few ulp off; code that runs once is fetched from a busy
    // L2, so it is kept short.)
    float total = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (left >> i & 1) total += __expf(static_cast<float>(moe_logit(key[i]) - top));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    const float p = lane < g.top_k ? __fdividef(__expf(static_cast<float>(moe_logit(my_key) - top)), total) : 0.f;
    float chosen = p;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) chosen += __shfl_xor_sync(0xffffffffu, chosen, o);
    if (lane < g.top_k) {
      const int at = t * g.top_k + lane;
      const float coef = g.renorm ? __fdividef(p, chosen) : p;
      for (int d = share ? 0 : rank; d < (share ? moe::CLUSTER : rank + 1); ++d) {
        rla_st_dsmem_u32(&r.ids[at], d, static_cast<uint32_t>(my_id));
        rla_st_dsmem_u32(&r.coef[at], d, __float_as_uint(coef));
        rla_or_dsmem_u32(&r.mask[my_id], d, 1u << t);
      }
    }
  }
}
RLA_DEVFN void moe_choose(const MoeArgs& g, int rank, bool share, const double* mine, MoeRoute& r) {
  if (g.E <= 32)
    moe_choose_of<1>(g, rank, share, mine, r);
  else if (g.E <= 64)
    moe_choose_of<2>(g, rank, share, mine, r);
  else if (g.E <= 128)
    moe_choose_of<4>(g, rank, share, mine, r);
  else
    moe_choose_of<8>(g, rank, share, mine, r);
}

// A unit of the gate/up kernel: 16 gate rows and the same 16 up rows of one
// expert; a lane holds gate and up of the rows moe_row(lane / 4) and 8 + that.
struct MoeUnitScales {
  float gate[2], up[2];
  RLA_DEVFN void load(const MoeArgs& g, int e, int group, int lane) {
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      const int64_t channel = (int64_t)e * g.I + group * 16 + m * 8 + moe_row(lane >> 2);
      gate[m] = moe_scale(g.s_gate, g.scale_f32, channel);
      up[m] = moe_scale(g.s_up, g.scale_f32, channel);
    }
  }
};
template <int NTM>
RLA_DEVFN void moe_finish_unit(const MoeArgs& g, const MoeRoute& r, int e, int group, const float (&acc)[2][NTM][4],
                               const MoeUnitScales& sc, int lane) {
  const int q = lane & 3;
  const int first = r.begin[e], count = __popc(r.mask[e]);
#pragma unroll
  for (int t = 0; t < NTM; ++t) {
    if (t * 8 >= count) break;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int col = t * 8 + 2 * q + j;
      if (col < count) {
        __nv_bfloat16* to = g.a + (int64_t)r.entry[first + col] * 2 * g.I + group * 16 + moe_place(moe_row(lane >> 2));
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          const float gate = acc[m][t][j] * sc.gate[m], up = acc[m][t][2 + j] * sc.up[m];
          moe_split(rla_silu_mul(gate, up), to[m * 8], to[g.I + m * 8]);
        }
      }
    }
  }
}

template <int NT>  // tiles of 8 tokens
__global__ void __cluster_dims__(moe::CLUSTER, 1, 1) __launch_bounds__(32 * moe::warps(NT), 1)
    moe_gate_up_kernel(const __grid_constant__ CUtensorMap gate_map, const __grid_constant__ CUtensorMap up_map,
                       const MoeArgs g, int stages) {
  constexpr int WARPS = moe::warps(NT);
  extern __shared__ uint8_t moe_smem[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(moe_smem) + 1023) & ~uintptr_t(1023));
  MoeShared& sm = *reinterpret_cast<MoeShared*>(smem);
  MoeRoute& r = sm.r;
  float* heads = reinterpret_cast<float*>(smem + moe_sums_offset());
  uint8_t* rings = smem + moe_ring_offset(g.T);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rank = static_cast<int>(rla_cluster_ctarank());

  MoeRing ring(rings, sm, warp, lane, stages);
  if (threadIdx.x == 0) {
    r.abort_flag = 0;
    rla_tma_prefetch_desc(&gate_map);
    rla_tma_prefetch_desc(&up_map);
  }
  static_assert(32 * WARPS >= moe::MAX_E, "one thread an expert");
  if (threadIdx.x < moe::MAX_E) r.mask[threadIdx.x] = 0;
  rla_fence_barrier_init();
  rla_griddep_launch_dependents();
  {  // this CTA's part of the router into L2 while the previous kernel finishes
    const int64_t lines = ((int64_t)g.E * g.H * 2 + 127) / 128;
    const char* p = reinterpret_cast<const char*>(g.router);
    for (int64_t i = rank * 32 * WARPS + threadIdx.x; i < lines; i += moe::CLUSTER * 32 * WARPS)
      rla_prefetch_l2(p + i * 128);
  }
  rla_griddep_wait();

  // routing; its scratch lies in the ring, which is not in use yet
  static_assert(moe_logit_most(8 * NT, WARPS) <= WARPS * 2 * moe::SLOT, "routing scratch fits the ring");
  double* logits = reinterpret_cast<double*>(rings);
  moe_logits<NT>(g, rank, logits);
  rla_cluster_sync();
  const bool share = g.T > WARPS;
  moe_choose(g, rank, share, logits, r);
  rla_cluster_arrive();  // this CTA has read the others' logits (and told them its choices) ...
  if (share) rla_cluster_wait();
  moe_build_lists(r, g.T, g.E, g.top_k);
  if (!share) rla_cluster_wait();  // ... and the others this one's: the ring is free
  rla_fence_proxy_async();  // plain accesses to the ring come before the copies into it

  // This CTA's units, and of their stages this warp's run.
  const int groups = g.I / 16;
  const int per = (g.H + moe::KB - 1) / moe::KB;  // stages of a unit
  const int units = r.num_active * groups;
  const int u0 = moe_part(units, blockIdx.x, gridDim.x);
  const int items = (moe_part(units, blockIdx.x + 1, gridDim.x) - u0) * per;
  const int i0 = moe_part(items, warp, WARPS);
  int left = moe_part(items, warp + 1, WARPS) - i0;
  const int unit = u0 + i0 / per;
  int ca = unit / groups, cg = unit % groups, cs = i0 % per;  // the products' place

  int pa = ca, pg = cg, ps = cs, to_put = left;  // the copies' place
  int prow = to_put > 0 ? r.active[pa] * g.I + pg * 16 : 0;
  auto put = [&]() {
    if (to_put == 0) return;
    --to_put;
    ring.issue<2>(&gate_map, &up_map, ps * moe::KB, prow, lane);
    if (++ps == per) {
      ps = 0;
      prow += 16;
      if (++pg == groups) {
        pg = 0, ++pa;
        if (to_put > 0) prow = r.active[pa] * g.I;
      }
    }
  };
  for (int i = 0; i < stages; ++i) put();
  if (blockIdx.x == 0) {  // for the second kernel
    const uint4* from = reinterpret_cast<const uint4*>(static_cast<MoeTables*>(&r));
    uint4* to = reinterpret_cast<uint4*>(g.tables);
    for (int i = threadIdx.x; i < (int)(sizeof(MoeTables) / 16); i += 32 * WARPS) to[i] = from[i];
  }

  bool head = left > 0 && cs != 0;  // the current unit began in an earlier warp
  bool tail = false, ok = true;
  MoeAcc<NT> acc;
  MoeUnitScales scales;
  moe_zero(acc);
  // One place finishes all units: code that a warp meets for the first time is
  // fetched from an L2 that is busy with weights.
  for (bool last = false; !last;) {
    bool whole = false;
    if (left > 0) {
      const int e = r.active[ca], first = r.begin[e];
      const int n = min(per - cs, left);
      scales.load(g, e, cg, lane);  // (read before the products, used after them)
      ok = moe_run<1, false, 1024, moe::SLOT / 2>(acc, ring, n, cs * moe::KB, g.H, 0, __popc(r.mask[e]), lane,
                                                  &r.abort_flag, nullptr, [&](int i) {
                                                    return reinterpret_cast<const uint16_t*>(g.x + r.token[first + i] * g.ldx);
                                                  }, put);
      left = ok ? left - n : 0;
      cs += n;
      if (!ok) {
        ring.drain();
      } else if (head) {
        float* h = heads + warp * NT * 256 + lane;
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) h[((m * NT + t) * 4 + j) * 32] = acc[m][t][j];
        head = false;
      } else {
        whole = cs == per;
        tail = !whole;  // goes on in the next warps
      }
    }
    last = left == 0;
    if (last) {
      __syncthreads();  // all heads are there
      if (tail) {
        const int end = (ca * groups + cg - u0 + 1) * per;  // the unit's last stage + 1
        for (int w = warp + 1; w < WARPS; ++w) {
          const int w0 = moe_part(items, w, WARPS), w1 = moe_part(items, w + 1, WARPS);
          if (w0 >= end) break;
          if (w0 == w1) continue;
          const float* h = heads + w * NT * 256 + lane;
#pragma unroll
          for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
              for (int j = 0; j < 4; ++j) acc[m][t][j] += h[((m * NT + t) * 4 + j) * 32];
        }
        whole = true;
      }
    }
    if (whole) moe_finish_unit(g, r, r.active[ca], cg, acc, scales, lane);
    if (cs == per) {
      cs = 0;
      if (++cg == groups) cg = 0, ++ca;
    }
    moe_zero(acc);
  }
}

// Blocks of 32 output rows; of a block's (active expert, stage) list each
// warp of each of the `splits` CTAs of the cluster takes an equal run, and
// adds each expert's part (x channel scale x token coefficient) to its sums
// [T][32] in shared memory.  (Rows behind H in the last block belong to the
// next expert, or are zeros; their sums are not stored.)
template <int NT>  // tiles of 8 tokens
__global__ void __launch_bounds__(32 * moe::warps(NT), 1)
    moe_down_kernel(const __grid_constant__ CUtensorMap down_map, const MoeArgs g, int stages) {
  constexpr int WARPS = moe::warps(NT);
  extern __shared__ uint8_t moe_smem[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(moe_smem) + 1023) & ~uintptr_t(1023));
  MoeShared& sm = *reinterpret_cast<MoeShared*>(smem);
  MoeRoute& r = sm.r;
  float* sums = reinterpret_cast<float*>(smem + moe_sums_offset());
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int gr = moe_row(lane >> 2), q = lane & 3;
  const int splits = gridDim.y, split = blockIdx.y;  // == cluster rank

  MoeRing ring(smem + moe_ring_offset(g.T), sm, warp, lane, stages);
  if (threadIdx.x == 0) {
    r.abort_flag = 0;
    rla_tma_prefetch_desc(&down_map);
  }
  rla_fence_barrier_init();
  rla_griddep_launch_dependents();
  rla_griddep_wait();
  {
    const uint4* from = reinterpret_cast<const uint4*>(g.tables);
    uint4* to = reinterpret_cast<uint4*>(static_cast<MoeTables*>(&r));
#pragma unroll
    for (int i = 0; i < (int)(sizeof(MoeTables) / 16); i += 32 * WARPS)
      if (i + threadIdx.x < sizeof(MoeTables) / 16) to[i + threadIdx.x] = __ldcg(from + i + threadIdx.x);
  }
  __syncthreads();

  const int blocks = (g.H + moe::ROWS - 1) / moe::ROWS;
  const int per = (g.I + moe::KB - 1) / moe::KB;
  const int items = r.num_active * per;
  const int parts = splits * WARPS, mine = split * WARPS + warp;
  const int i0 = moe_part(items, mine, parts), n = moe_part(items, mine + 1, parts) - i0;
  const int a0 = i0 / per, s0 = i0 - a0 * per;

  // the copies run through all blocks of this CTA without a break
  int pb = blockIdx.x, pa = a0, ps = s0, pi = 0;
  auto put = [&]() {
    if (n == 0 || pb >= blocks) return;
    ring.issue<1>(&down_map, nullptr, ps * moe::KB, r.active[pa] * g.H + pb * moe::ROWS, lane);
    if (++ps == per) ps = 0, ++pa;
    if (++pi == n) pi = 0, pa = a0, ps = s0, pb += gridDim.x;
  };
  for (int i = 0; i < stages; ++i) put();

  bool ok = true;
  const int values = g.T * moe::ROWS;
  float* own = sums + warp * values;
  const uint16_t* a = reinterpret_cast<const uint16_t*>(g.a);  // (at most 2^28 elements: 32-bit indices)
  for (int b = blockIdx.x; b < blocks; b += gridDim.x) {
    for (int p = lane; p < values; p += 32) own[p] = 0.f;
    int ca = a0, cs = s0, left = n;
    while (left > 0 && ok) {
      const int e = r.active[ca], first = r.begin[e], count = __popc(r.mask[e]);
      const int m = min(per - cs, left);
      float scale[2][2];  // (read before the products, used after them)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        scale[i >> 1][i & 1] =
            moe_scale(g.s_down, g.scale_f32, (int64_t)e * g.H + min(b * moe::ROWS + gr + i * 8, g.H - 1));
      MoeAcc<NT> acc;
      moe_zero(acc);
      // up to 4 tokens: columns 2 i and 2 i + 1 are the terms of entry i
      const bool paired = count <= 4;
      if (paired)
        ok = moe_run_tiles<1, 1, true, 2048, 1024>(
            acc, ring, m, cs * moe::KB, g.I, 0, 2 * count, lane, &r.abort_flag, a,
            [&](int i) { return (r.entry[first + (i >> 1)] * 2 + (i & 1)) * g.I; }, put);
      else
        ok = moe_run<2, true, 2048, 1024>(acc, ring, m, cs * moe::KB, g.I, g.I, count, lane, &r.abort_flag, a,
                                          [&](int i) { return r.entry[first + i] * 2 * g.I; }, put);
      if (!ok) break;
      if (paired) {  // both terms into the column of the lane's first
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i >> 1][0][2 * (i & 1)] += acc[i >> 1][0][2 * (i & 1) + 1];
      }
      __syncwarp();  // the zeros, or another expert's sums, are in place
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        if (t * 8 >= count) break;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          if (j == 1 && paired) break;
          const int col = paired ? q : t * 8 + 2 * q + j;
          if (col < count) {
            const float c = r.coef[r.entry[first + col]];
            float* v = own + r.token[first + col] * moe::ROWS + gr;
#pragma unroll
            for (int i = 0; i < 4; ++i)
              v[i * 8] = fmaf(acc[i >> 1][t][2 * (i & 1) + j] * scale[i >> 1][i & 1], c, v[i * 8]);
          }
        }
      }
      left -= m;
      cs = 0, ++ca;
    }
    __syncthreads();
    // the CTA's sum into warp 0's (each thread its own values), then the ranks'
    for (int p = threadIdx.x; p < values; p += 32 * WARPS) {
      float v = sums[p];
#pragma unroll
      for (int w = 1; w < WARPS; ++w) v += sums[w * values + p];
      sums[p] = v;
    }
    if (splits > 1) rla_cluster_sync();
    if (split == 0) {
      for (int p = threadIdx.x; p < values; p += 32 * WARPS) {
        float v = sums[p];
        for (int c = 1; c < splits; ++c) v += rla_ld_dsmem_f32(&sums[p], c);
        const int row = b * moe::ROWS + p % moe::ROWS;
        if (row < g.H) g.y[(int64_t)(p / moe::ROWS) * g.ldy + row] = __float2half_rn(v);
      }
    }
    if (splits > 1)
      rla_cluster_sync();  // no CTA goes on while rank 0 may still read it
    else
      __syncthreads();
  }
  if (!ok) ring.drain();
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
// Clusters of the gate/up kernel that run at once: its grid.  Per device.
template <int NT>
static int moe_up_clusters(size_t smem) {
  static std::atomic<int> cache[64];
  int dev = -1;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) dev = -1;
  if (dev >= 0) {
    const int c = cache[dev].load(std::memory_order_relaxed);
    if (c > 0) return c;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(moe::CLUSTER);
  cfg.blockDim = dim3(32 * moe::warps(NT));
  cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = moe::CLUSTER;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int n = 0;
  if (cudaOccupancyMaxActiveClusters(&n, moe_gate_up_kernel<NT>, &cfg) != cudaSuccess || n < 1) {
    (void)cudaGetLastError();
    return std::max(1, device_sm_count() / moe::CLUSTER);
  }
  if (dev >= 0) cache[dev].store(n, std::memory_order_relaxed);
  return n;
}

template <int NT>
static cudaError_t launch_moe(const MoeArgs& g, cudaStream_t s) {
  CUtensorMap gate_map, up_map, down_map;
  const uint64_t E = g.E, H = g.H, I = g.I;
  if (!make_tmap_2d(&gate_map, CU_TENSOR_MAP_DATA_TYPE_UINT8, g.w_gate, H, E * I, H, 128, 16, CU_TENSOR_MAP_SWIZZLE_128B) ||
      !make_tmap_2d(&up_map, CU_TENSOR_MAP_DATA_TYPE_UINT8, g.w_up, H, E * I, H, 128, 16, CU_TENSOR_MAP_SWIZZLE_128B) ||
      !make_tmap_2d(&down_map, CU_TENSOR_MAP_DATA_TYPE_UINT8, g.w_down, I, E * H, I, 128, 32, CU_TENSOR_MAP_SWIZZLE_128B))
    return cudaErrorInvalidValue;
  const int sms = device_sm_count();
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(32 * moe::warps(NT));
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;

  int stages = moe::MAX_STAGES;  // 3 up to 8 tokens and above 16, 2 between
  while (moe_smem_bytes(g.T, stages) > moe::SMEM) --stages;
  cfg.dynamicSmemBytes = moe_smem_bytes(g.T, stages);
  static std::atomic<uint64_t> up_done{0}, down_done{0};
  cudaError_t e = allow_smem(moe_gate_up_kernel<NT>, (int)moe::SMEM, up_done);
  if (e != cudaSuccess) return e;
  const int64_t most = (int64_t)std::min(g.E, g.T * g.top_k) * (g.I / 16);  // units, at most
  const int64_t clusters = std::min<int64_t>(moe_up_clusters<NT>(cfg.dynamicSmemBytes),
                                             (most + moe::CLUSTER - 1) / moe::CLUSTER);
  cfg.gridDim = dim3((unsigned)(clusters * moe::CLUSTER));
  e = cudaLaunchKernelEx(&cfg, moe_gate_up_kernel<NT>, gate_map, up_map, g, stages);
  if (e != cudaSuccess) return e;

  e = allow_smem(moe_down_kernel<NT>, (int)moe::SMEM, down_done);
  if (e != cudaSuccess) return e;
  const int blocks = (g.H + moe::ROWS - 1) / moe::ROWS;
  const int splits = std::max(1, std::min(moe::MAX_SPLITS, sms / blocks));
  cfg.gridDim = dim3(splits > 1 ? blocks : std::min(blocks, sms), splits);
  if (splits > 1) {
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = 1;
    attr[1].val.clusterDim.y = static_cast<unsigned>(splits);
    attr[1].val.clusterDim.z = 1;
    cfg.numAttrs = 2;
  }
  return cudaLaunchKernelEx(&cfg, moe_down_kernel<NT>, down_map, g, stages);
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
  return rla::moe_up256(n * (size_t)I * 4) + rla::moe_up256(sizeof(rla::MoeTables));
}

int rla_moe(const void* x, int64_t ldx, const void* router, const int8_t* w_gate, const void* scale_gate,
            const int8_t* w_up, const void* scale_up, const int8_t* w_down, const void* scale_down, int scale_dtype,
            int renormalize, void* y, int64_t ldy, int64_t T, int64_t H, int64_t I, int64_t E, int64_t top_k,
            void* workspace, size_t workspace_bytes, void* stream) {
  using namespace rla;
  static_assert(moe::MAX_T == RLA_MOE_MAX_TOKENS && moe::MAX_E == RLA_MOE_MAX_EXPERTS && moe::MAX_K == RLA_MOE_MAX_TOP_K,
                "limits of the header");
  if (T < 0 || H < 1 || I < 1 || E < 1 || H > (1 << 17) || I > (1 << 17))
    return moe_fail(RLA_ERR_INVALID_ARGUMENT, "T must be >= 0, H and I in [1, 2^17], E >= 1");
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
  const size_t a_bytes = moe_up256(n * (size_t)I * 4);
  const MoeArgs g{static_cast<const __half*>(x), ldx, static_cast<const __half*>(router), w_gate, w_up, w_down,
                  scale_gate, scale_up, scale_down, scale_dtype == RLA_DTYPE_F32 ? 1 : 0, static_cast<__half*>(y), ldy,
                  reinterpret_cast<__nv_bfloat16*>(ws), reinterpret_cast<MoeTables*>(ws + a_bytes), (int)T, (int)H, (int)I, (int)E, (int)top_k,
                  renormalize ? 1 : 0};
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = moe_tiles((int)T) == 1   ? launch_moe<1>(g, s)
                        : moe_tiles((int)T) == 2 ? launch_moe<2>(g, s)
                                                 : launch_moe<4>(g, s);
  if (e != cudaSuccess) {
    set_error("rla_moe: %s", cudaGetErrorString(e));
    return RLA_ERR_CUDA;
  }
  note_launch();
  note_launch();
  return RLA_OK;
}

}  // extern "C"
