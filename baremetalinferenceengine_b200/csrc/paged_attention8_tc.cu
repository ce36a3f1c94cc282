// Tree attention over an 8-bit paged KV cache on the tensor cores (tcgen05 kind::f8f6f4, TMA,
// TMEM), for bf16 queries and head_dim up to 128. Same contract as paged_attention.cu.
//
// Mathematics: the running softmax of paged_attention.cu on tiles of 128 slots, K and V as the
// codes they are held in: nothing is widened on its way to the tensor cores.
//   scores  S[row][slot] = (Qh + Ql)[row][:] . Kc[slot][:]         e4m3 x e4m3 and e5m2 x e4m3
//   mix     O[row][:]   += (P1 + P2 + P3)[row][slot] Vc[slot][:]   three e5m2 x e4m3
// Qh is the query times a power of two that puts its largest element in [128, 256), rounded to
// e4m3, and Ql what that leaves, e5m2: together all 8 bits of a bf16 element down to 2^-13 of the largest, and off by
// 2^-21 of the largest at most below. Scales are powers of two, so they meet the softmax as exponents:
//   t = S f + e_v,  f = 2^(e_k - e_q) scale log2(e),  P = 2^(t - m + 12),  l += P 2^(-e_v)
// with e_k and e_v the exponents of K's and V's scale at the slot, e_q the query's and m the running maximum
// of t: the weight times V's scale is what the mix takes, so its rounding is relative to the
// largest term of the sum, however far blocks' scales lie apart. P is at most 2^15 (a row is rescaled when m rises by
// more than 3). Its fp16 value has 11 bits, of which each e5m2 part takes three, the first two a bit more by the next
// one's sign: together all 11, down to steps of 2^-16, the smallest that e5m2 has. So a weight is off by 2^-11 of itself at
// most, or by 2^-17 of 2^12 where it is small, which 2^17 slots cannot add up to 2^-11 of the sum. (Two parts do not hold
// that: e5m2 and e4m3 leave 2^-10, which for thousands of small weights next to a large one came to 7 % of the sum of
// weights times |v|.)
//
// Bound: memory while group * tokens is below about 100 (a slot is half the bytes of a bf16 cache's, for the same
// tensor time), above it the products. What it takes is neither: it is the chain scores, softmax, weights, mix of each
// row tile, whose waits two groups of warps leave open (counters of 64 tokens at group 8: tensor pipe 24 % of its
// cycles, conversions and exponentials 20 %, issue slots 38 %), and for few rows the ends of segments.
// Measured, heads of 128, 8 kv heads: 1 sequence, 12 tokens at group 4 over 8000 slots 25 us; 64 ragged sequences of up
// to 8192 slots, 8 tokens at group 4 188 to 193 us (2.7 TB/s of codes); 16 sequences of 4096 to 8192 slots, 64 tokens at group 8
// 369 to 374 us (540 TFLOP/s of the formula's products). With weights of two parts 24, 171 and 337.
//
// Split and roles are paged_attention_tc.cu's, but for the queries, the scales and the MMAs. The warp that fetches V
// converts a segment's queries into two operands in shared memory, some rows between two tiles, while the segment before
// is computed (all warps but those of TMA together for a CTA's first, which all wait for). The warp that fetches K
// looks up the scales of its tile's slots, eight neighbouring ones of which share one. With two row tiles each softmax
// group has an MMA issuer of its own (warps 1 and 2), else one has both.
#include <cuda.h>

#include "kv8.cuh"
#include "paged_attention_tc.cuh"

namespace bm {
namespace paged {
namespace {

constexpr float kRescaleAt8 = 3.f;  // rise of the maximum (log2) that a row's sums are rescaled at (4 and 6: no faster; 2: 4 % slower)
constexpr float kLift = 12.f;       // P is 2^12 at the running maximum, so at most 2^15: e5m2 ends at 1.75 * 2^15
constexpr int kGroupSlots = 8;      // slots of a tile that share a scale
constexpr int kGroups = kTile / kGroupSlots;
// What beginning and ending an item costs a CTA, in tiles. 0, 1, 2, 4, 6, 8 take, us: the cases above 36, 27, 26, 26, 26,
// 26; 227, 198, 191, 173, 166, 171; 383, 384, 370, 362, 358, 357; the same with heads of 64 33, 23, 23, 23, 23, 23; 214,
// 188, 179, 163, 150, 152; 359, 355, 347, 336, 330, 327; one token for each of 64 sequences 219, 203, 188, 173, 170, 173;
// 32 sequences of 500 to 3000, up to 12 tokens at group 8 150, 140, 131, 126, 115, 112.
constexpr int kItemCost = 6;
constexpr int kConvert = 8;         // pairs of rows of the next queries that are converted between two tiles
constexpr int kQRing = 4;           // segments whose queries' factors are kept
constexpr int kQWarps = 10;         // warps that convert a CTA's first queries: all but the two of TMA

template <int HD, int COPIES>
struct Layout8 : RowLayout<HD, COPIES> {
  using Rows = RowLayout<HD, COPIES>;
  // Scores and mixes are issued for parts of a tile, each with TMEM columns of its own: where rows fill a tile a group
  // weighs one part while the other's mix and the next unit's scores are computed; copies' tiles wait for memory.
  static constexpr int kParts = Rows::kCopies > 1 ? 1 : 2;
  static constexpr int kPart = kTile / kParts;              // slots
  // Warps that issue MMAs: with two row tiles each group has one of its own.
  static constexpr int kIssuers = Rows::kTiles;
  static constexpr int kOperand = kTile * HD;               // a tile of K or V, one part of Q
  static constexpr int kQTile = 2 * kOperand;               // both parts of a row tile
  static constexpr int kQBuf = Rows::kTiles * kQTile;       // of two: a segment's, and the next one's
  static constexpr int kKS = HD == 64 ? 6 : Rows::kTwo ? 2 : 4;                          // K ring: freed by the scores
  static constexpr int kVS = HD == 64 ? 8 : Rows::kTwo ? 3 : Rows::kCopies > 1 ? 4 : 5;  // V ring: freed by the mix
  static constexpr int kOffK = 2 * kQBuf;
  static constexpr int kOffV = kOffK + kKS * kOperand;
  static constexpr int kOffMl = kOffV + kVS * kOperand;
  static constexpr int kOffSum = kOffMl + Rows::kMlBytes;
  static constexpr int kOffScale = kOffSum + Rows::kSumBytes;  // [kBadRing][kGroups] (f of K, e_v, 2^-e_v, -)
  static constexpr int kOffFactor = kOffScale + kBadRing * kGroups * 16;  // [kQRing][rows]
  static constexpr int kOffBar = kOffFactor + kQRing * Rows::kRows * 4;
  static constexpr int kBars = 2 * kKS + 2 * kVS + 12 + 7;
  static constexpr int kOffPlan = kOffBar + kBars * 8;      // Plan, scan, bad-page ring
  static constexpr int kBytes = kOffPlan + 96 + 16 * 8 + kBadRing * 4 + 16 + 1024 /* alignment slack */;
  static_assert(kBytes <= 232448, "shared memory of a CTA");
  // Tiles between the one whose scores are issued next and the one a softmax group may still read.
  static_assert(kKS + 6 <= kBadRing, "rings by tile");
};

// Instruction descriptors for kind::f8f6f4 with an fp32 accumulator: A e4m3 or e5m2, B e4m3.
__host__ __device__ constexpr uint32_t instr_desc_e4m3(bool a_e5m2, bool b_mn_major, int n, int m) {
  return (1u << 4) | ((a_e5m2 ? 1u : 0u) << 7) | ((b_mn_major ? 1u : 0u) << 16) | (static_cast<uint32_t>(n >> 3) << 17) |
         (static_cast<uint32_t>(m >> 4) << 24);
}
// The matrix descriptor of rows of HD bytes, 8-row groups HD * 8 bytes apart, with the swizzle
// of such rows (128 or 64 bytes). Both operands' tiles are one swizzle atom wide.
template <int HD>
__device__ __forceinline__ uint64_t byte_desc(uint32_t addr) {
  return static_cast<uint64_t>((addr >> 4) & 0x3FFFu) | (1ull << 16) | (static_cast<uint64_t>((HD * 8) >> 4) << 32) | (1ull << 46) |
         ((HD == 128 ? 2ull : 4ull) << 61);
}
__device__ __forceinline__ void mma_f8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// A's rows are TMEM lanes, four codes a column.
__device__ __forceinline__ void mma_f8_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// N consecutive 32-bit columns of this thread's TMEM lane.
template <int N>
__device__ __forceinline__ void tmem_load_n(uint32_t taddr, uint32_t (&r)[N]) {
  if constexpr (N == 32) {
    tmem_load32(taddr, r);
  } else {
    static_assert(N == 16, "columns");
    tmem_load16(taddr, r);
  }
}
template <int N>
__device__ __forceinline__ void tmem_store_n(uint32_t taddr, const uint32_t (&r)[N]) {
  if constexpr (N == 16) {
    tmem_store16(taddr, r);
  } else if constexpr (N == 8) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]),
        "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(taddr)
        : "memory");
  } else {
    static_assert(N == 4, "columns");
    asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%4], {%0, %1, %2, %3};" ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(taddr)
                 : "memory");
  }
}
// The phase's bytes to come, without an arrival.
__device__ __forceinline__ void mbar_expect_only(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive_n(uint64_t* bar, uint32_t count) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(count) : "memory");
}

// Two values as e5m2 (lo in the low byte), as kv8::to_codes makes e4m3.
__device__ __forceinline__ uint32_t e5m2x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
// Four weights' fp16 values as three e5m2 parts: the upper byte of an fp16 value, rounded, is its e5m2 value, so each part
// is taken off what the last one leaves. Weights are not negative. (Of a NaN the parts are zeros; its row's sum
// is one.)
__device__ __forceinline__ void weight_parts(float p0, float p1, float p2, float p3, uint32_t* first, uint32_t* second, uint32_t* third) {
  uint32_t a, b;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(a) : "f"(p1), "f"(p0));
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(b) : "f"(p3), "f"(p2));
  auto part = [&](uint32_t* to) {
    const uint32_t ha = a + 0x00800080u, hb = b + 0x00800080u;
    *to = __byte_perm(ha, hb, 0x7531);
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(a) : "r"(a), "r"(ha & 0xff00ff00u));
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(b) : "r"(b), "r"(hb & 0xff00ff00u));
  };
  part(first);
  part(second);
  part(third);
}

// Converts the queries of an item into its two parts in the buffer at `to`, row tile after row
// tile, copies and all, and their factors scale * log2(e) * 2^-e_q into factor[row]. Warp
// `worker` of `workers` takes every workers-th pair of rows of [from, until), half a warp a row; rows of no
// token are zero.
template <typename L, int HD>
__device__ __forceinline__ void convert_queries(const TreeArgs& a, const Seq& s, int kvh, int p, int tpt, unsigned char* to, float* factor,
                                                int worker, int workers, int from, int until) {
  constexpr int kBatch = 4;  // pairs of rows that are converted side by side
  const int lane = threadIdx.x & 31, half = lane >> 4, c = lane & 15;
  const int i_first = p * tpt * L::kTiles;
  const uint32_t by_group = (65536u + a.group - 1) / a.group;  // r / group = r * by_group >> 16 for r < 128
  const bf16* q = static_cast<const bf16*>(a.q) + (s.row0 * a.hq + static_cast<int64_t>(kvh) * a.group) * a.hd + c * 8;
  const int64_t token_step = static_cast<int64_t>(a.hq) * a.hd;
  for (int pair0 = from + worker; pair0 < until; pair0 += workers * kBatch) {
    uint4 raw[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int row = 2 * (pair0 + k * workers) + half, r = row % L::kCopyRows;
      const int token = static_cast<int>(r * by_group >> 16), i = i_first + row / L::kCopyRows * tpt + token;
      raw[k] = make_uint4(0u, 0u, 0u, 0u);
      if (row < 2 * until && token < tpt && i < s.n && c * 8 < a.hd) raw[k] = ld_keep(q + i * token_step + (r - token * a.group) * a.hd);
    }
    uint32_t top[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      // the larger of two neighbours' magnitudes, as bf16 in either half of a word
      const uint32_t m01 = __vmaxu2(raw[k].x & 0x7fff7fffu, raw[k].y & 0x7fff7fffu), m23 = __vmaxu2(raw[k].z & 0x7fff7fffu, raw[k].w & 0x7fff7fffu);
      const uint32_t m = __vmaxu2(m01, m23);
      top[k] = max(m & 0xffffu, m >> 16);
    }
#pragma unroll
    for (int off = 8; off > 0; off >>= 1) {
#pragma unroll
      for (int k = 0; k < kBatch; ++k) top[k] = max(top[k], __shfl_xor_sync(0xffffffffu, top[k], off));
    }
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int row = 2 * (pair0 + k * workers) + half, r = row % L::kCopyRows;
      if (row >= 2 * until) continue;
      const int e = min(max(static_cast<int>(top[k] >> 7) - 127, -60), 127);
      const float f = kv8::power(7 - e);
      if (c * 8 < HD) {
        float x[8];
        unpack16<bf16>(raw[k], x);
        uint32_t hi[2], lo[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float back[4];
          hi[j] = kv8::to_codes(x[4 * j] * f, x[4 * j + 1] * f) | kv8::to_codes(x[4 * j + 2] * f, x[4 * j + 3] * f) << 16;
          kv8::from_codes(hi[j], back);
#pragma unroll
          for (int d = 0; d < 4; ++d) back[d] = fmaf(x[4 * j + d], f, -back[d]);
          lo[j] = e5m2x2(back[0], back[1]) | e5m2x2(back[2], back[3]) << 16;
        }
#pragma unroll
        for (int copy = 0; copy < L::kCopies; ++copy) {
          const int at = copy * L::kCopyRows + r;
          const int chunk = (c >> 1) ^ (HD == 128 ? at & 7 : (at >> 1) & 3);  // the swizzle of 16-byte chunks
          unsigned char* dst = to + row / L::kCopyRows * L::kQTile + at * HD + chunk * 16 + (c & 1) * 8;
          *reinterpret_cast<uint2*>(dst) = make_uint2(hi[0], hi[1]);
          *reinterpret_cast<uint2*>(dst + L::kOperand) = make_uint2(lo[0], lo[1]);
        }
      }
      // a query that is not finite spoils its row
      if (c == 0) factor[row] = top[k] >= 0x7f80u ? __int_as_float(0x7fffffff) : a.qscale * kv8::power(e - 7);
    }
  }
  fence_proxy_async_smem();
  __syncwarp();
}

template <int HD, int COPIES>
__global__ void __launch_bounds__(kThreadsTc, 1)
    tree_tc8_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv, const TreeArgs a) {
  grid_dependency_wait();
  using L = Layout8<HD, COPIES>;
  constexpr bool DUAL = L::kTwo;
  constexpr uint32_t kIdescH = instr_desc_e4m3(false, false, L::kPart, kTile);
  constexpr uint32_t kIdescL = instr_desc_e4m3(true, false, L::kPart, kTile);
  constexpr uint32_t kIdescO = instr_desc_e4m3(true, true, HD, kTile);
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                                         ~static_cast<uintptr_t>(1023));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int cta = static_cast<int>(blockIdx.x);
  const int tpt = L::kCopyRows / a.group;  // tokens of a row tile
  const int per = tpt * L::kTiles;         // and of an item

  uint64_t* kfull = reinterpret_cast<uint64_t*>(smem + L::kOffBar);  // K, and its tile's scales
  uint64_t* kempty = kfull + L::kKS;
  uint64_t* vfull = kempty + L::kKS;
  uint64_t* vempty = vfull + L::kVS;
  // of group w's part h of a unit, at kParts w + h:
  uint64_t* sfull = vempty + L::kVS;    // scores in TMEM       (commit)
  uint64_t* pfull = sfull + 4;          // weights in TMEM      (one arrival per warp of the group)
  uint64_t* pvdone = pfull + 4;         // mix done             (commit)
  uint64_t* qfull = pvdone + 4;         // queries converted    (kQWarps arrivals)
  uint64_t* qempty = qfull + 2;         // the segment's last scores are done (a commit of each issuer)
  uint64_t* ofree = qempty + 2;         // the segment's O has been read (one arrival per softmax warp)
  uint64_t* mma_done = ofree + 1;      // of each issuer
  Plan* plan = reinterpret_cast<Plan*>(smem + L::kOffPlan);
  int64_t* scan = reinterpret_cast<int64_t*>(smem + L::kOffPlan + 96);
  volatile uint32_t* bad_ring = reinterpret_cast<volatile uint32_t*>(scan + 16);
  uint32_t* tmem_base_s = const_cast<uint32_t*>(bad_ring) + kBadRing;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_base_s + 1);
  float4* scales = reinterpret_cast<float4*>(smem + L::kOffScale);
  float* factors = reinterpret_cast<float*>(smem + L::kOffFactor);
  Record* records = reinterpret_cast<Record*>(a.ws);
  float* slots = a.ws + records_bytes(gridDim.x) / sizeof(float);

  // ---------------- the plan ----------------
  int64_t plan_total;
  int plan_nc;
  {
    // barriers and TMEM come up while the lengths are read
    if (tid == 0) {
      for (int i = 0; i < L::kKS; ++i) {
        mbar_init(&kfull[i], 1);
        mbar_init(&kempty[i], L::kTiles);  // read for each row tile
      }
      for (int i = 0; i < L::kVS; ++i) {
        mbar_init(&vfull[i], 1);
        mbar_init(&vempty[i], L::kTiles);
      }
      for (int i = 0; i < 4; ++i) {
        mbar_init(&sfull[i], 1);
        mbar_init(&pfull[i], 4);
        mbar_init(&pvdone[i], 1);
      }
      for (int i = 0; i < 2; ++i) {
        mbar_init(&qfull[i], kQWarps);
        mbar_init(&qempty[i], L::kIssuers);
        mbar_init(&mma_done[i], 1);
      }
      mbar_init(ofree, 8);
      *abort_flag = 0;
      fence_barrier_init();
    }
    if (warp == 1) tmem_alloc(tmem_base_s, L::kTmemCols);
    if (a.tile < kTile) {  // V rows that no copy ever fills: zero, since their weights of 0 meet them
      const int rows = kTile - a.tile;
      for (int c = tid; c < L::kVS * rows * (HD / 16); c += kThreadsTc) {
        const int row = a.tile + c / (HD / 16) % rows, stage = c / (HD / 16) / rows;
        *reinterpret_cast<uint4*>(smem + L::kOffV + stage * L::kOperand + row * HD + c % (HD / 16) * 16) = make_uint4(0u, 0u, 0u, 0u);
      }
      fence_proxy_async_smem();
    }
    if (!plan_share(a, per, scan, plan, records, &plan_total, &plan_nc)) {
      if (warp == 1) tmem_dealloc(*tmem_base_s, L::kTmemCols);
      return;
    }
  }
  const uint32_t tmem = *tmem_base_s;
  Walk walk;
  walk.start(a, plan->s, plan->b, plan->off, plan->hi - plan->lo, per);
  if (tid == 0) {
    records[cta] = Record{plan->lo, plan_total, static_cast<int32_t>(walk.b), walk.kvh, walk.p, walk.t, walk.tiles, plan_nc};
  }
  if (warp != 0 && warp != 3) {
    const int worker = warp < 3 ? warp - 1 : warp - 2;
    convert_queries<L, HD>(a, walk.s, walk.kvh, walk.p, tpt, smem, factors, worker, kQWarps, 0, L::kRows / 2);
    if (lane == 0) mbar_arrive(&qfull[0]);
    __syncwarp();
  }

  if (warp == 0 || warp == 3) {
    // ---------------- K with the scales (warp 0), V and the next segment's queries (warp 3) ----------------
    // Lanes 0 to 15 each fetch a box of the tile; warp 0's others look up the scales of eight slots
    // each, one step ahead, and their pages two.
    const bool is_v = warp == 3;
    const CUtensorMap* map = is_v ? &tv : &tk;
    uint64_t* full = is_v ? vfull : kfull;
    uint64_t* empty = is_v ? vempty : kempty;
    unsigned char* ring = smem + (is_v ? L::kOffV : L::kOffK);
    const int stages = is_v ? L::kVS : L::kKS;
    const int boxes = a.tile / a.box;    // of a tile: at most 16
    const bool scaler = !is_v && lane >= 16;
    const int first_slot = lane < 16 ? lane * a.box : (lane - 16) * kGroupSlots;  // of this lane in a tile
    int kt = 0, stage = 0;               // tiles asked for; the next one's ring slot
    uint32_t phase = 1;
    bool ok = true;
    for (int seg = 0; ok && walk.left > 0; walk.next(a, per), ++seg) {
      const int n = walk.segment();
      const int32_t* pages = a.page_table + static_cast<int64_t>(walk.s.seq) * a.max_pages;
      const int total = walk.s.ctx + walk.s.n, t0 = walk.t, kvh = walk.kvh;
      const bool mine = lane < 16 ? lane < boxes : scaler && first_slot < a.tile;
      // This lane's slot of tile i of the segment: its row in the tensor map, -1 bad, -2 none.
      auto row_of = [&](int i) {
        const int slot = (t0 + i) * a.tile + first_slot;
        if (!mine || i >= n || slot >= total) return -2;
        const int nth = slot / a.page_size;
        const int32_t page = __ldg(pages + nth);
        if (page < 0 || page >= a.num_pages) return -1;
        return (page * a.hkv + kvh) * a.page_size + (slot - nth * a.page_size);
      };
      // The scales of a row, as bytes; 127 (2^0) where there are none.
      auto scales_of = [&](int row, uint32_t* k, uint32_t* v) {
        *k = *v = 127;
        if (!scaler || row < 0) return;
        const int at = row / a.block;  // blocks divide pages
        *k = __ldg(a.k_scales + at);
        *v = __ldg(a.v_scales + at);
      };
      // the next segment's queries, whose buffer is the segment before's
      Walk ahead = walk;
      if (is_v) ahead.next(a, per);
      const bool converts = is_v && ahead.left > 0;
      int pairs = 0;  // of their rows converted
      int row = row_of(0), row1 = scaler ? row_of(1) : -2;
      uint32_t k, v;
      scales_of(row, &k, &v);
      for (int i = 0; i < n; ++i) {
        // looked up while this tile waits
        const int next = row_of(i + (scaler ? 2 : 1));
        uint32_t k1 = 127, v1 = 127;
        scales_of(row1, &k1, &v1);
        const uint32_t have = __ballot_sync(0xffffffffu, lane < 16 && row >= 0);
        const uint32_t bad = __ballot_sync(0xffffffffu, lane < 16 && row == -1);
        if (!(ok = warp_wait(&empty[stage], phase, abort_flag, a.status))) break;
        if (lane == 0) {
          const uint32_t bytes = __popc(have) * a.box * HD;
          if (is_v) {
            mbar_expect_tx(&full[stage], bytes);
          } else {
            mbar_expect_only(&full[stage], bytes);  // the arrival follows the scales
            bad_ring[kt % kBadRing] = bad;
            if (bad) raise_status(a.status, BM_DEVERR_BAD_PAGE);
          }
        }
        __syncwarp();
        if (lane < 16 && row >= 0) tma_load_2d(ring + stage * L::kOperand + lane * a.box * HD, map, &full[stage], 0, row);
        if (!is_v) {
          if (scaler) {
            const int ev = kv8::exponent(static_cast<uint8_t>(v));
            scales[kt % kBadRing * kGroups + lane - 16] =
                make_float4(kv8::power(kv8::exponent(static_cast<uint8_t>(k))), static_cast<float>(ev), kv8::power(-ev), 0.f);
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&full[stage]);
        }
        ++kt;
        if (++stage == stages) {
          stage = 0;
          phase ^= 1;
        }
        row = scaler ? row1 : next;
        row1 = next;
        k = k1;
        v = v1;
        if (converts) {  // a few rows at a time, so that V's ring stays full
          if (pairs == 0 && !(ok = warp_wait(&qempty[(seg + 1) & 1], (((seg + 1) >> 1) & 1) ^ 1u, abort_flag, a.status))) break;
          const int until = i + 1 < n ? min(pairs + kConvert, L::kRows / 2) : L::kRows / 2;
          if (pairs < until) {
            convert_queries<L, HD>(a, ahead.s, ahead.kvh, ahead.p, tpt, smem + ((seg + 1) & 1) * L::kQBuf,
                                   factors + (seg + 1) % kQRing * L::kRows, 0, 1, pairs, until);
            if (until == L::kRows / 2 && lane == 0) mbar_arrive_n(&qfull[(seg + 1) & 1], kQWarps);
            __syncwarp();
          }
          pairs = until;
        }
      }
    }
    if (lane == 0) {  // copies still in flight land before the CTA ends
      for (int i = max(0, kt - stages); i < kt; ++i) {
        wait_phase(&full[i % stages], (i / stages) & 1, abort_flag, a.status, kDrainNs, false);
      }
    }
    __syncwarp();
  } else if (warp < 1 + L::kIssuers) {
    // ---------------- MMA issuers ----------------
    // Units number through the CTA's segments, group x & 1 has unit x. An issuer has all of them, or with two row tiles
    // those of its group. Either way it passes through every phase of every barrier that it waits for, as a wait by
    // parity asks: a group that a segment of one tile passes by would lose count of the segments' queries and the tiles.
    // Scores go one unit of each group ahead of the mixes. The whole warp walks, one thread issues.
    const uint64_t q_desc = byte_desc<HD>(smem_u32(smem));
    const uint64_t k_desc = byte_desc<HD>(smem_u32(smem + L::kOffK));
    const uint64_t v_desc = byte_desc<HD>(smem_u32(smem + L::kOffV));
    constexpr uint32_t kStage = L::kOperand >> 4, kPartRows = L::kPart * HD >> 4;
    struct Place {
      int x, u, units, seg;  // unit, its number in its segment, units of that, segments before
    };
    const int first = warp - 1;  // of the issuer's units in a segment
    // Moves on to the issuer's next unit; false when there is none.
    auto advance = [&](Place& p, Walk& at) {
      p.x += L::kIssuers;
      p.u += L::kIssuers;
      if (p.u < p.units) return true;
      at.next(a, per);
      if (__shfl_sync(0xffffffffu, at.left > 0 ? 1 : 0, 0) == 0) return false;
      p.units = __shfl_sync(0xffffffffu, at.segment(), 0) * L::kTiles;
      p.u = first;
      ++p.seg;
      return true;
    };
    bool ok = true;
    auto score = [&](const Place& p, int h) {
      const int w = p.x & 1, buf = L::kParts * w + h, kt = p.x / L::kTiles, ks = kt % L::kKS, qbuf = p.seg & 1;
      if (h == 0) {
        if (p.u == first && !(ok = warp_wait(&qfull[qbuf], (p.seg >> 1) & 1, abort_flag, a.status))) return;
        if (!(ok = warp_wait(&kfull[ks], (kt / L::kKS) & 1, abort_flag, a.status))) return;
      }
      // the last weights in these columns have been mixed (before the first: passes)
      if (!(ok = warp_wait(&pvdone[buf], ((p.x >> 1) & 1) ^ 1u, abort_flag, a.status))) return;
      tc_fence_after();
      if (elect_one()) {
        const uint64_t q_at = q_desc + ((qbuf * L::kQBuf + (DUAL ? w * L::kQTile : 0)) >> 4), k_at = k_desc + ks * kStage + h * kPartRows;
#pragma unroll
        for (int kk = 0; kk < HD / 32; ++kk) mma_f8(tmem + buf * L::kPart, q_at + kk * 2, k_at + kk * 2, kIdescH, kk > 0 ? 1u : 0u);
#pragma unroll
        for (int kk = 0; kk < HD / 32; ++kk) mma_f8(tmem + buf * L::kPart, q_at + kStage + kk * 2, k_at + kk * 2, kIdescL, 1u);
        mma_commit(&sfull[buf]);
        if (h == L::kParts - 1) {
          mma_commit(&kempty[ks]);
          if (p.u + L::kIssuers >= p.units) mma_commit(&qempty[qbuf]);
        }
      }
      __syncwarp();
    };
    auto mix = [&](const Place& p, int h) {
      const int w = p.x & 1, buf = L::kParts * w + h, kt = p.x / L::kTiles, vs = kt % L::kVS;
      if (!(ok = warp_wait(&pfull[buf], (p.x >> 1) & 1, abort_flag, a.status))) return;
      if (h == 0) {
        // the segment's first mix overwrites O: its last reader was the previous segment's end
        if (p.u == first && p.seg > 0 && !(ok = warp_wait(ofree, (p.seg - 1) & 1, abort_flag, a.status))) return;
        if (!(ok = warp_wait(&vfull[vs], (kt / L::kVS) & 1, abort_flag, a.status))) return;
      }
      tc_fence_after();
      if (elect_one()) {
        // fresh: the group's first of the segment
        const uint32_t o = tmem + L::kColO + w * HD, at = tmem + buf * L::kPart, fresh = p.u < 2 && h == 0 ? 0u : 1u;
        const uint64_t v_at = v_desc + vs * kStage + h * kPartRows;
        constexpr uint32_t kStep = 32 * HD >> 4;  // 32 slots of V
#pragma unroll
        for (int i = 0; i < 3; ++i) {  // the weights' parts
#pragma unroll
          for (int kk = 0; kk < L::kPart / 32; ++kk) {
            mma_f8_ts(o, at + i * (L::kPart / 4) + kk * 8, v_at + kk * kStep, kIdescO, i > 0 || kk > 0 ? 1u : fresh);
          }
        }
        mma_commit(&pvdone[buf]);
        if (h == L::kParts - 1) mma_commit(&vempty[vs]);
      }
      __syncwarp();
    };
    Place mx{first, first, __shfl_sync(0xffffffffu, walk.segment(), 0) * L::kTiles, 0}, sc = mx;
    Walk mix_walk = walk;
    bool more = true, any = true;
    for (int lead = 0; more && lead < 2; lead += L::kIssuers) {
      for (int h = 0; ok && h < L::kParts; ++h) score(sc, h);
      more = ok && advance(sc, walk);
    }
    while (ok && any) {
      for (int h = 0; ok && h < L::kParts; ++h) {
        mix(mx, h);
        if (ok && more) score(sc, h);
      }
      if (more) more = advance(sc, walk);
      any = advance(mx, mix_walk);
    }
    if (elect_one()) mma_commit(&mma_done[first]);
    __syncwarp();
    if (lane == 0) wait_phase(&mma_done[first], 0, abort_flag, a.status, kDrainNs, false);
    __syncwarp();
  } else if (warp >= 4) {
    // ---------------- softmax ----------------
    constexpr int NC = L::kPart / L::kCopies;  // slots of a part that a copy weighs
    const int w = (warp - 4) >> 2;      // group
    const int quarter = warp & 3;
    const int copy = quarter * 32 / L::kCopyRows;
    const int r = quarter * 32 % L::kCopyRows + lane;  // row of the row tile; lane quarter * 32 + lane of TMEM is its
    const uint32_t lane_addr = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t o_addr = tmem + lane_addr + L::kColO + w * HD;
    int tiles = 0;         // before this segment
    for (int seg = 0; walk.left > 0; walk.next(a, per), ++seg) {
      const int n = walk.segment();
      const int units = n * L::kTiles;
      const Seq s = walk.s;
      const int i0 = walk.p * per + (DUAL ? w * tpt : 0);
      const int live = max(0, min(tpt, s.n - i0)) * a.group;
      const bool warp_live = r - lane < live;
      const int token = i0 + r / a.group;  // a row past `live` computes on zeros and is not stored
      const int total = s.ctx + s.n;
      float m = -INFINITY, l = 0.f, factor = 0.f;
      const int x0 = tiles * L::kTiles, first_u = (x0 ^ w) & 1;  // the segment's first unit; this group's first of them
      for (int u = first_u; u < units; u += 2) {
        const int kt = tiles + (DUAL ? u >> 1 : u);
        const uint32_t parity = (x0 + u) >> 1 & 1;
        const int slot0 = (walk.t + (DUAL ? u >> 1 : u)) * a.tile;
#pragma unroll 1
        for (int h = 0; h < L::kParts; ++h) {
          const int buf = L::kParts * w + h;
          const uint32_t s_addr = tmem + lane_addr + buf * L::kPart;
          warp_wait(&sfull[buf], parity, abort_flag, a.status);
          tc_fence_after();
          const uint32_t bad = bad_ring[kt % kBadRing];
          if (u == first_u && h == 0) factor = factors[seg % kQRing * L::kRows + (DUAL ? w * kTile : 0) + r];
          if (warp_live) {
            const int first = h * L::kPart + copy * NC;  // this copy's first slot of the tile
            const float4* group = scales + kt % kBadRing * kGroups + first / kGroupSlots;
            constexpr int kChunk = NC < 32 ? NC : 32;
            uint32_t v[NC / kChunk][kChunk];
#pragma unroll
            for (int c = 0; c < NC / kChunk; ++c) tmem_load_n<kChunk>(s_addr + copy * NC + kChunk * c, v[c]);
            tmem_wait_ld();
            if (slot0 + a.tile > s.ctx || a.tile < kTile || bad != 0) {
#pragma unroll
              for (int c = 0; c < NC / kChunk; ++c) {
                const int at = first + kChunk * c;
                uint32_t see = r < live ? seen32(a, s, token, slot0 + at) & low_bits(a.tile - at) : 0xffffffffu;
                if (bad) see &= sound32(bad, at, a.box);
                if (kChunk < 32) see |= 0xffffffffu << (kChunk & 31);
                if (__all_sync(0xffffffffu, see == 0xffffffffu)) continue;  // a prompt's chunks are mostly seen
#pragma unroll
                for (int e = 0; e < kChunk; ++e) {
                  if (!((see >> e) & 1)) v[c][e] = 0xff800000u;  // -inf: no weight
                }
              }
              __syncwarp();
            }
            // what a group's scores are multiplied by: never 0, since -inf times it has to stay
            auto times = [&](float k) {
              const float f = k * factor;
              return f < 1.17549435e-38f ? 1.17549435e-38f : f;
            };
            float top = -INFINITY;
#pragma unroll
            for (int c = 0; c < NC / kChunk; ++c) {
#pragma unroll
              for (int j = 0; j < kChunk / 8; ++j) {
                const float4 sc = group[4 * c + j];
                float most = __uint_as_float(v[c][8 * j]);
#pragma unroll
                for (int e = 1; e < 7; e += 2) most = max3(most, __uint_as_float(v[c][8 * j + e]), __uint_as_float(v[c][8 * j + e + 1]));
                most = fmaxf(most, __uint_as_float(v[c][8 * j + 7]));
                top = fmaxf(top, fmaf(most, times(sc.x), sc.y));
              }
            }
            if (r >= live) top = -INFINITY;
            if (factor != factor) top = 0.f;  // a row of NaN stays one through its merges
            const bool rise = top > m + kRescaleAt8 || (m == -INFINITY && top > -INFINITY);
            const float m_new = rise ? top : m;
            const float alpha = rise ? ex2(m - m_new) : 1.f;  // m = -inf: 0
            if ((u != first_u || h > 0) && __any_sync(0xffffffffu, rise)) {
              // the group's previous mix
              const int last = h > 0 ? buf - 1 : buf + L::kParts - 1;
              warp_wait(&pvdone[last], h > 0 ? parity : parity ^ 1, abort_flag, a.status);
              tc_fence_after();
              l *= alpha;
#pragma unroll 1
              for (int c = 0; c < HD / 16; ++c) {
                uint32_t o[16];
                tmem_load16(o_addr + 16 * c, o);
                tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
                tmem_store16(o_addr + 16 * c, o);
              }
            }
            m = m_new;
            const float base = m == -INFINITY ? 0.f : m - kLift;
#pragma unroll
            for (int c = 0; c < NC / kChunk; ++c) {
              uint32_t part[3][kChunk / 4];
#pragma unroll
              for (int j = 0; j < kChunk / 8; ++j) {
                const float4 sc = group[4 * c + j];
                const float f = times(sc.x), up = sc.y - base;
                const uint64_t f2 = pair(f, f), up2 = pair(up, up);
                uint64_t sum = 0;
#pragma unroll
                for (int e = 0; e < 8; e += 4) {
                  const float2 y0 = unpair(fma2(pair(v[c][8 * j + e], v[c][8 * j + e + 1]), f2, up2));
                  const float2 y1 = unpair(fma2(pair(v[c][8 * j + e + 2], v[c][8 * j + e + 3]), f2, up2));
                  const float p0 = ex2(y0.x), p1 = ex2(y0.y), p2 = ex2(y1.x), p3 = ex2(y1.y);
                  sum = add2(sum, add2(pair(p0, p1), pair(p2, p3)));
                  weight_parts(p0, p1, p2, p3, &part[0][2 * j + e / 4], &part[1][2 * j + e / 4], &part[2][2 * j + e / 4]);
                }
                const float2 two = unpair(sum);
                l = fmaf(two.x + two.y, sc.z, l);
              }
              const uint32_t to = s_addr + copy * (NC / 4) + kChunk / 4 * c;
#pragma unroll
              for (int i = 0; i < 3; ++i) tmem_store_n<kChunk / 4>(to + i * (L::kPart / 4), part[i]);
            }
            if constexpr (L::kCopies > 1) {  // no weights for the slots of the other copies
              uint32_t zero[NC / 4];
#pragma unroll
              for (int e = 0; e < NC / 4; ++e) zero[e] = 0;
#pragma unroll
              for (int c = 0; c < L::kCopies; ++c) {
                if (c != copy) {
#pragma unroll
                  for (int i = 0; i < 3; ++i) tmem_store_n<NC / 4>(s_addr + i * (L::kPart / 4) + c * (NC / 4), zero);
                }
              }
            }
            tmem_wait_st();
          }
          if ((slot0 + a.tile > total || bad != 0) && quarter * L::kParts >> 2 == h) {
            // V rows that no copy filled, or stale slots behind the last token: zero
            const int vs = kt % L::kVS;
            warp_wait(&vfull[vs], (kt / L::kVS) & 1, abort_flag, a.status);
            const int vr = quarter * 32 + lane;
            if (slot0 + vr >= total || (vr < a.tile && ((bad >> (vr / a.box)) & 1))) {
              unsigned char* row = smem + L::kOffV + vs * L::kOperand + vr * HD;
#pragma unroll
              for (int c = 0; c < HD / 16; ++c) *reinterpret_cast<uint4*>(row + c * 16) = make_uint4(0u, 0u, 0u, 0u);
            }
            fence_proxy_async_smem();
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&pfull[buf]);
        }
      }

      // the groups' last mixes of the segment: of both where finish_segment reads both O, else of this one's
      const bool had0 = units > 1 || (x0 & 1) == 0, had1 = units > 1 || (x0 & 1) == 1;
      constexpr bool kOwnOnly = DUAL || L::kCopies > 1;
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const int last = x0 + units - 1 - ((x0 + units - 1 - g) & 1);  // group g's
        if ((g == 0 ? had0 : had1) && (!kOwnOnly || g == w)) warp_wait(&pvdone[L::kParts * (g + 1) - 1], (last >> 1) & 1, abort_flag, a.status);
      }
      tc_fence_after();
      finish_segment<L, HD>(a, smem, walk, s, slots, tmem, w, copy, r, had0, had1, seg, i0, live, m, l);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(ofree);
      tiles += n;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, L::kTmemCols);
  }
}

template <int HD, int COPIES>
int launch_form(TreeArgs a, cudaStream_t stream, const char* what) {
  using L = Layout8<HD, COPIES>;
  tile_of(a.page_size, &a.tile, &a.box);
  const uint64_t rows = static_cast<uint64_t>(a.num_pages) * a.hkv * a.page_size;
  CUtensorMap tk, tv;
  if (int st = make_tensor_map_bytes(&tk, a.k_pages, a.hd, rows, HD, a.box, what)) return st;
  if (int st = make_tensor_map_bytes(&tv, a.v_pages, a.hd, rows, HD, a.box, what)) return st;
  auto kernel = tree_tc8_kernel<HD, COPIES>;
  if (int st = allow_dynamic_smem(reinterpret_cast<const void*>(kernel), L::kBytes, what)) return st;
  a.whole = whole_items(a, tokens_of(COPIES, a.group));
  a.item_cost = kItemCost;
  const int nc = ctas_for(a.batch, a.hkv, a.group, a.max_ctx, a.max_tree);
  if (int st = launch_kernel(what, kernel, dim3(nc), dim3(kThreadsTc), L::kBytes, stream, nullptr, tk, tv, a)) return st;
  if (nc == 1 || a.whole) return BM_OK;  // no item is cut
  return launch_kernel(what, tree_merge_kernel<L, HD>, dim3(nc - 1, std::min(L::kRows / 8, 8)), dim3(256), 0, stream, nullptr, a, nc);
}

template <int HD>
int launch_hd(const TreeArgs& a, cudaStream_t stream, const char* what) {
  switch (copies_for(a.group, a.max_tree)) {
    case 4:
      return launch_form<HD, 4>(a, stream, what);
    case 2:
      return launch_form<HD, 2>(a, stream, what);
    case 1:
      return launch_form<HD, 1>(a, stream, what);
    default:
      return launch_form<HD, kDual>(a, stream, what);
  }
}

}  // namespace

// Eight neighbouring slots of a tile, from its beginning on, share a scale: blocks and boxes of whole
// eights, or a tile that is one part of a page inside one block.
bool tc8_takes(const TreeArgs& a, bm_dtype_t dtype) {
  const int64_t rows = static_cast<int64_t>(a.num_pages) * a.hkv * a.page_size;
  int tile, box;
  return dtype == BM_BF16 && a.hd <= 128 && tile_of(a.page_size, &tile, &box) && rows + kTile < (int64_t{1} << 31) &&
         ((a.block % kGroupSlots == 0 && box % kGroupSlots == 0) || (tile == box && a.block % box == 0));
}

int launch_tc8(const TreeArgs& a, cudaStream_t stream, const char* what) {
  return a.hd > 64 ? launch_hd<128>(a, stream, what) : launch_hd<64>(a, stream, what);
}

}  // namespace paged
}  // namespace bm
