// Tree attention over an 8-bit paged KV cache on the tensor cores (tcgen05 kind::f8f6f4, TMA,
// TMEM), for bf16 queries and head_dim up to 128. Same contract as paged_attention.cu.
//
// Mathematics: the running softmax of paged_attention.cu on tiles of 128 slots, K and V as the
// codes they are held in: nothing is widened on its way to the tensor cores.
//   scores  S[row][slot] = (Qh + Ql)[row][:] . Kc[slot][:]    two e4m3 x e4m3 products
//   mix     O[row][:]   += (Ph + Pl)[row][slot] Vc[slot][:]   e4m3 x e4m3 and e5m2 x e4m3
// Qh is the query times a power of two that puts its largest element in [128, 256), rounded to
// e4m3, and Ql what that leaves: together all 8 bits of a bf16 element down to 2^-9 of the largest, and
// 2^-17 of the largest below. Scales are powers of two, so they meet the softmax as exponents:
//   t = S f + e_v,  f = 2^(e_k - e_q) scale log2(e),  P = 2^(t - m + 2),  l += P 2^(-e_v)
// with e_k and e_v the exponents of K's and V's scale at the slot, e_q the query's and m the running maximum
// of t: the weight times V's scale is what the mix takes, so its rounding is relative to the
// largest term of the sum, however far blocks' scales lie apart. P is at most 2^8 (a row is rescaled when m rises by more than 6); as
// fp16 it splits into Ph (e4m3) and Pl = P - Ph (e5m2, whose exponents reach down to 2^-16): off by 2^-8 of itself
// at most, by 2^-16 of the largest where it is small: the precision of bf16 weights, for two products of
// twice bf16's rate.
//
// Bound: memory while group * tokens is below about 100 (a slot is half the bytes of a bf16
// cache's, for the same tensor time), above it the softmax: exponentials, and the conversions of P.
//
// Split and roles are paged_attention_tc.cu's, but for the queries and the scales: warp 2 converts a
// segment's queries into two operands in shared memory while the segment before is computed (all
// warps but those of TMA together for a CTA's first, which all wait for), and the warp that fetches K looks up
// the scales of its tile's slots, eight neighbouring ones of which share one.
#include <cuda.h>

#include "kv8.cuh"
#include "paged_attention_tc.cuh"

namespace bm {
namespace paged {
namespace {

constexpr float kRescaleAt8 = 6.f;  // rise of the maximum (log2) that a row's sums are rescaled at
constexpr float kLift = 2.f;        // P is 2^2 at the running maximum, so at most 2^8
constexpr int kGroupSlots = 8;      // slots of a tile that share a scale
constexpr int kGroups = kTile / kGroupSlots;
constexpr int kQRing = 4;           // segments whose queries' factors are kept
constexpr int kQWarps = 10;         // warps that convert a CTA's first queries: all but the two of TMA

template <int HD, int COPIES>
struct Layout8 : RowLayout<HD, COPIES> {
  using Rows = RowLayout<HD, COPIES>;
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
  static constexpr int kBars = 2 * kKS + 2 * kVS + 6 + 6;
  static constexpr int kOffPlan = kOffBar + kBars * 8;      // Plan, scan, bad-page ring
  static constexpr int kBytes = kOffPlan + 96 + 16 * 8 + kBadRing * 4 + 16 + 1024 /* alignment slack */;
  static_assert(kBytes <= 232448, "shared memory of a CTA");
  // Tiles between the one whose scores are issued next and the one a softmax group may still read.
  static_assert(kKS + 4 <= kBadRing, "rings by tile");
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
// 8 consecutive 32-bit columns of this thread's TMEM lane.
__device__ __forceinline__ void tmem_store8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]),
      "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(taddr)
      : "memory");
}
// The phase's bytes to come, without an arrival.
__device__ __forceinline__ void mbar_expect_only(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive_n(uint64_t* bar, uint32_t count) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(count) : "memory");
}

// Two values as e4m3 (lo in the low byte); ends at +-448.
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
// Two weights: e4m3 of their fp16 values, and e5m2 of what that leaves.
__device__ __forceinline__ void weight_parts(float lo, float hi, uint32_t* part, uint32_t* rest) {
  uint32_t p, back;
  uint16_t h, l;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(p) : "f"(hi), "f"(lo));
  asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(h) : "r"(p));
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(back) : "h"(h));
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(back) : "r"(p), "r"(back));
  asm("cvt.rn.satfinite.e5m2x2.f16x2 %0, %1;" : "=h"(l) : "r"(back));
  *part = h;
  *rest = l;
}

// Converts the queries of an item into its two parts in the buffer at `to`, row tile after row
// tile, copies and all, and their factors scale * log2(e) * 2^-e_q into factor[row]. Warp
// `worker` of `workers` takes every workers-th pair of rows, half a warp a row; rows of no token are zero.
template <typename L, int HD>
__device__ __forceinline__ void convert_queries(const TreeArgs& a, const Seq& s, int kvh, int p, int tpt, unsigned char* to, float* factor,
                                                int worker, int workers) {
  constexpr int kBatch = 4;  // pairs of rows that are converted side by side
  const int lane = threadIdx.x & 31, half = lane >> 4, c = lane & 15;
  const int i_first = p * tpt * L::kTiles;
  const uint32_t by_group = (65536u + a.group - 1) / a.group;  // r / group = r * by_group >> 16 for r < 128
  const bf16* q = static_cast<const bf16*>(a.q) + (s.row0 * a.hq + static_cast<int64_t>(kvh) * a.group) * a.hd + c * 8;
  const int64_t token_step = static_cast<int64_t>(a.hq) * a.hd;
  for (int pair0 = worker; pair0 < L::kRows / 2; pair0 += workers * kBatch) {
    uint4 raw[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int row = 2 * (pair0 + k * workers) + half, r = row % L::kCopyRows;
      const int token = static_cast<int>(r * by_group >> 16), i = i_first + row / L::kCopyRows * tpt + token;
      raw[k] = make_uint4(0u, 0u, 0u, 0u);
      if (row < L::kRows && token < tpt && i < s.n && c * 8 < a.hd) raw[k] = ld_keep(q + i * token_step + (r - token * a.group) * a.hd);
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
      if (row >= L::kRows) continue;
      const int e = min(max(static_cast<int>(top[k] >> 7) - 127, -60), 127);
      const float f = kv8::power(7 - e);
      if (c * 8 < HD) {
        float x[8];
        unpack16<bf16>(raw[k], x);
        uint32_t hi[2], lo[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float back[4];
          hi[j] = e4m3x2(x[4 * j] * f, x[4 * j + 1] * f) | e4m3x2(x[4 * j + 2] * f, x[4 * j + 3] * f) << 16;
          kv8::from_codes(hi[j], back);
#pragma unroll
          for (int d = 0; d < 4; ++d) back[d] = fmaf(x[4 * j + d], f, -back[d]);
          lo[j] = e4m3x2(back[0], back[1]) | e4m3x2(back[2], back[3]) << 16;
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
  constexpr uint32_t kIdescS = instr_desc_e4m3(false, false, kTile, kTile);
  constexpr uint32_t kIdescH = instr_desc_e4m3(false, true, HD, kTile);
  constexpr uint32_t kIdescL = instr_desc_e4m3(true, true, HD, kTile);
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
  uint64_t* sfull = vempty + L::kVS;    // scores in TMEM       (commit)
  uint64_t* pfull = sfull + 2;          // weights in TMEM      (one arrival per warp of the group)
  uint64_t* pvdone = pfull + 2;         // mix done             (commit)
  uint64_t* qfull = pvdone + 2;         // queries converted    (kQWarps arrivals)
  uint64_t* qempty = qfull + 2;         // the segment's last scores are done (commit)
  uint64_t* ofree = qempty + 2;         // the segment's O has been read (one arrival per softmax warp)
  uint64_t* mma_done = ofree + 1;
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
        mbar_init(&kempty[i], 1);
      }
      for (int i = 0; i < L::kVS; ++i) {
        mbar_init(&vfull[i], 1);
        mbar_init(&vempty[i], 1);
      }
      for (int i = 0; i < 2; ++i) {
        mbar_init(&sfull[i], 1);
        mbar_init(&pfull[i], 4);
        mbar_init(&pvdone[i], 1);
        mbar_init(&qfull[i], kQWarps);
        mbar_init(&qempty[i], 1);
      }
      mbar_init(ofree, 8);
      mbar_init(mma_done, 1);
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
    convert_queries<L, HD>(a, walk.s, walk.kvh, walk.p, tpt, smem, factors, worker, kQWarps);
    if (lane == 0) mbar_arrive(&qfull[0]);
    __syncwarp();
  }

  if (warp == 0 || warp == 3) {
    // ---------------- K with the scales (warp 0) and V (warp 3) ----------------
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
    for (; ok && walk.left > 0; walk.next(a, per)) {
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
      }
    }
    if (lane == 0) {  // copies still in flight land before the CTA ends
      for (int i = max(0, kt - stages); i < kt; ++i) {
        wait_phase(&full[i % stages], (i / stages) & 1, abort_flag, a.status, kDrainNs, false);
      }
    }
    __syncwarp();
  } else if (warp == 2) {
    // ---------------- the queries of the segments behind the first, one ahead ----------------
    int seg = 0;
    for (walk.next(a, per); walk.left > 0; walk.next(a, per)) {
      ++seg;
      const int buf = seg & 1;
      if (!warp_wait(&qempty[buf], ((seg >> 1) & 1) ^ 1u, abort_flag, a.status)) break;
      convert_queries<L, HD>(a, walk.s, walk.kvh, walk.p, tpt, smem + buf * L::kQBuf, factors + seg % kQRing * L::kRows, 0, 1);
      if (lane == 0) mbar_arrive_n(&qfull[buf], kQWarps);
      __syncwarp();
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer ----------------
    // Step x: the mix of unit x - 2, then the scores of unit x into the TMEM buffer that
    // mix has done with. The whole warp walks, one thread issues.
    const uint64_t q_desc = byte_desc<HD>(smem_u32(smem));
    const uint64_t k_desc = byte_desc<HD>(smem_u32(smem + L::kOffK));
    const uint64_t v_desc = byte_desc<HD>(smem_u32(smem + L::kOffV));
    constexpr uint32_t kStage = L::kOperand >> 4;
    bool issued = false, ok = true, first = true;
    int seg = 0, mix_seg = -1, end = -1;  // segments of the scores and of the mix; units in all, once known
    int ks = 0, vs = 0;                   // ring slots of the next scores and mix
    uint32_t k_phase = 0, v_phase = 0;
    uint32_t firsts = 0;                  // bit i: unit x - 1 - i is its segment's first
    int left = __shfl_sync(0xffffffffu, walk.segment(), 0) * L::kTiles;
    for (int x = 0; ok; ++x) {
      const int w = x & 1;
      if (x >= 2) {
        const bool opens = (firsts & 2) != 0;
        if (opens) ++mix_seg;
        ok = warp_wait(&pfull[w], ((x - 2) >> 1) & 1, abort_flag, a.status);
        // the segment's first mix overwrites O: its last reader was the previous segment's end
        if (ok && opens && mix_seg > 0) ok = warp_wait(ofree, (mix_seg - 1) & 1, abort_flag, a.status);
        if (ok) ok = warp_wait(&vfull[vs], v_phase, abort_flag, a.status);
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          const uint32_t fresh = (firsts & 6) != 0 ? 0u : 1u;  // the group's first unit of the segment
          constexpr uint32_t kStep = 32 * HD >> 4;             // 32 slots of V
#pragma unroll
          for (int kk = 0; kk < kTile / 32; ++kk) {
            mma_f8_ts(tmem + L::kColO + w * HD, tmem + w * kTile + kk * 8, v_desc + vs * kStage + kk * kStep, kIdescH, kk > 0 ? 1u : fresh);
          }
#pragma unroll
          for (int kk = 0; kk < kTile / 32; ++kk) {
            mma_f8_ts(tmem + L::kColO + w * HD, tmem + w * kTile + 32 + kk * 8, v_desc + vs * kStage + kk * kStep, kIdescL, 1u);
          }
          mma_commit(&pvdone[w]);
          if (!DUAL || w == 1) mma_commit(&vempty[vs]);
        }
        __syncwarp();
        issued = true;
        if ((!DUAL || w == 1) && ++vs == L::kVS) {
          vs = 0;
          v_phase ^= 1;
        }
      }
      if (left > 0) {
        const int buf = seg & 1;
        if (first) ok = warp_wait(&qfull[buf], (seg >> 1) & 1, abort_flag, a.status);
        if (ok) ok = warp_wait(&kfull[ks], k_phase, abort_flag, a.status);
        if (ok && x >= 2) ok = warp_wait(&pvdone[w], ((x - 2) >> 1) & 1, abort_flag, a.status);
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          const uint64_t q_at = q_desc + ((buf * L::kQBuf + (DUAL ? w * L::kQTile : 0)) >> 4);
#pragma unroll
          for (int kk = 0; kk < HD / 32; ++kk) {
            mma_f8(tmem + w * kTile, q_at + kk * 2, k_desc + ks * kStage + kk * 2, kIdescS, kk > 0 ? 1u : 0u);
          }
#pragma unroll
          for (int kk = 0; kk < HD / 32; ++kk) {
            mma_f8(tmem + w * kTile, q_at + kStage + kk * 2, k_desc + ks * kStage + kk * 2, kIdescS, 1u);
          }
          mma_commit(&sfull[w]);
          if (!DUAL || w == 1) mma_commit(&kempty[ks]);
          if (left == 1) mma_commit(&qempty[buf]);
        }
        __syncwarp();
        issued = true;
        firsts = firsts << 1 | (first ? 1u : 0u);
        first = false;
        if ((!DUAL || w == 1) && ++ks == L::kKS) {
          ks = 0;
          k_phase ^= 1;
        }
        if (--left == 0) {
          walk.next(a, per);
          ++seg;
          left = __shfl_sync(0xffffffffu, walk.left > 0 ? walk.segment() : 0, 0) * L::kTiles;
          first = left > 0;
          if (left == 0) end = x + 1;
        }
      } else {
        firsts <<= 1;
        if (x == end + 1) break;  // the last unit's mix is issued
      }
    }
    if (issued) {
      if (elect_one()) mma_commit(mma_done);
      __syncwarp();
      if (lane == 0) wait_phase(mma_done, 0, abort_flag, a.status, kDrainNs, false);
      __syncwarp();
    }
  } else {
    // ---------------- softmax ----------------
    constexpr int NC = L::kCols;
    const int w = (warp - 4) >> 2;      // group
    const int quarter = warp & 3;
    const int copy = quarter * 32 / L::kCopyRows;
    const int r = quarter * 32 % L::kCopyRows + lane;  // row of the row tile; lane quarter * 32 + lane of TMEM is its
    const uint32_t lane_addr = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t s_addr = tmem + lane_addr + w * kTile;
    const uint32_t o_addr = tmem + lane_addr + L::kColO + w * HD;
    int x = 0;  // the segment's first unit
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
      const int u0 = x + ((x & 1) == w ? 0 : 1);
      for (int u = u0; u < x + units; u += 2) {
        const int kt = DUAL ? u >> 1 : u;
        const int t = walk.t + (DUAL ? (u - x) >> 1 : u - x);  // tile of the item
        warp_wait(&sfull[w], (u >> 1) & 1, abort_flag, a.status);
        tc_fence_after();
        const int slot0 = t * a.tile;
        const uint32_t bad = bad_ring[kt % kBadRing];
        if (u == u0) factor = factors[seg % kQRing * L::kRows + (DUAL ? w * kTile : 0) + r];
        if (warp_live) {
          // This copy's scores of the row: at most 64 are held, of 128 the second half is
          // loaded twice (its weights go where the first half's scores were).
          constexpr int kHeld = NC < 64 ? NC : 64;
          const float4* group = scales + kt % kBadRing * kGroups + copy * (NC / kGroupSlots);
          uint32_t v[kHeld / 32][32];
          auto load = [&](int col) {
#pragma unroll
            for (int c = 0; c < kHeld / 32; ++c) tmem_load32(s_addr + copy * NC + col + 32 * c, v[c]);
            tmem_wait_ld();
            if (slot0 + a.tile > s.ctx || a.tile < kTile || bad != 0) {
#pragma unroll
              for (int c = 0; c < kHeld / 32; ++c) {
                const int at = copy * NC + col + 32 * c;
                uint32_t see = r < live ? seen32(a, s, token, slot0 + at) & low_bits(a.tile - at) : 0xffffffffu;
                if (bad) see &= sound32(bad, at, a.box);
                if (__all_sync(0xffffffffu, see == 0xffffffffu)) continue;  // a prompt's chunks are mostly seen
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                  if (!((see >> e) & 1)) v[c][e] = 0xff800000u;  // -inf: no weight
                }
              }
              __syncwarp();
            }
          };
          // what a group's scores are multiplied by: never 0, since -inf times it has to stay
          auto times = [&](float k) {
            const float f = k * factor;
            return f < 1.17549435e-38f ? 1.17549435e-38f : f;
          };
          float top = -INFINITY;
          auto highest = [&](int col) {
#pragma unroll
            for (int c = 0; c < kHeld / 32; ++c) {
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const float4 sc = group[col / kGroupSlots + 4 * c + j];
                float most = __uint_as_float(v[c][8 * j]);
#pragma unroll
                for (int e = 1; e < 7; e += 2) most = max3(most, __uint_as_float(v[c][8 * j + e]), __uint_as_float(v[c][8 * j + e + 1]));
                most = fmaxf(most, __uint_as_float(v[c][8 * j + 7]));
                top = fmaxf(top, fmaf(most, times(sc.x), sc.y));
              }
            }
          };
          if constexpr (NC == 128) {
            load(64);
            highest(64);
          }
          load(0);
          highest(0);
          if (r >= live) top = -INFINITY;
          if (factor != factor) top = 0.f;  // a row of NaN stays one through its merges
          const bool rise = top > m + kRescaleAt8 || (m == -INFINITY && top > -INFINITY);
          const float m_new = rise ? top : m;
          const float alpha = rise ? ex2(m - m_new) : 1.f;  // m = -inf: 0
          if (u != u0 && __any_sync(0xffffffffu, rise)) {
            // the group's previous mix is done: these scores were issued after it
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
          auto weigh = [&](int col) {
#pragma unroll
            for (int c = 0; c < kHeld / 32; ++c) {
              uint32_t part[8], rest[8];
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const float4 sc = group[col / kGroupSlots + 4 * c + j];
                const float f = times(sc.x), up = sc.y - base;
                const uint64_t f2 = pair(f, f), up2 = pair(up, up);
                uint64_t sum = 0;
#pragma unroll
                for (int e = 0; e < 8; e += 4) {
                  const float2 y0 = unpair(fma2(pair(v[c][8 * j + e], v[c][8 * j + e + 1]), f2, up2));
                  const float2 y1 = unpair(fma2(pair(v[c][8 * j + e + 2], v[c][8 * j + e + 3]), f2, up2));
                  const float p0 = ex2(y0.x), p1 = ex2(y0.y), p2 = ex2(y1.x), p3 = ex2(y1.y);
                  sum = add2(sum, add2(pair(p0, p1), pair(p2, p3)));
                  uint32_t h0, h1, l0, l1;
                  weight_parts(p0, p1, &h0, &l0);
                  weight_parts(p2, p3, &h1, &l1);
                  part[2 * j + e / 4] = h0 | h1 << 16;
                  rest[2 * j + e / 4] = l0 | l1 << 16;
                }
                const float2 two = unpair(sum);
                l = fmaf(two.x + two.y, sc.z, l);
              }
              const uint32_t to = s_addr + (copy * NC + col) / 4 + 8 * c;
              tmem_store8(to, part);
              tmem_store8(to + 32, rest);
            }
          };
          weigh(0);
          if constexpr (NC == 128) {
            load(64);
            weigh(64);
          }
          if constexpr (L::kCopies > 1) {  // no weights for the slots of the other copies
            uint32_t zero[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) zero[e] = 0;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              if (c / (NC / 32) != copy) {
                tmem_store8(s_addr + 8 * c, zero);
                tmem_store8(s_addr + 32 + 8 * c, zero);
              }
            }
          }
          tmem_wait_st();
        }
        if (slot0 + a.tile > total || bad != 0) {
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
        if (lane == 0) mbar_arrive(&pfull[w]);
      }

      // the groups' last mixes of the segment: of both where finish_segment reads both O, else of this one's
      const int end = x + units;
      const int last0 = end - 1 - ((end - 1) & 1), last1 = end - 1 - (~(end - 1) & 1);
      const bool had0 = last0 >= x, had1 = last1 >= x;
      constexpr bool kOwnOnly = DUAL || L::kCopies > 1;
      if (had0 && (!kOwnOnly || w == 0)) warp_wait(&pvdone[0], (last0 >> 1) & 1, abort_flag, a.status);
      if (had1 && (!kOwnOnly || w == 1)) warp_wait(&pvdone[1], (last1 >> 1) & 1, abort_flag, a.status);
      tc_fence_after();
      finish_segment<L, HD>(a, smem, walk, s, slots, tmem, w, copy, r, had0, had1, seg, i0, live, m, l);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(ofree);
      x += units;
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
