// Tree attention over an 8-bit paged KV cache on the tensor cores for few rows per kv head (up to
// 64: decoding, small trees): the products of paged_attention8_tc.cu transposed.
//
// Mathematics, precision and scales are paged_attention8_tc.cu's; here slots are the rows of the products:
//   scores  S[slot][row] = Kc[slot][:] . (Qh + Ql)[row][:]    M = 128 slots, N = 32 rows
//   mix     O[dim][row] += Vc[slot][dim] (Ph + Pl)[slot][row]  M = 128 dims,  N = 32 rows
// so that a tile costs the tensor cores what its 32 rows need (a fourth of the form with rows as
// M), a softmax thread owns one slot, with the scales of its own (blocks of any size), and weighs it
// for all rows, and a row's sums meet without copies. What moves in return: a row's maximum lies over
// threads. It may lag by 2^4, so each thread compares its scores with the maxima that
// the group of threads holds, one barrier of the group tells whether any exceeds, and only then (in a
// sequence's first tiles, mostly) maxima are taken. Weights go through shared memory as
// the mix's second operand, 32 bytes of a slot's rows for each part. Weight sums stay with the threads
// until a segment ends.
//
// Bound: memory. Per tile of 128 slots (32 KB of 128 dims, 1300 cycles at the SM's share of HBM)
// a group of four warps takes some 700 cycles, and two groups take tiles in turn (or, with more
// than 32 rows, both the same tile, each its own 32 rows). Scores run three tiles ahead of the mix.
//
// Split, plan and walk are paged_attention_tc.cu's. Twelve warps:
//   warps 0, 3 TMA of K and of V;  warp 1 owns TMEM, one thread issues every MMA;
//   warp 2     queries of the next segment (all warps but those of TMA convert a CTA's first);
//   warps 4-7, 8-11  two softmax groups.
#include <cuda.h>

#include "paged_attention8_tc.cuh"

namespace bm {
namespace paged {
namespace {

constexpr int kRowsFew = 32;  // rows of a unit
constexpr int kBufs = 4;      // units in flight: scores in TMEM, weights in shared memory

template <bool TWO, int HDS = 128>
struct LayoutFew {
  static constexpr int kTiles = TWO ? 2 : 1;                // row tiles of an item
  static constexpr int kCopies = 1;
  static constexpr int kCopyRows = kRowsFew;
  static constexpr int kRows = kTiles * kRowsFew;           // rows of an item
  static constexpr int kSlotFloats = kRows * (HDS + 2);     // a partial: sums, then maxima, then weight sums
  static constexpr int kTileBytes = kTile * 128;            // a tile of K or V: rows of 128 bytes, past head_dim zeros
  static constexpr int kQTile = 2 * kRowsFew * 128;         // both parts of a row tile
  static constexpr int kOperand = kRowsFew * 128;           // one part
  static constexpr int kQBuf = kTiles * kQTile;
  static constexpr int kPart = kTile * kRowsFew;            // one part of a unit's weights
  static constexpr int kKS = TWO ? 4 : 5;
  static constexpr int kVS = 5;
  static constexpr int kOffK = 2 * kQBuf;
  static constexpr int kOffV = kOffK + kKS * kTileBytes;
  static constexpr int kOffP = kOffV + kVS * kTileBytes;
  static constexpr int kOffFactor = kOffP + kBufs * 2 * kPart;       // [kQRing][kRows]
  static constexpr int kOffMax = kOffFactor + kQRing * kRows * 4;    // [2][32] a group's maxima, as subtracted: m - lift
  static constexpr int kOffAlpha = kOffMax + 2 * kRowsFew * 4;       // [2][32]
  static constexpr int kOffTop = kOffAlpha + 2 * kRowsFew * 4;       // [2][4][32] of each warp; sums at the end
  static constexpr int kOffMl = kOffTop + 2 * 4 * kRowsFew * 4;      // [2][32] (factor, -) of the segment's end
  static constexpr int kOffBar = kOffMl + 2 * kRowsFew * 8;
  static constexpr int kBars = 2 * kKS + 2 * kVS + 3 * kBufs + 6;
  static constexpr int kOffPlan = kOffBar + kBars * 8;
  static constexpr int kBytes = kOffPlan + 96 + 16 * 8 + 16 + 1024 /* alignment slack */;
  static_assert(kBytes <= 232448, "shared memory of a CTA");
  static constexpr uint32_t kColO = kBufs * kRowsFew;       // TMEM: S of four units, O of two groups, 32 columns each
  static constexpr uint32_t kTmemCols = 256;
};

// The matrix descriptor of rows of 32 bytes, eight of them a swizzle atom (32-byte swizzle).
__device__ __forceinline__ uint64_t weight_desc(uint32_t addr) {
  return static_cast<uint64_t>((addr >> 4) & 0x3FFFu) | (1ull << 16) | (static_cast<uint64_t>(256 >> 4) << 32) | (1ull << 46) | (6ull << 61);
}
// kind::f8f6f4, A and B each e4m3 or (B) e5m2, fp32 accumulator.
__host__ __device__ constexpr uint32_t instr_desc_few(bool a_mn_major, bool b_mn_major, bool b_e5m2) {
  return (1u << 4) | ((b_e5m2 ? 1u : 0u) << 10) | ((a_mn_major ? 1u : 0u) << 15) | ((b_mn_major ? 1u : 0u) << 16) |
         (static_cast<uint32_t>(kRowsFew >> 3) << 17) | (static_cast<uint32_t>(kTile >> 4) << 24);
}

__device__ __forceinline__ void group_sync(int w) { asm volatile("bar.sync %0, 128;" ::"r"(2 + w) : "memory"); }
// Whether any thread of the group says so (and all have come here).
__device__ __forceinline__ bool group_any(int w, bool mine) {
  uint32_t any;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 q, %2, 0;\n\t"
      "bar.red.or.pred p, %1, 128, q;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(any)
      : "r"(2 + w), "r"(mine ? 1u : 0u)
      : "memory");
  return any != 0;
}
__device__ __forceinline__ float warp_max(float x) {
  float r;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(x));
  return r;
}
// 32 consecutive 32-bit columns of this thread's TMEM lane.
__device__ __forceinline__ void tmem_store32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
      "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]),
      "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(taddr)
      : "memory");
}

template <bool TWO>
__global__ void __launch_bounds__(kThreadsTc, 1)
    tree_few8_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv, const TreeArgs a, int hds) {
  grid_dependency_wait();
  using L = LayoutFew<TWO>;
  constexpr uint32_t kIdescS = instr_desc_few(false, false, false);
  constexpr uint32_t kIdescH = instr_desc_few(true, true, false);
  constexpr uint32_t kIdescL = instr_desc_few(true, true, true);
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                                         ~static_cast<uintptr_t>(1023));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int cta = static_cast<int>(blockIdx.x);
  const int tpt = kRowsFew / a.group;  // tokens of a row tile
  const int per = tpt * L::kTiles;     // and of an item

  uint64_t* kfull = reinterpret_cast<uint64_t*>(smem + L::kOffBar);
  uint64_t* kempty = kfull + L::kKS;
  uint64_t* vfull = kempty + L::kKS;
  uint64_t* vempty = vfull + L::kVS;
  uint64_t* sfull = vempty + L::kVS;  // scores in TMEM              (commit)
  uint64_t* pfull = sfull + kBufs;    // weights in shared memory    (one arrival per warp of the group)
  uint64_t* pvdone = pfull + kBufs;   // mix done                    (commit)
  uint64_t* qfull = pvdone + kBufs;   // queries converted           (kQWarps arrivals)
  uint64_t* qempty = qfull + 2;       // the segment's last scores are done (commit)
  uint64_t* ofree = qempty + 2;       // the segment's O has been read (one arrival per softmax warp)
  uint64_t* mma_done = ofree + 1;
  Plan* plan = reinterpret_cast<Plan*>(smem + L::kOffPlan);
  int64_t* scan = reinterpret_cast<int64_t*>(smem + L::kOffPlan + 96);
  uint32_t* tmem_base_s = reinterpret_cast<uint32_t*>(scan + 16);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_base_s + 1);
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
      for (int i = 0; i < kBufs; ++i) {
        mbar_init(&sfull[i], 1);
        mbar_init(&pfull[i], 4);
        mbar_init(&pvdone[i], 1);
      }
      for (int i = 0; i < 2; ++i) {
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
      for (int c = tid; c < L::kVS * rows * 8; c += kThreadsTc) {
        const int row = a.tile + c / 8 % rows, stage = c / 8 / rows;
        *reinterpret_cast<uint4*>(smem + L::kOffV + stage * L::kTileBytes + row * 128 + c % 8 * 16) = make_uint4(0u, 0u, 0u, 0u);
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
    convert_queries<L, 128>(a, walk.s, walk.kvh, walk.p, tpt, smem, factors, warp < 3 ? warp - 1 : warp - 2, kQWarps);
    if (lane == 0) mbar_arrive(&qfull[0]);
    __syncwarp();
  }

  if (warp == 0 || warp == 3) {
    // ---------------- K (warp 0) and V (warp 3) ----------------
    const bool is_v = warp == 3;
    const CUtensorMap* map = is_v ? &tv : &tk;
    uint64_t* full = is_v ? vfull : kfull;
    uint64_t* empty = is_v ? vempty : kempty;
    unsigned char* ring = smem + (is_v ? L::kOffV : L::kOffK);
    const int stages = is_v ? L::kVS : L::kKS;
    const int boxes = a.tile / a.box;    // of a tile: at most 16
    int kt = 0, stage = 0;               // tiles asked for; the next one's ring slot
    uint32_t phase = 1;
    bool ok = true;
    for (; ok && walk.left > 0; walk.next(a, per)) {
      const int n = walk.segment();
      const int32_t* pages = a.page_table + static_cast<int64_t>(walk.s.seq) * a.max_pages;
      const int total = walk.s.ctx + walk.s.n;
      auto row_of = [&](int t) {  // this lane's box of tile t: its row in the tensor map, -1 bad, -2 none
        const int slot = t * a.tile + lane * a.box;
        if (lane >= boxes || slot >= total) return -2;
        const int nth = slot / a.page_size;
        const int32_t page = __ldg(pages + nth);
        if (page < 0 || page >= a.num_pages) return -1;
        return (page * a.hkv + walk.kvh) * a.page_size + (slot - nth * a.page_size);
      };
      int row = row_of(walk.t);
      for (int i = 0; i < n; ++i) {
        const int next_row = i + 1 < n ? row_of(walk.t + i + 1) : -2;  // looked up while this tile waits
        const uint32_t have = __ballot_sync(0xffffffffu, row >= 0);
        const uint32_t bad = __ballot_sync(0xffffffffu, row == -1);
        if (!(ok = warp_wait(&empty[stage], phase, abort_flag, a.status))) break;
        if (lane == 0) {
          if (bad && !is_v) raise_status(a.status, BM_DEVERR_BAD_PAGE);
          mbar_expect_tx(&full[stage], __popc(have) * a.box * 128);
        }
        __syncwarp();
        if (row >= 0) tma_load_2d(ring + stage * L::kTileBytes + lane * a.box * 128, map, &full[stage], 0, row);
        ++kt;
        if (++stage == stages) {
          stage = 0;
          phase ^= 1;
        }
        row = next_row;
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
      convert_queries<L, 128>(a, walk.s, walk.kvh, walk.p, tpt, smem + buf * L::kQBuf, factors + seg % kQRing * L::kRows, 0, 1);
      if (lane == 0) mbar_arrive_n(&qfull[buf], kQWarps);
      __syncwarp();
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer ----------------
    // Step x: the mix of unit x - 3, then the scores of unit x, whose buffer unit x - 4 has left: its
    // weights are in shared memory. The whole warp walks, one thread issues.
    constexpr int kAhead = kBufs - 1;
    const uint64_t q_desc = byte_desc<128>(smem_u32(smem));
    const uint64_t k_desc = byte_desc<128>(smem_u32(smem + L::kOffK));
    const uint64_t v_desc = byte_desc<128>(smem_u32(smem + L::kOffV));
    const uint64_t p_desc = weight_desc(smem_u32(smem + L::kOffP));
    const int steps = (a.hd + 31) / 32;   // of the scores: 32 dims each
    bool issued = false, ok = true, first = true;
    int seg = 0, mix_seg = -1, end = -1;  // segments of the scores and of the mix; units in all, once known
    int ks = 0, vs = 0;                   // ring slots of the next scores and mix
    uint32_t k_phase = 0, v_phase = 0;
    uint32_t firsts = 0;                  // bit i: unit x - 1 - i is its segment's first
    int left = __shfl_sync(0xffffffffu, walk.segment(), 0) * L::kTiles;
    for (int x = 0; ok; ++x) {
      if (x >= kAhead) {
        const int u = x - kAhead, buf = u % kBufs, w = u & 1;
        const bool opens = (firsts >> (kAhead - 1)) & 1;
        if (opens) ++mix_seg;
        ok = warp_wait(&pfull[buf], (u / kBufs) & 1, abort_flag, a.status);
        // the segment's first mix overwrites O: its last reader was the previous segment's end
        if (ok && opens && mix_seg > 0) ok = warp_wait(ofree, (mix_seg - 1) & 1, abort_flag, a.status);
        if (ok) ok = warp_wait(&vfull[vs], v_phase, abort_flag, a.status);
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          // the group's first unit of the segment: the segment's first or second
          const uint32_t fresh = ((firsts >> (kAhead - 1)) & 3) != 0 ? 0u : 1u;
          const uint32_t o = tmem + L::kColO + w * kRowsFew;
          const uint64_t p = p_desc + (buf * 2 * L::kPart >> 4), v = v_desc + vs * (L::kTileBytes >> 4);
#pragma unroll
          for (int kk = 0; kk < kTile / 32; ++kk) mma_f8(o, v + kk * (32 * 128 >> 4), p + kk * (32 * 32 >> 4), kIdescH, kk > 0 ? 1u : fresh);
#pragma unroll
          for (int kk = 0; kk < kTile / 32; ++kk) mma_f8(o, v + kk * (32 * 128 >> 4), p + (L::kPart >> 4) + kk * (32 * 32 >> 4), kIdescL, 1u);
          mma_commit(&pvdone[buf]);
          if (!TWO || w == 1) mma_commit(&vempty[vs]);
        }
        __syncwarp();
        issued = true;
        if ((!TWO || w == 1) && ++vs == L::kVS) {
          vs = 0;
          v_phase ^= 1;
        }
      }
      if (left > 0) {
        const int qbuf = seg & 1, buf = x % kBufs, w = x & 1;
        if (first) ok = warp_wait(&qfull[qbuf], (seg >> 1) & 1, abort_flag, a.status);
        if (ok) ok = warp_wait(&kfull[ks], k_phase, abort_flag, a.status);
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          const uint64_t q_at = q_desc + ((qbuf * L::kQBuf + (TWO ? w * L::kQTile : 0)) >> 4), k_at = k_desc + ks * (L::kTileBytes >> 4);
          for (int kk = 0; kk < steps; ++kk) mma_f8(tmem + buf * kRowsFew, k_at + kk * 2, q_at + kk * 2, kIdescS, kk > 0 ? 1u : 0u);
          for (int kk = 0; kk < steps; ++kk) mma_f8(tmem + buf * kRowsFew, k_at + kk * 2, q_at + (L::kOperand >> 4) + kk * 2, kIdescS, 1u);
          mma_commit(&sfull[buf]);
          if (!TWO || w == 1) mma_commit(&kempty[ks]);
          if (left == 1) mma_commit(&qempty[qbuf]);
        }
        __syncwarp();
        issued = true;
        firsts = firsts << 1 | (first ? 1u : 0u);
        first = false;
        if ((!TWO || w == 1) && ++ks == L::kKS) {
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
        if (x >= end + kAhead - 1) break;  // the last unit's mix is issued
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
    const int w = (warp - 4) >> 2;      // group
    const int quarter = warp & 3;
    const int own = quarter * 32 + lane;  // this thread's slot of a tile, and its dim of O
    const uint32_t lane_addr = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t o_addr = tmem + lane_addr + L::kColO + w * kRowsFew;
    float* maxima = reinterpret_cast<float*>(smem + L::kOffMax) + w * kRowsFew;   // m - lift; -inf: none yet
    float* alphas = reinterpret_cast<float*>(smem + L::kOffAlpha) + w * kRowsFew;
    float* tops = reinterpret_cast<float*>(smem + L::kOffTop);                    // [2][4][32]
    float2* ends = reinterpret_cast<float2*>(smem + L::kOffMl);                   // [2][32]
    int x = 0;  // the segment's first unit
    for (int seg = 0; walk.left > 0; walk.next(a, per), ++seg) {
      const int n = walk.segment();
      const int units = n * L::kTiles;
      const Seq s = walk.s;
      const int i0 = walk.p * per + (TWO ? w * tpt : 0);
      const int live = max(0, min(tpt, s.n - i0)) * a.group;
      const int total = s.ctx + s.n;
      const int32_t* pages = a.page_table + static_cast<int64_t>(s.seq) * a.max_pages;
      const int u0 = x + ((x & 1) == w ? 0 : 1);
      const int t_step = TWO ? 1 : 2;   // tiles from one of this group's units to the next
      // The row of this thread's slot in tile t of the item, among all pages' rows; -1 where it has none.
      auto row_of = [&](int t) {
        const int slot = t * a.tile + own;
        if (own >= a.tile || slot >= total || t >= walk.t + n) return -1;
        const int nth = slot / a.page_size;
        const int32_t page = __ldg(pages + nth);
        return page < 0 || page >= a.num_pages ? -1 : (page * a.hkv + walk.kvh) * a.page_size + (slot - nth * a.page_size);
      };
      uint32_t kb = 127, vb = 127;
      auto scales_of = [&](int row, uint32_t* k, uint32_t* v) {
        *k = *v = 127;
        if (row < 0) return;
        *k = __ldg(a.k_scales + row / a.block);  // blocks divide pages
        *v = __ldg(a.v_scales + row / a.block);
      };
      const int t_first = walk.t + (TWO ? 0 : u0 - x);
      int row = row_of(t_first), row1 = row_of(t_first + t_step);
      scales_of(row, &kb, &vb);
      if (quarter == 0) maxima[lane] = lane < live ? -INFINITY : INFINITY;  // rows of nobody never rise, and weigh nothing
      group_sync(w);
      const float* factor = factors + seg % kQRing * L::kRows + (TWO ? w * kRowsFew : 0);
      uint64_t l2[kRowsFew / 2];  // this thread's share of the rows' weight sums
#pragma unroll
      for (int j = 0; j < kRowsFew / 2; ++j) l2[j] = 0;

      for (int u = u0; u < x + units; u += 2) {
        const int kt = TWO ? u >> 1 : u, buf = u % kBufs;
        const int t = walk.t + (TWO ? (u - x) >> 1 : u - x);  // tile of the item
        // on their way while this unit waits and computes
        const int row2 = row_of(t + 2 * t_step);
        uint32_t kb1, vb1;
        scales_of(row1, &kb1, &vb1);
        warp_wait(&sfull[buf], (u / kBufs) & 1, abort_flag, a.status);
        tc_fence_after();
        const int slot = t * a.tile + own;
        uint32_t seen = row < 0 ? 0u : 0xffffffffu;  // bit r: row r sees this slot
        if (seen != 0 && slot >= s.ctx) {
          const int j = slot - s.ctx;
          seen = 0;
          for (int i = 0; i < tpt && i0 + i < s.n; ++i) {
            if (sees(a, s.row0, i0 + i, j)) seen |= low_bits(a.group) << (i * a.group);
          }
        }
        __syncwarp();
        uint32_t v[kRowsFew];
        tmem_load32(tmem + lane_addr + buf * kRowsFew, v);
        const float kf = kv8::power(kv8::exponent(static_cast<uint8_t>(kb)));
        const int ev = kv8::exponent(static_cast<uint8_t>(vb));
        const uint64_t kf2 = pair(kf, kf), up2 = pair(static_cast<float>(ev), static_cast<float>(ev));
        tmem_wait_ld();
        // t = S f + e_v of every row, and whether any exceeds its maximum by more than it may
        bool over = false;
#pragma unroll
        for (int c = 0; c < kRowsFew; c += 8) {
          if (c >= live) break;  // the same for the CTA's group
#pragma unroll
          for (int e = c; e < c + 8; e += 4) {
            const ulonglong2 f = *reinterpret_cast<const ulonglong2*>(factor + e);
            const float4 m = *reinterpret_cast<const float4*>(maxima + e);
            const float2 y0 = unpair(fma2(pair(v[e], v[e + 1]), mul2(f.x, kf2), up2));
            const float2 y1 = unpair(fma2(pair(v[e + 2], v[e + 3]), mul2(f.y, kf2), up2));
            const float y[4] = {y0.x, y0.y, y1.x, y1.y}, top[4] = {m.x, m.y, m.z, m.w};
#pragma unroll
            for (int d = 0; d < 4; ++d) {
              const float z = (seen >> (e + d)) & 1 ? y[d] : -INFINITY;
              over = over || z > top[d] + (kLift + kRescaleAt8);
              v[e + d] = __float_as_uint(z);
            }
          }
        }
        if (group_any(w, over)) {
          // a row whose maximum has to rise: its new one, and what its sums are multiplied by
#pragma unroll
          for (int e = 0; e < kRowsFew; ++e) {
            if ((e & 7) == 0 && e >= live) break;
            const float top = warp_max(__uint_as_float(v[e]));
            if (lane == e) tops[(w * 4 + quarter) * kRowsFew + e] = top;
          }
          group_sync(w);
          if (quarter == 0) {
            float top = -INFINITY;
#pragma unroll
            for (int q = 0; q < 4; ++q) top = fmaxf(top, tops[(w * 4 + q) * kRowsFew + lane]);
            const float before = maxima[lane];
            const bool rise = top > before + (kLift + kRescaleAt8);
            alphas[lane] = rise ? ex2(before - (top - kLift)) : 1.f;  // before = -inf: 0
            if (rise) maxima[lane] = top - kLift;
          }
          group_sync(w);
          if (u != u0) {
            warp_wait(&pvdone[(u - 2) % kBufs], ((u - 2) / kBufs) & 1, abort_flag, a.status);
            tc_fence_after();
            uint32_t o[kRowsFew];
            tmem_load32(o_addr, o);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < kRowsFew; e += 4) {
              const float4 f = *reinterpret_cast<const float4*>(alphas + e);
              l2[e / 2] = mul2(l2[e / 2], pair(f.x, f.y));
              l2[e / 2 + 1] = mul2(l2[e / 2 + 1], pair(f.z, f.w));
              o[e] = __float_as_uint(__uint_as_float(o[e]) * f.x);
              o[e + 1] = __float_as_uint(__uint_as_float(o[e + 1]) * f.y);
              o[e + 2] = __float_as_uint(__uint_as_float(o[e + 2]) * f.z);
              o[e + 3] = __float_as_uint(__uint_as_float(o[e + 3]) * f.w);
            }
            tmem_store32(o_addr, o);
            tmem_wait_st();
          }
        }
        // weights, their sums without V's scale, and their parts
        if (u >= kBufs) warp_wait(&pvdone[buf], ((u - kBufs) / kBufs) & 1, abort_flag, a.status);  // the buffer has been read
        const float down = kv8::power(-ev);
        const uint64_t down2 = pair(down, down);
        unsigned char* to = smem + L::kOffP + buf * 2 * L::kPart + own * 32;
        const int flip = (own >> 2 & 1) * 16;  // the 32-byte swizzle
#pragma unroll
        for (int c = 0; c < kRowsFew; c += 16) {
          if (c >= live) break;
          uint32_t part[4], rest[4];
#pragma unroll
          for (int e = c; e < c + 16; e += 4) {
            const float4 m = *reinterpret_cast<const float4*>(maxima + e);
            const float b[4] = {m.x, m.y, m.z, m.w};
            float p[4];
#pragma unroll
            for (int d = 0; d < 4; ++d) p[d] = ex2(__uint_as_float(v[e + d]) - (b[d] == -INFINITY ? 0.f : b[d]));
            l2[e / 2] = fma2(pair(p[0], p[1]), down2, l2[e / 2]);
            l2[e / 2 + 1] = fma2(pair(p[2], p[3]), down2, l2[e / 2 + 1]);
            uint32_t h0, h1, r0, r1;
            weight_parts(p[0], p[1], &h0, &r0);
            weight_parts(p[2], p[3], &h1, &r1);
            part[(e - c) / 4] = h0 | h1 << 16;
            rest[(e - c) / 4] = r0 | r1 << 16;
          }
          *reinterpret_cast<uint4*>(to + (c ^ flip)) = make_uint4(part[0], part[1], part[2], part[3]);
          *reinterpret_cast<uint4*>(to + L::kPart + (c ^ flip)) = make_uint4(rest[0], rest[1], rest[2], rest[3]);
        }
        if (row < 0) {
          // a V row that no copy filled, or a stale slot behind the last token: zero
          const int vs = kt % L::kVS;
          wait_phase(&vfull[vs], (kt / L::kVS) & 1, abort_flag, a.status, kWaitNs, true);
          unsigned char* v_row = smem + L::kOffV + vs * L::kTileBytes + own * 128;
#pragma unroll
          for (int c = 0; c < 8; ++c) *reinterpret_cast<uint4*>(v_row + c * 16) = make_uint4(0u, 0u, 0u, 0u);
        }
        fence_proxy_async_smem();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&pfull[buf]);
        row = row1;
        row1 = row2;
        kb = kb1;
        vb = vb1;
      }

      // The segment's end. Weight sums: halves of the rows change sides until lane r holds row r's, then
      // over the group's warps.
      float l[kRowsFew];
#pragma unroll
      for (int e = 0; e < kRowsFew; e += 2) {
        const float2 two = unpair(l2[e / 2]);
        l[e] = two.x;
        l[e + 1] = two.y;
      }
#pragma unroll
      for (int keep = 16; keep >= 1; keep >>= 1) {
        const bool upper = lane & keep;
#pragma unroll
        for (int e = 0; e < keep; ++e) {
          const float give = upper ? l[e] : l[e + keep], have = upper ? l[e + keep] : l[e];
          l[e] = have + __shfl_xor_sync(0xffffffffu, give, keep);
        }
      }
      tops[(w * 4 + quarter) * kRowsFew + lane] = l[0];
      const int end = x + units;
      const int last = end - 1 - ((end - 1 - w) & 1);  // this group's last unit; below x: its O is stale
      if (last >= x) warp_wait(&pvdone[last % kBufs], (last / kBufs) & 1, abort_flag, a.status);
      tc_fence_after();
      both_groups_sync();
      const bool whole = walk.t == 0 && n == walk.tiles;
      float* slot = slots + (2 * static_cast<int64_t>(cta) + (seg > 0)) * (L::kRows * (hds + 2));
      // One warp of each group (TWO) or of the first works out the rows' maxima, sums and factors.
      if (quarter == 0 && (TWO || w == 0)) {
        auto sum_of = [&](int g) {
          float t = 0.f;
#pragma unroll
          for (int q = 0; q < 4; ++q) t += tops[(g * 4 + q) * kRowsFew + lane];
          return t;
        };
        const float m0 = maxima[lane];  // this group's (w is 0 unless TWO)
        if (TWO) {
          const float sum = sum_of(w);
          const float inv = !whole ? 1.f : sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;
          ends[w * kRowsFew + lane] = make_float2(inv, 0.f);
          if (!whole && lane < live) {
            slot[L::kRows * hds + w * kRowsFew + lane] = m0;
            slot[L::kRows * (hds + 1) + w * kRowsFew + lane] = sum;
          }
        } else {
          const float m1 = maxima[kRowsFew + lane];
          const float top = fmaxf(m0, m1), base = top == -INFINITY ? 0.f : top;
          const float f0 = ex2(m0 - base), f1 = ex2(m1 - base);  // a maximum of -inf: 0
          const float s0 = sum_of(0), s1 = sum_of(1), sum = s0 * f0 + s1 * f1;
          const float inv = !whole ? 1.f : sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;
          ends[lane] = make_float2(f0 * inv, f1 * inv);
          if (!whole && lane < live) {
            slot[L::kRows * hds + lane] = top;
            slot[L::kRows * (hds + 1) + lane] = sum;
          }
        }
      }
      both_groups_sync();
      // Values: a thread has a dim of every row; without TWO each group adds both groups' for half of the rows.
      const bool had0 = TWO || end - 1 - ((end - 1) & 1) >= x, had1 = end - 1 - (~(end - 1) & 1) >= x;
      constexpr int kShare = TWO ? kRowsFew : kRowsFew / 2;
      const int r_lo = TWO ? 0 : w * kShare;
#pragma unroll
      for (int c = 0; c < kShare; c += 16) {
        uint32_t o0[16], o1[16];
        if (r_lo + c < live) {
          if (TWO) {
            tmem_load16(o_addr + c, o0);
          } else {
            if (had0) tmem_load16(tmem + lane_addr + L::kColO + r_lo + c, o0);
            if (had1) tmem_load16(tmem + lane_addr + L::kColO + kRowsFew + r_lo + c, o1);
          }
          tmem_wait_ld();
          int token = i0 + (r_lo + c) / a.group, g = (r_lo + c) % a.group;
#pragma unroll
          for (int e = 0; e < 16; ++e, ++g) {
            const int r = r_lo + c + e;
            if (g == a.group) {
              g = 0;
              ++token;
            }
            if (r >= live || own >= a.hd) continue;
            const float2 f = ends[(TWO ? w * kRowsFew : 0) + r];
            float y;
            if (TWO) {
              y = __uint_as_float(o0[e]) * f.x;
            } else {
              y = had0 && f.x != 0.f ? __uint_as_float(o0[e]) * f.x : 0.f;
              if (had1 && f.y != 0.f) y = fmaf(__uint_as_float(o1[e]), f.y, y);
            }
            if (whole) {
              static_cast<bf16*>(a.out)[((s.row0 + token) * a.hq + walk.kvh * a.group + g) * a.hd + own] = __float2bfloat16_rn(y);
            } else {
              slot[((TWO ? w * kRowsFew : 0) + r) * hds + own] = y;
            }
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(ofree);
      x = end;
      both_groups_sync();  // maxima and sums have been read
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, L::kTmemCols);
  }
}

template <bool TWO>
int launch_form(TreeArgs a, int nc, cudaStream_t stream, const char* what) {
  using L = LayoutFew<TWO>;
  const uint64_t rows = static_cast<uint64_t>(a.num_pages) * a.hkv * a.page_size;
  CUtensorMap tk, tv;
  if (int st = make_tensor_map_bytes(&tk, a.k_pages, a.hd, rows, 128, a.box, what)) return st;
  if (int st = make_tensor_map_bytes(&tv, a.v_pages, a.hd, rows, 128, a.box, what)) return st;
  auto kernel = tree_few8_kernel<TWO>;
  if (int st = allow_dynamic_smem(reinterpret_cast<const void*>(kernel), L::kBytes, what)) return st;
  const int per = L::kTiles * (kRowsFew / a.group), hds = a.hd > 64 ? 128 : 64;
  a.whole = whole_items(a, per);
  if (int st = launch_kernel(what, kernel, dim3(nc), dim3(kThreadsTc), L::kBytes, stream, nullptr, tk, tv, a, hds)) return st;
  if (nc == 1 || a.whole) return BM_OK;  // no item is cut
  const dim3 grid(nc - 1, L::kRows / 8);
  return hds == 128 ? launch_kernel(what, tree_merge_kernel<LayoutFew<TWO, 128>, 128>, grid, dim3(256), 0, stream, nullptr, a, nc)
                    : launch_kernel(what, tree_merge_kernel<LayoutFew<TWO, 64>, 64>, grid, dim3(256), 0, stream, nullptr, a, nc);
}

}  // namespace

int launch_few8(const TreeArgs& a, int nc, cudaStream_t stream, const char* what) {
  return a.max_tree <= kRowsFew / a.group ? launch_form<false>(a, nc, stream, what) : launch_form<true>(a, nc, stream, what);
}

}  // namespace paged
}  // namespace bm
