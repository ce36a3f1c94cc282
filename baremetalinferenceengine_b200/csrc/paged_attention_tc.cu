// Tree attention over a paged KV cache on the tensor cores (tcgen05, TMA, TMEM), for
// bf16 caches with head_dim up to 128 (filled up with zeros to 64 or 128 by TMA). Same
// contract as paged_attention.cu.
//
// Mathematics: the running softmax of paged_attention.cu on tiles of 128 slots (fewer
// where whole pages do not make 128), with both products as tcgen05.mma:
//   scores  S[row][slot] = Q[row][:] . K[slot][:]    M = 128 rows, N = 128 slots
//   mix     O[row][:]   += P[row][slot] V[slot][:]   M = 128 rows, N = head_dim
// A row is (token, head of the group), token-major: 128 / group tokens share a tile of
// K and V. Each softmax thread owns one row (one TMEM lane), so maxima and sums need no
// exchange between threads; P overwrites S in TMEM as bf16 and is the A operand of the
// mix from there. O stays in TMEM; a row whose maximum rises by more than 2^8 (in the
// exponent's base) is rescaled there, smaller rises leave its weights up to 2^8 (fp32
// sums, bf16's exponent range: nothing is lost by it).
//
// Weights are rounded to bf16 for the mix, as bm_decode_attention does: both operands of these
// MMAs have V's type. The row sums take them before rounding. Outputs are off 64 bits by
// 1.9e-3 to 2.3e-3 in the 2-norm, of which 1.7e-3 is their own rounding. A weight in two bf16 parts
// (16 MMAs a mix, twice the stores to TMEM) brings that to 1.7e-3 and the three cases measured
// below to 246, 364 and 27 us; not kept.
//
// Bound: memory while group * tokens is below about 200 (two operations per K and V
// element and row against 2.25 bytes per ns and SM), the tensor cores and the
// exponentials above. Padding to M = 128 costs nothing that bounds: a tile's two
// products take 1024 cycles, its 64 KB of K and V 2800 at the SM's share of HBM. What few
// rows would leave idle is the softmax: a thread walks its row's 128 scores however few
// rows there are. So with at most 64 (32) rows the row tile holds them twice (four times),
// and each copy weighs a half (quarter) of the tile's slots, with zero weights elsewhere;
// the copies' sums meet at the segment's end. Measured on a B200 with both launches, calls
// one after the other (in brackets before the power limit lowers the SM clock from 1965 to 1600
// MHz): 64 sequences of 1 to 8192 and up to 8 drafted tokens, 32 / 8 heads of 128: 214 (189) us
// (1.03 GB, floor 157; one copy everywhere 16 us more); 16 of 4096 to 8192 and 64, 64 / 8 heads:
// 285 (241) us (floor 124 by products, 120 by bytes); one of 8000 and 12: 25 us (floor 5); a
// prompt's 2048 tokens behind 6144 without a mask, 64 / 8 heads: 547 us (floor 290 by products).
//
// Split: the host does not see the lengths, so one CTA per SM takes an equal share of
// all tiles of the batch, counted on the device: items (sequence, kv head, row tile) laid
// end to end, CTA c walking tiles [c T / nc, (c + 1) T / nc). An item cut at a CTA border
// leaves partials in the workspace (at most two per CTA), which tree_merge_kernel adds
// up; a whole one is written directly. Where the bounds allow no item of more than
// kWholeTiles tiles, borders move on to the next item instead: walking the rest of a short
// item costs less than a merge.
//
// Twelve warps:
//   warps 0, 3 TMA of K and of V, pages looked up by their lanes, one box of a page's
//              rows (or an equal part of them) x 64 dims each, into separate rings;
//   warp 1     owns TMEM; one thread issues every MMA;
//   warp 2     TMA of the queries, once per segment (an item's part in this CTA);
//   warps 4-7, 8-11  two softmax groups. Unit u of the CTA's sequence goes to group
//              u & 1 with TMEM buffers S[u & 1] and O[u & 1]: with one row tile per
//              item units are its tiles in turn, and both groups' sums meet at the
//              segment's end; with more rows (kDual) a tile is two units, one per row
//              tile, so K and V are read once for 256 rows.
// Every mbarrier wait is bounded in time: past the limit the CTA raises
// BM_DEVERR_TIMEOUT, lets its copies and MMAs land, frees TMEM and returns.
#include <cuda.h>

#include "paged_attention_tc.cuh"

namespace bm {
namespace paged {

namespace {

constexpr float kRescaleAt = 8.f;

template <int HD, int COPIES>
struct Layout : RowLayout<HD, COPIES> {
  using Rows = RowLayout<HD, COPIES>;
  static constexpr int kBox = kTile * 128;                  // 128 rows x 64 dims of bf16
  static constexpr int kOperand = HD / 64 * kBox;           // a tile of Q, K or V
  static constexpr int kKS = HD == 128 ? 2 : 4;             // K ring: freed by the scores
  static constexpr int kVS = HD == 128 ? 3 : 6;             // V ring: freed by the mix
  static constexpr int kOffK = Rows::kTiles * kOperand;
  static constexpr int kOffV = kOffK + kKS * kOperand;
  static constexpr int kOffMl = kOffV + kVS * kOperand;
  static constexpr int kOffSum = kOffMl + Rows::kMlBytes;
  static constexpr int kOffBar = kOffSum + Rows::kSumBytes;
  static constexpr int kBars = 2 * kKS + 2 * kVS + 6 + 4;
  static constexpr int kOffPlan = kOffBar + kBars * 8;      // Plan, scan, bad-page ring
  static constexpr int kBytes = kOffPlan + 96 + 16 * 8 + kBadRing * 4 + 16 + 1024 /* alignment slack */;
  static_assert(kBytes <= 232448, "shared memory of a CTA");
};

// D[tmem] (+)= A[tmem] * B[smem], kind::f16: A's rows are TMEM lanes, two bf16 a column.
__device__ __forceinline__ void mma_bf16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
      ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}

template <int HD, int COPIES>
__global__ void __launch_bounds__(kThreadsTc, 1)
    tree_tc_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                   const __grid_constant__ CUtensorMap tv, const TreeArgs a) {
  grid_dependency_wait();
  using L = Layout<HD, COPIES>;
  constexpr bool DUAL = L::kTwo;
  constexpr uint32_t kIdescS = instr_desc_bf16(false, false, kTile, kTile);
  constexpr uint32_t kIdescO = instr_desc_bf16(false, true, HD, kTile);
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                                         ~static_cast<uintptr_t>(1023));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int cta = static_cast<int>(blockIdx.x);
  const int tpt = L::kCopyRows / a.group;  // tokens of a row tile
  const int per = tpt * L::kTiles;         // and of an item

  uint64_t* kfull = reinterpret_cast<uint64_t*>(smem + L::kOffBar);
  uint64_t* kempty = kfull + L::kKS;
  uint64_t* vfull = kempty + L::kKS;
  uint64_t* vempty = vfull + L::kVS;
  uint64_t* sfull = vempty + L::kVS;  // scores in TMEM       (commit)
  uint64_t* pfull = sfull + 2;        // weights in TMEM      (one arrival per warp of the group)
  uint64_t* pvdone = pfull + 2;       // mix done             (commit)
  uint64_t* qfull = pvdone + 2;
  uint64_t* qempty = qfull + 1;       // the segment's last scores are done (commit)
  uint64_t* ofree = qempty + 1;       // the segment's O has been read (one arrival per softmax warp)
  uint64_t* mma_done = ofree + 1;
  Plan* plan = reinterpret_cast<Plan*>(smem + L::kOffPlan);
  int64_t* scan = reinterpret_cast<int64_t*>(smem + L::kOffPlan + 96);
  volatile uint32_t* bad_ring = reinterpret_cast<volatile uint32_t*>(scan + 16);
  uint32_t* tmem_base_s = const_cast<uint32_t*>(bad_ring) + kBadRing;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_base_s + 1);
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
      }
      mbar_init(qfull, 1);
      mbar_init(qempty, 1);
      mbar_init(ofree, 8);
      mbar_init(mma_done, 1);
      *abort_flag = 0;
      fence_barrier_init();
    }
    if (warp == 1) tmem_alloc(tmem_base_s, L::kTmemCols);
    if (a.tile < kTile) {  // V rows that no copy ever fills: zero, since their weights of 0 meet them
      const int rows = kTile - a.tile;
      for (int c = tid; c < L::kVS * (HD / 64) * rows * 8; c += kThreadsTc) {
        const int row = a.tile + c / 8 % rows, block = c / 8 / rows;
        *reinterpret_cast<uint4*>(smem + L::kOffV + block * L::kBox + row * 128 + c % 8 * 16) = make_uint4(0u, 0u, 0u, 0u);
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

  if (warp == 0 || warp == 3) {
    // ---------------- K (warp 0) and V (warp 3) ----------------
    const bool is_v = warp == 3;
    const CUtensorMap* map = is_v ? &tv : &tk;
    uint64_t* full = is_v ? vfull : kfull;
    uint64_t* empty = is_v ? vempty : kempty;
    unsigned char* ring = smem + (is_v ? L::kOffV : L::kOffK);
    const int stages = is_v ? L::kVS : L::kKS;
    constexpr int halves = HD / 64;      // 64 dims each; past head_dim the copy fills in zeros
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
          if (!is_v) {
            bad_ring[kt % kBadRing] = bad;
            if (bad) raise_status(a.status, BM_DEVERR_BAD_PAGE);
          }
          mbar_expect_tx(&full[stage], __popc(have) * a.box * 128 * halves);
        }
        __syncwarp();
        if (row >= 0) {
          unsigned char* to = ring + stage * L::kOperand + lane * a.box * 128;
          for (int h = 0; h < halves; ++h) tma_load_2d(to + h * L::kBox, map, &full[stage], 64 * h, row);
        }
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
  } else if (warp == 2 && lane == 0) {
    // ---------------- queries ----------------
    int seg = 0;
    for (; walk.left > 0; walk.next(a, per), ++seg) {
      if (!wait_phase(qempty, (seg & 1) ^ 1u, abort_flag, a.status, kWaitNs, true)) break;
      mbar_expect_tx(qfull, L::kTiles * L::kCopies * (HD / 64) * a.group * tpt * 128);
#pragma unroll
      for (int w = 0; w < L::kTiles; ++w) {
        const int token = static_cast<int>(walk.s.row0) + walk.p * per + w * tpt;
#pragma unroll
        for (int h = 0; h < HD / 64; ++h) {
#pragma unroll
          for (int c = 0; c < L::kCopies; ++c) {
            tma_load_3d(smem + w * L::kOperand + h * L::kBox + c * L::kCopyRows * 128, &tq, qfull, 64 * h, walk.kvh * a.group, token);
          }
        }
      }
    }
    if (seg > 0) wait_phase(qfull, (seg - 1) & 1, abort_flag, a.status, kDrainNs, false);
  } else if (warp == 1) {
    // ---------------- MMA issuer ----------------
    // Step x: the mix of unit x - 2, then the scores of unit x into the TMEM buffer that
    // mix has done with. The whole warp walks, one thread issues: descriptors stay in
    // uniform registers, and a product of 64 cycles is not held up by its issue.
    const uint64_t q_desc = smem_desc(smem_u32(smem), 16, 1024);
    const uint64_t k_desc = smem_desc(smem_u32(smem + L::kOffK), 16, 1024);
    const uint64_t v_desc = smem_desc(smem_u32(smem + L::kOffV), L::kBox, 1024);
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
#pragma unroll
          for (int kk = 0; kk < kTile / 16; ++kk) {
            mma_bf16_ts(tmem + L::kColO + w * HD, tmem + w * kTile + kk * 8, v_desc + vs * kStage + kk * 128, kIdescO,
                        kk > 0 ? 1u : fresh);
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
        if (first) ok = warp_wait(qfull, seg & 1, abort_flag, a.status);
        if (ok) ok = warp_wait(&kfull[ks], k_phase, abort_flag, a.status);
        if (ok && x >= 2) ok = warp_wait(&pvdone[w], ((x - 2) >> 1) & 1, abort_flag, a.status);
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < HD / 16; ++kk) {
            constexpr uint32_t kAtom = L::kBox >> 4;
            const uint32_t off = (kk >> 2) * kAtom + (kk & 3) * 2;
            mma_bf16(tmem + w * kTile, q_desc + (DUAL ? w * kStage : 0) + off, k_desc + ks * kStage + off, kIdescS,
                     kk > 0 ? 1u : 0u);
          }
          mma_commit(&sfull[w]);
          if (!DUAL || w == 1) mma_commit(&kempty[ks]);
          if (left == 1) mma_commit(qempty);
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
  } else if (warp >= 4) {
    // ---------------- softmax ----------------
    constexpr int NC = L::kCols;
    const int w = (warp - 4) >> 2;      // group
    const int quarter = warp & 3;
    const int copy = quarter * 32 / L::kCopyRows;
    const int r = quarter * 32 % L::kCopyRows + lane;  // row of the row tile; lane quarter * 32 + lane of TMEM is its
    const uint32_t lane_addr = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t s_addr = tmem + lane_addr + w * kTile;
    const uint32_t o_addr = tmem + lane_addr + L::kColO + w * HD;
    const uint64_t scale2 = pair(a.qscale, a.qscale);
    int x = 0;  // the segment's first unit
    for (int seg = 0; walk.left > 0; walk.next(a, per), ++seg) {
      const int n = walk.segment();
      const int units = n * L::kTiles;
      const Seq s = walk.s;
      const int i0 = walk.p * per + (DUAL ? w * tpt : 0);
      const int live = max(0, min(tpt, s.n - i0)) * a.group;
      const bool warp_live = r - lane < live;
      const int token = i0 + r / a.group;  // a row past `live` computes on what it finds and is not stored
      const int total = s.ctx + s.n;
      float m = -INFINITY, l = 0.f;
      const int u0 = x + ((x & 1) == w ? 0 : 1);
      for (int u = u0; u < x + units; u += 2) {
        const int kt = DUAL ? u >> 1 : u;
        const int t = walk.t + (DUAL ? (u - x) >> 1 : u - x);  // tile of the item
        warp_wait(&sfull[w], (u >> 1) & 1, abort_flag, a.status);
        tc_fence_after();
        const int slot0 = t * a.tile;
        const uint32_t bad = bad_ring[kt % kBadRing];
        if (warp_live) {
          // This copy's scores of the row: at most 64 are held, of 128 the second half is
          // loaded twice (its weights go where the first half's scores were).
          constexpr int kHeld = NC < 64 ? NC : 64;
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
          float top = -INFINITY, top1 = -INFINITY;
          auto highest = [&]() {
#pragma unroll
            for (int c = 0; c < kHeld / 32; ++c) {
#pragma unroll
              for (int e = 0; e < 32; e += 4) {
                top = max3(top, __uint_as_float(v[c][e]), __uint_as_float(v[c][e + 1]));
                top1 = max3(top1, __uint_as_float(v[c][e + 2]), __uint_as_float(v[c][e + 3]));
              }
            }
          };
          if constexpr (NC == 128) {
            load(64);
            highest();
          }
          load(0);
          highest();
          top = r < live ? fmaxf(top, top1) * a.qscale : -INFINITY;
          const bool rise = top > m + kRescaleAt || (m == -INFINITY && top > -INFINITY);
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
          const float base = m == -INFINITY ? 0.f : m;
          const uint64_t minus = pair(-base, -base);
          uint64_t sum[2] = {0, 0};
          auto weigh = [&](int col) {
#pragma unroll
            for (int c = 0; c < kHeld / 32; ++c) {
              uint32_t pk[16];
#pragma unroll
              for (int e = 0; e < 32; e += 2) {
                const float2 y = unpair(fma2(pair(v[c][e], v[c][e + 1]), scale2, minus));
                const float p0 = ex2(y.x), p1 = ex2(y.y);
                sum[e / 2 % 2] = add2(sum[e / 2 % 2], pair(p0, p1));
                pk[e / 2] = pack_bf16x2(p0, p1);
              }
              tmem_store16(s_addr + (copy * NC + col) / 2 + 16 * c, pk);
            }
          };
          weigh(0);
          if constexpr (NC == 128) {
            load(64);
            weigh(64);
          }
          if constexpr (L::kCopies > 1) {  // no weights for the slots of the other copies
            uint32_t zero[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) zero[e] = 0;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              if (c / (NC / 32) != copy) tmem_store16(s_addr + 16 * c, zero);
            }
          }
          const float2 sums = unpair(add2(sum[0], sum[1]));
          l += sums.x + sums.y;
          tmem_wait_st();
        }
        if (slot0 + a.tile > total || bad != 0) {
          // V rows that no copy filled, or stale slots behind the last token: zero
          const int vs = kt % L::kVS;
          warp_wait(&vfull[vs], (kt / L::kVS) & 1, abort_flag, a.status);
          const int vr = quarter * 32 + lane;
          if (slot0 + vr >= total || (vr < a.tile && ((bad >> (vr / a.box)) & 1))) {
            unsigned char* row = smem + L::kOffV + vs * L::kOperand + vr * 128;
#pragma unroll
            for (int h = 0; h < HD / 64; ++h) {
#pragma unroll
              for (int c = 0; c < 8; ++c) *reinterpret_cast<uint4*>(row + h * L::kBox + c * 16) = make_uint4(0u, 0u, 0u, 0u);
            }
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
  using L = Layout<HD, COPIES>;
  tile_of(a.page_size, &a.tile, &a.box);
  const int tpt = L::kCopyRows / a.group;
  const uint64_t rows = static_cast<uint64_t>(a.num_pages) * a.hkv * a.page_size;
  CUtensorMap tq, tk, tv;
  if (int st = make_tensor_map_bf16(&tk, a.k_pages, a.hd, rows, 64, a.box, what)) return st;
  if (int st = make_tensor_map_bf16(&tv, a.v_pages, a.hd, rows, 64, a.box, what)) return st;
  if (int st = make_tensor_map_3d_bf16(&tq, a.q, a.hd, a.hq, a.total_q, 64, a.group, tpt, what)) return st;
  auto kernel = tree_tc_kernel<HD, COPIES>;
  if (int st = allow_dynamic_smem(reinterpret_cast<const void*>(kernel), L::kBytes, what)) return st;
  a.whole = whole_items(a, tokens_of(COPIES, a.group));
  const int nc = ctas_for(a.batch, a.hkv, a.group, a.max_ctx, a.max_tree);
  if (int st = launch_kernel(what, kernel, dim3(nc), dim3(kThreadsTc), L::kBytes, stream, nullptr, tq, tk, tv, a)) return st;
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

bool tc_takes(const TreeArgs& a, bm_dtype_t dtype) {
  const int64_t rows = static_cast<int64_t>(a.num_pages) * a.hkv * a.page_size;
  int tile, box;
  return dtype == BM_BF16 && a.hd <= 128 && tile_of(a.page_size, &tile, &box) && rows + kTile < (int64_t{1} << 31);
}

size_t tc_workspace_bytes(int64_t batch, int hkv, int hd, int group, int max_ctx, int max_tree) {
  if (hd > 128 || hd % 8) return 0;
  const int nc = ctas_for(batch, hkv, group, max_ctx, max_tree);
  const size_t rows = static_cast<size_t>(rows_of(copies_for(group, max_tree)));
  return records_bytes(nc) + 2 * static_cast<size_t>(nc) * rows * ((hd <= 64 ? 64 : 128) + 2) * sizeof(float);
}

int launch_tc(const TreeArgs& a, cudaStream_t stream, const char* what) {
  return a.hd > 64 ? launch_hd<128>(a, stream, what) : launch_hd<64>(a, stream, what);
}

}  // namespace paged
}  // namespace bm
