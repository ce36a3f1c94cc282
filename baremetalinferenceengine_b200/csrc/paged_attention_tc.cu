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

#include <algorithm>

#include "bm_tc.cuh"
#include "bm_tma.h"
#include "paged_attention.cuh"

namespace bm {
namespace paged {

using namespace bm::tc;

namespace {

constexpr int kTile = 128;      // slots per tile, rows per row tile
constexpr int kThreadsTc = 384;
constexpr int kMinTiles = 2;    // tiles that make a CTA worth starting, where items are cut
constexpr int kWholeTiles = 8;  // of the longest item, up to which items stay whole
constexpr int kBadRing = 16;    // tiles whose bad-page bits are kept
constexpr uint64_t kWaitNs = 2000000000ull;
constexpr uint64_t kDrainNs = 200000000ull;
constexpr float kRescaleAt = 8.f;

// How an item's rows lie in row tiles: two tiles of rows, or one holding them COPIES times.
constexpr int kDual = 0;

template <int HD, int COPIES>
struct Layout {
  static constexpr bool kTwo = COPIES == kDual;
  static constexpr int kTiles = kTwo ? 2 : 1;               // row tiles of an item
  static constexpr int kCopies = kTwo ? 1 : COPIES;
  static constexpr int kCopyRows = kTile / kCopies;         // rows of a copy
  static constexpr int kCols = kTile / kCopies;             // slots of a tile that a copy weighs
  static constexpr int kRows = kTiles * kCopyRows;          // rows of an item
  static constexpr int kBox = kTile * 128;                  // 128 rows x 64 dims of bf16
  static constexpr int kOperand = HD / 64 * kBox;           // a tile of Q, K or V
  static constexpr int kKS = HD == 128 ? 2 : 4;             // K ring: freed by the scores
  static constexpr int kVS = HD == 128 ? 3 : 6;             // V ring: freed by the mix
  static constexpr int kOffK = kTiles * kOperand;
  static constexpr int kOffV = kOffK + kKS * kOperand;
  static constexpr int kOffMl = kOffV + kVS * kOperand;     // [2][2][128] (maximum, sum), not with two tiles
  // The copies' sums meet in shared memory, kDims dims of all rows at a time, each of the
  // kWriters (group, copy) adding its own kStep dims in turn.
  static constexpr int kWriters = 2 * kCopies;  // (unused with one copy)
  static constexpr int kDims = 4096 / kCopyRows < HD ? 4096 / kCopyRows : HD;
  static constexpr int kStep = kDims / kWriters;
  static constexpr int kPitch = kDims + 4;
  static constexpr int kOffSum = kOffMl + (kTwo ? 0 : 2 * 2 * kTile * 8);
  static constexpr int kOffBar = kOffSum + (kCopies > 1 ? kCopyRows * kPitch * 4 : 0);
  static constexpr int kBars = 2 * kKS + 2 * kVS + 6 + 4;
  static constexpr int kOffPlan = kOffBar + kBars * 8;      // Plan, scan, bad-page ring
  static constexpr int kBytes = kOffPlan + 96 + 16 * 8 + kBadRing * 4 + 16 + 1024 /* alignment slack */;
  static_assert(kBytes <= 232448, "shared memory of a CTA");
  static constexpr uint32_t kColO = 256;                    // TMEM: S0, S1 (128 each), O0, O1 (HD each)
  static constexpr uint32_t kTmemCols = 512;
  static constexpr int kSlotFloats = kRows * (HD + 2);      // a partial: sums, then maxima, then weight sums
};

// What a CTA left of its first segment, for the merge.
struct Record {
  int64_t lo, total;   // its first tile, and all tiles
  int32_t b, kvh, p;   // the item
  int32_t t0, tiles;   // the segment's first tile in it (-1: no segment), the item's tiles
  int32_t nc;          // CTAs with tiles
};
static_assert(sizeof(Record) == 40, "record layout");

__host__ __device__ constexpr size_t records_bytes(int nc) { return (static_cast<size_t>(nc) * sizeof(Record) + 255) / 256 * 256; }

// Tiles of item p (its row tiles hold `per` tokens) of a sequence.
__device__ __forceinline__ int item_tiles(const TreeArgs& a, const Seq& s, int p, int per) {
  const int seen = s.ctx + (a.mask ? s.n : min(s.n, (p + 1) * per));
  return (seen + a.tile - 1) / a.tile;
}
// All tiles of one kv head of a sequence, and its items.
__device__ __forceinline__ int64_t head_tiles(const TreeArgs& a, const Seq& s, int per, int* items) {
  *items = (s.n + per - 1) / per;
  if (a.mask) return static_cast<int64_t>(*items) * item_tiles(a, s, 0, per);
  int64_t t = 0;
  for (int p = 0; p < *items; ++p) t += item_tiles(a, s, p, per);
  return t;
}

// Tiles from tile `off` of a sequence to the next beginning of an item (0: it is one).
__device__ __forceinline__ int64_t to_next_item(const TreeArgs& a, const Seq& s, int64_t off, int64_t head, int per) {
  off %= head;
  for (int p = 0;; ++p) {
    const int tiles = item_tiles(a, s, p, per);
    if (off < tiles) return off == 0 ? 0 : tiles - off;
    off -= tiles;
  }
}

// The walk over a CTA's segments: every role runs its own, with the same results.
struct Walk {
  int64_t b, left;
  int items, kvh, p, t, tiles;
  Seq s;

  // Tile `off` of sequence b is the CTA's first, and `n` tiles are its own.
  __device__ void start(const TreeArgs& a, const Seq& sequence, int64_t b0, int64_t off, int64_t n, int per) {
    b = b0;
    left = n;
    s = sequence;
    int64_t head = head_tiles(a, s, per, &items);
    if (off >= a.hkv * head) {  // behind the sequence's last item: the next one with tiles
      do {
        ++b;
        read_seq(a, b, &s);
      } while (s.n == 0);
      head = head_tiles(a, s, per, &items);
      off = 0;
    }
    kvh = static_cast<int>(off / head);
    off -= kvh * head;
    p = 0;
    while (off >= (tiles = item_tiles(a, s, p, per))) {
      off -= tiles;
      ++p;
    }
    t = static_cast<int>(off);
  }
  // Tiles of the current segment (0 when the walk is over).
  __device__ int segment() const { return static_cast<int>(left < tiles - t ? left : tiles - t); }
  __device__ void next(const TreeArgs& a, int per) {
    left -= segment();
    if (left == 0) return;
    t = 0;
    if (++p == items) {
      p = 0;
      if (++kvh == a.hkv) {
        kvh = 0;
        do {
          ++b;  // a later sequence has tiles: the plan counted them
          read_seq(a, b, &s);
        } while (s.n == 0);
        items = (s.n + per - 1) / per;
      }
    }
    tiles = item_tiles(a, s, p, per);
  }
};

struct Plan {
  int64_t lo, hi, b, off;  // this CTA's tiles; the first is tile `off` of sequence b
  Seq s;                   // sequence b
};
static_assert(sizeof(Plan) <= 96, "room in the layout");

// The whole warp waits; lane 0 watches the clock where it is not over at once.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int32_t* status) {
  if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
  int ok = 1;
  if ((threadIdx.x & 31) == 0) ok = wait_phase(bar, parity, abort_flag, status, kWaitNs, true);
  return __shfl_sync(0xffffffffu, ok, 0) != 0;
}
// One thread of a converged warp, always the same.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(p));
  return p != 0;
}

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
// 16 consecutive 32-bit columns of this thread's TMEM lane.
__device__ __forceinline__ void tmem_store16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
      : "memory");
}
// 8 consecutive fp32 columns of this thread's TMEM lane, into r's first.
__device__ __forceinline__ void tmem_load8(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr));
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
      ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}

__device__ __forceinline__ uint32_t low_bits(int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; }

// Which of the 32 slots from slot0 on row i of the sequence sees.
__device__ __forceinline__ uint32_t seen32(const TreeArgs& a, const Seq& s, int i, int slot0) {
  const int lead = min(max(s.ctx - slot0, 0), 32);
  uint32_t v = low_bits(lead);
  const int j0 = slot0 + lead - s.ctx;  // the first drafted slot among them
  if (lead < 32 && j0 < s.n) {
    uint32_t tree;
    if (a.mask == nullptr) {
      tree = low_bits(min(i + 1, s.n) - j0);
    } else {
      const uint64_t* m = a.mask + (s.row0 + i) * a.words;
      uint64_t bits = __ldg(m + (j0 >> 6)) >> (j0 & 63);
      if ((j0 & 63) > 32 && (j0 >> 6) + 1 < a.words) bits |= __ldg(m + (j0 >> 6) + 1) << (64 - (j0 & 63));
      tree = static_cast<uint32_t>(bits) & low_bits(s.n - j0);
    }
    v |= tree << lead;
  }
  return v;
}

// Which of the 32 slots at column 32c of a tile have a sound page (bit b of bad: the
// tile's box b has not). Two boxes or more hold whole groups of 8 slots each.
__device__ __forceinline__ uint32_t sound32(uint32_t bad, int c, int box_rows) {
  uint32_t v = 0xffffffffu;
  for (int e = 0; e < 32; e += 8) {
    if ((bad >> min((32 * c + e) / box_rows, 31)) & 1) v &= ~(0xffu << e);
  }
  return v;
}

__device__ __forceinline__ float max3(float a, float b, float c) { return fmaxf(fmaxf(a, b), c); }

__device__ __forceinline__ void both_groups_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
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
    const int64_t share = (a.batch + kThreadsTc - 1) / kThreadsTc;
    const int64_t b_lo = min(a.batch, tid * share), b_hi = min(a.batch, b_lo + share);
    int64_t mine = 0;
    Seq s;
    for (int64_t b = b_lo; b < b_hi; ++b) {
      const int32_t bad = read_seq(a, b, &s);
      if (bad && cta == 0) raise_status(a.status, bad);
      int items;
      mine += a.hkv * head_tiles(a, s, per, &items);
    }
    int64_t incl = mine;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int64_t v = __shfl_up_sync(0xffffffffu, incl, off);
      if (lane >= off) incl += v;
    }
    if (lane == 31) scan[warp] = incl;
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    int64_t total = 0, before = incl - mine;
    for (int w = 0; w < kThreadsTc / 32; ++w) {
      if (w < warp) before += scan[w];
      total += scan[w];
    }
    const int nc = static_cast<int>(min(static_cast<int64_t>(gridDim.x), a.whole ? total : (total + kMinTiles - 1) / kMinTiles));
    if (cta >= nc) {  // nothing for this CTA (the same for all its threads)
      if (tid == 0) records[cta] = Record{0, total, -1, 0, 0, -1, 0, nc};
      if (warp == 1) tmem_dealloc(*tmem_base_s, L::kTmemCols);
      return;
    }
    // Tile x lies in one thread's sequences; a.whole moves both ends on to the next beginning
    // of an item.
    const int64_t lo = total * cta / nc, hi = total * (cta + 1) / nc;
    auto locate = [&](int64_t x, bool first) {
      if (x < before || x >= before + mine) return;
      int64_t at = before;
      for (int64_t b = b_lo; b < b_hi; ++b) {
        if (share > 1) read_seq(a, b, &s);
        int items;
        const int64_t head = head_tiles(a, s, per, &items), n = a.hkv * head;
        if (x < at + n) {
          const int64_t on = a.whole ? to_next_item(a, s, x - at, head, per) : 0;
          if (first) {
            plan->lo = x + on;
            plan->b = b;
            plan->off = x - at + on;
            plan->s = s;
          } else {
            plan->hi = x + on;
          }
          return;
        }
        at += n;
      }
    };
    locate(lo, true);
    locate(hi, false);
    if (tid == 0 && hi == total) plan->hi = total;
    __syncthreads();
    plan_total = total;
    plan_nc = nc;
    if (plan->lo >= plan->hi) {  // another CTA's item fills the whole range
      if (tid == 0) records[cta] = Record{0, total, -1, 0, 0, -1, 0, nc};
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
    float2* ml = reinterpret_cast<float2*>(smem + L::kOffMl);
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
                if (bad) see &= sound32(bad, at / 32, a.box);
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

      // The segment's end: sums out of TMEM, to out (whole item) or to a partial.
      const bool whole = walk.t == 0 && n == walk.tiles;
      float* slot = slots + (2 * static_cast<int64_t>(cta) + (seg > 0)) * L::kSlotFloats;
      const int end = x + units;
      const int h = r - (r / a.group) * a.group;
      bf16* out = static_cast<bf16*>(a.out) + ((s.row0 + token) * a.hq + walk.kvh * a.group + h) * a.hd;
      if constexpr (DUAL) {
        warp_wait(&pvdone[w], ((end - 2 + w) >> 1) & 1, abort_flag, a.status);
        tc_fence_after();
        const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;
        if (warp_live) {
#pragma unroll
          for (int c = 0; c < HD / 32; ++c) {
            uint32_t v[32];
            tmem_load32(o_addr + 32 * c, v);
            tmem_wait_ld();
            if (r < live) {
              if (whole) {
#pragma unroll
                for (int e = 0; e < 32; e += 8) {
                  float f[8];
#pragma unroll
                  for (int d = 0; d < 8; ++d) f[d] = __uint_as_float(v[e + d]) * inv;
                  if (32 * c + e < a.hd) st_plain(out + 32 * c + e, pack16<bf16>(f));
                }
              } else {
                float* dst = slot + (w * kTile + r) * HD + 32 * c;
#pragma unroll
                for (int e = 0; e < 32; e += 4) st_plain(dst + e, make_uint4(v[e], v[e + 1], v[e + 2], v[e + 3]));
              }
            }
          }
          if (!whole && r < live) {
            slot[L::kRows * HD + w * kTile + r] = m;
            slot[L::kRows * (HD + 1) + w * kTile + r] = l;
          }
        }
      } else if constexpr (L::kCopies > 1) {
        // maxima and sums of every group and copy, then their sums of values in shared memory
        ml[((seg & 1) * 2 + w) * kTile + copy * L::kCopyRows + r] = make_float2(m, l);
        both_groups_sync();
        float top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int i = 0; i < L::kWriters; ++i) {
          top = fmaxf(top, ml[((seg & 1) * 2 + i / L::kCopies) * kTile + i % L::kCopies * L::kCopyRows + r].x);
        }
        const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int i = 0; i < L::kWriters; ++i) {
          const float2 part = ml[((seg & 1) * 2 + i / L::kCopies) * kTile + i % L::kCopies * L::kCopyRows + r];
          sum = fmaf(part.y, ex2(part.x - base), sum);  // a maximum of -inf: 0
        }
        const float inv = !whole ? 1.f : sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;
        const int last = end - 1 - ((end - 1 - w) & 1);  // this group's last unit; none: its O is stale
        const bool had = last >= x && warp_live;
        if (last >= x) warp_wait(&pvdone[w], (last >> 1) & 1, abort_flag, a.status);
        tc_fence_after();
        const float f = m == -INFINITY || r >= live ? 0.f : ex2(m - base) * inv;
        float* acc = reinterpret_cast<float*>(smem + L::kOffSum);
        for (int d0 = 0; d0 < HD; d0 += L::kDims) {
#pragma unroll 1
          for (int step = 0; step < L::kWriters; ++step) {
            const int col = (w * L::kCopies + copy + step) % L::kWriters * L::kStep;
            uint32_t o[16];
            if (had) {  // the same for the warp
              if constexpr (L::kStep == 16) {
                tmem_load16(o_addr + d0 + col, o);
              } else {
                tmem_load8(o_addr + d0 + col, o);
              }
              tmem_wait_ld();
            }
            float* to = acc + r * L::kPitch + col;
#pragma unroll
            for (int e = 0; e < L::kStep; e += 4) {
              float4 add = make_float4(0.f, 0.f, 0.f, 0.f);
              if (had && f != 0.f) {
                add = make_float4(__uint_as_float(o[e]) * f, __uint_as_float(o[e + 1]) * f, __uint_as_float(o[e + 2]) * f,
                                  __uint_as_float(o[e + 3]) * f);
              }
              if (step > 0) {
                const float4 old = *reinterpret_cast<const float4*>(to + e);
                add = make_float4(add.x + old.x, add.y + old.y, add.z + old.z, add.w + old.w);
              }
              *reinterpret_cast<float4*>(to + e) = add;
            }
            __syncwarp();
            both_groups_sync();
          }
          for (int c = tid - 128; c < live * (L::kDims / 8); c += 256) {
            const int row = c / (L::kDims / 8), d = c % (L::kDims / 8) * 8;
            const float* from = acc + row * L::kPitch + d;
            if (whole) {
              const int tok = i0 + row / a.group, head = row % a.group;
              float f8[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) f8[e] = from[e];
              if (d0 + d < a.hd) {
                st_plain(static_cast<bf16*>(a.out) + ((s.row0 + tok) * a.hq + walk.kvh * a.group + head) * a.hd + d0 + d, pack16<bf16>(f8));
              }
            } else {
              float* to = slot + row * HD + d0 + d;
              *reinterpret_cast<float4*>(to) = *reinterpret_cast<const float4*>(from);
              *reinterpret_cast<float4*>(to + 4) = *reinterpret_cast<const float4*>(from + 4);
            }
          }
          __syncwarp();
          both_groups_sync();  // the sums have been read
        }
        if (!whole && w == 0 && copy == 0 && r < live) {
          slot[L::kRows * HD + r] = top;
          slot[L::kRows * (HD + 1) + r] = sum;
        }
      } else {
        // both groups' maxima and sums, then each takes half of the dims of both
        ml[((seg & 1) * 2 + w) * kTile + r] = make_float2(m, l);
        both_groups_sync();
        const float2 other = ml[((seg & 1) * 2 + (w ^ 1)) * kTile + r];
        const int last0 = end - 1 - ((end - 1) & 1), last1 = end - 1 - (~(end - 1) & 1);  // last units of groups 0, 1
        if (last0 >= x) warp_wait(&pvdone[0], (last0 >> 1) & 1, abort_flag, a.status);
        if (last1 >= x) warp_wait(&pvdone[1], (last1 >> 1) & 1, abort_flag, a.status);
        tc_fence_after();
        if (warp_live) {
          const float top = fmaxf(m, other.x), base = top == -INFINITY ? 0.f : top;
          const float own_f = m == -INFINITY ? 0.f : ex2(m - base), other_f = other.x == -INFINITY ? 0.f : ex2(other.x - base);
          const float sum = l * own_f + other.y * other_f;
          const float inv = !whole ? 1.f : sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;
          const float f0 = (w == 0 ? own_f : other_f) * inv, f1 = (w == 0 ? other_f : own_f) * inv;
          const bool two = last0 >= x && last1 >= x;  // otherwise one group had no unit and its O is stale
#pragma unroll
          for (int c = 0; c < HD / 64; ++c) {
            const int col = w * (HD / 2) + 32 * c;
            uint32_t v[32];
            float f[32];
            tmem_load32(tmem + lane_addr + L::kColO + (last0 >= x ? 0 : HD) + col, v);
            tmem_wait_ld();
            const float fa = last0 >= x ? f0 : f1;
#pragma unroll
            for (int e = 0; e < 32; ++e) f[e] = fa == 0.f ? 0.f : __uint_as_float(v[e]) * fa;
            if (two) {
              tmem_load32(tmem + lane_addr + L::kColO + HD + col, v);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 32; ++e) f[e] = f1 == 0.f ? f[e] : fmaf(__uint_as_float(v[e]), f1, f[e]);
            }
            if (r < live) {
              if (whole) {
#pragma unroll
                for (int e = 0; e < 32; e += 8) {
                  if (col + e < a.hd) st_plain(out + col + e, pack16<bf16>(f + e));
                }
              } else {
                float* dst = slot + r * HD + col;
#pragma unroll
                for (int e = 0; e < 32; e += 4) *reinterpret_cast<float4*>(dst + e) = make_float4(f[e], f[e + 1], f[e + 2], f[e + 3]);
              }
            }
          }
          if (!whole && w == 0 && r < live) {
            slot[L::kRows * HD + r] = top;
            slot[L::kRows * (HD + 1) + r] = sum;
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(ofree);
      x = end;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, L::kTmemCols);
  }
}

// Adds up the partials of the item that CTA k's first tile continues: block (k, rows
// 8 y .. 8 y + 7, and so on) by the first border inside the item. A warp takes a row, its halves
// every other part: an item of few rows and many parts is bound by the latency of the
// parts' loads, so many are in flight over many SMs.
template <int HD, int COPIES>
__global__ void __launch_bounds__(256) tree_merge_kernel(const TreeArgs a, int ctas) {
  grid_dependency_wait();
  using L = Layout<HD, COPIES>;
  const Record* records = reinterpret_cast<const Record*>(a.ws);
  const float* slots = a.ws + records_bytes(ctas) / sizeof(float);
  const int k = static_cast<int>(blockIdx.x) + 1;
  const Record rec = records[k];
  if (rec.t0 <= 0) return;  // no tiles, or its first tile begins an item
  const int64_t first = rec.lo - rec.t0;  // the item's first tile
  auto border = [&](int c) { return rec.total * c / rec.nc; };
  if (border(k - 1) > first) return;  // an earlier border is inside it, too
  Seq s;
  read_seq(a, rec.b, &s);
  const int tpt = L::kCopyRows / a.group;
  constexpr int kLanes = 16;  // threads of a part's row
  const int lane = threadIdx.x & 31;
  // one past the last CTA with a part: the one that holds the item's last tile
  const int last = static_cast<int>(((first + rec.tiles) * rec.nc - 1) / rec.total) + 1;
  const int skip = border(k - 1) != first;  // in the first CTA the item is not the first segment
  auto part = [&](int c) { return slots + (2 * static_cast<int64_t>(c) + (c == k - 1 ? skip : 0)) * L::kSlotFloats; };
  for (int r = static_cast<int>(blockIdx.y) * 8 + threadIdx.x / 32; r < L::kRows; r += 8 * gridDim.y) {
    const int tile = r / kTile, rr = r - tile * kTile;
    const int i0 = rec.p * tpt * L::kTiles + tile * tpt;
    if (rr >= max(0, min(tpt, s.n - i0)) * a.group) continue;
    // the first parts' maxima, sums and values at once: two parts are all there is, mostly
    constexpr int kDims = HD / kLanes;  // 4 or 8 dims of a thread
    const int d = lane % kLanes * kDims, half = lane / kLanes;
    auto values = [&](int c, int e) { return *reinterpret_cast<const float4*>(part(min(c, last - 1)) + r * HD + d + e); };
    const bool own = k - 1 + lane < last;
    const float own_m = own ? part(k - 1 + lane)[L::kRows * HD + r] : -INFINITY;
    const float own_l = own ? part(k - 1 + lane)[L::kRows * (HD + 1) + r] : 0.f;
    float4 own_v[kDims / 4];
#pragma unroll
    for (int e = 0; e < kDims; e += 4) own_v[e / 4] = values(k - 1 + half, e);
    float m = own_m;
    for (int c = k - 1 + lane + 32; c < last; c += 32) m = fmaxf(m, part(c)[L::kRows * HD + r]);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
    const float base = m == -INFINITY ? 0.f : m;
    float l = 0.f, o[kDims];
#pragma unroll
    for (int e = 0; e < kDims; ++e) o[e] = 0.f;
    auto add = [&](const float4& v, float w, int e) {
      o[e] = fmaf(v.x, w, o[e]);
      o[e + 1] = fmaf(v.y, w, o[e + 1]);
      o[e + 2] = fmaf(v.z, w, o[e + 2]);
      o[e + 3] = fmaf(v.w, w, o[e + 3]);
    };
    for (int c0 = k - 1; c0 < last; c0 += 32) {
      float f = 0.f;  // of part c0 + lane
      if (c0 == k - 1) {
        f = ex2(own_m - base);
        l = own_l * f;
      } else if (c0 + lane < last) {
        f = ex2(part(c0 + lane)[L::kRows * HD + r] - base);
        l = fmaf(part(c0 + lane)[L::kRows * (HD + 1) + r], f, l);
      }
      const int n = min(32, last - c0);
      int i = half;
      if (c0 == k - 1) {
        const float w = __shfl_sync(0xffffffffu, f, i);  // past n: 0
#pragma unroll
        for (int e = 0; e < kDims; e += 4) add(own_v[e / 4], w, e);
        i += 2;
      }
#pragma unroll 8
      for (; i < n + half; i += 2) {
        const float w = __shfl_sync(0xffffffffu, f, i & 31);
#pragma unroll
        for (int e = 0; e < kDims; e += 4) add(values(c0 + i, e), w, e);
      }
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
#pragma unroll
    for (int e = 0; e < kDims; ++e) o[e] += __shfl_xor_sync(0xffffffffu, o[e], 16);
    if (half != 0) continue;
    const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;
    const int token = i0 + rr / a.group, h = rr - (rr / a.group) * a.group;
    if (d >= a.hd) continue;
    bf16* out = static_cast<bf16*>(a.out) + ((s.row0 + token) * a.hq + rec.kvh * a.group + h) * a.hd + d;
#pragma unroll
    for (int e = 0; e < kDims; e += 4) {  // head_dim is a multiple of 8
      *reinterpret_cast<uint2*>(out + e) = make_uint2(pack_bf16x2(o[e] * inv, o[e + 1] * inv),
                                                      pack_bf16x2(o[e + 2] * inv, o[e + 3] * inv));
    }
  }
}

// The form for the bounds' rows per kv head: the widest that holds them in one item, else
// two row tiles.
int copies_for(int group, int max_tree) {
  const int64_t rows = static_cast<int64_t>(group) * max_tree;
  return rows <= 32 ? 4 : rows <= 64 ? 2 : rows <= kTile / group * group ? 1 : kDual;
}
int rows_of(int copies) { return copies == kDual ? 2 * kTile : kTile / copies; }
int tokens_of(int copies, int group) { return copies == kDual ? kTile / group * 2 : kTile / copies / group; }

// Slots of a tile and rows of the boxes that fill it: whole pages or equal parts of one,
// so that a box never crosses a page, at 1024-byte steps of shared memory unless there is
// one. A tile below half full is left to the CUDA cores.
bool tile_of(int page_size, int* tile, int* box) {
  if (page_size <= kTile) {
    const int n = page_size % 8 == 0 ? kTile / page_size : 1;
    *box = page_size;
    *tile = n * page_size;
  } else {
    int parts = (page_size + kTile - 1) / kTile;
    while (page_size % parts != 0) ++parts;  // ends at parts = page_size
    *box = *tile = page_size / parts;
  }
  return *tile >= kTile / 2;
}

// CTAs for the bounds: one per SM, no more than the tiles there can be (a tile holds at
// least half of 128 slots).
int ctas_for(int64_t batch, int hkv, int group, int max_ctx, int max_tree) {
  const int per = tokens_of(copies_for(group, max_tree), group);
  const int64_t tiles = batch * hkv * ((max_tree + per - 1) / per) *
                        ((static_cast<int64_t>(max_ctx) + max_tree + kTile / 2 - 1) / (kTile / 2));
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(sm_count(), tiles)));
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
  // Whole items up to kWholeTiles tiles where they make CTAs for a quarter of the SMs or more
  // (80 items of 5 tiles: 15.9 us, cut 18.6), else up to half of that (8 items of 8: 18.7,
  // cut 15.8).
  const int per = tokens_of(COPIES, a.group);
  const int64_t items = a.batch * a.hkv * ((a.max_tree + per - 1) / per);
  a.whole = a.max_ctx + a.max_tree <= (4 * items >= sm_count() ? kWholeTiles : kWholeTiles / 2) * a.tile;
  const int nc = ctas_for(a.batch, a.hkv, a.group, a.max_ctx, a.max_tree);
  if (int st = launch_kernel(what, kernel, dim3(nc), dim3(kThreadsTc), L::kBytes, stream, nullptr, tq, tk, tv, a)) return st;
  if (nc == 1 || a.whole) return BM_OK;  // no item is cut
  return launch_kernel(what, tree_merge_kernel<HD, COPIES>, dim3(nc - 1, std::min(L::kRows / 8, 8)), dim3(256), 0, stream, nullptr, a, nc);
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
