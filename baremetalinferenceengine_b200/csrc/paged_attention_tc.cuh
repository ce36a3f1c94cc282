// Pieces that the tensor-core forms of the paged tree attention have in common
// (paged_attention_tc.cu, paged_attention8_tc.cu): how an item's rows lie in row tiles, the
// plan that shares tiles out over CTAs and the walk over a CTA's part of it, masks, the end
// of a segment and the merge of partials.
#pragma once

#include <algorithm>

#include "bm_tc.cuh"
#include "bm_tma.h"
#include "paged_attention.cuh"

namespace bm {
namespace paged {

using namespace bm::tc;

constexpr int kTile = 128;      // slots per tile, rows per row tile
constexpr int kThreadsTc = 384;
constexpr int kMinTiles = 2;    // places (tiles, and items' costs) that make a CTA worth starting, where items are cut
constexpr int kWholeTiles = 8;  // of the longest item, up to which items stay whole
constexpr int kBadRing = 16;    // tiles whose bad-page bits are kept
constexpr uint64_t kWaitNs = 2000000000ull;
constexpr uint64_t kDrainNs = 200000000ull;

// How an item's rows lie in row tiles: two tiles of rows, or one holding them COPIES times.
constexpr int kDual = 0;

template <int HD, int COPIES>
struct RowLayout {
  static constexpr bool kTwo = COPIES == kDual;
  static constexpr int kTiles = kTwo ? 2 : 1;               // row tiles of an item
  static constexpr int kCopies = kTwo ? 1 : COPIES;
  static constexpr int kCopyRows = kTile / kCopies;         // rows of a copy
  static constexpr int kCols = kTile / kCopies;             // slots of a tile that a copy weighs
  static constexpr int kRows = kTiles * kCopyRows;          // rows of an item
  // The copies' sums meet in shared memory, kDims dims of all rows at a time, each of the
  // kWriters (group, copy) adding its own kStep dims in turn.
  static constexpr int kWriters = 2 * kCopies;  // (unused with one copy)
  static constexpr int kDims = 4096 / kCopyRows < HD ? 4096 / kCopyRows : HD;
  static constexpr int kStep = kDims / kWriters;
  static constexpr int kPitch = kDims + 4;
  static constexpr int kMlBytes = kTwo ? 0 : 2 * 2 * kTile * 8;  // [2][2][128] (maximum, sum)
  static constexpr int kSumBytes = kCopies > 1 ? kCopyRows * kPitch * 4 : 0;
  static constexpr uint32_t kColO = 256;                    // TMEM: S0, S1 (128 each), O0, O1 (HD each)
  static constexpr uint32_t kTmemCols = 512;
  static constexpr int kSlotFloats = kRows * (HD + 2);      // a partial: sums, then maxima, then weight sums
};

// CTAs share out places: a.item_cost of them for each item, ahead of one for each of its tiles.

// What a CTA left of its first segment, for the merge.
struct Record {
  int64_t lo, total;   // its first place, and all places
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
// Its places.
__device__ __forceinline__ int item_places(const TreeArgs& a, const Seq& s, int p, int per) { return a.item_cost + item_tiles(a, s, p, per); }
// All places of one kv head of a sequence, and its items.
__device__ __forceinline__ int64_t head_places(const TreeArgs& a, const Seq& s, int per, int* items) {
  *items = (s.n + per - 1) / per;
  if (a.mask) return static_cast<int64_t>(*items) * item_places(a, s, 0, per);
  int64_t t = 0;
  for (int p = 0; p < *items; ++p) t += item_places(a, s, p, per);
  return t;
}

// From place `off` of a sequence to where a CTA's part may begin or end: back to an item's beginning
// from the places ahead of its first tile; with a.whole on to the next beginning. 0: it may here.
__device__ __forceinline__ int64_t to_border(const TreeArgs& a, const Seq& s, int64_t off, int64_t head, int per) {
  off %= head;
  for (int p = 0;; ++p) {
    const int places = item_places(a, s, p, per);
    if (off < places) return off == 0 ? 0 : a.whole ? places - off : off <= a.item_cost ? -off : 0;
    off -= places;
  }
}

// The walk over a CTA's segments: every role runs its own, with the same results.
struct Walk {
  int64_t b, left;                // places left
  int items, kvh, p, t, tiles;
  Seq s;

  // Place `off` of sequence b is the CTA's first, and `n` places are its own.
  __device__ void start(const TreeArgs& a, const Seq& sequence, int64_t b0, int64_t off, int64_t n, int per) {
    b = b0;
    left = n;
    s = sequence;
    int64_t head = head_places(a, s, per, &items);
    if (off >= a.hkv * head) {  // behind the sequence's last item: the next one with tiles
      do {
        ++b;
        read_seq(a, b, &s);
      } while (s.n == 0);
      head = head_places(a, s, per, &items);
      off = 0;
    }
    kvh = static_cast<int>(off / head);
    off -= kvh * head;
    p = 0;
    while (off >= (tiles = item_places(a, s, p, per))) {
      off -= tiles;
      ++p;
    }
    tiles -= a.item_cost;
    t = static_cast<int>(off);
    if (t == 0) {
      left -= a.item_cost;
    } else {
      t -= a.item_cost;  // behind the places ahead of its first tile
    }
  }
  // Tiles of the current segment (0 when the walk is over).
  __device__ int segment() const { return static_cast<int>(left < tiles - t ? left : tiles - t); }
  __device__ void next(const TreeArgs& a, int per) {
    left -= segment();
    if (left == 0) return;
    left -= a.item_cost;
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
  int64_t lo, hi, b, off;  // this CTA's places; the first is place `off` of sequence b
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

// Which of the 32 slots from slot `at` of a tile on have a sound page (bit b of bad: the
// tile's box b has not). Two boxes or more hold whole groups of 8 slots each.
__device__ __forceinline__ uint32_t sound32(uint32_t bad, int at, int box_rows) {
  uint32_t v = 0xffffffffu;
  for (int e = 0; e < 32; e += 8) {
    if ((bad >> min((at + e) / box_rows, 31)) & 1) v &= ~(0xffu << e);
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

// Shares the places of the batch out: this CTA's into *plan, and the number of all places and
// of the CTAs that have some. False (with the CTA's empty record written) where it has none.
// All threads of the CTA call it; barriers and TMEM that they set up before are visible behind it.
__device__ __forceinline__ bool plan_share(const TreeArgs& a, int per, int64_t* scan, Plan* plan, Record* records, int64_t* total_out,
                                           int* nc_out) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, cta = static_cast<int>(blockIdx.x);
  const int64_t share = (a.batch + kThreadsTc - 1) / kThreadsTc;
  const int64_t b_lo = min(a.batch, tid * share), b_hi = min(a.batch, b_lo + share);
  int64_t mine = 0;
  Seq s;
  for (int64_t b = b_lo; b < b_hi; ++b) {
    const int32_t bad = read_seq(a, b, &s);
    if (bad && cta == 0) raise_status(a.status, bad);
    int items;
    mine += a.hkv * head_places(a, s, per, &items);
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
    return false;
  }
  // Place x lies in one thread's sequences.
  const int64_t lo = total * cta / nc, hi = total * (cta + 1) / nc;
  auto locate = [&](int64_t x, bool first) {
    if (x < before || x >= before + mine) return;
    int64_t at = before;
    for (int64_t b = b_lo; b < b_hi; ++b) {
      if (share > 1) read_seq(a, b, &s);
      int items;
      const int64_t head = head_places(a, s, per, &items), n = a.hkv * head;
      if (x < at + n) {
        const int64_t on = a.whole || a.item_cost > 0 ? to_border(a, s, x - at, head, per) : 0;
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
  *total_out = total;
  *nc_out = nc;
  if (plan->lo < plan->hi) return true;
  if (tid == 0) records[cta] = Record{0, total, -1, 0, 0, -1, 0, nc};  // another CTA's item fills the whole range
  return false;
}

// A segment's end, by the softmax threads: sums out of TMEM, to out (whole item) or to a
// partial. Group w's thread for row r of the row tile (and copy) has the running maximum m and sum
// l of its units; had0 and had1 tell which groups had some (O of the other is stale), and their mixes are
// done. L is the kernel's layout.
template <typename L, int HD>
__device__ __forceinline__ void finish_segment(const TreeArgs& a, unsigned char* smem, const Walk& walk, const Seq& s, float* slots,
                                               uint32_t tmem, int w, int copy, int r, bool had0, bool had1, int seg, int i0,
                                               int live, float m, float l) {
  const int tid = threadIdx.x, lane = tid & 31, quarter = (tid >> 5) & 3;
  const bool warp_live = r - lane < live;
  const int token = i0 + r / a.group;
  const uint32_t lane_addr = static_cast<uint32_t>(quarter * 32) << 16;
  const uint32_t o_addr = tmem + lane_addr + L::kColO + w * HD;
  float2* ml = reinterpret_cast<float2*>(smem + L::kOffMl);
  const bool whole = walk.t == 0 && walk.segment() == walk.tiles;
  float* slot = slots + (2 * static_cast<int64_t>(blockIdx.x) + (seg > 0)) * L::kSlotFloats;
  const int h = r - (r / a.group) * a.group;
  bf16* out = static_cast<bf16*>(a.out) + ((s.row0 + token) * a.hq + walk.kvh * a.group + h) * a.hd;
  if constexpr (L::kTwo) {
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
    const bool had = (w == 0 ? had0 : had1) && warp_live;
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
    if (warp_live) {
      const float top = fmaxf(m, other.x), base = top == -INFINITY ? 0.f : top;
      const float own_f = m == -INFINITY ? 0.f : ex2(m - base), other_f = other.x == -INFINITY ? 0.f : ex2(other.x - base);
      const float sum = l * own_f + other.y * other_f;
      const float inv = !whole ? 1.f : sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;
      const float f0 = (w == 0 ? own_f : other_f) * inv, f1 = (w == 0 ? other_f : own_f) * inv;
      const bool two = had0 && had1;
#pragma unroll
      for (int c = 0; c < HD / 64; ++c) {
        const int col = w * (HD / 2) + 32 * c;
        uint32_t v[32];
        float f[32];
        tmem_load32(tmem + lane_addr + L::kColO + (had0 ? 0 : HD) + col, v);
        tmem_wait_ld();
        const float fa = had0 ? f0 : f1;
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
}

// Adds up the partials of the item that CTA k's first tile continues: block (k, rows
// 8 y .. 8 y + 7, and so on) by the first border inside the item. A warp takes a row, its halves
// every other part: an item of few rows and many parts is bound by the latency of the
// parts' loads, so many are in flight over many SMs.
template <typename L, int HD>
__global__ void __launch_bounds__(256) tree_merge_kernel(const TreeArgs a, int ctas) {
  grid_dependency_wait();
  const Record* records = reinterpret_cast<const Record*>(a.ws);
  const float* slots = a.ws + records_bytes(ctas) / sizeof(float);
  const int k = static_cast<int>(blockIdx.x) + 1;
  const Record rec = records[k];
  if (rec.t0 <= 0) return;  // no tiles, or its first tile begins an item
  const int64_t first = rec.lo - rec.t0;  // the place of the item's first tile
  const int64_t begin = first - a.item_cost;
  auto border = [&](int c) { return rec.total * c / rec.nc; };
  if (border(k - 1) > first) return;  // an earlier border is inside it, too
  Seq s;
  read_seq(a, rec.b, &s);
  const int tpt = L::kCopyRows / a.group;
  constexpr int kLanes = 16;  // threads of a part's row
  const int lane = threadIdx.x & 31;
  // one past the last CTA with a part: the one that holds the item's last tile
  const int last = static_cast<int>(((first + rec.tiles) * rec.nc - 1) / rec.total) + 1;
  const int skip = border(k - 1) < begin;  // in the first CTA the item is not the first segment
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
inline int copies_for(int group, int max_tree) {
  const int64_t rows = static_cast<int64_t>(group) * max_tree;
  return rows <= 32 ? 4 : rows <= 64 ? 2 : rows <= kTile / group * group ? 1 : kDual;
}
inline int rows_of(int copies) { return copies == kDual ? 2 * kTile : kTile / copies; }
inline int tokens_of(int copies, int group) { return copies == kDual ? kTile / group * 2 : kTile / copies / group; }

// Slots of a tile and rows of the boxes that fill it: whole pages or equal parts of one,
// so that a box never crosses a page, at 1024-byte steps of shared memory unless there is
// one. A tile below half full is left to the CUDA cores.
inline bool tile_of(int page_size, int* tile, int* box) {
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
inline int ctas_for(int64_t batch, int hkv, int group, int max_ctx, int max_tree) {
  const int per = tokens_of(copies_for(group, max_tree), group);
  const int64_t tiles = batch * hkv * ((max_tree + per - 1) / per) *
                        ((static_cast<int64_t>(max_ctx) + max_tree + kTile / 2 - 1) / (kTile / 2));
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(sm_count(), tiles)));
}

// Whole items up to kWholeTiles tiles where they make CTAs for a quarter of the SMs or more
// (80 items of 5 tiles: 15.9 us, cut 18.6), else up to half of that (8 items of 8: 18.7,
// cut 15.8).
inline bool whole_items(const TreeArgs& a, int per) {
  const int64_t items = a.batch * a.hkv * ((a.max_tree + per - 1) / per);
  return a.max_ctx + a.max_tree <= (4 * items >= sm_count() ? kWholeTiles : kWholeTiles / 2) * a.tile;
}

}  // namespace paged
}  // namespace bm
