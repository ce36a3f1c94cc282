// Sampling one token per row of logits with temperature, top-k, top-p and min-p, from
// given uniform numbers (bm_sample).
//
// Mathematics: w_i = exp((x_i - max x) / T). Ordered by (x descending, index ascending),
// top-k, top-p and min-p each keep a beginning of the row, so what stays is described
// by a key t and an index e: every logit above t and those equal to it up to index e.
// The token is the first index whose running weight passes u times the total.
//
// Exactness: a token is a whole number, so a rounding next to a border changes the
// answer. Weights are 64-bit fixed point, 2^bits for the largest with 2^bits * vocab <=
// 2^62, rounded once from fp64; every sum that decides is an integer sum, the same in any
// order, and p * sum and u * sum are compared exactly. The fp64 2^-y is table-driven (the
// method of Tang, ACM TOMS 15, 1989): y = (j + r) / 128, a table of 2^(-j/128) and a
// polynomial of degree 4 in r, off by less than 2^-49 of the weight.
//
// Bound: a row is read from HBM once (the passes below find it in L2), so bytes count
// only for many rows; there the fp64 operations (eleven a logit where all weigh) cost as
// much, and one or few rows are bound by the chain of passes. Measured on a B200, calls one
// after the other on changing rows: with top-p alone 9 to 21 us for one fp32 row of 32000 (by
// the row), 22 for one of 128256 and 202 for 256 bf16 rows of 128256 (floor 10; 100 without
// a filter, 85 with top-k alone, 17 at temperature 0); all settings mixed by row, fp32: 19 us for
// 8 rows of 128256, 55 for 64 (floor 5). A row of up to 1024 logits stays in one CTA's
// registers (11 us for 64 rows of 1000, 22 with the passes; 18 for 256). A cluster of up to 8 CTAs
// shares a longer row:
//   1. the largest logit and its first index;
//   2. for a small top-k: the logits that reach the k-th largest of the maxima of 512 or
//      1024 parts of the row, which one CTA then finishes alone. For others, first top-k,
//      then top-p: a histogram over 4096 bins of equal ratio of weight, in
//      32-bit counts (top-k) or fixed-point fp32 weights (top-p; shared-memory atomics
//      on 64 bits are many times slower). Each CTA adds up a slice of the bins over the
//      cluster. The bins that can hold the border are one or, with the fp32 weights'
//      error bounds, few; the next pass sums the exact weights (over the row and above
//      these bins) and collects their logits, which the leader splits by the bits of
//      their keys down to t. More than 1024 of them (rows of almost equal logits) are
//      split by the whole cluster first;
//   3. the weights of what stays, by stretches of the row in index order (known from
//      2. but for the collected logits); the stretch that holds u * total is walked.
#include <cooperative_groups.h>

#include <algorithm>

#include "bm_common.cuh"
#include "bm_host.h"

namespace bm {
namespace {

namespace cg = cooperative_groups;

using u64 = unsigned long long;

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;
constexpr int kBins = 4096;
constexpr int kCoarse = kBins / 64;
constexpr int kList = 1024;  // logits of the border's bins that are collected
constexpr double kLog2e = 1.4426950408889634074;

struct SampleArgs {
  int32_t* tokens;
  const void* logits;
  const float* uniforms;
  const float* temperature;
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  int64_t rows, stride;
  int vocab;
  int bits;   // the largest weight is 2^bits
  int chunk;  // logits of a row per CTA of the cluster
  int unit;   // bits of a fp32 weight in the histogram: chunk * 2^unit * 129 / 128 < 2^32
  bool vec;   // rows are 16-byte aligned
  int32_t* status;
};

// Keys order as the logits do: -inf (and NaN) lowest, -0 and +0 alike.
__device__ __forceinline__ uint32_t key_of(float x) {
  if (x != x) x = -INFINITY;
  const uint32_t u = __float_as_uint(x + 0.f);
  return u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float logit_of(uint32_t key) {
  return __uint_as_float(key ^ (key >> 31 ? 0x80000000u : 0xffffffffu));
}

// A finite fp32 value in fp64 by its bits: the conversion instruction runs at a quarter
// of the fp64 units' rate. What is below 2^-126 comes out as 2^-126 at most, which is
// nothing beside a temperature of 2^-60 or more.
__device__ __forceinline__ double widen(float x) {
  const int u = __float_as_int(x);
  return __hiloint2double(((u >> 3) & 0x8fffffff) + 0x38000000, u << 29);
}

// Weights of a row.
struct Weigher {
  double top;            // the largest logit (finite: see `remap`)
  double scale;          // 128 log2(e) / T
  double least;          // min_p in units of the weights
  const double* table;   // 2^(bits - j/128), j < 128
  float top_f, bins;     // bins of the histogram per logit

  // The weight's place in the histogram, from 0 at the largest logit; never falls as the
  // logit does. Below kLimit the weight may round to something; NaN for a NaN logit, and
  // for -inf at T = inf. Rounded here in every use: fused with the addition of kMagic in some
  // of them, a place half way between two bins would be now in one, now in the other.
  static constexpr float kLimit = kBins - 1.5f;
  __device__ __forceinline__ float place(float x) const { return __fmul_rn(top_f - x, bins); }
  // The weight before it is rounded to a whole number, for places below kLimit (anything
  // for others).
  __device__ __forceinline__ double real(float x) const {
    constexpr double kRound = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to a whole number
    constexpr double c1 = -0.69314718055994530942 / 128, c2 = c1 * c1 / 2, c3 = c1 * c2 / 3, c4 = c1 * c3 / 4;
    const double d = top - widen(x);
    const double shifted = fma(d, scale, kRound);
    const int j = __double2loint(shifted);
    const double r = fma(d, scale, kRound - shifted);
    double q = fma(r, c4, c3);
    q = fma(r, q, c2);
    q = fma(r, q, c1);
    q = fma(r, q, 1.0);
    const double w = q * table[j & 127];
    return __hiloint2double(__double2hiint(w) - ((j >> 7) << 20), __double2loint(w));
  }
  __device__ __forceinline__ static u64 whole(double w) {  // w < 2^52, rounded
    return static_cast<u64>(__double_as_longlong(w + 4503599627370496.0)) & 0xfffffffffffffull;
  }
  // A whole number that never rises as the logit falls, linear in it: kEven for the
  // largest, 0 for those without a weight.
  static constexpr uint32_t kEven = 1u << 31;
  __device__ __forceinline__ uint32_t even(float x) const {
    const float b = place(x);
    return b < kLimit ? kEven - static_cast<uint32_t>(b * 524288.f) : 0;
  }
  __device__ __forceinline__ u64 operator()(float x) const { return place(x) < kLimit ? whole(real(x)) : 0; }
};

// Of a row with this largest logit. Past bits + 2 octaves a weight rounds to 0.
__device__ __forceinline__ Weigher weigher(float top, float temperature, float min_p, int bits, const double* table) {
  const float bins_per_octave = Weigher::kLimit / static_cast<float>(bits + 2);
  const double per_logit = kLog2e / fmax(static_cast<double>(temperature), 0x1p-60);
  Weigher w;
  w.top_f = top;
  w.top = widen(top);
  w.scale = 128.0 * per_logit;
  w.least = exp2(static_cast<double>(bits)) * static_cast<double>(fminf(min_p, 1.f));
  w.table = table;
  w.bins = static_cast<float>(per_logit * static_cast<double>(bins_per_octave));
  return w;
}

// Adding it to 0 <= x < 2^22 rounds x to a whole number, in the sum's low bits.
constexpr float kMagic = 12582912.f;  // 1.5 * 2^23
__device__ __forceinline__ int bits_of(float magic_sum) { return __float_as_int(magic_sum) - 0x4b400000; }

struct Shared {
  union {
    uint32_t hist[kBins];
    u64 split[kThreads];   // of an interval of keys
  };
  double table[128];
  u64 coarse[kCoarse];     // the histogram by 64 bins
  u64 best[kMaxCluster];   // per CTA of the cluster: key << 32 | ~index
  u64 sum[kMaxCluster], above[kMaxCluster];
  u64 warp[kWarps], sub[kWarps];
  u64 before, through;     // value above the bin found, and up to its end
  u64 ties;                // how many logits equal to t stay
  u64 cand_weight[kList];  // the leader's: collected logits
  uint32_t cand_key[kList], cand_index[kList];
  uint32_t list_key[kList], list_index[kList];  // this CTA's share of them
  uint32_t own_count, offset;
  uint32_t count, key_min, key_max;             // the leader's: logits of the border's bins
  uint32_t bin_lo, bin_hi, bin;
  uint32_t members, member[32];                 // of the border's part of a split
  u64 member_value[32];
  uint32_t key;            // t
  uint32_t index;
  bool cut;                // not all logits equal to t stay
};

__device__ __forceinline__ u64 warp_sum64(u64 v) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  return v;
}
// The sum before this thread's v over the block's threads; *all: of all of them.
__device__ __forceinline__ u64 block_scan64(u64 v, u64* scratch, u64* all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  u64 incl = v;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const u64 o = __shfl_up_sync(0xffffffffu, incl, off);
    if (lane >= off) incl += o;
  }
  __syncthreads();
  if (lane == 31) scratch[warp] = incl;
  __syncthreads();
  u64 at = incl - v, s = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) at += scratch[w];
    s += scratch[w];
  }
  *all = s;
  return at;
}

// floor(f * s) and whether f * s has a fraction, f in [0, 1).
__device__ __forceinline__ u64 portion(float f, u64 s, bool* fraction) {
  const u64 f64 = static_cast<u64>(static_cast<double>(f) * 18446744073709551616.0);
  *fraction = f64 * s != 0;
  return __umul64hi(f64, s);
}

// In a row with +inf these are its largest logits and the others have no weight.
__device__ __forceinline__ float remapped(float x, bool remap) {
  return remap ? (x == INFINITY ? 0.f : -INFINITY) : x;
}

// The logits [lo, hi) of a row by one warp: f(index, logit), U 16-byte loads in flight
// per lane besides those being worked on. Lanes may call f a different number of times.
template <int U, typename T, typename F>
__device__ __forceinline__ void each(const T* x, int lo, int hi, bool vec, bool remap, F f) {
  constexpr int VEC = VecWidth<T>::value;
  const int lane = threadIdx.x & 31;
  if (!vec) {
    for (int i = lo + lane; i < hi; i += 32) f(i, remapped(load1(x + i), remap));
    return;
  }
  const int whole = lo + (hi - lo) / VEC * VEC;  // a multiple of VEC, as lo is
  uint4 next[U];
  auto fetch = [&](int i0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * 32 * VEC;
      if (i < whole) next[u] = __ldg(reinterpret_cast<const uint4*>(x + i));
    }
  };
  fetch(lo + lane * VEC);
  for (int i0 = lo + lane * VEC; i0 < whole; i0 += 32 * VEC * U) {
    uint4 raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u] = next[u];
    fetch(i0 + 32 * VEC * U);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * 32 * VEC;
      if (i < whole) {
        float v[VEC];
        unpack16<T>(raw[u], v);
        if (remap) {
#pragma unroll
          for (int e = 0; e < VEC; ++e) v[e] = remapped(v[e], true);
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) f(i + e, v[e]);
      }
    }
  }
  if (whole + lane < hi) f(whole + lane, remapped(load1(x + whole + lane), remap));  // fewer than VEC are left
}

// The border among the block's elements, kEach a thread, taken by descending `fine`: the
// fine of the first whose running value (equal ones together) reaches the target, and in
// *before the value above it. All values together reach the target; elements of value 0
// are none. `coarse` never rises where fine falls: the range that is left of it is split
// in 512 equal parts a round, so elements should lie evenly in it (64-bit shared-memory
// atomics on one address take turns). Up to 32 elements in the border's part are ranked by
// every warp alike; more that share one coarse are split by their fine.
constexpr int kEach = kList / kThreads;
__device__ uint32_t border(Shared& sh, const uint32_t (&coarse)[kEach], const uint32_t (&fine)[kEach],
                           const u64 (&value)[kEach], u64 target, u64* before) {
  const int tid = threadIdx.x, lane = tid & 31;
  u64 passed = 0;
  uint32_t from = 0, to = 0xffffffffu, fine_from = 0, fine_to = 0xffffffffu;
  bool by_fine = false;
  for (int round = 0; round < 10; ++round) {  // at most 4 by coarse, 5 by fine
    __syncthreads();
    sh.split[tid] = 0;
    if (tid == 0) {
      sh.members = 0;
      sh.key_min = 0xffffffffu;
      sh.key_max = 0;
    }
    __syncthreads();
    {  // the range that is left
      uint32_t mn = 0xffffffffu, mx = 0;
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        const uint32_t f = by_fine ? fine[e] : coarse[e];
        if (value[e] != 0 && coarse[e] >= from && coarse[e] <= to && fine[e] >= fine_from && fine[e] <= fine_to) {
          mn = min(mn, f);
          mx = max(mx, f);
        }
      }
      mn = __reduce_min_sync(0xffffffffu, mn);
      mx = __reduce_max_sync(0xffffffffu, mx);
      if (lane == 0) {
        atomicMin(&sh.key_min, mn);
        atomicMax(&sh.key_max, mx);
      }
      __syncthreads();
      if (by_fine) {
        fine_from = sh.key_min;
        fine_to = sh.key_max;
        if (fine_from >= fine_to) {
          *before = passed;
          return fine_to;
        }
      } else {
        from = sh.key_min;
        to = sh.key_max;
      }
    }
    const uint32_t range = by_fine ? fine_to - fine_from : to - from;
    const int shift = max(0, 32 - __clz(range) - 9);
    auto part = [&](int e) { return by_fine ? (fine_to - fine[e]) >> shift : (to - coarse[e]) >> shift; };
    auto within = [&](int e) {
      if (value[e] == 0) return false;
      return by_fine ? coarse[e] == to && fine[e] >= fine_from && fine[e] <= fine_to : coarse[e] >= from && coarse[e] <= to;
    };
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      if (within(e)) atomicAdd(&sh.split[part(e)], value[e]);
    }
    __syncthreads();
    const u64 v = sh.split[tid];
    u64 total;
    const u64 at = block_scan64(v, sh.sub, &total) + passed;
    if (at < target && target <= at + v) {
      sh.bin = tid;
      sh.before = at;
    }
    __syncthreads();
    passed = sh.before;
    const uint32_t bin = sh.bin;
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      if (within(e) && part(e) == bin) {
        const uint32_t n = atomicAdd(&sh.members, 1u);
        if (n < 32) {
          sh.member[n] = fine[e];
          sh.member_value[n] = value[e];
        }
      }
    }
    __syncthreads();
    if (sh.members <= 32) {
      const bool is = lane < static_cast<int>(sh.members);
      const uint32_t own = is ? sh.member[lane] : 0;
      const u64 worth = is ? sh.member_value[lane] : 0;
      u64 above = passed;
      for (int j = 0; j < static_cast<int>(sh.members); ++j) {
        if (sh.member[j] > own) above += sh.member_value[j];
      }
      // the lowest of those with less than the target above them
      const uint32_t found = __reduce_min_sync(0xffffffffu, worth != 0 && above < target ? own : 0xffffffffu);
      const int who = __ffs(__ballot_sync(0xffffffffu, is && own == found)) - 1;
      *before = __shfl_sync(0xffffffffu, above, who);
      return found;
    }
    if (by_fine) {
      fine_to -= bin << shift;
      if (shift < 31) fine_from = max(fine_from, fine_to - min(fine_to, (1u << shift) - 1));
    } else {
      to -= bin << shift;
      from = max(from, to - min(to, (1u << shift) - 1));
      by_fine = from == to;
    }
  }
  *before = passed;
  return fine_to;
}

// The rest of a row whose top-k logits are in the leader's list (some more may be), or all
// of whose logits are (k at least their number).
__device__ __noinline__ void finish_alone(Shared& sh, const SampleArgs& a, const Weigher& weigh, int k, float p, float u,
                                          int64_t row) {
  const int tid = threadIdx.x;
  const uint32_t n = sh.count;
  uint32_t key[kEach], even[kEach], later[kEach];  // even: as the logits lie; later: descends as the index rises
  u64 one[kEach], weight[kEach], before, all;
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const uint32_t i = tid + e * kThreads;
    key[e] = i < n ? sh.cand_key[i] : 0;
    even[e] = weigh.even(logit_of(key[e]));
    later[e] = i < n ? ~sh.cand_index[i] : 0;
    one[e] = i < n;
    weight[e] = i < n ? weigh(logit_of(key[e])) : 0;
  }
  // top-k, then top-p: a key, how many of those equal to it stay, and (if not all) the last
  for (int stage = 0; stage < 2; ++stage) {
    if (stage == 1 ? !(p < 1.f) : k >= static_cast<int>(n)) continue;
    u64 target = k;
    if (stage == 1) {
      u64 mine = 0;
#pragma unroll
      for (int e = 0; e < kEach; ++e) mine += weight[e];
      block_scan64(mine, sh.sub, &all);
      bool fraction;
      target = portion(fmaxf(p, 0.f), all, &fraction);
      if (fraction || target == 0) ++target;
    }
    const uint32_t t = border(sh, even, key, stage == 0 ? one : weight, target, &before);
    u64 tie[kEach], equal = 0;
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      tie[e] = one[e] != 0 && key[e] == t;
      equal += tie[e];
    }
    block_scan64(equal, sh.sub, &all);
    const u64 w = stage == 0 ? 1 : max(weigh(logit_of(t)), static_cast<u64>(1));
    const u64 rest = (target - before + w - 1) / w;
    uint32_t last = 0;  // of the `later` order: those below it go
    if (rest < all) last = border(sh, later, later, tie, rest, &before);
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      if (key[e] < t || (key[e] == t && later[e] < last)) one[e] = weight[e] = 0;
    }
  }
  u64 mine = 0;
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    if (weight[e] != 0 && weigh.real(logit_of(key[e])) < weigh.least) weight[e] = 0;  // min-p
    mine += weight[e];
  }
  block_scan64(mine, sh.sub, &all);
  bool fraction;
  const u64 want = portion(u, all, &fraction);
  const uint32_t token = ~border(sh, later, later, weight, want + 1, &before);
  if (tid == 0) a.tokens[row] = static_cast<int32_t>(token);
}

// A row of at most kList logits: one CTA holds it, and there is nothing to search for
// in memory.
template <typename T>
__global__ void __launch_bounds__(kThreads) sample_short_kernel(const SampleArgs a) {
  grid_dependency_wait();
  extern __shared__ __align__(16) unsigned char smem[];
  Shared& sh = *reinterpret_cast<Shared*>(smem);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(a.logits) + row * a.stride;
  float v[kEach];
  uint32_t most = 0;
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const int i = tid + e * kThreads;
    v[e] = i < a.vocab ? load1(x + i) : -INFINITY;
    most = max(most, key_of(v[e]));
  }
  const float temp = a.temperature ? a.temperature[row] : 1.f;
  const float u = a.uniforms[row];
  const int k = a.top_k ? a.top_k[row] : 0;
  const float p = a.top_p ? a.top_p[row] : 1.f;
  const float mp = a.min_p ? a.min_p[row] : 0.f;
  if (!(temp >= 0.f) || !(u >= 0.f && u < 1.f) || p != p || mp != mp) {
    if (tid == 0) {
      a.tokens[row] = -1;
      raise_status(a.status, BM_DEVERR_BAD_PARAMETER);
    }
    return;
  }
  most = __reduce_max_sync(0xffffffffu, most);
  if (lane == 0) sh.list_key[warp] = most;
  if (tid < 128) sh.table[tid] = exp2(static_cast<double>(a.bits) - tid / 128.0);
  if (tid == 0) sh.index = 0xffffffffu;
  __syncthreads();
  for (int w = 0; w < kWarps; ++w) most = max(most, sh.list_key[w]);
  const float top = logit_of(most);
  if (top == -INFINITY || temp == 0.f) {
    uint32_t first = 0xffffffffu;
#pragma unroll
    for (int e = kEach - 1; e >= 0; --e) {
      if (tid + e * kThreads < a.vocab && key_of(v[e]) == most) first = tid + e * kThreads;
    }
    first = __reduce_min_sync(0xffffffffu, first);
    if (lane == 0) atomicMin(&sh.index, first);
    __syncthreads();
    if (tid == 0) a.tokens[row] = top == -INFINITY ? -1 : static_cast<int32_t>(sh.index);
    return;
  }
  const bool remap = top == INFINITY;
  const Weigher weigh = weigher(remap ? 0.f : top, temp, mp, a.bits, sh.table);
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const int i = tid + e * kThreads;
    if (i < a.vocab) {
      sh.cand_key[i] = key_of(remapped(v[e], remap));
      sh.cand_index[i] = i;
    }
  }
  if (tid == 0) sh.count = a.vocab;
  __syncthreads();
  finish_alone(sh, a, weigh, k > 0 ? min(k, a.vocab) : a.vocab, p, u, row);
}

// RESIDENT: CTAs per SM that the registers are cut for.
template <typename T, int RESIDENT>
__global__ void __launch_bounds__(kThreads, RESIDENT) sample_kernel(const SampleArgs a) {
  grid_dependency_wait();
  extern __shared__ __align__(16) unsigned char smem[];
  Shared& sh = *reinterpret_cast<Shared*>(smem);
  cg::cluster_group cluster = cg::this_cluster();
  const int C = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  auto peer = [&](int r) { return cluster.map_shared_rank(&sh, r); };
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t row = blockIdx.x / C;
  const float temp = a.temperature ? a.temperature[row] : 1.f;
  const float u = a.uniforms[row];
  const int k = a.top_k ? a.top_k[row] : 0;
  const float p = a.top_p ? a.top_p[row] : 1.f;
  const float mp = a.min_p ? a.min_p[row] : 0.f;
  if (!(temp >= 0.f) || !(u >= 0.f && u < 1.f) || p != p || mp != mp) {
    if (rank == 0 && tid == 0) {
      a.tokens[row] = -1;
      raise_status(a.status, BM_DEVERR_BAD_PARAMETER);
    }
    return;  // the whole cluster
  }
  cluster.barrier_arrive();  // the others' shared memory is there once all have
  const T* x = static_cast<const T*>(a.logits) + row * a.stride;
  constexpr int VEC = VecWidth<T>::value;
  // this CTA's stretch and this warp's stretch of it
  const int c_lo = min(a.vocab, rank * a.chunk), c_hi = min(a.vocab, c_lo + a.chunk);
  const int span = ((c_hi - c_lo + kWarps - 1) / kWarps + VEC - 1) / VEC * VEC;
  const int lo = min(c_hi, c_lo + warp * span), hi = min(c_hi, lo + span);

  // A small top-k: the k-th largest of the maxima of `groups` parts of the row is a bound
  // that k logits reach, and few more where k is small beside the groups.
  const int share = max(1, C / 2);                   // threads of a group
  const int groups = C * (kThreads / share);         // 512 or 1024
  const bool bounded = k > 0 && k < a.vocab && 2 * k <= groups && temp > 0.f;

  // ---------------- the largest logit ----------------
  {
    float m = -INFINITY;
    int at = c_hi;
    if (temp == 0.f) {  // and its first index
      each<4>(x, lo, hi, a.vec, false, [&](int i, float v) {
        if (v > m) {  // a lane's indexes ascend
          m = v;
          at = i;
        }
      });
    } else {
      each<4>(x, lo, hi, a.vec, false, [&](int, float v) { m = fmaxf(m, v); });
    }
    cluster.barrier_wait();
    if (temp > 0.f) {
      if (bounded) {
        float g = m;
        if (share > 1) g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, 1));
        if (share > 2) g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, 2));
        if (tid % share == 0) peer(0)->cand_key[(rank * kThreads + tid) / share] = key_of(g);
      }
    }
    u64 best = static_cast<u64>(key_of(m)) << 32 | static_cast<uint32_t>(~at);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
      const u64 o = __shfl_xor_sync(0xffffffffu, best, off);
      best = o > best ? o : best;
    }
    if (lane == 0) sh.warp[warp] = best;
    if (tid < 128) sh.table[tid] = exp2(static_cast<double>(a.bits) - tid / 128.0);
    __syncthreads();
    if (tid < C) {
      for (int w = 0; w < kWarps; ++w) best = sh.warp[w] > best ? sh.warp[w] : best;
      peer(tid)->best[rank] = best;
    }
  }
  cluster.sync();
  u64 best = 0;
  for (int r = 0; r < C; ++r) best = sh.best[r] > best ? sh.best[r] : best;
  const float top = logit_of(static_cast<uint32_t>(best >> 32));
  if (top == -INFINITY || temp == 0.f) {
    if (rank == 0 && tid == 0) a.tokens[row] = top == -INFINITY ? -1 : static_cast<int32_t>(~static_cast<uint32_t>(best));
    return;  // nobody reads another CTA's shared memory after the sync above
  }
  const bool remap = top == INFINITY;
  const float bins_per_octave = Weigher::kLimit / static_cast<float>(a.bits + 2);
  const Weigher weigh = weigher(remap ? 0.f : top, temp, mp, a.bits, sh.table);

  uint32_t t = 0;         // what stays: keys above t,
  u64 ties = 0;           // and the first `ties` equal to it,
  bool cut = false;       // which are not all
  bool summed = false;    // kept: the weights of what stays by warp's stretch
  u64 kept = 0;

  // Logits set aside on the way, in no order, with the range of their keys.
  uint32_t from = 0xffffffffu, to = 0;
  auto collect = [&](int i, float lv) {
    const uint32_t key = key_of(lv);
    from = min(from, key);
    to = max(to, key);
    const uint32_t n = atomicAdd(&sh.own_count, 1u);
    if (n < kList) {
      sh.list_key[n] = key;
      sh.list_index[n] = static_cast<uint32_t>(i);
    }
  };
  // This CTA's go behind the others' in the leader's list: put(place, key, index).
  auto hand_over = [&](auto put) {
    from = __reduce_min_sync(0xffffffffu, from);
    to = __reduce_max_sync(0xffffffffu, to);
    if (lane == 0 && to != 0) {
      atomicMin(&peer(0)->key_min, from);
      atomicMax(&peer(0)->key_max, to);
    }
    __syncthreads();
    const uint32_t own = sh.own_count;
    if (tid == 0 && own != 0) sh.offset = atomicAdd(&peer(0)->count, own);
    __syncthreads();
    for (uint32_t i = tid; i < min(own, static_cast<uint32_t>(kList)); i += kThreads) {
      const uint32_t at = sh.offset + i;
      if (at < kList) put(at, sh.list_key[i], sh.list_index[i]);
    }
  };
  auto clear_lists = [&]() {
    if (tid == 0) {
      sh.own_count = 0;
      sh.count = 0;
      sh.key_min = 0xffffffffu;
      sh.key_max = 0;
    }
  };
  auto put_index = [&](uint32_t at, uint32_t key, uint32_t index) {
    peer(0)->cand_key[at] = key;
    peer(0)->cand_index[at] = index;
  };

  if (bounded && !remap) {
    if (rank == 0) {
      uint32_t key[kEach], even[kEach];
      u64 one[kEach], before;
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        one[e] = tid + e * kThreads < groups;
        key[e] = one[e] != 0 ? sh.cand_key[tid + e * kThreads] : 0;
        even[e] = weigh.even(logit_of(key[e]));
      }
      const uint32_t bound = border(sh, even, key, one, k, &before);
      if (tid < C) peer(tid)->key = bound;
      __syncthreads();
    }
    clear_lists();
    cluster.sync();
    const float bound = logit_of(sh.key);
    if (bound > -INFINITY) {
      each<1>(x, lo, hi, a.vec, false, [&](int i, float v) {
        if (v >= bound) collect(i, v);
      });
      hand_over(put_index);
      cluster.sync();
      if (peer(0)->count <= kList) {
        cluster.sync();  // the count has been read: a CTA's shared memory outlives its readers
        if (rank == 0) finish_alone(sh, a, weigh, k, p, u, row);
        return;
      }
      cluster.sync();
    }
  }

  // ---------------- t for top-k (stage 0) and top-p (stage 1) ----------------
  const bool has_min_p = mp > 0.f;
  for (int stage = 0; stage < 2; ++stage) {
    if (stage == 0 ? !(k > 0 && k < a.vocab) : !(p < 1.f)) continue;
    const uint32_t t0 = t;  // top-p works on what top-k left: keys above t0
    const float t0_f = t0 != 0 ? logit_of(t0) : -INFINITY;
    const u64 tied = stage == 1 && t0 != 0 ? ties * weigh(t0_f) : 0;  // and these
    auto bin_of = [&](float x) -> int {  // a logit without a weight has the last
      const float b = weigh.place(x);
      return b < Weigher::kLimit ? bits_of(b + kMagic) : kBins - 1;
    };
    for (int b = tid; b < kBins / 4; b += kThreads) reinterpret_cast<uint4*>(sh.hist)[b] = make_uint4(0u, 0u, 0u, 0u);
    clear_lists();
    __syncthreads();
    if (stage == 0) {
      each<1>(x, lo, hi, a.vec, remap, [&](int, float v) { atomicAdd(&sh.hist[bin_of(v)], 1u); });
    } else {
      // the fp32 weight in units of its bin's middle, 2^unit: linear within the bin
      const float unit = exp2f(static_cast<float>(a.unit));
      const float slope = unit * -0.69314718f / bins_per_octave;
      each<1>(x, lo, hi, a.vec, remap, [&](int, float v) {
        const float b = weigh.place(v);
        if (b < Weigher::kLimit && v > t0_f) {
          const float m = b + kMagic;
          atomicAdd(&sh.hist[bits_of(m)], static_cast<uint32_t>(bits_of(fmaf(b - (m - kMagic), slope, unit) + kMagic)));
        }
      });
    }
    __syncthreads();
    // a bin's value: its count, or its weight in units of 2^-40 of the largest
    auto bin_value = [&](u64 h, int bin) -> u64 {
      if (stage == 0) return h;
      return static_cast<u64>(static_cast<double>(h) * static_cast<double>(exp2f(static_cast<float>(40 - a.unit) - static_cast<float>(bin) / bins_per_octave)));
    };
    const u64 tied_value = tied == 0 ? 0 : static_cast<u64>(static_cast<double>(tied) * exp2(40.0 - a.bits));
    const int tied_bin = tied == 0 ? -1 : bin_of(t0_f);
    {
      u64 v = 0;  // eight bins a thread, 64 by eight threads
#pragma unroll
      for (int i = 0; i < kBins / kThreads; ++i) v += bin_value(sh.hist[tid * (kBins / kThreads) + i], tid * (kBins / kThreads) + i);
#pragma unroll
      for (int off = 4; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
      if ((lane & 7) == 0) sh.coarse[tid >> 3] = v + (rank == 0 && tied_bin >> 6 == tid >> 3 ? tied_value : 0);
    }
    cluster.sync();
    // The bins that can hold the border: the first whose running value reaches the target,
    // for top-p from the least to the most that the sums' errors allow. A place is off by
    // 4 * 2^-24 of at most 53 octaves, the line within a bin by 2^-16.5 of the weight (half a
    // bin is 53 / 8192 octaves at most), a coarse weight by half a unit of at least
    // 0.99 * 2^unit: a sum by e = 2^-15.5 + 1.01 * 2^-(unit + 1) of itself, a running sum
    // against p * sum by 2 e (1 + e), below the 2^-13 + 2^(1 - unit) taken.
    if (warp == 0) {
      static_assert(kCoarse == 64, "two coarse bins a lane");
      u64 c0 = 0, c1 = 0;
      for (int r = 0; r < C; ++r) {
        c0 += peer(r)->coarse[2 * lane];
        c1 += peer(r)->coarse[2 * lane + 1];
      }
      auto scan = [&](u64 v) {  // the sum of the lanes before, v included
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
          const u64 o = __shfl_up_sync(0xffffffffu, v, off);
          if (lane >= off) v += o;
        }
        return v;
      };
      const u64 coarse_incl = scan(c0 + c1);
      const u64 sum = __shfl_sync(0xffffffffu, coarse_incl, 31);
      u64 least_target = k, most_target = k;
      if (stage == 1) {
        const double ps = static_cast<double>(fmaxf(p, 0.f)) * static_cast<double>(sum);
        const double width = 0x1p-13 + exp2f(static_cast<float>(1 - a.unit));
        least_target = max(static_cast<u64>(ps * fmax(1.0 - width, 0.0)), static_cast<u64>(1));
        most_target = static_cast<u64>(ps * (1.0 + width)) + 2 * kBins;  // each bin's value was cut to a whole number
      }
#pragma unroll 1
      for (int side = 0; side < 2; ++side) {
        const u64 target = side == 0 ? least_target : most_target;
        int bin = kBins - 1;
        u64 at = 0, through = 0;
        const uint32_t hit = __ballot_sync(0xffffffffu, target <= coarse_incl);
        if (hit != 0) {
          const int l = __ffs(hit) - 1;
          const u64 before = __shfl_sync(0xffffffffu, coarse_incl - c0 - c1, l), first = __shfl_sync(0xffffffffu, c0, l);
          const int group = 2 * l + (target > before + first);
          at = before + (target > before + first ? first : 0);
          // its 64 bins, two a lane; rounding by bin and by CTA sums to what coarse holds
          u64 f0 = 0, f1 = 0;
          const int b0 = group * 64 + 2 * lane;
          for (int r = 0; r < C; ++r) {
            f0 += bin_value(peer(r)->hist[b0], b0);
            f1 += bin_value(peer(r)->hist[b0 + 1], b0 + 1);
          }
          if (tied_bin == b0) f0 += tied_value;
          if (tied_bin == b0 + 1) f1 += tied_value;
          const u64 incl = at + scan(f0 + f1);
          const int fl = __ffs(__ballot_sync(0xffffffffu, target <= incl)) - 1;
          const u64 fine = __shfl_sync(0xffffffffu, incl - f0 - f1, fl), f = __shfl_sync(0xffffffffu, f0, fl);
          const bool second = target > fine + f;
          bin = group * 64 + 2 * fl + second;
          at = fine + (second ? f : 0);
          through = second ? __shfl_sync(0xffffffffu, incl, fl) : fine + f;
        }
        if (lane == 0) {
          if (side == 0) {
            sh.bin_lo = bin;
            sh.before = at;
            sh.through = through;
          }
          sh.bin_hi = bin;
        }
        if (most_target <= through) break;  // both ends in one bin
      }
    }
    __syncthreads();
    const int bin_lo = static_cast<int>(sh.bin_lo), bin_hi = static_cast<int>(sh.bin_hi);
    // Exact weights: of the row, of what is above these bins, and of that what min_p keeps;
    // and the bins' logits.
    u64 own_sum = 0, own_above = 0;
    from = 0xffffffffu;
    to = 0;
    kept = 0;
    // All of a small top-k's logits, and those that share its last bin, fit the list: the
    // leader goes on alone.
    const bool alone = stage == 0 && sh.through <= kList;
    if (alone) {
      each<1>(x, lo, hi, a.vec, remap, [&](int i, float lv) {
        if (bin_of(lv) <= bin_hi && i < hi) collect(i, lv);
      });
    } else if (stage == 0) {
      each<1>(x, lo, hi, a.vec, remap, [&](int i, float lv) {
        const int b = bin_of(lv);
        if (b > bin_hi) return;
        if (b >= bin_lo) {
          collect(i, lv);
        } else {
          const double w = weigh.real(lv);
          if (w >= weigh.least) kept += Weigher::whole(w);
        }
      });
    } else {
      const float m_lo = kMagic + static_cast<float>(bin_lo), m_hi = kMagic + static_cast<float>(bin_hi);
      each<1>(x, lo, hi, a.vec, remap, [&](int i, float lv) {
        const float b = weigh.place(lv), m = b + kMagic;
        const double w = weigh.real(lv);
        const u64 n = b < Weigher::kLimit && lv > t0_f ? Weigher::whole(w) : 0;
        own_sum += n;
        if (m < m_lo) {
          own_above += n;
          if (has_min_p && w >= weigh.least) kept += n;
        } else if (m <= m_hi && n != 0) {  // a logit without weight is no border
          collect(i, lv);
        }
        if (t0 != 0 && lv == t0_f && m <= m_hi) collect(i, lv);
      });
      if (!has_min_p) kept = own_above;
      own_sum = warp_sum64(own_sum);
      own_above = warp_sum64(own_above);
      if (lane == 0) {
        sh.warp[warp] = own_sum;
        sh.sub[warp] = own_above;
      }
    }
    auto value = [&](uint32_t key) -> u64 { return stage == 0 ? 1 : key == t0 ? 0 : weigh(logit_of(key)); };
    auto put_weight = [&](uint32_t at, uint32_t key, uint32_t) {
      peer(0)->cand_key[at] = key;
      peer(0)->cand_weight[at] = value(key);
    };
    if (alone) {
      hand_over(put_index);
    } else {
      hand_over(put_weight);
    }
    if (stage == 1 && tid < C) {
      u64 s = 0, b = 0;
      for (int w = 0; w < kWarps; ++w) {
        s += sh.warp[w];
        b += sh.sub[w];
      }
      peer(tid)->sum[rank] = s;
      peer(tid)->above[rank] = b;
    }
    cluster.sync();
    if (alone) {
      if (rank == 0) finish_alone(sh, a, weigh, k, p, u, row);
      return;  // nobody reads another CTA's shared memory any more
    }
    u64 target = k, passed = stage == 0 ? sh.before : 0;
    if (stage == 1) {
      u64 s = tied;
      for (int r = 0; r < C; ++r) {
        s += sh.sum[r];
        passed += sh.above[r];
      }
      bool fraction;
      target = portion(fmaxf(p, 0.f), s, &fraction);
      if (fraction || target == 0) ++target;  // a token stays while the weight before it is below target
    }
    uint32_t count = peer(0)->count;
    from = peer(0)->key_min;
    to = peer(0)->key_max;
    summed = count <= kList;
    // Split the keys from..to, 512 equal parts a round, down to the border's key: by the
    // whole cluster while the list does not hold them, then by the leader.
    for (int round = 0; round < 4 && from != to; ++round) {
      const bool all = count > kList;
      if (!all && rank != 0) break;
      if (all) {  // the leader's counters have been read
        cluster.sync();
      } else {
        __syncthreads();
      }
      int shift = 0;
      while (((to - from) >> shift) >= static_cast<uint32_t>(kThreads)) ++shift;
      sh.split[tid] = 0;
      if (tid == 0) {
        sh.own_count = all ? 0 : sh.own_count;
        if (all) sh.count = 0;
        sh.key_min = 0xffffffffu;
        sh.key_max = 0;
      }
      __syncthreads();
      if (all) {
        each<1>(x, lo, hi, a.vec, remap, [&](int, float lv) {
          const uint32_t key = key_of(lv);
          if (key >= from && key <= to) atomicAdd(&sh.split[(to - key) >> shift], value(key));
        });
        cluster.sync();
      } else {
        for (uint32_t i = tid; i < count; i += kThreads) {
          const uint32_t key = sh.cand_key[i];
          if (key >= from && key <= to) atomicAdd(&sh.split[(to - key) >> shift], sh.cand_weight[i]);
        }
        __syncthreads();
      }
      u64 v = 0, total;
      if (all) {
        for (int r = 0; r < C; ++r) v += peer(r)->split[tid];
      } else {
        v = sh.split[tid];
      }
      if (tied != 0 && t0 >= from && t0 <= to && (to - t0) >> shift == static_cast<uint32_t>(tid)) v += tied;
      const u64 at = block_scan64(v, sh.sub, &total) + passed;
      if (at < target && target <= at + v) {
        sh.bin = tid;
        sh.before = at;
      }
      __syncthreads();
      passed = sh.before;
      const uint32_t bin = sh.bin, old_from = from, old_to = to;
      if (all) {
        from = 0xffffffffu;
        to = 0;
        each<1>(x, lo, hi, a.vec, remap, [&](int i, float lv) {
          const uint32_t key = key_of(lv);
          if (key >= old_from && key <= old_to && (old_to - key) >> shift == bin) collect(i, lv);
        });
        hand_over(put_weight);
        cluster.sync();
        count = peer(0)->count;
        from = peer(0)->key_min;
        to = peer(0)->key_max;
      } else {
        for (uint32_t i = tid; i < count; i += kThreads) {
          const uint32_t key = sh.cand_key[i];
          if (key >= from && key <= to && (to - key) >> shift == bin) {
            atomicMin(&sh.key_min, key);
            atomicMax(&sh.key_max, key);
          }
        }
        __syncthreads();
        from = sh.key_min;
        to = sh.key_max;
      }
    }
    if (rank == 0) {
      int n = 0;
      for (uint32_t i = tid; i < count && count <= kList; i += kThreads) n += sh.cand_key[i] == from;
      u64 total;
      block_scan64(static_cast<u64>(n), sh.sub, &total);
      if (tid < C) {
        const u64 equal = count > kList ? count : total;  // logits of key t (over the list: one key)
        const u64 w = max(stage == 1 && from == t0 ? weigh(t0_f) : value(from), static_cast<u64>(1));
        u64 rest = min((target - passed + w - 1) / w, equal);
        if (stage == 1 && from == t0) rest = min(rest, ties);
        peer(tid)->key = from;
        peer(tid)->ties = rest;
        peer(tid)->cut = rest < equal;
      }
    }
    cluster.sync();
    t = sh.key;
    ties = sh.ties;
    cut = sh.cut;
  }

  // ---------------- the token ----------------
  // An index by running sums of values: the sums by warp's stretch (own) meet over the
  // cluster; then those by sixteenths of the stretch that holds the target, then its
  // logits. First (if not all logits equal to t stay) the last of those that do, then the
  // token.
  const float t_f = t != 0 ? logit_of(t) : -INFINITY;
  uint32_t last_tie = 0xffffffffu;
  for (int what = cut ? 0 : 1; what < 2; ++what) {
    auto value = [&](int i, float v) -> u64 {
      if (what == 0) return v == t_f;
      if (!(weigh.place(v) < Weigher::kLimit) || v < t_f || (v == t_f && static_cast<uint32_t>(i) > last_tie)) return 0;
      const double w = weigh.real(v);
      return w >= weigh.least ? Weigher::whole(w) : 0;
    };
    // What stays above the border's bins was summed on the way; their logits are collected.
    u64 own = 0;
    const bool have = what == 1 && summed;
    if (have) {
      own = kept;
    } else {
      each<1>(x, lo, hi, a.vec, remap, [&](int i, float v) { own += value(i, v); });
    }
    own = warp_sum64(own);
    __syncthreads();
    if (lane == 0) sh.warp[warp] = own;
    __syncthreads();
    if (have) {
      for (uint32_t i = tid; i < sh.own_count; i += kThreads) {
        const int index = static_cast<int>(sh.list_index[i]);
        const u64 w = value(index, logit_of(sh.list_key[i]));
        if (w != 0) atomicAdd(&sh.warp[(index - c_lo) / span], w);
      }
      __syncthreads();
    }
    if (tid < C) {
      u64 s = 0;
      for (int w = 0; w < kWarps; ++w) s += sh.warp[w];
      peer(tid)->sum[rank] = s;
    }
    cluster.sync();
    u64 total = 0, at = 0;
    for (int r = 0; r < C; ++r) {
      if (r < rank) at += sh.sum[r];
      total += sh.sum[r];
    }
    bool fraction;
    const u64 want = what == 0 ? ties - 1 : portion(u, total, &fraction);  // the first index whose running sum exceeds it
    if (at <= want && want < at + sh.sum[rank]) {  // this CTA's stretch (all its threads agree)
      int w = 0;
      while (w < kWarps - 1 && want >= at + sh.warp[w]) at += sh.warp[w++];
      const int w_lo = min(c_hi, c_lo + w * span), w_hi = min(c_hi, w_lo + span);
      const int part = ((w_hi - w_lo + kWarps - 1) / kWarps + VEC - 1) / VEC * VEC;
      int s_lo = min(w_hi, w_lo + warp * part), s_hi = min(w_hi, s_lo + part);
      own = 0;
      each<1>(x, s_lo, s_hi, a.vec, remap, [&](int i, float v) { own += value(i, v); });
      own = warp_sum64(own);
      if (lane == 0) sh.sub[warp] = own;
      __syncthreads();
      if (warp == 0) {
        int q = 0;
        while (q < kWarps - 1 && want >= at + sh.sub[q]) at += sh.sub[q++];
        s_lo = min(w_hi, w_lo + q * part);
        s_hi = min(w_hi, s_lo + part);
        for (int i0 = s_lo; i0 < s_hi; i0 += 32) {
          const int i = i0 + lane;
          u64 incl = i < s_hi ? value(i, remapped(load1(x + i), remap)) : 0;
#pragma unroll
          for (int off = 1; off < 32; off <<= 1) {
            const u64 o = __shfl_up_sync(0xffffffffu, incl, off);
            if (lane >= off) incl += o;
          }
          const uint32_t hit = __ballot_sync(0xffffffffu, want < at + incl);
          if (hit != 0) {
            const int index = i0 + __ffs(hit) - 1;
            if (what == 1) {
              if (lane == 0) a.tokens[row] = index;
            } else if (lane < C) {
              peer(lane)->index = index;
            }
            break;
          }
          at += __shfl_sync(0xffffffffu, incl, 31);
        }
      }
    }
    if (what == 0) {
      cluster.sync();
      last_tie = sh.index;
    }
  }
}

}  // namespace
}  // namespace bm

extern "C" int bm_sample(int32_t* tokens, const void* logits, const float* uniforms, const float* temperature,
                         const int32_t* top_k, const float* top_p, const float* min_p, int64_t rows, int64_t vocab,
                         int64_t row_stride, bm_dtype_t dtype, int32_t* d_status, void* stream) {
  using namespace bm;
  const char* what = "bm_sample";
  if (!valid_dtype(dtype)) return fail(BM_ERR_INVALID_ARGUMENT, "%s: bad dtype %d", what, static_cast<int>(dtype));
  if (rows < 0 || rows > INT32_MAX / kMaxCluster) return fail(BM_ERR_INVALID_ARGUMENT, "%s: bad rows", what);
  if (vocab <= 0 || vocab > (1 << 24)) return fail(BM_ERR_INVALID_ARGUMENT, "%s: vocab outside [1, 2^24]", what);
  if (row_stride < vocab) return fail(BM_ERR_INVALID_ARGUMENT, "%s: row_stride below vocab", what);
  if (rows == 0) return BM_OK;
  if (!tokens || !logits || !uniforms) return fail(BM_ERR_INVALID_ARGUMENT, "%s: NULL pointer", what);
  const int es = dtype_size(dtype);
  if (!aligned_to(logits, es) || !aligned_to({tokens, uniforms, temperature, top_k, top_p, min_p, d_status}, 4)) {
    return fail(BM_ERR_INVALID_ARGUMENT, "%s: a pointer is not aligned to its elements", what);
  }
  SampleArgs a{};
  a.tokens = tokens;
  a.logits = logits;
  a.uniforms = uniforms;
  a.temperature = temperature;
  a.top_k = top_k;
  a.top_p = top_p;
  a.min_p = min_p;
  a.rows = rows;
  a.stride = row_stride;
  a.vocab = static_cast<int>(vocab);
  int log2_up = 0;
  while ((int64_t{1} << log2_up) < vocab) ++log2_up;
  a.bits = std::min(51, 62 - log2_up);  // an fp64 weight is made whole below 2^52
  a.vec = aligned16(logits) && row_stride * es % 16 == 0;
  a.status = d_status;
  // CTAs per row: as many as leave every SM at most one, with all the registers they like;
  // then twice as many, at half the registers, while a CTA has more than 16384 logits and an
  // SM gets at most four (rows cost unevenly and SMs fill unevenly: 64 mixed rows of 128256
  // with 4 CTAs 51, with 8 44 us; 256 rows of 128256 with 1 and 2: top-k 126 and 105, top-p 199
  // and 193, no filter 94 and 96; 128 rows of 32000 with 2 and 4: 38 and 44). None with fewer
  // than 2048.
  int c = 1;
  while (c < kMaxCluster && rows * c * 2 <= sm_count() && vocab >= int64_t{2048} * c * 2) c *= 2;
  while (c < kMaxCluster && rows * c * 2 <= 4 * sm_count() && vocab > int64_t{16384} * c) c *= 2;
  const bool crowded = rows * c > sm_count();
  a.chunk = static_cast<int>(((vocab + c - 1) / c + 7) / 8 * 8);
  // A bin of the histogram holds a CTA's whole stretch without passing 32 bits. A weight is at
  // most 2^unit (1 + 0.35 / 77) + 0.5: half a bin above its middle (0.5 ln 2 of an octave's 77
  // bins or more: kLimit / (51 + 2)), and rounded, where unit is 7 at least (and then an octave has
  // 102 bins): below 2^unit * 129 / 128.
  a.unit = 16;
  while ((static_cast<int64_t>(a.chunk) * 129 << a.unit) >= int64_t{128} << 32) --a.unit;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = static_cast<unsigned>(c);
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = 1;
  const dim3 grid(static_cast<unsigned>(rows * c));
  if (vocab <= kList) {
    auto kernel = dtype == BM_F32 ? sample_short_kernel<float> : sample_short_kernel<bf16>;
    if (int st = allow_dynamic_smem(reinterpret_cast<const void*>(kernel), sizeof(Shared), what)) return st;
    return launch_kernel(what, kernel, dim3(static_cast<unsigned>(rows)), dim3(kThreads), sizeof(Shared), as_stream(stream), nullptr, a);
  }
  auto go = [&](auto kernel) {
    if (int st = allow_dynamic_smem(reinterpret_cast<const void*>(kernel), sizeof(Shared), what)) return st;
    return launch_kernel(what, kernel, grid, dim3(kThreads), sizeof(Shared), as_stream(stream), &attr, a);
  };
  if (dtype == BM_F32) return crowded ? go(sample_kernel<float, 2>) : go(sample_kernel<float, 1>);
  return crowded ? go(sample_kernel<bf16, 2>) : go(sample_kernel<bf16, 1>);
}
