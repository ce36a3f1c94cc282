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
// method of Tang, ACM TOMS 15, 1989): y = (j + r) / 64, a table of 2^(-j/64) and a
// polynomial of degree 5 in r, off by less than 2^-50 of the weight.
//
// Bound: a row is read from HBM once (the passes below find it in L2), so bytes count
// only for many rows; there the fp64 operations (eleven a logit where all weigh) cost as
// much, and one or few rows are bound by the chain of passes. A cluster of up to 8 CTAs
// shares a row:
//   1. the largest logit and its first index;
//   2. for top-k, then for top-p: a histogram over 4096 bins of equal ratio of weight, in
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
constexpr int kBinsPerThread = kBins / kThreads;
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
  int unit;   // bits of a fp32 weight in the histogram: chunk * 2^unit < 2^32
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
// of the fp64 units' rate.
__device__ __forceinline__ double widen(float x) {
  const uint32_t u = __float_as_uint(x);
  if ((u & 0x7f800000u) == 0) return static_cast<double>(x);  // zeros and denormals
  return __hiloint2double(static_cast<int>((u & 0x80000000u) | (((u & 0x7fffffffu) >> 3) + 0x38000000u)),
                          static_cast<int>(u << 29));
}

// Weights of a row.
struct Weigher {
  double top;            // the largest logit (0 when it is +inf: no other has a weight)
  double scale;          // 64 log2(e) / T
  double one, least;     // 2^bits; min_p in it
  const double* table;   // 2^(bits - j/64), j < 64
  float top_f, scale_f;  // the same in fp32, scale_f per octave
  float limit;           // octaves past which a weight rounds to 0

  // log2 of the largest weight over this one, rounded: never falls as the logit does.
  // NaN for -inf at T = inf.
  __device__ __forceinline__ float octaves(float x) const { return (top_f - x) * scale_f; }
  // The weight before it is rounded to a whole number, for x < top with octaves < limit.
  __device__ __forceinline__ double real(float x) const {
    constexpr double kRound = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to a whole number
    constexpr double kStep = 0.010830424696249145;  // ln(2) / 64
    const double y = (top - widen(x)) * scale;
    const double shifted = y + kRound;
    const int j = __double2loint(shifted);
    const double z = (y - (shifted - kRound)) * -kStep;
    double q = fma(z, 1.0 / 120.0, 1.0 / 24.0);
    q = fma(z, q, 1.0 / 6.0);
    q = fma(z, q, 0.5);
    q = fma(z, q, 1.0);
    q = fma(z, q, 1.0);
    const double w = q * table[j & 63];
    return __hiloint2double(__double2hiint(w) - ((j >> 6) << 20), __double2loint(w));
  }
  __device__ __forceinline__ static u64 whole(double w) {  // w < 2^52, rounded
    return static_cast<u64>(__double_as_longlong(w + 4503599627370496.0)) & 0xfffffffffffffull;
  }
  // The weight, and (kept) the same or 0 where min_p drops it.
  __device__ __forceinline__ u64 weigh(float x, u64* kept) const {
    if (x == top_f) {
      *kept = static_cast<u64>(one);
      return *kept;
    }
    *kept = 0;
    if (!(octaves(x) < limit)) return 0;
    const double w = real(x);
    const u64 n = whole(w);
    if (w >= least) *kept = n;
    return n;
  }
  __device__ __forceinline__ u64 operator()(float x) const {
    u64 kept;
    return weigh(x, &kept);
  }
};

struct Shared {
  union {
    u64 wide[kBins];
    uint32_t hist[kBins];
  };
  double table[64];
  u64 best[kMaxCluster];   // per CTA of the cluster: key << 32 | ~index
  u64 sum[kMaxCluster], above[kMaxCluster], slice[kMaxCluster];
  u64 warp[kWarps], sub[kWarps], kept[kWarps];
  u64 before;              // value above the bin found
  u64 ties;                // how many logits equal to t stay,
  u64 cand_weight[kList];  // the leader's: collected logits
  uint32_t cand_key[kList];
  uint32_t list_key[kList], list_index[kList];  // this CTA's share of them
  uint32_t own_count;
  uint32_t count, key_min, key_max;             // the leader's: logits of the border's bins
  uint32_t bin_lo, bin_hi, bin;
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

// The logits [lo, hi) of a row by one warp: f(index, logit), U 16-byte loads in flight
// per lane besides those being worked on. Lanes may call f a different number of times.
template <int U, typename T, typename F>
__device__ __forceinline__ void each(const T* x, int lo, int hi, bool vec, F f) {
  constexpr int VEC = VecWidth<T>::value;
  const int lane = threadIdx.x & 31;
  if (!vec) {
    for (int i = lo + lane; i < hi; i += 32) f(i, load1(x + i));
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
#pragma unroll
        for (int e = 0; e < VEC; ++e) f(i + e, v[e]);
      }
    }
  }
  if (whole + lane < hi) f(whole + lane, load1(x + whole + lane));  // fewer than VEC are left
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const SampleArgs a) {
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
  const T* x = static_cast<const T*>(a.logits) + row * a.stride;
  constexpr int VEC = VecWidth<T>::value;
  // this CTA's stretch and this warp's stretch of it
  const int c_lo = min(a.vocab, rank * a.chunk), c_hi = min(a.vocab, c_lo + a.chunk);
  const int span = ((c_hi - c_lo + kWarps - 1) / kWarps + VEC - 1) / VEC * VEC;
  const int lo = min(c_hi, c_lo + warp * span), hi = min(c_hi, lo + span);

  // ---------------- the largest logit ----------------
  {
    uint32_t key = 0;
    int at = 0;
    each<4>(x, lo, hi, a.vec, [&](int i, float v) {
      const uint32_t c = key_of(v);
      if (c > key) {  // a lane's indexes ascend
        key = c;
        at = i;
      }
    });
    u64 best = static_cast<u64>(key) << 32 | static_cast<uint32_t>(~at);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
      const u64 o = __shfl_xor_sync(0xffffffffu, best, off);
      best = o > best ? o : best;
    }
    if (lane == 0) sh.warp[warp] = best;
    if (tid < 64) sh.table[tid] = exp2(static_cast<double>(a.bits) - tid / 64.0);
    __syncthreads();
    if (tid < C) {
      for (int w = 0; w < kWarps; ++w) best = sh.warp[w] > best ? sh.warp[w] : best;
      peer(tid)->best[rank] = best;
    }
  }
  cluster.sync();
  u64 best = 0;
  for (int r = 0; r < C; ++r) best = sh.best[r] > best ? sh.best[r] : best;
  const uint32_t top = static_cast<uint32_t>(best >> 32);
  Weigher weigh;
  weigh.top_f = logit_of(top);
  if (weigh.top_f == -INFINITY || temp == 0.f) {
    if (rank == 0 && tid == 0) a.tokens[row] = weigh.top_f == -INFINITY ? -1 : static_cast<int32_t>(~static_cast<uint32_t>(best));
    return;  // nobody reads another CTA's shared memory after the sync above
  }
  weigh.top = weigh.top_f == INFINITY ? 0.0 : widen(weigh.top_f);
  weigh.scale = 64.0 * kLog2e / static_cast<double>(temp);
  weigh.one = exp2(static_cast<double>(a.bits));
  weigh.least = weigh.one * static_cast<double>(fminf(mp, 1.f));
  weigh.table = sh.table;
  weigh.scale_f = static_cast<float>(kLog2e / static_cast<double>(temp));
  weigh.limit = static_cast<float>(a.bits + 2);
  const float bins_per_octave = static_cast<float>(kBins - 1) / weigh.limit;

  uint32_t t = 0;         // what stays: keys above t,
  u64 ties = 0;           // and the first `ties` equal to it,
  bool cut = false;       // which are not all
  bool summed = false;    // kept: the weights of what stays by warp's stretch
  u64 kept = 0;

  // ---------------- t for top-k (stage 0) and top-p (stage 1) ----------------
  for (int stage = 0; stage < 2; ++stage) {
    if (stage == 0 ? !(k > 0 && k < a.vocab) : !(p < 1.f)) continue;
    const uint32_t t0 = t;  // top-p works on what top-k left: keys above t0
    const u64 tied = stage == 1 && t0 != 0 ? ties * weigh(logit_of(t0)) : 0;  // and these
    auto bin_of = [&](float x) -> int {  // by octaves; a logit without a weight has the last
      if (x == weigh.top_f) return 0;
      const float b = weigh.octaves(x) * bins_per_octave;
      return b < static_cast<float>(kBins - 1) ? static_cast<int>(b) : kBins - 1;
    };
    // the fp32 weight in units of its bin's: at most 2^unit
    auto coarse = [&](float x, int bin) -> uint32_t {
      const float y = x == weigh.top_f ? 0.f : weigh.octaves(x) - static_cast<float>(bin) / bins_per_octave;
      return __float2uint_rn(exp2f(static_cast<float>(a.unit) - fmaxf(y, 0.f)));
    };
    for (int b = tid; b < kBins; b += kThreads) sh.hist[b] = 0;
    if (tid == 0) {
      sh.own_count = 0;
      sh.count = 0;
      sh.key_min = 0xffffffffu;
      sh.key_max = 0;
      sh.bin_lo = sh.bin_hi = kBins - 1;
    }
    __syncthreads();
    each<1>(x, lo, hi, a.vec, [&](int, float v) {
      if (stage == 0) {
        atomicAdd(&sh.hist[bin_of(v == v ? v : -INFINITY)], 1u);
      } else if (key_of(v) > t0 && (v == weigh.top_f || weigh.octaves(v) < weigh.limit)) {
        const int b = bin_of(v);
        atomicAdd(&sh.hist[b], coarse(v, b));
      }
    });
    cluster.sync();
    // this CTA's slice of the bins, over the cluster
    const int per_thread = kBins / C / kThreads;  // 8, 4, 2 or 1 bins
    const int first_bin = rank * (kBins / C) + tid * per_thread;
    u64 v[kBinsPerThread], mine = 0;
#pragma unroll
    for (int i = 0; i < kBinsPerThread; ++i) {
      v[i] = 0;
      if (i < per_thread) {
        for (int r = 0; r < C; ++r) v[i] += peer(r)->hist[first_bin + i];
        if (stage == 1) {  // units of the bin to units of the largest weight's 2^-40
          v[i] = static_cast<u64>(static_cast<double>(v[i]) *
                                  static_cast<double>(exp2f(static_cast<float>(40 - a.unit) -
                                                            static_cast<float>(first_bin + i) / bins_per_octave)));
          if (tied != 0 && bin_of(logit_of(t0)) == first_bin + i) v[i] += static_cast<u64>(static_cast<double>(tied) / weigh.one * 1099511627776.0);
        }
      }
      mine += v[i];
    }
    u64 all;
    u64 at = block_scan64(mine, sh.sub, &all);
    if (tid < C) peer(tid)->slice[rank] = all;
    cluster.sync();
    u64 sum = 0;
    for (int r = 0; r < C; ++r) {
      if (r < rank) at += sh.slice[r];
      sum += sh.slice[r];
    }
    // The bins that can hold the border: the first whose running value reaches the target,
    // for top-p from the least to the most that the sums' errors allow. Octave counts here
    // and above are off by 5 * 2^-24 of at most 53 octaves, a coarse weight by half a unit
    // of at least 0.99 * 2^unit: a sum by e = 2^-16 + 1.01 * 2^-(unit + 1) of itself, a
    // running sum against p * sum by 2 e (1 + e), below the 2^-13 + 2^(1 - unit) taken.
    u64 least_target = k, most_target = k;
    if (stage == 1) {
      const double ps = static_cast<double>(fmaxf(p, 0.f)) * static_cast<double>(sum);
      const double width = 0x1p-13 + exp2f(static_cast<float>(1 - a.unit));
      least_target = max(static_cast<u64>(ps * fmax(1.0 - width, 0.0)), static_cast<u64>(1));
      most_target = static_cast<u64>(ps * (1.0 + width)) + 2 * kBins;  // each bin's sum was cut to a whole number
    }
#pragma unroll
    for (int i = 0; i < kBinsPerThread; ++i) {
      const u64 next = at + v[i];
      if (at < least_target && least_target <= next) {
        for (int r = 0; r < C; ++r) peer(r)->bin_lo = first_bin + i;
        if (stage == 0) {
          for (int r = 0; r < C; ++r) peer(r)->before = at;
        }
      }
      if (at < most_target && most_target <= next) {
        for (int r = 0; r < C; ++r) peer(r)->bin_hi = first_bin + i;
      }
      at = next;
    }
    cluster.sync();
    const int bin_lo = static_cast<int>(sh.bin_lo), bin_hi = static_cast<int>(sh.bin_hi);
    // Exact weights: of the row's part (sum), of what is above these bins, and of that
    // what min_p keeps; and the bins' logits.
    u64 own_sum = 0, own_above = 0;
    uint32_t key_lo = 0xffffffffu, key_hi = 0;
    kept = 0;
    each<1>(x, lo, hi, a.vec, [&](int i, float lv) {
      const uint32_t key = key_of(lv);
      if (key < t0) return;
      const int b = bin_of(lv == lv ? lv : -INFINITY);
      u64 w = 0, keep = 0;
      if (key > t0 && (stage == 1 || b < bin_lo)) w = weigh.weigh(lv, &keep);
      own_sum += w;
      if (b < bin_lo) {
        own_above += w;
        kept += keep;
      } else if (b <= bin_hi && (stage == 0 || w != 0 || key == t0)) {  // a logit without weight is no border
        key_lo = min(key_lo, key);
        key_hi = max(key_hi, key);
        const uint32_t n = atomicAdd(&sh.own_count, 1u);
        if (n < kList) {
          sh.list_key[n] = key;
          sh.list_index[n] = static_cast<uint32_t>(i);
        }
      }
    });
    if (stage == 1) {
      own_sum = warp_sum64(own_sum);
      own_above = warp_sum64(own_above);
      if (lane == 0) {
        sh.warp[warp] = own_sum;
        sh.sub[warp] = own_above;
      }
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
      key_lo = min(key_lo, __shfl_xor_sync(0xffffffffu, key_lo, off));
      key_hi = max(key_hi, __shfl_xor_sync(0xffffffffu, key_hi, off));
    }
    if (lane == 0 && key_hi != 0) {
      atomicMin(&peer(0)->key_min, key_lo);
      atomicMax(&peer(0)->key_max, key_hi);
    }
    __syncthreads();
    // this CTA's collected logits go behind the others' in the leader's list
    const uint32_t own_count = sh.own_count;
    if (tid == 0) sh.bin = own_count == 0 ? 0 : atomicAdd(&peer(0)->count, own_count);
    if (stage == 1 && tid < C) {
      u64 s = 0, b = 0;
      for (int w = 0; w < kWarps; ++w) {
        s += sh.warp[w];
        b += sh.sub[w];
      }
      peer(tid)->sum[rank] = s;
      peer(tid)->above[rank] = b;
    }
    __syncthreads();
    for (uint32_t i = tid; i < own_count; i += kThreads) {
      if (sh.bin + i >= kList || i >= kList) break;
      peer(0)->cand_key[sh.bin + i] = sh.list_key[i];
      peer(0)->cand_weight[sh.bin + i] = stage == 0 ? 1 : sh.list_key[i] == t0 ? 0 : weigh(logit_of(sh.list_key[i]));
    }
    cluster.sync();
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
    key_lo = peer(0)->key_min;
    key_hi = peer(0)->key_max;
    summed = count <= kList;
    auto value = [&](uint32_t key) -> u64 { return stage == 0 ? 1 : key == t0 ? 0 : weigh(logit_of(key)); };
    // the interval's bins, descending, at most kBins of 2^shift keys
    auto shift_of = [](uint32_t from, uint32_t to) {
      int s = 0;
      while (((to - from) >> s) >= static_cast<uint32_t>(kBins)) ++s;
      return s;
    };
    // More than the list holds: the cluster splits the interval of keys until it does.
    for (int round = 0; round < 3 && count > kList && key_lo != key_hi; ++round) {  // 12 bits a round
      cluster.sync();  // the leader's counters have been read
      const int shift = shift_of(key_lo, key_hi);
      for (int b = tid; b < kBins; b += kThreads) sh.wide[b] = 0;
      if (tid == 0) {
        sh.own_count = 0;
        sh.count = 0;
        sh.key_min = 0xffffffffu;
        sh.key_max = 0;
      }
      __syncthreads();
      each<1>(x, lo, hi, a.vec, [&](int, float lv) {
        const uint32_t key = key_of(lv);
        if (key < key_lo || key > key_hi) return;
        const u64 w = value(key);
        if (w != 0) atomicAdd(&sh.wide[(key_hi - key) >> shift], w);
      });
      cluster.sync();
      mine = 0;
#pragma unroll
      for (int i = 0; i < kBinsPerThread; ++i) {
        v[i] = 0;
        if (i < per_thread) {
          for (int r = 0; r < C; ++r) v[i] += peer(r)->wide[first_bin + i];
          if (tied != 0 && t0 >= key_lo && t0 <= key_hi && (key_hi - t0) >> shift == static_cast<uint32_t>(first_bin + i)) v[i] += tied;
        }
        mine += v[i];
      }
      at = block_scan64(mine, sh.sub, &all) + passed;
      if (tid < C) peer(tid)->slice[rank] = all;
      cluster.sync();
      for (int r = 0; r < rank; ++r) at += sh.slice[r];
#pragma unroll
      for (int i = 0; i < kBinsPerThread; ++i) {
        if (at < target && target <= at + v[i]) {
          for (int r = 0; r < C; ++r) {
            peer(r)->bin = first_bin + i;
            peer(r)->before = at;
          }
        }
        at += v[i];
      }
      cluster.sync();
      passed = sh.before;
      const uint32_t bin = sh.bin;
      const uint32_t from = key_lo, to = key_hi;
      key_lo = 0xffffffffu;
      key_hi = 0;
      __syncthreads();  // sh.bin has been read
      each<1>(x, lo, hi, a.vec, [&](int i, float lv) {
        const uint32_t key = key_of(lv);
        if (key < from || key > to || (to - key) >> shift != bin) return;
        key_lo = min(key_lo, key);
        key_hi = max(key_hi, key);
        const uint32_t n = atomicAdd(&sh.own_count, 1u);
        if (n < kList) sh.list_key[n] = key;
      });
      if (key_hi != 0) {
        atomicMin(&peer(0)->key_min, key_lo);
        atomicMax(&peer(0)->key_max, key_hi);
      }
      __syncthreads();
      const uint32_t own = sh.own_count;
      if (tid == 0) sh.bin = own == 0 ? 0 : atomicAdd(&peer(0)->count, own);
      __syncthreads();
      for (uint32_t i = tid; i < own; i += kThreads) {
        if (sh.bin + i >= kList || i >= kList) break;
        peer(0)->cand_key[sh.bin + i] = sh.list_key[i];
        peer(0)->cand_weight[sh.bin + i] = value(sh.list_key[i]);
      }
      cluster.sync();
      count = peer(0)->count;
      key_lo = peer(0)->key_min;
      key_hi = peer(0)->key_max;
    }
    if (rank == 0) {
      uint32_t from = key_lo, to = key_hi;
      for (int round = 0; round < 3 && from != to; ++round) {  // count <= kList; 12 bits a round
        const int shift = shift_of(from, to);
        __syncthreads();
        for (int b = tid; b < kBins; b += kThreads) sh.wide[b] = 0;
        __syncthreads();
        for (uint32_t i = tid; i < count; i += kThreads) {
          const uint32_t key = sh.cand_key[i];
          if (key >= from && key <= to) atomicAdd(&sh.wide[(to - key) >> shift], sh.cand_weight[i]);
        }
        if (tid == 0 && tied != 0 && t0 >= from && t0 <= to) atomicAdd(&sh.wide[(to - t0) >> shift], tied);
        __syncthreads();
        mine = 0;
#pragma unroll
        for (int i = 0; i < kBinsPerThread; ++i) {
          v[i] = sh.wide[tid * kBinsPerThread + i];
          mine += v[i];
        }
        at = block_scan64(mine, sh.sub, &all) + passed;
#pragma unroll
        for (int i = 0; i < kBinsPerThread; ++i) {
          if (at < target && target <= at + v[i]) {
            sh.bin = tid * kBinsPerThread + i;
            sh.before = at;
            sh.key_min = 0xffffffffu;
            sh.key_max = 0;
          }
          at += v[i];
        }
        __syncthreads();
        passed = sh.before;
        for (uint32_t i = tid; i < count; i += kThreads) {
          const uint32_t key = sh.cand_key[i];
          if (key >= from && key <= to && (to - key) >> shift == sh.bin) {
            atomicMin(&sh.key_min, key);
            atomicMax(&sh.key_max, key);
          }
        }
        __syncthreads();
        from = sh.key_min;
        to = sh.key_max;
      }
      uint32_t equal = count;  // logits of key t
      if (count <= kList) {
        int n = 0;
        for (uint32_t i = tid; i < count; i += kThreads) n += sh.cand_key[i] == from;
        u64 total;
        block_scan64(n, sh.sub, &total);
        equal = static_cast<uint32_t>(total);
      }
      if (tid == 0) {
        u64 rest;
        if (stage == 1 && from == t0) {
          const u64 w = max(weigh(logit_of(t0)), static_cast<u64>(1));
          rest = min((target - passed + w - 1) / w, ties);
        } else {
          const u64 w = max(value(from), static_cast<u64>(1));  // a border lies in logits of some value
          rest = (target - passed + w - 1) / w;
        }
        if (rest > equal) rest = equal;
        for (int r = 0; r < C; ++r) {
          peer(r)->key = from;
          peer(r)->ties = rest;
          peer(r)->cut = rest < equal;
        }
      }
    }
    cluster.sync();
    t = sh.key;
    ties = sh.ties;
    cut = sh.cut;
  }

  // ---------------- the index where a running sum passes a target ----------------
  // f(index, logit) -> its value. The sums by warp's stretch are in sh.warp; then those by
  // sixteenths of the stretch that holds the target, then its logits. Writes the index to
  // every CTA's sh.index.
  auto find = [&](auto f, auto target_of) -> void {
    __syncthreads();
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
    const u64 want = target_of(total);             // the first index whose running sum exceeds it
    if (at <= want && want < at + sh.sum[rank]) {  // this CTA's stretch (all its threads agree)
      int w = 0;
      while (want >= at + sh.warp[w]) at += sh.warp[w++];
      const int w_lo = min(c_hi, c_lo + w * span), w_hi = min(c_hi, w_lo + span);
      const int part = ((w_hi - w_lo + kWarps - 1) / kWarps + VEC - 1) / VEC * VEC;
      int s_lo = min(w_hi, w_lo + warp * part), s_hi = min(w_hi, s_lo + part);
      u64 own = 0;
      each<1>(x, s_lo, s_hi, a.vec, [&](int i, float v) { own += f(i, v); });
      own = warp_sum64(own);
      if (lane == 0) sh.sub[warp] = own;
      __syncthreads();
      if (warp == 0) {
        int q = 0;
        while (want >= at + sh.sub[q]) at += sh.sub[q++];
        s_lo = min(w_hi, w_lo + q * part);
        s_hi = min(w_hi, s_lo + part);
        for (int i0 = s_lo; i0 < s_hi; i0 += 32) {
          const int i = i0 + lane;
          u64 incl = i < s_hi ? f(i, load1(x + i)) : 0;
#pragma unroll
          for (int off = 1; off < 32; off <<= 1) {
            const u64 o = __shfl_up_sync(0xffffffffu, incl, off);
            if (lane >= off) incl += o;
          }
          const unsigned int hit = __ballot_sync(0xffffffffu, want < at + incl);
          if (hit != 0) {
            if (lane < C) peer(lane)->index = i0 + __ffs(hit) - 1;
            break;
          }
          at += __shfl_sync(0xffffffffu, incl, 31);
        }
      }
    }
    cluster.sync();
  };

  uint32_t last_tie = 0xffffffffu;  // index of the last logit equal to t that stays
  if (cut) {
    auto is_tie = [&](int, float v) -> u64 { return key_of(v) == t; };
    u64 own = 0;
    each<1>(x, lo, hi, a.vec, [&](int i, float v) { own += is_tie(i, v); });
    own = warp_sum64(own);
    __syncthreads();
    if (lane == 0) sh.warp[warp] = own;
    find(is_tie, [&](u64) { return ties - 1; });
    last_tie = sh.index;
  }
  auto staying = [&](int i, float v) -> u64 {
    const uint32_t key = key_of(v);
    if (key < t || (key == t && static_cast<uint32_t>(i) > last_tie)) return 0;
    u64 keep;
    weigh.weigh(v, &keep);
    return keep;
  };
  // What stays, by warp's stretch: summed above the border's bins on the way, and of
  // their collected logits here; or all of it now.
  if (!summed) {
    kept = 0;
    each<1>(x, lo, hi, a.vec, [&](int i, float v) { kept += staying(i, v); });
  }
  kept = warp_sum64(kept);
  __syncthreads();
  if (lane == 0) sh.warp[warp] = kept;
  if (summed) {
    __syncthreads();
    for (uint32_t i = tid; i < min(sh.own_count, static_cast<uint32_t>(kList)); i += kThreads) {
      const u64 w = staying(static_cast<int>(sh.list_index[i]), logit_of(sh.list_key[i]));
      if (w != 0) atomicAdd(&sh.warp[(static_cast<int>(sh.list_index[i]) - c_lo) / span], w);
    }
  }
  find(staying, [&](u64 total) {
    bool fraction;
    return portion(u, total, &fraction);
  });
  if (rank == 0 && tid == 0) a.tokens[row] = static_cast<int32_t>(sh.index);
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
  // CTAs per row: enough to fill two per SM, none with fewer than 2048 logits.
  int c = 1;
  while (c < kMaxCluster && rows * c < 2 * sm_count() && vocab > int64_t{2048} * c) c *= 2;
  a.chunk = static_cast<int>(((vocab + c - 1) / c + 7) / 8 * 8);
  a.unit = 16;
  while ((static_cast<int64_t>(a.chunk) << a.unit) >= int64_t{1} << 32) --a.unit;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = static_cast<unsigned>(c);
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = 1;
  const dim3 grid(static_cast<unsigned>(rows * c));
  auto go = [&](auto kernel) {
    if (int st = allow_dynamic_smem(reinterpret_cast<const void*>(kernel), sizeof(Shared), what)) return st;
    return launch_kernel(what, kernel, grid, dim3(kThreads), sizeof(Shared), as_stream(stream), &attr, a);
  };
  return dtype == BM_F32 ? go(sample_kernel<float>) : go(sample_kernel<bf16>);
}
