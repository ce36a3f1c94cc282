// Sampling one token per row of logits with temperature, top-k, top-p and min-p, from
// given uniform numbers (bm_sample).
//
// Mathematics: w_i = exp((x_i - max x) / T). Ordered by (x descending, index ascending),
// top-k, top-p and min-p each keep a beginning of the row, so what stays is described
// by a key t and a count c: every logit above t and the first c of those equal to it.
// The token is the first index whose running weight passes u times the total.
//
// Exactness: a token is a whole number, so a rounding next to a border changes the
// answer. Weights are 64-bit fixed point, 2^bits for the largest with 2^bits * vocab <=
// 2^62, rounded once from fp64; every sum is an integer sum, the same in any order, and
// p * sum and u * sum are compared exactly.
#include <algorithm>

#include "bm_common.cuh"
#include "bm_host.h"

namespace bm {
namespace {

constexpr int kThreads = 512;
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
  int bits;  // the largest weight is 2^bits
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

struct Weigher {
  float top;      // the largest logit
  double scale;   // log2(e) / T
  double one;     // 2^bits
  __device__ __forceinline__ double real(float x) const {
    if (x == top) return 1.0;  // +inf too
    if (x == -INFINITY || top == INFINITY) return 0.0;
    return exp2((static_cast<double>(x) - static_cast<double>(top)) * scale);
  }
  __device__ __forceinline__ uint64_t operator()(float x) const { return __double2ull_rn(real(x) * one); }
};

template <typename V>
__device__ __forceinline__ V block_sum(V v, V* scratch) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  V s = 0;
  for (int w = 0; w < kThreads / 32; ++w) s += scratch[w];
  return s;
}

// floor(f * s) and whether f * s has a fraction, f in [0, 1].
__device__ __forceinline__ uint64_t portion(float f, uint64_t s, bool* fraction) {
  const uint64_t f64 = static_cast<uint64_t>(static_cast<double>(f) * 18446744073709551616.0);  // f < 1
  *fraction = f64 * s != 0;
  return __umul64hi(f64, s);
}

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_kernel(const SampleArgs a) {
  grid_dependency_wait();
  __shared__ uint64_t scratch[kThreads / 32];
  __shared__ uint64_t shares[kThreads];
  const int tid = threadIdx.x;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
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
      continue;
    }
    const T* x = static_cast<const T*>(a.logits) + row * a.stride;
    const int per = (a.vocab + kThreads - 1) / kThreads;
    const int lo = min(a.vocab, tid * per), hi = min(a.vocab, lo + per);
    uint32_t top = 0;
    for (int i = lo; i < hi; ++i) top = max(top, key_of(load1(x + i)));
    shares[tid] = top;
    __syncthreads();
    for (int w = 0; w < kThreads; ++w) top = max(top, static_cast<uint32_t>(shares[w]));
    __syncthreads();
    const Weigher weigh{logit_of(top), temp > 0.f ? kLog2e / static_cast<double>(temp) : 0.0, exp2(static_cast<double>(a.bits))};
    auto count_from = [&](uint32_t t) {  // logits with a key of at least t
      int n = 0;
      for (int i = lo; i < hi; ++i) n += key_of(load1(x + i)) >= t;
      return block_sum<uint64_t>(n, scratch);
    };
    auto weight_above = [&](uint32_t t) {
      uint64_t w = 0;
      for (int i = lo; i < hi; ++i) {
        const float v = load1(x + i);
        if (key_of(v) > t) w += weigh(logit_of(key_of(v)));
      }
      return block_sum<uint64_t>(w, scratch);
    };
    uint32_t t = 0;            // what stays: keys above t,
    uint64_t ties = a.vocab;   // and the first `ties` equal to it
    if (temp == 0.f) {
      t = top;
      ties = 1;
    } else {
      if (k > 0 && k < a.vocab) {
        for (int bit = 31; bit >= 0; --bit) {
          const uint32_t cand = t | (1u << bit);
          if (count_from(cand) >= static_cast<uint64_t>(k)) t = cand;
        }
        ties = k - (t == 0xffffffffu ? 0 : count_from(t + 1));
      }
      if (p < 1.f) {
        const uint64_t equal = count_from(t) - (t == 0xffffffffu ? 0 : count_from(t + 1));
        const uint64_t sum = weight_above(t) + min(ties, equal) * weigh(logit_of(t));
        bool fraction;
        uint64_t target = portion(max(p, 0.f), sum, &fraction);
        if (fraction || target == 0) ++target;  // stays while the weight before it is below target
        uint32_t lowest = t;
        if (weight_above(t) >= target) {
          // the lowest key whose weight above it is below target, in (t, top]
          uint32_t hi_key = top, lo_key = t;
          while (hi_key - lo_key > 1) {
            const uint32_t mid = lo_key + (hi_key - lo_key) / 2;
            if (weight_above(mid) < target) {
              hi_key = mid;
            } else {
              lo_key = mid;
            }
          }
          lowest = hi_key;
          ties = a.vocab;
        }
        const uint64_t above = weight_above(lowest), w = weigh(logit_of(lowest));
        if (w > 0) ties = min(ties, (target - above + w - 1) / w);
        t = lowest;
      }
    }
    // this thread's indexes: how many tie, then what stays
    uint64_t mine = 0;
    for (int i = lo; i < hi; ++i) mine += key_of(load1(x + i)) == t;
    __syncthreads();
    shares[tid] = mine;
    __syncthreads();
    uint64_t before = 0;
    for (int w = 0; w < tid; ++w) before += shares[w];
    __syncthreads();
    const double least = min(mp, 1.f);
    uint64_t own = 0;
    auto staying = [&](int i, uint64_t* tied) -> uint64_t {
      const uint32_t key = key_of(load1(x + i));
      if (key < t) return 0;
      if (key == t && (*tied)++ >= ties) return 0;
      const double w = weigh.real(logit_of(key));
      return w >= least ? __double2ull_rn(w * weigh.one) : 0;
    };
    uint64_t tied = before;
    for (int i = lo; i < hi; ++i) own += staying(i, &tied);
    shares[tid] = own;
    const uint64_t total = block_sum<uint64_t>(own, scratch);
    bool fraction;
    const uint64_t want = portion(temp == 0.f ? 0.f : u, total, &fraction);
    uint64_t at = 0;
    for (int w = 0; w < tid; ++w) at += shares[w];
    if (logit_of(top) == -INFINITY) {
      if (tid == 0) a.tokens[row] = -1;
    } else if (at <= want && want < at + own) {
      tied = before;
      for (int i = lo; i < hi; ++i) {
        at += staying(i, &tied);
        if (at > want) {
          a.tokens[row] = i;
          break;
        }
      }
    }
    __syncthreads();
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
  if (rows < 0 || rows > INT32_MAX) return fail(BM_ERR_INVALID_ARGUMENT, "%s: bad rows", what);
  if (vocab <= 0 || vocab > (1 << 24)) return fail(BM_ERR_INVALID_ARGUMENT, "%s: vocab outside [1, 2^24]", what);
  if (row_stride < vocab) return fail(BM_ERR_INVALID_ARGUMENT, "%s: row_stride below vocab", what);
  if (rows == 0) return BM_OK;
  if (!tokens || !logits || !uniforms) return fail(BM_ERR_INVALID_ARGUMENT, "%s: NULL pointer", what);
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
  a.bits = 62 - log2_up;
  if (a.bits > 52) a.bits = 52;  // an fp64 weight has no more
  a.status = d_status;
  const dim3 grid(static_cast<unsigned>(std::min<int64_t>(rows, 1 << 16)));
  auto go = [&](auto kernel) { return launch_kernel(what, kernel, grid, dim3(kThreads), 0, as_stream(stream), nullptr, a); };
  return dtype == BM_F32 ? go(sample_kernel<float>) : go(sample_kernel<bf16>);
}
