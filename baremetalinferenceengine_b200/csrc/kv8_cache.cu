// RMSNorm of every head of Q and K and their rotary positions in one pass
// (bm_qk_norm_rotary); the same on the way into a paged cache held in 8 bits, which
// quantises K and V as it writes them (bm_paged_kv8_append); and a stretch of that cache
// read back as dense rows (bm_paged_kv8_read).
//
// Mathematics: per head x of hd elements, with r = rsqrt(mean(x^2) + eps),
//   y = x r w,  then the pairs (a, b) of its first rd elements become (a c - b s, b c + a s),
// fp32 throughout, rounded once at the end: to the storage type, or to e4m3 as
//   code = rne(y 2^-E),  E = max(E before, ceil(log2(max |y| / 448)))
// over the block's new rows and elements of the head. A block with slots of earlier calls
// keeps its scale unless it has to grow; then its earlier codes move with it. (A scale left
// by rows that a later call overwrites is at worst larger than needed, which costs a floating
// code nothing above 2^-6.)
//
// Bound: memory; q, k and v are read once, and q and the codes written once. But where a block has more rows than its job
// holds in registers (in bf16 more than 64 of 128 elements, or 32 of 256; in fp32 half of that; fewer where alignment
// allows only narrower loads), its K and V are read twice.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "kv8.cuh"
#include "rotary_device.cuh"

namespace bm {
namespace {

using namespace bm::rot;
using namespace bm::kv8;

constexpr int kMaxHeadDim = 256;
constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;
constexpr int kAppendThreads = 256;
constexpr int kAppendWarps = kAppendThreads / 32;
// Passes whose loads a lane keeps in flight, of Q's (and norm_rotary's) heads and of K's and V's rows; and the blocks
// that an SM has room for at the registers these take. A prompt's 16384 rows of 64 + 8 heads of 128, us: 4 and 5 blocks
// 114, 4 and 4 123, 2 and 6 116. K and V of 32768 tokens, 8 heads, in one
// kernel: 2 and 2 blocks 118, 1 and 3 154, 4 and 1 146; jobs of several heads, the next one's rows asked for early: no gain.
constexpr int kUQ = 4, kUK = 2;
constexpr int kQBlocks = 5, kKvBlocks = 2, kVBlocks = 3;

struct HeadArgs {
  void* q_out;
  void* k_out;               // norm_rotary only
  const void* q;
  const void* k;
  const void* v;             // append only
  const void* q_weight;      // NULL: no norm
  const void* k_weight;
  const int32_t* positions;  // norm_rotary: NULL = pos0 + row; append: NULL = the slot
  const float2* table;       // NULL: no rotation (append only)
  int64_t rows, q_stride, k_stride, v_stride, q_out_stride, k_out_stride;
  int32_t pos0, table_len;
  float eps;
  int hq, hkv, hd, rd;
  int units, rest;           // rotated and copied units of a head
  int heads_per_pass;        // lanes of a warp hold so many heads, or rows of one
  int parts;                 // warps per row of Q (and K, norm_rotary)
  int32_t* status;
  // append
  bm_paged_kv8_t cache;
  const int32_t* ctx_lens;
  const int32_t* starts;
  const int32_t* seq_ids;
  int64_t batch, kv_ctas;
  int max_tokens, blocks, warps_per_job;
};

// A lane's share of a head: J units of two chunks of N elements. FULL: every lane of a warp has a rotated
// unit (heads of 32, 64, 128 or 256 elements in a power of two of units, all of them rotated), so that nothing of it is asked.
template <int N, int J, bool FULL>
struct Share {
  int first[J], second[J];
  bool own_[J], pair_[J], turns_[J];
  __device__ __forceinline__ bool own(int j) const { return FULL || own_[j]; }
  __device__ __forceinline__ bool pair(int j) const { return FULL || pair_[j]; }
  __device__ __forceinline__ bool turns(int j) const { return FULL || turns_[j]; }
  template <bool INTER>
  __device__ __forceinline__ void place(const HeadArgs& a, int c0, bool live) {
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int c = c0 + 32 * j;
      own_[j] = live && c < a.units + a.rest;
      turns_[j] = c < a.units;
      first[j] = turns(j) ? c * (INTER ? 2 * N : N) : a.rd + (c - a.units) * 2 * N;
      second[j] = first[j] + (turns(j) && !INTER ? a.rd / 2 : N);
      pair_[j] = own(j) && second[j] < a.hd;  // the last copied unit may have one chunk
    }
  }
};

// The sum over the n lanes of a head (lane = head * n + c), for each of them.
__device__ __forceinline__ float head_sum(float v, int c, int n, int lane) {
  if ((n & (n - 1)) == 0) {
    for (int off = n >> 1; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
    return v;
  }
  int region = n;  // the lanes below it hold what is left to add
  for (int off = 16; off > 0; off >>= 1) {
    if (off >= n) continue;
    const float other = __shfl_down_sync(0xffffffffu, v, off);
    if (c < off && c + off < region) v += other;
    region = min(region, off);
  }
  return __shfl_sync(0xffffffffu, v, lane - c);
}

template <typename T, int N, int J, bool FULL>
struct Head {
  Piece<T, N> p1[J], p2[J];

  __device__ __forceinline__ void load(const T* x, const Share<N, J, FULL>& s) {
#pragma unroll
    for (int j = 0; j < J; ++j) {
      if (s.own(j)) p1[j].load(x + s.first[j]);
      if (s.pair(j)) p2[j].load(x + s.second[j]);
    }
  }
  __device__ __forceinline__ void get(float (&x)[J][2 * N], const Share<N, J, FULL>& s) const {
#pragma unroll
    for (int j = 0; j < J; ++j) {
#pragma unroll
      for (int e = 0; e < 2 * N; ++e) x[j][e] = 0.f;
      if (s.own(j)) p1[j].get(x[j]);
      if (s.pair(j)) p2[j].get(x[j] + N);
    }
  }
  __device__ __forceinline__ void set_store(T* to, const float (&x)[J][2 * N], const Share<N, J, FULL>& s) {
#pragma unroll
    for (int j = 0; j < J; ++j) {
      p1[j].set(x[j]);
      p2[j].set(x[j] + N);
      if (s.own(j)) p1[j].store(to + s.first[j]);
      if (s.pair(j)) p2[j].store(to + s.second[j]);
    }
  }
};

// x r w, w unpacked. Every lane of the warp takes part, whether it holds elements or not.
template <int N, int J>
__device__ __forceinline__ void norm(float (&x)[J][2 * N], const float (&w)[J][2 * N], const HeadArgs& a, int c, int n, int lane) {
  uint64_t sum2 = 0;
#pragma unroll
  for (int j = 0; j < J; ++j) {
#pragma unroll
    for (int e = 0; e < 2 * N; e += 2) sum2 = fma2(pair(x[j][e], x[j][e + 1]), pair(x[j][e], x[j][e + 1]), sum2);
  }
  const float2 sums = unpair(sum2);
  const float r = rsqrtf(head_sum(sums.x + sums.y, c, n, lane) / a.hd + a.eps);
  const uint64_t r2 = pair(r, r);
#pragma unroll
  for (int j = 0; j < J; ++j) {
#pragma unroll
    for (int e = 0; e < 2 * N; e += 2) {
      const float2 y = unpair(mul2(mul2(pair(x[j][e], x[j][e + 1]), r2), pair(w[j][e], w[j][e + 1])));
      x[j][e] = y.x;
      x[j][e + 1] = y.y;
    }
  }
}
// The lane's share of a norm's weights, from global or shared memory (Piece::load streams from global memory only).
template <typename T, int N, int J, bool FULL>
__device__ __forceinline__ void load_weight(float (&w)[J][2 * N], const T* weight, const Share<N, J, FULL>& s) {
  using Raw = decltype(Piece<T, N>::raw);
  Head<T, N, J, FULL> raw;
#pragma unroll
  for (int j = 0; j < J; ++j) {
    if (s.own(j)) raw.p1[j].raw = *reinterpret_cast<const Raw*>(weight + s.first[j]);
    if (s.pair(j)) raw.p2[j].raw = *reinterpret_cast<const Raw*>(weight + s.second[j]);
  }
  raw.get(w, s);
}

template <int N, int J, bool FULL>
struct Angles {
  float2 cs[J][N];
  __device__ __forceinline__ void load(const HeadArgs& a, int pos, int c0, const Share<N, J, FULL>& s) {
    const float2* t = a.table + static_cast<int64_t>(pos) * (a.rd / 2);
#pragma unroll
    for (int j = 0; j < J; ++j) {
      if (s.own(j) && s.turns(j)) load_angles<N>(t + (c0 + 32 * j) * N, cs[j]);
    }
  }
};
template <int N, int J, bool INTER, bool FULL>
__device__ __forceinline__ void turn(float (&x)[J][2 * N], const Angles<N, J, FULL>& t, const Share<N, J, FULL>& s) {
#pragma unroll
  for (int j = 0; j < J; ++j) {
    if (s.own(j) && s.turns(j)) {
      if constexpr (!INTER && N % 2 == 0) {
        rotate2<N>(x[j], t.cs[j]);
      } else {
        rotate<N, INTER>(x[j], t.cs[j]);
      }
    }
  }
}

// The weights of Q's and K's norms as a block keeps them, in shared memory (a lane's share of either would take
// a dozen registers): q's hd elements, then k's.
template <typename T>
__device__ __forceinline__ void stage_weights(T* to, const HeadArgs& a, int threads) {
  for (int i = threadIdx.x; i < 2 * a.hd; i += threads) {
    const T* w = static_cast<const T*>(i < a.hd ? a.q_weight : a.k_weight);
    if (w != nullptr) to[i < a.hd ? i : i - a.hd + kMaxHeadDim] = w[i < a.hd ? i : i - a.hd];
  }
  __syncthreads();
}

// One warp's share of a row's heads: part `part` of a.parts of Q's heads and, behind them, `hkv` of K's.
template <typename T, int N, int J, bool INTER, bool FULL>
__device__ __forceinline__ void turn_heads(const HeadArgs& a, int64_t row, int hkv, int part, bool normed, const T* weights, int pos, int lane) {
  const int n = min(32, a.units + a.rest), hpi = a.heads_per_pass, heads = a.hq + hkv;
  const int hl = lane / n, c = lane - hl * n;
  Share<N, J, FULL> s;
  s.template place<INTER>(a, c, hl < hpi);
  const int passes = (heads + hpi - 1) / hpi, mine = (passes + a.parts - 1) / a.parts;
  const int h_end = min(heads, (part + 1) * mine * hpi);
  if (part * mine * hpi >= h_end) return;
  const T* q = static_cast<const T*>(a.q) + row * a.q_stride;
  const T* k = static_cast<const T*>(a.k) + row * a.k_stride;
  T* q_out = static_cast<T*>(a.q_out) + row * a.q_out_stride;
  T* k_out = static_cast<T*>(a.k_out) + row * a.k_out_stride;
  Angles<N, J, FULL> t;
  bool have = false;
  for (int hb = part * mine * hpi; hb < h_end; hb += hpi * kUQ) {  // the same for the warp
    Head<T, N, J, FULL> x[kUQ];
#pragma unroll
    for (int u = 0; u < kUQ; ++u) {
      const int h = hb + u * hpi + hl;
      if (h < h_end) x[u].load(h < a.hq ? q + h * a.hd : k + (h - a.hq) * a.hd, s);
    }
    if (!have) {
      if (a.table) t.load(a, pos, c, s);
      have = true;
    }
#pragma unroll
    for (int u = 0; u < kUQ; ++u) {
      const int h = hb + u * hpi + hl;
      if (hb + u * hpi >= h_end) break;
      float y[J][2 * N];
      x[u].get(y, s);
      if (normed) {
        float w[J][2 * N];
        load_weight<T, N, J, FULL>(w, weights + (h < a.hq ? 0 : kMaxHeadDim), s);
        norm<N, J>(y, w, a, c, n, lane);
      }
      if (a.table) turn<N, J, INTER, FULL>(y, t, s);
      if (h < h_end) x[u].set_store(h < a.hq ? q_out + h * a.hd : k_out + (h - a.hq) * a.hd, y, s);
    }
  }
}

template <typename T, int N, int J, bool INTER, bool FULL>
__global__ void __launch_bounds__(kThreads, kQBlocks) norm_rotary_kernel(const __grid_constant__ HeadArgs a) {
  grid_dependency_wait();
  __shared__ __align__(16) T weights[2 * kMaxHeadDim];
  const int lane = threadIdx.x & 31;
  const int64_t job = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  const int64_t row = job / a.parts;
  const int part = static_cast<int>(job - row * a.parts);
  const int32_t pos = row >= a.rows ? 0 : a.positions ? __ldg(a.positions + row) : static_cast<int32_t>(a.pos0 + row);
  stage_weights(weights, a, kThreads);
  if (row >= a.rows) return;
  if (pos < 0 || pos >= a.table_len) {
    if (lane == 0) raise_status(a.status, BM_DEVERR_BAD_POSITION);
    return;
  }
  turn_heads<T, N, J, INTER, FULL>(a, row, a.hkv, part, true, weights, pos, lane);
}

// A sequence of the batch: its cache sequence, cached slots, new rows and the first of them.
struct Span {
  int seq, ctx, n;
  int64_t row0;
};
// Reads and checks sequence b (starts[b], starts[b + 1], first[b], seq_ids[b]): its rows go
// to the slots from `first` on. The BM_DEVERR_* bits are 0 when it is sound.
__device__ __forceinline__ int32_t read_span(const bm_paged_kv8_t& c, const int32_t* starts, const int32_t* first,
                                             const int32_t* seq_ids, int64_t rows, int most, int64_t b, Span* s) {
  const int32_t r0 = __ldg(starts + b), r1 = __ldg(starts + b + 1);
  s->ctx = __ldg(first + b);
  s->seq = seq_ids ? __ldg(seq_ids + b) : static_cast<int>(b);
  s->row0 = r0;
  const int64_t n = static_cast<int64_t>(r1) - r0;
  s->n = static_cast<int>(n);
  int32_t bad = 0;
  if (r0 < 0 || r1 > rows || n < 0 || n > most || s->ctx < 0 || (n > 0 && s->ctx + n > static_cast<int64_t>(c.max_pages) * c.page_size)) {
    bad |= BM_DEVERR_BAD_POSITION;
  }
  if (s->seq < 0 || s->seq >= c.num_seqs) bad |= BM_DEVERR_BAD_SEQUENCE;
  if (bad) s->n = 0;
  return bad;
}

// N codes to memory.
template <int N>
__device__ __forceinline__ void store_codes(uint8_t* to, const float* x, float f) {
  if constexpr (N == 1) {
    *to = static_cast<uint8_t>(to_codes(x[0] * f, 0.f));
  } else {
    uint32_t w[N / 4];
#pragma unroll
    for (int e = 0; e < N; e += 4) w[e / 4] = to_codes(x[e] * f, x[e + 1] * f) | to_codes(x[e + 2] * f, x[e + 3] * f) << 16;
    if constexpr (N == 8) {
      *reinterpret_cast<uint2*>(to) = make_uint2(w[0], w[1]);
    } else {
      *reinterpret_cast<uint32_t*>(to) = w[0];
    }
  }
}

// One warp's share of a token's Q on the way of an append.
template <typename T, int N, int J, bool INTER, bool FULL>
__device__ __forceinline__ void append_q(const HeadArgs& a, int64_t job, const T* weights, int lane) {
  const int64_t token = job / a.parts;
  const int part = static_cast<int>(job - token * a.parts);
  const int64_t b = token / a.max_tokens;
  const int j = static_cast<int>(token - b * a.max_tokens);
  if (b >= a.batch) return;
  Span s;
  if (read_span(a.cache, a.starts, a.ctx_lens, a.seq_ids, a.rows, a.max_tokens, b, &s) || j >= s.n) return;
  const int64_t row = s.row0 + j;
  const int32_t pos = a.positions ? __ldg(a.positions + row) : s.ctx + j;
  if (a.table && (pos < 0 || pos >= a.table_len)) return;  // K's and V's jobs tell
  turn_heads<T, N, J, INTER, FULL>(a, row, 0, part, a.q_weight != nullptr, weights, pos, lane);
}
template <typename T, int N, int J, bool INTER, bool FULL>
__global__ void __launch_bounds__(kThreads, kQBlocks) append_q_kernel(const __grid_constant__ HeadArgs a) {
  grid_dependency_wait();
  __shared__ __align__(16) T weights[2 * kMaxHeadDim];
  if (a.q_weight) stage_weights(weights, a, kThreads);
  append_q<T, N, J, INTER, FULL>(a, static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5), weights, threadIdx.x & 31);
}

// What a launch appends: all of a call, or K or V alone.
enum class Jobs { kAll, kK, kV };

// The first kv_ctas blocks take K and V: one job is K or V of one head in one block of slots,
// held by warps_per_job warps of a block. A lane group holds a row, so the norm is a sum over a group and the scale a
// maximum over the warp, then over the job's warps. The other blocks rotate Q.
template <typename T, int N, int J, bool INTER, bool FULL, Jobs JOBS>
__global__ void __launch_bounds__(kAppendThreads, JOBS == Jobs::kV ? kVBlocks : kKvBlocks) append_kernel(const __grid_constant__ HeadArgs a) {
  grid_dependency_wait();
  __shared__ uint32_t tops[kAppendWarps];
  __shared__ __align__(16) T weights[2 * kMaxHeadDim];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const bm_paged_kv8_t& c8 = a.cache;
  if (JOBS == Jobs::kAll && blockIdx.x >= a.kv_ctas) {
    if (a.q_weight) stage_weights(weights, a, kAppendThreads);
    append_q<T, N, J, INTER, FULL>(a, (static_cast<int64_t>(blockIdx.x) - a.kv_ctas) * kAppendWarps + warp, weights, lane);
    return;
  }
  // ---------------- K and V ----------------
  const int wpj = a.warps_per_job, sub = warp % wpj;
  const int64_t job = static_cast<int64_t>(blockIdx.x) * (kAppendWarps / wpj) + warp / wpj;
  const int kinds = JOBS == Jobs::kAll ? 2 * a.hkv : a.hkv;
  const int which = static_cast<int>(job % kinds);
  const int head = JOBS == Jobs::kAll ? which >> 1 : which;
  const bool is_v = JOBS == Jobs::kAll ? which & 1 : JOBS == Jobs::kV;
  const int64_t bj = job / kinds, b = bj / a.blocks;
  const int jb = static_cast<int>(bj - b * a.blocks);
  Span s{};
  int lo = 0, hi = 0, begin = 0;     // the block's new slots; its first slot
  uint8_t *pages = nullptr, *scale = nullptr;
  bool active = b < a.batch;
  if (active) {
    const int32_t bad = read_span(c8, a.starts, a.ctx_lens, a.seq_ids, a.rows, a.max_tokens, b, &s);
    if (bad && jb == 0 && which == 0 && !is_v && lane == 0 && sub == 0) raise_status(a.status, bad);
    // 64 bits: a block's end may pass the last slot there can be
    const int64_t from = (static_cast<int64_t>(s.ctx / c8.block) + jb) * c8.block;
    lo = static_cast<int>(max(static_cast<int64_t>(s.ctx), min(from, static_cast<int64_t>(s.ctx) + s.n)));
    hi = static_cast<int>(min(static_cast<int64_t>(s.ctx) + s.n, from + c8.block));
    active = !bad && lo < hi;
    begin = static_cast<int>(active ? from : 0);
  }
  if (!active) lo = hi = 0;
  const int n = min(32, a.units + a.rest), rpi = a.heads_per_pass;
  const int rl = lane / n, c = lane - rl * n;
  Share<N, J, FULL> sh;
  sh.template place<INTER>(a, c, rl < rpi);
  const T* src = static_cast<const T*>(is_v ? a.v : a.k) + static_cast<int64_t>(head) * a.hd;
  const int64_t stride = is_v ? a.v_stride : a.k_stride;
  const bool normed = !is_v && a.k_weight, turned = !is_v && a.table;

  // Batches of kUK passes, of rpi rows each, in turn over the job's warps. One batch stays in
  // registers until its scale is known; more are read again. The first one's loads are on their way before
  // the chain of page and scale is walked.
  const int step = kUK * rpi * wpj;
  Head<T, N, J, FULL> x[kUK];
  int32_t pos[kUK];
  float y[kUK][J][2 * N];
  bool good[kUK];
  auto fetch = [&](int from) {
#pragma unroll
    for (int u = 0; u < kUK; ++u) {
      const int slot = from + (sub * kUK + u) * rpi + rl;
      good[u] = active && slot < hi && (FULL || rl < rpi);
      const int64_t r = s.row0 + (slot - s.ctx);
      if (good[u]) x[u].load(src + r * stride, sh);
      pos[u] = good[u] && a.table && a.positions ? __ldg(a.positions + r) : slot;
    }
  };
  fetch(lo);
  float w[J][2 * N];
  if (normed && active) load_weight<T, N, J, FULL>(w, static_cast<const T*>(a.k_weight), sh);
  if (active) {
    const int nth = begin / c8.page_size;
    const int32_t page = __ldg(c8.page_table + static_cast<int64_t>(s.seq) * c8.max_pages + nth);
    if (page < 0 || page >= c8.num_pages) {
      if (lane == 0 && sub == 0) raise_status(a.status, BM_DEVERR_BAD_PAGE);
      active = false;
      lo = hi = 0;
#pragma unroll
      for (int u = 0; u < kUK; ++u) good[u] = false;
    } else {
      const int64_t ph = static_cast<int64_t>(page) * a.hkv + head;
      const int off = begin - nth * c8.page_size;
      pages = static_cast<uint8_t*>(is_v ? c8.v_pages : c8.k_pages) + (ph * c8.page_size + off) * a.hd;
      scale = static_cast<uint8_t*>(is_v ? c8.v_scales : c8.k_scales) + ph * (c8.page_size / c8.block) + off / c8.block;
    }
  }
  // A block with slots of earlier calls has a scale: read here, since the job's first warp
  // writes it at its own end, behind the barrier.
  const bool keeps = active && begin < s.ctx;
  const int before = keeps ? exponent(*scale) : kLowest;

  uint32_t top = 0;
  int bad_position = 0;
  auto compute = [&]() {
#pragma unroll
    for (int u = 0; u < kUK; ++u) {
      if (a.table && good[u] && (pos[u] < 0 || pos[u] >= a.table_len)) {  // V, too, leaves out the rows whose position is bad
        good[u] = false;
        bad_position = 1;
      }
      Angles<N, J, FULL> t;
      if (turned && good[u]) t.load(a, pos[u], c, sh);
      x[u].get(y[u], sh);
      if (normed) norm<N, J>(y[u], w, a, c, n, lane);
      if (turned && good[u]) turn<N, J, INTER, FULL>(y[u], t, sh);
    }
  };
  // The lane's largest finite magnitude (elements that it does not own are 0); what is not finite becomes NaN and
  // sets no scale.
  auto examine = [&]() {
    uint32_t most = 0;
#pragma unroll
    for (int u = 0; u < kUK; ++u) {
      uint32_t m = 0;
#pragma unroll
      for (int j = 0; j < J; ++j) {
#pragma unroll
        for (int e = 0; e < 2 * N; ++e) m = max(m, magnitude(y[u][j][e]));
      }
      if (!good[u]) m = 0;
      if (m >= kNotFinite) {
        m = 0;
#pragma unroll
        for (int j = 0; j < J; ++j) {
#pragma unroll
          for (int e = 0; e < 2 * N; ++e) {
            if (magnitude(y[u][j][e]) >= kNotFinite) {
              y[u][j][e] = __int_as_float(0x7fffffff);
            } else {
              m = max(m, magnitude(y[u][j][e]));
            }
          }
        }
      }
      most = max(most, m);
    }
    return most;
  };
  const int batches = (hi - lo + step - 1) / step;
  for (int i = 0; i < batches; ++i) {
    if (i > 0) fetch(lo + i * step);
    compute();
    top = max(top, examine());
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if (wpj > 1) {
    if (lane == 0) tops[warp] = top;
    __syncthreads();
    for (int i = 0; i < wpj; ++i) top = max(top, tops[warp - sub + i]);
  }
  if (bad_position) raise_status(a.status, BM_DEVERR_BAD_POSITION);
  if (!active) return;
  const int e = max(exponent_for(top), before);
  if (keeps && e > before) {
    const float f = power(before - e);
    const int chunks = (s.ctx - begin) * (a.hd / 16);
    for (int i = sub * 32 + lane; i < chunks; i += wpj * 32) {
      uint4* at = reinterpret_cast<uint4*>(pages) + i;
      uint4 raw = *at;
      uint32_t* words = &raw.x;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float v[4];
        from_codes(words[k], v);
        words[k] = to_codes(v[0] * f, v[1] * f) | to_codes(v[2] * f, v[3] * f) << 16;
      }
      *at = raw;
    }
  }
  const float f = power(-e);
  for (int i = 0; i < batches; ++i) {
    if (batches > 1) {
      fetch(lo + i * step);
      compute();
      examine();
    }
#pragma unroll
    for (int u = 0; u < kUK; ++u) {
      const int slot = lo + i * step + (sub * kUK + u) * rpi + rl;
      uint8_t* to = pages + static_cast<int64_t>(slot - begin) * a.hd;
#pragma unroll
      for (int j = 0; j < J; ++j) {
        if (good[u] && sh.own(j)) store_codes<N>(to + sh.first[j], y[u][j], f);
        if (good[u] && sh.pair(j)) store_codes<N>(to + sh.second[j], y[u][j] + N, f);
      }
    }
  }
  if (lane == 0 && sub == 0) *scale = static_cast<uint8_t>(e + 127);
}

struct ReadArgs {
  void* k_out;
  void* v_out;
  bm_paged_kv8_t cache;
  const int32_t* first;
  const int32_t* starts;
  const int32_t* seq_ids;
  int64_t rows, batch;
  int max_rows, chunks;  // the most rows of a sequence; jobs of them
  int32_t* status;
};

// 16 values to memory, past the caches' other contents. (Neighbouring lanes that swap halves, so that each store
// fills whole sectors, are 3 % faster on even batches and 20 % slower on uneven ones.)
template <typename T>
__device__ __forceinline__ void store16(T* to, const uint4& codes, float f) {
  float v[16];
  from_codes(codes.x, v);
  from_codes(codes.y, v + 4);
  from_codes(codes.z, v + 8);
  from_codes(codes.w, v + 12);
#pragma unroll
  for (int e = 0; e < 16; ++e) v[e] *= f;
#pragma unroll
  for (int e = 0; e < 16; e += VecWidth<T>::value) st_stream(to + e, pack16<T>(v + e));
}

constexpr int kReadU = 4;
// A warp takes K and V of one head in kReadU passes of rows; a lane 16 codes of each.
template <typename T>
__global__ void __launch_bounds__(kThreads) read_kernel(const __grid_constant__ ReadArgs a) {
  grid_dependency_wait();
  const bm_paged_kv8_t& c8 = a.cache;
  const int lane = threadIdx.x & 31;
  const int64_t job = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  const int head = static_cast<int>(job % c8.num_kv_heads);
  const int64_t rest = job / c8.num_kv_heads, b = rest / a.chunks;
  const int chunk = static_cast<int>(rest - b * a.chunks);
  if (b >= a.batch) return;
  Span s;
  const int32_t bad = read_span(c8, a.starts, a.first, a.seq_ids, a.rows, a.max_rows, b, &s);
  if (bad) {
    if (chunk == 0 && head == 0 && lane == 0) raise_status(a.status, bad);
    return;
  }
  const int n = c8.head_dim / 16, rpi = 32 / n;  // lanes of a row, rows of a pass
  const int rl = lane / n, c = lane - rl * n;
  const int64_t i0 = static_cast<int64_t>(chunk) * (kReadU * rpi) + rl;
  if (rl >= rpi) return;
  uint4 k[kReadU], v[kReadU];
  float kf[kReadU], vf[kReadU];
  bool good[kReadU];
#pragma unroll
  for (int u = 0; u < kReadU; ++u) {
    const int64_t i = i0 + u * rpi;
    good[u] = i < s.n;
    if (good[u]) {
      const int slot = static_cast<int>(s.ctx + i), nth = slot / c8.page_size;
      const int32_t page = __ldg(c8.page_table + static_cast<int64_t>(s.seq) * c8.max_pages + nth);
      good[u] = page >= 0 && page < c8.num_pages;
      if (good[u]) {
        const int64_t ph = static_cast<int64_t>(page) * c8.num_kv_heads + head;
        const int off = slot - nth * c8.page_size;
        const int64_t at = (ph * c8.page_size + off) * c8.head_dim + c * 16;
        const int64_t sc = ph * (c8.page_size / c8.block) + off / c8.block;
        k[u] = ld_stream(static_cast<const uint8_t*>(c8.k_pages) + at);
        v[u] = ld_stream(static_cast<const uint8_t*>(c8.v_pages) + at);
        kf[u] = power(exponent(static_cast<const uint8_t*>(c8.k_scales)[sc]));
        vf[u] = power(exponent(static_cast<const uint8_t*>(c8.v_scales)[sc]));
      } else if (c == 0) {
        raise_status(a.status, BM_DEVERR_BAD_PAGE);
      }
    }
  }
#pragma unroll
  for (int u = 0; u < kReadU; ++u) {
    if (!good[u]) continue;
    const int64_t to = ((s.row0 + i0 + u * rpi) * c8.num_kv_heads + head) * c8.head_dim + c * 16;
    store16(static_cast<T*>(a.k_out) + to, k[u], kf[u]);
    store16(static_cast<T*>(a.v_out) + to, v[u], vf[u]);
  }
}

// Sets the units of a head and calls go(N, J): the widest chunk that divides every run of
// elements and suits every pointer and stride, as rotary.cu picks it: 16 bytes, 8 (bf16),
// else single elements, of which a lane holds up to four pairs.
template <typename F>
int with_chunk(HeadArgs* a, bm_dtype_t dtype, F go) {
  const int es = dtype_size(dtype);
  auto fits = [&](int n) {
    if ((a->rd / 2) % n || (a->hd - a->rd) % n || a->hd % n) return false;
    const uintptr_t bytes = static_cast<uintptr_t>(n) * es;
    for (const void* p : {a->q, a->k, a->v, static_cast<const void*>(a->q_out), static_cast<const void*>(a->k_out), a->q_weight, a->k_weight}) {
      if (reinterpret_cast<uintptr_t>(p) % bytes) return false;
    }
    for (int64_t s : {a->q_stride, a->k_stride, a->v_stride, a->q_out_stride, a->k_out_stride}) {
      if (s % n) return false;
    }
    return n % 2 != 0 || aligned16(a->table);
  };
  int n = 16 / es;
  if (!fits(n)) n = es == 2 && fits(4) ? 4 : 1;
  a->units = a->rd / 2 / n;
  a->rest = (a->hd - a->rd + 2 * n - 1) / (2 * n);
  a->heads_per_pass = 32 / std::min(32, a->units + a->rest);
  return go(n);
}

// Warps of a row of heads: one where the rows fill the GPU (2048 warps: 14 per SM), else up to 8.
int parts_for(int64_t rows) {
  return static_cast<int>(std::min<int64_t>(8, std::max<int64_t>(1, 2048 / std::max<int64_t>(1, rows))));
}

int check_heads(const char* what, int64_t rows, int hq, int hkv, int hd) {
  if (rows < 0 || rows > INT32_MAX || hq < 0 || hkv < 0 || hq > (1 << 16) || hkv > (1 << 16)) {
    return fail(BM_ERR_INVALID_ARGUMENT, "%s: bad rows or head count", what);
  }
  if (hd <= 0 || hd > kMaxHeadDim) return fail(BM_ERR_INVALID_ARGUMENT, "%s: head_dim %d outside [1, %d]", what, hd, kMaxHeadDim);
  return BM_OK;
}
int check_eps(const char* what, float eps) {
  if (!(eps >= 0.f) || !std::isfinite(eps)) return fail(BM_ERR_INVALID_ARGUMENT, "%s: eps must be finite and >= 0", what);
  return BM_OK;
}
// Whether the weights of a norm (hd elements, or NULL) meet an output.
bool meets_weight(const Rows& out, const void* w, int hd, int64_t rows, int es) {
  if (w == nullptr || out.p == nullptr || out.n == 0) return false;
  const uintptr_t o = reinterpret_cast<uintptr_t>(out.p), i = reinterpret_cast<uintptr_t>(w);
  return o < i + static_cast<uintptr_t>(hd) * es && i < o + static_cast<uintptr_t>((rows - 1) * out.stride + out.n) * es;
}

}  // namespace

int check_paged_kv8(const char* what, const bm_paged_kv8_t* c) {
  if (!c) return fail(BM_ERR_INVALID_ARGUMENT, "%s: NULL cache", what);
  if (!c->k_pages || !c->v_pages || !c->k_scales || !c->v_scales || !c->page_table) {
    return fail(BM_ERR_INVALID_ARGUMENT, "%s: NULL pointer in the cache", what);
  }
  if (c->num_pages <= 0 || c->page_size <= 0 || c->block <= 0 || c->max_pages <= 0 || c->num_seqs <= 0 || c->num_kv_heads <= 0 ||
      c->num_kv_heads > (1 << 16)) {
    return fail(BM_ERR_INVALID_ARGUMENT, "%s: bad sizes in the cache", what);
  }
  if (c->head_dim <= 0 || c->head_dim > kMaxHeadDim || c->head_dim % 16) {
    return fail(BM_ERR_INVALID_ARGUMENT, "%s: head_dim %d of an 8-bit cache must be a multiple of 16 up to %d", what, c->head_dim, kMaxHeadDim);
  }
  if (c->page_size % c->block) return fail(BM_ERR_INVALID_ARGUMENT, "%s: block %d does not divide page_size %d", what, c->block, c->page_size);
  if (static_cast<int64_t>(c->page_size) * c->max_pages > INT32_MAX - 4095) {  // a pass may look past a sequence's last slot
    return fail(BM_ERR_INVALID_ARGUMENT, "%s: page_size * max_pages above 2^31 - 4096", what);
  }
  if (!aligned16(c->k_pages) || !aligned16(c->v_pages)) return fail(BM_ERR_INVALID_ARGUMENT, "%s: pages must be 16-byte aligned", what);
  if (!aligned_to(c->page_table, 4)) return fail(BM_ERR_INVALID_ARGUMENT, "%s: a pointer is not aligned to its elements", what);
  return BM_OK;
}

bool meets_pages8(const bm_paged_kv8_t& c, const void* p, uintptr_t bytes) {
  const uintptr_t from = reinterpret_cast<uintptr_t>(p);
  const uintptr_t slots = static_cast<uintptr_t>(c.num_pages) * c.num_kv_heads * c.page_size;
  auto meets = [&](const void* q, uintptr_t n) {
    const uintptr_t lo = reinterpret_cast<uintptr_t>(q);
    return from < lo + n && lo < from + bytes;
  };
  return meets(c.k_pages, slots * c.head_dim) || meets(c.v_pages, slots * c.head_dim) || meets(c.k_scales, slots / c.block) ||
         meets(c.v_scales, slots / c.block);
}

}  // namespace bm

extern "C" int bm_qk_norm_rotary(void* q_out, void* k_out, const void* q, const void* k, const void* q_weight, const void* k_weight,
                                 float eps, const int32_t* positions, int32_t pos0, const void* table, int32_t table_len,
                                 int32_t rotary_dim, int32_t interleaved, int64_t rows, int32_t num_q_heads, int32_t num_kv_heads,
                                 int32_t head_dim, int64_t q_stride, int64_t k_stride, int64_t q_out_stride, int64_t k_out_stride,
                                 bm_dtype_t dtype, int32_t* d_status, void* stream) {
  using namespace bm;
  const char* what = "bm_qk_norm_rotary";
  if (!valid_dtype(dtype)) return fail(BM_ERR_INVALID_ARGUMENT, "%s: bad dtype %d", what, static_cast<int>(dtype));
  if (int st = check_heads(what, rows, num_q_heads, num_kv_heads, head_dim)) return st;
  if (int st = check_eps(what, eps)) return st;
  if (!table) return fail(BM_ERR_INVALID_ARGUMENT, "%s: NULL table", what);
  if (int st = check_rotation(what, table, table_len, rotary_dim, head_dim)) return st;
  if (rows == 0 || (num_q_heads == 0 && num_kv_heads == 0)) return BM_OK;
  if ((num_q_heads > 0 && (!q || !q_out || !q_weight)) || (num_kv_heads > 0 && (!k || !k_out || !k_weight))) {
    return fail(BM_ERR_INVALID_ARGUMENT, "%s: NULL pointer", what);
  }
  const int64_t qn = static_cast<int64_t>(num_q_heads) * head_dim, kn = static_cast<int64_t>(num_kv_heads) * head_dim;
  if ((qn && (q_stride < qn || q_out_stride < qn)) || (kn && (k_stride < kn || k_out_stride < kn))) {
    return fail(BM_ERR_INVALID_ARGUMENT, "%s: a row stride below heads * head_dim", what);
  }
  if (!positions && (pos0 < 0 || pos0 + rows > INT32_MAX)) return fail(BM_ERR_INVALID_ARGUMENT, "%s: bad pos0", what);
  const int es = dtype_size(dtype);
  if (!aligned_to({q, k, q_out, k_out, q_weight, k_weight}, es) || !aligned_to({positions, d_status}, 4)) {
    return fail(BM_ERR_INVALID_ARGUMENT, "%s: a pointer is not aligned to its elements", what);
  }
  const Rows qi{q, q_stride, qn}, ki{k, k_stride, kn}, qo{q_out, q_out_stride, qn}, ko{k_out, k_out_stride, kn};
  if ((meet(qo, qi, rows, es) && !same(qo, qi, rows)) || (meet(ko, ki, rows, es) && !same(ko, ki, rows)) ||
      meet(qo, ki, rows, es) || meet(ko, qi, rows, es) || meet(qo, ko, rows, es)) {
    return fail(BM_ERR_INVALID_ARGUMENT, "%s: an output overlaps an input or the other output", what);
  }
  for (const void* w : {num_q_heads ? q_weight : nullptr, num_kv_heads ? k_weight : nullptr}) {
    if (meets_weight(qo, w, head_dim, rows, es) || meets_weight(ko, w, head_dim, rows, es)) {
      return fail(BM_ERR_INVALID_ARGUMENT, "%s: an output overlaps a weight", what);
    }
  }
  HeadArgs a{};
  if (num_q_heads) {
    a.q_out = q_out;
    a.q = q;
    a.q_weight = q_weight;
    a.q_stride = q_stride;
    a.q_out_stride = q_out_stride;
  }
  if (num_kv_heads) {
    a.k_out = k_out;
    a.k = k;
    a.k_weight = k_weight;
    a.k_stride = k_stride;
    a.k_out_stride = k_out_stride;
  }
  a.eps = eps;
  a.positions = positions;
  a.pos0 = pos0;
  a.table = static_cast<const float2*>(table);
  a.table_len = table_len;
  a.rd = rotary_dim;
  a.rows = rows;
  a.hq = num_q_heads;
  a.hkv = num_kv_heads;
  a.hd = head_dim;
  a.status = d_status;
  a.parts = parts_for(rows);
  const int64_t blocks = (rows * a.parts + kWarps - 1) / kWarps;
  return with_chunk(&a, dtype, [&](int n) {
    const bool full = a.rest == 0 && 32 % a.units == 0;
    auto go = [&](auto kernel) {
      return launch_kernel(what, kernel, dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0, as_stream(stream), nullptr, a);
    };
    auto pick = [&](auto inter) {
      constexpr bool I = decltype(inter)::value;
      if (dtype == BM_F32) {
        if (n == 4) return full ? go(norm_rotary_kernel<float, 4, 1, I, true>) : go(norm_rotary_kernel<float, 4, 1, I, false>);
        return go(norm_rotary_kernel<float, 1, 4, I, false>);
      }
      if (n == 8) return full ? go(norm_rotary_kernel<bf16, 8, 1, I, true>) : go(norm_rotary_kernel<bf16, 8, 1, I, false>);
      if (n == 4) return go(norm_rotary_kernel<bf16, 4, 1, I, false>);
      return go(norm_rotary_kernel<bf16, 1, 4, I, false>);
    };
    return interleaved ? pick(std::true_type{}) : pick(std::false_type{});
  });
}

extern "C" int bm_paged_kv8_append(void* q_out, const void* q, const void* k, const void* v, const void* q_weight,
                                   const void* k_weight, float eps, const int32_t* positions, const bm_paged_kv8_t* cache,
                                   const int32_t* seq_ids, const int32_t* ctx_lens, const int32_t* q_starts, const void* table,
                                   int32_t table_len, int32_t rotary_dim, int32_t interleaved, int64_t rows, int64_t batch,
                                   int32_t num_q_heads, int32_t max_tokens, int64_t q_stride, int64_t k_stride, int64_t v_stride,
                                   int64_t q_out_stride, bm_dtype_t dtype, int32_t* d_status, void* stream) {
  using namespace bm;
  const char* what = "bm_paged_kv8_append";
  if (!valid_dtype(dtype)) return fail(BM_ERR_INVALID_ARGUMENT, "%s: bad dtype %d", what, static_cast<int>(dtype));
  if (int st = check_paged_kv8(what, cache)) return st;
  const bm_paged_kv8_t& c = *cache;
  if (int st = check_heads(what, rows, num_q_heads, c.num_kv_heads, c.head_dim)) return st;
  if (int st = check_eps(what, eps)) return st;
  if (batch < 0 || batch > INT32_MAX || max_tokens < 0) return fail(BM_ERR_INVALID_ARGUMENT, "%s: bad batch or max_tokens", what);
  if (table) {
    if (int st = check_rotation(what, table, table_len, rotary_dim, c.head_dim)) return st;
  }
  if (rows == 0 || batch == 0 || max_tokens == 0) return BM_OK;
  if (!k || !v || !ctx_lens || !q_starts || (num_q_heads > 0 && (!q || !q_out))) return fail(BM_ERR_INVALID_ARGUMENT, "%s: NULL pointer", what);
  if (!seq_ids && batch > c.num_seqs) return fail(BM_ERR_INVALID_ARGUMENT, "%s: more sequences than the cache holds", what);
  const int64_t qn = static_cast<int64_t>(num_q_heads) * c.head_dim, kn = static_cast<int64_t>(c.num_kv_heads) * c.head_dim;
  if ((qn && (q_stride < qn || q_out_stride < qn)) || k_stride < kn || v_stride < kn) {
    return fail(BM_ERR_INVALID_ARGUMENT, "%s: a row stride below heads * head_dim", what);
  }
  const int es = dtype_size(dtype);
  if (!aligned_to({q, k, v, q_out, q_weight, k_weight}, es) || !aligned_to({positions, seq_ids, ctx_lens, q_starts, d_status}, 4)) {
    return fail(BM_ERR_INVALID_ARGUMENT, "%s: a pointer is not aligned to its elements", what);
  }
  const Rows qi{q, q_stride, qn}, qo{q_out, q_out_stride, qn}, ki{k, k_stride, kn}, vi{v, v_stride, kn};
  if ((meet(qo, qi, rows, es) && !same(qo, qi, rows)) || meet(qo, ki, rows, es) || meet(qo, vi, rows, es) ||
      meets_weight(qo, q_weight, c.head_dim, rows, es) || meets_weight(qo, k_weight, c.head_dim, rows, es)) {
    return fail(BM_ERR_INVALID_ARGUMENT, "%s: q_out overlaps an input", what);
  }
  auto in_cache = [&](const Rows& r) { return r.n != 0 && meets_pages8(c, r.p, static_cast<uintptr_t>((rows - 1) * r.stride + r.n) * es); };
  if (in_cache(qo) || in_cache(qi) || in_cache(ki) || in_cache(vi)) {
    return fail(BM_ERR_INVALID_ARGUMENT, "%s: q, k, v or q_out overlaps the cache", what);
  }
  max_tokens = static_cast<int32_t>(std::min<int64_t>(max_tokens, rows));  // no sequence has more
  HeadArgs a{};
  if (num_q_heads) {
    a.q_out = q_out;
    a.q = q;
    a.q_weight = q_weight;
    a.q_stride = q_stride;
    a.q_out_stride = q_out_stride;
  }
  a.k = k;
  a.v = v;
  a.k_weight = k_weight;
  a.k_stride = k_stride;
  a.v_stride = v_stride;
  a.eps = eps;
  a.positions = positions;
  a.table = static_cast<const float2*>(table);
  a.table_len = table_len;
  a.rd = table ? rotary_dim : 0;
  a.rows = rows;
  a.hq = num_q_heads;
  a.hkv = c.num_kv_heads;
  a.hd = c.head_dim;
  a.status = d_status;
  a.cache = c;
  a.ctx_lens = ctx_lens;
  a.starts = q_starts;
  a.seq_ids = seq_ids;
  a.batch = batch;
  a.max_tokens = max_tokens;
  a.blocks = static_cast<int>((static_cast<int64_t>(max_tokens) - 1 + c.block - 1) / c.block + 1);  // that max_tokens neighbouring slots can meet
  const int64_t most_rows = std::min<int64_t>(rows, batch * static_cast<int64_t>(max_tokens));
  a.parts = parts_for(most_rows);
  return with_chunk(&a, dtype, [&](int n) {
    // A warp holds kUK passes of a block's rows in registers (of 128 elements in bf16: 8 rows); the widest blocks are
    // read twice.
    const int rows_at_once = std::min(max_tokens, c.block);
    a.warps_per_job = 1;
    while (a.warps_per_job < kAppendWarps && a.warps_per_job * kUK * a.heads_per_pass < rows_at_once) a.warps_per_job *= 2;
    const int64_t per = kAppendWarps / a.warps_per_job;
    const double jobs = static_cast<double>(batch) * a.blocks * 2 * a.hkv, q_jobs = static_cast<double>(batch) * max_tokens * a.parts;
    if (jobs + q_jobs > INT32_MAX) return fail(BM_ERR_INVALID_ARGUMENT, "%s: batch * max_tokens too large", what);
    // Fewer than kApartRows rows go in one launch, more in one each for K, V and Q, since K's registers leave room for only 16
    // warps on an SM; two launches more are 6 to 8 us. In one and apart, us: 1030 rows of 64 + 2 x 8 heads of 128 in bf16
    // 21 and 28, 4096 48 and 55, 8192 90 and 89, 16384 167 and 159; of 32 + 2 x 8 4096 34 and 40, 8192 62 and 64, 12000 89
    // and 89, 16384 118 and 113; of 32 + 2 x 4 of 64 8192 29 and 31, 16384 53 and 54; of 6 + 2 x 6 of 48 in fp32 4096 19
    // and 23, 12000 50 and 50, 16384 67 and 64.
    constexpr int64_t kApartRows = 12288;
    const bool apart = most_rows >= kApartRows;
    a.kv_ctas = (batch * a.blocks * (apart ? 1 : 2) * a.hkv + per - 1) / per;
    const int64_t q_warps = num_q_heads ? batch * max_tokens * a.parts : 0;
    const int64_t q_ctas = apart ? 0 : (q_warps + kAppendWarps - 1) / kAppendWarps;
    const bool full = a.rest == 0 && 32 % a.units == 0;
    auto go = [&](auto inter, auto whole, auto type, auto width) {
      constexpr bool I = decltype(inter)::value, F = decltype(whole)::value;
      using T = decltype(type);
      constexpr int N = decltype(width)::value, J = N == 1 ? 4 : 1;
      auto launch = [&](auto kernel, int64_t ctas, int threads) {
        return launch_kernel(what, kernel, dim3(static_cast<unsigned>(ctas)), dim3(threads), 0, as_stream(stream), nullptr, a);
      };
      if (!apart) return launch(append_kernel<T, N, J, I, F, Jobs::kAll>, a.kv_ctas + q_ctas, kAppendThreads);
      if (int st = launch(append_kernel<T, N, J, I, F, Jobs::kK>, a.kv_ctas, kAppendThreads)) return st;
      if (int st = launch(append_kernel<T, N, J, I, F, Jobs::kV>, a.kv_ctas, kAppendThreads)) return st;
      return num_q_heads ? launch(append_q_kernel<T, N, J, I, F>, (q_warps + kWarps - 1) / kWarps, kThreads) : BM_OK;
    };
    auto pick = [&](auto inter) {
      const std::true_type yes;
      const std::false_type no;
      const std::integral_constant<int, 1> one;
      const std::integral_constant<int, 4> four;
      const std::integral_constant<int, 8> eight;
      if (dtype == BM_F32) {
        if (n == 4) return full ? go(inter, yes, 0.f, four) : go(inter, no, 0.f, four);
        return go(inter, no, 0.f, one);
      }
      if (n == 8) return full ? go(inter, yes, bf16{}, eight) : go(inter, no, bf16{}, eight);
      return n == 4 ? go(inter, no, bf16{}, four) : go(inter, no, bf16{}, one);
    };
    return interleaved ? pick(std::true_type{}) : pick(std::false_type{});
  });
}

extern "C" int bm_paged_kv8_read(void* k_out, void* v_out, const bm_paged_kv8_t* cache, const int32_t* seq_ids, const int32_t* first,
                                 const int32_t* starts, int64_t rows, int64_t batch, int32_t max_rows, bm_dtype_t dtype,
                                 int32_t* d_status, void* stream) {
  using namespace bm;
  const char* what = "bm_paged_kv8_read";
  if (!valid_dtype(dtype)) return fail(BM_ERR_INVALID_ARGUMENT, "%s: bad dtype %d", what, static_cast<int>(dtype));
  if (int st = check_paged_kv8(what, cache)) return st;
  const bm_paged_kv8_t& c = *cache;
  if (rows < 0 || rows > INT32_MAX || batch < 0 || batch > INT32_MAX || max_rows < 0) {
    return fail(BM_ERR_INVALID_ARGUMENT, "%s: bad rows, batch or max_rows", what);
  }
  if (rows == 0 || batch == 0 || max_rows == 0) return BM_OK;
  if (!k_out || !v_out || !first || !starts) return fail(BM_ERR_INVALID_ARGUMENT, "%s: NULL pointer", what);
  if (!seq_ids && batch > c.num_seqs) return fail(BM_ERR_INVALID_ARGUMENT, "%s: more sequences than the cache holds", what);
  if (!aligned16(k_out) || !aligned16(v_out)) return fail(BM_ERR_INVALID_ARGUMENT, "%s: k_out and v_out must be 16-byte aligned", what);
  if (!aligned_to({seq_ids, first, starts, d_status}, 4)) return fail(BM_ERR_INVALID_ARGUMENT, "%s: a pointer is not aligned to its elements", what);
  const uintptr_t bytes = static_cast<uintptr_t>(rows) * c.num_kv_heads * c.head_dim * dtype_size(dtype);
  const uintptr_t ko = reinterpret_cast<uintptr_t>(k_out), vo = reinterpret_cast<uintptr_t>(v_out);
  if ((ko < vo + bytes && vo < ko + bytes) || meets_pages8(c, k_out, bytes) || meets_pages8(c, v_out, bytes)) {
    return fail(BM_ERR_INVALID_ARGUMENT, "%s: an output overlaps the other or the cache", what);
  }
  max_rows = static_cast<int32_t>(std::min<int64_t>(max_rows, rows));  // no sequence has more
  ReadArgs a{k_out, v_out, c, first, starts, seq_ids, rows, batch, max_rows, 0, d_status};
  const int per = kReadU * (32 / (c.head_dim / 16));
  a.chunks = static_cast<int>((static_cast<int64_t>(max_rows) + per - 1) / per);
  const double jobs = static_cast<double>(batch) * a.chunks * c.num_kv_heads;
  if (jobs > INT32_MAX) return fail(BM_ERR_INVALID_ARGUMENT, "%s: batch * max_rows too large", what);
  const int64_t blocks = (batch * a.chunks * c.num_kv_heads + kWarps - 1) / kWarps;
  auto go = [&](auto kernel) {
    return launch_kernel(what, kernel, dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0, as_stream(stream), nullptr, a);
  };
  return dtype == BM_F32 ? go(read_kernel<float>) : go(read_kernel<bf16>);
}
