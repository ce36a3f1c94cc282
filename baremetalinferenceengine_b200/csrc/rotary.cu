// Rotary positions in half-split and interleaved pairs, on part of the head, from
// scaled (cos, sin) tables; and the same rotation on the way into a paged KV cache
// (bm_rotary, bm_paged_kv_append, bm_rotary_table_fill).
//
// Mathematics: a pair (a, b) at position p and frequency f becomes
//   (a c - b s, b c + a s),  (c, s) = mscale * (cos, sin)(p f),
// the expression of rope_rotate, whose roundings are pinned. Pairs are (i, i + rd/2)
// (half) or (2i, 2i + 1) (interleaved); elements past the rotary_dim rd are copied.
//
// Bound: memory. Every element of q, k (and v) is read once and written once; the
// table rows come from L2. Layout of the work: a unit is N pairs of one head, two
// 16-byte chunks (i and i + rd/2, or two chunks side by side; copied elements are units of
// two chunks, too), and a lane keeps the N (cos, sin) of its unit's place in the head for
// all heads that it visits, so the table is read once per token and lane and not once
// per head, and neighbouring lanes cover whole heads. A warp takes one token,
// or one of `parts` shares of a token's heads when there are few tokens: a decode
// batch is bound by the chain position -> (cos, sin), sequence -> page -> store, which
// more warps with one pass each overlap. Data loads are issued before that chain is
// waited for. Measured on a B200, bf16, calls one after the other: 16384 rows of 64 + 8 heads
// of 128 in 101 to 103 us (604 MB, 0.91 to 0.89 of the copy rate: the power limit), 32768 rows
// of 64 + 8 appended to pages of 64 in 224 to 227 us (0.92 to 0.90), a decode batch of 64 rows in 4 us
// either way.
#include <algorithm>
#include <cmath>

#include "bm_common.cuh"
#include "bm_host.h"

namespace bm {
namespace {

constexpr int kMaxHeadDim = 1024;
constexpr int kThreads = 128;  // 256: 1 to 3 % slower on prompts

struct RotaryArgs {
  void* q_out;
  void* k_out;              // rotary: k_out; append: unused
  const void* q;
  const void* k;
  const void* v;            // append only
  const int32_t* positions; // NULL: pos0 + row (append without rotation: unused)
  const int32_t* slots;     // append: NULL = positions
  const int32_t* seq_ids;   // append: NULL = 0
  const float2* table;      // NULL: no rotation (append only)
  void* k_pages;
  void* v_pages;
  const int32_t* page_table;
  int64_t rows;
  int64_t q_stride, k_stride, v_stride, q_out_stride, k_out_stride;
  int32_t pos0, table_len;
  int hq, hkv, hd, rd;      // rd: rotated elements of a head (0 without a table)
  int num_pages, page_size, max_pages, num_seqs;
  int parts;                // warps per token
  int units, rest;          // rotated and copied units of a head
  int32_t* status;
};

// N consecutive elements of T held between load and store.
template <typename T>
struct Piece16 {
  uint4 raw;
  __device__ __forceinline__ void load(const T* p) { raw = ld_stream(p); }
  __device__ __forceinline__ void store(T* p) const { st_plain(p, raw); }
  __device__ __forceinline__ void get(float* f) const { unpack16<T>(raw, f); }
  __device__ __forceinline__ void set(const float* f) { raw = pack16<T>(f); }
};
template <typename T, int N>
struct Piece;
template <>
struct Piece<float, 4> : Piece16<float> {};
template <>
struct Piece<bf16, 8> : Piece16<bf16> {};
template <>
struct Piece<bf16, 4> {
  uint2 raw;
  __device__ __forceinline__ void load(const bf16* p) { raw = __ldcs(reinterpret_cast<const uint2*>(p)); }
  __device__ __forceinline__ void store(bf16* p) const { *reinterpret_cast<uint2*>(p) = raw; }
  __device__ __forceinline__ void get(float* f) const {
    f[0] = bf16_lo(raw.x);
    f[1] = bf16_hi(raw.x);
    f[2] = bf16_lo(raw.y);
    f[3] = bf16_hi(raw.y);
  }
  __device__ __forceinline__ void set(const float* f) {
    raw.x = pack_bf16x2(f[0], f[1]);
    raw.y = pack_bf16x2(f[2], f[3]);
  }
};
template <typename T>
struct Piece<T, 1> {
  T raw;
  __device__ __forceinline__ void load(const T* p) { raw = *p; }
  __device__ __forceinline__ void store(T* p) const { *p = raw; }
  __device__ __forceinline__ void get(float* f) const { f[0] = load1<T>(&raw); }
  __device__ __forceinline__ void set(const float* f) { store1<T>(&raw, f[0]); }
};

template <typename T, int N, bool INTER>
__device__ __forceinline__ void rotate(Piece<T, N>& p1, Piece<T, N>& p2, const float2* cs) {
  float x[2 * N];
  p1.get(x);
  p2.get(x + N);
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const int a = INTER ? 2 * e : e, b = INTER ? 2 * e + 1 : N + e;
    rope_rotate(x[a], x[b], cs[e], &x[a], &x[b]);
  }
  p1.set(x);
  p2.set(x + N);
}

// PAGED: k goes into the cache's pages and v with it; otherwise k into k_out.
template <typename T, int N, bool INTER, bool PAGED>
__global__ void __launch_bounds__(kThreads) rotary_kernel(RotaryArgs a) {
  constexpr int U = PAGED ? 4 : 2;  // passes whose loads a lane keeps in flight (the other way round: 9 % and 4 % slower on prompts)
  const int lane = threadIdx.x & 31;
  const int64_t job0 = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) >> 5;
  const int64_t njobs = a.rows * a.parts;
  if (job0 < njobs && lane == 0) {
    const int64_t r = job0 / a.parts;
    if (a.positions) prefetch_l2(a.positions + r);
    if (PAGED && a.slots) prefetch_l2(a.slots + r);
    if (PAGED && a.seq_ids) prefetch_l2(a.seq_ids + r);
  }
  grid_dependency_wait();
  const int64_t step = (static_cast<int64_t>(gridDim.x) * kThreads) >> 5;
  const int heads = a.hq + a.hkv + (PAGED ? a.hkv : 0);
  constexpr int kUnit = INTER ? 2 * N : N;  // elements between neighbouring units

  for (int64_t job = job0; job < njobs; job += step) {
    const int64_t row = job / a.parts;
    const int part = static_cast<int>(job - row * a.parts);
    const int32_t pos = a.positions ? __ldg(a.positions + row) : static_cast<int32_t>(a.pos0 + row);
    int64_t cache_base = 0;
    const int64_t head_stride = PAGED ? static_cast<int64_t>(a.page_size) * a.hd : 0;
    int32_t bad = 0;
    if (a.table != nullptr && (pos < 0 || pos >= a.table_len)) bad |= BM_DEVERR_BAD_POSITION;
    if constexpr (PAGED) {
      const int32_t slot = a.slots ? __ldg(a.slots + row) : pos;
      if (slot == -1) continue;  // a padding row
      const int32_t seq = a.seq_ids ? __ldg(a.seq_ids + row) : 0;
      const int32_t nth = slot / a.page_size;
      if (slot < 0 || nth >= a.max_pages) bad |= BM_DEVERR_BAD_POSITION;
      if (seq < 0 || seq >= a.num_seqs) bad |= BM_DEVERR_BAD_SEQUENCE;
      if (!bad) {
        const int32_t page = __ldg(a.page_table + static_cast<int64_t>(seq) * a.max_pages + nth);
        if (page < 0 || page >= a.num_pages) bad |= BM_DEVERR_BAD_PAGE;
        cache_base = static_cast<int64_t>(page) * a.hkv * head_stride + static_cast<int64_t>(slot - nth * a.page_size) * a.hd;
      }
    }
    if (bad) {  // uniform across the warp
      if (lane == 0) raise_status(a.status, bad);
      continue;
    }
    const T* qrow = static_cast<const T*>(a.q) + row * a.q_stride;
    const T* krow = static_cast<const T*>(a.k) + row * a.k_stride;
    const T* vrow = static_cast<const T*>(a.v) + row * a.v_stride;
    T* qdst = static_cast<T*>(a.q_out) + row * a.q_out_stride;
    T* kdst = PAGED ? static_cast<T*>(a.k_pages) + cache_base : static_cast<T*>(a.k_out) + row * a.k_out_stride;
    T* vdst = static_cast<T*>(a.v_pages) + cache_base;
    // heads in turn: q's, k's, then (PAGED) v's
    auto src = [&](int h) -> const T* {
      if (h < a.hq) return qrow + static_cast<int64_t>(h) * a.hd;
      if (!PAGED || h < a.hq + a.hkv) return krow + static_cast<int64_t>(h - a.hq) * a.hd;
      return vrow + static_cast<int64_t>(h - a.hq - a.hkv) * a.hd;
    };
    auto dst = [&](int h) -> T* {
      if (h < a.hq) return qdst + static_cast<int64_t>(h) * a.hd;
      if (!PAGED) return kdst + static_cast<int64_t>(h - a.hq) * a.hd;
      if (h < a.hq + a.hkv) return kdst + (h - a.hq) * head_stride;
      return vdst + (h - a.hq - a.hkv) * head_stride;
    };
    const int turning = a.hq + a.hkv;

    for (int c0 = 0; c0 < a.units + a.rest; c0 += 32) {
      const int n = min(32, a.units + a.rest - c0);
      const int hpi = 32 / n;
      const int c = c0 + lane % n;
      const int hl = lane / n;
      if (hl >= hpi) continue;
      const bool turns = c < a.units;
      // this unit's two chunks of every head; the last copied one may have no second
      const int first = turns ? c * kUnit : a.rd + (c - a.units) * 2 * N;
      const int second = first + (turns && !INTER ? a.rd / 2 : N);
      const bool pair = second < a.hd;
      const int passes = (heads + hpi - 1) / hpi;
      const int mine = (passes + a.parts - 1) / a.parts;
      const int h_end = min(heads, (part + 1) * mine * hpi);
      float2 cs[N];
      bool have = false;
      for (int hb = part * mine * hpi + hl; hb < h_end; hb += hpi * U) {
        Piece<T, N> x1[U], x2[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int h = hb + u * hpi;
          if (h < h_end) {
            x1[u].load(src(h) + first);
            if (pair) x2[u].load(src(h) + second);
          }
        }
        if (turns && !have) {
          const float2* t = a.table + static_cast<int64_t>(pos) * (a.rd / 2) + c * N;
          if constexpr (N % 2 == 0) {  // 16-byte loads: the host checked the table's alignment
#pragma unroll
            for (int e = 0; e < N; e += 2) {
              const float4 two = __ldg(reinterpret_cast<const float4*>(t + e));
              cs[e] = make_float2(two.x, two.y);
              cs[e + 1] = make_float2(two.z, two.w);
            }
          } else {
#pragma unroll
            for (int e = 0; e < N; ++e) cs[e] = __ldg(t + e);
          }
          have = true;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int h = hb + u * hpi;
          if (h < h_end) {
            if (turns && h < turning) rotate<T, N, INTER>(x1[u], x2[u], cs);
            x1[u].store(dst(h) + first);
            if (pair) x2[u].store(dst(h) + second);
          }
        }
      }
    }
  }
}

template <bool PAGED>
int launch(RotaryArgs a, bool interleaved, bm_dtype_t dtype, cudaStream_t stream, const char* what) {
  // The widest chunk that divides every run of elements and suits every pointer and
  // stride: 16 bytes, 8 (bf16 heads such as 24 rotated elements), else one element.
  const int es = dtype_size(dtype);
  auto fits = [&](int n) {
    if ((a.rd / 2) % n || (a.hd - a.rd) % n || a.hd % n) return false;
    const uintptr_t bytes = static_cast<uintptr_t>(n) * es;
    const void* ptrs[] = {a.q, a.k, a.v, a.q_out, a.k_out, a.k_pages, a.v_pages};
    for (const void* p : ptrs) {
      if (reinterpret_cast<uintptr_t>(p) % bytes) return false;
    }
    for (int64_t s : {a.q_stride, a.k_stride, a.v_stride, a.q_out_stride, a.k_out_stride}) {
      if (s % n) return false;
    }
    return n % 2 != 0 || aligned16(a.table);
  };
  int n = 16 / es;
  if (!fits(n)) n = es == 2 && fits(4) ? 4 : 1;
  a.units = a.rd / 2 / n;
  a.rest = (a.hd - a.rd + 2 * n - 1) / (2 * n);
  // One warp per token for a batch that fills the GPU (2048 warps: 14 per SM); fewer
  // tokens are shared out over up to 8 warps each.
  a.parts = static_cast<int>(std::min<int64_t>(8, std::max<int64_t>(1, 2048 / std::max<int64_t>(1, a.rows))));
  const int64_t blocks = (a.rows * a.parts + kThreads / 32 - 1) / (kThreads / 32);
  const dim3 grid(static_cast<unsigned>(std::min<int64_t>(blocks, static_cast<int64_t>(sm_count()) * 32)));
  auto go = [&](auto kernel) { return launch_kernel(what, kernel, grid, dim3(kThreads), 0, stream, nullptr, a); };
  if (dtype == BM_F32) {
    if (n == 4) return interleaved ? go(rotary_kernel<float, 4, true, PAGED>) : go(rotary_kernel<float, 4, false, PAGED>);
    return interleaved ? go(rotary_kernel<float, 1, true, PAGED>) : go(rotary_kernel<float, 1, false, PAGED>);
  }
  if (n == 8) return interleaved ? go(rotary_kernel<bf16, 8, true, PAGED>) : go(rotary_kernel<bf16, 8, false, PAGED>);
  if (n == 4) return interleaved ? go(rotary_kernel<bf16, 4, true, PAGED>) : go(rotary_kernel<bf16, 4, false, PAGED>);
  return interleaved ? go(rotary_kernel<bf16, 1, true, PAGED>) : go(rotary_kernel<bf16, 1, false, PAGED>);
}

// Rows of `n` elements, `stride` apart.
struct Rows {
  const void* p;
  int64_t stride, n;
};

// Whether two runs of rows share memory. Slices of one buffer's rows (q, k and v of a
// fused projection) interleave without meeting.
bool meet(const Rows& a, const Rows& b, int64_t rows, int es) {
  if (a.p == nullptr || b.p == nullptr || a.n == 0 || b.n == 0) return false;
  const uintptr_t pa = reinterpret_cast<uintptr_t>(a.p), pb = reinterpret_cast<uintptr_t>(b.p);
  if (pa + static_cast<uintptr_t>((rows - 1) * a.stride + a.n) * es <= pb) return false;
  if (pb + static_cast<uintptr_t>((rows - 1) * b.stride + b.n) * es <= pa) return false;
  if (rows > 1 && a.stride == b.stride) {
    const int64_t pitch = a.stride * es;
    const int64_t d = ((static_cast<int64_t>(pa - pb) % pitch) + pitch) % pitch;  // a's offset behind b in a row
    return !(d >= b.n * es && d + a.n * es <= pitch);
  }
  return true;
}
bool same(const Rows& a, const Rows& b, int64_t rows) { return a.p == b.p && (rows == 1 || a.stride == b.stride); }

int check_rotation(const char* what, const void* table, int32_t table_len, int rd, int hd) {
  if (table_len <= 0) return fail(BM_ERR_INVALID_ARGUMENT, "%s: table_len must be > 0", what);
  if (reinterpret_cast<uintptr_t>(table) & 7u) return fail(BM_ERR_INVALID_ARGUMENT, "%s: table not 8-byte aligned", what);
  if (rd <= 0 || rd % 2 || rd > hd) {
    return fail(BM_ERR_INVALID_ARGUMENT, "%s: rotary_dim %d must be even, positive and at most head_dim %d", what, rd, hd);
  }
  return BM_OK;
}

struct Frequencies {
  int kind;
  double theta, factor, low, high, mscale;  // YARN: low and high hold the ramp's ends
  double original;
};

__global__ void rotary_table_kernel(float2* table, int32_t max_pos, int half, int rd, Frequencies f) {
  grid_dependency_wait();
  const int64_t n = static_cast<int64_t>(max_pos) * half;
  for (int64_t idx = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; idx < n;
       idx += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int64_t p = idx / half;
    const int i = static_cast<int>(idx - p * half);
    const double base = pow(f.theta, 2.0 * i / rd);
    double angle;
    if (f.kind == BM_ROPE_SCALING_NONE || f.kind == BM_ROPE_SCALING_NTK) {  // NTK: theta is the stretched base
      angle = static_cast<double>(p) / base;
    } else {
      const double freq = 1.0 / base;
      double part = 1.0;  // share of the frequency that is divided by factor
      if (f.kind == BM_ROPE_SCALING_BANDS) {
        const double turns = f.original * freq / 6.283185307179586476925287;
        part = 1.0 - fmin(fmax((turns - f.low) / (f.high - f.low), 0.0), 1.0);
      } else if (f.kind == BM_ROPE_SCALING_YARN) {
        part = fmin(fmax((i - f.low) / fmax(f.high - f.low, 0.001), 0.0), 1.0);
      }
      angle = static_cast<double>(p) * (freq / f.factor * part + freq * (1.0 - part));
    }
    double s, c;
    sincos(angle, &s, &c);
    table[idx] = make_float2(static_cast<float>(f.mscale * c), static_cast<float>(f.mscale * s));
  }
}

}  // namespace
}  // namespace bm

extern "C" int bm_rotary_table_fill(void* table, int32_t max_pos, int32_t rotary_dim, double theta,
                                    const bm_rope_scaling_t* scaling, void* stream) {
  using namespace bm;
  const char* what = "bm_rotary_table_fill";
  if (max_pos <= 0 || rotary_dim <= 0 || rotary_dim % 2 || !(theta > 0.0) || !std::isfinite(theta)) {
    return fail(BM_ERR_INVALID_ARGUMENT, "%s: need max_pos > 0, even rotary_dim > 0, finite theta > 0", what);
  }
  if (!table || (reinterpret_cast<uintptr_t>(table) & 7u)) return fail(BM_ERR_INVALID_ARGUMENT, "%s: bad table pointer", what);
  Frequencies f{};
  f.theta = theta;
  f.factor = 1.0;
  f.mscale = 1.0;
  if (scaling != nullptr) {
    const bm_rope_scaling_t& s = *scaling;
    f.kind = s.kind;
    f.factor = s.factor;
    f.low = s.low;
    f.high = s.high;
    f.original = s.original_max_pos;
    if (s.kind < BM_ROPE_SCALING_NONE || s.kind > BM_ROPE_SCALING_YARN) {
      return fail(BM_ERR_INVALID_ARGUMENT, "%s: bad scaling kind %d", what, static_cast<int>(s.kind));
    }
    if (s.kind != BM_ROPE_SCALING_NONE && !(s.factor >= 1.0 && std::isfinite(s.factor))) {
      return fail(BM_ERR_INVALID_ARGUMENT, "%s: factor must be finite and >= 1", what);
    }
    if (!std::isfinite(s.mscale)) return fail(BM_ERR_INVALID_ARGUMENT, "%s: mscale must be finite", what);
    if (s.kind == BM_ROPE_SCALING_NTK) {
      if (rotary_dim < 4) return fail(BM_ERR_INVALID_ARGUMENT, "%s: NTK needs rotary_dim >= 4", what);
      f.theta = theta * std::pow(s.factor, rotary_dim / (rotary_dim - 2.0));
    }
    if (s.kind == BM_ROPE_SCALING_BANDS &&
        !(s.low < s.high && std::isfinite(s.low) && std::isfinite(s.high) && s.original_max_pos > 0)) {
      return fail(BM_ERR_INVALID_ARGUMENT, "%s: BANDS needs finite low < high and original_max_pos > 0", what);
    }
    if (s.kind == BM_ROPE_SCALING_YARN) {
      if (!(s.low >= s.high && s.high > 0.0 && std::isfinite(s.low) && s.original_max_pos > 0 && theta > 1.0)) {
        return fail(BM_ERR_INVALID_ARGUMENT, "%s: YARN needs low >= high > 0, original_max_pos > 0 and theta > 1", what);
      }
      const auto edge = [&](double turns) {
        return rotary_dim * std::log(s.original_max_pos / (turns * 6.283185307179586476925287)) / (2.0 * std::log(theta));
      };
      f.low = std::max(std::floor(edge(s.low)), 0.0);
      f.high = std::min(std::ceil(edge(s.high)), rotary_dim - 1.0);
    }
    f.mscale = s.mscale > 0.0 ? s.mscale : s.kind == BM_ROPE_SCALING_YARN ? 0.1 * std::log(s.factor) + 1.0 : 1.0;
  }
  const int half = rotary_dim / 2;
  const int64_t n = static_cast<int64_t>(max_pos) * half;
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>((n + 255) / 256, static_cast<int64_t>(sm_count()) * 8));
  return launch_kernel("rotary_table_kernel", rotary_table_kernel, dim3(grid), dim3(256), 0, as_stream(stream), nullptr,
                       static_cast<float2*>(table), max_pos, half, rotary_dim, f);
}

extern "C" int bm_rotary(void* q_out, void* k_out, const void* q, const void* k, const int32_t* positions, int32_t pos0,
                         const void* table, int32_t table_len, int32_t rotary_dim, int32_t interleaved, int64_t rows,
                         int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim, int64_t q_stride,
                         int64_t k_stride, int64_t q_out_stride, int64_t k_out_stride, bm_dtype_t dtype,
                         int32_t* d_status, void* stream) {
  using namespace bm;
  const char* what = "bm_rotary";
  if (!valid_dtype(dtype)) return fail(BM_ERR_INVALID_ARGUMENT, "%s: bad dtype %d", what, static_cast<int>(dtype));
  if (rows < 0 || num_q_heads < 0 || num_kv_heads < 0) return fail(BM_ERR_INVALID_ARGUMENT, "%s: negative rows or head count", what);
  if (head_dim <= 0 || head_dim > kMaxHeadDim) return fail(BM_ERR_INVALID_ARGUMENT, "%s: head_dim %d outside [1, %d]", what, head_dim, kMaxHeadDim);
  if (num_q_heads > (1 << 16) || num_kv_heads > (1 << 16)) return fail(BM_ERR_INVALID_ARGUMENT, "%s: more than 65536 heads", what);
  if (!table) return fail(BM_ERR_INVALID_ARGUMENT, "%s: NULL table", what);
  if (int st = check_rotation(what, table, table_len, rotary_dim, head_dim)) return st;
  if (rows == 0 || (num_q_heads == 0 && num_kv_heads == 0)) return BM_OK;
  if ((num_q_heads > 0 && (!q || !q_out)) || (num_kv_heads > 0 && (!k || !k_out))) {
    return fail(BM_ERR_INVALID_ARGUMENT, "%s: NULL pointer", what);
  }
  const int64_t qn = static_cast<int64_t>(num_q_heads) * head_dim, kn = static_cast<int64_t>(num_kv_heads) * head_dim;
  if ((qn && (q_stride < qn || q_out_stride < qn)) || (kn && (k_stride < kn || k_out_stride < kn))) {
    return fail(BM_ERR_INVALID_ARGUMENT, "%s: a row stride below heads * head_dim", what);
  }
  if (!positions && (pos0 < 0 || pos0 + rows > INT32_MAX)) return fail(BM_ERR_INVALID_ARGUMENT, "%s: bad pos0", what);
  const int es = dtype_size(dtype);
  if (!aligned_to({q, k, q_out, k_out}, es) || !aligned_to({positions, d_status}, 4)) {
    return fail(BM_ERR_INVALID_ARGUMENT, "%s: a pointer is not aligned to its elements", what);
  }
  const Rows qi{q, q_stride, qn}, ki{k, k_stride, kn}, qo{q_out, q_out_stride, qn}, ko{k_out, k_out_stride, kn};
  if ((meet(qo, qi, rows, es) && !same(qo, qi, rows)) || (meet(ko, ki, rows, es) && !same(ko, ki, rows)) ||
      meet(qo, ki, rows, es) || meet(ko, qi, rows, es) || meet(qo, ko, rows, es)) {
    return fail(BM_ERR_INVALID_ARGUMENT, "%s: an output overlaps an input or the other output", what);
  }
  RotaryArgs a{};
  a.q_out = q_out;
  a.k_out = k_out;
  a.q = q;
  a.k = k;
  a.positions = positions;
  a.pos0 = pos0;
  a.table = static_cast<const float2*>(table);
  a.table_len = table_len;
  a.rd = rotary_dim;
  a.rows = rows;
  a.hq = num_q_heads;
  a.hkv = num_kv_heads;
  a.hd = head_dim;
  a.q_stride = q_stride;
  a.k_stride = k_stride;
  a.q_out_stride = q_out_stride;
  a.k_out_stride = k_out_stride;
  a.status = d_status;
  return launch<false>(a, interleaved != 0, dtype, as_stream(stream), what);
}

extern "C" int bm_paged_kv_append(void* q_out, const void* q, const void* k, const void* v, const int32_t* positions,
                                  const int32_t* slots, const int32_t* seq_ids, const bm_paged_kv_t* cache,
                                  const void* table, int32_t table_len, int32_t rotary_dim, int32_t interleaved,
                                  int64_t rows, int32_t num_q_heads, int64_t q_stride, int64_t k_stride,
                                  int64_t v_stride, int64_t q_out_stride, bm_dtype_t dtype, int32_t* d_status,
                                  void* stream) {
  using namespace bm;
  const char* what = "bm_paged_kv_append";
  if (!valid_dtype(dtype)) return fail(BM_ERR_INVALID_ARGUMENT, "%s: bad dtype %d", what, static_cast<int>(dtype));
  if (rows < 0 || num_q_heads < 0 || num_q_heads > (1 << 16)) return fail(BM_ERR_INVALID_ARGUMENT, "%s: bad rows or head count", what);
  if (int st = check_paged_kv(what, cache)) return st;
  const bm_paged_kv_t& c = *cache;
  if (c.head_dim > kMaxHeadDim) return fail(BM_ERR_INVALID_ARGUMENT, "%s: head_dim %d outside [1, %d]", what, c.head_dim, kMaxHeadDim);
  if (table) {
    if (int st = check_rotation(what, table, table_len, rotary_dim, c.head_dim)) return st;
  }
  if (rows == 0) return BM_OK;
  if (!k || !v || (num_q_heads > 0 && (!q || !q_out))) return fail(BM_ERR_INVALID_ARGUMENT, "%s: NULL pointer", what);
  if (!positions && (table || !slots)) return fail(BM_ERR_INVALID_ARGUMENT, "%s: NULL positions", what);
  const int64_t qn = static_cast<int64_t>(num_q_heads) * c.head_dim, kn = static_cast<int64_t>(c.num_kv_heads) * c.head_dim;
  if ((qn && (q_stride < qn || q_out_stride < qn)) || k_stride < kn || v_stride < kn) {
    return fail(BM_ERR_INVALID_ARGUMENT, "%s: a row stride below heads * head_dim", what);
  }
  const int es = dtype_size(dtype);
  if (!aligned_to({q, k, v, q_out, c.k_pages, c.v_pages}, es) || !aligned_to({positions, slots, seq_ids, c.page_table, d_status}, 4)) {
    return fail(BM_ERR_INVALID_ARGUMENT, "%s: a pointer is not aligned to its elements", what);
  }
  const Rows qi{q, q_stride, qn}, qo{q_out, q_out_stride, qn};
  if ((meet(qo, qi, rows, es) && !same(qo, qi, rows)) || meet(qo, Rows{k, k_stride, kn}, rows, es) ||
      meet(qo, Rows{v, v_stride, kn}, rows, es)) {
    return fail(BM_ERR_INVALID_ARGUMENT, "%s: q_out overlaps an input", what);
  }
  if (qn != 0 && meets_pages(c, q_out, static_cast<uintptr_t>((rows - 1) * q_out_stride + qn) * es, es)) {
    return fail(BM_ERR_INVALID_ARGUMENT, "%s: q_out overlaps the cache's pages", what);
  }
  RotaryArgs a{};
  a.q_out = q_out;
  a.q = q;
  a.k = k;
  a.v = v;
  a.positions = positions;
  a.slots = slots;
  a.seq_ids = seq_ids;
  a.table = static_cast<const float2*>(table);
  a.table_len = table_len;
  a.rd = table ? rotary_dim : 0;
  a.k_pages = c.k_pages;
  a.v_pages = c.v_pages;
  a.page_table = c.page_table;
  a.num_pages = c.num_pages;
  a.page_size = c.page_size;
  a.max_pages = c.max_pages;
  a.num_seqs = c.num_seqs;
  a.rows = rows;
  a.hq = num_q_heads;
  a.hkv = c.num_kv_heads;
  a.hd = c.head_dim;
  a.q_stride = q_stride;
  a.k_stride = k_stride;
  a.v_stride = v_stride;
  a.q_out_stride = q_out_stride;
  a.status = d_status;
  return launch<true>(a, interleaved != 0, dtype, as_stream(stream), what);
}
