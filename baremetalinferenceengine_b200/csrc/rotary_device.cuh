// Pieces that the kernels which rotate heads in shares of a warp have in common (rotary.cu,
// kv8_cache.cu): a lane's chunks of a head, the rotation of a unit's pairs, and the host
// checks of rows and tables.
//
// A unit is N pairs of one head: the chunks of N elements at i and i + rd/2 (half pairs), or
// two side by side (interleaved pairs, and elements past rotary_dim, which are copied).
#pragma once

#include "bm_common.cuh"
#include "bm_host.h"

namespace bm {
namespace rot {

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

// The N pairs of a unit's two chunks x[0, N) and x[N, 2N).
template <int N, bool INTER>
__device__ __forceinline__ void rotate(float* x, const float2* cs) {
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const int a = INTER ? 2 * e : e, b = INTER ? 2 * e + 1 : N + e;
    rope_rotate(x[a], x[b], cs[e], &x[a], &x[b]);
  }
}
// The same for half pairs, two to an instruction (N even): rope_rotate's roundings, since a product with -s is
// the negative of the one with s.
template <int N>
__device__ __forceinline__ void rotate2(float* x, const float2* cs) {
#pragma unroll
  for (int e = 0; e < N; e += 2) {
    const uint64_t a = pair(x[e], x[e + 1]), b = pair(x[N + e], x[N + e + 1]), c = pair(cs[e].x, cs[e + 1].x);
    const float2 first = unpair(fma2(a, c, mul2(b, pair(-cs[e].y, -cs[e + 1].y))));
    const float2 second = unpair(fma2(b, c, mul2(a, pair(cs[e].y, cs[e + 1].y))));
    x[e] = first.x;
    x[e + 1] = first.y;
    x[N + e] = second.x;
    x[N + e + 1] = second.y;
  }
}
template <typename T, int N, bool INTER>
__device__ __forceinline__ void rotate(Piece<T, N>& p1, Piece<T, N>& p2, const float2* cs) {
  float x[2 * N];
  p1.get(x);
  p2.get(x + N);
  rotate<N, INTER>(x, cs);
  p1.set(x);
  p2.set(x + N);
}

// The (cos, sin) of a unit: N of them from t, by 16-byte loads where N is even (the host
// checks the table's alignment).
template <int N>
__device__ __forceinline__ void load_angles(const float2* t, float2* cs) {
  if constexpr (N % 2 == 0) {
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
}

// Rows of `n` elements, `stride` apart.
struct Rows {
  const void* p;
  int64_t stride, n;
};

// Whether two runs of rows share memory. Slices of one buffer's rows (q, k and v of a
// fused projection) interleave without meeting.
inline bool meet(const Rows& a, const Rows& b, int64_t rows, int es) {
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
inline bool same(const Rows& a, const Rows& b, int64_t rows) { return a.p == b.p && (rows == 1 || a.stride == b.stride); }

inline int check_rotation(const char* what, const void* table, int32_t table_len, int rd, int hd) {
  if (table_len <= 0) return fail(BM_ERR_INVALID_ARGUMENT, "%s: table_len must be > 0", what);
  if (reinterpret_cast<uintptr_t>(table) & 7u) return fail(BM_ERR_INVALID_ARGUMENT, "%s: table not 8-byte aligned", what);
  if (rd <= 0 || rd % 2 || rd > hd) {
    return fail(BM_ERR_INVALID_ARGUMENT, "%s: rotary_dim %d must be even, positive and at most head_dim %d", what, rd, hd);
  }
  return BM_OK;
}

}  // namespace rot
}  // namespace bm
