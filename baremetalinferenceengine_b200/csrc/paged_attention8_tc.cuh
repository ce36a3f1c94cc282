// Pieces that the tensor-core forms of the tree attention over an 8-bit paged cache have in
// common (paged_attention8_tc.cu, for many rows, whose header comment has the mathematics;
// paged_attention8_few.cu): the two parts of queries and weights, and operands of single bytes.
#pragma once

#include "kv8.cuh"
#include "paged_attention_tc.cuh"

namespace bm {
namespace paged {

constexpr float kRescaleAt8 = 4.f;  // rise of the maximum (log2) that a row's sums are rescaled at
constexpr float kLift = 4.f;        // P is 2^4 at the running maximum, so at most 2^8
constexpr int kQRing = 4;           // segments whose queries' factors are kept
constexpr int kQWarps = 10;         // warps that convert a CTA's first queries: all but the two of TMA

// The matrix descriptor of rows of HD bytes, 8-row groups HD * 8 bytes apart, with the swizzle
// of such rows (128 or 64 bytes). Both operands' tiles are one swizzle atom wide.
template <int HD>
__device__ __forceinline__ uint64_t byte_desc(uint32_t addr) {
  return static_cast<uint64_t>((addr >> 4) & 0x3FFFu) | (1ull << 16) | (static_cast<uint64_t>((HD * 8) >> 4) << 32) | (1ull << 46) |
         ((HD == 128 ? 2ull : 4ull) << 61);
}
__device__ __forceinline__ void mma_f8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void mbar_arrive_n(uint64_t* bar, uint32_t count) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(count) : "memory");
}

// Two values as e4m3 (lo in the low byte); ends at +-448.
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
// Two weights: e4m3 of their fp16 values, and e5m2 of what that leaves.
__device__ __forceinline__ void weight_parts(float lo, float hi, uint32_t* part, uint32_t* rest) {
  uint32_t p, back;
  uint16_t h, l;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(p) : "f"(hi), "f"(lo));
  asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(h) : "r"(p));
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(back) : "h"(h));
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(back) : "r"(p), "r"(back));
  asm("cvt.rn.satfinite.e5m2x2.f16x2 %0, %1;" : "=h"(l) : "r"(back));
  *part = h;
  *rest = l;
}

// Converts the queries of an item into its two parts in the buffer at `to`, row tile after row
// tile, copies and all, and their factors scale * log2(e) * 2^-e_q into factor[row]. Warp
// `worker` of `workers` takes every workers-th pair of rows, half a warp a row; rows of no token are zero.
template <typename L, int HD>
__device__ __forceinline__ void convert_queries(const TreeArgs& a, const Seq& s, int kvh, int p, int tpt, unsigned char* to, float* factor,
                                                int worker, int workers) {
  constexpr int kBatch = 4;  // pairs of rows that are converted side by side
  const int lane = threadIdx.x & 31, half = lane >> 4, c = lane & 15;
  const int i_first = p * tpt * L::kTiles;
  const uint32_t by_group = (65536u + a.group - 1) / a.group;  // r / group = r * by_group >> 16 for r < 128
  const bf16* q = static_cast<const bf16*>(a.q) + (s.row0 * a.hq + static_cast<int64_t>(kvh) * a.group) * a.hd + c * 8;
  const int64_t token_step = static_cast<int64_t>(a.hq) * a.hd;
  for (int pair0 = worker; pair0 < L::kRows / 2; pair0 += workers * kBatch) {
    uint4 raw[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int row = 2 * (pair0 + k * workers) + half, r = row % L::kCopyRows;
      const int token = static_cast<int>(r * by_group >> 16), i = i_first + row / L::kCopyRows * tpt + token;
      raw[k] = make_uint4(0u, 0u, 0u, 0u);
      if (row < L::kRows && token < tpt && i < s.n && c * 8 < a.hd) raw[k] = ld_keep(q + i * token_step + (r - token * a.group) * a.hd);
    }
    uint32_t top[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      // the larger of two neighbours' magnitudes, as bf16 in either half of a word
      const uint32_t m01 = __vmaxu2(raw[k].x & 0x7fff7fffu, raw[k].y & 0x7fff7fffu), m23 = __vmaxu2(raw[k].z & 0x7fff7fffu, raw[k].w & 0x7fff7fffu);
      const uint32_t m = __vmaxu2(m01, m23);
      top[k] = max(m & 0xffffu, m >> 16);
    }
#pragma unroll
    for (int off = 8; off > 0; off >>= 1) {
#pragma unroll
      for (int k = 0; k < kBatch; ++k) top[k] = max(top[k], __shfl_xor_sync(0xffffffffu, top[k], off));
    }
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int row = 2 * (pair0 + k * workers) + half, r = row % L::kCopyRows;
      if (row >= L::kRows) continue;
      const int e = min(max(static_cast<int>(top[k] >> 7) - 127, -60), 127);
      const float f = kv8::power(7 - e);
      if (c * 8 < HD) {
        float x[8];
        unpack16<bf16>(raw[k], x);
        uint32_t hi[2], lo[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float back[4];
          hi[j] = e4m3x2(x[4 * j] * f, x[4 * j + 1] * f) | e4m3x2(x[4 * j + 2] * f, x[4 * j + 3] * f) << 16;
          kv8::from_codes(hi[j], back);
#pragma unroll
          for (int d = 0; d < 4; ++d) back[d] = fmaf(x[4 * j + d], f, -back[d]);
          lo[j] = e4m3x2(back[0], back[1]) | e4m3x2(back[2], back[3]) << 16;
        }
#pragma unroll
        for (int copy = 0; copy < L::kCopies; ++copy) {
          const int at = copy * L::kCopyRows + r;
          const int chunk = (c >> 1) ^ (HD == 128 ? at & 7 : (at >> 1) & 3);  // the swizzle of 16-byte chunks
          unsigned char* dst = to + row / L::kCopyRows * L::kQTile + at * HD + chunk * 16 + (c & 1) * 8;
          *reinterpret_cast<uint2*>(dst) = make_uint2(hi[0], hi[1]);
          *reinterpret_cast<uint2*>(dst + L::kOperand) = make_uint2(lo[0], lo[1]);
        }
      }
      // a query that is not finite spoils its row
      if (c == 0) factor[row] = top[k] >= 0x7f80u ? __int_as_float(0x7fffffff) : a.qscale * kv8::power(e - 7);
    }
  }
  fence_proxy_async_smem();
  __syncwarp();
}

// The few-row form: up to two row tiles of 32 rows.
inline bool few8_takes(int group, int max_tree) { return group <= 32 && max_tree <= 2 * (32 / group); }
int launch_few8(const TreeArgs& a, int nc, cudaStream_t stream, const char* what);

}  // namespace paged
}  // namespace bm
