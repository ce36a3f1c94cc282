// Attention of a tree of drafted tokens per sequence over a paged KV cache: the entry
// points (bm_paged_tree_attention), and the CUDA-core kernels that serve fp32, every
// head_dim and every page size. The tensor-core form is paged_attention_tc.cu.
//
// Mathematics: for row r = (token i, head) of a sequence, over the slots t that it sees,
//   out = sum_t 2^(s_t - m) v_t / sum_t 2^(s_t - m),  s_t = q . k_t * scale * log2(e),
// in one pass: m and the sums are running values, rescaled by 2^(m_old - m_new) when a
// tile of slots raises m (fp32 throughout).
//
// Bound: with R = group * n rows per kv head a slot costs 4 R hd operations and
// 2 hd * es bytes, so few rows are bound by memory and many, in fp32 on CUDA cores, by
// the multiply-adds. All rows of a kv head therefore share a CTA's tile of K and V
// (64 rows against 64 slots), and both products run from shared memory in register
// tiles (4 x 4 scores and 4 x hd/16 outputs per thread), 64 multiply-adds for 8 16-byte
// shared loads; up to 32 rows have a kernel of their own, bound by its shared loads of Q
// (8 rows of 128 in fp32 over 16 sequences of 1000 to 2000, 8 heads: 84 us, floor 30; of 256 in
// bf16, which the tensor-core form does not take, 4 rows 72, 32 rows 318, 512 rows 4870 us,
// floors 27, 28 and 60). Slots
// are shared out over CTAs when the (sequence, kv head, row tile) triples do not fill the
// GPU; the shares' partial sums meet in tree_combine_kernel.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "paged_attention.cuh"

namespace bm {
namespace paged {
namespace {

constexpr int kThreads = 256;
constexpr int BM = 64;   // query rows of a CTA
constexpr int kBN = 64;  // slots per tile

// NJ: 16-byte groups of four outputs a thread owns per row, ceil(hd / 64).
template <typename T, int NJ>
__global__ void __launch_bounds__(kThreads) tree_attention_kernel(const TreeArgs a) {
  grid_dependency_wait();
  constexpr int MR = BM / 16;
  constexpr int VEC = VecWidth<T>::value;
  const int hd = a.hd, ld = hd + 4;
  int64_t id = blockIdx.x;
  const int split = static_cast<int>(id % a.splits);
  id /= a.splits;
  const int rt = static_cast<int>(id % a.row_tiles);
  id /= a.row_tiles;
  const int kvh = static_cast<int>(id % a.hkv);
  const int64_t b = id / a.hkv;
  const int tid = threadIdx.x, ty = tid >> 4, tx = tid & 15;
  Seq s;
  const int32_t bad = read_seq(a, b, &s);
  if (bad) {
    if (tid == 0 && split == 0 && rt == 0 && kvh == 0) raise_status(a.status, bad);
    return;
  }
  const int R = a.group * s.n;
  const int r_lo = rt * BM;
  if (r_lo >= R) return;
  const int total = s.ctx + s.n;
  // without a mask the last row of the tile sees the most
  const int seen = a.mask ? total : s.ctx + min(s.n, (min(R, r_lo + BM) - 1) / a.group + 1);
  const int start = split * a.split_len;
  const int end = min(seen, start + a.split_len);

  extern __shared__ __align__(16) float smem[];
  float* Qs = smem;
  float* Ks = Qs + BM * ld;
  float* Vs = Ks + kBN * ld;
  float* Ps = Vs + kBN * ld;                                  // [BM][kBN + 4]
  int* valid = reinterpret_cast<int*>(Ps + BM * (kBN + 4));   // [kBN]: the slot's page is sound

  const int cpr = hd / VEC;  // 16-byte chunks of a row
  const T* q = static_cast<const T*>(a.q);
  for (int c = tid; c < BM * cpr; c += kThreads) {
    const int r = c / cpr, col = (c - r * cpr) * VEC;
    float f[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) f[e] = 0.f;
    if (r_lo + r < R) {
      const int i = (r_lo + r) / a.group, g = (r_lo + r) - i * a.group;
      unpack16<T>(ld_keep(q + ((s.row0 + i) * a.hq + kvh * a.group + g) * hd + col), f);
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) Qs[r * ld + col + e] = f[e] * a.qscale;
  }

  float m[MR], l[MR], acc[MR][NJ][4];
#pragma unroll
  for (int r = 0; r < MR; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.f;
#pragma unroll
    for (int j = 0; j < NJ; ++j) acc[r][j][0] = acc[r][j][1] = acc[r][j][2] = acc[r][j][3] = 0.f;
  }
  const T* kp = static_cast<const T*>(a.k_pages);
  const T* vp = static_cast<const T*>(a.v_pages);
  const int32_t* pages = a.page_table + static_cast<int64_t>(s.seq) * a.max_pages;
  const int nchunks = hd / 4;

  for (int t0 = start; t0 < end; t0 += kBN) {
    __syncthreads();  // the last tile has been read
    for (int c = tid; c < kBN * cpr; c += kThreads) {
      const int r = c / cpr, col = (c - r * cpr) * VEC;
      const int slot = t0 + r;
      float kf[VEC], vf[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) kf[e] = vf[e] = 0.f;
      bool ok = slot < end;
      if (ok) {
        const int nth = slot / a.page_size;
        const int32_t page = __ldg(pages + nth);
        ok = page >= 0 && page < a.num_pages;
        if (ok) {
          const int64_t at = ((static_cast<int64_t>(page) * a.hkv + kvh) * a.page_size + (slot - nth * a.page_size)) * hd + col;
          unpack16<T>(ld_stream(kp + at), kf);
          unpack16<T>(ld_stream(vp + at), vf);
        } else if (col == 0) {
          raise_status(a.status, BM_DEVERR_BAD_PAGE);
        }
      }
      if (col == 0) valid[r] = ok;
#pragma unroll
      for (int e = 0; e < VEC; e += 4) {
        *reinterpret_cast<float4*>(Ks + r * ld + col + e) = make_float4(kf[e], kf[e + 1], kf[e + 2], kf[e + 3]);
        *reinterpret_cast<float4*>(Vs + r * ld + col + e) = make_float4(vf[e], vf[e + 1], vf[e + 2], vf[e + 3]);
      }
    }
    __syncthreads();
    float sc[MR][4];
#pragma unroll
    for (int r = 0; r < MR; ++r) sc[r][0] = sc[r][1] = sc[r][2] = sc[r][3] = 0.f;
#pragma unroll 4
    for (int d = 0; d < hd; d += 4) {
      float4 k4[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) k4[c] = *reinterpret_cast<const float4*>(Ks + (tx + 16 * c) * ld + d);
#pragma unroll
      for (int r = 0; r < MR; ++r) {
        const float4 q4 = *reinterpret_cast<const float4*>(Qs + (ty * MR + r) * ld + d);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          sc[r][c] = fmaf(q4.x, k4[c].x, sc[r][c]);
          sc[r][c] = fmaf(q4.y, k4[c].y, sc[r][c]);
          sc[r][c] = fmaf(q4.z, k4[c].z, sc[r][c]);
          sc[r][c] = fmaf(q4.w, k4[c].w, sc[r][c]);
        }
      }
    }
#pragma unroll
    for (int r = 0; r < MR; ++r) {
      const int row = r_lo + ty * MR + r;
      const int i = row / a.group;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int slot = t0 + tx + 16 * c, j = slot - s.ctx;
        if (!valid[tx + 16 * c] || row >= R || (j >= 0 && !sees(a, s.row0, i, j))) sc[r][c] = -INFINITY;
      }
      // the 16 threads of a row are half a warp
      float mx = fmaxf(fmaxf(sc[r][0], sc[r][1]), fmaxf(sc[r][2], sc[r][3]));
#pragma unroll
      for (int off = 8; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
      const float m_new = fmaxf(m[r], mx);
      const float base = m_new == -INFINITY ? 0.f : m_new;  // nothing seen yet: every weight is 0
      const float alpha = exp2f(m[r] - base);
      m[r] = m_new;
      float sum = 0.f;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float p = exp2f(sc[r][c] - base);
        sum += p;
        Ps[(ty * MR + r) * (kBN + 4) + tx + 16 * c] = p;
      }
      l[r] = l[r] * alpha + sum;  // this thread's share of the row's sum
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[r][j][e] *= alpha;
      }
    }
    __syncwarp();  // a row's weights are written and read by the same half-warp
#pragma unroll 2
    for (int t = 0; t < kBN; t += 4) {
      float4 p4[MR];
#pragma unroll
      for (int r = 0; r < MR; ++r) p4[r] = *reinterpret_cast<const float4*>(Ps + (ty * MR + r) * (kBN + 4) + t);
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const int c = tx + 16 * j;
        if (c < nchunks) {
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const float4 v4 = *reinterpret_cast<const float4*>(Vs + (t + u) * ld + c * 4);
#pragma unroll
            for (int r = 0; r < MR; ++r) {
              const float p = u == 0 ? p4[r].x : u == 1 ? p4[r].y : u == 2 ? p4[r].z : p4[r].w;
              acc[r][j][0] = fmaf(p, v4.x, acc[r][j][0]);
              acc[r][j][1] = fmaf(p, v4.y, acc[r][j][1]);
              acc[r][j][2] = fmaf(p, v4.z, acc[r][j][2]);
              acc[r][j][3] = fmaf(p, v4.w, acc[r][j][3]);
            }
          }
        }
      }
    }
  }

#pragma unroll
  for (int r = 0; r < MR; ++r) {
#pragma unroll
    for (int off = 8; off > 0; off >>= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], off);
    const int row = r_lo + ty * MR + r;
    if (row >= R) continue;
    const int i = row / a.group, h = kvh * a.group + (row - i * a.group);
    const int64_t at = (s.row0 + i) * a.hq + h;
    if (a.splits == 1) {
      const float inv = l[r] > 0.f ? 1.f / l[r] : l[r] == 0.f ? 0.f : l[r];  // a NaN sum stays one
      T* out = static_cast<T*>(a.out) + at * hd;
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const int c = tx + 16 * j;
        if (c < nchunks) {
          if constexpr (sizeof(T) == 4) {
            *reinterpret_cast<float4*>(out + c * 4) = make_float4(acc[r][j][0] * inv, acc[r][j][1] * inv,
                                                                  acc[r][j][2] * inv, acc[r][j][3] * inv);
          } else {
            *reinterpret_cast<uint2*>(out + c * 4) = make_uint2(pack_bf16x2(acc[r][j][0] * inv, acc[r][j][1] * inv),
                                                                pack_bf16x2(acc[r][j][2] * inv, acc[r][j][3] * inv));
          }
        }
      }
    } else {
      // partial of (row, head, split): hd sums, then the sum of weights and the maximum
      float* w = a.ws + (at * a.splits + split) * (hd + 4);
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const int c = tx + 16 * j;
        if (c < nchunks) *reinterpret_cast<float4*>(w + c * 4) = make_float4(acc[r][j][0], acc[r][j][1], acc[r][j][2], acc[r][j][3]);
      }
      if (tx == 0) {
        w[hd] = l[r];
        w[hd + 1] = m[r];
      }
    }
  }
}

// Few rows (MR at most): each warp walks groups of eight slots of its own with its own
// running softmax; K and V of the next groups are on their way into its ring of shared
// memory (cp.async) meanwhile, and no barrier but the warp's own stands between. Four lanes
// share a slot: each makes a quarter of all its scores, then, these summed up, weighs a
// quarter of the rows; and a lane owns 16-byte chunks of every row of V. Multiply-adds go
// two to an instruction. The four warps' sums meet at the end. The tiled kernel above would
// read its shared K and V eight times over for a few rows. J: 16-byte chunks of a row of V
// per lane.
constexpr int kRowThreads = 128;
constexpr int kGroup = 8;   // slots of a warp's step
constexpr int kStages = 2;  // groups of a warp in flight or in use

// The ring, in whose place the warps' sums [4][MR][hd] meet at the end; then Q [MR][hd], the
// warps' weights [4][kGroup][MR], their maxima and sums.
__host__ __device__ constexpr int ring_bytes(int hd, int es) { return kRowThreads / 32 * kStages * 2 * kGroup * hd * es; }
__host__ __device__ constexpr int rows_smem(int hd, int es, int mr) {
  return ring_bytes(hd, es) + (mr * hd + kRowThreads / 32 * mr * (kGroup + 2)) * 4;
}

__device__ __forceinline__ void copy16_async(void* to, const void* from, bool real) {  // zeros where not real
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(to))),
               "l"(from), "r"(real ? 16 : 0)
               : "memory");
}

// A 16-byte chunk as pairs of fp32.
template <typename T>
__device__ __forceinline__ void unpack_pairs(const uint4& raw, uint64_t* f) {
  if constexpr (sizeof(T) == 4) {
    f[0] = pair(raw.x, raw.y);
    f[1] = pair(raw.z, raw.w);
  } else {
    f[0] = pair(bf16_lo(raw.x), bf16_hi(raw.x));
    f[1] = pair(bf16_lo(raw.y), bf16_hi(raw.y));
    f[2] = pair(bf16_lo(raw.z), bf16_hi(raw.z));
    f[3] = pair(bf16_lo(raw.w), bf16_hi(raw.w));
  }
}

template <typename T, int MR, int J>
__global__ void __launch_bounds__(kRowThreads) tree_rows_kernel(const TreeArgs a) {
  grid_dependency_wait();
  constexpr int VEC = VecWidth<T>::value;
  constexpr int kWarps = kRowThreads / 32;
  const int hd = a.hd, cpr = hd / VEC;
  int64_t id = blockIdx.x;
  const int split = static_cast<int>(id % a.splits);
  id /= a.splits;
  const int rt = static_cast<int>(id % a.row_tiles);
  id /= a.row_tiles;
  const int kvh = static_cast<int>(id % a.hkv);
  const int64_t b = id / a.hkv;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  Seq s;
  const int32_t bad = read_seq(a, b, &s);
  if (bad) {
    if (tid == 0 && split == 0 && rt == 0 && kvh == 0) raise_status(a.status, bad);
    return;
  }
  const int R = a.group * s.n, r_lo = rt * MR;
  if (r_lo >= R) return;
  const int rows = min(MR, R - r_lo);
  const int total = s.ctx + s.n;
  const int seen = a.mask ? total : s.ctx + min(s.n, (r_lo + rows - 1) / a.group + 1);
  const int start = split * a.split_len, end = min(seen, start + a.split_len);

  extern __shared__ __align__(16) float smem[];
  T* ring = reinterpret_cast<T*>(smem) + warp * kStages * 2 * kGroup * hd;
  float* Qs = smem + ring_bytes(hd, sizeof(T)) / 4;       // [MR][hd]
  float* Ps = Qs + MR * hd + warp * kGroup * MR;          // this warp's weights [kGroup][MR]
  float* ml = Qs + MR * (hd + kWarps * kGroup);           // [kWarps][MR] maxima, then sums
  const T* kp = static_cast<const T*>(a.k_pages);
  const T* vp = static_cast<const T*>(a.v_pages);
  const int32_t* pages = a.page_table + static_cast<int64_t>(s.seq) * a.max_pages;
  const int own = lane >> 2, sub = lane & 3;  // this lane's slot of the group, its quarter of K's chunks
  // Neighbouring rows' chunks lie 64 bytes apart in the banks, by the pitch or by a swap.
  const int swap = cpr % 8 == 0 ? 4 : 0;

  uint32_t sound = 0;  // bit i: this lane's slot in stage i has a sound page
  auto fetch = [&](int g0, int stage) {
    const int slot = g0 + own;
    int64_t at = -1;  // the slot's row of the pages
    if (slot < end) {
      const int nth = slot / a.page_size;
      const int32_t page = __ldg(pages + nth);
      if (page >= 0 && page < a.num_pages) {
        at = ((static_cast<int64_t>(page) * a.hkv + kvh) * a.page_size + (slot - nth * a.page_size)) * hd;
      } else if (sub == 0) {
        raise_status(a.status, BM_DEVERR_BAD_PAGE);
      }
    }
    const bool real = at >= 0;
    sound = (sound & ~(1u << stage)) | (real ? 1u << stage : 0u);
    if (g0 < end) {
      const T* k_from = kp + (real ? at : 0);
      const T* v_from = vp + (real ? at : 0);
      T* k_to = ring + (stage * 2 * kGroup + own) * hd;
      T* v_to = k_to + kGroup * hd;
      for (int c = sub; c < cpr; c += 4) copy16_async(k_to + (c ^ (own & 1 ? swap : 0)) * VEC, k_from + c * VEC, real);
      for (int c = sub; c < cpr; c += 4) copy16_async(v_to + (c ^ (own & 1 ? swap : 0)) * VEC, v_from + c * VEC, real);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  const int first = start + warp * kGroup;
  for (int i = 0; i < kStages; ++i) fetch(first + i * kWarps * kGroup, i);

  const T* q = static_cast<const T*>(a.q);
  for (int c = tid; c < MR * cpr; c += kRowThreads) {
    const int r = c / cpr, col = (c - r * cpr) * VEC;
    float f[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) f[e] = 0.f;
    if (r < rows) {
      const int i = (r_lo + r) / a.group, g = (r_lo + r) - i * a.group;
      unpack16<T>(ld_keep(q + ((s.row0 + i) * a.hq + kvh * a.group + g) * hd + col), f);
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) Qs[r * hd + col + e] = f[e] * a.qscale;
  }
  __syncthreads();

  constexpr int RL = MR / 4;        // rows that a lane weighs for its slot, from
  const int r_own = sub * RL;       // this one on
  constexpr int P2 = J * VEC / 2;   // pairs of a row's dims that a lane owns
  float m[RL], l[RL];
  uint64_t acc[MR][P2];
#pragma unroll
  for (int r = 0; r < RL; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.f;
  }
#pragma unroll
  for (int r = 0; r < MR; ++r) {
#pragma unroll
    for (int e = 0; e < P2; ++e) acc[r][e] = 0;
  }
  int stage = 0;
  for (int g0 = first; g0 < end; g0 += kWarps * kGroup) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
    __syncwarp();  // all lanes' copies of this group are there
    const T* ks = ring + (stage * 2 * kGroup + own) * hd;
    const T* vs = ring + (stage * 2 + 1) * kGroup * hd;
    uint64_t s2[MR];
#pragma unroll
    for (int r = 0; r < MR; ++r) s2[r] = 0;
#pragma unroll 4
    for (int c = sub; c < cpr; c += 4) {
      uint64_t k2[VEC / 2];
      unpack_pairs<T>(*reinterpret_cast<const uint4*>(ks + (c ^ (own & 1 ? swap : 0)) * VEC), k2);
#pragma unroll
      for (int r = 0; r < MR; ++r) {
#pragma unroll
        for (int e = 0; e < VEC; e += 4) {
          const ulonglong2 q4 = *reinterpret_cast<const ulonglong2*>(Qs + r * hd + c * VEC + e);
          s2[r] = fma2(q4.x, k2[e / 2], s2[r]);
          s2[r] = fma2(q4.y, k2[e / 2 + 1], s2[r]);
        }
      }
    }
    __syncwarp();  // lanes may have left the loop apart; the last group's weights have been read
    float sc[MR];
#pragma unroll
    for (int r = 0; r < MR; ++r) {
      const float2 two = unpair(s2[r]);
      sc[r] = two.x + two.y;
    }
    // the four quarters' sums: half of the rows stay with a lane, then half of these
#pragma unroll
    for (int keep = MR / 2; keep >= RL; keep /= 2) {
      const int bit = keep == MR / 2 ? 2 : 1;
      const bool upper = sub & bit;
#pragma unroll
      for (int r = 0; r < keep; ++r) {
        const float give = upper ? sc[r] : sc[r + keep], have = upper ? sc[r + keep] : sc[r];
        sc[r] = have + __shfl_xor_sync(0xffffffffu, give, bit);
      }
    }
    const bool real = (sound >> stage) & 1;
    const int j0 = g0 + own - s.ctx;
    float alpha[RL], p[RL];
    bool rise = false;
#pragma unroll
    for (int r = 0; r < RL; ++r) {
      if (!real || r_own + r >= rows || (j0 >= 0 && !sees(a, s.row0, (r_lo + r_own + r) / a.group, j0))) sc[r] = -INFINITY;
      float mx = sc[r];
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
      const float m_new = fmaxf(m[r], mx);
      const float base = m_new == -INFINITY ? 0.f : m_new;
      rise = rise || m_new > m[r];
      alpha[r] = exp2f(m[r] - base);
      p[r] = exp2f(sc[r] - base);
      m[r] = m_new;
      l[r] = l[r] * alpha[r] + p[r];  // this slot's share
      Ps[own * MR + r_own + r] = p[r];
    }
    if (__any_sync(0xffffffffu, rise)) {
#pragma unroll
      for (int r = 0; r < MR; ++r) {
        const float f = __shfl_sync(0xffffffffu, alpha[r % RL], r / RL);
#pragma unroll
        for (int e = 0; e < P2; ++e) acc[r][e] = mul2(acc[r][e], pair(f, f));
      }
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < kGroup; ++i) {
      uint64_t w[MR];
#pragma unroll
      for (int r = 0; r < MR; r += 4) {
        const float4 p4 = *reinterpret_cast<const float4*>(Ps + i * MR + r);
        w[r] = pair(p4.x, p4.x);
        w[r + 1] = pair(p4.y, p4.y);
        w[r + 2] = pair(p4.z, p4.z);
        w[r + 3] = pair(p4.w, p4.w);
      }
#pragma unroll
      for (int j = 0; j < J; ++j) {
        if (lane + 32 * j >= cpr) continue;
        uint64_t v2[VEC / 2];
        unpack_pairs<T>(*reinterpret_cast<const uint4*>(vs + i * hd + ((lane + 32 * j) ^ (i & 1 ? swap : 0)) * VEC), v2);
#pragma unroll
        for (int r = 0; r < MR; ++r) {
#pragma unroll
          for (int e = 0; e < VEC / 2; ++e) acc[r][j * VEC / 2 + e] = fma2(w[r], v2[e], acc[r][j * VEC / 2 + e]);
        }
      }
    }
    __syncwarp();  // this group has been read
    fetch(g0 + kStages * kWarps * kGroup, stage);
    if (++stage == kStages) stage = 0;
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  // the warps' maxima, sums of weights and of values
#pragma unroll
  for (int r = 0; r < RL; ++r) {
#pragma unroll
    for (int off = 4; off < 32; off <<= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], off);
    if (own == 0) {
      ml[warp * MR + r_own + r] = m[r];
      ml[(kWarps + warp) * MR + r_own + r] = l[r];
    }
  }
  __syncthreads();  // the rings have been read
#pragma unroll
  for (int r = 0; r < MR; ++r) {
#pragma unroll
    for (int j = 0; j < J; ++j) {
      if (lane + 32 * j < cpr) {
#pragma unroll
        for (int e = 0; e < VEC; e += 4) {
          *reinterpret_cast<ulonglong2*>(smem + (warp * MR + r) * hd + (lane + 32 * j) * VEC + e) =
              make_ulonglong2(acc[r][(j * VEC + e) / 2], acc[r][(j * VEC + e) / 2 + 1]);
        }
      }
    }
  }
  __syncthreads();
  for (int c = tid; c < rows * (hd / 4); c += kRowThreads) {
    const int r = c / (hd / 4), d = (c - r * (hd / 4)) * 4;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, ml[w * MR + r]);
    const float base = top == -INFINITY ? 0.f : top;
    float sum = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = exp2f(ml[w * MR + r] - base);
      sum = fmaf(ml[(kWarps + w) * MR + r], f, sum);
      const float4 part = *reinterpret_cast<const float4*>(smem + (w * MR + r) * hd + d);
      o = make_float4(fmaf(part.x, f, o.x), fmaf(part.y, f, o.y), fmaf(part.z, f, o.z), fmaf(part.w, f, o.w));
    }
    const int i = (r_lo + r) / a.group, h = kvh * a.group + (r_lo + r - i * a.group);
    const int64_t row = (s.row0 + i) * a.hq + h;
    if (a.splits == 1) {
      const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;
      T* out = static_cast<T*>(a.out) + row * hd + d;
      if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4*>(out) = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
      } else {
        *reinterpret_cast<uint2*>(out) = make_uint2(pack_bf16x2(o.x * inv, o.y * inv), pack_bf16x2(o.z * inv, o.w * inv));
      }
    } else {
      float* w = a.ws + (row * a.splits + split) * (hd + 4);
      *reinterpret_cast<float4*>(w + d) = o;
      if (d == 0) {
        w[hd] = sum;
        w[hd + 1] = top;
      }
    }
  }
}

// One warp per (row, head): the splits' partials, each scaled to the common maximum.
template <typename T>
__global__ void __launch_bounds__(kThreads) tree_combine_kernel(const TreeArgs a) {
  grid_dependency_wait();
  const int lane = threadIdx.x & 31;
  const int64_t warp = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) >> 5;
  const int h = static_cast<int>(warp % a.hq);
  const int64_t bi = warp / a.hq;
  const int i = static_cast<int>(bi % a.max_tree);
  const int64_t b = bi / a.max_tree;
  if (b >= a.batch) return;
  Seq s;
  if (read_seq(a, b, &s) || i >= s.n) return;
  const int64_t at = (s.row0 + i) * a.hq + h;
  const float* w = a.ws + at * a.splits * (a.hd + 4);
  float m = -INFINITY;
  for (int k = 0; k < a.splits; ++k) m = fmaxf(m, w[k * (a.hd + 4) + a.hd + 1]);
  const float base = m == -INFINITY ? 0.f : m;
  float l = 0.f;
  for (int k = 0; k < a.splits; ++k) {
    l = fmaf(w[k * (a.hd + 4) + a.hd], exp2f(w[k * (a.hd + 4) + a.hd + 1] - base), l);
  }
  const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;
  for (int c = lane; c < a.hd / 4; c += 32) {
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k = 0; k < a.splits; ++k) {
      const float f = exp2f(w[k * (a.hd + 4) + a.hd + 1] - base) * inv;
      const float4 p = *reinterpret_cast<const float4*>(w + k * (a.hd + 4) + c * 4);
      o.x = fmaf(f, p.x, o.x);
      o.y = fmaf(f, p.y, o.y);
      o.z = fmaf(f, p.z, o.z);
      o.w = fmaf(f, p.w, o.w);
    }
    T* out = static_cast<T*>(a.out) + at * a.hd + c * 4;
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<float4*>(out) = o;
    } else {
      *reinterpret_cast<uint2*>(out) = make_uint2(pack_bf16x2(o.x, o.y), pack_bf16x2(o.z, o.w));
    }
  }
}

// Rows of a CTA: 4 and 8 are tree_rows_kernel's, the others the tiled kernel's. Up to 32
// rows, tiles of 8 of them beat a tiled kernel cut to 32 rows (16 sequences of 1000 to 2000,
// 8 heads: 24 rows of 128 in fp32 193 against 244 us, 32 rows of 256 in bf16 361 against 563,
// though 32 rows of 128 in fp32 268 against 255); a tile of 8 for 4 rows costs twice as much
// (4 rows of 256 in bf16: 210 against 107 us).
int rows_per_tile(int rows) { return rows > 32 ? BM : rows > 4 ? 8 : 4; }

// The CUDA-core form's split: enough CTAs for four per SM (eight of the few-row kernel's),
// none shorter than a tile.
void plan(int64_t batch, int hkv, int group, int max_ctx, int max_tree, int* row_tiles, int* splits, int* split_len) {
  const int rows = group * max_tree, bm = rows_per_tile(rows);
  *row_tiles = (rows + bm - 1) / bm;
  const int len = max_ctx + max_tree;
  const int64_t ctas = batch * hkv * *row_tiles;
  const int64_t want = ((bm <= 8 ? 8 : 4) * static_cast<int64_t>(sm_count()) + ctas - 1) / ctas;
  const int most = std::max(1, len / kBN);
  const int n = static_cast<int>(std::min<int64_t>(want, std::min(most, 64)));
  *split_len = ((len + n - 1) / n + kBN - 1) / kBN * kBN;
  *splits = (len + *split_len - 1) / *split_len;
}

template <typename T, int NJ>
int launch_one(const TreeArgs& a, cudaStream_t stream, const char* what) {
  const int ld = a.hd + 4;
  const int smem = ((BM + 2 * kBN) * ld + BM * (kBN + 4) + kBN) * 4;
  auto kernel = tree_attention_kernel<T, NJ>;
  if (int st = allow_dynamic_smem(reinterpret_cast<const void*>(kernel), smem, what)) return st;
  const int64_t grid = a.batch * a.hkv * a.row_tiles * a.splits;
  return launch_kernel(what, kernel, dim3(static_cast<unsigned>(grid)), dim3(kThreads), smem, stream, nullptr, a);
}

template <typename T>
int launch(TreeArgs a, cudaStream_t stream, const char* what) {
  const int nj = (a.hd + 63) / 64;
  auto few = [&](auto mr) {
    constexpr int MR = decltype(mr)::value;
    const int smem = rows_smem(a.hd, sizeof(T), MR);
    const int64_t grid = a.batch * a.hkv * a.row_tiles * a.splits;
    auto kernel = tree_rows_kernel<T, MR, 1>;
    if constexpr (sizeof(T) == 4) {
      if (a.hd > 128) kernel = tree_rows_kernel<T, MR, 2>;
    }
    if (int st = allow_dynamic_smem(reinterpret_cast<const void*>(kernel), smem, what)) return st;
    return launch_kernel(what, kernel, dim3(static_cast<unsigned>(grid)), dim3(kRowThreads), smem, stream, nullptr, a);
  };
  const int rows = rows_per_tile(a.group * a.max_tree);
  const int st = rows == 4   ? few(std::integral_constant<int, 4>{})
                 : rows == 8 ? few(std::integral_constant<int, 8>{})
                 : nj == 1   ? launch_one<T, 1>(a, stream, what)
                 : nj == 2   ? launch_one<T, 2>(a, stream, what)
                             : launch_one<T, 4>(a, stream, what);
  if (st != BM_OK || a.splits == 1) return st;
  const int64_t warps = a.batch * a.max_tree * a.hq;
  const int64_t grid = (warps + kThreads / 32 - 1) / (kThreads / 32);
  return launch_kernel(what, tree_combine_kernel<T>, dim3(static_cast<unsigned>(grid)), dim3(kThreads), 0, stream,
                       nullptr, a);
}

int check_sizes(const char* what, int64_t total_q, int64_t batch, int hq, int hkv, int hd, int max_ctx, int max_tree) {
  if (total_q < 0 || batch < 0 || total_q > INT32_MAX || batch > INT32_MAX) {
    return fail(BM_ERR_INVALID_ARGUMENT, "%s: bad total_q or batch", what);
  }
  if (hq <= 0 || hkv <= 0 || hq % hkv || hq / hkv > 64) {
    return fail(BM_ERR_INVALID_ARGUMENT, "%s: num_q_heads must be a multiple (at most 64) of num_kv_heads", what);
  }
  if (hd <= 0 || hd > 256) return fail(BM_ERR_INVALID_ARGUMENT, "%s: head_dim %d outside [1, 256]", what, hd);
  if (max_ctx < 0 || max_tree < 0 || static_cast<int64_t>(max_ctx) + max_tree > (1 << 30)) {
    return fail(BM_ERR_INVALID_ARGUMENT, "%s: bad max_ctx or max_tree", what);
  }
  // One CTA per (sequence, kv head, row tile, split) and one warp per (row, head) of the
  // bounds: both grids, and the row numbers, stay within 32 bits.
  if (batch > 0 && max_tree > 0 && static_cast<int64_t>(max_tree) * hq > INT32_MAX / 64 / batch) {
    return fail(BM_ERR_INVALID_ARGUMENT, "%s: batch * max_tree * num_q_heads above 2^25", what);
  }
  return BM_OK;
}

size_t simt_workspace_bytes(int64_t total_q, int64_t batch, int hq, int hkv, int hd, int max_ctx, int max_tree) {
  if (batch == 0 || max_tree == 0) return 0;
  int row_tiles, splits, split_len;
  plan(batch, hkv, hq / hkv, max_ctx, max_tree, &row_tiles, &splits, &split_len);
  return splits == 1 ? 0 : static_cast<size_t>(total_q) * hq * splits * (hd + 4) * sizeof(float);
}

}  // namespace
}  // namespace paged

int check_paged_kv(const char* what, const bm_paged_kv_t* c) {
  if (!c) return fail(BM_ERR_INVALID_ARGUMENT, "%s: NULL cache", what);
  if (!c->k_pages || !c->v_pages || !c->page_table) return fail(BM_ERR_INVALID_ARGUMENT, "%s: NULL pointer in the cache", what);
  if (c->num_pages <= 0 || c->page_size <= 0 || c->max_pages <= 0 || c->num_seqs <= 0 || c->num_kv_heads <= 0 ||
      c->head_dim <= 0 || c->num_kv_heads > (1 << 16)) {
    return fail(BM_ERR_INVALID_ARGUMENT, "%s: bad sizes in the cache", what);
  }
  if (static_cast<int64_t>(c->page_size) * c->max_pages > INT32_MAX) {
    return fail(BM_ERR_INVALID_ARGUMENT, "%s: page_size * max_pages above 2^31 - 1", what);
  }
  return BM_OK;
}

bool meets_pages(const bm_paged_kv_t& c, const void* p, uintptr_t bytes, int es) {
  const uintptr_t from = reinterpret_cast<uintptr_t>(p);
  const uintptr_t all = static_cast<uintptr_t>(c.num_pages) * c.num_kv_heads * c.page_size * c.head_dim * es;
  for (const void* pages : {c.k_pages, c.v_pages}) {
    const uintptr_t lo = reinterpret_cast<uintptr_t>(pages);
    if (from < lo + all && lo < from + bytes) return true;
  }
  return false;
}

}  // namespace bm

extern "C" int bm_paged_tree_attention_workspace_size(int64_t total_q, int64_t batch, int32_t num_q_heads,
                                                      int32_t num_kv_heads, int32_t head_dim, int32_t max_ctx,
                                                      int32_t max_tree, size_t* bytes_out) {
  using namespace bm;
  const char* what = "bm_paged_tree_attention_workspace_size";
  if (!bytes_out) return fail(BM_ERR_INVALID_ARGUMENT, "%s: NULL bytes_out", what);
  *bytes_out = 0;
  if (int st = paged::check_sizes(what, total_q, batch, num_q_heads, num_kv_heads, head_dim, max_ctx, max_tree)) return st;
  if (batch == 0 || max_tree == 0) return BM_OK;
  *bytes_out = std::max(paged::simt_workspace_bytes(total_q, batch, num_q_heads, num_kv_heads, head_dim, max_ctx, max_tree),
                        paged::tc_workspace_bytes(batch, num_kv_heads, head_dim, num_q_heads / num_kv_heads,
                                                  max_ctx, max_tree));
  return BM_OK;
}

extern "C" int bm_paged_tree_attention(void* out, const void* q, const bm_paged_kv_t* cache, const int32_t* seq_ids,
                                       const int32_t* ctx_lens, const int32_t* q_starts, const uint64_t* tree_mask,
                                       int32_t mask_words, int64_t total_q, int64_t batch, int32_t num_q_heads,
                                       int32_t max_ctx, int32_t max_tree, float scale, void* workspace,
                                       size_t workspace_bytes, bm_dtype_t dtype, int32_t* d_status, void* stream) {
  using namespace bm;
  const char* what = "bm_paged_tree_attention";
  if (!valid_dtype(dtype)) return fail(BM_ERR_INVALID_ARGUMENT, "%s: bad dtype %d", what, static_cast<int>(dtype));
  if (int st = check_paged_kv(what, cache)) return st;
  const bm_paged_kv_t& c = *cache;
  if (int st = paged::check_sizes(what, total_q, batch, num_q_heads, c.num_kv_heads, c.head_dim, max_ctx, max_tree)) return st;
  if (c.head_dim * dtype_size(dtype) % 16) {
    return fail(BM_ERR_INVALID_ARGUMENT, "%s: head_dim %d is not whole 16-byte rows", what, c.head_dim);
  }
  if (tree_mask && (mask_words <= 0 || max_tree > 64 * static_cast<int64_t>(mask_words))) {
    return fail(BM_ERR_INVALID_ARGUMENT, "%s: max_tree %d does not fit %d mask words", what, max_tree, mask_words);
  }
  const float s = scale > 0.f ? scale : 1.f / std::sqrt(static_cast<float>(c.head_dim));
  const float qscale = s * 1.4426950408889634f;  // the softmax runs in base 2
  if (scale != scale || !std::isfinite(qscale)) return fail(BM_ERR_INVALID_ARGUMENT, "%s: scale is not finite", what);
  if (batch == 0 || total_q == 0 || max_tree == 0) return BM_OK;
  if (!out || !q || !ctx_lens || !q_starts) return fail(BM_ERR_INVALID_ARGUMENT, "%s: NULL pointer", what);
  if (!aligned16(out) || !aligned16(q) || !aligned16(c.k_pages) || !aligned16(c.v_pages) || !aligned16(workspace)) {
    return fail(BM_ERR_INVALID_ARGUMENT, "%s: q, out, pages and workspace must be 16-byte aligned", what);
  }
  if (!aligned_to({seq_ids, ctx_lens, q_starts, c.page_table, d_status}, 4) || !aligned_to(tree_mask, 8)) {
    return fail(BM_ERR_INVALID_ARGUMENT, "%s: a pointer is not aligned to its elements", what);
  }
  if (!seq_ids && batch > c.num_seqs) return fail(BM_ERR_INVALID_ARGUMENT, "%s: more sequences than the cache holds", what);
  const uintptr_t o = reinterpret_cast<uintptr_t>(out), i = reinterpret_cast<uintptr_t>(q);
  const uintptr_t bytes = static_cast<uintptr_t>(total_q) * num_q_heads * c.head_dim * dtype_size(dtype);
  if (o < i + bytes && i < o + bytes) return fail(BM_ERR_INVALID_ARGUMENT, "%s: out overlaps q", what);
  if (meets_pages(c, out, bytes, dtype_size(dtype))) return fail(BM_ERR_INVALID_ARGUMENT, "%s: out overlaps the cache's pages", what);
  const size_t simt = paged::simt_workspace_bytes(total_q, batch, num_q_heads, c.num_kv_heads, c.head_dim, max_ctx, max_tree);
  const size_t tc = paged::tc_workspace_bytes(batch, c.num_kv_heads, c.head_dim, num_q_heads / c.num_kv_heads, max_ctx,
                                              max_tree);
  if (std::max(simt, tc) > 0 && (!workspace || workspace_bytes < std::max(simt, tc))) {
    return fail(BM_ERR_INVALID_ARGUMENT, "%s: workspace of %zu bytes is smaller than %zu", what, workspace_bytes,
                std::max(simt, tc));
  }
  paged::TreeArgs a{};
  a.out = out;
  a.q = q;
  a.k_pages = c.k_pages;
  a.v_pages = c.v_pages;
  a.page_table = c.page_table;
  a.seq_ids = seq_ids;
  a.ctx_lens = ctx_lens;
  a.q_starts = q_starts;
  a.mask = tree_mask;
  a.words = mask_words;
  a.ws = static_cast<float*>(workspace);
  a.total_q = total_q;
  a.batch = batch;
  a.hq = num_q_heads;
  a.hkv = c.num_kv_heads;
  a.hd = c.head_dim;
  a.group = num_q_heads / c.num_kv_heads;
  a.num_pages = c.num_pages;
  a.page_size = c.page_size;
  a.max_pages = c.max_pages;
  a.num_seqs = c.num_seqs;
  a.max_ctx = max_ctx;
  a.max_tree = max_tree;
  a.qscale = qscale;
  a.status = d_status;
  if (paged::tc_takes(a, dtype)) return paged::launch_tc(a, as_stream(stream), what);
  paged::plan(batch, a.hkv, a.group, max_ctx, max_tree, &a.row_tiles, &a.splits, &a.split_len);
  return dtype == BM_F32 ? paged::launch<float>(a, as_stream(stream), what) : paged::launch<bf16>(a, as_stream(stream), what);
}
