// Pieces of the paged tree attention shared by its CUDA-core kernels
// (paged_attention.cu) and its tensor-core kernel (paged_attention_tc.cu).
#pragma once

#include "bm_common.cuh"
#include "bm_host.h"

namespace bm {
namespace paged {

struct TreeArgs {
  void* out;                  // [total_q][hq][hd]
  const void* q;
  const void* k_pages;        // [num_pages][hkv][page_size][hd]
  const void* v_pages;
  const uint8_t* k_scales;    // an 8-bit cache's: [num_pages][hkv][page_size / block]
  const uint8_t* v_scales;
  int block;
  const int32_t* page_table;  // [num_seqs][max_pages]
  const int32_t* seq_ids;     // NULL: b
  const int32_t* ctx_lens;
  const int32_t* q_starts;    // [batch + 1]
  const uint64_t* mask;       // [total_q][words]; NULL: drafted slot j is seen by rows i >= j
  float* ws;
  int64_t total_q, batch;
  int words;
  int hq, hkv, hd, group;
  int num_pages, page_size, max_pages, num_seqs;
  int max_ctx, max_tree;
  int tile, box;              // tensor-core form: slots of a tile, rows of the boxes that fill it
  bool whole;                 // and whether items stay whole
  int item_cost;              // what beginning and ending an item costs, in tiles (0: not counted)
  int splits, split_len;      // CUDA-core form: the slots shared out over CTAs
  int row_tiles;              // and the query rows of a sequence and kv head
  float qscale;               // scale * log2(e): the softmax runs in base 2
  int32_t* status;
};

// One sequence of the batch: its cache sequence, context, rows and first row.
struct Seq {
  int seq, ctx, n;
  int64_t row0;
};

// Reads and checks sequence b; the returned BM_DEVERR_* bits are 0 when it is sound.
// Reads q_starts[b], q_starts[b + 1], ctx_lens[b] and seq_ids[b] only.
__device__ __forceinline__ int32_t read_seq(const TreeArgs& a, int64_t b, Seq* s) {
  const int32_t r0 = __ldg(a.q_starts + b), r1 = __ldg(a.q_starts + b + 1);
  s->ctx = __ldg(a.ctx_lens + b);
  s->seq = a.seq_ids ? __ldg(a.seq_ids + b) : static_cast<int>(b);
  s->row0 = r0;
  const int64_t n = static_cast<int64_t>(r1) - r0;
  s->n = static_cast<int>(n);
  int32_t bad = 0;
  if (r0 < 0 || r1 > a.total_q || n < 0 || n > a.max_tree || s->ctx < 0 || s->ctx > a.max_ctx ||
      (n > 0 && s->ctx + n > static_cast<int64_t>(a.max_pages) * a.page_size)) {
    bad |= BM_DEVERR_BAD_POSITION;
  }
  if (s->seq < 0 || s->seq >= a.num_seqs) bad |= BM_DEVERR_BAD_SEQUENCE;
  if (bad) s->n = 0;
  return bad;
}

// Whether drafted slot j is seen by row i of the sequence whose first row is row0
// (0 <= j < n is the caller's).
__device__ __forceinline__ bool sees(const TreeArgs& a, int64_t row0, int i, int j) {
  if (a.mask == nullptr) return j <= i;
  return (__ldg(a.mask + (row0 + i) * a.words + (j >> 6)) >> (j & 63)) & 1;
}

// The tensor-core forms (paged_attention_tc.cu; tc8: paged_attention8_tc.cu): whether they take
// these arguments, the scratch they need (the same), and their launches.
bool tc_takes(const TreeArgs& a, bm_dtype_t dtype);
size_t tc_workspace_bytes(int64_t batch, int hkv, int hd, int group, int max_ctx, int max_tree);
int launch_tc(const TreeArgs& a, cudaStream_t stream, const char* what);
bool tc8_takes(const TreeArgs& a, bm_dtype_t dtype);
int launch_tc8(const TreeArgs& a, cudaStream_t stream, const char* what);

}  // namespace paged
}  // namespace bm
