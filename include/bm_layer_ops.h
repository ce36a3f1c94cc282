/*
 * bm_layer_ops.h — C ABI of the B200 (sm_100a) fused transformer-layer kernels.
 *
 * The memory-bound per-token ops of a Llama layer, batched over rows (tokens):
 * token-embedding gather, RMSNorm (optionally fused with the residual add),
 * RoPE on Q and the GQA K heads written into a static KV cache, and SwiGLU.
 *
 * Conventions shared by every entry point:
 *   - Plain pointers and sizes only. Every data pointer is a device pointer on
 *     the CUDA device that is current on the calling thread; `stream` is a
 *     cudaStream_t of that device passed as void* (NULL = legacy default stream).
 *   - Launches are asynchronous and stream-ordered; no entry point synchronises,
 *     except bm_status_read, which says so.
 *   - Nothing allocates device memory, except bm_rope_table_create.
 *   - The return value is a bm_status_t. Host-side argument checks happen before
 *     any launch: on failure nothing is launched. No entry point calls exit().
 *   - Data types: BM_F32 (IEEE fp32) or BM_BF16 (bfloat16 storage, 2 bytes).
 *     Arithmetic is fp32 in every kernel; outputs are rounded to nearest-even.
 *   - Rows are dense and row-major unless a stride argument says otherwise.
 *     16-byte aligned pointers with 16-byte multiple row pitches take the
 *     128-bit vector path; anything else runs a scalar path with the same
 *     results. Every pointer is aligned to its elements.
 *   - Values that only the device can check (token ids, positions and sequence
 *     ids held in device arrays) are checked by the kernels. A bad row is skipped
 *     (its outputs are left unwritten) and a BM_DEVERR_* bit is OR-ed into
 *     *d_status when d_status is not NULL. Read it with bm_status_read.
 *
 * Each entry point cites the reference interface it replaces
 * (NolanKisser/BareMetalInferenceEngine, paths within that project).
 */
#ifndef BM_LAYER_OPS_H
#define BM_LAYER_OPS_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define BM_ABI_VERSION 1

typedef enum bm_dtype {
  BM_F32 = 0,
  BM_BF16 = 1
} bm_dtype_t;

typedef enum bm_status {
  BM_OK = 0,
  BM_ERR_INVALID_ARGUMENT = 1, /* a size, pointer or dtype fails a host-side check */
  BM_ERR_CUDA = 2,             /* a CUDA runtime call or launch failed */
  BM_ERR_DEVICE = 3            /* bm_status_read found BM_DEVERR_* bits set */
} bm_status_t;

/* Bits a kernel OR-s into *d_status. */
#define BM_DEVERR_BAD_ID 0x1       /* token id outside [0, vocab) */
#define BM_DEVERR_BAD_POSITION 0x2 /* position outside [0, max_seq) or beyond the RoPE table */
#define BM_DEVERR_BAD_SEQUENCE 0x4 /* sequence id outside [0, num_seqs) */
#define BM_DEVERR_TIMEOUT 0x8      /* a tensor-core pipeline wait passed its time limit; outputs incomplete */
#define BM_DEVERR_BAD_PAGE 0x10    /* page id of a page table outside [0, num_pages) */
#define BM_DEVERR_BAD_PARAMETER 0x20 /* a sampling setting or uniform number of a row outside its range */

/* Human-readable name of a bm_status_t. Never NULL. */
const char* bm_status_string(int status);

/* BM_ABI_VERSION of the loaded library. */
int bm_abi_version(void);

/* Message of the last BM_ERR_* returned on this host thread ("" if none). */
const char* bm_last_error_message(void);

/* Synchronises `stream`, copies *d_status into *flags_out (host) and clears
 * *d_status to 0. Returns BM_ERR_DEVICE when any bit was set, else BM_OK. */
int bm_status_read(int32_t* d_status, int32_t* flags_out, void* stream);

/* ---------------------------------------------------------------------------
 * Embedding gather: out[r, :] = table[ids[r], :]  (bit-exact copy).
 * Replaces the per-token row copy in ExecutionEngine::run_layers
 * (src/execution_engine.cu:98-99) and the host id check of forward()
 * (src/execution_engine.cu:63-65), which becomes BM_DEVERR_BAD_ID.
 * table: [vocab][dim]; out: rows of `dim` elements, `out_row_stride` elements
 * apart (>= dim).
 */
int bm_embed_gather(void* out, const void* table, const int32_t* ids,
                    int64_t rows, int64_t dim, int64_t vocab,
                    int64_t out_row_stride, bm_dtype_t dtype,
                    int32_t* d_status, void* stream);

/* ---------------------------------------------------------------------------
 * RMSNorm over rows: out[r,i] = in[r,i] * rsqrt(mean_i(in[r,:]^2) + eps) * weight[i].
 * Replaces launch_rms_norm (include/kernels.cuh:9, src/kernels.cu:59-78), which
 * normalises one vector per launch. out may equal in (in place).
 * in/out rows are in_stride / out_stride elements apart (>= dim).
 */
int bm_rmsnorm(void* out, const void* in, const void* weight,
               int64_t rows, int64_t dim, float eps,
               int64_t in_stride, int64_t out_stride,
               bm_dtype_t dtype, void* stream);

/* ---------------------------------------------------------------------------
 * Fused residual add + RMSNorm:
 *   residual[r,:] <- residual[r,:] + delta[r,:]      (fp32 add, stored in dtype)
 *   out[r,:]       = rmsnorm(residual[r,:]) * weight (on the stored values)
 * Replaces the pair launch_add(hidden, hidden, projected) followed by
 * launch_rms_norm(normed, hidden, w) (src/execution_engine.cu:118+121 and
 * :126+:109/:80; include/kernels.cuh:9,32). Rows are dense ([rows][dim]).
 * out must not overlap residual or delta.
 */
int bm_add_rmsnorm(void* residual, const void* delta, const void* weight,
                   void* out, int64_t rows, int64_t dim, float eps,
                   bm_dtype_t dtype, void* stream);

/* ---------------------------------------------------------------------------
 * Element-wise add: out = a + b over n elements. out may equal a or b.
 * Replaces launch_add (include/kernels.cuh:32, src/kernels.cu:199-207).
 */
int bm_add(void* out, const void* a, const void* b, int64_t n,
           bm_dtype_t dtype, void* stream);

/* ---------------------------------------------------------------------------
 * SwiGLU: out = silu(gate) * up = gate / (1 + exp(-gate)) * up over n elements.
 * Replaces launch_swiglu (include/kernels.cuh:29, src/kernels.cu:185-195).
 * out may equal gate or up.
 */
int bm_swiglu(void* out, const void* gate, const void* up, int64_t n,
              bm_dtype_t dtype, void* stream);

/* ---------------------------------------------------------------------------
 * One layer step: the five ops above in the order ExecutionEngine::run_layers
 * issues them for a token (src/execution_engine.cu:98-126), for a batch of
 * rows, equivalent to
 *   bm_embed_gather(hidden <- embed[ids])
 *   bm_add_rmsnorm(hidden += attn_out; y_attn = rmsnorm(hidden) * w_attn)
 *   bm_rope_kv_store(q in place; rotated k and v into the caches)
 *   bm_add_rmsnorm(hidden += ffn_out; y_ffn = rmsnorm(hidden) * w_ffn)
 *   bm_swiglu(act = silu(gate) * up)
 * No single reference function: it groups the reference's per-token calls.
 * Every input (the GEMM and attention outputs included) must be ready when it is
 * called; inside one transformer layer they are not (attn_out depends on y_attn
 * through the projections and the attention), so a layer loop calls the ops
 * separately and this one-call form serves steps whose inputs are at hand together.
 * Batches of at most 512 tokens with 16-byte aligned buffers and whole-vector
 * rows run as ONE launch (the only dependency between the ops is the row-local
 * residual, so the launch holds independent row, token and SwiGLU jobs); larger
 * batches issue the five batched kernels. Results are the same either way (the
 * residual and the cache copies bit for bit). Every array is row-major and
 * contiguous: hidden, attn_out, y_attn, ffn_out, y_ffn [rows][dim]; q
 * [rows][num_q_heads][head_dim]; k, v [rows][num_kv_heads][head_dim]; gate, up,
 * act [rows][ffn]; caches [num_seqs][num_kv_heads][max_seq][head_dim];
 * positions and ids int32[rows]; seq_ids int32[rows] or NULL (all 0);
 * rope_table as for bm_rope_kv_store (NULL: fp64 angles from theta). Bad ids,
 * positions and sequences flag *d_status and skip that row's op, as the
 * separate calls do. */
typedef struct bm_layer_step {
  int64_t rows;
  int32_t dim, ffn;
  int64_t vocab;
  int32_t num_q_heads, num_kv_heads, head_dim, max_seq, num_seqs;
  float eps;
  double theta;
  const int32_t* ids;
  const void* embed;
  void* hidden;
  const void* attn_out;
  const void* w_attn;
  void* y_attn;
  void* q;
  const void* k;
  const void* v;
  const int32_t* positions;
  const int32_t* seq_ids;
  void* k_cache;
  void* v_cache;
  const void* rope_table;
  int32_t rope_table_len;
  const void* ffn_out;
  const void* w_ffn;
  void* y_ffn;
  const void* gate;
  const void* up;
  void* act;
} bm_layer_step_t;

int bm_layer_step(const bm_layer_step_t* step, bm_dtype_t dtype, int32_t* d_status, void* stream);

/* ---------------------------------------------------------------------------
 * RoPE table: fp32 (cos, sin) pairs laid out [max_pos][head_dim/2], entry
 * (p, i) for angle p / theta^(2i/head_dim), computed on the device in fp64
 * (the angle formula of the reference's CPU check loop,
 * tests/kernel_tests.cu:180, rounded once to fp32).
 * bm_rope_table_fill writes caller memory of max_pos*head_dim*4 bytes;
 * bm_rope_table_create allocates it (cudaMalloc) and fills it, synchronously.
 */
int bm_rope_table_fill(void* table, int32_t max_pos, int32_t head_dim,
                       double theta, void* stream);
int bm_rope_table_create(int32_t max_pos, int32_t head_dim, double theta,
                         void** table_out);
int bm_rope_table_destroy(void* table);

/* ---------------------------------------------------------------------------
 * Fused RoPE + KV-cache store for `rows` tokens.
 *   q [rows][num_q_heads][head_dim]  rotated in place;
 *   k [rows][num_kv_heads][head_dim] rotated and written to k_cache (k itself
 *                                    is not modified);
 *   v [rows][num_kv_heads][head_dim] copied to v_cache.
 * Caches are [num_seqs][num_kv_heads][max_seq][head_dim] (include/kv_cache.h:37-40).
 * Token r goes to sequence seq_ids[r] (all 0 when seq_ids is NULL) at position
 * positions[r] (pos0 + r when positions is NULL).
 * Rotation: the half-split pairing (i, i + head_dim/2) of launch_rope
 * (include/kernels.cuh:12-15, src/kernels.cu:126-140). Replaces the sequence
 * launch_rope + launch_kv_store(k) + launch_kv_store(v)
 * (src/execution_engine.cu:113-115; include/kernels.cuh:15,36).
 * rope_table from bm_rope_table_*, with table_len positions; NULL computes
 * cos/sin per pair on the device in fp64 from theta.
 */
int bm_rope_kv_store(void* q, const void* k, const void* v,
                     const int32_t* positions, int32_t pos0,
                     const int32_t* seq_ids,
                     void* k_cache, void* v_cache,
                     const void* rope_table, int32_t table_len, double theta,
                     int64_t rows, int32_t num_q_heads, int32_t num_kv_heads,
                     int32_t head_dim, int32_t max_seq, int32_t num_seqs,
                     bm_dtype_t dtype, int32_t* d_status, void* stream);

/* ---------------------------------------------------------------------------
 * RoPE in place on q [rows][num_q_heads][head_dim] and k [rows][num_kv_heads]
 * [head_dim] (either may be NULL with its head count 0). Batched launch_rope
 * (include/kernels.cuh:15, src/kernels.cu:126-148); positions/pos0,
 * rope_table/theta as in bm_rope_kv_store.
 */
int bm_rope(void* q, void* k, const int32_t* positions, int32_t pos0,
            const void* rope_table, int32_t table_len, double theta,
            int64_t rows, int32_t num_q_heads, int32_t num_kv_heads,
            int32_t head_dim, bm_dtype_t dtype, int32_t* d_status,
            void* stream);

/* ---------------------------------------------------------------------------
 * KV store: cache[seq][h][pos][:] = src[r][h][:] for `rows` tokens.
 * Batched launch_kv_store (include/kernels.cuh:36, src/kernels.cu:211-222);
 * positions/pos0 and seq_ids as in bm_rope_kv_store.
 */
int bm_kv_store(void* cache, const void* src, const int32_t* positions,
                int32_t pos0, const int32_t* seq_ids, int64_t rows,
                int32_t num_heads, int32_t head_dim, int32_t max_seq,
                int32_t num_seqs, bm_dtype_t dtype, int32_t* d_status,
                void* stream);

/* ---------------------------------------------------------------------------
 * Decode attention: one query token per entry of a batch, GQA.
 *   out[b][h][:] = softmax_j(q[b][h] . K[s][h/G][j] * scale) . V[s][h/G][j]
 * over positions j in [0, lens[b]) of cache sequence s = seq_ids[b] (0 when
 * seq_ids is NULL), G = num_q_heads / num_kv_heads (<= 16), scale <= 0 meaning
 * 1/sqrt(head_dim). q and out are [batch][num_q_heads][head_dim]; the caches are
 * [num_seqs][num_kv_heads][max_seq][head_dim] (bm_kv_cache_layer,
 * bm_rope_kv_store). lens is a device array; max_len is a host-side upper bound
 * of its entries that sizes the work split. head_dim <= 256 with whole 16-byte
 * rows. Replaces launch_attention (include/kernels.cuh:41,
 * src/kernels.cu:225-264: one token, heads = kv heads, three launches).
 * Long sequences are split across CTAs; the split results need
 * bm_decode_attention_workspace_size() bytes of device scratch, passed as
 * `workspace` (caller-owned; its contents need no initialisation). With less
 * scratch than that (or NULL) each (query, kv head) runs unsplit in one CTA:
 * same results, less parallelism. A query with an out-of-range sequence or a
 * length outside [1, max_len] (max_len <= max_seq) is skipped and flags
 * *d_status. */
int bm_decode_attention_workspace_size(int64_t batch, int32_t num_q_heads, int32_t num_kv_heads,
                                       int32_t head_dim, int32_t max_len, size_t* bytes_out);
int bm_decode_attention(void* out, const void* q, const void* k_cache, const void* v_cache,
                        const int32_t* seq_ids, const int32_t* lens, int32_t max_len, int64_t batch,
                        int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim, int32_t max_seq,
                        int32_t num_seqs, float scale, void* workspace, size_t workspace_bytes,
                        bm_dtype_t dtype, int32_t* d_status, void* stream);

/* Decode attention with the new token's RoPE and K/V store in the same launch:
 * the engine's step for one token, launch_rope + launch_kv_store twice +
 * launch_attention (src/execution_engine.cu:113-116), equivalent to
 *   bm_rope_kv_store(q, k, v, positions, 0, seq_ids, k_cache, v_cache, rope_table, ...)
 *   bm_decode_attention(out, q, k_cache, v_cache, seq_ids, lens, ...)
 * for queries whose token sits at positions[b] < lens[b] of its own sequence (no
 * two queries of one call share a sequence). k and v are [batch][num_kv_heads]
 * [head_dim]; rope_table is required (bm_rope_table_*, rope_table_len positions).
 * On the CUDA-core path (head_dims other than 128) ONE launch: the CTA that attends
 * to the new position rotates k into the K cache, copies v into the V cache and
 * every CTA rotates its queries as it stages them, with the arithmetic of
 * bm_rope_kv_store. Head_dim 128 caches, read by TMA-fed kernels, take the two
 * calls. q is consumed: afterwards it holds its input or its rotation. On the
 * one-launch path a position outside [0, lens[b]) or past the table flags
 * BM_DEVERR_BAD_POSITION and that token is neither rotated nor stored (its query
 * attends over the cache as it is); the two-call path checks positions as
 * bm_rope_kv_store does. */
int bm_rope_kv_decode_attention(void* out, void* q, const void* k, const void* v, const int32_t* positions,
                                const void* rope_table, int32_t rope_table_len, const int32_t* seq_ids,
                                void* k_cache, void* v_cache, const int32_t* lens, int32_t max_len, int64_t batch,
                                int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim, int32_t max_seq,
                                int32_t num_seqs, float scale, void* workspace, size_t workspace_bytes,
                                bm_dtype_t dtype, int32_t* d_status, void* stream);

/* Decode attention that allocates nothing, for callers that cannot call
 * cudaMalloc (a host application whose own arena owns all device memory, a
 * plugin in a process that reserved the GPU up front, a latency-critical path
 * that cannot afford cudaMalloc's implicit synchronisation). No counterpart in
 * the reference. Same arguments and results as bm_decode_attention, without the
 * workspace: the split partials live in an 8 MiB array compiled into the
 * library (one copy per GPU, held until the process exits). Arguments are
 * checked as bm_decode_attention checks them; then a batch whose split plan
 * (the one bm_decode_attention runs with a workspace of this array's size)
 * needs more than 8 MiB is rejected with BM_ERR_INVALID_ARGUMENT. The first
 * call in a CUDA context looks up that context's copy of the array (cached under
 * the context's unique id); make it before capturing any stream. All calls
 * share the array: calls that overlap on the GPU race on it and must be
 * serialised by the caller. */
int bm_decode_attention_static_scratch(void* out, const void* q, const void* k_cache, const void* v_cache,
                                       const int32_t* seq_ids, const int32_t* lens, int32_t max_len,
                                       int64_t batch, int32_t num_q_heads, int32_t num_kv_heads,
                                       int32_t head_dim, int32_t max_seq, int32_t num_seqs, float scale,
                                       bm_dtype_t dtype, int32_t* d_status, void* stream);

/* ---------------------------------------------------------------------------
 * Tensor-core GEMMs (tcgen05, bf16 operands, fp32 accumulation, bf16 output).
 * The activation is [rows][K] row-major; weights are [K][N] row-major, the
 * layout of launch_gemm's B operand (include/kernels.cuh:20, src/kernels.cu:83-121).
 * For BM_BF16: N and K multiples of 8, every pointer 16-byte aligned, any row
 * count (tcgen05). BM_F32 (any shape, no alignment needed) runs on CUDA cores in
 * fp32 (below).
 *
 * bm_gemm_swiglu: out[r][f] = silu(sum_d x[r][d] w_gate[d][f]) * sum_d x[r][d] w_up[d][f]
 * for x [rows][dim], w_gate and w_up [dim][hidden], out [rows][hidden]: the two
 * FFN input projections and the SwiGLU of src/execution_engine.cu:122-124 in one
 * kernel, the products kept in fp32 until the SwiGLU. bm_gemm: c[M][N] = a[M][K] b[K][N].
 * A pipeline wait that passes its time limit (a fault, never a slow input) sets
 * BM_DEVERR_TIMEOUT in *d_status.
 * BM_F32: fp32 arithmetic on CUDA cores, built for few rows (the reference
 * engine's one-token products, src/execution_engine.cu:81,110-125), K split over a
 * thread-block cluster and reduced in a fixed order (deterministic); d_status is
 * not used. bm_gemm_swiglu's fp32 SwiGLU is g / (1 + expf(-g)) * u, as bm_swiglu,
 * so it equals bm_gemm twice and bm_swiglu bit for bit.
 *
 * bm_gemm_shared_a: c[o] = a . b[o] for o < count (1 to 3), the products of one
 * activation with several weights (an attention block's Q, K and V projections):
 * c, b and n are host arrays of count device pointers and widths, a is [m][k],
 * b[o] [k][n[o]], c[o] [m][n[o]]. BM_F32 runs all of them in one launch; BM_BF16
 * runs bm_gemm once per product. */
int bm_gemm_swiglu(void* out, const void* x, const void* w_gate, const void* w_up, int64_t rows, int32_t dim,
                   int32_t hidden, bm_dtype_t dtype, int32_t* d_status, void* stream);
int bm_gemm(void* c, const void* a, const void* b, int64_t m, int32_t n, int32_t k, bm_dtype_t dtype,
            int32_t* d_status, void* stream);
int bm_gemm_shared_a(void* const* c, const void* a, const void* const* b, const int32_t* n, int32_t count,
                     int64_t m, int32_t k, bm_dtype_t dtype, int32_t* d_status, void* stream);

/* The RMSNorm before a projection and the projection together (the norms of
 * src/execution_engine.cu:80,109,121, after the residual adds of :118,126, each
 * followed by its products :81,110-112,122-123):
 *   x = h + d                      (d may be NULL: x = h)
 *   y = x * rsqrt(mean(x^2) + eps) * norm_weight       (as bm_rmsnorm computes it)
 *   swiglu == 0: c[o] = y . b[o] for o < count (1 to 3)   (as bm_gemm_shared_a)
 *   swiglu != 0: count 2, c[0] = silu(y . b[0]) * (y . b[1])   (as bm_gemm_swiglu)
 * h, d, residual_out and normed are [m][k]; b[o] is [k][n[o]]. residual_out
 * (may be NULL) receives x, the updated residual stream, when d is given; it must
 * not overlap h or d, which the kernel still reads while it is written.
 * BM_F32 with the normalised rows of a CTA's share of K fitting its shared memory
 * (one-token and few-token products): ONE launch, y never written to memory (its
 * sum of squares is ordered as the product kernel's threads hold the row, so y can
 * differ from bm_rmsnorm's in the last bit). Otherwise, and for BM_BF16, the norm
 * runs first into `normed` (scratch, always required), then the products. k > 0. */
int bm_rmsnorm_gemm(void* const* c, const void* h, const void* d, const void* norm_weight, float eps,
                    void* residual_out, void* normed, const void* const* b, const int32_t* n, int32_t count,
                    int32_t swiglu, int64_t m, int32_t k, bm_dtype_t dtype, int32_t* d_status, void* stream);

/* Softmax in place over num_vectors vectors of `size` elements, `stride`
 * elements apart (the gaps untouched): x = exp(x - max) / sum exp(x - max), fp32
 * arithmetic. Replaces launch_softmax(_batch) (include/kernels.cuh:23-26,
 * src/kernels.cu:150-180). */
int bm_softmax(void* x, int64_t size, int64_t num_vectors, int64_t stride, bm_dtype_t dtype, void* stream);

/* ---------------------------------------------------------------------------
 * Batch-aware static KV cache. Replaces the reference's KVCache
 * (include/kv_cache.h:10-40, src/kv_cache.cu:4-47), which allocates
 * [max_batch][kv_heads][max_seq][head_dim] fp32 per layer but keeps one
 * current_seq_pos_ for the whole cache (src/kv_cache.cu:38-47). Here every
 * sequence has its own length, and the cache stores fp32 or bf16.
 *
 * bm_kv_cache_create allocates, per layer, one K and one V buffer of
 * num_seqs * num_kv_heads * max_seq * head_dim elements (cudaMalloc, zeroed) on
 * the current device, plus two int32 device arrays of max_tokens entries for the
 * positions and sequence ids of one batch. bm_kv_cache_append takes the
 * sequence id of each of `rows` new tokens (host array), gives each token the
 * next position of its sequence (tokens of one sequence in the order given),
 * copies positions and sequence ids to the device arrays on `stream`, and
 * returns their device pointers for bm_rope_kv_store. It fails, changing
 * nothing, if a sequence would pass max_seq or rows exceeds max_tokens.
 * The host copy is synchronous with respect to the host buffer (the call
 * returns after the upload is queued from the cache's own pinned staging).
 * Every append overwrites the same two device arrays, so issue each append and
 * the bm_rope_kv_store calls that read its arrays on one stream: stream order
 * then keeps the next append's upload behind the previous step's readers. */
typedef struct bm_kv_cache bm_kv_cache_t;

int bm_kv_cache_create(int32_t num_layers, int32_t num_seqs, int32_t num_kv_heads, int32_t max_seq,
                       int32_t head_dim, int32_t max_tokens, bm_dtype_t dtype, bm_kv_cache_t** cache_out);
int bm_kv_cache_destroy(bm_kv_cache_t* cache);
/* Device pointers of layer `layer`'s K and V caches, [num_seqs][kv_heads][max_seq][head_dim]. */
int bm_kv_cache_layer(const bm_kv_cache_t* cache, int32_t layer, void** keys, void** values);
/* Current length (next position) of sequence `seq`. */
int bm_kv_cache_seq_len(const bm_kv_cache_t* cache, int32_t seq, int32_t* len_out);
/* Starts sequence `seq` over (length 0); seq = -1 resets every sequence. */
int bm_kv_cache_reset(bm_kv_cache_t* cache, int32_t seq);
int bm_kv_cache_append(bm_kv_cache_t* cache, const int32_t* seq_ids, int64_t rows,
                       const int32_t** positions_dev, const int32_t** seq_ids_dev, void* stream);

/* ---------------------------------------------------------------------------
 * Rotary positions in their other forms. No counterpart in the reference, whose
 * launch_rope (src/kernels.cu:126-140) rotates whole heads, half-split, unscaled.
 *
 * Scaled tables. A table is fp32 (cos, sin) pairs [max_pos][rotary_dim/2], the
 * layout of bm_rope_table_fill, entry (p, i) = mscale * (cos, sin)(p * f_i), angles in
 * fp64, with f_i = theta^(-2i/rotary_dim) changed by `kind`:
 *   NONE    f_i (bm_rope_table_fill's table, bit for bit, when mscale is 1)
 *   LINEAR  f_i / factor
 *   NTK     theta replaced by theta * factor^(rotary_dim / (rotary_dim - 2))
 *   BANDS   with t = original_max_pos * f_i / 2pi turns in the original context and
 *           k = clamp((t - low) / (high - low), 0, 1):  k f_i + (1 - k) f_i / factor
 *           (low, high: the low and high frequency factors, low < high)
 *   YARN    r = clamp((i - a) / max(b - a, 0.001), 0, 1):  (1 - r) f_i + r f_i / factor,
 *           a = max(floor(e(low)), 0), b = min(ceil(e(high)), rotary_dim - 1),
 *           e(n) = rotary_dim ln(original_max_pos / (2pi n)) / (2 ln theta)
 *           (low, high: beta_fast and beta_slow, low >= high > 0; theta > 1)
 * factor >= 1. mscale <= 0 means the kind's own: 0.1 ln(factor) + 1 for YARN, else 1.
 * Such a table serves every entry point that takes a rope_table, too. */
typedef enum bm_rope_scaling_kind {
  BM_ROPE_SCALING_NONE = 0,
  BM_ROPE_SCALING_LINEAR = 1,
  BM_ROPE_SCALING_NTK = 2,
  BM_ROPE_SCALING_BANDS = 3,
  BM_ROPE_SCALING_YARN = 4
} bm_rope_scaling_kind_t;

typedef struct bm_rope_scaling {
  int32_t kind; /* bm_rope_scaling_kind_t */
  int32_t original_max_pos;
  double factor, low, high, mscale;
} bm_rope_scaling_t;

/* scaling NULL: NONE. */
int bm_rotary_table_fill(void* table, int32_t max_pos, int32_t rotary_dim, double theta,
                         const bm_rope_scaling_t* scaling, void* stream);

/* Rotates the first rotary_dim elements of every head and copies the rest:
 * q_out [rows][num_q_heads][head_dim] from q, k_out [rows][num_kv_heads][head_dim]
 * from k (either pair may be NULL with its head count 0). The heads of a row are
 * dense; rows are *_stride elements apart (a slice of a fused Q/K/V projection), so
 * every stride is at least heads * head_dim. Outputs may be their inputs (same pointer
 * and stride: in place) and must not overlap them otherwise.
 * interleaved 0: pairs (i, i + rotary_dim/2), as bm_rope; 1: pairs (2i, 2i + 1).
 * positions int32[rows] or NULL (pos0 + r); the table is required. With
 * rotary_dim = head_dim and interleaved 0 the results equal bm_rope's bit for bit. A
 * position outside [0, table_len) flags BM_DEVERR_BAD_POSITION and leaves its row
 * unwritten. rotary_dim even, <= head_dim <= 1024. */
int bm_rotary(void* q_out, void* k_out, const void* q, const void* k, const int32_t* positions, int32_t pos0,
              const void* table, int32_t table_len, int32_t rotary_dim, int32_t interleaved, int64_t rows,
              int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim, int64_t q_stride, int64_t k_stride,
              int64_t q_out_stride, int64_t k_out_stride, bm_dtype_t dtype, int32_t* d_status, void* stream);

/* ---------------------------------------------------------------------------
 * Paged KV cache. No counterpart in the reference, whose cache is one static run of
 * max_seq positions (include/kv_cache.h:37-40).
 * k_pages and v_pages are [num_pages][num_kv_heads][page_size][head_dim] (the static
 * cache's layout with a page in a sequence's place); slot t of sequence s lives in page
 * page_table[s][t / page_size] at t % page_size. page_table is a device array
 * int32 [num_seqs][max_pages], read by every call: entries behind a sequence's last
 * slot are never read and may hold anything. */
typedef struct bm_paged_kv {
  void* k_pages;
  void* v_pages;
  const int32_t* page_table;
  int32_t num_pages, page_size, max_pages, num_seqs, num_kv_heads, head_dim;
} bm_paged_kv_t;

/* RoPE + K/V store into a paged cache (bm_rope_kv_store for pages), for `rows` tokens:
 *   q_out[r] = q[r] rotated (q_out may be q);
 *   slot slots[r] of sequence seq_ids[r]: K = k[r] rotated, V = v[r].
 * slots NULL: slot = positions[r]. A drafted tree's tokens share rotary positions and
 * have slots of their own. seq_ids NULL: all 0. table NULL: nothing is rotated (q_out
 * and K are copies; positions may be NULL when slots is given). q, k, v and q_out rows
 * are *_stride elements apart; num_q_heads may be 0 (q and q_out NULL). Rows whose slot is -1 are padding: nothing of
 * theirs is read or written. Bad positions (outside the table), slots (negative or
 * outside max_pages pages), sequences and page ids flag *d_status; such a row is
 * skipped. The rows of one call name distinct slots: with two rows on one slot either
 * row's values may be kept, chunk by chunk. q_out must not overlap the pages, nor k and v
 * slots that the call writes. */
int bm_paged_kv_append(void* q_out, const void* q, const void* k, const void* v, const int32_t* positions,
                       const int32_t* slots, const int32_t* seq_ids, const bm_paged_kv_t* cache, const void* table,
                       int32_t table_len, int32_t rotary_dim, int32_t interleaved, int64_t rows, int32_t num_q_heads,
                       int64_t q_stride, int64_t k_stride, int64_t v_stride, int64_t q_out_stride, bm_dtype_t dtype,
                       int32_t* d_status, void* stream);

/* Attention of a tree of drafted tokens per sequence over a paged cache (of one token:
 * decode attention; without a mask: a chunk of a prompt behind its cached beginning).
 * Sequence b (cache sequence seq_ids[b], b when NULL) has the query rows
 * [q_starts[b], q_starts[b+1]) of q and out, [total_q][num_q_heads][head_dim], and
 * n_b of them. Its context is the cache slots [0, ctx_lens[b]); its drafted tokens'
 * K and V sit in slots ctx_lens[b] + j, j < n_b (bm_paged_kv_append). Row i of it gets
 *   out[i][h] = softmax_t(q[i][h] . K[t][h/G] * scale) . V[t][h/G]
 * over the context and the drafted slots j that it sees: bit j%64 of
 * tree_mask[row][j/64] (uint64 [total_q][mask_words], bits past n_b ignored), or j <= i
 * when tree_mask is NULL. G = num_q_heads / num_kv_heads <= 64, scale <= 0 means
 * 1/sqrt(head_dim) (a scale that is not finite is refused), head_dim <= 256 with whole 16-byte rows, and
 * batch * max_tree * num_q_heads <= 2^25. q and out are dense, and out must not overlap
 * q or the pages. A row that sees nothing gets zeros. With batch, total_q or max_tree 0
 * nothing runs and nothing is flagged. Rows outside [q_starts[0], q_starts[batch]) are left as they were.
 * max_ctx and max_tree are host-side upper bounds of ctx_lens and n_b that size the
 * work split; with a mask max_tree <= 64 * mask_words. K and V of the ctx + n_b slots
 * must be finite; slots behind them may hold anything. Softmax statistics and sums are
 * fp32. bf16 caches with head_dim a multiple of 8 up to 128 run on the tensor cores, with
 * weights rounded to bf16 as bm_decode_attention does, for page sizes up to 128 that are
 * multiples of 8 or at least 64, and larger ones with an equal part of 64 to 128 slots;
 * all others run on the CUDA cores.
 * A sequence with n_b or ctx outside [0, bound], slots outside its max_pages pages or
 * rows outside [0, total_q) flags BM_DEVERR_BAD_POSITION, one with a bad sequence id
 * BM_DEVERR_BAD_SEQUENCE: it is skipped, its rows unwritten. A bad page id flags
 * BM_DEVERR_BAD_PAGE and its slots count as unseen.
 * workspace: bm_paged_tree_attention_workspace_size() bytes of device scratch (16-byte aligned),
 * contents of no matter, for calls of the same sizes; calls that overlap on the GPU
 * need their own. */
int bm_paged_tree_attention_workspace_size(int64_t total_q, int64_t batch, int32_t num_q_heads, int32_t num_kv_heads,
                                           int32_t head_dim, int32_t max_ctx, int32_t max_tree, size_t* bytes_out);
int bm_paged_tree_attention(void* out, const void* q, const bm_paged_kv_t* cache, const int32_t* seq_ids,
                            const int32_t* ctx_lens, const int32_t* q_starts, const uint64_t* tree_mask,
                            int32_t mask_words, int64_t total_q, int64_t batch, int32_t num_q_heads, int32_t max_ctx,
                            int32_t max_tree, float scale, void* workspace, size_t workspace_bytes, bm_dtype_t dtype,
                            int32_t* d_status, void* stream);

/* ---------------------------------------------------------------------------
 * RMSNorm of every head of Q and K, then rotary positions, in one pass. No counterpart in
 * the reference, whose heads are rotated as they are (src/kernels.cu:126-140). For each head
 * x of q and k, with w its norm's weight [head_dim] (of the storage type):
 *   y = x * rsqrt(mean(x^2) + eps) * w, then bm_rotary's rotation of y,
 * in fp32 throughout, rounded once. Every argument that bm_rotary has means what it means
 * there (strides, positions, outputs that may be their inputs, bad positions);
 * head_dim <= 256. A head of zeros stays one (with eps 0: NaN). */
int bm_qk_norm_rotary(void* q_out, void* k_out, const void* q, const void* k, const void* q_weight, const void* k_weight,
                      float eps, const int32_t* positions, int32_t pos0, const void* table, int32_t table_len,
                      int32_t rotary_dim, int32_t interleaved, int64_t rows, int32_t num_q_heads, int32_t num_kv_heads,
                      int32_t head_dim, int64_t q_stride, int64_t k_stride, int64_t q_out_stride, int64_t k_out_stride,
                      bm_dtype_t dtype, int32_t* d_status, void* stream);

/* ---------------------------------------------------------------------------
 * Paged KV cache held in 8 bits. bm_paged_kv_t with pages of e4m3 codes (sign, four bits of
 * exponent, three of mantissa; largest 448) and a scale for each block of `block`
 * neighbouring slots of a page (block divides page_size) and head:
 *   K[t] = k_pages[p][h][o][:] * k_scales[p][h][o / block],  p = page_table[s][t / page_size],
 *   o = t % page_size;  V alike.
 * A scale is a power of two in one byte, 2^(byte - 127) (e8m0), from 2^-40 to 2^40; a byte
 * outside these counts as the nearest. k_scales and v_scales are
 * [num_pages][num_kv_heads][page_size / block]. head_dim is a multiple of 16 up to 256, and
 * page_size * max_pages at most 2^31 - 4096. */
typedef struct bm_paged_kv8 {
  void* k_pages;
  void* v_pages;
  void* k_scales;
  void* v_scales;
  const int32_t* page_table;
  int32_t num_pages, page_size, block, max_pages, num_seqs, num_kv_heads, head_dim;
} bm_paged_kv8_t;

/* Norm, RoPE and K/V store into an 8-bit paged cache. Sequence b (cache sequence seq_ids[b],
 * b when NULL) appends the rows [q_starts[b], q_starts[b+1]) of k and v, n_b of them, as its
 * slots ctx_lens[b] + i: the arguments of bm_paged_kv8_tree_attention, which reads them.
 *   q_out[r] = q[r], K = k[r]: each head normed (q_weight, k_weight; NULL: not) and rotated
 *   (table; NULL: not) as bm_qk_norm_rotary does, at positions[r] (NULL: the row's slot);
 *   V = v[r] as it is.
 * K and V are quantised from fp32, one rounding to the nearest (even) code. The scale of a
 * block is 2^E, E = ceil(log2(a / 448)) with a its largest new magnitude, at least 2^-40 and at
 * most 2^40 (larger values end at 448 * 2^40). A block that has slots before ctx_lens[b] keeps
 * its scale where that is larger; else its earlier codes are moved to the new scale (exactly,
 * unless they fall below 2^-6). Slots behind the new ones keep their codes, which mean nothing under another
 * scale. A value that is not finite becomes NaN and sets no scale.
 * q, k, v and q_out rows are *_stride elements apart; num_q_heads may be 0 (q, q_out NULL);
 * q_out may be q and must not overlap anything else. max_tokens is a host-side upper bound of
 * n_b. Rows outside [q_starts[0], q_starts[batch]) are neither read nor written. A call names
 * no block twice: with one sequence in it twice, or one page under two of its sequences,
 * where both append, the codes and scale of the blocks they share are either one's, or mixed.
 * A sequence with n_b outside [0, max_tokens], slots outside its max_pages pages or rows
 * outside [0, rows) flags BM_DEVERR_BAD_POSITION, a bad sequence id BM_DEVERR_BAD_SEQUENCE: it
 * is skipped. A bad page id flags BM_DEVERR_BAD_PAGE: K and V of its slots are skipped. A
 * position outside the table flags BM_DEVERR_BAD_POSITION: its row is skipped. */
int bm_paged_kv8_append(void* q_out, const void* q, const void* k, const void* v, const void* q_weight,
                        const void* k_weight, float eps, const int32_t* positions, const bm_paged_kv8_t* cache,
                        const int32_t* seq_ids, const int32_t* ctx_lens, const int32_t* q_starts, const void* table,
                        int32_t table_len, int32_t rotary_dim, int32_t interleaved, int64_t rows, int64_t batch,
                        int32_t num_q_heads, int32_t max_tokens, int64_t q_stride, int64_t k_stride, int64_t v_stride,
                        int64_t q_out_stride, bm_dtype_t dtype, int32_t* d_status, void* stream);

/* Reads cached slots back: rows [starts[b], starts[b+1]) of k_out and v_out
 * [rows][num_kv_heads][head_dim] (dense, 16-byte aligned) get slots first[b] + i of sequence b
 * (seq_ids[b], b when NULL) as values of dtype: exact in fp32 and in bf16. max_rows bounds a
 * sequence's rows; other rows of the outputs are left as they were. Bad sequences are
 * skipped as bm_paged_kv8_append does, and rows whose page id is bad. */
int bm_paged_kv8_read(void* k_out, void* v_out, const bm_paged_kv8_t* cache, const int32_t* seq_ids,
                      const int32_t* first, const int32_t* starts, int64_t rows, int64_t batch, int32_t max_rows,
                      bm_dtype_t dtype, int32_t* d_status, void* stream);

/* bm_paged_tree_attention over an 8-bit paged cache: every argument and every rule as there, with
 * q and out of dtype, K and V the values that the cache stands for. Those of the ctx + n slots
 * must be finite (no NaN code). Statistics and sums are fp32. bf16 with head_dim up to 128 and
 * page sizes as there runs on the tensor cores where eight neighbouring slots of a tile of 128 share a
 * scale (blocks that are multiples of 8, in pages or equal parts of pages that are multiples of 8, or
 * a part inside one block); all others run on the CUDA cores. The tensor cores take a query
 * as an e4m3 and an e5m2 part (together its bf16 value down to 2^-13 of its head's largest, off by at most 2^-21
 * of that below) and a weight as three e5m2 parts (off by 2^-11 of itself, or by 2^-29 of the sum's largest
 * weight times V's scale). */
int bm_paged_kv8_tree_attention_workspace_size(int64_t total_q, int64_t batch, int32_t num_q_heads, int32_t num_kv_heads,
                                               int32_t head_dim, int32_t max_ctx, int32_t max_tree, size_t* bytes_out);
int bm_paged_kv8_tree_attention(void* out, const void* q, const bm_paged_kv8_t* cache, const int32_t* seq_ids,
                                const int32_t* ctx_lens, const int32_t* q_starts, const uint64_t* tree_mask,
                                int32_t mask_words, int64_t total_q, int64_t batch, int32_t num_q_heads, int32_t max_ctx,
                                int32_t max_tree, float scale, void* workspace, size_t workspace_bytes, bm_dtype_t dtype,
                                int32_t* d_status, void* stream);

/* ---------------------------------------------------------------------------
 * Sampling: one token per row of logits [rows][vocab], rows row_stride elements apart,
 * from given uniform numbers in [0, 1). The reference leaves this to its callers (an
 * argmax on the host, src/benchmark.cpp). For each row, in this order:
 *   weights w_i = exp((x_i - max x) / temperature[r])
 *   top_k[r] = k > 0: only the k largest stay
 *   top_p[r] = p < 1: in descending order, a token stays while the weights before it
 *     sum to less than p times what is left after top-k (the first always stays)
 *   min_p[r] = m > 0: w_i >= m stay (the largest always stay)
 *   token: the lowest index whose running sum of staying weights, in index order,
 *     exceeds uniforms[r] times their total.
 * Equal logits are ordered by index, the lowest first. temperature 0: the largest
 * logit's lowest index. temperature, top_k, top_p and min_p are device arrays of one
 * entry per row, or NULL (1, off, off, off); k <= 0 or >= vocab, p >= 1 and m <= 0 are
 * off, p <= 0 leaves the largest alone. A NaN logit counts as -inf; -inf has no weight;
 * with +inf logits only these have one, all alike; a logit more than FLT_MAX below the
 * largest has none. A row without any weight gets token -1. Weights are held in 64-bit
 * fixed point (2^min(51, 62 - ceil(log2 vocab)) for the largest, from fp64 exponentials)
 * and summed as integers, so a result does not depend on the order of any sum.
 * Temperatures between 0 and 2^-60 count as 2^-60. A row whose temperature, top_p, min_p or uniform number is
 * NaN, or whose temperature is negative or uniform outside [0, 1), gets -1 and flags
 * BM_DEVERR_BAD_PARAMETER. vocab <= 2^24. */
int bm_sample(int32_t* tokens, const void* logits, const float* uniforms, const float* temperature,
              const int32_t* top_k, const float* top_p, const float* min_p, int64_t rows, int64_t vocab,
              int64_t row_stride, bm_dtype_t dtype, int32_t* d_status, void* stream);

/* Self-test of the bounded waits behind BM_DEVERR_TIMEOUT (the tensor-core
 * kernels' mbarrier waits): one CTA waits on a barrier that nothing completes,
 * with a limit of limit_ns in [1 ms, 2 s]. The wait gives up, ORs
 * BM_DEVERR_TIMEOUT into *d_status and the kernel finishes; the context stays
 * usable. d_result (device, 4 x int64): [0] 1 if the wait reported success
 * (expected 0), [1] its duration in ns (about limit_ns), [2] and [3] the same for
 * a second wait that honours the first one's abort (gives up at once). */
int bm_selftest_bounded_wait(int64_t limit_ns, int32_t* d_status, int64_t* d_result, void* stream);

#ifdef __cplusplus
} /* extern "C" */
#endif

#endif /* BM_LAYER_OPS_H */
