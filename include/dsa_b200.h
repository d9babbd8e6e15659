/* C ABI of libdsa_b200.so: the sm_100a kernels of the DeepSeek Sparse Attention
 * (DSA) hot path -- lightning-indexer logits, per-row top-k selection and sparse
 * MLA -- behind plain pointers and sizes.
 *
 * The reference project (sparse_attn/DSA.py) has no native ABI: it reaches its
 * GPU kernels through late-bound Python imports.  Each entry point below names
 * the reference call site it stands in for.
 *
 * Conventions
 *   - Every pointer is a DEVICE pointer unless its comment says "host".
 *   - The caller owns all buffers (inputs, outputs, workspace, status word); the
 *     library allocates nothing and keeps no pointer after the call returns.
 *   - Calls are asynchronous on `stream` (a cudaStream_t passed as void*; NULL =
 *     the default stream) and never synchronise.
 *   - Return value: 0 on success, a negative DSA_ERR_* code otherwise; nothing is
 *     launched on error and dsa_last_error_string() describes it.
 *   - `status` (may be NULL) is one int32 in device memory, zeroed by the caller.
 *     Kernels write a non-zero code there instead of faulting: 1 = an internal
 *     bounded wait expired, 2 = an index or page id was out of range (the access
 *     was skipped), 3 = too few free pages (the call changed nothing).  Read it after synchronising when you want to check.
 */
#ifndef DSA_B200_H_
#define DSA_B200_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define DSA_OK 0
#define DSA_ERR_SHAPE (-1)     /* unsupported or inconsistent sizes */
#define DSA_ERR_ALIGN (-2)     /* pointer or stride alignment */
#define DSA_ERR_WORKSPACE (-3) /* workspace missing or too small */
#define DSA_ERR_CUDA (-4)      /* a CUDA runtime / driver call failed */
#define DSA_ERR_ARG (-5)       /* NULL pointer or bad flag */

#define DSA_W_F32 0
#define DSA_W_BF16 1
#define DSA_X_F32 0
#define DSA_X_BF16 1

/* Library version (major*10000 + minor*100 + patch). */
int dsa_version(void);
/* Message of the most recent error on the calling thread ("" if none). */
const char* dsa_last_error_string(void);

/* Per-block FP8 quantiser, one kernel.  Stands in for fp8_quant_per_block
 * (sparse_attn/DSA.py:102-132): for every block of block_size (64 or 128)
 * consecutive values, scale = max(absmax, 1e-6) / 448 (fp32) and
 * q = round_to_e4m3(x / scale).  x is fp32 (DSA_X_F32) or bf16 (DSA_X_BF16),
 * n_blocks * block_size values, 16-byte aligned; q_fp8 gets one byte per value,
 * scale one fp32 per block.  Bytes and scales equal the reference's CPU result. */
int dsa_fp8_quant_per_block(const void* x, int x_dtype, int64_t n_blocks, int block_size, void* q_fp8, float* scale,
                            void* stream);

/* Write side of the paged FP8 latent cache, one kernel: rows kv [n_tokens, 576] (fp32 DSA_X_F32 or bf16 DSA_X_BF16,
 * row_stride values apart, every row 16-byte aligned) -> records [n_tokens, 656] bytes (16-byte aligned, dense): the 512
 * latent values as e4m3, their four fp32 scales (one per 128 values, quantised as above), the 64 rope values as bf16. */
int dsa_pack_latent_cache(const void* kv, int kv_dtype, int64_t row_stride, int64_t n_tokens, void* records, void* stream);

/* RoPE + per-row FP8 quantiser in one pass: stands in for DsaIndexer.rope followed by fp8_quant_per_block
 * (sparse_attn/DSA.py:513-524, 530-531).  x_bf16 [n_rows, head_dim] (head_dim 64 or 128 = one FP8 block per
 * row); row r is at position r / rows_per_pos (heads per token for q, 1 for k); cos_table / sin_table
 * [n_pos, rope_dim / 2] fp32 as built by the reference's _rope_cossin (DSA.py:430-441).  The first rope_dim values
 * of a row are rotated -- halves form (interleave = 0: fp32 products, not rounded, DSA.py:444-454) or even/odd
 * pairs (interleave = 1: rounded to bf16, DSA.py:457-469) -- with the reference's operation order, then the row is
 * quantised: bytes and scales equal the eager chain's. */
int dsa_rope_fp8_quant(const void* x_bf16, int64_t n_rows, int head_dim, int rope_dim, int interleave, int rows_per_pos,
                       const float* cos_table, const float* sin_table, int64_t n_pos, void* q_fp8, float* scale,
                       void* stream);

/* The same, and with gate_bf16 [n_rows] the scorer's weights of the rows as well: gate_out[r] =
 * ((float(gate[r]) * gate_mul0) * scale[r]) * gate_mul1 in fp32, every product rounded (sparse_attn/DSA.py:327-331, 505-511). */
int dsa_rope_fp8_quant_gated(const void* x_bf16, int64_t n_rows, int head_dim, int rope_dim, int interleave, int rows_per_pos,
                             const float* cos_table, const float* sin_table, int64_t n_pos, void* q_fp8, float* scale,
                             const void* gate_bf16, float gate_mul0, float gate_mul1, float* gate_out, void* stream);

/* Lightning-indexer logits, contiguous keys.
 *   logits[t, s] = k_scale[s] * sum_h w[t,h] * relu(q[t,h,:] . k[s,:])  for ks[t] <= s < ke[t].
 * Stands in for deep_gemm.fp8_mqa_logits(q_fp8, (k_fp8, k_scale), w, ks, ke) as
 * called at sparse_attn/DSA.py:343-345, 547-552, 654-659.
 *   q_fp8   [T, H, D] e4m3, contiguous, 16-byte aligned
 *   k_fp8   [S, D]    e4m3, contiguous, 16-byte aligned
 *   k_scale [S] fp32;  w [T, H] fp32 (DSA_W_F32) or bf16 (DSA_W_BF16), q scale folded in
 *   ks, ke  [T] int32 (ks may be NULL = 0)
 *   logits  [T, ld_logits] fp32, ld_logits >= S
 * Supported: H in {4,8,16,32,64} with D = 128, and H in {4,64} with D = 64.
 * clean != 0 also writes -inf to every column outside the window (the library
 * call's default); clean == 0 leaves columns that lie in fully masked 128-key
 * tiles untouched, which is all dsa_topk_select needs. */
int dsa_indexer_logits(const void* q_fp8, const void* k_fp8, const float* k_scale, const void* w, int w_dtype,
                       const int32_t* ks, const int32_t* ke, float* logits, int64_t ld_logits, int T, int S,
                       int H, int D, int clean, int32_t* status, void* stream);

/* Lightning-indexer logits for decode over a paged FP8 key cache: one query
 * token per sequence.  No counterpart call in the reference (it has no cache,
 * sparse_attn/DSA.py:475-477); same arithmetic as dsa_indexer_logits with
 * ks = 0, ke = ctx_len[b] and key s of sequence b stored at physical row
 * block_table[b, s/64]*64 + s%64.
 *   q_fp8 [B, H, 128] e4m3; w [B, H]; kcache [num_pages*64, 128] e4m3;
 *   kscale [num_pages*64] fp32; block_table [B, table_stride] int32;
 *   ctx_len [B] int32; logits [B, ld_logits] fp32, ld_logits >= max_ctx.
 * Columns >= ctx_len[b] inside a processed tile get -inf; beyond are untouched. */
int dsa_indexer_logits_paged(const void* q_fp8, const void* w, int w_dtype, const void* kcache,
                             const float* kscale, const int32_t* block_table, int64_t table_stride,
                             const int32_t* ctx_len, float* logits, int64_t ld_logits, int B, int H, int D,
                             int num_pages, int max_ctx, int32_t* status, void* stream);

/* Per-row top-k by radix select.  Stands in for logits.topk(k).indices at
 * sparse_attn/DSA.py:361, 567, 675-676.  Row t considers columns
 * [ks[t], min(ke[t], S)) only (ks NULL = 0, ke NULL = S) and writes k int32
 * column indices to out_idx[t, 0:k]: the indices of the k largest values,
 * unsorted, ties at the k-th value going to the lower column; when fewer than k
 * columns are in the window all of them are written followed by -1 padding.
 * Output is bit-identical from run to run. */
int dsa_topk_select(const float* logits, int64_t ld_logits, const int32_t* ks, const int32_t* ke, int T, int S,
                    int k, int32_t* out_idx, void* stream);

/* Indexer logits + top-k in one call (the whole of IndexerSimulator.logits_step,
 * sparse_attn/DSA.py:336-362).  `workspace` holds the fp32 logits of one chunk
 * of query rows; dsa_indexer_topk_workspace_bytes gives the size that does the
 * whole call in one chunk, smaller workspaces (>= one 256-row chunk) make it
 * loop. */
size_t dsa_indexer_topk_workspace_bytes(int T, int S);
int dsa_indexer_topk(const void* q_fp8, const void* k_fp8, const float* k_scale, const void* w, int w_dtype,
                     const int32_t* ks, const int32_t* ke, int T, int S, int H, int D, int k, int32_t* out_idx,
                     void* workspace, size_t workspace_bytes, int32_t* status, void* stream);

/* Token-sparse MLA attention, prefill (MQA over the shared latent KV):
 *   out[t,h,:] = sum_j softmax_j(scale * q[t,h,:576] . kv[idx[t,j],:576]) * kv[idx[t,j],:512]
 * over the slots with idx[t,j] >= 0; a row without any valid slot gives zeros.
 * Takes the place of the block-sparse attention stand-in reached through
 * register_sparse_fa().run (sparse_attn/DSA.py:208-249); the reference has no
 * sparse-MLA kernel of its own.
 *   q_bf16 [T, H, 576] bf16; kv_bf16 [S_kv, 576] bf16; idx [T, K] int32 positions
 *   into kv (negative = empty; >= S_kv is skipped and sets status 2);
 *   out_bf16 [T, H, 512] bf16.  All contiguous and 16-byte aligned.  K <= 2048; scale > 0.  Any H >= 1
 *   (up to 16 and up to 32 heads have kernels of their own, more are processed in groups of 128). */
int dsa_sparse_mla_prefill(const void* q_bf16, const void* kv_bf16, const int32_t* idx, void* out_bf16, int T, int H,
                           int S_kv, int K, float scale, int32_t* status, void* stream);

/* Block-sparse multi-head attention, the call behind register_sparse_fa().run
 * (sparse_attn/DSA.py:232-247: triton_block_sparse_attn_fwd_openai_prefetch(q, k, v, idx, num,
 * sm_scale) -> (out, _), whose source is not part of the reference).  Non-causal; 64-token blocks:
 *   out[b,s,h,:] = softmax_j(scale * q[b,s,h,:] . k[b,j,h,:]) v[b,j,h,:],  j over the key blocks
 *   lut[b,h,s/64,0..num[b,h,s/64]) of query block s/64.
 *   q, k, v, out [B, S, H, 128] bf16, contiguous, 16-byte aligned; S a multiple of 64;
 *   lut [B, H, S/64, topk] int32 key-block ids (an id outside [0, S/64) contributes nothing and
 *   sets status 2); num [B, H, S/64] int32, clamped to [0, topk]; scale > 0. */
int dsa_block_sparse_mha(const void* q_bf16, const void* k_bf16, const void* v_bf16, const int32_t* lut,
                         const int32_t* num, void* out_bf16, int B, int S, int H, int D, int topk, float scale,
                         int32_t* status, void* stream);

/* The same attention for decode over the paged FP8 latent cache (no counterpart
 * in the reference, which has no cache: sparse_attn/DSA.py:475-477).  One query
 * token per sequence; idx[b, j] is a logical position of sequence b, stored at
 * cache row block_table[b, pos/64]*64 + pos%64.  A cache row is 656 bytes:
 * 512 e4m3 latent values, 4 fp32 scales (one per 128 values), 64 bf16 rope
 * values; latent = e4m3 * scale is rounded to bf16 before the tensor-core math.
 *   q_bf16 [B, H, 576]; cache [num_pages*64, 656] bytes; block_table
 *   [B, table_stride] int32; idx [B, K] int32 (K <= 2048); out_bf16 [B, H, 512].
 * Sequences run in rounds of one per pair of SMs (per group of 128 heads).  The
 * slot lists of a partly filled last round -- every sequence of a small batch, the
 * last B mod pairs of a larger one -- are cut into up to eight parts that run on
 * different SMs and are merged by a second kernel in fp32, so that a row's last
 * bits depend on the batch it is computed in.  The parts need `workspace` (16-byte
 * aligned): dsa_sparse_mla_decode_workspace_bytes(B, H, K) bytes are enough for
 * every batch of up to B sequences.  A smaller workspace holds fewer parts; with
 * NULL, or less than two parts a sequence, the call works with one. */
size_t dsa_sparse_mla_decode_workspace_bytes(int B, int H, int K);
int dsa_sparse_mla_decode_paged(const void* q_bf16, const void* cache, const int32_t* block_table,
                                int64_t table_stride, const int32_t* idx, void* out_bf16, int B, int H, int K,
                                int num_pages, int max_ctx, float scale, void* workspace, size_t workspace_bytes,
                                int32_t* status, void* stream);

/* One decode step: dsa_indexer_logits_paged, dsa_topk_select over [0, ctx_len) and dsa_sparse_mla_decode_paged with the arguments
 * of those calls, for hosts whose calls cost as much as the kernels.  The caches may have different numbers of pages. */
int dsa_decode_step(const void* q_fp8, const void* w, int w_dtype, const void* kcache, const float* kscale, int k_pages,
                    const int32_t* block_table, int64_t table_stride, const int32_t* ctx_len, float* logits, int64_t ld_logits,
                    int B, int idx_heads, int idx_dim, int max_ctx, int k, int32_t* idx, const void* q_bf16, const void* latent,
                    int latent_pages, void* out_bf16, int H, float scale, void* workspace, size_t workspace_bytes,
                    int32_t* status, void* stream);

/* ---- the paged latent cache in 4 bits -------------------------------------------
 * No counterpart in the reference (it has no cache, sparse_attn/DSA.py:475-477).
 * A record is 416 bytes a token, two halves of 208.  Half c holds latent values
 * 256c .. 256c+255 and rope values 32c .. 32c+31:
 *   128 bytes  codes, eight values to a little-endian 32-bit word
 *    16 bytes  scales of the sixteen groups of 16 values
 *    64 bytes  rope values, bf16
 * A scale byte (e << 3) + m, e = 0..30, stands for (8 + m) * 2^(e - 18); 255 is a NaN.
 * A code is a sign and the number of one of 0, .5, 1, 1.5, 2, 3, 4, 6.  Of a word's
 * values the even ones are in the low 16 bits, the odd ones in the high 16; value k
 * of a half has its sign and the bits of its number, highest first, at
 *   k=0: 15, 8 7 6    k=1: 12, 5 4 3    k=2: 9, 2 1 0    k=3: 14, 11 10 13.
 * value = code * scale (exact in bf16).  Quantising: scale = (largest magnitude of
 * the group) / 6, held to [2^-15, 61440] and rounded to nearest even; code = value /
 * scale to nearest, ties to the even number, saturating.  A group with an infinity
 * or a NaN gets the scale 255 and reads as NaN. */

/* Write side: rows kv [n_tokens, 576] (as for dsa_pack_latent_cache) -> records at the
 * rows slots[i] of cache [cache_rows, 416] (slots may be NULL: row i).  A negative
 * slot is skipped, one >= cache_rows is skipped and sets status 2; the slots of a
 * call must differ.  With k_fp8 (NULL: none) the tokens' indexer keys go to the same
 * rows of the paged key cache: k_fp8 [n_tokens, 128] e4m3 -> kcache [cache_rows, 128],
 * k_scale [n_tokens] -> kscale [cache_rows]. */
int dsa_pack_latent4(const void* kv, int kv_dtype, int64_t row_stride, int64_t n_tokens, void* cache, int64_t cache_rows,
                     const int32_t* slots, const void* k_fp8, const float* k_scale, void* kcache, float* kscale,
                     int32_t* status, void* stream);
/* Read side: positions 0 .. n_tokens-1 of one sequence -> rows out_bf16 [n_tokens, 576], row_stride values apart (a
 * multiple of 8).  Position p is the record block_table[p/64]*64 + p%64 (block_table may be NULL: record p); a page that
 * is out of range gives rows of zeros and sets status 2. */
int dsa_unpack_latent4(const void* cache, int64_t cache_rows, const int32_t* block_table, int64_t n_tokens, void* out_bf16,
                       int64_t row_stride, int32_t* status, void* stream);

/* dsa_sparse_mla_decode_paged over records of record_bytes = 656 (FP8) or 416 (4 bits), for tokens_per_seq query rows of
 * each sequence: rows r = b*tokens_per_seq .. of q [T, H, 576], idx [T, K] and out [T, H, 512] go by row b of block_table.
 * T and tokens_per_seq may be as large as the tensors.  The kernels that work in pairs of SMs -- FP8 records, more than 32
 * heads, or calls of few rows -- exchange the two halves of a score q.k (256 latent and 32 rope values each) in fp16: a half
 * beyond 65504, before the softmax scale, saturates, and the two halves of an output row disagree.  (4-bit values reach 368640.
 * |q| of the latent part must stay below 2^113 there.)  Lists may be cut into parts that different SMs take and a second
 * kernel merges in fp32; the parts' `workspace` (16-byte aligned) of dsa_sparse_mla_decode_records_workspace_bytes bytes is
 * enough for every call of up to T rows.  With a smaller one, or NULL, the call works with fewer parts or none. */
size_t dsa_sparse_mla_decode_records_workspace_bytes(int record_bytes, int T, int H, int K);
int dsa_sparse_mla_decode_records(const void* q_bf16, const void* cache, int record_bytes, const int32_t* block_table,
                                  int64_t table_stride, int tokens_per_seq, const int32_t* idx, void* out_bf16, int T, int H,
                                  int K, int num_pages, int max_ctx, float scale, void* workspace, size_t workspace_bytes,
                                  int32_t* status, void* stream);
/* dsa_decode_step with such records. */
int dsa_decode_step_records(const void* q_fp8, const void* w, int w_dtype, const void* kcache, const float* kscale, int k_pages,
                            const int32_t* block_table, int64_t table_stride, const int32_t* ctx_len, float* logits,
                            int64_t ld_logits, int B, int idx_heads, int idx_dim, int max_ctx, int k, int32_t* idx,
                            const void* q_bf16, const void* latent, int record_bytes, int latent_pages, void* out_bf16, int H,
                            float scale, void* workspace, size_t workspace_bytes, int32_t* status, void* stream);

/* ---- pages of the paged caches ----------------------------------------------------
 * No counterpart in the reference.  The state is the caller's, in device memory:
 *   refs [num_pages] int32       how many sequences hold the page, 0 = free
 *   block_table [B, table_stride] int32, P entries used: the pages of a sequence in
 *                                order, -1 behind the last one
 *   ctx_len [B] int32            its tokens (64 to a page); 0 = an empty row
 * Pages are taken lowest free id first, in the order of the call's list: the ids
 * depend on the state alone.  A call that takes pages is all or nothing: with a bad
 * argument, a partly filled last page that it copies or fills and that is no page of the
 * pool (status 2), or too few free pages (status 3) it changes nothing.  Entries of full
 * pages are believed: a fork copies one that is no page as it stands and sets status 2.
 * B <= 262144.  `workspace` (4-byte aligned): dsa_pages_workspace_bytes(num_pages, n). */

/* A cache whose pages are copied (host struct): `layers` times [num_pages*64, token_bytes] bytes, layer_stride bytes
 * apart; every layer 16-byte aligned, token_bytes a multiple of 4. */
typedef struct {
  void* base;
  int64_t layer_stride;
  int32_t layers;
  int32_t token_bytes;
} dsa_page_cache;

size_t dsa_pages_workspace_bytes(int num_pages, int n);
/* Page src[i] -> page dst[i], i < n, in every layer of every cache (`caches`: host array); with tokens [n], the first
 * tokens[i] of its 64 tokens (held to 0..64).  Entries with a negative id are skipped, ids >= num_pages are skipped and set
 * status 2.  No page may be written twice, nor be written and read. */
int dsa_copy_pages(const dsa_page_cache* caches, int n_caches, int num_pages, const int32_t* src, const int32_t* dst,
                   const int32_t* tokens, int n, int32_t* status, void* stream);
/* Room for n_new[i] more tokens (0..max_new) in row rows[i], rows all different: pages are taken, ctx_len grows, and
 * slots [n, max_new] gets the cache rows of the new tokens, -1 behind them (refused: -1 everywhere).  B * P < 2^31. */
int dsa_extend_pages(int32_t* block_table, int64_t table_stride, int P, int B, int32_t* ctx_len, int32_t* refs, int num_pages,
                     const int32_t* rows, const int32_t* n_new, int n, int max_new, int32_t* slots, void* workspace,
                     size_t workspace_bytes, int32_t* status, void* stream);
/* Row children[i] (empty, all different, no parent of the call) becomes a copy of row parents[i]: its full pages are
 * shared, a partly filled last one is copied to a page of the child's own, in every layer of every cache. */
int dsa_fork_pages(int32_t* block_table, int64_t table_stride, int P, int B, int32_t* ctx_len, int32_t* refs, int num_pages,
                   const int32_t* parents, const int32_t* children, int n, const dsa_page_cache* caches, int n_caches,
                   void* workspace, size_t workspace_bytes, int32_t* status, void* stream);
/* Rows rows[i] become empty and give their pages back (one that is named twice does so once; one that is out of range
 * is skipped and sets status 2, and so does a page that was free already). */
int dsa_free_pages(int32_t* block_table, int64_t table_stride, int P, int B, int32_t* ctx_len, int32_t* refs, int num_pages,
                   const int32_t* rows, int n, int32_t* status, void* stream);
/* The L pages in use move to ids 0 .. L-1: the i-th lowest free page below L takes the contents of the i-th highest page
 * in use, in every layer of every cache.  new_table [B, new_stride] and new_refs are the tables that go with it (they may be
 * block_table and refs).  The pages moved from are not written: the old table reads right until one of them is taken. */
int dsa_compact_pages(const int32_t* block_table, int64_t table_stride, int32_t* new_table, int64_t new_stride, int P, int B,
                      const int32_t* refs, int32_t* new_refs, int num_pages, const dsa_page_cache* caches, int n_caches,
                      void* workspace, size_t workspace_bytes, int32_t* status, void* stream);

/* dsa_indexer_topk without a caller-supplied workspace.  No counterpart in the
 * reference: it exists for hosts that cannot allocate device memory at the call
 * site (a runtime that owns the whole device heap and forbids allocation inside
 * its operator callbacks, a serving loop whose pool is frozen once it starts).
 * Same inputs, outputs and results as dsa_indexer_topk; the fp32 logits scratch
 * is a 64 MiB array built into the library, which every GPU that loads the
 * library keeps until the process exits.  Limits and rules:
 *   - min(T, 256) * round_up(S, 4) * 4 bytes must fit in 64 MiB (S <= 65536 when
 *     T >= 256); larger problems are refused with DSA_ERR_WORKSPACE.
 *   - The first call on each device looks up the array's device address, and
 *     that lookup is when the driver materialises the 64 MiB on that device (CUDA
 *     loads modules lazily): it can fail with DSA_ERR_CUDA "out of memory" on a
 *     GPU that is already full.  Make one warm-up call with T = 0 per device at
 *     start-up -- before the host freezes its pool and outside any stream
 *     capture; it launches nothing.
 *   - All calls on one device share the array, which keeps whatever the last
 *     call left there (every call overwrites what it reads).  Two calls whose
 *     kernels overlap on the GPU (different streams) race: serialise them.
 *   - It calls no cudaMalloc / cudaFree and no allocating library routine; after
 *     the warm-up call no device memory changes hands at all. */
size_t dsa_indexer_topk_static_max_bytes(void);
int dsa_indexer_topk_static(const void* q_fp8, const void* k_fp8, const float* k_scale, const void* w, int w_dtype,
                            const int32_t* ks, const int32_t* ke, int T, int S, int H, int D, int k,
                            int32_t* out_idx, int32_t* status, void* stream);

/* ---- test hooks ---------------------------------------------------------------
 * No counterpart in the reference.  They exist so that the parity tests can reach,
 * through this ABI, code paths that the normal entry points choose by themselves.
 *
 * dsa_test_indexer_logits_general: dsa_indexer_logits with 64 heads x 128 kept on
 *   the general kernel (the normal call takes the register-weight kernel for that
 *   shape); the two must agree bit for bit.
 * dsa_test_topk_select_two_pass: dsa_topk_select with every row on the two-pass
 *   radix path (the normal call takes the sampled single pass for long rows and
 *   falls back to this path when the sample misleads it); same sets, same order.
 * dsa_test_bounded_wait: launches one thread that waits, with the wait helper all
 *   pipeline roles use, on a barrier nobody arrives at; after poll_limit
 *   (1..65536) polls it must give up and write status 1 to *status.
 * dsa_test_few_heads_plan: how the 4-bit attention of few heads divides T lists of K
 *   slots among `sms` CTAs (parts != 0: lists may be cut), on the host, launch by
 *   launch: adds to seen[T][blocks of a list] (host bytes; a block is 64 slots, a list
 *   has at least one) how often a CTA has the block, and returns the most pieces of
 *   lists that a CTA has in a launch (at most 1024), or a negative error. */
int dsa_test_indexer_logits_general(const void* q_fp8, const void* k_fp8, const float* k_scale, const void* w,
                                    int w_dtype, const int32_t* ks, const int32_t* ke, float* logits,
                                    int64_t ld_logits, int T, int S, int H, int D, int clean, int32_t* status,
                                    void* stream);
int dsa_test_topk_select_two_pass(const float* logits, int64_t ld_logits, const int32_t* ks, const int32_t* ke, int T,
                                  int S, int k, int32_t* out_idx, void* stream);
int dsa_test_bounded_wait(int poll_limit, int32_t* status, void* stream);
int dsa_test_few_heads_plan(int T, int K, int sms, int parts, uint8_t* seen);

#ifdef __cplusplus
}
#endif
#endif /* DSA_B200_H_ */
