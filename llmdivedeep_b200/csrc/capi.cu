// extern "C" surface of libdsa_b200.so (declared in include/dsa_b200.h): argument
// checks, error strings and the calls into the kernel launchers.
#include <stdarg.h>
#include <stdio.h>
#include <string.h>

#include "dsa_host.h"

namespace dsa {

struct IndexerArgs;   // defined with the kernel

static thread_local char g_err[512] = "";

int set_error(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
  return code;
}

int check_launch(const char* what) {
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_error(DSA_ERR_CUDA, "%s: launch failed: %s", what, cudaGetErrorString(e));
  return DSA_OK;
}

int sm_count() {
  static int cached[64] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  if (!cached[dev]) {
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) n = 148;
    cached[dev] = n;
  }
  return cached[dev];
}

bool allow_smem(const void* kern, int bytes, uint64_t* done) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return false;
  const uint64_t bit = dev >= 0 && dev < 64 ? 1ull << dev : 0;
  if (__atomic_load_n(done, __ATOMIC_RELAXED) & bit) return true;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return false;
  __atomic_fetch_or(done, bit, __ATOMIC_RELAXED);
  return true;
}

// launchers implemented next to their kernels
int indexer_logits_contiguous(const void* q, const void* k, const float* k_scale, const void* w, int w_dtype,
                              const int32_t* ks, const int32_t* ke, float* logits, int64_t ld, int T, int S,
                              int H, int D, int clean, int general, int32_t* status, cudaStream_t stream);
int indexer_logits_paged(const void* q, const void* w, int w_dtype, const void* kcache, const float* kscale,
                         const int32_t* block_table, int64_t table_stride, const int32_t* ctx_len, float* logits,
                         int64_t ld, int B, int H, int D, int num_pages, int max_ctx, int32_t* status,
                         cudaStream_t stream);
int topk_select_launch(const float* logits, int64_t ld, const int32_t* ks, const int32_t* ke, int T, int S, int k,
                       int32_t* out, int sample, int overlapped, cudaStream_t stream);
int bounded_wait_probe_launch(uint32_t poll_limit, int32_t* status, cudaStream_t stream);

int sparse_mla_prefill_launch(const void* q, const void* kv, const int32_t* idx, void* out, int T, int H, int S_kv,
                              int K, float scale, int32_t* status, cudaStream_t stream);
int sparse_mla_decode_launch(const void* q, const void* cache, int record_bytes, const int32_t* block_table, int64_t table_stride,
                             int tokens_per_seq, const int32_t* idx, void* out, int B, int H, int K, int num_pages, int max_ctx,
                             float scale, void* workspace, size_t workspace_bytes, int32_t* status, int overlapped,
                             cudaStream_t stream);
size_t mla_decode_workspace_bytes(int B, int H, int K);
size_t mla_decode_records_workspace_bytes(int record_bytes, int T, int H, int K);
int few4_plan_probe(int T, int K, int sms, int parts, uint8_t* seen);
int block_sparse_mha_launch(const void* q, const void* k, const void* v, const int32_t* lut, const int32_t* num,
                            void* out, int B, int S, int H, int topk, float scale, int32_t* status,
                            cudaStream_t stream);

int fp8_quant_launch(const void* x, int x_is_bf16, int64_t n_blocks, int block, void* q, float* scale,
                     cudaStream_t stream);
int pack_latent4_launch(const void* kv, int kv_is_bf16, int64_t row_stride, int64_t n, void* cache, const int32_t* slots, int64_t cache_rows, const void* k8,
                        const float* k_scale, void* kcache, float* kscale, int32_t* status, cudaStream_t stream);
int unpack_latent4_launch(const void* cache, int64_t cache_rows, const int32_t* table, int64_t n, void* out, int64_t out_stride, int32_t* status,
                          cudaStream_t stream);
int copy_pages_launch(const dsa_page_cache* caches, int n_caches, int num_pages, const int32_t* src, const int32_t* dst, const int32_t* tokens, int n,
                      int32_t* status, cudaStream_t stream);
int extend_pages_launch(int32_t* table, int64_t stride, int P, int B, int32_t* ctx, int32_t* refs, int num_pages, const int32_t* rows, const int32_t* n_new, int n,
                        int max_new, int32_t* slots, int32_t* workspace, int32_t* status, cudaStream_t stream);
int fork_pages_launch(int32_t* table, int64_t stride, int P, int B, int32_t* ctx, int32_t* refs, int num_pages, const int32_t* parents, const int32_t* children,
                      int n, const dsa_page_cache* caches, int n_caches, int32_t* workspace, int32_t* status, cudaStream_t stream);
int free_pages_launch(int32_t* table, int64_t stride, int P, int B, int32_t* ctx, int32_t* refs, int num_pages, const int32_t* rows, int n, int32_t* status,
                      cudaStream_t stream);
int compact_pages_launch(const int32_t* table, int64_t stride, int32_t* new_table, int64_t new_stride, int P, int B, const int32_t* refs, int32_t* new_refs,
                         int num_pages, const dsa_page_cache* caches, int n_caches, int32_t* workspace, int32_t* status, cudaStream_t stream);
size_t pages_workspace_bytes(int num_pages, int n);
int accept_drafts_launch(int32_t* table, int64_t stride, int P, int B, int32_t* ctx, int32_t* refs, int num_pages, const int32_t* rows, const int32_t* n_new,
                         const int32_t* path, int path_stride, const int32_t* n_keep, int n, const dsa_page_cache* caches, int n_caches, int32_t* workspace,
                         int32_t* status, cudaStream_t stream);
int indexer_logits_drafts_launch(const void* q, const void* w, int w_is_bf16, const void* kcache, const float* kscale, const int32_t* block_table,
                                 int64_t table_stride, const int32_t* ctx_len, const int32_t* n_new, const int64_t* tree, int tokens_per_seq, float* logits,
                                 int64_t ld, int B, int H, int num_pages, int max_ctx, int32_t* status, cudaStream_t stream);
int topk_select_drafts_launch(const float* logits, int64_t ld, const int32_t* ctx_len, const int32_t* n_new, const int64_t* tree, int tokens_per_seq, int B,
                              int max_ctx, int k, int32_t* out, int32_t* ends, cudaStream_t stream);
int window_mla_prefill_launch(const void* q, const void* kv, const int32_t* ks, const int32_t* ke, void* out, int T, int H, int S, int window, int first,
                              float scale, void* workspace, size_t workspace_bytes, int32_t* status, cudaStream_t stream);
size_t window_mla_prefill_workspace(int T, int H, int window, int first);
size_t window_mla_decode_workspace(int record_bytes, int B, int tokens_per_seq, int H, int window, int first, int max_ctx);
int window_mla_decode_launch(const void* q, const void* cache, int record_bytes, const int32_t* block_table, int64_t table_stride, const int32_t* ctx_len,
                             const int32_t* n_new, const int64_t* tree, int tokens_per_seq, void* out, int B, int H, int window, int first, int num_pages,
                             int max_ctx, float scale, void* workspace, size_t workspace_bytes, int32_t* status, cudaStream_t stream);
int pack_latent_launch(const void* kv, int kv_is_bf16, int64_t row_stride, int64_t n, void* rec, cudaStream_t stream);
int rope_fp8_quant_launch(const void* x, int64_t n_rows, int head_dim, int rope_dim, int interleave, int rows_per_pos,
                          const float* cos_t, const float* sin_t, void* q, float* scale, const void* gate, float mul0,
                          float mul1, float* gate_out, cudaStream_t stream);

static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace dsa

using namespace dsa;

static int indexer_logits_checked(const void* q_fp8, const void* k_fp8, const float* k_scale, const void* w, int w_dtype,
                                  const int32_t* ks, const int32_t* ke, float* logits, int64_t ld_logits, int T, int S,
                                  int H, int D, int clean, int general, int32_t* status, void* stream) {
  g_err[0] = 0;
  if (T < 0 || S < 0) return set_error(DSA_ERR_SHAPE, "indexer_logits: negative size (T=%d, S=%d)", T, S);
  if (T == 0 || S == 0) return DSA_OK;
  if (!q_fp8 || !k_fp8 || !k_scale || !w || !ke || !logits)
    return set_error(DSA_ERR_ARG, "indexer_logits: NULL pointer argument");
  if (w_dtype != DSA_W_F32 && w_dtype != DSA_W_BF16)
    return set_error(DSA_ERR_ARG, "indexer_logits: w_dtype must be DSA_W_F32 or DSA_W_BF16");
  if (ld_logits < S) return set_error(DSA_ERR_SHAPE, "indexer_logits: ld_logits (%lld) < S (%d)", (long long)ld_logits, S);
  if (!aligned16(q_fp8) || !aligned16(k_fp8))
    return set_error(DSA_ERR_ALIGN, "indexer_logits: q_fp8 and k_fp8 must be 16-byte aligned");
  if ((int64_t)T * H > 0x7fffffffLL) return set_error(DSA_ERR_SHAPE, "indexer_logits: T*H exceeds 2^31");
  if (ld_logits * 64 > 0x7fffffffLL)
    return set_error(DSA_ERR_SHAPE, "indexer_logits: ld_logits (%lld) too large (64 * ld must stay below 2^31)",
                     (long long)ld_logits);
  return indexer_logits_contiguous(q_fp8, k_fp8, k_scale, w, w_dtype, ks, ke, logits, ld_logits, T, S, H, D, clean,
                                   general, status, static_cast<cudaStream_t>(stream));
}

static int topk_select_checked(const float* logits, int64_t ld_logits, const int32_t* ks, const int32_t* ke, int T, int S,
                               int k, int32_t* out_idx, int sample, int overlapped, void* stream) {
  g_err[0] = 0;
  if (T < 0 || S < 0 || k < 0) return set_error(DSA_ERR_SHAPE, "topk_select: negative size");
  if (T == 0 || k == 0) return DSA_OK;
  if (!logits || !out_idx) return set_error(DSA_ERR_ARG, "topk_select: NULL pointer argument");
  if (ld_logits < S) return set_error(DSA_ERR_SHAPE, "topk_select: ld_logits < S");
  if (k > 65535) return set_error(DSA_ERR_SHAPE, "topk_select: k (%d) exceeds 65535", k);
  return topk_select_launch(logits, ld_logits, ks, ke, T, S, k, out_idx, sample, overlapped, static_cast<cudaStream_t>(stream));
}

extern "C" {

int dsa_version(void) { return 100; }

const char* dsa_last_error_string(void) { return g_err; }

int dsa_indexer_logits(const void* q_fp8, const void* k_fp8, const float* k_scale, const void* w, int w_dtype,
                       const int32_t* ks, const int32_t* ke, float* logits, int64_t ld_logits, int T, int S,
                       int H, int D, int clean, int32_t* status, void* stream) {
  return indexer_logits_checked(q_fp8, k_fp8, k_scale, w, w_dtype, ks, ke, logits, ld_logits, T, S, H, D, clean,
                                /*general=*/0, status, stream);
}

/* Test hooks (declared in include/dsa_b200.h under "test hooks"): the same calls pinned to the code path that the
 * normal entry points only take for some shapes or rows, so that tests can compare the two. */
int dsa_test_indexer_logits_general(const void* q_fp8, const void* k_fp8, const float* k_scale, const void* w,
                                    int w_dtype, const int32_t* ks, const int32_t* ke, float* logits,
                                    int64_t ld_logits, int T, int S, int H, int D, int clean, int32_t* status,
                                    void* stream) {
  return indexer_logits_checked(q_fp8, k_fp8, k_scale, w, w_dtype, ks, ke, logits, ld_logits, T, S, H, D, clean,
                                /*general=*/1, status, stream);
}

int dsa_test_topk_select_two_pass(const float* logits, int64_t ld_logits, const int32_t* ks, const int32_t* ke, int T,
                                  int S, int k, int32_t* out_idx, void* stream) {
  return topk_select_checked(logits, ld_logits, ks, ke, T, S, k, out_idx, /*sample=*/0, /*overlapped=*/0, stream);
}

int dsa_test_few_heads_plan(int T, int K, int sms, int parts, uint8_t* seen) {
  g_err[0] = 0;
  if (T < 0 || K < 0 || K > 2048 || sms < 1) return set_error(DSA_ERR_SHAPE, "test_few_heads_plan: bad sizes");
  if (T > 0 && !seen) return set_error(DSA_ERR_ARG, "test_few_heads_plan: NULL pointer argument");
  return few4_plan_probe(T, K, sms, parts, seen);
}

int dsa_test_bounded_wait(int poll_limit, int32_t* status, void* stream) {
  g_err[0] = 0;
  if (poll_limit < 1 || poll_limit > (1 << 16)) return set_error(DSA_ERR_ARG, "test_bounded_wait: poll_limit must be in [1, 65536]");
  if (!status) return set_error(DSA_ERR_ARG, "test_bounded_wait: NULL status");
  return bounded_wait_probe_launch((uint32_t)poll_limit, status, static_cast<cudaStream_t>(stream));
}

int dsa_indexer_logits_paged(const void* q_fp8, const void* w, int w_dtype, const void* kcache,
                             const float* kscale, const int32_t* block_table, int64_t table_stride,
                             const int32_t* ctx_len, float* logits, int64_t ld_logits, int B, int H, int D,
                             int num_pages, int max_ctx, int32_t* status, void* stream) {
  g_err[0] = 0;
  if (B < 0 || max_ctx < 0 || num_pages < 0)
    return set_error(DSA_ERR_SHAPE, "indexer_logits_paged: negative size");
  if (B == 0 || max_ctx == 0) return DSA_OK;
  if (!q_fp8 || !w || !kcache || !kscale || !block_table || !ctx_len || !logits)
    return set_error(DSA_ERR_ARG, "indexer_logits_paged: NULL pointer argument");
  if (w_dtype != DSA_W_F32 && w_dtype != DSA_W_BF16)
    return set_error(DSA_ERR_ARG, "indexer_logits_paged: bad w_dtype");
  if (ld_logits < max_ctx) return set_error(DSA_ERR_SHAPE, "indexer_logits_paged: ld_logits < max_ctx");
  if (ld_logits * 64 > 0x7fffffffLL) return set_error(DSA_ERR_SHAPE, "indexer_logits_paged: ld_logits too large");
  if (table_stride * 64 < max_ctx)
    return set_error(DSA_ERR_SHAPE, "indexer_logits_paged: block table row (%lld pages) shorter than max_ctx %d",
                     (long long)table_stride, max_ctx);
  if (!aligned16(q_fp8) || !aligned16(kcache) || !aligned16(kscale))
    return set_error(DSA_ERR_ALIGN, "indexer_logits_paged: q_fp8, kcache and kscale must be 16-byte aligned");
  if ((int64_t)num_pages * 64 > 0x7fffffffLL) return set_error(DSA_ERR_SHAPE, "indexer_logits_paged: cache too large");
  return indexer_logits_paged(q_fp8, w, w_dtype, kcache, kscale, block_table, table_stride, ctx_len, logits,
                              ld_logits, B, H, D, num_pages, max_ctx, status, static_cast<cudaStream_t>(stream));
}

int dsa_topk_select(const float* logits, int64_t ld_logits, const int32_t* ks, const int32_t* ke, int T, int S,
                    int k, int32_t* out_idx, void* stream) {
  return topk_select_checked(logits, ld_logits, ks, ke, T, S, k, out_idx, /*sample=*/1, /*overlapped=*/0, stream);
}

int dsa_sparse_mla_prefill(const void* q_bf16, const void* kv_bf16, const int32_t* idx, void* out_bf16, int T, int H,
                           int S_kv, int K, float scale, int32_t* status, void* stream) {
  g_err[0] = 0;
  if (T < 0 || H < 0 || S_kv < 0 || K < 0) return set_error(DSA_ERR_SHAPE, "sparse_mla_prefill: negative size");
  if (T == 0 || H == 0) return DSA_OK;
  if (!q_bf16 || !out_bf16 || (K > 0 && (!idx || !kv_bf16)))
    return set_error(DSA_ERR_ARG, "sparse_mla_prefill: NULL pointer argument");
  if (!aligned16(q_bf16) || !aligned16(kv_bf16) || !aligned16(out_bf16))
    return set_error(DSA_ERR_ALIGN, "sparse_mla_prefill: q, kv and out must be 16-byte aligned");
  if ((int64_t)T * H > 0x7fffffffLL || T > 0x7fffffff / 2) return set_error(DSA_ERR_SHAPE, "sparse_mla_prefill: T*H too large");
  if (H > 128 * 65535) return set_error(DSA_ERR_SHAPE, "sparse_mla_prefill: too many heads");
  if (K > 2048) return set_error(DSA_ERR_SHAPE, "sparse_mla_prefill: K (%d) exceeds 2048 selected keys per query", K);
  if (!(scale > 0.f)) return set_error(DSA_ERR_ARG, "sparse_mla_prefill: the softmax scale must be positive");
  return sparse_mla_prefill_launch(q_bf16, kv_bf16, idx, out_bf16, T, H, S_kv, K, scale, status,
                                   static_cast<cudaStream_t>(stream));
}

int dsa_block_sparse_mha(const void* q_bf16, const void* k_bf16, const void* v_bf16, const int32_t* lut,
                         const int32_t* num, void* out_bf16, int B, int S, int H, int D, int topk, float scale,
                         int32_t* status, void* stream) {
  g_err[0] = 0;
  if (B < 0 || S < 0 || H < 0 || topk < 0) return set_error(DSA_ERR_SHAPE, "block_sparse_mha: negative size");
  if (D != 128) return set_error(DSA_ERR_SHAPE, "block_sparse_mha: head dim %d, only 128 is built", D);
  if (!(scale > 0.f)) return set_error(DSA_ERR_ARG, "block_sparse_mha: the softmax scale must be positive");
  if (S % 64) return set_error(DSA_ERR_SHAPE, "block_sparse_mha: S (%d) must be a multiple of the 64-token block", S);
  if (B == 0 || S == 0 || H == 0) return DSA_OK;
  if (!q_bf16 || !k_bf16 || !v_bf16 || !out_bf16 || !num || (topk > 0 && !lut))
    return set_error(DSA_ERR_ARG, "block_sparse_mha: NULL pointer argument");
  if (!aligned16(q_bf16) || !aligned16(k_bf16) || !aligned16(v_bf16) || !aligned16(out_bf16))
    return set_error(DSA_ERR_ALIGN, "block_sparse_mha: q, k, v and out must be 16-byte aligned");
  if ((int64_t)B * S > 0x7fffffffLL || H > 65535 || B > 65535)
    return set_error(DSA_ERR_SHAPE, "block_sparse_mha: B*S, H or B too large");
  return block_sparse_mha_launch(q_bf16, k_bf16, v_bf16, lut, num, out_bf16, B, S, H, topk, scale, status,
                                 static_cast<cudaStream_t>(stream));
}

static int sparse_mla_decode_checked(const void* q_bf16, const void* cache, int record_bytes, const int32_t* block_table,
                                int64_t table_stride, int tokens_per_seq, const int32_t* idx, void* out_bf16, int B, int H, int K,
                                int num_pages, int max_ctx, float scale, void* workspace, size_t workspace_bytes,
                                int32_t* status, int overlapped, void* stream) {
  g_err[0] = 0;
  if (B < 0 || H < 0 || K < 0 || num_pages < 0 || max_ctx < 0)
    return set_error(DSA_ERR_SHAPE, "sparse_mla_decode_paged: negative size");
  if (record_bytes != 656 && record_bytes != 416)
    return set_error(DSA_ERR_SHAPE, "sparse_mla_decode_paged: records of %d bytes, only 656 (FP8) and 416 (4 bits) are built", record_bytes);
  if (tokens_per_seq < 1) return set_error(DSA_ERR_SHAPE, "sparse_mla_decode_paged: tokens_per_seq (%d) must be at least 1", tokens_per_seq);
  if (B == 0 || H == 0) return DSA_OK;
  if (!q_bf16 || !out_bf16 || (K > 0 && (!idx || !cache || !block_table)))
    return set_error(DSA_ERR_ARG, "sparse_mla_decode_paged: NULL pointer argument");
  if (!aligned16(q_bf16) || !aligned16(cache) || !aligned16(out_bf16))
    return set_error(DSA_ERR_ALIGN, "sparse_mla_decode_paged: q, cache and out must be 16-byte aligned");
  if (table_stride * 64 < max_ctx)
    return set_error(DSA_ERR_SHAPE, "sparse_mla_decode_paged: block table row shorter than max_ctx");
  if (K > 2048) return set_error(DSA_ERR_SHAPE, "sparse_mla_decode_paged: K (%d) exceeds 2048 selected keys per query", K);
  if (!(scale > 0.f)) return set_error(DSA_ERR_ARG, "sparse_mla_decode_paged: the softmax scale must be positive");
  if ((int64_t)num_pages * 64 > 0x7fffffffLL || (int64_t)B * H > 0x7fffffffLL)
    return set_error(DSA_ERR_SHAPE, "sparse_mla_decode_paged: problem too large");
  if (workspace && (reinterpret_cast<uintptr_t>(workspace) & 15))
    return set_error(DSA_ERR_WORKSPACE, "sparse_mla_decode_paged: workspace must be 16-byte aligned");
  return sparse_mla_decode_launch(q_bf16, cache, record_bytes, block_table, table_stride, tokens_per_seq, idx, out_bf16, B, H, K, num_pages,
                                  max_ctx, scale, workspace, workspace_bytes, status, overlapped,
                                  static_cast<cudaStream_t>(stream));
}

int dsa_sparse_mla_decode_paged(const void* q_bf16, const void* cache, const int32_t* block_table,
                                int64_t table_stride, const int32_t* idx, void* out_bf16, int B, int H, int K,
                                int num_pages, int max_ctx, float scale, void* workspace, size_t workspace_bytes,
                                int32_t* status, void* stream) {
  return sparse_mla_decode_checked(q_bf16, cache, /*record_bytes=*/656, block_table, table_stride, /*tokens_per_seq=*/1, idx, out_bf16, B, H, K,
                                   num_pages, max_ctx, scale, workspace, workspace_bytes, status, /*overlapped=*/0, stream);
}

int dsa_sparse_mla_decode_records(const void* q_bf16, const void* cache, int record_bytes, const int32_t* block_table, int64_t table_stride,
                                  int tokens_per_seq, const int32_t* idx, void* out_bf16, int T, int H, int K, int num_pages, int max_ctx, float scale,
                                  void* workspace, size_t workspace_bytes, int32_t* status, void* stream) {
  return sparse_mla_decode_checked(q_bf16, cache, record_bytes, block_table, table_stride, tokens_per_seq, idx, out_bf16, T, H, K, num_pages, max_ctx,
                                   scale, workspace, workspace_bytes, status, /*overlapped=*/0, stream);
}

int dsa_decode_step_records(const void* q_fp8, const void* w, int w_dtype, const void* kcache, const float* kscale, int k_pages,
                    const int32_t* block_table, int64_t table_stride, const int32_t* ctx_len, float* logits, int64_t ld_logits,
                    int B, int idx_heads, int idx_dim, int max_ctx, int k, int32_t* idx, const void* q_bf16, const void* latent,
                    int record_bytes, int latent_pages, void* out_bf16, int H, float scale, void* workspace, size_t workspace_bytes,
                    int32_t* status, void* stream) {
  int rc = dsa_indexer_logits_paged(q_fp8, w, w_dtype, kcache, kscale, block_table, table_stride, ctx_len, logits, ld_logits, B,
                                    idx_heads, idx_dim, k_pages, max_ctx, status, stream);
  // Small batches leave SMs to the next kernel while one still runs: each is launched so that it may set itself up under the end
  // of the one before.  us a step in a plain loop over one set of inputs: 1 x 2000 37.0 -> 29.5, 2 x 9000 43.1 -> 36.9, 7 x 33000 50.3 -> 45.1,
  // 12 x 30000 57.5 -> 52.3, 20 x 20000 65.7 -> 61.6; 30 x 9000 70.2 both.  In a CUDA graph, whose launches are closer, 40 batches of 4 to 24
  // with contexts of 3000 to 60000 take 1.4 % less on average: 6 % less at 3000 tokens, up to 6 % more at 20000 and from 18 sequences on
  // (23 x 20000 62.3 -> 66.5), 2 % more with 8 of 9000 and over, the others less.  From 64 up the top-k's blocks take the first SMs that come
  // free, and the rest waits.
  const int overlapped = B <= 24;
  if (!rc) rc = topk_select_checked(logits, ld_logits, nullptr, ctx_len, B, max_ctx, k, idx, /*sample=*/1, overlapped, stream);
  if (!rc) rc = sparse_mla_decode_checked(q_bf16, latent, record_bytes, block_table, table_stride, /*tokens_per_seq=*/1, idx, out_bf16, B, H, k, latent_pages, max_ctx,
                                          scale, workspace, workspace_bytes, status, overlapped, stream);
  return rc;
}

int dsa_decode_step(const void* q_fp8, const void* w, int w_dtype, const void* kcache, const float* kscale, int k_pages,
                    const int32_t* block_table, int64_t table_stride, const int32_t* ctx_len, float* logits, int64_t ld_logits,
                    int B, int idx_heads, int idx_dim, int max_ctx, int k, int32_t* idx, const void* q_bf16, const void* latent,
                    int latent_pages, void* out_bf16, int H, float scale, void* workspace, size_t workspace_bytes,
                    int32_t* status, void* stream) {
  return dsa_decode_step_records(q_fp8, w, w_dtype, kcache, kscale, k_pages, block_table, table_stride, ctx_len, logits, ld_logits, B, idx_heads,
                                 idx_dim, max_ctx, k, idx, q_bf16, latent, /*record_bytes=*/656, latent_pages, out_bf16, H, scale, workspace,
                                 workspace_bytes, status, stream);
}

size_t dsa_sparse_mla_decode_workspace_bytes(int B, int H, int K) {
  if (B <= 0 || H <= 0 || K <= 0) return 0;
  return mla_decode_workspace_bytes(B, H, K);
}

size_t dsa_sparse_mla_decode_records_workspace_bytes(int record_bytes, int T, int H, int K) {
  if (T <= 0 || H <= 0 || K <= 0) return 0;
  return mla_decode_records_workspace_bytes(record_bytes, T, H, K);
}

int dsa_fp8_quant_per_block(const void* x, int x_dtype, int64_t n_blocks, int block_size, void* q_fp8, float* scale,
                            void* stream) {
  g_err[0] = 0;
  if (n_blocks < 0) return set_error(DSA_ERR_SHAPE, "fp8_quant_per_block: negative size");
  if (n_blocks == 0) return DSA_OK;
  if (!x || !q_fp8 || !scale) return set_error(DSA_ERR_ARG, "fp8_quant_per_block: NULL pointer argument");
  if (x_dtype != DSA_X_F32 && x_dtype != DSA_X_BF16) return set_error(DSA_ERR_ARG, "fp8_quant_per_block: bad x_dtype");
  if (!aligned16(x) || (reinterpret_cast<uintptr_t>(q_fp8) & 3))
    return set_error(DSA_ERR_ALIGN, "fp8_quant_per_block: x must be 16-byte and q_fp8 4-byte aligned");
  return fp8_quant_launch(x, x_dtype == DSA_X_BF16, n_blocks, block_size, q_fp8, scale, static_cast<cudaStream_t>(stream));
}

int dsa_pack_latent_cache(const void* kv, int kv_dtype, int64_t row_stride, int64_t n_tokens, void* records, void* stream) {
  g_err[0] = 0;
  if (n_tokens < 0) return set_error(DSA_ERR_SHAPE, "pack_latent_cache: negative size");
  if (n_tokens == 0) return DSA_OK;
  if (!kv || !records) return set_error(DSA_ERR_ARG, "pack_latent_cache: NULL pointer argument");
  if (kv_dtype != DSA_X_F32 && kv_dtype != DSA_X_BF16) return set_error(DSA_ERR_ARG, "pack_latent_cache: bad kv_dtype");
  const int64_t elt = kv_dtype == DSA_X_BF16 ? 2 : 4;
  if (n_tokens > 1 && row_stride < 576) return set_error(DSA_ERR_SHAPE, "pack_latent_cache: row_stride below 576");
  if (!aligned16(kv) || !aligned16(records) || (n_tokens > 1 && (row_stride * elt) % 16))
    return set_error(DSA_ERR_ALIGN, "pack_latent_cache: every row and the records must be 16-byte aligned");
  return pack_latent_launch(kv, kv_dtype == DSA_X_BF16, row_stride, n_tokens, records, static_cast<cudaStream_t>(stream));
}

int dsa_pack_latent4(const void* kv, int kv_dtype, int64_t row_stride, int64_t n_tokens, void* cache, int64_t cache_rows, const int32_t* slots,
                     const void* k_fp8, const float* k_scale, void* kcache, float* kscale, int32_t* status, void* stream) {
  g_err[0] = 0;
  if (n_tokens < 0 || cache_rows < 0) return set_error(DSA_ERR_SHAPE, "pack_latent4: negative size");
  if (n_tokens == 0) return DSA_OK;
  if (!kv || !cache) return set_error(DSA_ERR_ARG, "pack_latent4: NULL pointer argument");
  if (kv_dtype != DSA_X_F32 && kv_dtype != DSA_X_BF16) return set_error(DSA_ERR_ARG, "pack_latent4: bad kv_dtype");
  if (!slots && cache_rows < n_tokens)
    return set_error(DSA_ERR_SHAPE, "pack_latent4: %lld tokens in order need as many records, the cache has %lld", (long long)n_tokens, (long long)cache_rows);
  const int64_t elt = kv_dtype == DSA_X_BF16 ? 2 : 4;
  if (n_tokens > 1 && row_stride < 576) return set_error(DSA_ERR_SHAPE, "pack_latent4: row_stride below 576");
  if (!aligned16(kv) || !aligned16(cache) || (n_tokens > 1 && (row_stride * elt) % 16))
    return set_error(DSA_ERR_ALIGN, "pack_latent4: every row and the cache must be 16-byte aligned");
  if (k_fp8 && (!k_scale || !kcache || !kscale)) return set_error(DSA_ERR_ARG, "pack_latent4: NULL pointer argument");
  if (k_fp8 && (!aligned16(k_fp8) || !aligned16(kcache))) return set_error(DSA_ERR_ALIGN, "pack_latent4: keys and their cache must be 16-byte aligned");
  return pack_latent4_launch(kv, kv_dtype == DSA_X_BF16, row_stride, n_tokens, cache, slots, cache_rows, k_fp8, k_scale, kcache, kscale, status,
                             static_cast<cudaStream_t>(stream));
}

int dsa_unpack_latent4(const void* cache, int64_t cache_rows, const int32_t* block_table, int64_t n_tokens, void* out_bf16, int64_t row_stride,
                       int32_t* status, void* stream) {
  g_err[0] = 0;
  if (n_tokens < 0 || cache_rows < 0) return set_error(DSA_ERR_SHAPE, "unpack_latent4: negative size");
  if (n_tokens == 0) return DSA_OK;
  if (!cache || !out_bf16) return set_error(DSA_ERR_ARG, "unpack_latent4: NULL pointer argument");
  if (!block_table && cache_rows < n_tokens)
    return set_error(DSA_ERR_SHAPE, "unpack_latent4: %lld tokens in order, the cache has %lld", (long long)n_tokens, (long long)cache_rows);
  if (n_tokens > 1 && row_stride < 576) return set_error(DSA_ERR_SHAPE, "unpack_latent4: row_stride below 576");
  if (!aligned16(cache) || !aligned16(out_bf16) || (n_tokens > 1 && row_stride % 8))
    return set_error(DSA_ERR_ALIGN, "unpack_latent4: the cache and every row must be 16-byte aligned");
  return unpack_latent4_launch(cache, cache_rows, block_table, n_tokens, out_bf16, row_stride, status, static_cast<cudaStream_t>(stream));
}

// The caches that a call copies pages of: 0, or an error.
static int check_page_caches(const char* who, const dsa_page_cache* caches, int n_caches) {
  if (n_caches < 0) return set_error(DSA_ERR_SHAPE, "%s: negative number of caches", who);
  if (n_caches > 0 && !caches) return set_error(DSA_ERR_ARG, "%s: NULL pointer argument", who);
  int64_t layers = 0;
  for (int c = 0; c < n_caches; ++c) {
    const dsa_page_cache& h = caches[c];
    if (h.layers < 0 || h.token_bytes <= 0 || h.token_bytes > (1 << 20) || h.token_bytes % 4)
      return set_error(DSA_ERR_SHAPE, "%s: cache %d: a token's bytes (%d) must be a multiple of 4, up to 1 MiB", who, c, h.token_bytes);
    if (h.layers > 0 && !h.base) return set_error(DSA_ERR_ARG, "%s: NULL pointer argument", who);
    if (!aligned16(h.base) || (h.layers > 1 && h.layer_stride % 16))
      return set_error(DSA_ERR_ALIGN, "%s: cache %d: every layer must be 16-byte aligned", who, c);
    layers += (int64_t)h.layers * ((h.token_bytes * 64 >> 14) + 1);
  }
  if (layers > (1 << 24)) return set_error(DSA_ERR_SHAPE, "%s: too many layers", who);
  return DSA_OK;
}
// Sizes of the page tables: 0, or an error.
static int check_pool(const char* who, const void* table, int64_t stride, int P, int B, const void* refs, int num_pages, int n) {
  if (P < 0 || B < 0 || num_pages < 0 || n < 0) return set_error(DSA_ERR_SHAPE, "%s: negative size", who);
  if ((int64_t)num_pages * 64 > 0x7fffffffLL || (int64_t)P * 64 > 0x7fffffffLL) return set_error(DSA_ERR_SHAPE, "%s: too many pages", who);
  if (B > (1 << 18)) return set_error(DSA_ERR_SHAPE, "%s: %d table rows, 262144 are the most", who, B);
  if (B > 1 && stride < P) return set_error(DSA_ERR_SHAPE, "%s: table rows overlap", who);
  if ((B > 0 && P > 0 && !table) || (num_pages > 0 && !refs)) return set_error(DSA_ERR_ARG, "%s: NULL pointer argument", who);
  return DSA_OK;
}
static int check_pages_workspace(const char* who, const void* workspace, size_t bytes, int num_pages, int n) {
  if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 3) || bytes < pages_workspace_bytes(num_pages, n))
    return set_error(DSA_ERR_WORKSPACE, "%s: workspace missing, unaligned or smaller than %zu B", who, pages_workspace_bytes(num_pages, n));
  return DSA_OK;
}

size_t dsa_pages_workspace_bytes(int num_pages, int n) { return num_pages < 0 || n < 0 ? 0 : pages_workspace_bytes(num_pages, n); }

int dsa_copy_pages(const dsa_page_cache* caches, int n_caches, int num_pages, const int32_t* src, const int32_t* dst, const int32_t* tokens, int n,
                   int32_t* status, void* stream) {
  g_err[0] = 0;
  int rc = check_page_caches("copy_pages", caches, n_caches);
  if (rc) return rc;
  if (n < 0 || num_pages < 0) return set_error(DSA_ERR_SHAPE, "copy_pages: negative size");
  if (n == 0 || n_caches == 0) return DSA_OK;
  if (!src || !dst) return set_error(DSA_ERR_ARG, "copy_pages: NULL pointer argument");
  return copy_pages_launch(caches, n_caches, num_pages, src, dst, tokens, n, status, static_cast<cudaStream_t>(stream));
}

int dsa_extend_pages(int32_t* block_table, int64_t table_stride, int P, int B, int32_t* ctx_len, int32_t* refs, int num_pages, const int32_t* rows,
                     const int32_t* n_new, int n, int max_new, int32_t* slots, void* workspace, size_t workspace_bytes, int32_t* status, void* stream) {
  g_err[0] = 0;
  int rc = check_pool("extend_pages", block_table, table_stride, P, B, refs, num_pages, n);
  if (rc || n == 0) return rc;
  if ((int64_t)B * P > 0x7fffffffLL)                   // the pages that a call asks for are summed in 32 bits
    return set_error(DSA_ERR_SHAPE, "extend_pages: more than 2147483647 table entries (%d rows of %d)", B, P);
  if (max_new < 0 || max_new > (1 << 30)) return set_error(DSA_ERR_SHAPE, "extend_pages: bad max_new (%d)", max_new);
  if (!ctx_len || !rows || !n_new || (max_new > 0 && !slots)) return set_error(DSA_ERR_ARG, "extend_pages: NULL pointer argument");
  if ((rc = check_pages_workspace("extend_pages", workspace, workspace_bytes, num_pages, n))) return rc;
  return extend_pages_launch(block_table, table_stride, P, B, ctx_len, refs, num_pages, rows, n_new, n, max_new, slots, static_cast<int32_t*>(workspace),
                             status, static_cast<cudaStream_t>(stream));
}

int dsa_fork_pages(int32_t* block_table, int64_t table_stride, int P, int B, int32_t* ctx_len, int32_t* refs, int num_pages, const int32_t* parents,
                   const int32_t* children, int n, const dsa_page_cache* caches, int n_caches, void* workspace, size_t workspace_bytes,
                   int32_t* status, void* stream) {
  g_err[0] = 0;
  int rc = check_pool("fork_pages", block_table, table_stride, P, B, refs, num_pages, n);
  if (!rc) rc = check_page_caches("fork_pages", caches, n_caches);
  if (rc || n == 0) return rc;
  if (!ctx_len || !parents || !children) return set_error(DSA_ERR_ARG, "fork_pages: NULL pointer argument");
  if ((rc = check_pages_workspace("fork_pages", workspace, workspace_bytes, num_pages, n))) return rc;
  return fork_pages_launch(block_table, table_stride, P, B, ctx_len, refs, num_pages, parents, children, n, caches, n_caches,
                           static_cast<int32_t*>(workspace), status, static_cast<cudaStream_t>(stream));
}

int dsa_free_pages(int32_t* block_table, int64_t table_stride, int P, int B, int32_t* ctx_len, int32_t* refs, int num_pages, const int32_t* rows, int n,
                   int32_t* status, void* stream) {
  g_err[0] = 0;
  const int rc = check_pool("free_pages", block_table, table_stride, P, B, refs, num_pages, n);
  if (rc || n == 0) return rc;
  if (!ctx_len || !rows) return set_error(DSA_ERR_ARG, "free_pages: NULL pointer argument");
  return free_pages_launch(block_table, table_stride, P, B, ctx_len, refs, num_pages, rows, n, status, static_cast<cudaStream_t>(stream));
}

int dsa_compact_pages(const int32_t* block_table, int64_t table_stride, int32_t* new_table, int64_t new_stride, int P, int B, const int32_t* refs,
                      int32_t* new_refs, int num_pages, const dsa_page_cache* caches, int n_caches, void* workspace, size_t workspace_bytes,
                      int32_t* status, void* stream) {
  g_err[0] = 0;
  int rc = check_pool("compact_pages", block_table, table_stride, P, B, refs, num_pages, 0);
  if (!rc) rc = check_pool("compact_pages", new_table, new_stride, P, B, new_refs, num_pages, 0);
  if (!rc) rc = check_page_caches("compact_pages", caches, n_caches);
  if (rc) return rc;
  if ((rc = check_pages_workspace("compact_pages", workspace, workspace_bytes, num_pages, 0))) return rc;
  return compact_pages_launch(block_table, table_stride, new_table, new_stride, P, B, refs, new_refs, num_pages, caches, n_caches,
                              static_cast<int32_t*>(workspace), status, static_cast<cudaStream_t>(stream));
}

// ---- window layers and drafted tokens ------------------------------------------------------------------------------------
static int check_drafts(const char* who, int B, int tokens_per_seq, const void* tree, int max_ctx) {
  if (B < 0 || max_ctx < 0) return set_error(DSA_ERR_SHAPE, "%s: negative size", who);
  if (tokens_per_seq < 1) return set_error(DSA_ERR_SHAPE, "%s: tokens_per_seq (%d) must be at least 1", who, tokens_per_seq);
  if (tree && tokens_per_seq > 64) return set_error(DSA_ERR_SHAPE, "%s: a tree has at most 64 drafts, not %d", who, tokens_per_seq);
  if ((int64_t)B * tokens_per_seq > 0x7fffffffLL) return set_error(DSA_ERR_SHAPE, "%s: more than 2147483647 query rows", who);
  if (reinterpret_cast<uintptr_t>(tree) & 7) return set_error(DSA_ERR_ALIGN, "%s: tree must be 8-byte aligned", who);
  return DSA_OK;
}
static int check_window(const char* who, int H, int window, int first, float scale) {
  if (H < 0) return set_error(DSA_ERR_SHAPE, "%s: negative size", who);
  if (window < 1 || first < 0) return set_error(DSA_ERR_SHAPE, "%s: window (%d) must be at least 1 and first (%d) at least 0", who, window, first);
  if (!(scale > 0.f)) return set_error(DSA_ERR_ARG, "%s: the softmax scale must be positive", who);
  return DSA_OK;
}

size_t dsa_window_mla_prefill_workspace_bytes(int T, int H, int window, int first) {
  return T <= 0 || H <= 0 || window < 1 || first < 0 ? 0 : window_mla_prefill_workspace(T, H, window, first);
}

int dsa_window_mla_prefill(const void* q_bf16, const void* kv_bf16, const int32_t* ks, const int32_t* ke, void* out_bf16, int T, int H, int S, int window,
                           int first, float scale, void* workspace, size_t workspace_bytes, int32_t* status, void* stream) {
  g_err[0] = 0;
  if (T < 0 || S < 0) return set_error(DSA_ERR_SHAPE, "window_mla_prefill: negative size");
  const int rc = check_window("window_mla_prefill", H, window, first, scale);
  if (rc || T == 0 || H == 0) return rc;
  if (!q_bf16 || !out_bf16 || (S > 0 && !kv_bf16)) return set_error(DSA_ERR_ARG, "window_mla_prefill: NULL pointer argument");
  if (!aligned16(q_bf16) || !aligned16(kv_bf16) || !aligned16(out_bf16))
    return set_error(DSA_ERR_ALIGN, "window_mla_prefill: q, kv and out must be 16-byte aligned");
  if ((int64_t)T * H > 0x7fffffffLL) return set_error(DSA_ERR_SHAPE, "window_mla_prefill: T*H exceeds 2^31");
  if (workspace && (reinterpret_cast<uintptr_t>(workspace) & 15))
    return set_error(DSA_ERR_WORKSPACE, "window_mla_prefill: workspace must be 16-byte aligned");
  return window_mla_prefill_launch(q_bf16, kv_bf16, ks, ke, out_bf16, T, H, S, window, first, scale, workspace, workspace_bytes, status,
                                   static_cast<cudaStream_t>(stream));
}

size_t dsa_window_mla_decode_workspace_bytes(int record_bytes, int B, int tokens_per_seq, int H, int window, int first, int max_ctx) {
  return B <= 0 || tokens_per_seq < 1 || H <= 0 || window < 1 || first < 0 || max_ctx <= 0 ? 0 : window_mla_decode_workspace(record_bytes, B, tokens_per_seq, H, window, first, max_ctx);
}

int dsa_window_mla_decode_paged(const void* q_bf16, const void* cache, int record_bytes, const int32_t* block_table, int64_t table_stride,
                                const int32_t* ctx_len, const int32_t* n_new, const int64_t* tree, int tokens_per_seq, void* out_bf16, int B, int H,
                                int window, int first, int num_pages, int max_ctx, float scale, void* workspace, size_t workspace_bytes, int32_t* status,
                                void* stream) {
  const char* who = "window_mla_decode_paged";
  g_err[0] = 0;
  int rc = check_drafts(who, B, tokens_per_seq, tree, max_ctx);
  if (!rc) rc = check_window(who, H, window, first, scale);
  if (rc) return rc;
  if (num_pages < 0) return set_error(DSA_ERR_SHAPE, "%s: negative size", who);
  if (record_bytes != 656 && record_bytes != 416) return set_error(DSA_ERR_SHAPE, "%s: records of %d bytes, only 656 (FP8) and 416 (4 bits) are built", who, record_bytes);
  if (B == 0 || H == 0) return DSA_OK;
  if (!q_bf16 || !out_bf16 || !ctx_len || (max_ctx > 0 && (!cache || !block_table))) return set_error(DSA_ERR_ARG, "%s: NULL pointer argument", who);
  if (!aligned16(q_bf16) || !aligned16(cache) || !aligned16(out_bf16)) return set_error(DSA_ERR_ALIGN, "%s: q, cache and out must be 16-byte aligned", who);
  if (table_stride * 64 < max_ctx) return set_error(DSA_ERR_SHAPE, "%s: block table row shorter than max_ctx", who);
  if ((int64_t)num_pages * 64 > 0x7fffffffLL || (int64_t)B * tokens_per_seq * H > 0x7fffffffLL) return set_error(DSA_ERR_SHAPE, "%s: problem too large", who);
  if (workspace && (reinterpret_cast<uintptr_t>(workspace) & 15)) return set_error(DSA_ERR_WORKSPACE, "%s: workspace must be 16-byte aligned", who);
  return window_mla_decode_launch(q_bf16, cache, record_bytes, block_table, table_stride, ctx_len, n_new, tree, tokens_per_seq, out_bf16, B, H, window, first,
                                  num_pages, max_ctx, scale, workspace, workspace_bytes, status, static_cast<cudaStream_t>(stream));
}

int dsa_indexer_logits_drafts(const void* q_fp8, const void* w, int w_dtype, const void* kcache, const float* kscale, const int32_t* block_table,
                              int64_t table_stride, const int32_t* ctx_len, const int32_t* n_new, const int64_t* tree, int tokens_per_seq, float* logits,
                              int64_t ld_logits, int B, int H, int D, int num_pages, int max_ctx, int32_t* status, void* stream) {
  const char* who = "indexer_logits_drafts";
  g_err[0] = 0;
  const int rc = check_drafts(who, B, tokens_per_seq, tree, max_ctx);
  if (rc) return rc;
  if (num_pages < 0) return set_error(DSA_ERR_SHAPE, "%s: negative size", who);
  if (D != 128 || (H != 64 && H != 32 && H != 16)) return set_error(DSA_ERR_SHAPE, "%s: unsupported (heads=%d, head_dim=%d)", who, H, D);
  if (B == 0 || max_ctx == 0) return DSA_OK;
  if (!q_fp8 || !w || !kcache || !kscale || !block_table || !ctx_len || !logits) return set_error(DSA_ERR_ARG, "%s: NULL pointer argument", who);
  if (w_dtype != DSA_W_F32 && w_dtype != DSA_W_BF16) return set_error(DSA_ERR_ARG, "%s: bad w_dtype", who);
  if (ld_logits < max_ctx) return set_error(DSA_ERR_SHAPE, "%s: ld_logits < max_ctx", who);
  if (ld_logits * 64 > 0x7fffffffLL) return set_error(DSA_ERR_SHAPE, "%s: ld_logits too large", who);
  if (table_stride * 64 < max_ctx) return set_error(DSA_ERR_SHAPE, "%s: block table row (%lld pages) shorter than max_ctx %d", who, (long long)table_stride, max_ctx);
  if (!aligned16(q_fp8) || !aligned16(kcache) || !aligned16(kscale)) return set_error(DSA_ERR_ALIGN, "%s: q_fp8, kcache and kscale must be 16-byte aligned", who);
  if ((int64_t)num_pages * 64 > 0x7fffffffLL || (int64_t)B * tokens_per_seq * H > 0x7fffffffLL) return set_error(DSA_ERR_SHAPE, "%s: problem too large", who);
  return indexer_logits_drafts_launch(q_fp8, w, w_dtype == DSA_W_BF16, kcache, kscale, block_table, table_stride, ctx_len, n_new, tree, tokens_per_seq, logits,
                                      ld_logits, B, H, num_pages, max_ctx, status, static_cast<cudaStream_t>(stream));
}

size_t dsa_topk_select_drafts_workspace_bytes(int B, int tokens_per_seq) { return B < 0 || tokens_per_seq < 1 ? 0 : (size_t)B * tokens_per_seq * sizeof(int32_t); }

int dsa_topk_select_drafts(const float* logits, int64_t ld_logits, const int32_t* ctx_len, const int32_t* n_new, const int64_t* tree, int tokens_per_seq,
                           int B, int max_ctx, int k, int32_t* out_idx, void* workspace, size_t workspace_bytes, void* stream) {
  const char* who = "topk_select_drafts";
  g_err[0] = 0;
  const int rc = check_drafts(who, B, tokens_per_seq, tree, max_ctx);
  if (rc) return rc;
  if (k < 0) return set_error(DSA_ERR_SHAPE, "%s: negative size", who);
  if (B == 0 || k == 0) return DSA_OK;
  if ((max_ctx > 0 && !logits) || !ctx_len || !out_idx) return set_error(DSA_ERR_ARG, "%s: NULL pointer argument", who);
  if (ld_logits < max_ctx) return set_error(DSA_ERR_SHAPE, "%s: ld_logits < max_ctx", who);
  if (k > 65535) return set_error(DSA_ERR_SHAPE, "%s: k (%d) exceeds 65535", who, k);
  const size_t need = dsa_topk_select_drafts_workspace_bytes(B, tokens_per_seq);
  if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 3) || workspace_bytes < need)
    return set_error(DSA_ERR_WORKSPACE, "%s: workspace missing, unaligned or smaller than %zu B", who, need);
  return topk_select_drafts_launch(logits, ld_logits, ctx_len, n_new, tree, tokens_per_seq, B, max_ctx, k, out_idx, static_cast<int32_t*>(workspace),
                                   static_cast<cudaStream_t>(stream));
}

int dsa_accept_drafts(int32_t* block_table, int64_t table_stride, int P, int B, int32_t* ctx_len, int32_t* refs, int num_pages, const int32_t* rows,
                      const int32_t* n_new, const int32_t* path, int path_stride, const int32_t* n_keep, int n, const dsa_page_cache* caches, int n_caches,
                      void* workspace, size_t workspace_bytes, int32_t* status, void* stream) {
  const char* who = "accept_drafts";
  g_err[0] = 0;
  int rc = check_pool(who, block_table, table_stride, P, B, refs, num_pages, n);
  if (!rc) rc = check_page_caches(who, caches, n_caches);
  if (rc || n == 0) return rc;
  if (path_stride < 0) return set_error(DSA_ERR_SHAPE, "%s: negative size", who);
  if (!ctx_len || !rows || !n_new || !n_keep || (path_stride > 0 && !path)) return set_error(DSA_ERR_ARG, "%s: NULL pointer argument", who);
  if ((rc = check_pages_workspace(who, workspace, workspace_bytes, 0, n))) return rc;
  return accept_drafts_launch(block_table, table_stride, P, B, ctx_len, refs, num_pages, rows, n_new, path, path_stride, n_keep, n, caches, n_caches,
                              static_cast<int32_t*>(workspace), status, static_cast<cudaStream_t>(stream));
}

int dsa_rope_fp8_quant_gated(const void* x_bf16, int64_t n_rows, int head_dim, int rope_dim, int interleave, int rows_per_pos,
                             const float* cos_table, const float* sin_table, int64_t n_pos, void* q_fp8, float* scale,
                             const void* gate_bf16, float gate_mul0, float gate_mul1, float* gate_out, void* stream) {
  g_err[0] = 0;
  if (n_rows < 0 || n_pos < 0) return set_error(DSA_ERR_SHAPE, "rope_fp8_quant: negative size");
  if (n_rows == 0) return DSA_OK;
  if (!x_bf16 || !cos_table || !sin_table || !q_fp8 || !scale) return set_error(DSA_ERR_ARG, "rope_fp8_quant: NULL pointer argument");
  if (head_dim != 64 && head_dim != 128) return set_error(DSA_ERR_SHAPE, "rope_fp8_quant: head dim %d, only 64 and 128 are built", head_dim);
  if (gate_bf16 && !gate_out) return set_error(DSA_ERR_ARG, "rope_fp8_quant: NULL pointer argument");
  // the rotated part is made of whole lanes (head_dim / 32 values each) and, in the halves form, of two equal lane groups
  const int per = head_dim / 32;
  if (rope_dim <= 0 || rope_dim > head_dim || rope_dim % (2 * per)) return set_error(DSA_ERR_SHAPE, "rope_fp8_quant: rope_dim %d does not fit head dim %d", rope_dim, head_dim);
  if (!interleave && ((rope_dim / 2 / per) & (rope_dim / 2 / per - 1))) return set_error(DSA_ERR_SHAPE, "rope_fp8_quant: rope_dim / 2 must span a power-of-two number of lanes");
  if (rows_per_pos <= 0 || (n_rows + rows_per_pos - 1) / rows_per_pos > n_pos)
    return set_error(DSA_ERR_SHAPE, "rope_fp8_quant: %lld rows at %d per position need more than the %lld positions of the tables",
                     (long long)n_rows, rows_per_pos, (long long)n_pos);
  if (!aligned16(x_bf16) || (reinterpret_cast<uintptr_t>(q_fp8) & 3)) return set_error(DSA_ERR_ALIGN, "rope_fp8_quant: x must be 16-byte and q_fp8 4-byte aligned");
  return rope_fp8_quant_launch(x_bf16, n_rows, head_dim, rope_dim, interleave, rows_per_pos, cos_table, sin_table, q_fp8, scale,
                               gate_bf16, gate_mul0, gate_mul1, gate_out, static_cast<cudaStream_t>(stream));
}

int dsa_rope_fp8_quant(const void* x_bf16, int64_t n_rows, int head_dim, int rope_dim, int interleave, int rows_per_pos,
                       const float* cos_table, const float* sin_table, int64_t n_pos, void* q_fp8, float* scale,
                       void* stream) {
  return dsa_rope_fp8_quant_gated(x_bf16, n_rows, head_dim, rope_dim, interleave, rows_per_pos, cos_table, sin_table, n_pos, q_fp8, scale,
                                  nullptr, 0.f, 0.f, nullptr, stream);
}

static const int kMinChunkRows = 256;

static int64_t logits_ld(int S) { return ((int64_t)S + 3) & ~int64_t(3); }

size_t dsa_indexer_topk_workspace_bytes(int T, int S) {
  if (T <= 0 || S <= 0) return 0;
  return (size_t)T * (size_t)logits_ld(S) * sizeof(float);
}

int dsa_indexer_topk(const void* q_fp8, const void* k_fp8, const float* k_scale, const void* w, int w_dtype,
                     const int32_t* ks, const int32_t* ke, int T, int S, int H, int D, int k, int32_t* out_idx,
                     void* workspace, size_t workspace_bytes, int32_t* status, void* stream) {
  g_err[0] = 0;
  if (T < 0 || S < 0 || k < 0) return set_error(DSA_ERR_SHAPE, "indexer_topk: negative size");
  if (T == 0 || k == 0) return DSA_OK;
  if (S == 0) return set_error(DSA_ERR_SHAPE, "indexer_topk: S = 0 with k > 0");
  if (!out_idx || !ke) return set_error(DSA_ERR_ARG, "indexer_topk: NULL pointer argument");
  const int64_t ld = logits_ld(S);
  const size_t row_bytes = (size_t)ld * sizeof(float);
  if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15))
    return set_error(DSA_ERR_WORKSPACE, "indexer_topk: workspace missing or not 16-byte aligned");
  int64_t rows = (int64_t)(workspace_bytes / row_bytes);
  const int min_rows = T < kMinChunkRows ? T : kMinChunkRows;
  if (rows < min_rows)
    return set_error(DSA_ERR_WORKSPACE, "indexer_topk: workspace %zu B holds %lld rows, need >= %d (%zu B)",
                     workspace_bytes, (long long)rows, min_rows, (size_t)min_rows * row_bytes);
  if (rows > T) rows = T;
  if (rows < T) rows &= ~int64_t(kMinChunkRows - 1);   // whole query groups per chunk
  float* logits = static_cast<float*>(workspace);
  const size_t w_elt = w_dtype == DSA_W_BF16 ? 2 : 4;
  for (int64_t r0 = 0; r0 < T; r0 += rows) {
    const int n = (int)((T - r0 < rows) ? T - r0 : rows);
    int rc = dsa_indexer_logits(static_cast<const uint8_t*>(q_fp8) + (size_t)r0 * H * D, k_fp8, k_scale,
                                static_cast<const uint8_t*>(w) + (size_t)r0 * H * w_elt, w_dtype,
                                ks ? ks + r0 : nullptr, ke + r0, logits, ld, n, S, H, D, /*clean=*/0, status, stream);
    if (rc) return rc;
    rc = dsa_topk_select(logits, ld, ks ? ks + r0 : nullptr, ke + r0, n, S, k, out_idx + (size_t)r0 * k, stream);
    if (rc) return rc;
  }
  return DSA_OK;
}

}  // extern "C"
