// Lightning-indexer logits of drafted tokens over the paged FP8 key cache, and the ends of their rows for the selection:
//   logits[r, s] = k_scale[s] * sum_h w[r, h] * relu(q[r, h, :] . k[s, :])   where draft r sees position s (drafts.cuh), -inf where not.
#include <cuda.h>
#include <cuda_fp8.h>
#include <math_constants.h>

#include "dsa_common.cuh"
#include "dsa_host.h"
#include "drafts.cuh"

namespace dsa {

constexpr int kDraftKeys = 128;                        // columns of a row are written up to a multiple of this
constexpr int kDraftPage = 64;

struct DraftLogitsArgs {
  const uint8_t* q;                                    // [T, H, 128] e4m3
  const void* w;                                       // [T, H]
  int w_is_bf16;
  const uint8_t* kcache;                               // [num_pages*64, 128] e4m3
  const float* kscale;
  const int32_t* block_table;
  int64_t table_stride;
  DraftArgs drafts;
  float* logits;
  int64_t ld;
  int B, num_pages;
  int* status;
};

// A CTA for 128 keys of a row, a thread per key.
template <int H>
__global__ void __launch_bounds__(kDraftKeys) draft_logits_kernel(const DraftLogitsArgs a) {
  __shared__ float q_s[H][128];
  __shared__ float w_s[H];
  const int per = a.drafts.per_seq, r = blockIdx.y, b = r / per, i = r - b * per;
  const Drafts dr = drafts_of(a.drafts, b);
  if (dr.bad && a.status) atomicCAS(a.status, kStatusOk, kStatusBadIndex);
  if ((int64_t)blockIdx.x * kDraftKeys >= dr.ctx) return;
  for (int e = threadIdx.x; e < H * 128; e += kDraftKeys) {
    __nv_fp8_e4m3 v;
    v.__x = a.q[(int64_t)r * H * 128 + e];
    q_s[e >> 7][e & 127] = float(v);
  }
  for (int h = threadIdx.x; h < H; h += kDraftKeys)
    w_s[h] = a.w_is_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(a.w)[(int64_t)r * H + h]) : static_cast<const float*>(a.w)[(int64_t)r * H + h];
  __syncthreads();
  const int s = blockIdx.x * kDraftKeys + threadIdx.x, P = dr.ctx - dr.m;
  if (s >= a.drafts.max_ctx) return;
  bool seen = i < dr.m && s < dr.ctx;
  if (seen && s >= P) seen = a.drafts.tree ? (draft_mask(a.drafts, b, i) >> (s - P)) & 1 : s - P <= i;
  float score = -CUDART_INF_F;
  if (seen) {
    const int page = __ldg(a.block_table + (int64_t)b * a.table_stride + s / kDraftPage);
    if (page >= 0 && page < a.num_pages) {
      const int64_t row = (int64_t)page * kDraftPage + s % kDraftPage;
      float k[128];
      for (int c = 0; c < 128; ++c) {
        __nv_fp8_e4m3 v;
        v.__x = a.kcache[row * 128 + c];
        k[c] = float(v);
      }
      score = 0.f;
      for (int h = 0; h < H; ++h) {
        float d = 0.f;
#pragma unroll
        for (int c = 0; c < 128; ++c) d += q_s[h][c] * k[c];
        score += w_s[h] * fmaxf(d, 0.f);
      }
      score *= a.kscale[row];
    } else if (a.status) {
      atomicCAS(a.status, kStatusOk, kStatusBadIndex);
    }
  }
  a.logits[(int64_t)r * a.ld + s] = score;
}

int indexer_logits_drafts_launch(const void* q, const void* w, int w_is_bf16, const void* kcache, const float* kscale, const int32_t* block_table,
                                 int64_t table_stride, const int32_t* ctx_len, const int32_t* n_new, const int64_t* tree, int tokens_per_seq, float* logits,
                                 int64_t ld, int B, int H, int num_pages, int max_ctx, int32_t* status, cudaStream_t stream) {
  DraftLogitsArgs a{};
  a.q = static_cast<const uint8_t*>(q);
  a.w = w; a.w_is_bf16 = w_is_bf16;
  a.kcache = static_cast<const uint8_t*>(kcache);
  a.kscale = kscale;
  a.block_table = block_table; a.table_stride = table_stride;
  a.drafts = {ctx_len, n_new, tree, tokens_per_seq, max_ctx};
  a.logits = logits; a.ld = ld;
  a.B = B; a.num_pages = num_pages;
  a.status = status;
  const dim3 grid((max_ctx + kDraftKeys - 1) / kDraftKeys, B * tokens_per_seq);
  if (H == 64) draft_logits_kernel<64><<<grid, kDraftKeys, 0, stream>>>(a);
  else if (H == 32) draft_logits_kernel<32><<<grid, kDraftKeys, 0, stream>>>(a);
  else draft_logits_kernel<16><<<grid, kDraftKeys, 0, stream>>>(a);
  return check_launch("indexer_logits_drafts");
}

// ---- selection -------------------------------------------------------------------------------------------------------
// ends[r]: the position behind the last one that row r sees, 0 for a row without a token.
__global__ void __launch_bounds__(256) draft_ends_kernel(const DraftArgs d, int T, int32_t* ends) {
  const int r = blockIdx.x * 256 + threadIdx.x;
  if (r >= T) return;
  const int b = r / d.per_seq, i = r - b * d.per_seq;
  const Drafts dr = drafts_of(d, b);
  ends[r] = i < dr.m ? dr.ctx - dr.m + i + 1 : 0;
}
// A selection of a row that sees fewer positions than it has slots holds all that the row does not see as well: those become empty slots.
__global__ void __launch_bounds__(256) draft_unsee_kernel(const DraftArgs d, int k, int32_t* idx) {
  const int r = blockIdx.x, b = r / d.per_seq, i = r - b * d.per_seq;
  const Drafts dr = drafts_of(d, b);
  const int P = dr.ctx - dr.m;
  if (i >= dr.m) return;
  const uint64_t bits = draft_mask(d, b, i);
  if (P + __popcll(bits) >= min(k, P + i + 1)) return;
  int32_t* row = idx + (int64_t)r * k;
  for (int j = threadIdx.x; j < k; j += 256) {
    const int at = row[j] - P;
    if (at >= 0 && !(bits >> at & 1)) row[j] = -1;     // at <= i < 64
  }
}

int topk_select_launch(const float* logits, int64_t ld, const int32_t* ks, const int32_t* ke, int T, int S, int k, int32_t* out, int sample, int overlapped,
                       cudaStream_t stream);

int topk_select_drafts_launch(const float* logits, int64_t ld, const int32_t* ctx_len, const int32_t* n_new, const int64_t* tree, int tokens_per_seq, int B,
                              int max_ctx, int k, int32_t* out, int32_t* ends, cudaStream_t stream) {
  const DraftArgs d{ctx_len, n_new, tree, tokens_per_seq, max_ctx};
  const int T = B * tokens_per_seq;
  draft_ends_kernel<<<(T + 255) / 256, 256, 0, stream>>>(d, T, ends);
  int rc = check_launch("topk_select_drafts");
  if (!rc) rc = topk_select_launch(logits, ld, nullptr, ends, T, max_ctx, k, out, /*sample=*/1, /*overlapped=*/0, stream);
  if (rc || !tree || k == 0) return rc;
  draft_unsee_kernel<<<T, 256, 0, stream>>>(d, k, out);
  return check_launch("topk_select_drafts");
}

}  // namespace dsa
