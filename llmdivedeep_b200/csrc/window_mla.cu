// MLA attention over a sliding window and the first tokens (MQA over the shared 576-dim latent KV, 512-dim V): a query row at position p of its
// sequence sees the positions < first and the last `window` ones, p itself included,
//   o[r, :] = sum_s softmax_s(scale * q[r, :] . kv[s, :]) * kv[s, :512],   s < first or p - window < s <= p,
// over bf16 rows (prompts) or the records of the paged latent caches (decode, one or several query tokens a sequence: a chain, or a tree of
// drafts, drafts.cuh).
#include <cuda.h>
#include <cudaTypedefs.h>
#include <math_constants.h>

#include "dsa_common.cuh"
#include "dsa_host.h"
#include "drafts.cuh"
#include "mla_pair.cuh"

namespace dsa {

struct WinArgs {
  const __nv_bfloat16* q;         // [T, H, 576]
  const uint8_t* kv;              // prompts: [S, 576] bf16 rows; decode: [num_phys_rows] records
  const int32_t *ks, *ke;         // prompts: [T] rows' windows; null: 0, and the last T positions of S
  const int32_t* block_table;     // decode: [B, table_stride]
  int64_t table_stride;
  DraftArgs drafts;               // decode
  __nv_bfloat16* out;             // [T, H, 512]
  int T, H, S;                    // S: prompts, rows of kv
  int window, first;
  int num_phys_rows;
  float scale_log2e;
  int* status;
};

// What a row sees: two stretches of positions, a1 <= b0, and single ones behind `at`.
struct Sees {
  int a0, a1, b0, b1, at;
  uint64_t bits;
};
__device__ __forceinline__ Sees sees_prompt(const WinArgs& a, int t) {
  const int ks = a.ks ? max(__ldg(a.ks + t), 0) : 0, ke = a.ke ? min(__ldg(a.ke + t), a.S) : a.S - a.T + t + 1;
  Sees s{};
  if (ke <= ks) return s;
  s.a0 = ks;
  s.a1 = a.first < ke - ks ? ks + a.first : ke;
  s.b0 = max(s.a1, ke - a.window);
  s.b1 = ke;
  return s;
}
__device__ __forceinline__ Sees sees_draft(const WinArgs& a, const Drafts& dr, int b, int i) {
  Sees s{};
  if (i >= dr.m) return s;
  const int P = dr.ctx - dr.m;
  s.at = P;
  if (!a.drafts.tree) {
    const int ke = P + i + 1;
    s.a1 = min(a.first, ke);
    s.b0 = max(s.a1, ke - a.window);
    s.b1 = ke;
    return s;
  }
  s.bits = draft_mask(a.drafts, b, i);
  const int n = __popcll(s.bits);
  s.a1 = min(a.first, P);
  s.b0 = max(s.a1, P + n - a.window);                  // its own position is P + n - 1
  s.b1 = max(s.b0, P);
  uint64_t left = s.bits;
  for (int k = 0; k < n - a.window; ++k) {             // drafts of its path that the window has passed
    const uint64_t lowest = left & (0 - left);
    left ^= lowest;
    if (P + k >= a.first) s.bits ^= lowest;
  }
  return s;
}

// A lane's share of a row: values 8 lane .. of either half of the latent, rope values 2 lane ..
struct RowShare {
  float x[2][8], r[2];
};
template <int SRC>
__device__ __forceinline__ RowShare load_share(const uint8_t* __restrict__ row, int lane) {
  RowShare v;
  uint32_t rope;
  if constexpr (SRC == kSrcRows) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint4 w = __ldg(reinterpret_cast<const uint4*>(row + h * 512 + lane * 16));
      const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int i = 0; i < 8; ++i) v.x[h][i] = __uint_as_float(i & 1 ? u[i >> 1] & 0xffff0000u : u[i >> 1] << 16);
    }
    rope = __ldg(reinterpret_cast<const uint32_t*>(row + 1024) + lane);
  } else if constexpr (SRC == kSrcFp8) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint2 w = __ldg(reinterpret_cast<const uint2*>(row + h * 256 + lane * 8));
      const uint4 b = e4m3x8_to_bf16(w, __ldg(reinterpret_cast<const float*>(row + 512) + h * 2 + (lane >> 4)));
      const uint32_t u[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
      for (int i = 0; i < 8; ++i) v.x[h][i] = __uint_as_float(i & 1 ? u[i >> 1] & 0xffff0000u : u[i >> 1] << 16);
    }
    rope = __ldg(reinterpret_cast<const uint32_t*>(row + 528) + lane);
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint8_t* half = row + h * kLatent4Half;
      uint32_t u[4];
      latent4_codes(__ldg(reinterpret_cast<const uint32_t*>(half) + lane), u);
      const uint32_t sc = latent4_scale(__ldg(half + kLatent4Scales + (lane >> 1)));
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t p = mul_bf16x2(u[i], sc);
        v.x[h][2 * i] = __uint_as_float(p << 16) * kLatent4Gain;
        v.x[h][2 * i + 1] = __uint_as_float(p & 0xffff0000u) * kLatent4Gain;
      }
    }
    rope = __ldg(reinterpret_cast<const uint32_t*>(row + (lane >> 4) * kLatent4Half + kLatent4Rope) + (lane & 15));
  }
  v.r[0] = __uint_as_float(rope << 16);
  v.r[1] = __uint_as_float(rope & 0xffff0000u);
  return v;
}

// One row's softmax and output, key by key.
struct RowState {
  float m, l, o[2][8];
};
__device__ __forceinline__ void row_step(RowState& st, const RowShare& q, const RowShare& k, float scale_log2e) {
  float d = q.r[0] * k.r[0] + q.r[1] * k.r[1];
#pragma unroll
  for (int i = 0; i < 8; ++i) d += q.x[0][i] * k.x[0][i] + q.x[1][i] * k.x[1][i];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
  const float s = d * scale_log2e, m = fmaxf(st.m, s), at = m == -CUDART_INF_F ? 0.f : m;
  const float keep = st.m == -CUDART_INF_F ? 0.f : exp2f(st.m - at), p = exp2f(s - at);
  st.m = m;
  st.l = st.l * keep + p;
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int i = 0; i < 8; ++i) st.o[h][i] = st.o[h][i] * keep + p * k.x[h][i];
}

// A warp per query row (token, head).
template <int SRC>
__global__ void __launch_bounds__(256) window_rows_kernel(const WinArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t rows = (int64_t)a.T * a.H, warps = (int64_t)gridDim.x * 8;
  for (int64_t g = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); g < rows; g += warps) {
    const int t = (int)(g / a.H);
    Sees s;
    const int32_t* table = nullptr;
    if constexpr (SRC == kSrcRows) {
      s = sees_prompt(a, t);
    } else {
      const int b = t / a.drafts.per_seq, i = t - b * a.drafts.per_seq;
      const Drafts dr = drafts_of(a.drafts, b);
      if (dr.bad && a.status) atomicCAS(a.status, kStatusOk, kStatusBadIndex);
      s = sees_draft(a, dr, b, i);
      table = a.block_table + (int64_t)b * a.table_stride;
    }
    const RowShare q = load_share<kSrcRows>(reinterpret_cast<const uint8_t*>(a.q + g * kMlaDqk), lane);
    RowState st{-CUDART_INF_F, 0.f, {}};
    auto key = [&](int pos) {
      int64_t row = pos;
      constexpr int kBytes = SRC == kSrcRows ? kMlaDqk * 2 : SRC == kSrcFp8 ? kLatentTokenBytes : kLatent4Bytes;
      if constexpr (SRC != kSrcRows) {
        const int page = __ldg(table + pos / kLatentPage);
        if (page < 0 || (int64_t)(page + 1) * kLatentPage > a.num_phys_rows) {
          if (a.status) atomicCAS(a.status, kStatusOk, kStatusBadIndex);
          return;
        }
        row = (int64_t)page * kLatentPage + pos % kLatentPage;
      }
      row_step(st, q, load_share<SRC>(a.kv + row * kBytes, lane), a.scale_log2e);
    };
    for (int p = s.a0; p < s.a1; ++p) key(p);
    for (int p = s.b0; p < s.b1; ++p) key(p);
    for (uint64_t left = s.bits; left; left &= left - 1) key(s.at + __ffsll(left) - 1);
    const float inv = st.l > 0.f ? 1.f / st.l : st.l;  // (a NaN stays one)
    uint4* o = reinterpret_cast<uint4*>(a.out + g * kMlaDv);
#pragma unroll
    for (int h = 0; h < 2; ++h)
      o[h * 32 + lane] = make_uint4(pack_bf16x2(st.o[h][0] * inv, st.o[h][1] * inv), pack_bf16x2(st.o[h][2] * inv, st.o[h][3] * inv),
                                    pack_bf16x2(st.o[h][4] * inv, st.o[h][5] * inv), pack_bf16x2(st.o[h][6] * inv, st.o[h][7] * inv));
  }
}

template <int SRC>
static int launch_window(const WinArgs& a, cudaStream_t stream) {
  if (a.T == 0 || a.H == 0) return DSA_OK;
  const int64_t ctas = ((int64_t)a.T * a.H + 7) / 8;
  window_rows_kernel<SRC><<<(unsigned)min(ctas, (int64_t)sm_count() * 64), 256, 0, stream>>>(a);
  return check_launch("window_mla");
}

int window_mla_prefill_launch(const void* q, const void* kv, const int32_t* ks, const int32_t* ke, void* out, int T, int H, int S, int window, int first,
                              float scale, int32_t* status, cudaStream_t stream) {
  WinArgs a{};
  a.q = static_cast<const __nv_bfloat16*>(q);
  a.kv = static_cast<const uint8_t*>(kv);
  a.ks = ks; a.ke = ke;
  a.out = static_cast<__nv_bfloat16*>(out);
  a.T = T; a.H = H; a.S = S;
  a.window = window; a.first = first;
  a.scale_log2e = scale * 1.4426950408889634f;
  a.status = status;
  return launch_window<kSrcRows>(a, stream);
}

int window_mla_decode_launch(const void* q, const void* cache, int record_bytes, const int32_t* block_table, int64_t table_stride, const int32_t* ctx_len,
                             const int32_t* n_new, const int64_t* tree, int tokens_per_seq, void* out, int B, int H, int window, int first, int num_pages,
                             int max_ctx, float scale, int32_t* status, cudaStream_t stream) {
  WinArgs a{};
  a.q = static_cast<const __nv_bfloat16*>(q);
  a.kv = static_cast<const uint8_t*>(cache);
  a.block_table = block_table;
  a.table_stride = table_stride;
  a.drafts = {ctx_len, n_new, tree, tokens_per_seq, max_ctx};
  a.out = static_cast<__nv_bfloat16*>(out);
  a.T = B * tokens_per_seq; a.H = H;
  a.window = window; a.first = first;
  a.num_phys_rows = num_pages * kLatentPage;
  a.scale_log2e = scale * 1.4426950408889634f;
  a.status = status;
  return record_bytes == kLatent4Bytes ? launch_window<kSrc4>(a, stream) : launch_window<kSrcFp8>(a, stream);
}

}  // namespace dsa
