// Drafted tokens of the sequences of a batch: the last m of a sequence's ctx tokens, whose query rows are b * per_seq + i, i < m (rows i >= m
// belong to no token).  P = ctx - m tokens stand before them.  Draft i sees those, the drafts before it that its mask names (no masks: all
// of them, a chain) and itself.
#pragma once
#include <stdint.h>

#include "dsa_common.cuh"

namespace dsa {

constexpr int kMaxTreeDrafts = 64;                     // bits of a mask

struct DraftArgs {
  const int32_t* ctx_len;                              // [B]
  const int32_t* n_new;                                // [B], null: min(ctx, per_seq)
  const int64_t* tree;                                 // [B, per_seq], null: chains
  int per_seq;
  int max_ctx;
};

struct Drafts {
  int ctx, m;                                          // of a sequence whose lengths make no sense: 0 and 0
  bool bad;
};

__device__ __forceinline__ Drafts drafts_of(const DraftArgs& d, int b) {
  Drafts r;
  r.ctx = __ldg(d.ctx_len + b);
  r.m = d.n_new ? __ldg(d.n_new + b) : min(r.ctx, d.per_seq);
  r.bad = r.ctx < 0 || r.ctx > d.max_ctx || r.m < 0 || r.m > d.per_seq || r.m > r.ctx;
  if (r.bad) r.ctx = r.m = 0;
  return r;
}

// The drafts that draft i of sequence b sees, of a tree: those before it that its mask names, and itself.
__device__ __forceinline__ uint64_t draft_mask(const DraftArgs& d, int b, int i) {
  const uint64_t named = static_cast<uint64_t>(__ldg(d.tree + (int64_t)b * d.per_seq + i));
  return (named & ((1ull << i) - 1)) | (1ull << i);
}

}  // namespace dsa
