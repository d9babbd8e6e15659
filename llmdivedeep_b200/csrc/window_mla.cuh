// What the two kernels of window attention share (window_prompt.cu: bf16 rows; window_mla.cu: records of the paged caches): their arguments, what a
// row sees, a row taken key by key, and the plan of parts.
#pragma once
#include <math_constants.h>

#include "dsa_common.cuh"
#include "dsa_host.h"
#include "drafts.cuh"
#include "mla_pair.cuh"

namespace dsa {

// A block's partial scores cross between the pair as they are, in fp32: both sides add the same two numbers, so that one softmax weights all of a row's columns.  It
// is 32 KB a block and direction, and that costs: 2048 tokens x 128 heads, window 4096, 2236 us, 1.23 a block, where half of the bits took 1821 (24 of them
// 2068), 64 sequences of decode, FP8, 128 for 103.  But a half rounded to fp16 is off by 2^-11 of itself, which the sum of two that cancel need not be large
// against (an output 7 % off with halves of 4000), and it is lost beyond 65504.  A form with 16 bits for numbers that a rounding to 2^-10 does not hurt and
// 32 for others took 2016 and 112, but few blocks more time than this (160 sequences of drafts 78 for 73), and its time went by the data; two messages of half a part 2530.
// Every thread has its counterpart's row and keys: it stores its 32 numbers straight into the peer's shared memory, a warp's 16-byte pieces side by side, with no copy
// of its own in between.
constexpr int kWinXWarp = 32 * 32 * 4;                 // a warp's part of a tile: 32 rows x 32 keys
constexpr int kWinXBytes = 8 * kWinXWarp;
static_assert(kWinXBytes == 2 * kMlaXBytes, "in the place of a tile on its way out and one that comes in");
__device__ __forceinline__ void send_scores(uint32_t dst_cluster, uint32_t bar_cluster, const uint32_t (&sv)[32]) {
#pragma unroll
  for (int c = 0; c < 8; ++c)
    asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, [%5];"
                 ::"r"(dst_cluster + c * 512), "r"(sv[4 * c]), "r"(sv[4 * c + 1]), "r"(sv[4 * c + 2]), "r"(sv[4 * c + 3]), "r"(bar_cluster) : "memory");
}
// The peer's numbers have come.  (The stores belong to the cluster's scope, and so does this wait.)
__device__ __forceinline__ bool wait_scores(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* status) {
  return mbar_wait_warp<4, true>(bar, parity, abort_flag, status);
}
// s = this side's scores + the peer's
__device__ __forceinline__ void add_scores(const uint8_t* recv, const uint32_t (&sv)[32], float (&s)[32]) {
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    const float4 x = *reinterpret_cast<const float4*>(recv + c * 512);
    s[4 * c + 0] = __uint_as_float(sv[4 * c + 0]) + x.x;
    s[4 * c + 1] = __uint_as_float(sv[4 * c + 1]) + x.y;
    s[4 * c + 2] = __uint_as_float(sv[4 * c + 2]) + x.z;
    s[4 * c + 3] = __uint_as_float(sv[4 * c + 3]) + x.w;
  }
}

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
  int seq_rows, seq_units;        // query rows (token, head) of a sequence, and its units; prompts: all rows are one sequence's
  int unit_rows;                  // rows of a unit: 128, fewer where a prompt's rows of few heads are many tokens
  int n_full;                     // the first n_full units are a CTA pair each; ...
  int n_split;                    // ... the keys of every later one are cut into n_split parts, a pair each
  float* part_o;                  // [parts, 128, 512] fp32 normalised partial outputs
  float* part_lse;                // [parts, 2, 128] their log2-sum-exp as each CTA of the pair has it (-inf: nothing seen)
  int tma_out;                    // the output tensor map is valid: full units leave through TMA stores
  // drafts over rows that were made bf16 first: kv is [B * pad] rows, slot j of sequence b row b * pad + j, with a bit for each that has a page
  int pad;
  uint32_t* valid;
  int live;                       // only units with drafts in them are jobs; the other rows' zeros come with the rows of the keys
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

// The score of a row and a key, times log2(e): every lane has it.
__device__ __forceinline__ float row_score(const RowShare& q, const RowShare& k, float scale_log2e) {
  float d = q.r[0] * k.r[0] + q.r[1] * k.r[1];
#pragma unroll
  for (int i = 0; i < 8; ++i) d += q.x[0][i] * k.x[0][i] + q.x[1][i] * k.x[1][i];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
  return d * scale_log2e;
}


__device__ __forceinline__ uint32_t low_bits(int n) { return n >= 32 ? 0xffffffffu : (1u << max(n, 0)) - 1u; }
// which of the 32 keys from k0 on are in [lo, hi)
__device__ __forceinline__ uint32_t range_bits(int lo, int hi, int k0) { return low_bits(hi - k0) & ~low_bits(lo - k0); }

// which of the 32 keys from k0 on have their bit set, bit j at `at` + j
__device__ __forceinline__ uint32_t draft_bits(uint64_t bits, int at, int k0) {
  const int sh = k0 - at;
  return sh >= 64 || sh <= -32 ? 0u : sh >= 0 ? static_cast<uint32_t>(bits >> sh) : static_cast<uint32_t>(bits) << -sh;
}

// The keys of tokens tok0 .. tok1 of a sequence by slots: the first tokens' [0, head) and behind them the windows' [shift + head, ...); slot j is
// position j, from head on j + shift.  Slots [full0, full1) are seen by all of these tokens.
struct Slots {
  int head, shift, n, full0, full1;
};
__device__ __forceinline__ Slots slots_of(const WinArgs& a, const Drafts& dr, int tok0, int tok1) {
  Slots s{};
  if (tok0 >= dr.m) return s;
  const bool tree = a.drafts.tree != nullptr;
  const int P = dr.ctx - dr.m, hi = P + min(tok1, dr.m - 1) + 1, near = P + 1 + (tree ? 0 : tok0), lo = max(0, near - a.window);
  const int least = tree ? P : near;                   // positions up to here are seen by every row
  s.head = min(a.first, hi);
  if (lo <= s.head) s.head = 0;
  else s.shift = lo - s.head;
  s.n = hi - s.shift;
  s.full0 = max(min(a.first, hi), hi - a.window);      // (of a tree: its path may be shorter)
  s.full0 = s.full0 <= min(a.first, least) ? 0 : s.full0 - s.shift;
  s.full1 = least - s.shift;
  return s;
}

// Units run in rounds of one to a pair of SMs.  The keys of a partly filled last round's units are cut into parts, as many as there are pairs for.
constexpr int kWinMaxParts = 16;
constexpr int kWinPartBlocks = 2;                      // blocks of a part at least
constexpr size_t kWinPartBytes = (size_t)128 * (kMlaDv + 2) * sizeof(float);
inline int window_parts(int64_t units, int64_t keys) {
  const int pairs = max(1, sm_count() / 2), rest = (int)(units % pairs);
  const int64_t blocks = (keys + kMlaBlk - 1) / kMlaBlk;
  return rest == 0 ? 1 : (int)max((int64_t)1, min(min((int64_t)kWinMaxParts, blocks / kWinPartBlocks), (int64_t)(pairs / rest)));
}
// of every call of up to `units` of them
inline size_t window_workspace(int64_t units, int64_t keys) {
  const int pairs = max(1, sm_count() / 2);
  size_t most = 0;
  for (int64_t u = 1; u < pairs && u <= units; ++u) {
    const int parts = window_parts(u, keys);
    if (parts > 1) most = max(most, (size_t)u * parts);
  }
  return most * kWinPartBytes;
}
// Keys of a unit at most, that parts are worth: first tokens, window, and the tokens of the unit.
inline int64_t window_keys(int H, int64_t window, int64_t first, int64_t tokens, int64_t most) {
  return min(most, window + first + min(tokens, (int64_t)(127 / H + 2)));
}
// Sets a.n_full, a.n_split and where the parts go.
inline void window_plan(WinArgs& a, int64_t units, int64_t keys, void* workspace, size_t workspace_bytes) {
  const int rest = (int)(units % max(1, sm_count() / 2));
  int ns = window_parts(units, keys);
  if (ns > 1) {                                        // a smaller workspace: as many parts as it holds
    const size_t fit = workspace ? workspace_bytes / kWinPartBytes / rest : 0;
    if (fit < (size_t)ns) ns = fit > 1 ? (int)fit : 1;
  }
  a.n_full = (int)(ns > 1 ? units - rest : units);
  a.n_split = ns;
  if (ns > 1) {
    a.part_o = static_cast<float*>(workspace);
    a.part_lse = a.part_o + (size_t)rest * ns * 128 * kMlaDv;
  }
}
// Drafts of sequences over rows that were made bf16 first (window_prompt.cu); a.kv and what goes with it is set.
int window_prompt_drafts(const WinArgs& a, void* workspace, size_t workspace_bytes, cudaStream_t stream);
void window_prompt_units(WinArgs& a);                  // sets unit_rows, seq_units and live
size_t window_prompt_drafts_workspace(int B, int64_t seq_rows, int H, int64_t keys);
// The kernel that merges the parts of units n_full .. of `units` (window_mla.cu).
void window_combine(const WinArgs& a, int64_t units, cudaStream_t stream);
int make_tmap_2d_bytes(CUtensorMap* m, const void* base, uint64_t rows, uint64_t inner_bytes, uint64_t row_pitch, uint32_t box_bytes, uint32_t box_rows);

}  // namespace dsa
