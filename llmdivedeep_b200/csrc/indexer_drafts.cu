// Lightning-indexer logits of drafted tokens over the paged FP8 key cache, and the ends of their rows for the selection:
//   logits[r, s] = k_scale[s] * sum_h w[r, h] * relu(q[r, h, :] . k[s, :])   where draft r sees position s (drafts.cuh), -inf where not.
// The drafts of a sequence share the fetch of its keys: a persistent CTA takes units of up to four drafts and 16 tiles of keys; one warp writes units, one fetches
// pages and scales, one issues the MMAs of two accumulators in turn, sixteen sum the heads.  What bounds it: the epilogue, an FMA with saturation and one more a
// head and key, at the power cap where it is long.  64 sequences of 128K x 4 drafts x 64 heads: 538 us with scales by plain loads, 475 by TMA, 415 with units from
// shared memory, 360 with one barrier a tile and one test a warp before the store (410 to 420 in loops at the power cap); 190 us for its bytes.
#include <cuda.h>
#include <cudaTypedefs.h>
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

// A work unit is NT drafts of a sequence against a chunk of its keys: the accumulator of a tile is 128 SUB keys by NT drafts x H heads, SUB = 4 / NT, so
// that each of four epilogue warpgroups has one draft and 128 keys of every tile: a thread is a key and holds the draft's H head weights in
// registers.  The arithmetic, and its order, is that of indexer_logits_rw_kernel (indexer_logits.cu), so that a draft's scores are those of a
// decode step of its own, bit for bit.
constexpr float kDraftRelu = 0x1p-25f;                 // relu(d) = 2^25 sat(2^-25 d): exact, and on the FMA pipe
constexpr int kDraftChunk = 16;                        // tiles of a unit at most
template <int H, int NT>
struct DraftCfg {
  static constexpr int SUB = 4 / NT, N = NT * H, KSTEPS = 4;
  static constexpr int TILE_KEYS = SUB * kDraftKeys, PAGES = TILE_KEYS / kDraftPage;
  static constexpr int K_TILE_BYTES = TILE_KEYS * 128, Q_TILE_BYTES = N * 128;
  static constexpr int STAGES = NT == 4 ? 6 : NT == 2 ? 4 : 3;
  static constexpr int COLS = 4 * H, TMEM_COLS = 2 * COLS;           // of an accumulator stage; two of them
  static constexpr int EPI_WARPS = 16, THREADS = 128 + 512;
  static constexpr int REGS_EPI = 104, REGS_OTHER = 64;
  static_assert(512 * REGS_EPI + 128 * REGS_OTHER <= THREADS * 96, "more registers than the launch has");
  // A slot of the scales' ring is written again when the MMAs of STAGES tiles before have been done, and for them the epilogue has read two tiles more.
  static constexpr int SCALES = STAGES + 2, SCALE_BYTES = TILE_KEYS * 4;
  static constexpr int SMEM_BYTES = 1024 + STAGES * K_TILE_BYTES + 2 * Q_TILE_BYTES + SCALES * SCALE_BYTES + 2 * N * 4 + 256 + 2 * 64 + 2 * PAGES * kDraftChunk * 4;
  static_assert(SMEM_BYTES <= 227 * 1024, "shared memory budget");
};

// A unit as its roles find it in shared memory.
struct DraftUnit {
  int b, g, t_lo, t_hi;                                // sequence, group of NT drafts, tiles; t_lo < 0: there are no more
  int P, m, columns;                                   // tokens before the drafts, drafts, columns that are written
  int holes;                                           // a page of the tiles is none
  uint64_t bits[4];                                    // of the group's drafts: which drafts they see
};
static_assert(sizeof(DraftUnit) == 64, "");
// Unit u: whether it has tiles, and drafts.
template <int TILE_KEYS, int NT>
__device__ __forceinline__ bool draft_unit(const DraftLogitsArgs& a, int u, int groups, int chunk, DraftUnit& x, bool& live, bool& bad) {
  const int c = u / (a.B * groups), bg = u - c * a.B * groups;
  x.b = bg / groups;
  x.g = bg - x.b * groups;
  const Drafts dr = drafts_of(a.drafts, x.b);
  bad = dr.bad;
  x.P = dr.ctx - dr.m;
  x.m = dr.m;
  x.columns = min(a.drafts.max_ctx, (dr.ctx + kDraftKeys - 1) / kDraftKeys * kDraftKeys);
  x.t_lo = c * chunk;
  x.t_hi = min(x.t_lo + chunk, (dr.ctx + TILE_KEYS - 1) / TILE_KEYS);
  live = x.g * NT < dr.m;
  return x.t_lo < x.t_hi;
}

template <int H, int NT>
__global__ void __launch_bounds__(DraftCfg<H, NT>::THREADS, 1)
draft_logits_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k, const DraftLogitsArgs a, const int groups,
                    const int chunk, const int n_units) {
  using C = DraftCfg<H, NT>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* k_s = smem;                                        // STAGES x [TILE_KEYS x 128]
  uint8_t* q_s = k_s + C::STAGES * C::K_TILE_BYTES;           // 2 x [N rows x 128]
  float* scale_s = reinterpret_cast<float*>(q_s + 2 * C::Q_TILE_BYTES);      // SCALES x [TILE_KEYS]
  float* w_s = scale_s + C::SCALES * C::TILE_KEYS;            // 2 x N head weights
  uint64_t* bars = reinterpret_cast<uint64_t*>(w_s + 2 * C::N);
  uint64_t *k_full = bars, *k_empty = k_full + C::STAGES, *q_full = k_empty + C::STAGES, *q_empty = q_full + 2, *acc_full = q_empty + 2, *acc_empty = acc_full + 2,
           *w_full = acc_empty + 2, *w_empty = w_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(w_empty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  static_assert((2 * C::STAGES + 12 + 1) * 8 <= 256, "barriers");
  DraftUnit* unit_s = reinterpret_cast<DraftUnit*>(bars + 32);       // two units deep, like q_s, w_s and
  int* pages_s = reinterpret_cast<int*>(unit_s + 2);          // the first cache row of every page of the unit's chunk, -1 = none

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < C::STAGES; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 1);
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], C::EPI_WARPS);
      mbar_init(&w_full[i], 1);
      mbar_init(&w_empty[i], C::EPI_WARPS + 2);
    }
    *abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_desc(&tmap_q);
    tma_prefetch_desc(&tmap_k);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, C::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::REGS_OTHER));
    if (warp == 0) {
      // ------------------------------ TMA producer ------------------------------
      uint32_t it = 0;
      bool ok = true;
      for (uint32_t nu = 0;; ++nu) {
        const int ub = nu & 1;
        ok = mbar_wait_warp(&w_full[ub], (nu >> 1) & 1, abort_flag, a.status);
        if (!ok) break;
        const int b = unit_s[ub].b, g = unit_s[ub].g, t_lo = unit_s[ub].t_lo, t_hi = unit_s[ub].t_hi;
        if (t_lo < 0) break;
        ok = mbar_wait_warp(&q_empty[ub], ((nu >> 1) & 1) ^ 1, abort_flag, a.status);
        if (!ok) break;
        if (lane == 0) {
          mbar_expect_tx(&q_full[ub], C::Q_TILE_BYTES);
          tma_load_2d(q_s + ub * C::Q_TILE_BYTES, &tmap_q, 0, (b * a.drafts.per_seq + g * NT) * H, &q_full[ub]);
        }
        for (int kt = t_lo; kt < t_hi; ++kt, ++it) {
          const int st = it % C::STAGES, sc = it % C::SCALES;
          ok = mbar_wait_warp(&k_empty[st], ((it / C::STAGES) & 1) ^ 1, abort_flag, a.status);
          if (!ok) break;
          const int r = lane < C::PAGES ? pages_s[ub * C::PAGES * kDraftChunk + C::PAGES * (kt - t_lo) + lane] : -1;      // a page that is none is skipped, its scores are not used
          const int n_valid = __popc(__ballot_sync(0xffffffffu, r >= 0));
          if (lane == 0) {
            if (n_valid) mbar_expect_tx(&k_full[st], n_valid * (kDraftPage * (128 + 4)));
            else mbar_arrive(&k_full[st]);
          }
          __syncwarp();
          if (r >= 0) {
            tma_load_2d(k_s + st * C::K_TILE_BYTES + lane * (kDraftPage * 128), &tmap_k, 0, r, &k_full[st]);
            asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                         ::"r"(smem_u32(scale_s + sc * C::TILE_KEYS + lane * kDraftPage)), "l"(a.kscale + r), "r"(kDraftPage * 4), "r"(smem_u32(&k_full[st])) : "memory");
          }
        }
        if (!ok) break;
        __syncwarp();
        if (lane == 0) mbar_arrive(&w_empty[ub]);
      }
      if (lane == 0 && *abort_flag) {               // on abort, give copies already in flight a bounded chance to land
        for (int st = 0; st < C::STAGES; ++st)
          for (uint32_t spin = 0; spin < (1u << 16) && !mbar_try_wait(&k_full[st], 0) && !mbar_try_wait(&k_full[st], 1); ++spin) {
          }
      }
    } else if (warp == 1) {
      // ------------------------------- MMA issuer -------------------------------
      constexpr uint32_t idesc = umma_idesc(0, 0, 0, 0, kDraftKeys, C::N);
      uint32_t it = 0;
      for (uint32_t nu = 0;; ++nu) {
        const int ub = nu & 1;
        bool ok = mbar_wait_warp(&w_full[ub], (nu >> 1) & 1, abort_flag, a.status);
        if (!ok) break;
        const int n = __shfl_sync(0xffffffffu, unit_s[ub].t_hi - unit_s[ub].t_lo, 0), more = __shfl_sync(0xffffffffu, unit_s[ub].t_lo, 0);
        if (more < 0) break;
        if (lane == 0) mbar_arrive(&w_empty[ub]);
        ok = mbar_wait_warp(&q_full[ub], (nu >> 1) & 1, abort_flag, a.status);
        const uint64_t qdesc = umma_smem_desc(smem_u32(q_s + ub * C::Q_TILE_BYTES), 16, 1024, kSwz128);
        for (int t = 0; t < n && ok; ++t, ++it) {
          const int st = it % C::STAGES, acc = it & 1;
          ok = mbar_wait_warp(&k_full[st], (it / C::STAGES) & 1, abort_flag, a.status) &&
               mbar_wait_warp(&acc_empty[acc], ((it >> 1) & 1) ^ 1, abort_flag, a.status);
          if (!ok) break;
          tc_fence_after();
          const uint64_t kdesc = umma_smem_desc(smem_u32(k_s + st * C::K_TILE_BYTES), 16, 1024, kSwz128);
          if (elect_one()) {
#pragma unroll
            for (int sub = 0; sub < C::SUB; ++sub)
#pragma unroll
              for (int k = 0; k < C::KSTEPS; ++k)
                umma_f8(tmem_base + acc * C::COLS + sub * C::N, kdesc + (sub * kDraftKeys * 128 >> 4) + (k * 32 >> 4), qdesc + (k * 32 >> 4), idesc, k > 0);
            umma_commit(&acc_full[acc]);
            umma_commit(&k_empty[st]);
          }
          __syncwarp();
        }
        if (!ok) break;
        if (elect_one()) umma_commit(&q_empty[ub]);
        __syncwarp();
      }
    } else if (warp == 2) {
      // ------------------- stager: what the other roles need of the next unit, so that none of them waits for global memory -------------------
      uint32_t nu = 0;
      bool ok = true;
      for (int u = blockIdx.x; u < n_units && !aborted_warp(abort_flag); u += gridDim.x) {
        DraftUnit x;
        bool live, bad;
        const bool work = draft_unit<C::TILE_KEYS, NT>(a, u, groups, chunk, x, live, bad);
        if (bad && lane == 0 && a.status) atomicCAS(a.status, kStatusOk, kStatusBadIndex);
        if (!work || !live) continue;
        const int ub = nu & 1;
        const int64_t off = (int64_t)(x.b * a.drafts.per_seq + x.g * NT) * H;
        const int left = (a.drafts.per_seq - x.g * NT) * H;           // values of the sequence's drafts from here on; zeros behind
        constexpr int kRounds = (C::N + 31) / 32, kPages = (C::PAGES * kDraftChunk + 31) / 32;
        float v[kRounds];
        int pr[kPages];
#pragma unroll
        for (int i = 0; i < kRounds; ++i) {
          const int e = lane + 32 * i;
          v[i] = e >= left || e >= C::N ? 0.f : a.w_is_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(a.w)[off + e]) : static_cast<const float*>(a.w)[off + e];
        }
        const int n_pages = (x.P + x.m + kDraftPage - 1) / kDraftPage;
#pragma unroll
        for (int i = 0; i < kPages; ++i) {
          const int page = C::PAGES * x.t_lo + lane + 32 * i;
          pr[i] = page < n_pages && lane + 32 * i < C::PAGES * (x.t_hi - x.t_lo) ? __ldg(a.block_table + (int64_t)x.b * a.table_stride + page) : -2;
        }
        uint64_t bits = 0;
        const int d = x.g * NT + lane;
        if (lane < NT && d < x.m && a.drafts.tree) bits = draft_mask(a.drafts, x.b, d);
        if (!mbar_wait_warp(&w_empty[ub], ((nu >> 1) & 1) ^ 1, abort_flag, a.status)) {
          ok = false;
          break;
        }
#pragma unroll
        for (int i = 0; i < kRounds; ++i)
          if (lane + 32 * i < C::N) w_s[ub * C::N + lane + 32 * i] = v[i];
        bool holes = false;
#pragma unroll
        for (int i = 0; i < kPages; ++i) {
          int r = -1;
          holes |= pr[i] != -2 && (pr[i] < 0 || pr[i] >= a.num_pages);
          if (pr[i] >= 0 && pr[i] < a.num_pages) r = pr[i] * kDraftPage;
          else if (pr[i] != -2 && a.status) atomicCAS(a.status, kStatusOk, kStatusBadIndex);
          if (lane + 32 * i < C::PAGES * kDraftChunk) pages_s[ub * C::PAGES * kDraftChunk + lane + 32 * i] = r;
        }
        if (lane < NT) unit_s[ub].bits[lane] = bits;
        holes = __any_sync(0xffffffffu, holes);
        if (lane == 0) {
          DraftUnit& to = unit_s[ub];
          to.b = x.b; to.g = x.g; to.t_lo = x.t_lo; to.t_hi = x.t_hi;
          to.P = x.P; to.m = x.m; to.columns = x.columns; to.holes = holes;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&w_full[ub]);
        ++nu;
      }
      if (ok && mbar_wait_warp(&w_empty[nu & 1], ((nu >> 1) & 1) ^ 1, abort_flag, a.status) && lane == 0) {
        unit_s[nu & 1].t_lo = -1;
        mbar_arrive(&w_full[nu & 1]);
      }
    } else {
      // ------------------- groups without a draft: -inf -------------------
      for (int u = blockIdx.x; u < n_units; u += gridDim.x) {
        DraftUnit x;
        bool live, bad;
        if (!draft_unit<C::TILE_KEYS, NT>(a, u, groups, chunk, x, live, bad) || live) continue;
        for (int i = x.g * NT; i < min(x.g * NT + NT, a.drafts.per_seq); ++i)
          for (int s = x.t_lo * C::TILE_KEYS + lane; s < min(x.t_hi * C::TILE_KEYS, x.columns); s += 32)
            a.logits[((int64_t)x.b * a.drafts.per_seq + i) * a.ld + s] = -CUDART_INF_F;
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::REGS_EPI));
    // ------------- epilogue: warpgroup = draft of the group and 128 keys of the tile, thread = key -------------
    const int wg = (warp - 4) >> 2, tok = wg % NT, sub = wg / NT;
    const int wq = warp & 3, row = wq * 32 + lane;
    const uint32_t t_lane = tmem_base + (uint32_t(wq * 32) << 16) + wg * H;
    uint32_t it = 0;
    int sc = 0;                                  // slot of the scales' ring
    bool ok = true;
    for (uint32_t nu = 0; ok; ++nu) {
      const int ub = nu & 1;
      ok = mbar_wait_warp(&w_full[ub], (nu >> 1) & 1, abort_flag, a.status);
      if (!ok) break;
      const DraftUnit& x = unit_s[ub];
      const int t_lo = x.t_lo, t_hi = x.t_hi;
      if (t_lo < 0) break;
      uint64_t wreg[H / 2];                      // this draft's head weights as packed pairs, for the whole unit
      {
        const float4* src = reinterpret_cast<const float4*>(w_s + ub * C::N + tok * H);
#pragma unroll
        for (int j = 0; j < H / 4; ++j) {
          const float4 w4 = src[j];
          wreg[2 * j] = pack_f32x2(w4.x, w4.y);
          wreg[2 * j + 1] = pack_f32x2(w4.z, w4.w);
        }
      }
      const int i = x.g * NT + tok, P = x.P;
      const int columns = i < a.drafts.per_seq ? x.columns : 0;
      const int plain = i >= x.m ? 0 : a.drafts.tree ? P : P + i + 1;      // positions before are all seen, of those behind the bits'
      const int easy = x.holes ? -1 : min(plain, columns) - 32;            // a warp whose first column is no further writes all of its scores
      float* out = a.logits + ((int64_t)x.b * a.drafts.per_seq + i) * a.ld + row;
      int s0 = t_lo * C::TILE_KEYS + sub * kDraftKeys;
      for (int n = t_hi - t_lo; n > 0; --n, ++it, s0 += C::TILE_KEYS) {
        const int stage = it & 1;
        ok = mbar_wait_warp(&acc_full[stage], (it >> 1) & 1, abort_flag, a.status);
        if (!ok) break;
        tc_fence_after();
        const uint32_t t_acc = t_lane + stage * C::COLS;
        uint32_t v[2][16];
        uint64_t chain[2];
        tmem_ld16(t_acc, v[0]);
        const float kscale = scale_s[sc * C::TILE_KEYS + sub * kDraftKeys + row];      // there since the MMAs began; read before the accumulator is given back
        if (++sc == C::SCALES) sc = 0;
#pragma unroll
        for (int c = 0; c < H; c += 16) {
          const int cur = (c >> 4) & 1;
          tmem_wait_ld();
          if (c + 16 < H) tmem_ld16(t_acc + c + 16, v[cur ^ 1]);
#pragma unroll
          for (int j = 0; j < 16; j += 2) {
            const int hp = (c + j) >> 1;               // head pair
            const float d0 = __saturatef(__uint_as_float(v[cur][j]) * kDraftRelu);
            const float d1 = __saturatef(__uint_as_float(v[cur][j + 1]) * kDraftRelu);
            if (hp < 2) chain[hp] = 0;
            chain[hp & 1] = fma_f32x2(pack_f32x2(d0, d1), wreg[hp], chain[hp & 1]);
          }
        }
        float e0, o0, e1, o1;
        unpack_f32x2(chain[0], e0, o0);
        unpack_f32x2(chain[1], e1, o1);
        const float score = (((0.f + (e0 + o0)) + (e1 + o1)) * (1.f / kDraftRelu)) * kscale;
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&acc_empty[stage]);   // the accumulator slice and the scale have been used
        if (s0 + wq * 32 <= easy) {
          out[s0] = score;
        } else {
          const int s = s0 + row;
          if (s < columns) {
            bool in = s < plain || (s >= P && s - P < kMaxTreeDrafts && (unit_s[ub].bits[tok] >> (s - P) & 1));
            if (unit_s[ub].holes && in) in = pages_s[ub * C::PAGES * kDraftChunk + (s >> 6) - unit_s[ub].t_lo * C::PAGES] >= 0;
            out[s0] = in ? score : -CUDART_INF_F;
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&w_empty[ub]);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, C::TMEM_COLS);
  }
}

int make_tmap_2d_u8(CUtensorMap* m, const void* base, uint64_t rows, uint32_t row_bytes, uint64_t row_pitch, uint32_t box_rows);

template <int H, int NT>
static int launch_draft_logits(const DraftLogitsArgs& a, cudaStream_t stream) {
  using C = DraftCfg<H, NT>;
  CUtensorMap tq, tk;
  int rc = make_tmap_2d_u8(&tq, a.q, (uint64_t)a.B * a.drafts.per_seq * H, 128, 128, C::N);
  if (!rc) rc = make_tmap_2d_u8(&tk, a.kcache, (uint64_t)a.num_pages * kDraftPage, 128, 128, kDraftPage);
  if (rc) return rc;
  const int groups = (a.drafts.per_seq + NT - 1) / NT, tiles = (a.drafts.max_ctx + C::TILE_KEYS - 1) / C::TILE_KEYS;
  // Tiles of a unit: the most of 1 .. kDraftChunk that leaves the CTA with most to do least, counting a unit's start as one tile.
  const auto units = [&](int c) { return (int64_t)a.B * groups * ((tiles + c - 1) / c); };
  const auto cost = [&](int c) { return (units(c) + sm_count() - 1) / sm_count() * (min(c, tiles) + 1); };
  int chunk = kDraftChunk;
  for (int c = kDraftChunk - 1; c >= 1; --c)
    if (cost(c) < cost(chunk)) chunk = c;
  if (units(chunk) > 0x7fffffff) return set_error(DSA_ERR_SHAPE, "indexer_logits_drafts: too many work units");
  const int n_units = (int)units(chunk);
  auto kern = draft_logits_kernel<H, NT>;
  static uint64_t allowed = 0;
  if (!allow_smem(reinterpret_cast<const void*>(kern), C::SMEM_BYTES, &allowed))
    return set_error(DSA_ERR_CUDA, "indexer_logits_drafts: cannot raise dynamic shared memory to %d", C::SMEM_BYTES);
  kern<<<min(n_units, sm_count()), C::THREADS, C::SMEM_BYTES, stream>>>(tq, tk, a, groups, chunk, n_units);
  return check_launch("indexer_logits_drafts");
}
// Drafts of a group: as few places as possible without a draft, then as many as possible.
template <int H>
static int launch_draft_logits(const DraftLogitsArgs& a, cudaStream_t stream) {
  const int n = a.drafts.per_seq;
  if (n == 1) return launch_draft_logits<H, 1>(a, stream);
  return (n + 1) / 2 * 2 < (n + 3) / 4 * 4 ? launch_draft_logits<H, 2>(a, stream) : launch_draft_logits<H, 4>(a, stream);
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
  if (num_pages == 0) return set_error(DSA_ERR_SHAPE, "indexer_logits_drafts: an empty cache");
  if (H == 64) return launch_draft_logits<64>(a, stream);
  return H == 32 ? launch_draft_logits<32>(a, stream) : launch_draft_logits<16>(a, stream);
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
// What a row does not see has the lowest score there is, and is selected where too few others are higher: where the row sees fewer positions than it has slots, or has
// scores that are no numbers.  Those become empty slots: drafts by the row's mask, whatever their scores are, and positions of pages that are none by theirs, which only the
// scores tell of.  It starts under the selection's end, and a thread has eight slots' scores under way (256 rows of 2048 slots at 128K: 4 us behind the selection's 39).
__global__ void __launch_bounds__(256) draft_unsee_kernel(const float* __restrict__ logits, int64_t ld, const DraftArgs d, int k, int32_t* idx) {
  constexpr int kAhead = 8;
  const int r = blockIdx.x, b = r / d.per_seq, i = r - b * d.per_seq;
  const Drafts dr = drafts_of(d, b);
  const int P = dr.ctx - dr.m;
  const uint64_t bits = d.tree ? draft_mask(d, b, i) : 0;
  const float* scores = logits + (int64_t)r * ld;
  int32_t* row = grid_wait(idx) + (int64_t)r * k;      // (no block goes before: what comes next waits for this kernel)
  if (i >= dr.m) return;
  for (int j0 = threadIdx.x; j0 < k; j0 += 256 * kAhead) {
    int at[kAhead];
    float score[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) at[u] = j0 + 256 * u < k ? row[j0 + 256 * u] : -1;
#pragma unroll
    for (int u = 0; u < kAhead; ++u) score[u] = at[u] >= 0 ? __ldg(scores + at[u]) : 0.f;
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const bool other = d.tree && at[u] >= P && !(bits >> (at[u] - P) & 1);     // at - P <= i < 64
      if (at[u] >= 0 && (other || score[u] == -CUDART_INF_F)) row[j0 + 256 * u] = -1;
    }
  }
}

int topk_select_launch(const float* logits, int64_t ld, const int32_t* ks, const int32_t* ke, int T, int S, int k, int32_t* out, int sample, int overlapped,
                       cudaStream_t stream);

int topk_select_drafts_launch(const float* logits, int64_t ld, const int32_t* ctx_len, const int32_t* n_new, const int64_t* tree, int tokens_per_seq, int B,
                              int max_ctx, int k, int32_t* out, int32_t* ends, cudaStream_t stream) {
  const DraftArgs d{ctx_len, n_new, tree, tokens_per_seq, max_ctx};
  const int T = B * tokens_per_seq;
  if (max_ctx == 0) {
    cudaMemsetAsync(out, 0xff, (size_t)T * k * sizeof(int32_t), stream);
    return check_launch("topk_select_drafts");
  }
  draft_ends_kernel<<<(T + 255) / 256, 256, 0, stream>>>(d, T, ends);
  int rc = check_launch("topk_select_drafts");
  if (!rc) rc = topk_select_launch(logits, ld, nullptr, ends, T, max_ctx, k, out, /*sample=*/1, /*overlapped=*/0, stream);
  if (rc || k == 0) return rc;
  launch_after(1, draft_unsee_kernel, dim3(T), 256, 0, stream, logits, ld, d, k, out);
  return check_launch("topk_select_drafts");
}

}  // namespace dsa
