// MLA attention over a sliding window and the first tokens (MQA over the shared 576-dim latent KV, 512-dim V): a query row at position p of its
// sequence sees the positions < first and the last `window` ones, p itself included,
//   o[r, :] = sum_s softmax_s(scale * q[r, :] . kv[s, :]) * kv[s, :512],   s < first or p - window < s <= p,
// here over the records of the paged latent caches: decode, one or several query tokens a sequence, a chain or a tree of drafts (drafts.cuh).  Prompts:
// window_prompt.cu.
//
// A unit is up to 128 query rows (token, head) of one sequence, and its keys are the union of what they see, as slots: the first tokens, then the window's,
// then the drafts.  Rows of one sequence share the fetch and the conversion of their records, which is why a unit has several tokens where heads are few.  A pair
// of CTAs has a unit, each half of the latent dims (sparse_mla.cu): whole, O of 128 rows and 512 dims and S, P and Q of 576 do not fit one SM's tensor memory.
// What bounds it: a block of 64 slots takes a pair 1.8 us from FP8 records and 1.5 from 4 bits, the chain of conversion, exchange (32 KB either way), softmax and
// P.V with half of the issue slots used (74 sequences x 128 heads, FP8, window 2048: 80 us under the profiler, issue slots 47 %, tensor pipe 26 %, DRAM 18 %).  64
// sequences x 128 heads at 128K, window 4096: 136 to 139 us for 29 us of bytes and 45 of operations; 160 x 4 drafts x 16 heads, 4 bits, window 1024: 75 to 78 us,
// of which a unit's start, a chain of lengths, pages, records and its first scores, takes 6 and its end 2 in each of three rounds.
#include <cuda.h>
#include <cudaTypedefs.h>

#include "window_mla.cuh"

namespace dsa {

// ---- the pair kernel ---------------------------------------------------------------------------------------------------
template <int SRC>
struct WinCfg {
  static constexpr int kBufs = kMlaBufs - 1;           // the fifth one's space holds raw rows
  static constexpr int kOffBars = kMlaBufs * kMlaKBytes + kWinXBytes;
  static constexpr int kOffValid = kOffBars + 640;
  static constexpr int kOffPm = kOffValid + kMlaValidRing * kMlaBlk;
  static constexpr int kOffSees = kOffPm + kMlaPairBytes;             // int4 a row
  static constexpr int kOffMore = kOffSees + 128 * 16;                // 8 bytes a row: the drafts it sees
  static constexpr int kOffRaw = kOffMore + 128 * 8;
  static constexpr int kSmem = kOffRaw + (MlaRaw<SRC>::kPieces - MlaRaw<SRC>::kInBuf) * MlaRaw<SRC>::kBytes;
  static_assert(kSmem <= 232448 && kOffRaw % 16 == 0, "shared memory budget of one CTA");
};

template <int SRC>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kMlaThreads, 1)
window_mla_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_o, const WinArgs a) {
  using C = WinCfg<SRC>;
  constexpr int NB = C::kBufs;
  extern __shared__ __align__(1024) uint8_t smem[];            // the swizzled panels need 1024-byte alignment
  launch_dependents();                                         // (the kernel that merges the parts)
  uint8_t* kv_s = smem;                                        // five buffers: four panels [64 keys x 128 B] and 64 x 64 B
  uint8_t* recv_s = kv_s + kMlaBufs * kMlaKBytes;              // the peer's partial score tile
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kOffBars);      // as in sparse_mla.cu
  uint64_t *q_full = bars + 0, *q_moved = bars + 1, *o_final = bars + 2, *s_free = bars + 3, *p_full = bars + 4, *s_full = bars + 5, *pv_done = bars + 7,
           *pm_full = bars + 9, *recv_full = bars + 17, *xchg_free = bars + 33, *kv_full = bars + 49, *kv_free = bars + 54;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 64);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  uint32_t* odd_s = tmem_slot + 2;                             // [4 quadrants] rows with a key that they do not see and that is no number
  volatile uint32_t* lost_s = odd_s + 4;                       // [4 quadrants] a warp of it has given up
  uint8_t* valid_s = smem + C::kOffValid;                      // decode: [kMlaValidRing][64] 1 = the slot of the block has a page
  uint16_t* pm_s = reinterpret_cast<uint16_t*>(smem + C::kOffPm);        // block maxima, rounded up to bf16
  int4* sees_s = reinterpret_cast<int4*>(smem + C::kOffSees);
  uint64_t* more_s = reinterpret_cast<uint64_t*>(smem + C::kOffMore);

  const int cta = blockIdx.x & 1, peer = cta ^ 1;              // rank in the cluster = V half = contraction part
  const int job = blockIdx.x >> 1;
  const int part = job < a.n_full ? -1 : job - a.n_full;       // >= 0: a part of a unit's keys
  const int n_split = part < 0 ? 1 : a.n_split, nth = part < 0 ? 0 : part / n_split, unit = part < 0 ? job : a.n_full + nth, split = part < 0 ? 0 : part - nth * n_split;
  const int warp = warp_index(), lane = threadIdx.x & 31;
  const int seq = a.seq_units == 1 ? unit : unit / a.seq_units;      // (divisions stand before the first load)
  const int row0 = (unit - seq * a.seq_units) * a.unit_rows;   // of the sequence's query rows
  const int rows_here = min(a.unit_rows, a.seq_rows - row0);
  const int64_t g0 = (int64_t)seq * a.seq_rows + row0;
  const int n_quad = (rows_here + 31) / 32;                    // quadrants of tensor memory with rows in them: the others' warps stand by
  const int tok0 = row0 == 0 ? 0 : row0 / a.H, tok1 = a.seq_units == 1 ? a.drafts.per_seq - 1 : (row0 + rows_here - 1) / a.H;
  // the five Q panels wait at the end of the KV buffers (from buffer kQBuf0 on) for their move into tensor memory
  constexpr int kQStage = NB * kMlaKBytes - kMlaPanels * kMlaQPanelBytes, kQBuf0 = kQStage / kMlaKBytes;
  static_assert(kQStage >= 0 && kQStage % 1024 == 0, "Q staging");
  auto q_stage = [&](int lp) -> uint8_t* { return kv_s + kQStage + lp * kMlaQPanelBytes; };

  // ---- set-up ----------------------------------------------------------------------------------------------------------
  if (warp == 0) {
    for (int i = lane; i < 59; i += 32) {
      const uint32_t count = i == 1 ? 16u                                            // q_moved: lane 0 of the softmax warps
                             : (i == 3 || i == 4) ? 2u * n_quad                      // s_free, p_full: lane 0 of a set's warps
                             : (i >= 9 && i <= 16) ? 2u                              // pm_full: the two warps of a quadrant
                             : (i >= 49 && i <= 53) ? uint32_t(kMlaGatherWarps)
                                                    : 1u;                   // the others
      mbar_init(bars + i, count);
    }
    mbar_fence_init();
    if (lane < 9) const_cast<int*>(abort_flag)[lane] = 0;      // and odd_s, lost_s
    __syncwarp();
    if (lane == 0) mbar_expect_tx(q_full, kMlaPanels * kMlaQPanelBytes);
    __syncwarp();
    if (lane < kMlaPanels)                             // x in 4-byte units: 32 per panel
      tma_load_2d(q_stage(lane), &tmap_q, (lane < 4 ? cta * 4 + lane : 8) * 32, (int)g0, q_full);
    if (lane == kMlaPanels && a.tma_out) tma_prefetch_desc(&tmap_o);
  } else if (warp == kMlaMmaWarp) {
    tmem_alloc(tmem_slot, kMlaTmemCols);
    tmem_relinquish();
  }
  const Drafts dr = drafts_of(a.drafts, seq);
  if (dr.bad && threadIdx.x == 0 && a.status) atomicCAS(a.status, kStatusOk, kStatusBadIndex);
  const Slots sl = slots_of(a, dr, tok0, tok1);
  const int head = sl.head, shift = sl.shift, n_slots = sl.n, full0 = sl.full0, full1 = sl.full1;
  const int blocks = (n_slots + kMlaBlk - 1) / kMlaBlk;
  const int per = (blocks + n_split - 1) / n_split, blk_lo = min(blocks, split * per), nblk = min(blocks, blk_lo + per) - blk_lo;
  // The records of 64 slots a block, each gather warp every eleventh: raw into shared memory two blocks ahead (cp.async), then to bf16.  The first two
  // blocks are sent for before anything of the set-up is waited for: a page's entry and a record are two times the way to memory.
  constexpr int kG = kMlaGatherWarps, kRows = kRawRows, kRawRow = MlaRaw<SRC>::kRow, kRawBytes = MlaRaw<SRC>::kBytes, kRawInBuf = MlaRaw<SRC>::kInBuf;
  constexpr int kBytes = SRC == kSrc4 ? kLatent4Bytes : kLatentTokenBytes;
  const int w4 = warp - kMlaGatherWarp0;
  const int slot = warp >= kMlaGatherWarp0 && lane < kRows ? w4 + lane * kG : kMlaBlk;      // lane j < 6 looks after slot w4 + 11 j
  const int32_t* table = a.block_table + (int64_t)seq * a.table_stride;
  auto position = [&](int i) -> int {
    const int j = (blk_lo + i) * kMlaBlk + slot;
    return slot < kMlaBlk && i < nblk && j < n_slots ? (j < head ? j : j + shift) : -1;
  };
  auto table_entry = [&](int pos) -> int { return pos >= 0 ? __ldg(table + pos / kLatentPage) : -1; };
  auto cache_row = [&](int pos, int page) -> int {   // -1 = no slot, or a page that is none: flagged
    if (pos < 0) return -1;
    if (page >= 0 && (int64_t)(page + 1) * kLatentPage <= a.num_phys_rows) return page * kLatentPage + pos % kLatentPage;
    if (a.status) atomicCAS(a.status, kStatusOk, kStatusBadIndex);
    return -1;
  };
  auto stage_of = [&](int i) -> uint8_t* {           // the fifth KV buffer, and what does not fit there behind everything else
    const int c = (i & 1) * kG + w4;
    return c < kRawInBuf ? kv_s + NB * kMlaKBytes + c * kRawBytes : smem + C::kOffRaw + (c - kRawInBuf) * kRawBytes;
  };
  auto fetch = [&](int i, int id) {                  // an empty slot is zero-filled, values and scales
    uint8_t* st = stage_of(i);
    if constexpr (SRC == kSrc4) {
#pragma unroll
      for (int u = 0; u < (kRows * 13 + 31) / 32; ++u) {         // 208 bytes a row: thirteen pieces
        const int c = u * 32 + lane, j = c / 13, rid = __shfl_sync(0xffffffffu, id, min(j, kRows - 1));
        if (c < kRows * 13)
          cp_async_16(st + c * 16, a.kv + (int64_t)max(rid, 0) * kBytes + cta * kLatent4Half + (c - j * 13) * 16, rid >= 0 ? 16 : 0);
      }
    } else {
#pragma unroll
      for (int u = 0; u < kRows / 2; ++u) {        // two rows of 256 values per instruction
        const int j = 2 * u + (lane >> 4), rid = __shfl_sync(0xffffffffu, id, j);
        cp_async_16(st + j * kRawRow + (lane & 15) * 16, a.kv + cta * kMlaDvHalf + (lane & 15) * 16 + (int64_t)max(rid, 0) * kBytes, rid >= 0 ? 16 : 0);
      }
      const int rid = __shfl_sync(0xffffffffu, id, lane >> 2);
      if (lane < kRows) cp_async_16(st + lane * kRawRow + 256, a.kv + kMlaDv + (int64_t)max(id, 0) * kBytes, id >= 0 ? 16 : 0);      // a row's four scales
      if (lane < 4 * kRows)                        // this CTA's two K-steps of the rope panel: 64 bytes per row
        cp_async_16(st + (lane >> 2) * kRawRow + 272 + (lane & 3) * 16, a.kv + kMlaDv + 16 + cta * 64 + (lane & 3) * 16 + (int64_t)max(rid, 0) * kBytes, rid >= 0 ? 16 : 0);
    }
    cp_async_commit();
  };
  int id_cur = -1, id_nxt = -1, pa = -1, ta = -1;      // row ids of blocks i and i+1, position and page of i+2
  if (warp >= kMlaGatherWarp0 && nblk > 0) {
    const int p0 = position(0), p1 = position(1), t0 = table_entry(p0), t1 = table_entry(p1);
    pa = position(2);
    ta = table_entry(pa);
    id_cur = cache_row(p0, t0);
    fetch(0, id_cur);
    id_nxt = cache_row(p1, t1);
    fetch(1, id_nxt);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (nblk == 0) {   // nothing seen: zeros (a part: weight zero in the combine); no cluster traffic yet
    if (part < 0) {
      for (int e = threadIdx.x; e < rows_here * 32; e += kMlaThreads)
        reinterpret_cast<uint4*>(a.out + (g0 + (e >> 5)) * kMlaDv + cta * kMlaDvHalf)[e & 31] = make_uint4(0, 0, 0, 0);
    } else if (threadIdx.x < 128) {
      a.part_lse[((int64_t)part * 2 + cta) * 128 + threadIdx.x] = -CUDART_INF_F;
    }
    if (threadIdx.x == 0) mbar_wait(q_full, 0, abort_flag, a.status);     // the Q copy must have landed before the CTA goes
    if (warp == kMlaMmaWarp) tmem_dealloc(*tmem_slot, kMlaTmemCols);
    return;
  }
  const uint32_t tmem = *tmem_slot;
  // The peer's barriers must be initialised before anything is sent to it: the softmax warps wait before their first remote access, the
  // others only before they leave.
  cluster_arrive();
  bool left = false;                                           // this warp has arrived at the barrier that the pair leaves through

  if (warp >= kMlaSoftmaxWarps) regs_dec<MlaRegs<true>::kOther>();
  else regs_inc<MlaRegs<true>::kSoftmax>();
  if (warp == kMlaMmaWarp) {
    // ------------------------------- MMA issuer: as in sparse_mla.cu -------------------------------
    constexpr uint32_t idesc_qk = umma_idesc(1, 1, 0, 0, 128, kMlaBlk);
    constexpr uint32_t idesc_pv = umma_idesc(1, 1, 0, 1, 128, kMlaDvHalf);
    bool ok = mla_wait(q_moved, 0, abort_flag, a.status);
    const uint64_t kdesc0 = umma_smem_desc(smem_u32(kv_s), 16, 1024, kSwz128);
    const uint64_t vdesc0 = umma_smem_desc(smem_u32(kv_s), kMlaKPanelBytes, 1024, kSwz128);
    const uint64_t rdesc0 = umma_smem_desc(smem_u32(kv_s + kMlaRopeOff), 16, 512, kSwz64);
    const uint32_t rope_ks = 2 * cta;                  // this CTA's two K-steps of the rope panel
    for (int n = 0; n < nblk + 2 && ok; ++n) {
      if (n < nblk) {
        const int buf = n % NB;
        ok = mla_wait(&kv_full[buf], (n / NB) & 1, abort_flag, a.status);
        if (ok && n > 0) ok = mla_wait(s_free, (n - 1) & 1, abort_flag, a.status);
        if (!ok) break;
        fence_async_smem();       // the rows were written by st, the tensor core reads through the async proxy
        tc_fence_after();
        if (elect_one()) {
          const uint64_t kd0 = kdesc0 + uint64_t(buf) * (kMlaKBytes >> 4);
#pragma unroll
          for (int lp = 0; lp < 4; ++lp)
#pragma unroll
            for (int ks = 0; ks < 4; ++ks)
              umma_f16_ts(tmem + kColS, tmem + kColQ + lp * 32 + 8 * ks, kd0 + uint64_t((lp * kMlaKPanelBytes) >> 4) + 2 * ks, idesc_qk, (lp | ks) != 0);
#pragma unroll
          for (int u = 0; u < 2; ++u)
            umma_f16_ts(tmem + kColS, tmem + kColQ + 4 * 32 + 8 * (rope_ks + u), rdesc0 + uint64_t(buf) * (kMlaKBytes >> 4) + 2 * u, idesc_qk, 1);
          umma_commit(&s_full[n & 1]);
        }
        __syncwarp();
      }
      if (n >= 2) {
        ok = mla_wait(p_full, n & 1, abort_flag, a.status);
        if (!ok) break;
        const int j = n - 2;
        tc_fence_after();
        if (elect_one()) {
          const uint64_t vd = vdesc0 + uint64_t(j % NB) * (kMlaKBytes >> 4);
#pragma unroll
          for (int ks = 0; ks < kMlaBlk / 16; ++ks)    // 16 keys per step: 16 rows x 128 B further into each panel
            umma_f16_ts(tmem + kColO, tmem + kColP + 8 * ks, vd + ks * (2048 >> 4), idesc_pv, (j | ks) != 0);
          umma_commit(&kv_free[j % NB]);
          umma_commit(&pv_done[j & 1]);
          if (j == nblk - 1) umma_commit(o_final);
        }
        __syncwarp();
      }
    }
  } else if (warp > kMlaMmaWarp) {
    // ----------------------------- records to bf16 -----------------------------
    bool ok = true;
    auto mark = [&](int i, bool used) {
      if (slot < kMlaBlk) valid_s[(i % kMlaValidRing) * kMlaBlk + slot] = used;
    };
    const int l16 = (lane & 3) | ((lane >> 3) << 2);         // 4 bits: sixteen lanes a row, two rows at a time (sparse_mla.cu)
    for (int i = 0, buf = 0; i < nblk; ++i) {
      const int id2 = cache_row(pa, ta);             // block i+2
      pa = position(i + 3);
      ta = table_entry(pa);
      if (i == kQBuf0) ok = mla_wait(q_moved, 0, abort_flag, a.status);   // from here on the buffers held Q
      if (i >= NB) ok = mla_wait(&kv_free[buf], ((i / NB) - 1) & 1, abort_flag, a.status);
      if (!ok) break;
      mark(i, id_cur >= 0);
      id_cur = id_nxt;
      id_nxt = id2;
      cp_async_wait<1>();                            // this lane's copies of block i have landed (block i+1 may be in flight) ...
      __syncwarp();                                  // ... and the other lanes'
      const uint8_t* st = stage_of(i);
      uint8_t* dst = kv_s + buf * kMlaKBytes;
      if constexpr (SRC == kSrc4) {
#pragma unroll
        for (int u = 0; u < kRows / 2; ++u) {
          const int j = 2 * u + ((lane >> 2) & 1), r = w4 + j * kG;
          const uint2 w = *reinterpret_cast<const uint2*>(st + j * kRawRow + l16 * 8);
          const uint32_t sc = latent4_scale(st[j * kRawRow + kLatent4Scales + l16]);
          uint8_t* row = dst + (l16 >> 2) * kMlaKPanelBytes + r * 128;
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            uint32_t p[4];
            latent4_codes(x == 0 ? w.x : w.y, p);
            const uint4 v = make_uint4(mul_bf16x2(p[0], sc), mul_bf16x2(p[1], sc), mul_bf16x2(p[2], sc), mul_bf16x2(p[3], sc));
            if (r < kMlaBlk) *reinterpret_cast<uint4*>(row + ((((2 * l16 + x) ^ r) & 7) << 4)) = v;
          }
        }
      } else {
        uint8_t* dst_lat = dst + (lane >> 3) * kMlaKPanelBytes;
#pragma unroll
        for (int j = 0; j < kRows; ++j) {
          const int r = w4 + j * kG;
          const uint2 raw = *reinterpret_cast<const uint2*>(st + j * kRawRow + lane * 8);
          const float sc = *reinterpret_cast<const float*>(st + j * kRawRow + 256 + cta * 8 + (lane >> 4) * 4);
          const uint4 v = e4m3x8_to_bf16(raw, sc);
          if (r < kMlaBlk) *reinterpret_cast<uint4*>(dst_lat + r * 128 + (((lane ^ r) & 7) << 4)) = v;
        }
      }
      {
        constexpr int kRope = SRC == kSrc4 ? kLatent4Rope : 272;
        const int r = w4 + (lane >> 2) * kG;
        if (lane < 4 * kRows && r < kMlaBlk)
          *reinterpret_cast<uint4*>(dst + kMlaRopeOff + r * 64 + (((lane ^ (r >> 1)) & 3) << 4)) =
              *reinterpret_cast<const uint4*>(st + (lane >> 2) * kRawRow + kRope + (lane & 3) * 16);
      }
      __syncwarp();                                  // (the MMA warp makes the writes visible to the tensor core's reads)
      if (lane == 0) mbar_arrive(&kv_full[buf]);
      fetch(i + 2, id2);                             // into the stage just read: what was loaded from it has been stored
      if (++buf == NB) buf = 0;
    }
    cp_async_wait_all();                             // nothing of this thread's is in flight when it leaves
  } else {
    // ------------- partial-score exchange, softmax and output: thread = (row, half of a block's keys); as in sparse_mla.cu but for the masks -------------
    const int qd = warp & 3, hf = (warp >> 2) & 1, set = warp >> 3;      // hf: key half; set: takes the blocks of that parity
    const int row = qd * 32 + lane;                    // TMEM lane
    const uint32_t t_row = tmem + (uint32_t(qd * 32) << 16);
    const uint32_t peer_xchg_free = mapa_u32(smem_u32(xchg_free + warp), peer);
    const uint32_t peer_recv_full = mapa_u32(smem_u32(recv_full + warp), peer);
    float m = -CUDART_INF_F, l = 0.f;                  // m: reference of the last block seen; l: this thread's keys only
    bool odd = false;                                  // what this row does not see is no number: P x V would let it in
    bool ok = mla_wait(q_full, 0, abort_flag, a.status);
    if (ok) {
#pragma unroll 1
      for (int hp = warp >> 2; hp < 2 * kMlaPanels; hp += 4) {
        uint32_t qv[16];
        const uint8_t* src = q_stage(hp >> 1) + row * 128;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const uint4 w = *reinterpret_cast<const uint4*>(src + ((((hp & 1) * 4 + c) ^ (row & 7)) << 4));
          qv[4 * c + 0] = w.x; qv[4 * c + 1] = w.y; qv[4 * c + 2] = w.z; qv[4 * c + 3] = w.w;
        }
        if constexpr (SRC == kSrc4) {                  // the latents come 2^-14 times what they are (latent4.cuh)
          if (hp < 8) {
#pragma unroll
            for (int i = 0; i < 16; ++i) qv[i] = mul_bf16x2(qv[i], kLatent4GainPair);
          }
        }
        tmem_st16(t_row + kColQ + hp * 16, qv);
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_moved);             // one arrival per warp
    }
    if (warp < 4) {                                    // what this quadrant's rows see, in slots
      const Sees v = row < rows_here ? sees_draft(a, dr, seq, (row0 + row) / a.H) : Sees{};
      sees_s[row] = make_int4(shift ? min(v.a1, head) : v.a1, v.b0 - shift, v.b1 - shift, v.at - shift);
      more_s[row] = v.bits;
    }
    named_bar_sync(3 + qd, 128);
    cluster_wait();
    const uint8_t* recv = recv_s + (hf * 4 + qd) * kWinXWarp + lane * 16;      // this thread's part of the set's partial tile
    const uint32_t peer_recv = mapa_u32(smem_u32(recv), peer);
    auto pm_of = [&](int blk) -> uint16_t* { return pm_s + (blk & 3) * 256 + row; };      // [key half][row]
    auto raise = [&](float m_old, float bmax) { return bmax - m_old > kMaxRaise ? bmax : m_old; };   // -inf - -inf: stays
    auto pair_max = [&](const uint16_t* pm) {
      return fmaxf(__uint_as_float(uint32_t(pm[0]) << 16), __uint_as_float(uint32_t(pm[128]) << 16));
    };
    // which of the 32 keys of this thread's half of block g this row sees
    auto seen_of = [&](int r, int g, int half) -> uint32_t {
      const int4 v = sees_s[r];
      const int k0 = g * kMlaBlk + 32 * half;
      return (range_bits(0, v.x, k0) | range_bits(v.y, v.z, k0) | draft_bits(more_s[r], v.w, k0)) & low_bits(n_slots - k0);
    };
    if (qd < n_quad && set < nblk && lane == 0) mbar_expect_tx(&recv_full[warp], kWinXWarp);
    for (int n = qd < n_quad ? set : nblk; n < nblk && ok; n += 2) {
      const uint32_t ph = (n >> 1) & 1;
      uint32_t sv[32];                                 // this CTA's partial scores
      ok = mla_wait(&s_full[set], ph, abort_flag, a.status);
      if (!ok) break;
      tc_fence_after();
      tmem_ld32(t_row + kColS + 32 * hf, sv);
      tmem_wait_ld();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(s_free);              // the next block's scores may overwrite S now
      if (n > 0) {                                     // the peer has read block n-1
        ok = mla_wait(&xchg_free[warp ^ 8], ((n - 1) >> 1) & 1, abort_flag, a.status);
        if (!ok) break;
      }
      send_scores(peer_recv, peer_recv_full, sv);
      uint32_t seen = 0xffffffffu;
      const int k0 = (blk_lo + n) * kMlaBlk;
      const bool whole = k0 >= full0 && k0 + kMlaBlk <= full1;
      if (!whole) {
        seen = seen_of(row, blk_lo + n, hf);
        float z = 0.f;
#pragma unroll
        for (int i = 0; i < 32; ++i) z = fmaf((seen >> i) & 1u ? 0.f : __uint_as_float(sv[i]), 0.f, z);
        odd |= z != 0.f;                               // NaN
      }
      // the reference of the block before, from that block's maxima: every thread follows the whole sequence by itself
      if (n > 0) {
        ok = mla_wait(&pm_full[(set ^ 1) * 4 + qd], ((n - 1) >> 1) & 1, abort_flag, a.status);
        if (!ok) break;
      }
      const float m_own = m;                           // what l is relative to
      if (n > 0) m = raise(m, pair_max(pm_of(n - 1)));
      const float m_prev = m;
      ok = wait_scores(&recv_full[warp], ph, abort_flag, a.status);
      if (!ok) break;
      float s[32];                                     // raw scores; the (positive) scale is folded into the exponent's FMA
      add_scores(recv, sv, s);
      seen &= __ballot_sync(0xffffffffu, valid_s[(n % kMlaValidRing) * kMlaBlk + 32 * hf + lane]);
      auto largest = [&]() {
        float bm[4] = {s[0], s[1], s[2], s[3]};        // four independent chains
#pragma unroll
        for (int i = 4; i < 32; ++i) bm[i & 3] = fmaxf(bm[i & 3], s[i]);
        return fmaxf(fmaxf(bm[0], bm[1]), fmaxf(bm[2], bm[3]));
      };
      const float top = largest();                     // of every value of the tile, seen or not
      float bmax = top;
      if (__any_sync(0xffffffffu, seen != 0xffffffffu)) {
#pragma unroll
        for (int i = 0; i < 32; ++i) s[i] = (seen >> i) & 1u ? s[i] : -CUDART_INF_F;
        bmax = largest();
      }
      pm_of(n)[hf * 128] = static_cast<uint16_t>(bf16_bits_round_up(bmax * a.scale_log2e));
      __syncwarp();
      if (lane == 0) mbar_arrive(&pm_full[set * 4 + qd]);
      mbar_arrive_remote_after(peer_xchg_free, top, lane == 0);      // the peer may send into this stage again
      if (lane == 0 && n + 2 < nblk) mbar_expect_tx(&recv_full[warp], kWinXWarp);
      ok = mla_wait(&pm_full[set * 4 + qd], ph, abort_flag, a.status);
      if (!ok) break;
      m = raise(m_prev, pair_max(pm_of(n)));
      if (m != m_own && m_own != -CUDART_INF_F) l *= fast_exp2(m_own - m);      // (without a reference l is 0, or NaN, and stays so)
      bool waited_pv = n == 0;
      if (__any_sync(0xffffffffu, m != m_prev) && n > 0) {
        // O must be quiescent: P.V of the previous block has to be complete.  This thread scales its half of the columns.
        ok = mla_wait(&pv_done[set ^ 1], ((n - 1) >> 1) & 1, abort_flag, a.status);
        if (!ok) break;
        waited_pv = true;
        tc_fence_after();
        const float alpha = m != m_prev ? fast_exp2(m_prev - m) : 1.f;
#pragma unroll 1
        for (int c = hf * (kMlaDvHalf / 2); c < (hf + 1) * (kMlaDvHalf / 2); c += 16) {
          uint32_t ov[16];
          tmem_ld16(t_row + kColO + c, ov);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 16; ++i) ov[i] = __float_as_uint(__uint_as_float(ov[i]) * alpha);
          tmem_st16(t_row + kColO + c, ov);
        }
      }
      const float m_eff = (m == -CUDART_INF_F) ? 0.f : m;
      uint32_t pk[16];
      const uint64_t scale2 = pack_f32x2(a.scale_log2e, a.scale_log2e), m2 = pack_f32x2(-m_eff, -m_eff);
      float ps[4] = {0.f, 0.f, 0.f, 0.f};              // sums of the even and odd keys, two chains each
#pragma unroll
      for (int i = 0; i < 32; i += 2) {
        float x0, x1;
        unpack_f32x2(fma_f32x2(pack_f32x2(s[i], s[i + 1]), scale2, m2), x0, x1);
        const float p0 = fast_exp2(x0), p1 = fast_exp2(x1);
        pk[i >> 1] = pack_bf16x2(p0, p1);
        add_bf16x2(pk[i >> 1], ps[i & 2], ps[(i & 2) + 1]);
      }
      l += (ps[0] + ps[1]) + (ps[2] + ps[3]);
      if (!waited_pv) {                                // P is single-buffered: P.V of the previous block must be done
        ok = mla_wait(&pv_done[set ^ 1], ((n - 1) >> 1) & 1, abort_flag, a.status);
        if (!ok) break;
        tc_fence_after();
      }
      tmem_st16(t_row + kColP + 16 * hf, pk);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_full);
    }
    if (ok) cluster_arrive();                          // nothing remote is left to do for this warp: the others need not wait for its output
    left = ok;
    if (ok) ok = mla_wait(o_final, 0, abort_flag, a.status);
    // A full unit leaves through shared memory and TMA stores: four [128 rows x 128 B] panels in the (now idle) first two KV buffers.
    const bool by_tma = a.tma_out && part < 0 && rows_here == 128;
    // the row sum over all keys: the four threads of a row add theirs, relative to the later reference, through the idle third KV buffer
    // (every warp comes to the barrier, whatever became of its waits)
    float2* sum_s = reinterpret_cast<float2*>(kv_s + 2 * kMlaKBytes);
    const int quarter = warp >> 2;                     // which quarter of the row's columns this thread writes
    const int4 mine = sees_s[row];
    const bool any = mine.x > 0 || mine.z > mine.y || more_s[row] != 0;      // the row sees something
    if (ok) sum_s[quarter * 128 + row] = make_float2(m, l);
    const uint32_t odds = __ballot_sync(0xffffffffu, odd && any && row < rows_here);
    if (odds && lane == 0) atomicOr(odd_s + qd, odds);
    if (!ok && lane == 0) lost_s[qd] = 1;
    named_bar_sync(3 + qd, 128);
    ok = lost_s[qd] == 0;                              // the same for the quadrant's four warps: there are barriers behind, and sums of all four
    uint32_t again = 0;                                // rows of the quadrant that have to be done again
    __nv_bfloat16* const orow = a.out + (g0 + row) * kMlaDv + cta * kMlaDvHalf;
    const int64_t prow = (int64_t)part * 128 + row;
    if (ok) {
      tc_fence_after();
      float mt = -CUDART_INF_F;
#pragma unroll
      for (int u = 0; u < 4; ++u) mt = fmaxf(mt, sum_s[u * 128 + row].x);
      l = 0.f;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const float2 ml = sum_s[u * 128 + row];
        l += ml.x != -CUDART_INF_F ? ml.y * fast_exp2(ml.x - mt) : ml.y;
      }
      // A key that a row does not see and that is no number has come in through 0 x NaN, unless the row is none anyway.
      again = __ballot_sync(0xffffffffu, (odd_s[qd] >> lane & 1u) && l == l);
      if (!any) l = 0.f;                               // a block that every other row sees is not masked
      const float inv = l > 0.f ? (SRC == kSrc4 ? kLatent4Gain : 1.f) / l : l;      // (a NaN stays one)
      if (part >= 0 && quarter == 0)                   // what this CTA's half of the columns is weighted with
        a.part_lse[((int64_t)part * 2 + cta) * 128 + row] = l > 0.f ? mt + log2f(l) : l == 0.f ? -CUDART_INF_F : l;
#pragma unroll 1
      for (int c = quarter * (kMlaDvHalf / 4); c < (quarter + 1) * (kMlaDvHalf / 4); c += 32) {
        uint32_t ov[32];
        tmem_ld32(t_row + kColO + c, ov);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 32; ++i) ov[i] = __float_as_uint(any ? __uint_as_float(ov[i]) * inv : 0.f);
        if (row < rows_here && part >= 0) {
          float4* po = reinterpret_cast<float4*>(a.part_o + prow * kMlaDv + cta * kMlaDvHalf + c);
#pragma unroll
          for (int i = 0; i < 32; i += 4)
            po[i >> 2] = make_float4(__uint_as_float(ov[i]), __uint_as_float(ov[i + 1]), __uint_as_float(ov[i + 2]), __uint_as_float(ov[i + 3]));
        } else if (row < rows_here) {
          uint8_t* prow_s = kv_s + (c >> 6) * kMlaQPanelBytes + row * 128;
          const int ch0 = (c & 63) >> 3;               // first of this iteration's four 16-byte chunks in the 128-byte row
#pragma unroll
          for (int i = 0; i < 32; i += 8) {
            uint4 w;
            w.x = pack_bf16x2(__uint_as_float(ov[i + 0]), __uint_as_float(ov[i + 1]));
            w.y = pack_bf16x2(__uint_as_float(ov[i + 2]), __uint_as_float(ov[i + 3]));
            w.z = pack_bf16x2(__uint_as_float(ov[i + 4]), __uint_as_float(ov[i + 5]));
            w.w = pack_bf16x2(__uint_as_float(ov[i + 6]), __uint_as_float(ov[i + 7]));
            if (by_tma) *reinterpret_cast<uint4*>(prow_s + (((ch0 + (i >> 3)) ^ (row & 7)) << 4)) = w;
            else *reinterpret_cast<uint4*>(orow + c + i) = w;
          }
        }
      }
    }
    if (again) {
      // Rare: these rows, each by a warp, key by key over what they see of this part: this CTA's half of the output from whole scores.
      named_bar_sync(3 + qd, 128);                     // what the four warps have written of them is overwritten
      constexpr int kBytes = SRC == kSrcFp8 ? kLatentTokenBytes : kLatent4Bytes;
#pragma unroll 1
      for (int nth = 0; again; again &= again - 1, ++nth) {
        if ((nth & 3) != quarter) continue;
        const int r = qd * 32 + __ffs(again) - 1;
        const RowShare q = load_share<kSrcRows>(reinterpret_cast<const uint8_t*>(a.q + (g0 + r) * kMlaDqk), lane);
        float rm = -CUDART_INF_F, rl = 0.f, o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
        for (int n = 0; n < 2 * nblk; ++n) {
          const int g = blk_lo + (n >> 1);
          uint32_t todo = seen_of(r, g, n & 1);
#pragma unroll 1
          for (; todo; todo &= todo - 1) {
            const int j = g * kMlaBlk + 32 * (n & 1) + __ffs(todo) - 1, pos = j < head ? j : j + shift;
            const int page = __ldg(a.block_table + (int64_t)seq * a.table_stride + pos / kLatentPage);
            if (page < 0 || (int64_t)(page + 1) * kLatentPage > a.num_phys_rows) continue;
            const int64_t key = (int64_t)page * kLatentPage + pos % kLatentPage;
            const RowShare k = load_share<SRC>(a.kv + key * kBytes, lane);
            const float s = row_score(q, k, a.scale_log2e), mx = fmaxf(rm, s), at = mx == -CUDART_INF_F ? 0.f : mx;
            const float keep = rm == -CUDART_INF_F ? 0.f : exp2f(rm - at), p = exp2f(s - at);
            rm = mx;
            rl = rl * keep + p;
#pragma unroll
            for (int i = 0; i < 8; ++i) o[i] = o[i] * keep + p * (cta ? k.x[1][i] : k.x[0][i]);
          }
        }
        const float inv = rl > 0.f ? 1.f / rl : rl;    // (a NaN stays one)
        const uint4 w = make_uint4(pack_bf16x2(o[0] * inv, o[1] * inv), pack_bf16x2(o[2] * inv, o[3] * inv), pack_bf16x2(o[4] * inv, o[5] * inv),
                                   pack_bf16x2(o[6] * inv, o[7] * inv));
        if (part >= 0) {
          float4* po = reinterpret_cast<float4*>(a.part_o + ((int64_t)part * 128 + r) * kMlaDv + cta * kMlaDvHalf + lane * 8);
          po[0] = make_float4(o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
          po[1] = make_float4(o[4] * inv, o[5] * inv, o[6] * inv, o[7] * inv);
          if (lane == 0) a.part_lse[((int64_t)part * 2 + cta) * 128 + r] = rl > 0.f ? rm + log2f(rl) : rl == 0.f ? -CUDART_INF_F : rl;
        } else if (by_tma) {
          *reinterpret_cast<uint4*>(kv_s + (lane >> 3) * kMlaQPanelBytes + r * 128 + (((lane ^ r) & 7) << 4)) = w;
        } else {
          reinterpret_cast<uint4*>(a.out + (g0 + r) * kMlaDv + cta * kMlaDvHalf)[lane] = w;
        }
      }
      fence_async_smem();
      named_bar_sync(3 + qd, 128);                     // a panel below has rows of all four warps
    }
    if (by_tma) {                                      // every softmax thread comes here, whatever became of its waits
      fence_async_smem();                              // the store below reads the panel through the async proxy
      named_bar_sync(7 + quarter, 128);
      if ((warp & 3) == 0 && elect_one() && !*abort_flag) {         // x in 4-byte units: 32 per 64-column panel
        tma_store_2d(&tmap_o, kv_s + quarter * kMlaQPanelBytes, (cta * 4 + quarter) * 32, (int)g0);
        bulk_commit_and_wait_read();                   // the panel has been read: the CTA may go
      }
    }
  }

  __syncwarp();
  if (warp >= kMlaSoftmaxWarps) cluster_wait();      // the wait that pairs with the arrive above
  if (!left) cluster_arrive();                       // nothing remote is left to do for this warp either
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    // a wait gave up: let the copies that may still be in flight into this CTA land (bounded) before its shared memory goes away
    if (threadIdx.x == 0)
      for (int w = 0; w < 64; ++w) __nanosleep(1000);
    __syncthreads();
  }
  cluster_wait();                 // neither CTA leaves while the other may still copy into it or arrive on its barriers
  if (warp == kMlaMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, kMlaTmemCols);
  }
}

// The parts of a unit's keys: out[r, :] = sum_s 2^(lse_s - M) o_s / sum_s 2^(lse_s - M), each half of the columns by the sums of the CTA that computed it.
template <int PARTS>
__global__ void __launch_bounds__(128) window_combine_kernel(const WinArgs a) {
  const float *lse = grid_wait(a.part_lse), *part = grid_wait(a.part_o);
  const int unit = a.n_full + blockIdx.x, r = blockIdx.y, seq = unit / a.seq_units, row = (unit - seq * a.seq_units) * a.unit_rows + r;
  if (row >= a.seq_rows) return;
  const int d = threadIdx.x * 4, cta = d / kMlaDvHalf;
  float wgt[PARTS];
  float4 v[PARTS];
#pragma unroll
  for (int sp = 0; sp < PARTS; ++sp) {
    const int64_t p = (int64_t)blockIdx.x * a.n_split + sp;
    wgt[sp] = sp < a.n_split ? lse[(p * 2 + cta) * 128 + r] : -CUDART_INF_F;
    v[sp] = sp < a.n_split ? *reinterpret_cast<const float4*>(part + (p * 128 + r) * kMlaDv + d) : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  float mx = -CUDART_INF_F, den = 0.f;
  bool nan = false;
#pragma unroll
  for (int sp = 0; sp < PARTS; ++sp) {
    mx = fmaxf(mx, wgt[sp]);
    nan |= wgt[sp] != wgt[sp];
  }
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int sp = 0; sp < PARTS; ++sp) {
    if (wgt[sp] == -CUDART_INF_F) continue;            // a part that saw nothing has written nothing
    const float w = exp2f(wgt[sp] - mx);
    den += w;
    acc.x += w * v[sp].x; acc.y += w * v[sp].y; acc.z += w * v[sp].z; acc.w += w * v[sp].w;
  }
  const float inv = nan ? CUDART_NAN_F : den > 0.f ? 1.f / den : 0.f;
  uint2 o;
  o.x = pack_bf16x2(acc.x * inv, acc.y * inv);
  o.y = pack_bf16x2(acc.z * inv, acc.w * inv);
  *reinterpret_cast<uint2*>(a.out + ((int64_t)seq * a.seq_rows + row) * kMlaDv + d) = o;
}

// ---- launches --------------------------------------------------------------------------------------------------------
void window_combine(const WinArgs& a, int64_t units, cudaStream_t stream) {
  launch_after(1, a.n_split > 8 ? window_combine_kernel<kWinMaxParts> : window_combine_kernel<8>, dim3((unsigned)(units - a.n_full), a.unit_rows), 128, 0, stream, a);
}

template <int SRC>
static int launch_window(WinArgs a, int64_t units, int64_t keys, void* workspace, size_t workspace_bytes, cudaStream_t stream) {
  using C = WinCfg<SRC>;
  if (a.T == 0 || a.H == 0) return DSA_OK;
  const int64_t rows = (int64_t)a.T * a.H;
  window_plan(a, units, keys, workspace, workspace_bytes);
  CUtensorMap tq, to;
  int rc = make_tmap_2d_bytes(&tq, a.q, rows, kMlaDqk * 2, kMlaDqk * 2, 128, 128);
  if (rc) return rc;
  to = tq;
  if (a.n_full > 0 && rows >= 128) {
    if ((rc = make_tmap_2d_bytes(&to, a.out, rows, kMlaDv * 2, kMlaDv * 2, 128, 128))) return rc;
    a.tma_out = 1;
  }
  auto kern = window_mla_kernel<SRC>;
  static uint64_t allowed = 0;
  if (!allow_smem(reinterpret_cast<const void*>(kern), C::kSmem, &allowed))
    return set_error(DSA_ERR_CUDA, "window_mla: cannot raise dynamic shared memory to %d", C::kSmem);
  const int64_t jobs = a.n_full + (units - a.n_full) * a.n_split;
  if (2 * jobs > 0x7fffffff) return set_error(DSA_ERR_SHAPE, "window_mla: too many work units");
  kern<<<(unsigned)(2 * jobs), kMlaThreads, C::kSmem, stream>>>(tq, to, a);
  if (a.n_split > 1) window_combine(a, units, stream);
  return check_launch("window_mla");
}

// ---- drafts of many rows: records to bf16 rows once, for all of a sequence's units -------------------------------------
// Slots of every sequence (those of all its drafts) -> rows [B * pad, 576], and a bit for each that has a page.  A warp for eight slots.
constexpr int kRowsSlots = 8;
template <int SRC>
__global__ void __launch_bounds__(256) window_rows_kernel(const WinArgs a, const uint8_t* __restrict__ cache, uint4* __restrict__ rows, int B) {
  constexpr int kBytes = SRC == kSrc4 ? kLatent4Bytes : kLatentTokenBytes;
  const int lane = threadIdx.x & 31, per = a.pad / kRowsSlots;
  const int64_t job = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int b = (int)(job / per), j0 = (int)(job - (int64_t)b * per) * kRowsSlots;
  if (b >= B) return;
  const Drafts dr = drafts_of(a.drafts, b);
  if (dr.bad && j0 == 0 && lane == 0 && a.status) atomicCAS(a.status, kStatusOk, kStatusBadIndex);
  const Slots sl = slots_of(a, dr, 0, a.drafts.per_seq - 1);
  if (a.live) {                                        // rows of units without a draft
    const int row0 = (dr.m * a.H + a.unit_rows - 1) / a.unit_rows * a.unit_rows;
    for (int r = row0 + j0 / kRowsSlots; r < a.seq_rows; r += per) {
      uint4* o = reinterpret_cast<uint4*>(a.out + ((int64_t)b * a.seq_rows + r) * kMlaDv);
      o[lane] = o[32 + lane] = make_uint4(0, 0, 0, 0);
    }
  }
  if (j0 >= sl.n) return;
  int id = -1;
  if (lane < kRowsSlots && j0 + lane < sl.n) {
    const int pos = j0 + lane < sl.head ? j0 + lane : j0 + lane + sl.shift;
    const int page = __ldg(a.block_table + (int64_t)b * a.table_stride + pos / kLatentPage);
    if (page >= 0 && (int64_t)(page + 1) * kLatentPage <= a.num_phys_rows) id = page * kLatentPage + pos % kLatentPage;
    else if (a.status) atomicCAS(a.status, kStatusOk, kStatusBadIndex);
  }
  const uint32_t have = __ballot_sync(0xffffffffu, id >= 0);
  if (lane == 0) reinterpret_cast<uint8_t*>(a.valid)[((int64_t)b * a.pad + j0) / 8] = (uint8_t)have;
  uint4* out = rows + ((int64_t)b * a.pad + j0) * (kMlaDqk / 8);
#pragma unroll 4
  for (int j = 0; j < kRowsSlots; ++j) {
    const int r = __shfl_sync(0xffffffffu, id, j);
    if (j0 + j >= sl.n) break;
    uint4 v[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
    uint32_t rope = 0;
    if (r >= 0) {
      const uint8_t* rec = cache + (int64_t)r * kBytes;
#pragma unroll
      for (int h = 0; h < 2; ++h) {                    // a lane has values 8 lane .. of either half
        if constexpr (SRC == kSrcFp8) {
          v[h] = e4m3x8_to_bf16(__ldg(reinterpret_cast<const uint2*>(rec + h * 256 + lane * 8)), __ldg(reinterpret_cast<const float*>(rec + 512) + h * 2 + (lane >> 4)));
        } else {
          const uint8_t* half = rec + h * kLatent4Half;
          uint32_t p[4];
          latent4_codes(__ldg(reinterpret_cast<const uint32_t*>(half) + lane), p);
          const uint32_t sc = latent4_scale(__ldg(half + kLatent4Scales + (lane >> 1)));
#pragma unroll
          for (int i = 0; i < 4; ++i) p[i] = mul_bf16x2(mul_bf16x2(p[i], sc), kLatent4GainPair);      // both exact
          v[h] = make_uint4(p[0], p[1], p[2], p[3]);
        }
      }
      rope = SRC == kSrcFp8 ? __ldg(reinterpret_cast<const uint32_t*>(rec + 528) + lane)
                            : __ldg(reinterpret_cast<const uint32_t*>(rec + (lane >> 4) * kLatent4Half + kLatent4Rope) + (lane & 15));
    }
    out[j * (kMlaDqk / 8) + lane] = v[0];
    out[j * (kMlaDqk / 8) + 32 + lane] = v[1];
    reinterpret_cast<uint32_t*>(out + j * (kMlaDqk / 8) + 64)[lane] = rope;
  }
}
constexpr int64_t kRowsMost = 512ll << 20;             // bytes of rows at most
static int rows_pad(int64_t keys) { return (int)((keys + 63) / 64 * 64); }
// Bytes of the rows, 0: not this way.  Made rows once, a sequence's records cost its units 1.17 us a block of 64 in place of 1.8 (FP8) and 1.5 (4 bits), and 64 rows
// 0.02 us of the whole GPU.  us with records and with rows, 128 heads, FP8: 32 sequences of 3 drafts, window 512, 51.5 / 50.0, of 4 55.0 / 50.7, of 5 77 / 65, of 13
// 162 / 111; 4 bits of 4 47.9 / 49.0, of 5 69 / 63, of 13 141 / 108.  Calls that leave pairs idle cut keys into parts instead, unless there are many: 4
// sequences of 13, window 512, 28.1 / 28.7 (4 bits 24.7 / 28.2), window 2048 71 / 59.
static int64_t rows_bytes(int record_bytes, int B, int64_t seq_rows, int64_t keys) {
  const int64_t bytes = (int64_t)B * rows_pad(keys) * (kMlaDqk * 2), units = (seq_rows + 127) / 128;
  return units >= (record_bytes == kLatent4Bytes ? 5 : 4) && (B * units >= sm_count() / 2 || keys >= 1024) && bytes <= kRowsMost ? bytes : 0;
}

// Rows of a unit.  Calls that leave most pairs idle have fewer: a block's exchange and softmax take less time, and there are more units to share its keys.
static int decode_unit_rows(int B, int64_t seq_rows) {
  const int pairs = max(1, sm_count() / 2);
  for (const int rows : {32, 64})
    if (seq_rows > rows && pairs / (B * ((seq_rows + rows - 1) / rows)) >= 256 / rows) return rows;
  return 128;
}
static int64_t decode_units(int B, int64_t seq_rows) {
  const int rows = decode_unit_rows(B, seq_rows);
  return B * ((seq_rows + rows - 1) / rows);
}
// Of every call of up to B sequences.
size_t window_mla_decode_workspace(int record_bytes, int B, int tokens_per_seq, int H, int window, int first, int max_ctx) {
  const int64_t seq_rows = (int64_t)tokens_per_seq * H, keys = window_keys(H, window, first, tokens_per_seq, max_ctx);
  size_t most = window_workspace(B * ((seq_rows + 127) / 128), keys);
  for (int b = 1; b <= min(B, 16); ++b) {              // more have units of 128 rows
    const int64_t units = decode_units(b, seq_rows);
    const int parts = window_parts(units, keys);
    if (parts > 1) most = max(most, (size_t)(units % max(1, sm_count() / 2)) * parts * kWinPartBytes);
  }
  const int64_t slots = min((int64_t)max_ctx, (int64_t)window + first + tokens_per_seq), rows = rows_bytes(record_bytes, B, seq_rows, slots);
  if (rows) most = max(most, (size_t)rows + (size_t)B * rows_pad(slots) / 8 + 256 + window_prompt_drafts_workspace(B, seq_rows, H, keys));
  return most;
}

int window_mla_decode_launch(const void* q, const void* cache, int record_bytes, const int32_t* block_table, int64_t table_stride, const int32_t* ctx_len,
                             const int32_t* n_new, const int64_t* tree, int tokens_per_seq, void* out, int B, int H, int window, int first, int num_pages,
                             int max_ctx, float scale, void* workspace, size_t workspace_bytes, int32_t* status, cudaStream_t stream) {
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
  a.seq_rows = tokens_per_seq * H;
  const int64_t slots = min((int64_t)max_ctx, (int64_t)window + first + tokens_per_seq), rows = rows_bytes(record_bytes, B, a.seq_rows, slots);
  if (rows && workspace) {
    a.pad = rows_pad(slots);
    const size_t valid = ((size_t)B * a.pad / 8 + 255) / 256 * 256;
    if (workspace_bytes >= rows + valid) {
      a.valid = reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(workspace) + rows);
      window_prompt_units(a);
      const unsigned grid = (unsigned)(((int64_t)B * (a.pad / kRowsSlots) + 7) / 8);
      auto kern = record_bytes == kLatent4Bytes ? window_rows_kernel<kSrc4> : window_rows_kernel<kSrcFp8>;
      kern<<<grid, 256, 0, stream>>>(a, a.kv, static_cast<uint4*>(workspace), B);
      a.kv = static_cast<const uint8_t*>(workspace);
      a.S = B * a.pad;
      return window_prompt_drafts(a, static_cast<uint8_t*>(workspace) + rows + valid, workspace_bytes - rows - valid, stream);
    }
  }
  a.unit_rows = decode_unit_rows(B, a.seq_rows);
  a.seq_units = (a.seq_rows - 1) / a.unit_rows + 1;
  const int64_t units = (int64_t)B * a.seq_units, keys = window_keys(H, window, first, tokens_per_seq, max_ctx);
  return record_bytes == kLatent4Bytes ? launch_window<kSrc4>(a, units, keys, workspace, workspace_bytes, stream)
                                       : launch_window<kSrcFp8>(a, units, keys, workspace, workspace_bytes, stream);
}

}  // namespace dsa
