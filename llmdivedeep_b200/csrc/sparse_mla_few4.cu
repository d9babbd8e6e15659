// Attention of at most 32 heads over the paged 4-bit latent cache (latent4.cuh) for calls of more than a few rows (sparse_mla.cu takes
// those): the function of that file's decode with scores and output TRANSPOSED, as in sparse_mla_few.cu, so that the heads are the N of
// the tensor-core tiles and not the M:
//   S^T [64 keys x N heads] = K Q^T     (M = 64, 36 K-steps over the 576 dims)
//   O^T [512 dims x N heads] += V^T P^T (four M = 128 tiles, 4 K-steps over a block's 64 keys)
// N is 16 or 32.  The latents are converted to bf16 times 2^-14, the rope values too: the scores come out 2^-14 times what they are and
// the output too, which the softmax scale and the quotient at the end make good.
//
// Persistent CTAs, one per SM.  As many lists as there are whole rounds of go to the CTAs one by one; the blocks of 64 slots of the lists
// that are left are dealt out in equal stretches.  Of a list that is cut every CTA leaves a normalised partial output and its
// log2-sum-exp in the workspace, and a second kernel merges them (fp32).  So calls of one row and of a thousand fill the GPU alike, and a
// row's last bits depend on its place in the call.
//   * warps 0-3: softmax and output; warp 4 issues the scores' MMAs, warp 6 those of P.V; warp 5: the end of every list, Q.
//   * warps 7-22: four rows of a block each, eight lanes a row: the records are requested two blocks ahead into registers and, converted,
//     go into a ring of half blocks (256 dims of 64 keys in four 128-byte swizzled panels, four such).  Positions and page-table entries
//     come for eight blocks at a time, one and two such groups ahead.
//
// What bounds it: shared memory.  Of the ~2450 cycles that a block takes the tensor cores read it for 1300 (K and V once each, Q and P
// with every instruction) and the warps use it for 860, the conversion's 73 KB most of it.  The number of MMAs does not: 34 a block in place of 52,
// with score tiles of 128 rows -- two panels at a time, their sums exchanged between softmax warps -- take 55.1 us where this takes
// 53.0 (148 rows, 16 heads).  Issued by one warp, though, scores and P.V took 69.9 us where two took 55.8.  A call adds ~12000 cycles until the first block's scores are complete, a
// further list two blocks, parts their merge.  2048 keys, 16 heads: 64 rows 33.3 us, 148 rows 53.0 (126 MB of records: 2.4 TB/s, 199 TFLOP/s),
// 160 rows 64.5, 296 rows 98.5; 32 heads: 64 rows 39.9, 148 rows 62.4 (339 TFLOP/s), 256 rows 116.
// Tried and dropped: rows by cp.async or bulk copies through a stage of raw records (65 to 84 us where this took 55.8), eight softmax warps
// (60 to 66), Q of two lists (no gain), a prefetch of the first records into L2 (+4 us).
// Every wait is bounded (dsa_common.cuh).
#include <cuda.h>
#include <cudaTypedefs.h>
#include <math_constants.h>

#include "dsa_common.cuh"
#include "dsa_host.h"
#include "latent4.cuh"

namespace dsa {

struct Few4Args {
  const uint8_t* cache;           // [num_rows, 416]
  const int32_t* block_table;     // [sequences, table_stride]: list t is of sequence (row0 + t) / tokens_per_seq
  const int32_t* idx;             // [T, K] positions (negative = empty)
  __nv_bfloat16* out;             // [T, H, 512]
  int64_t table_stride;
  int T, H, K, max_ctx, tokens_per_seq;
  int row0;                       // the call's row that this launch begins with
  int num_rows;
  int list_blocks;                // blocks of 64 slots of a list
  int ctas;
  int rounds;                     // CTA c has lists c, c + ctas, ... of so many rounds, ...
  int rest, rest_ctas;            // ... and if c < rest_ctas, a stretch of the rest blocks of the lists behind them:
  int per_list;                   // one of so many equal parts of a list, or (0) of all blocks
  float scale_log2e;
  float* part_o;                  // [2 ctas][H][512]: of a CTA's first piece of a list and of its last one
  float* part_lse;                // [2 ctas][H], log2 units, -inf = empty
  int* status;
};

constexpr int kF4GatherWarps = 16, kF4SoftmaxWarps = 4;
constexpr int kF4MmaWarp = kF4SoftmaxWarps, kF4StageWarp = kF4MmaWarp + 1, kF4PvWarp = kF4MmaWarp + 2, kF4GatherWarp0 = kF4MmaWarp + 3;
constexpr int kF4Threads = (kF4GatherWarp0 + kF4GatherWarps) * 32;
constexpr int kF4Blk = 64, kF4Rows = kF4Blk / kF4GatherWarps;      // keys of a block, rows of a gather warp
constexpr int kF4Panel = kF4Blk * 128;                 // 64 keys x 64 dims, 128-byte swizzled
constexpr int kF4Half = 4 * kF4Panel;                  // 256 dims of a block
constexpr int kF4Dv = 512, kF4QBytes = 1152;
constexpr int kF4Valid = 8;                            // ring of validity bytes, by block
constexpr int kF4Pieces = 1024;                        // pieces of a CTA at most: the launcher cuts longer calls, inside a sequence too
constexpr uint8_t kF4Unknown = 255;                    // a piece's length before the list's end is known
constexpr int kF4Look = 8;                             // 16-byte pieces of a list that a lane looks at together
constexpr uint32_t kF4RopeGain = 0x38803880u;          // 2^-14 as a pair of bf16

template <int N>
struct F4Cfg {
  // Ring of half blocks.  What is not shared memory is L1, and there the loads of the records under way need about 50 KB: five halves are
  // slower, of 32 heads most, where they leave it 28 KB (148 rows x 2048 keys: 16 heads 54.8 -> 53.5 us, 32 heads 73.7 -> 62.9); three
  // make the conversion wait for P.V (68.6, 81.2).
  static constexpr int HALVES = 4;
  static constexpr int PBUFS = 2;
  static constexpr int Q_BYTES = 9 * N * 128, P_BYTES = N * 128;
  static constexpr int BAR_BYTES = 512;
  static constexpr int SMEM = HALVES * kF4Half + kF4Panel + Q_BYTES + PBUFS * P_BYTES + BAR_BYTES + kF4Valid * kF4Blk + kF4Pieces + 3 * kF4SoftmaxWarps * N * 4;
  static constexpr uint32_t COL_O = 0, COL_S = 4 * N, COLS = COL_S + 2 * N <= 128 ? 128 : 256;
  static_assert(SMEM <= 232448 && COL_S + 2 * N <= COLS, "budget of one CTA");
};

__device__ __forceinline__ void f4_ld_s(uint32_t taddr, uint32_t (&r)[8]) {      // as few_ld_s
  asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr) : "memory");
}
// 16 bytes of a record: read once, so nothing is kept for it in L1 (16 heads, 148 rows 53.5 -> 52.9 us, 160 rows 66.6 -> 64.8).
__device__ __forceinline__ uint4 f4_ld_once(const uint8_t* p) {
  uint4 r;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
  return r;
}
__device__ __forceinline__ uint32_t f4_pack(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float f4_exp2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// Whether the phase is complete, without the pause that try_wait may make: for a warp that has more than one thing to look at.
__device__ __forceinline__ uint32_t f4_test(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok;
}
// What a CTA has to do, list by list: the whole lists of its rounds, then its stretch.
struct F4Piece {
  int cta;
  int done, all, start;                                // its blocks behind it, and all of them; first block of the stretch
  int t, b0, b1;                                       // the list and its blocks [b0, b1) in this piece
  static __host__ __device__ __forceinline__ int start_of(const Few4Args& a, int c) {
    if (a.per_list) return c / a.per_list * a.list_blocks + c % a.per_list * a.list_blocks / a.per_list;
    return a.rest ? (int)((int64_t)c * a.rest / a.rest_ctas) : 0;
  }
  __host__ __device__ __forceinline__ F4Piece(const Few4Args& a, int c) : cta(c) {
    start = start_of(a, c);
    done = t = b0 = b1 = 0;
    all = min(a.rounds, (a.T - c + a.ctas - 1) / a.ctas) * a.list_blocks + (c < a.rest_ctas ? start_of(a, c + 1) - start : 0);
  }
  __host__ __device__ __forceinline__ bool next(const Few4Args& a) {
    if (done >= all) return false;
    const int x = done - a.rounds * a.list_blocks;
    if (x < 0) {
      t = done / a.list_blocks * a.ctas + cta;
      b0 = 0;
      b1 = a.list_blocks;
    } else {
      t = (start + x) / a.list_blocks;
      b0 = start + x - t * a.list_blocks;
      b1 = min(a.list_blocks, b0 + all - done);
      t += a.rounds * a.ctas;
    }
    done += b1 - b0;
    return true;
  }
  // The part that this piece leaves if it is not a whole list: of the stretch's first list, or of its last.
  __device__ __forceinline__ int part(const Few4Args& a) const { return 2 * cta + (done - (b1 - b0) == a.rounds * a.list_blocks ? 0 : 1); }
};

// What one of `of` threads sees of the slots [lo, hi) of a list: the last used one, and the largest position.
struct F4Scan {
  int last, top;
  __device__ __forceinline__ void see(int id, int j, int max_ctx) {
    if (id >= 0 && id < max_ctx) last = j;
    top = max(top, id);
  }
  __device__ __forceinline__ F4Scan(const Few4Args& a, const int32_t* row, int lo, int hi, int me, int of) {
    last = top = -1;
    if (((reinterpret_cast<uintptr_t>(row + lo) | (hi - lo) * 4) & 15) == 0) {      // a few loads are requested before the first is looked at
#pragma unroll 1
      for (int j0 = lo + me * 4; j0 < hi; j0 += of * 4 * kF4Look) {
        int4 id[kF4Look];
#pragma unroll
        for (int i = 0; i < kF4Look; ++i)
          id[i] = j0 + i * of * 4 < hi ? *reinterpret_cast<const int4*>(row + j0 + i * of * 4) : make_int4(-1, -1, -1, -1);
#pragma unroll
        for (int i = 0; i < kF4Look; ++i) {
          const int j = j0 + i * of * 4;
          see(id[i].x, j, a.max_ctx); see(id[i].y, j + 1, a.max_ctx); see(id[i].z, j + 2, a.max_ctx); see(id[i].w, j + 3, a.max_ctx);
        }
      }
    } else {
#pragma unroll 4
      for (int j = lo + me; j < hi; j += of) see(row[j], j, a.max_ctx);
    }
    if (top >= a.max_ctx && a.status) atomicCAS(a.status, kStatusOk, kStatusBadIndex);
    last = __reduce_max_sync(0xffffffffu, last);
  }
};

template <int N>
__global__ void __launch_bounds__(kF4Threads, 1)
sparse_mla_few4_kernel(const __grid_constant__ CUtensorMap tmap_q, const Few4Args a) {
  using C = F4Cfg<N>;
  constexpr int NH = N / 8;                            // groups of eight heads: a thread has two adjacent heads of each
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* half_s = smem;                              // [HALVES][4 panels]
  uint8_t* rope_s = half_s + C::HALVES * kF4Half;      // one panel: free again after a block's scores
  uint8_t* q_s = rope_s + kF4Panel;                    // nine panels [N heads x 128 B]
  uint8_t* p_s = q_s + C::Q_BYTES;                     // P^T as [N heads][64 keys], swizzled
  uint64_t* bars = reinterpret_cast<uint64_t*>(p_s + C::PBUFS * C::P_BYTES);
  uint64_t* half_full = bars + 0;                      // [4] gather -> MMA; a block's second half: its rope values and validity bytes too
  uint64_t* half_free = bars + 4;                      // [4] P.V of those 256 dims has read the half
  uint64_t* rope_free = bars + 8;                      // the block's scores have read the rope panel
  uint64_t* q_full = bars + 9;
  uint64_t* q_free = bars + 10;
  uint64_t* s_full = bars + 11;                        // [2] MMA -> softmax
  uint64_t* pv_done = bars + 13;                       // [2] P.V of the block complete
  uint64_t* p_full = bars + 15;                        // [2] softmax -> MMA
  uint64_t* meet = bars + 17;                          // the four softmax warps
  uint64_t* s_free = bars + 18;                        // [2] the softmax has read S
  constexpr int kBars = 20;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + kBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  uint8_t* valid_s = reinterpret_cast<uint8_t*>(bars) + C::BAR_BYTES;
  volatile uint8_t* len_s = valid_s + kF4Valid * kF4Blk;            // [kF4Pieces] used blocks of the CTA's pieces
  int* last_s = reinterpret_cast<int*>(bars + kBars + 1);           // [warps] what each has seen of the first list
  float* max_s = reinterpret_cast<float*>(valid_s + kF4Valid * kF4Blk + kF4Pieces);      // [2][4 warps][N] block maxima by block parity
  float* wgt_s = max_s + 2 * kF4SoftmaxWarps * N;      // [4 warps][N]
  static_assert((kBars + 1) * 8 + kF4Threads / 32 * 4 <= C::BAR_BYTES, "barriers");

  const int warp = warp_index(), lane = threadIdx.x & 31;
  launch_dependents();
  if (warp == 0) {
    for (int i = lane; i < kBars; i += 32) {
      const uint32_t count = i < 4 ? uint32_t(kF4GatherWarps) : i >= 15 ? uint32_t(kF4SoftmaxWarps) : 1u;
      mbar_init(bars + i, count);
    }
    mbar_fence_init();
    if (lane == 0) *abort_flag = 0;
  } else if (warp == kF4MmaWarp) {
    tmem_alloc(tmem_slot, C::COLS);
    tmem_relinquish();
  }
  for (int i = threadIdx.x; i < kF4Pieces / 4; i += kF4Threads) reinterpret_cast<volatile uint32_t*>(len_s)[i] = 0x01010101u * kF4Unknown;
  const int32_t* idx = grid_wait(a.idx);               // a launch under the top-k's end reads its lists after the wait
  // The first piece's end is found by all threads together, so that it is known when the roles begin.
  int blocks0;
  {
    F4Piece p0(a, blockIdx.x);
    const bool there = p0.next(a);
    const int lo = p0.b0 * kF4Blk, hi = there ? min(a.K, p0.b1 * kF4Blk) : lo;
    const F4Scan scan(a, idx + (int64_t)p0.t * a.K, lo, hi, threadIdx.x, kF4Threads);
    if (lane == 0) last_s[warp] = scan.last;
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const int last0 = __reduce_max_sync(0xffffffffu, lane < kF4Threads / 32 ? last_s[lane] : -1);
    blocks0 = last0 < 0 ? 0 : (last0 - lo) / kF4Blk + 1;
  }
  const uint32_t tmem = *tmem_slot;

  // Used blocks of the CTA's nu-th piece, once the warp that reads the lists has come to it (it waits for nobody).
  auto piece_blocks = [&](uint32_t nu, bool& ok) -> int {
    if (nu == 0) return blocks0;
    for (uint32_t i = 0; i < kSpinLimit; ++i) {
      const int nb = len_s[nu];
      if (__all_sync(0xffffffffu, nb != kF4Unknown)) return nb;
      if (i > kFastSpins) {
        if (aborted_warp(abort_flag)) break;
        __nanosleep(40);
      }
    }
    *abort_flag = 1;
    if (a.status) atomicCAS(a.status, kStatusOk, kStatusWaitTimeout);
    ok = false;
    return 0;
  };
  F4Piece pc(a, blockIdx.x);
  constexpr uint64_t kHalf = kF4Half >> 4, kOne = kF4Panel >> 4, kQPanel = (N * 128) >> 4;      // descriptor steps

  if (warp == kF4StageWarp) {
    // ------------- the last used slot of every piece (it decides the number of blocks), and Q -------------
    // Whichever can go on; Q, which the tensor core waits for, first.
    F4Piece qc(a, blockIdx.x);
    uint32_t nu = 1, nq = 0, idle = 0;
    bool lists = pc.next(a), queries = true;           // (the first list's end is known)
    while (lists || queries) {
      if (queries && __all_sync(0xffffffffu, f4_test(q_free, (nq & 1) ^ 1))) {
        queries = qc.next(a);
        if (queries) {
          if (lane == 0) mbar_expect_tx(q_full, C::Q_BYTES);
          __syncwarp();
          if (lane < 9) tma_load_2d(q_s + lane * N * 128, &tmap_q, lane * 32, qc.t * a.H, q_full);      // x in 4-byte units
          ++nq;
        }
        idle = 0;
      } else if (lists) {
        lists = pc.next(a);
        if (!lists) continue;
        const int lo = pc.b0 * kF4Blk;
        const int last = F4Scan(a, idx + (int64_t)pc.t * a.K, lo, min(a.K, pc.b1 * kF4Blk), lane, 32).last;
        if (lane == 0) len_s[nu] = (uint8_t)(last < 0 ? 0 : (last - lo) / kF4Blk + 1);
        ++nu;
      } else if (++idle > kFastSpins) {
        if (idle > kSpinLimit || aborted_warp(abort_flag)) {
          *abort_flag = 1;
          if (a.status) atomicCAS(a.status, kStatusOk, kStatusWaitTimeout);
          break;
        }
        __nanosleep(40);
      }
    }
  } else if (warp == kF4MmaWarp) {
    // ------------------------------- scores -------------------------------
    constexpr uint32_t idesc_qk = umma_idesc(1, 1, 0, 0, kF4Blk, N);
    const uint64_t qdesc = umma_smem_desc(smem_u32(q_s), 16, 1024, kSwz128);
    const uint64_t kdesc = umma_smem_desc(smem_u32(half_s), 16, 1024, kSwz128);
    const uint64_t rdesc = umma_smem_desc(smem_u32(rope_s), 16, 1024, kSwz128);
    uint32_t nu = 0, n = 0;
    bool ok = true;
    for (; ok && pc.next(a); ++nu) {
      const int nb = piece_blocks(nu, ok);
      if (ok) ok = mbar_wait_warp(q_full, nu & 1, abort_flag, a.status);
      if (!ok) break;
      if (nb == 0) {                                   // Q was fetched before the list was known
        if (lane == 0) mbar_arrive(q_free);
        continue;
      }
      for (const uint32_t end = n + nb; n < end; ++n) {
        const uint32_t d = tmem + C::COL_S + (n & 1) * N;
        if (n >= 2) ok = mbar_wait_warp(&s_free[n & 1], ((n >> 1) - 1) & 1, abort_flag, a.status);
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          const uint32_t g = 2 * n + hf;
          if (ok) ok = mbar_wait_warp(&half_full[g % C::HALVES], (g / C::HALVES) & 1, abort_flag, a.status);
          if (!ok) break;
          fence_async_smem();                          // the rows were written through the generic proxy
          tc_fence_after();
          if (elect_one()) {
            const uint64_t kd = kdesc + (g % C::HALVES) * kHalf;
#pragma unroll
            for (int ks = 0; ks < 16; ++ks)
              umma_f16_ss(d, kd + (ks >> 2) * kOne + 2 * (ks & 3), qdesc + (4 * hf + (ks >> 2)) * kQPanel + 2 * (ks & 3), idesc_qk, hf | ks);
            if (hf == 1) {
#pragma unroll
              for (int ks = 0; ks < 4; ++ks) umma_f16_ss(d, rdesc + 2 * ks, qdesc + 8 * kQPanel + 2 * ks, idesc_qk, 1);
              umma_commit(&s_full[n & 1]);
              umma_commit(rope_free);
              if (n + 1 == end) umma_commit(q_free);
            }
          }
          __syncwarp();
        }
        if (!ok) break;
      }
    }
  } else if (warp == kF4PvWarp) {
    // ------------------------------- P.V -------------------------------
    constexpr uint32_t idesc_pv = umma_idesc(1, 1, 1, 0, 128, N);
    const uint64_t vdesc = umma_smem_desc(smem_u32(half_s), kF4Panel, 1024, kSwz128);
    const uint64_t pdesc = umma_smem_desc(smem_u32(p_s), 16, 1024, kSwz128);
    uint32_t nu = 0, n = 0;
    bool ok = true;
    for (; ok && pc.next(a); ++nu) {
      const int nb = piece_blocks(nu, ok);
      for (const uint32_t begun = n, end = n + nb; n < end; ++n) {      // a piece's first P says that the last one's O has been read
        ok = mbar_wait_warp(&p_full[n & 1], (n >> 1) & 1, abort_flag, a.status);
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          const uint64_t pd = pdesc + (n & 1) * (C::P_BYTES >> 4);
#pragma unroll
          for (int m = 0; m < 4; ++m) {
            const uint64_t vd = vdesc + ((2 * n + (m >> 1)) % C::HALVES) * kHalf + (m & 1) * 2 * kOne;
#pragma unroll
            for (int ks = 0; ks < 4; ++ks)             // 16 keys: 16 rows x 128 B further into each panel, 32 B along P's rows
              umma_f16_ss(tmem + C::COL_O + m * N, vd + ks * (2048 >> 4), pd + 2 * ks, idesc_pv, n != begun || ks != 0);
            if (m & 1) umma_commit(&half_free[(2 * n + (m >> 1)) % C::HALVES]);
          }
          umma_commit(&pv_done[n & 1]);
        }
        __syncwarp();
      }
    }
  } else if (warp >= kF4GatherWarp0) {
    // ----------------------------- gather: four rows of every block to a warp -----------------------------
    const int w = warp - kF4GatherWarp0, r0 = kF4Rows * w;
    bool ok = true, more = true;
    uint32_t nu = 0;
    int j = 0, jend = 0;                               // blocks of the current piece that are still to be looked up
    // Row ids come by groups of eight used blocks: lane 4 b + r has row r0 + r of the group's block b.  Positions are requested two
    // groups ahead, page-table entries one.
    struct Group { int pos, list, blocks; };
    auto look_up = [&]() -> Group {
      Group h{-1, 0, 0};
      int slot = -1;
      while (more && h.blocks < 8) {
        if (j == jend) {
          more = pc.next(a);
          if (!more) break;
          j = pc.b0;
          jend = j + piece_blocks(nu++, ok);
          if (!ok) more = false;
          continue;
        }
        const int take = min(8 - h.blocks, jend - j), b = (lane >> 2) - h.blocks;
        if (b >= 0 && b < take) {
          h.list = pc.t;
          slot = (j + b) * kF4Blk + r0 + (lane & 3);
        }
        j += take;
        h.blocks += take;
      }
      if (slot >= 0 && slot < a.K) h.pos = idx[(int64_t)h.list * a.K + slot];
      return h;
    };
    auto table_entry = [&](const Group& h) -> int {
      return h.pos >= 0 && h.pos < a.max_ctx ? __ldg(a.block_table + (int64_t)((a.row0 + h.list) / a.tokens_per_seq) * a.table_stride + h.pos / 64) : -1;
    };
    auto cache_row = [&](const Group& h, int page) -> int {        // -1 = empty; bad positions are flagged by the warp that reads the list
      if (h.pos < 0 || h.pos >= a.max_ctx) return -1;
      if (page >= 0 && (int64_t)(page + 1) * 64 <= a.num_rows) return page * 64 + h.pos % 64;
      if (a.status) atomicCAS(a.status, kStatusOk, kStatusBadIndex);
      return -1;
    };
    // ids of the group that the next block to fetch is in; entries and positions of the next, positions of the one after
    Group h1 = look_up(), h2{-1, 0, 0};
    int ids = cache_row(h1, table_entry(h1)), got = h1.blocks, e1 = -1;
    h1 = h2;
    uint32_t fetched = 0, group0 = 0;                  // blocks fetched; first block of the group
    // This lane's part of a row: of either half 32 neighbouring dims -- four words, two scales -- and eight rope values.
    struct Raw { uint4 word[2], rope; uint32_t scales[2]; bool used; };
    const int l8 = lane & 7;
    auto fetch_next = [&](Raw& x) {                    // an empty slot's row: zeros
      x.word[0] = x.word[1] = x.rope = make_uint4(0, 0, 0, 0);
      x.scales[0] = x.scales[1] = 0;
      x.used = false;
      if (fetched - group0 == (uint32_t)got) {
        group0 = fetched;
        got = h1.blocks;
        ids = cache_row(h1, e1);
        h1 = h2;
        e1 = table_entry(h1);
        h2 = look_up();
      }
      if (got == 0) return;
      const int id = __shfl_sync(0xffffffffu, ids, 4 * (fetched - group0) + (lane >> 3));
      if (id >= 0) {
        const uint8_t* src = a.cache + (int64_t)id * kLatent4Bytes;
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          x.word[hf] = f4_ld_once(src + hf * kLatent4Half + l8 * 16);
          x.scales[hf] = __ldg(reinterpret_cast<const uint16_t*>(src + hf * kLatent4Half + kLatent4Scales + l8 * 2));
        }
        x.rope = f4_ld_once(src + (l8 >> 2) * kLatent4Half + kLatent4Rope + (l8 & 3) * 16);
        x.used = true;
      }
      ++fetched;
    };
    // A lane stores its words in an order of its own, so that the eight lanes of a row hit all banks.
    const int rr = r0 + (lane >> 3), turn = l8 >> 1;
    uint32_t off[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) off[i] = turn * kF4Panel + rr * 128 + (((((l8 & 1) * 4 + ((i + turn) & 3)) ^ rr) & 7) << 4);
    auto put_block = [&](uint32_t n, const Raw& r) {
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        // words and scales in this lane's order
        uint32_t x[4] = {r.word[hf].x, r.word[hf].y, r.word[hf].z, r.word[hf].w}, y[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = turn & 1 ? x[(i + 1) & 3] : x[i];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = turn & 2 ? y[(i + 2) & 3] : y[i];
        const uint32_t lo = latent4_scale(r.scales[hf] & 255u), hi = latent4_scale(r.scales[hf] >> 8);
        const uint32_t g = 2 * n + hf, slot = g % C::HALVES;
        if (ok && g >= C::HALVES) ok = mbar_wait_warp(&half_free[slot], (g / C::HALVES - 1) & 1, abort_flag, a.status);
        if (!ok) break;
        uint8_t* dst = half_s + slot * kF4Half;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t c[4];
          latent4_codes(x[i], c);
          const uint32_t sc = (i + turn) & 2 ? hi : lo;
          *reinterpret_cast<uint4*>(dst + off[i]) = make_uint4(mul_bf16x2(c[0], sc), mul_bf16x2(c[1], sc), mul_bf16x2(c[2], sc), mul_bf16x2(c[3], sc));
        }
        if (hf == 1) {
          if (n >= 1) ok = mbar_wait_warp(rope_free, (n - 1) & 1, abort_flag, a.status);
          if (!ok) break;
          *reinterpret_cast<uint4*>(rope_s + rr * 128 + (((l8 ^ rr) & 7) << 4)) =
              make_uint4(mul_bf16x2(r.rope.x, kF4RopeGain), mul_bf16x2(r.rope.y, kF4RopeGain), mul_bf16x2(r.rope.z, kF4RopeGain), mul_bf16x2(r.rope.w, kF4RopeGain));
          if (l8 == 0) valid_s[(n % kF4Valid) * kF4Blk + rr] = r.used;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&half_full[slot]);
      }
    };
    Raw even, odd;                                     // blocks of either parity: nothing moves from register to register
    fetch_next(even);
    fetch_next(odd);                                   // (a group of fewer than two blocks is the last)
    h1 = look_up();
    e1 = table_entry(h1);
    h2 = look_up();
    for (uint32_t n = 0; ok && n < fetched; n += 2) {
      put_block(n, even);
      fetch_next(even);
      if (!ok || n + 1 >= fetched) break;
      put_block(n + 1, odd);
      fetch_next(odd);
    }
  } else {
    // ------------- softmax and output: warp w has keys 16 w.. of a block, and dims 32 w.. of every 128 of the output -------------
    const uint32_t t_row = tmem + (uint32_t(warp * 32) << 16);
    uint32_t nu = 0, n = 0, met = 0;
    bool ok = true;
    auto all_meet = [&]() -> bool {                    // the four warps: what was written to shared memory before is seen after
      __syncwarp();
      if (lane == 0) mbar_arrive(meet);
      return mbar_wait_warp(meet, met++ & 1, abort_flag, a.status);
    };
    auto put_row = [&](float* row, const float(&v)[2 * NH]) {      // heads 8 i + 2 (lane % 4), + 1 of every thread's values
      if (lane < 4) {
#pragma unroll
        for (int i = 0; i < NH; ++i) *reinterpret_cast<float2*>(row + 8 * i + 2 * lane) = make_float2(v[2 * i], v[2 * i + 1]);
      }
    };
    for (; ok && pc.next(a); ++nu) {
      const int nb = piece_blocks(nu, ok);
      if (!ok) break;
      const bool whole = pc.b0 == 0 && pc.b1 == a.list_blocks;
      __nv_bfloat16* out = a.out + (int64_t)pc.t * a.H * kF4Dv;
      const int64_t part = pc.part(a);
      if (nb == 0) {                                   // nothing selected: zero rows, or a part of no weight
        if (whole) {
          for (int i = warp * 32 + lane; i < a.H * (kF4Dv / 8); i += kF4SoftmaxWarps * 32) reinterpret_cast<uint4*>(out)[i] = make_uint4(0, 0, 0, 0);
        } else if (warp == 0) {
          for (int h = lane; h < a.H; h += 32) a.part_lse[part * a.H + h] = -CUDART_INF_F;
        }
        continue;
      }
      float m[2 * NH], l[2 * NH];                      // heads 8 i + 2 (lane % 4), + 1: references (log2), sums over this thread's keys
#pragma unroll
      for (int i = 0; i < 2 * NH; ++i) { m[i] = -CUDART_INF_F; l[i] = 0.f; }
      const uint32_t begun = n, stop = n + nb;
      for (; n != stop; ++n) {
        ok = mbar_wait_warp(&s_full[n & 1], (n >> 1) & 1, abort_flag, a.status);
        if (!ok) break;
        tc_fence_after();
        uint32_t sv[4 * NH];
#pragma unroll
        for (int i = 0; i < NH; i += 2) f4_ld_s(t_row + C::COL_S + (n & 1) * N + 8 * i, *reinterpret_cast<uint32_t(*)[8]>(&sv[4 * i]));
        const uint8_t* valid = valid_s + (n % kF4Valid) * kF4Blk + 16 * warp + (lane >> 2);
        const bool va = valid[0], vb = valid[8];
        tmem_wait_ld();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_free[n & 1]);
        float s[4 * NH], bm[2 * NH];
#pragma unroll
        for (int i = 0; i < NH; ++i) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            s[4 * i + e] = va ? __uint_as_float(sv[4 * i + e]) : -CUDART_INF_F;
            s[4 * i + 2 + e] = vb ? __uint_as_float(sv[4 * i + 2 + e]) : -CUDART_INF_F;
            bm[2 * i + e] = fmaxf(s[4 * i + e], s[4 * i + 2 + e]);
          }
        }
#pragma unroll
        for (int o = 4; o < 32; o <<= 1)
#pragma unroll
          for (int i = 0; i < 2 * NH; ++i) bm[i] = fmaxf(bm[i], __shfl_xor_sync(0xffffffffu, bm[i], o));
        float* mx = max_s + (n & 1) * 4 * N;
        put_row(mx + warp * N, bm);
        ok = all_meet();
        if (!ok) break;
        bool grown = false;
        float f[2 * NH];
#pragma unroll
        for (int i = 0; i < NH; ++i) {
          float2 b = make_float2(-CUDART_INF_F, -CUDART_INF_F);
#pragma unroll
          for (int v = 0; v < kF4SoftmaxWarps; ++v) {
            const float2 x = *reinterpret_cast<const float2*>(mx + v * N + 8 * i + 2 * (lane & 3));
            b.x = fmaxf(b.x, x.x);
            b.y = fmaxf(b.y, x.y);
          }
          const float bx[2] = {b.x * a.scale_log2e, b.y * a.scale_log2e};
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float m_old = m[2 * i + e];
            const bool up = bx[e] - m_old > kMaxRaise; // also true when m is still -inf and the maximum finite
            f[2 * i + e] = up ? f4_exp2(m_old - bx[e]) : 1.f;
            if (up) m[2 * i + e] = bx[e];
            grown |= up;
          }
        }
        if (__any_sync(0xffffffffu, grown)) {          // the same in all four warps
#pragma unroll
          for (int i = 0; i < 2 * NH; ++i) l[i] *= f[i];
          if (n != begun) {                            // O must be quiescent: P.V of the block before complete
            ok = mbar_wait_warp(&pv_done[(n - 1) & 1], ((n - 1) >> 1) & 1, abort_flag, a.status);
            if (!ok) break;
            tc_fence_after();
            float* fac = max_s + ((n + 1) & 1) * 4 * N + warp * N;      // the half that this block does not use
            put_row(fac, f);
            __syncwarp();
#pragma unroll 1
            for (int c = 0; c < 4 * N; c += 16) {
              uint32_t ov[16];
              tmem_ld16(t_row + C::COL_O + c, ov);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 16; ++i) ov[i] = __float_as_uint(__uint_as_float(ov[i]) * fac[(c & (N - 1)) + i]);
              tmem_st16(t_row + C::COL_O + c, ov);
            }
            tmem_wait_st();
            __syncwarp();
          }
        }
        uint32_t pk[2 * NH];                           // [group of eight heads][keys t / 4, t / 4 + 8]: two heads each
#pragma unroll
        for (int i = 0; i < NH; ++i) {
          const float m0 = m[2 * i] == -CUDART_INF_F ? 0.f : m[2 * i], m1 = m[2 * i + 1] == -CUDART_INF_F ? 0.f : m[2 * i + 1];
          const float p0 = f4_exp2(fmaf(s[4 * i], a.scale_log2e, -m0)), p1 = f4_exp2(fmaf(s[4 * i + 1], a.scale_log2e, -m1));
          const float p2 = f4_exp2(fmaf(s[4 * i + 2], a.scale_log2e, -m0)), p3 = f4_exp2(fmaf(s[4 * i + 3], a.scale_log2e, -m1));
          pk[2 * i] = f4_pack(p0, p1);
          pk[2 * i + 1] = f4_pack(p2, p3);
          add_bf16x2(pk[2 * i], l[2 * i], l[2 * i + 1]);            // of P as it was rounded (sparse_mla.cu)
          add_bf16x2(pk[2 * i + 1], l[2 * i], l[2 * i + 1]);
        }
        if (n >= C::PBUFS) {                           // that P buffer has been read
          ok = mbar_wait_warp(&pv_done[(n - C::PBUFS) & 1], ((n - C::PBUFS) >> 1) & 1, abort_flag, a.status);
          if (!ok) break;
        }
        // transposed on the way: row = head, 16-byte chunk = eight keys
        uint8_t* p = p_s + (n % C::PBUFS) * C::P_BYTES;
#pragma unroll
        for (int i = 0; i < NH; i += 2) {
          const int h = 8 * (i + (lane >> 4)) + (lane & 7), ch = 2 * warp + ((lane >> 3) & 1);
          asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};"
                       ::"r"(smem_u32(p + h * 128 + ((ch ^ (h & 7)) << 4))), "r"(pk[2 * i]), "r"(pk[2 * i + 1]), "r"(pk[2 * i + 2]), "r"(pk[2 * i + 3])
                       : "memory");
        }
        fence_async_smem();                            // visible to the tensor core's reads
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[n & 1]);
      }
      if (!ok) break;
      // row sums over the lanes that share a head, and over the warps
      float* sum_s = max_s + (n & 1) * 4 * N;          // the last block's maxima are in the other half
#pragma unroll
      for (int o = 4; o < 32; o <<= 1)
#pragma unroll
        for (int i = 0; i < 2 * NH; ++i) l[i] += __shfl_xor_sync(0xffffffffu, l[i], o);
      put_row(sum_s + warp * N, l);
      float* wgt = wgt_s + warp * N;
      put_row(wgt, m);
      ok = all_meet();
      if (!ok) break;
      if (lane < N) {                                  // a head's quotient is taken once
        const float sum = (sum_s[lane] + sum_s[N + lane]) + (sum_s[2 * N + lane] + sum_s[3 * N + lane]);
        if (!whole && warp == 0 && lane < a.H) a.part_lse[part * a.H + lane] = sum > 0.f ? wgt[lane] + log2f(sum) : sum == 0.f ? -CUDART_INF_F : sum;
        wgt[lane] = sum > 0.f ? kLatent4Gain / sum : sum == 0.f ? 0.f : sum;      // a sum that is no number stays visible
      }
      __syncwarp();
      ok = mbar_wait_warp(&pv_done[(n - 1) & 1], ((n - 1) >> 1) & 1, abort_flag, a.status);
      if (!ok) break;
      tc_fence_after();
#pragma unroll 1
      for (int c = 0; c < 4 * N; c += 16) {            // 16 heads of this lane's dim of a 128-dim tile
        uint32_t ov[16];
        tmem_ld16(t_row + C::COL_O + c, ov);
        float x[16];
        const int h0 = c & (N - 1), d0 = (c / N) * 128 + warp * 32;
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
          const float4 v = *reinterpret_cast<const float4*>(wgt + h0 + i);
          x[i] = v.x; x[i + 1] = v.y; x[i + 2] = v.z; x[i + 3] = v.w;
        }
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] *= __uint_as_float(ov[i]);
        if (whole) {
          // two neighbouring dims to a word: the even lane takes the pair of the even head, the odd lane that of the odd one
          const bool even = !(lane & 1);
          __nv_bfloat16* o = out + (int64_t)h0 * kF4Dv + d0 + (lane & ~1);
#pragma unroll
          for (int i = 0; i < 16; i += 2) {
            const float y = __shfl_xor_sync(0xffffffffu, even ? x[i + 1] : x[i], 1);
            const int h = i + (lane & 1);
            if (h0 + h < a.H) *reinterpret_cast<uint32_t*>(o + h * kF4Dv) = even ? f4_pack(x[i], y) : f4_pack(y, x[i + 1]);
          }
        } else {
          float* o = a.part_o + (part * a.H + h0) * kF4Dv + d0 + lane;
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (h0 + i < a.H) o[i * kF4Dv] = x[i];
        }
      }
      tc_fence_before();
      ok = all_meet();                                 // sum_s may be written again
    }
  }

  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {                                   // a wait gave up: let the copies in flight land (bounded)
    if (threadIdx.x == 0)
      for (int w = 0; w < 64; ++w) __nanosleep(1000);
    __syncthreads();
  }
  if (warp == kF4MmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, C::COLS);
  }
}

// out = sum_p 2^(lse_p - M) o_p / sum_p 2^(lse_p - M) over the parts of a list that was cut: at most one a block, 32.  A lane finds one
// part and its weight (each thread for itself: 13 us for parts of one list, mostly 64-bit divisions).
constexpr int kF4Parts = 32;
__global__ void __launch_bounds__(128) sparse_mla_few4_merge_kernel(const Few4Args a) {
  __shared__ float weight_s[kF4Parts];
  const float *lse = grid_wait(a.part_lse), *part = grid_wait(a.part_o);
  const int t = a.rounds * a.ctas + blockIdx.x, h = blockIdx.y, d = threadIdx.x * 4, lane = threadIdx.x & 31;
  // the CTAs whose stretches have the list's first and last block
  auto cta_of = [&](int x) { return (int)(((int64_t)(x + 1) * a.rest_ctas - 1) / a.rest); };
  const int blk0 = blockIdx.x * a.list_blocks, c0 = a.per_list ? blockIdx.x * a.per_list : cta_of(blk0);
  const int parts = a.per_list ? a.per_list : cta_of(blk0 + a.list_blocks - 1) - c0 + 1;
  if (parts == 1) return;                              // whole
  const int first = 2 * c0 + (F4Piece::start_of(a, c0) >= blk0 ? 0 : 1);      // the others' stretches begin in this list
  auto slot_of = [&](int p) { return p == 0 ? first : 2 * (c0 + p); };
  if (threadIdx.x < 32) {
    const float x = lane < parts ? lse[(int64_t)slot_of(lane) * a.H + h] : -CUDART_INF_F;
    float mx = x;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    const float w = x == -CUDART_INF_F ? 0.f : exp2f(x - mx);      // NaN stays NaN
    float den = w;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) den += __shfl_xor_sync(0xffffffffu, den, o);
    weight_s[lane] = den == 0.f ? 0.f : w / den;
  }
  float4 v[8], acc = make_float4(0.f, 0.f, 0.f, 0.f);
  const float* src = part + (int64_t)h * kF4Dv + d;
  auto load = [&](int p) { return *reinterpret_cast<const float4*>(src + (int64_t)slot_of(p) * a.H * kF4Dv); };
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = i < parts ? load(i) : acc;
  __syncthreads();
  for (int p0 = 0; p0 < parts; p0 += 8) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float w = p0 + i < parts ? weight_s[p0 + i] : 0.f;
      if (w != 0.f) {                                  // a part of no weight has left no output
        acc.x += w * v[i].x; acc.y += w * v[i].y; acc.z += w * v[i].z; acc.w += w * v[i].w;
      }
      if (p0 + 8 + i < parts) v[i] = load(p0 + 8 + i);
    }
  }
  uint2 o;
  o.x = f4_pack(acc.x, acc.y);
  o.y = f4_pack(acc.z, acc.w);
  *reinterpret_cast<uint2*>(a.out + ((int64_t)t * a.H + h) * kF4Dv + d) = o;
}

int make_tmap_2d_bytes(CUtensorMap* m, const void* base, uint64_t rows, uint64_t inner_bytes, uint64_t row_pitch,
                       uint32_t box_bytes, uint32_t box_rows);

constexpr int kF4LeastBlocks = 2;                      // of a CTA, in calls that have few
constexpr int kF4PieceBlocks = 2;                      // what a further piece costs a CTA, in blocks

static int f4_list_blocks(int K) { return max(1, (K + kF4Blk - 1) / kF4Blk); }
static int f4_ctas(int T, int list_blocks, int sms) {
  return (int)min((int64_t)sms, max((int64_t)T, (int64_t)T * list_blocks / kF4LeastBlocks));
}
static size_t f4_parts_bytes(int ctas, int H) { return (size_t)2 * ctas * H * (kF4Dv + 1) * sizeof(float); }
size_t few4_workspace_bytes(int T, int H, int K) { return f4_parts_bytes(f4_ctas(T, f4_list_blocks(K), sm_count()), H); }

// The lists from row t0 of the call's T that one launch takes, and which CTA has what of them; without parts, every list in one piece.  A CTA's
// pieces fit its table: it has a list of each round, and its stretch lies in three others at most.
static void f4_plan(Few4Args& a, int t0, int T, int sms, bool parts) {
  a.row0 = t0;
  a.T = min(T - t0, kF4Pieces / 2 * sms);
  a.list_blocks = f4_list_blocks(a.K);
  a.ctas = parts ? f4_ctas(a.T, a.list_blocks, sms) : min(a.T, sms);
  a.rounds = parts ? a.T / a.ctas : (a.T + a.ctas - 1) / a.ctas;
  a.rest = max(0, a.T - a.rounds * a.ctas) * a.list_blocks;
  a.rest_ctas = min(a.ctas, max(1, a.rest / kF4LeastBlocks));
  // Equal parts of each list while they keep the GPU as busy: a CTA whose stretch lies in two lists pays for the second's Q, output and
  // start what two blocks take.  2048 keys, us with stretches of all blocks and so: 16 heads 24 rows 21.4, 19.1; 64 rows 34.6, 32.5; 32 heads
  // 64 rows 44.9, 42.3.
  a.per_list = 0;
  if (a.rest) {
    const int lists = a.rest / a.list_blocks, p = min(a.ctas / lists, max(1, a.list_blocks / kF4LeastBlocks));
    if ((a.list_blocks + p - 1) / p <= (a.rest + a.rest_ctas - 1) / a.rest_ctas + kF4PieceBlocks) {
      a.per_list = p;
      a.rest_ctas = lists * p;
    }
  }
}

// Walks the plans of a call of T rows on the host: for every block of every list how often a CTA has it (`seen`, [T, blocks of a list]), and the most pieces
// that a CTA has in a launch, or -1 where a piece lies outside its lists.
int few4_plan_probe(int T, int K, int sms, int parts, uint8_t* seen) {
  Few4Args a{};
  a.K = K;
  int most = 0;
  for (int t0 = 0; t0 < T; t0 += a.T) {
    f4_plan(a, t0, T, sms, parts != 0);
    for (int c = 0; c < a.ctas; ++c) {
      int n = 0;
      for (F4Piece pc(a, c); pc.next(a); ++n) {
        if (pc.t < 0 || pc.t >= a.T || pc.b0 < 0 || pc.b1 <= pc.b0 || pc.b1 > a.list_blocks) return -1;
        for (int b = pc.b0; b < pc.b1; ++b) ++seen[(int64_t)(t0 + pc.t) * a.list_blocks + b];
      }
      most = max(most, n);
    }
  }
  return most;
}

template <int N>
static int launch_few4(const void* q, const Few4Args& a, int overlapped, cudaStream_t stream) {
  using C = F4Cfg<N>;
  CUtensorMap tq;
  const int rc = make_tmap_2d_bytes(&tq, q, (uint64_t)a.T * a.H, kF4QBytes, kF4QBytes, 128, N);
  if (rc) return rc;
  auto kern = sparse_mla_few4_kernel<N>;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM) != cudaSuccess)
    return set_error(DSA_ERR_CUDA, "sparse_mla: cannot raise dynamic shared memory to %d", C::SMEM);
  launch_after(overlapped, kern, dim3(a.ctas), kF4Threads, C::SMEM, stream, tq, a);
  if (a.per_list > 1 || (!a.per_list && a.rest && (a.rest % a.rest_ctas || a.rest / a.rest_ctas % a.list_blocks)))      // some list may be cut
    launch_after(1, sparse_mla_few4_merge_kernel, dim3(a.T - a.rounds * a.ctas, a.H), 128, 0, stream, a);
  return check_launch("sparse_mla");
}

int sparse_mla_few4_launch(const void* q, const void* cache, const int32_t* block_table, int64_t table_stride, int tokens_per_seq, const int32_t* idx,
                           void* out, int T, int H, int K, int num_pages, int max_ctx, float scale, void* workspace, size_t workspace_bytes,
                           int32_t* status, int overlapped, cudaStream_t stream) {
  Few4Args a{};
  a.cache = static_cast<const uint8_t*>(cache);
  a.block_table = block_table;
  a.table_stride = table_stride;
  a.tokens_per_seq = tokens_per_seq;
  a.H = H; a.K = K; a.max_ctx = max_ctx;
  a.num_rows = num_pages * 64;
  a.scale_log2e = scale * 1.4426950408889634f * kLatent4Gain;
  a.status = status;
  for (int t0 = 0; t0 < T; t0 += a.T) {
    f4_plan(a, t0, T, sm_count(), /*parts=*/true);
    if (workspace && workspace_bytes >= f4_parts_bytes(a.ctas, H)) {
      a.part_o = static_cast<float*>(workspace);
      a.part_lse = a.part_o + (size_t)2 * a.ctas * H * kF4Dv;
    } else {
      f4_plan(a, t0, T, sm_count(), /*parts=*/false);
    }
    a.idx = idx + (int64_t)t0 * K;
    a.out = static_cast<__nv_bfloat16*>(out) + (int64_t)t0 * H * kF4Dv;
    const void* qt = static_cast<const uint8_t*>(q) + (size_t)t0 * H * kF4QBytes;
    const int rc = H <= 16 ? launch_few4<16>(qt, a, overlapped, stream) : launch_few4<32>(qt, a, overlapped, stream);
    if (rc) return rc;
  }
  return DSA_OK;
}

}  // namespace dsa
