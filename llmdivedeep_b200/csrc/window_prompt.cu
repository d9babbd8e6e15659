// MLA attention over a sliding window and the first tokens, prompts: bf16 query rows over bf16 latent rows (the arithmetic: window_mla.cuh).
//
// A persistent cluster of two CTAs takes units of 128 query rows (token, head) one after the other.  Within a unit it is the kernel of
// sparse_mla.cu: CTA c has half of the latent dims (its half of V and of the scores' contraction), the partial scores of a block of 64 keys
// cross over in fp32, each side runs the softmax, P.V accumulates in tensor memory.  What differs:
//   * a block is 64 rows of a stretch of keys, fetched by five TMA boxes; rows of one sequence that follow one another share the blocks, and what
//     each of them sees of a block is a 32-bit mask to a thread, from two ranges;
//   * blocks, query panels and the output's staging go through one ring of five buffers, in the order Q(u) Q(u) Q(u)+O(u - 1) K(u, 0) K(u, 1) ..., so that
//     the next unit's queries and keys are on their way while the last blocks of this one are worked on.  (The third entry has one query panel; the
//     output before is staged behind it.)  An entry of the ring costs a unit about as much as a block does;
//   * four more warps move Q into tensor memory and O out of it, so that the softmax goes from unit to unit without a pause.
// Roles: warps 0-15 exchange + softmax, 16 MMA issuer, 17 loads, 18 zeros in the rows behind the end of a stretch, 19 plans the next unit, 20-23 Q and O.
// Every wait is bounded (dsa_common.cuh); the two CTAs leave together through a cluster barrier.
// What bounds it: 1.17 us a block, of which the tensor pipe works 0.58: the softmax warps' chain, in which 32 KB of scores cross to the other SM and as many come back (with
// half of the bits it was 0.93; window_mla.cuh) -- a buffer is held for 5.8 us, load, exchange, softmax and P.V -- and the entries of the ring that a unit needs
// besides.  us a unit, four first tokens, by window: 128 heads 64 7.6, 512 15.3, 2048 43.3; 8 tokens x 16 heads 64 8.6, 512 14.9, 1024 24.2 (a unit of one block 6.8).
// 8192 tokens x 128 heads at 128K, window 4096: 10.3 to 10.5 ms = 890 to 910 TFLOP/s; packed prompts of 16 heads, window 512, 220 us for 64 us of operations:
// their units have few blocks, and the last round of units is a part of one.  40 tokens x 128 heads: 10.4 to 10.9 us, a chain of set-up and plan 1.2, loads 1.6 to 2,
// scores 0.9, exchange and softmax 1.8, P.V 0.6, output 2.2.
#include <cuda.h>
#include <cudaTypedefs.h>

#include "window_mla.cuh"

namespace dsa {

constexpr int kWpThreads = 768, kWpMmaWarp = 16, kWpLoadWarp = 17, kWpFixWarp = 18, kWpPlanWarp = 19, kWpOutWarp = 20;
constexpr int kWpRegsSoftmax = 88, kWpRegsRoles = 64, kWpRegsOut = 64;
static_assert(512 * kWpRegsSoftmax + 128 * kWpRegsRoles + 128 * kWpRegsOut <= kWpThreads * 80, "more registers than the launch has");
constexpr int kWpTokens = 34;                          // tokens of a unit at most
constexpr int kWpSegs = 2 * kWpTokens;                 // ... and stretches of keys: two for each sequence in it
struct PromptPlan {
  int blocks, blk_lo;                                  // blocks of the job (-1: there are no more jobs), and which is its first
  int full0, full1;                                    // keys that every row sees which sees any (one sequence in the unit)
  int row0, rows, part, tok0;                          // first query row, rows, part (-1: a whole unit), token of the first row
  int job, at, holes;                                  // drafts: key of the first draft; a key without a page
  int ready;                                           // of the first plan: written before the CTA's first barrier
  int4 sees[kWpTokens];                                // of the unit's tokens: {a0, a1, b0, b1}
  // Drafts: which of them each sees.  Prompts, of the first token of a stretch: the last keys of the stretch may be the sequence's first ones, behind its own,
  // and are known by their places in the tokens' `sees`; which is the first of those | how many << 32.
  uint64_t more[kWpTokens];
  int4 segs[kWpSegs + 1];                              // {first key, end, blocks before, tokens of the unit that it is for}
};
constexpr int kWpHead = 16;                            // first keys that come behind a stretch at most
constexpr int kWpPlans = 4;                            // jobs that are planned ahead of the one whose output is on its way
constexpr int kWpOffBars = kMlaBufs * kMlaKBytes + kWinXBytes;
constexpr int kWpOffPm = kWpOffBars + 640;
constexpr int kWpOffSums = kWpOffPm + kMlaPairBytes;   // [4][128] (m, l)
constexpr int kWpOffPlans = kWpOffSums + 4 * 128 * 8;
constexpr int kWpOffRedo = kWpOffPlans + kWpPlans * (int)sizeof(PromptPlan);
constexpr int kWpRedo = 12;                            // quadrants of jobs that a warp has on its list of rows to be done key by key
constexpr int kWpSmem = kWpOffRedo + 4 * kWpRedo * 8;
static_assert(kWpSmem <= 232448 && sizeof(PromptPlan) % 16 == 0, "shared memory budget of one CTA");

__device__ __forceinline__ float dot_bf16x2(uint32_t x, uint32_t y, float d) {
  d = fmaf(__uint_as_float(x << 16), __uint_as_float(y << 16), d);
  return fmaf(__uint_as_float(x & 0xffff0000u), __uint_as_float(y & 0xffff0000u), d);
}

// The first keys behind a stretch: which is the first, and how many.
template <bool DRAFTS>
__device__ __forceinline__ int2 head_of(const PromptPlan& p, const int4& seg) {
  if (DRAFTS) return make_int2(0, 0);
  const uint64_t x = p.more[seg.w & 0xffff];
  return make_int2((int)(uint32_t)x, (int)(x >> 32));
}

// The keys of a unit of drafts, all of one sequence: one stretch of its slots' rows.
__device__ __forceinline__ int draft_segs(const WinArgs& a, int n_tok, PromptPlan& p) {
  const int lane = threadIdx.x & 31, seq = p.tok0 / a.drafts.per_seq, i0 = p.tok0 - seq * a.drafts.per_seq, base = seq * a.pad;
  const Drafts dr = drafts_of(a.drafts, seq);
  if (i0 >= dr.m) return 0;
  const Slots all = slots_of(a, dr, 0, a.drafts.per_seq - 1), mine = slots_of(a, dr, i0, i0 + n_tok - 1);
  const int n = mine.n + mine.shift - all.shift;       // up to the last of its tokens, by the sequence's slots
  for (int t = lane; t < n_tok; t += 32) {
    const Sees s = sees_draft(a, dr, seq, i0 + t);
    p.sees[t] = i0 + t < dr.m ? make_int4(base, base + (all.shift ? min(s.a1, all.head) : s.a1), base + s.b0 - all.shift, base + s.b1 - all.shift) : make_int4(0, 0, 0, 0);
    p.more[t] = s.bits;
  }
  bool holes = false;
  for (int w = lane; w < (n + 31) / 32; w += 32) holes |= (a.valid[base / 32 + w] & low_bits(n - 32 * w)) != low_bits(n - 32 * w);
  holes = __any_sync(0xffffffffu, holes);
  if (lane == 0) {
    p.at = base + dr.ctx - dr.m - all.shift;
    p.holes = holes;
    p.segs[0] = make_int4(base, base + n, 0, (n_tok - 1) << 16);
    p.segs[1] = make_int4(0, 0, 0x7fffffff, 0);
    p.full0 = holes ? 0x7fffffff : base + mine.full0 + mine.shift - all.shift;
    p.full1 = base + mine.full1 + mine.shift - all.shift;
  }
  return (n + kMlaBlk - 1) / kMlaBlk;
}

// The keys of a unit, by one warp.  Neighbouring rows of a sequence whose windows touch share two stretches: its first keys and those of their windows.  Where
// the first keys fit into the last block of the other stretch they are no block of their own (16 heads, window 512, 14.9 us a unit, 16.4 to 18 without; 64
// heads, window 1024, 24.2 and 26.3 to 28).
template <bool DRAFTS>
__device__ __forceinline__ int build_segs(const WinArgs& a, int n_tok, PromptPlan& p) {
  if constexpr (DRAFTS) return draft_segs(a, n_tok, p);
  const int lane = threadIdx.x & 31;
  int n = 0, blocks = 0, runs = 0;
  int rk = 0, ra = 0, rlo = 0, rhi = 0, r0 = 0, r1 = -1;             // the run that is open (r1 >= r0)
  int full0 = 0, full1 = 0x7fffffff, heads = 0x7fffffff;
  auto put = [&](int lo, int hi, int head) {
    if (lo >= hi) return;
    if (lane == 0) {
      p.segs[n] = make_int4(lo, hi, blocks, r0 | r1 << 16);
      p.more[r0] = (uint32_t)rk | (uint64_t)head << 32;
    }
    ++n;
    blocks += (hi - lo + kMlaBlk - 1) / kMlaBlk;
  };
  auto close = [&]() {
    if (r1 < r0) return;
    ++runs;
    // (with a gap between the stretches every row sees all of the first keys)
    const int head = ra - rk, tail = (rhi - rlo) % kMlaBlk;
    if (rlo <= ra || head > kWpHead || tail == 0 || tail + head > kMlaBlk) {
      put(rk, rlo <= ra ? rhi : ra, 0);
      if (rlo > ra) put(rlo, rhi, 0);
    } else {
      put(rlo, rhi + head, head);
      for (int t = r0 + (lane - r0 & 31); t <= r1; t += 32)
        if (p.sees[t].y > p.sees[t].x) p.sees[t].x = rhi, p.sees[t].y = rhi + head;
    }
  };
  for (int base = 0; base < n_tok; base += 32) {
    const Sees mine = base + lane < n_tok ? sees_prompt(a, p.tok0 + base + lane) : Sees{};
    if (base + lane < n_tok) p.sees[base + lane] = make_int4(mine.a0, mine.a1, mine.b0, mine.b1);
    for (int j = 0; j < min(32, n_tok - base); ++j) {
      const int k = __shfl_sync(0xffffffffu, mine.a0, j), a1 = __shfl_sync(0xffffffffu, mine.a1, j), lo = __shfl_sync(0xffffffffu, mine.b0, j),
                hi = __shfl_sync(0xffffffffu, mine.b1, j);
      if (hi <= k) continue;                           // sees nothing
      full0 = max(full0, lo);
      full1 = min(full1, hi);
      heads = min(heads, a1);
      if (r1 >= r0 && k == rk && lo <= rhi && hi >= rlo) {
        ra = max(ra, a1);
        rlo = min(rlo, lo);
        rhi = max(rhi, hi);
      } else {
        close();
        r0 = base + j;
        rk = k; ra = a1; rlo = lo; rhi = hi;
      }
      r1 = base + j;
    }
  }
  close();
  if (lane == 0) {
    p.segs[n] = make_int4(0, 0, 0x7fffffff, 0);
    p.full0 = runs != 1 ? 0x7fffffff : full0 <= heads ? rk : full0;
    p.full1 = full1;
  }
  return blocks;
}

// A job: a whole unit, or a part of the keys of one.
struct JobRows {
  int part, n_split, split, row0, rows;                // part < 0: a whole unit
};
template <bool DRAFTS>
__device__ __forceinline__ JobRows job_rows(const WinArgs& a, int job) {
  JobRows j;
  j.part = job < a.n_full ? -1 : job - a.n_full;
  j.n_split = j.part < 0 ? 1 : a.n_split;
  j.split = j.part < 0 ? 0 : j.part % j.n_split;
  const int unit = j.part < 0 ? job : a.n_full + j.part / j.n_split, seq = DRAFTS ? unit / a.seq_units : 0, row = (unit - seq * a.seq_units) * a.unit_rows;
  j.row0 = seq * a.seq_rows + row;
  j.rows = min(a.unit_rows, a.seq_rows - row);
  return j;
}

// The J-th unit that has a draft in it, for ascending J; -1: there are fewer.  By a warp.
struct LiveUnits {
  int s0 = -32, before = 0, total = 0, upto = 0, own = 0;      // 32 sequences: their first, units before them, of them, of a lane's up to its own, its own
  __device__ __forceinline__ int find(const WinArgs& a, int J) {
    const int lane = threadIdx.x & 31, B = a.T / a.drafts.per_seq;
    while (J >= before + total) {
      before += total;
      s0 += 32;
      if (s0 >= B) return -1;
      own = s0 + lane < B ? (drafts_of(a.drafts, s0 + lane).m * a.H + a.unit_rows - 1) / a.unit_rows : 0;
      upto = own;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += y;
      }
      total = __shfl_sync(0xffffffffu, upto, 31);
    }
    const int l = __ffs(__ballot_sync(0xffffffffu, upto > J - before)) - 1;
    return (s0 + l) * a.seq_units + J - before - __shfl_sync(0xffffffffu, upto - own, l);
  }
};

// DRAFTS: units of the drafts of one sequence, over the rows of its slots.
template <bool DRAFTS>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kWpThreads, 1)
window_prompt_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_o, const __grid_constant__ CUtensorMap tmap_lat,
                     const __grid_constant__ CUtensorMap tmap_rope, const WinArgs a, const int jobs) {
  constexpr int NB = kMlaBufs;
  extern __shared__ __align__(1024) uint8_t smem[];            // the swizzled panels need 1024-byte alignment
  uint8_t* recv_s = smem + NB * kMlaKBytes;                    // the peer's partial score tile
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kWpOffBars);
  uint64_t* q_ready = bars + 0;                      // Q of a unit is in tensor memory
  uint64_t* qk_done = bars + 1;                      // the unit's scores have all been computed: Q's columns are free
  uint64_t* o_final = bars + 2;                      // the unit's last P.V
  uint64_t* o_free = bars + 3;                       // O has been read
  uint64_t* s_free = bars + 4;                       // a set has read S into registers
  uint64_t* p_full = bars + 5;                       // softmax -> MMA
  // by parity of the blocks, counted over all units: a set of softmax warps takes every second block
  uint64_t* s_full = bars + 6;                       // [2] MMA -> softmax
  uint64_t* pv_done = bars + 8;                      // [2] P.V of a block finished: O is quiescent, P is free
  uint64_t* pm_full = bars + 10;                     // [2][4 quadrants] both key halves' block maxima are in pm_s
  uint64_t* recv_full = bars + 18;                   // [16 warps] the peer's part of a partial tile has landed in recv_s
  uint64_t* xchg_free = bars + 34;                   // [16] the peer has read what this CTA's warp sent
  uint64_t* ring_full = bars + 50;                   // [5] a buffer is ready to be read (the output's: to be written)
  uint64_t* part_full = bars + 55;                   // [5] a block that is no whole one has landed: it is ready when its other rows are zeros
  uint64_t* ring_free = bars + 60;                   // [5] the four warps of Q and O, or P.V of a block and three arrivals with it
  uint64_t* plan_full = bars + 65;                   // [4]
  uint64_t* plan_free = bars + 69;                   // [4]
  uint64_t* sums_full = bars + 73;                   // the row sums of a unit, and whether a row must be done key by key
  uint64_t* sums_free = bars + 74;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 75);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  uint32_t* odd_s = tmem_slot + 2;                   // [4 quadrants] rows with a key that they do not see and that is no number
  uint16_t* pm_s = reinterpret_cast<uint16_t*>(smem + kWpOffPm);         // block maxima, rounded up to bf16
  float2* sums_s = reinterpret_cast<float2*>(smem + kWpOffSums);
  PromptPlan* plans = reinterpret_cast<PromptPlan*>(smem + kWpOffPlans);

  launch_dependents();                                         // (the kernel that merges the parts)
  const int cta = blockIdx.x & 1, peer = cta ^ 1;              // rank in the cluster = V half = contraction part
  const int pair = blockIdx.x >> 1, n_pairs = gridDim.x >> 1;
  const int warp = warp_index(), lane = threadIdx.x & 31;
  if (warp == 0) {
    for (int i = lane; i < 75; i += 32) {
      const uint32_t count = (i == 0 || i == 3 || i == 74 || (i >= 60 && i <= 64)) ? 4u      // q_ready, o_free, sums_free, ring_free: the warps of Q and O
                             : (i == 4 || i == 5) ? 8u                               // s_free, p_full: lane 0 of a set's warps
                             : (i >= 10 && i <= 17) ? 2u                             // pm_full: the two warps of a quadrant
                             : (i >= 69 && i <= 72) ? 23u                            // plan_free: all that read it
                             : i == 73 ? 16u                                         // sums_full
                                       : 1u;
      mbar_init(bars + i, count);
    }
    mbar_fence_init();
    if (lane < 5) const_cast<int*>(abort_flag)[lane] = 0;      // and odd_s
    if (lane == 5) tma_prefetch_desc(&tmap_q);
    if (lane == 6) tma_prefetch_desc(&tmap_lat);
    if (lane == 7) tma_prefetch_desc(&tmap_rope);
    if (lane == 8) tma_prefetch_desc(&tmap_o);
  } else if (warp == kWpMmaWarp) {
    tmem_alloc(tmem_slot, kMlaTmemCols);
    tmem_relinquish();
  }
  // The plan of a job, by a warp: its blocks (0: nothing is seen), all else in p.
  LiveUnits found;
  auto job_at = [&](int nth) { return DRAFTS && a.live ? found.find(a, nth) : nth < jobs ? nth : -1; };
  auto make_plan = [&](int job, const JobRows& j, PromptPlan& p) {
    const int tok0 = j.row0 / a.H;
    __syncwarp();
    if (lane == 0) p.tok0 = tok0;
    __syncwarp();
    const int blocks = build_segs<DRAFTS>(a, (j.row0 + j.rows - 1) / a.H - tok0 + 1, p);
    const int per = j.n_split == 1 ? blocks : (blocks + j.n_split - 1) / j.n_split, blk_lo = min(blocks, j.split * per), n = min(blocks, blk_lo + per) - blk_lo;
    if (lane == 0) {
      p.blocks = n; p.blk_lo = blk_lo;
      p.row0 = j.row0; p.rows = j.rows; p.part = j.part; p.job = job;
    }
    return n;
  };
  int job0 = -1, n0 = 0;
  if (warp == kWpPlanWarp) {                                   // the first one while the others set up
    job0 = job_at(pair);
    if (job0 >= 0) n0 = make_plan(job0, job_rows<DRAFTS>(a, job0), plans[0]);
    if (lane == 0) plans[0].ready = n0 > 0;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  cluster_arrive();                                            // the peer's barriers must be initialised before anything is sent to it
  bool left = false;                                           // this warp has arrived at the barrier that the pair leaves through

  auto wait = [&](uint64_t* bar, uint32_t phase) { return mla_wait(bar, phase & 1, abort_flag, a.status); };
  // the plan of this CTA's k-th job; false: give up
  const bool ready = plans[0].ready != 0;
  auto plan_of = [&](uint32_t k) { return (k == 0 && ready) || wait(&plan_full[k % kWpPlans], k / kWpPlans); };
  auto plan_done = [&](uint32_t k) {
    __syncwarp();
    if (lane == 0) mbar_arrive(&plan_free[k % kWpPlans]);
  };
  // the stretch of block g, looked for from the one before on
  auto seg_of = [&](const PromptPlan& p, int& at, int g) -> int4 {
    while (g >= p.segs[at + 1].z) ++at;
    return p.segs[at];
  };

  if (warp < 16) {
    regs_inc<kWpRegsSoftmax>();
    // ------------- partial-score exchange and softmax: thread = (row, half of a block's keys); as in sparse_mla.cu but for masks and units -------------
    const int qd = warp & 3, hf = (warp >> 2) & 1, set = warp >> 3;      // hf: key half; set: takes the blocks of that parity
    const int row = qd * 32 + lane;                    // TMEM lane
    const uint32_t t_row = tmem + (uint32_t(qd * 32) << 16);
    const uint32_t peer_xchg_free = mapa_u32(smem_u32(xchg_free + warp), peer);
    const uint32_t peer_recv_full = mapa_u32(smem_u32(recv_full + warp), peer);
    const uint8_t* recv = recv_s + (hf * 4 + qd) * kWinXWarp + lane * 16;      // this thread's part of the set's partial tile
    const uint32_t peer_recv = mapa_u32(smem_u32(recv), peer);
    auto pm_of = [&](uint32_t blk) -> uint16_t* { return pm_s + (blk & 3) * 256 + row; };      // [key half][row]
    auto raise = [&](float m_old, float bmax) { return bmax - m_old > kMaxRaise ? bmax : m_old; };   // -inf - -inf: stays
    auto pair_max = [&](const uint16_t* pm) {
      return fmaxf(__uint_as_float(uint32_t(pm[0]) << 16), __uint_as_float(uint32_t(pm[128]) << 16));
    };
    if (lane == 0) mbar_expect_tx(&recv_full[warp], kWinXWarp);
    cluster_wait();
    bool ok = true;
    uint32_t n = set, base = 0;                        // this set's next block, the first block of the unit, both of all blocks
    for (uint32_t k = 0; ok; ++k) {
      if (!(ok = plan_of(k))) break;
      const PromptPlan& p = plans[k % kWpPlans];
      const int blocks = p.blocks;
      if (blocks < 0) break;
      const int tok = row < p.rows ? (p.row0 + row) / a.H - p.tok0 : kWpTokens;      // kWpTokens: no row
      int at = 0;
      float m = -CUDART_INF_F, l = 0.f;                // m: reference of the last block seen; l: this thread's keys only
      bool odd = false;                                // what this row does not see is no number: P x V would let it in
      for (; n < base + blocks; n += 2) {
        const uint32_t ph = n >> 1;
        const bool begun = n > base;                   // there is a block of this unit before
        uint32_t sv[32];                               // this CTA's partial scores
        if (!(ok = wait(&s_full[set], ph))) break;
        tc_fence_after();
        tmem_ld32(t_row + kColS + 32 * hf, sv);
        tmem_wait_ld();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(s_free);            // the next block's scores may overwrite S now
        if (n > 0 && !(ok = wait(&xchg_free[warp ^ 8], (n - 1) >> 1))) break;      // the peer has read block n-1
        send_scores(peer_recv, peer_recv_full, sv);
        uint32_t seen = 0xffffffffu;                   // which of this thread's keys its row sees
        {
          const int blk = p.blk_lo + (int)(n - base);
          const int4 s = seg_of(p, at, blk);
          const int k0 = s.x + (blk - s.z) * kMlaBlk;
          if (!(k0 >= p.full0 && k0 + kMlaBlk <= p.full1)) {
            seen = 0u;
            if (tok < kWpTokens) {
              const int4 v = p.sees[tok];
              if (tok >= (s.w & 0xffff) && tok <= (s.w >> 16))
                seen = range_bits(v.x, v.y, k0 + 32 * hf) | range_bits(v.z, v.w, k0 + 32 * hf);
              if constexpr (DRAFTS) {
                seen |= draft_bits(p.more[tok], p.at, k0 + 32 * hf);
                if (p.holes) seen &= a.valid[(k0 >> 5) + hf];
              }
              seen &= low_bits(s.y - k0 - 32 * hf);
              if (v.y > v.x || v.w > v.z || (DRAFTS && p.more[tok] != 0)) {
                float z = 0.f;
#pragma unroll
                for (int i = 0; i < 32; ++i) z = fmaf((seen >> i) & 1u ? 0.f : __uint_as_float(sv[i]), 0.f, z);
                odd |= z != 0.f;                       // NaN
              }
            }
          }
        }
        // the reference of the block before, from that block's maxima: every thread follows the whole sequence by itself
        if (begun && !(ok = wait(&pm_full[(set ^ 1) * 4 + qd], (n - 1) >> 1))) break;
        const float m_own = m;                         // what l is relative to
        if (begun) m = raise(m, pair_max(pm_of(n - 1)));
        const float m_prev = m;
        if (!(ok = wait_scores(&recv_full[warp], ph & 1, abort_flag, a.status))) break;
        float s[32];                                   // raw scores; the (positive) scale is folded into the exponent's FMA
        add_scores(recv, sv, s);
        auto largest = [&]() {
          float bm[4] = {s[0], s[1], s[2], s[3]};      // four independent chains
#pragma unroll
          for (int i = 4; i < 32; ++i) bm[i & 3] = fmaxf(bm[i & 3], s[i]);
          return fmaxf(fmaxf(bm[0], bm[1]), fmaxf(bm[2], bm[3]));
        };
        const float top = largest();                   // of every value of the tile, seen or not
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
        if (lane == 0) mbar_expect_tx(&recv_full[warp], kWinXWarp);
        if (!(ok = wait(&pm_full[set * 4 + qd], ph))) break;
        m = raise(m_prev, pair_max(pm_of(n)));
        if (m != m_own && m_own != -CUDART_INF_F) l *= fast_exp2(m_own - m);      // (without a reference l is 0, or NaN, and stays so)
        bool waited_pv = n == 0;
        if (__any_sync(0xffffffffu, m != m_prev) && begun) {
          // O must be quiescent: P.V of the previous block has to be complete.  This thread scales its half of the columns.
          if (!(ok = wait(&pv_done[set ^ 1], (n - 1) >> 1))) break;
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
        float ps[4] = {0.f, 0.f, 0.f, 0.f};            // sums of the even and odd keys, two chains each
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
          float x0, x1;
          unpack_f32x2(fma_f32x2(pack_f32x2(s[i], s[i + 1]), scale2, m2), x0, x1);
          const float p0 = fast_exp2(x0), p1 = fast_exp2(x1);
          pk[i >> 1] = pack_bf16x2(p0, p1);
          add_bf16x2(pk[i >> 1], ps[i & 2], ps[(i & 2) + 1]);
        }
        l += (ps[0] + ps[1]) + (ps[2] + ps[3]);
        if (!waited_pv) {                              // P is single-buffered: P.V of the previous block, of whatever unit, must be done
          if (!(ok = wait(&pv_done[set ^ 1], (n - 1) >> 1))) break;
          tc_fence_after();
        }
        tmem_st16(t_row + kColP + 16 * hf, pk);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full);
      }
      if (!ok) break;
      base += blocks;
      if (k > 0 && !(ok = wait(sums_free, k - 1))) break;
      sums_s[(warp >> 2) * 128 + row] = make_float2(m, l);
      const uint32_t odds = __ballot_sync(0xffffffffu, odd);
      __syncwarp();
      if (lane == 0) {
        if (odds) atomicOr(odd_s + qd, odds);
        mbar_arrive(sums_full);
        mbar_arrive(&plan_free[k % kWpPlans]);
      }
    }
  } else if (warp >= kWpOutWarp) {
    regs_dec<kWpRegsOut>();
    // ------------- Q into tensor memory, O out of it: thread = row -------------
    const int qd = warp & 3, row = qd * 32 + lane;
    const uint32_t t_row = tmem + (uint32_t(qd * 32) << 16);
    bool ok = true;
    uint2* redo_s = reinterpret_cast<uint2*>(smem + kWpOffRedo) + qd * kWpRedo;
    int redos = 0;
    // A buffer goes back when all four warps have said that they are done with it.  (They do not meet at a barrier: one may have given up, and a barrier has no limit.)
    auto give_back = [&](uint32_t e) {
      __syncwarp();
      if (lane == 0) mbar_arrive(&ring_free[e % NB]);
    };
    auto drain = [&](uint32_t k, uint32_t e, bool last) {      // the output of job k, staged in entry e, of the last job one of its own
      const PromptPlan& p = plans[k % kWpPlans];
      const int row0 = p.row0, rows = p.rows, part = p.part;
      const int tok = row < rows ? (row0 + row) / a.H - p.tok0 : 0;
      const int4 v = row < rows ? p.sees[tok] : make_int4(0, 0, 0, 0);
      const bool any = v.y > v.x || v.w > v.z || (DRAFTS && row < rows && p.more[tok] != 0);      // the row sees something
      ok = wait(sums_full, k) && wait(o_final, k) && wait(&ring_full[e % NB], e / NB);
      if (!ok) return;
      tc_fence_after();
      const uint32_t odd = odd_s[qd];
      float mt = -CUDART_INF_F, l = 0.f;
#pragma unroll
      for (int u = 0; u < 4; ++u) mt = fmaxf(mt, sums_s[u * 128 + row].x);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const float2 ml = sums_s[u * 128 + row];
        l += ml.x != -CUDART_INF_F ? ml.y * fast_exp2(ml.x - mt) : ml.y;
      }
      __syncwarp();
      if (lane == 0) {
        odd_s[qd] = 0;
        mbar_arrive(sums_free);
      }
      if (!any) l = 0.f;                               // a block that every other row sees is not masked
      const float inv = l > 0.f ? 1.f / l : l;         // (a NaN stays one)
      const bool by_tma = part < 0 && qd * 32 + 32 <= rows;
      // A key that a row does not see and that is no number has come in through 0 x NaN, unless the row is none anyway: done again when all jobs are done.
      const uint32_t again = __ballot_sync(0xffffffffu, (odd >> lane & 1u) && any && l == l);
      if (again) {
        if (lane == 0 && redos < kWpRedo) redo_s[redos] = make_uint2(p.job, again);
        ++redos;
      }
      if (part >= 0)                                   // what this CTA's half of the columns is weighted with
        a.part_lse[((int64_t)part * 2 + cta) * 128 + row] = l > 0.f ? mt + log2f(l) : l == 0.f ? -CUDART_INF_F : l;
      {
        // pieces of 32 rows x 32 columns, two to a warp, of the last job four
        uint8_t* const stage0 = smem + (e % NB) * kMlaKBytes + (last ? qd * 8192 : kMlaQPanelBytes + qd * 4096) + lane * 64;
        const uint32_t wrap = last ? 3 * 2048 : 2048;
        __nv_bfloat16* const orow = a.out + (int64_t)(row0 + row) * kMlaDv + cta * kMlaDvHalf;
        const uint64_t inv2 = pack_f32x2(inv, inv);
        const bool blind = __any_sync(0xffffffffu, !any);
        auto scaled = [&](uint32_t (&ov)[16]) {
#pragma unroll
          for (int i = 0; i < 16; i += 2) {
            float x, y;
            unpack_f32x2(mul_f32x2(pack_f32x2(__uint_as_float(ov[i]), __uint_as_float(ov[i + 1])), inv2), x, y);
            ov[i] = __float_as_uint(x);
            ov[i + 1] = __float_as_uint(y);
          }
          if (blind) {                                 // a row that sees nothing: zeros, whatever the blocks of the others gave it
#pragma unroll
            for (int i = 0; i < 16; ++i) ov[i] = any ? ov[i] : 0u;
          }
        };
        auto eight = [&](const uint32_t (&ov)[16], int i) {
          return make_uint4(pack_bf16x2(__uint_as_float(ov[i]), __uint_as_float(ov[i + 1])), pack_bf16x2(__uint_as_float(ov[i + 2]), __uint_as_float(ov[i + 3])),
                            pack_bf16x2(__uint_as_float(ov[i + 4]), __uint_as_float(ov[i + 5])), pack_bf16x2(__uint_as_float(ov[i + 6]), __uint_as_float(ov[i + 7])));
        };
        // the next sixteen columns are on their way while these are written; with every address known beforehand
        uint32_t ov[2][16];
        tmem_ld16(t_row + kColO, ov[0]);
        if (by_tma) {
#pragma unroll
          for (int c = 0; c < kMlaDvHalf; c += 16) {
            uint32_t (&now)[16] = ov[(c >> 4) & 1];
            tmem_wait_ld();
            if (c + 16 < kMlaDvHalf) tmem_ld16(t_row + kColO + c + 16, ov[((c >> 4) & 1) ^ 1]);
            if (c >= 64 && (c & 31) == 0 && (!last || c >= 128)) {      // the store of two, or four, pieces before has read its own
              if (lane == 0) {
                if (last) asm volatile("cp.async.bulk.wait_group.read 3;" ::: "memory");
                else asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
              }
              __syncwarp();
            }
            scaled(now);
            uint8_t* stage = stage0 + (((c >> 5) * 2048) & wrap);
            *reinterpret_cast<uint4*>(stage + (((((c & 31) >> 3) + 0) ^ (lane >> 1 & 3)) << 4)) = eight(now, 0);
            *reinterpret_cast<uint4*>(stage + (((((c & 31) >> 3) + 1) ^ (lane >> 1 & 3)) << 4)) = eight(now, 8);
            if ((c & 31) == 16) {
              fence_async_smem();                      // the store reads the piece through the async proxy
              __syncwarp();
              if (lane == 0) {
                tma_store_2d(&tmap_o, stage, (cta * 8 + (c >> 5)) * 16, row0 + qd * 32);      // x in 4-byte units: 16 per 32 columns
                asm volatile("cp.async.bulk.commit_group;" ::: "memory");
              }
            }
          }
        } else {
#pragma unroll 1
          for (int c = 0; c < kMlaDvHalf; c += 16) {
            tmem_ld16(t_row + kColO + c, ov[0]);
            tmem_wait_ld();
            scaled(ov[0]);
            if (row < rows && part >= 0) {
              float4* po = reinterpret_cast<float4*>(a.part_o + ((int64_t)part * 128 + row) * kMlaDv + cta * kMlaDvHalf + c);
#pragma unroll
              for (int i = 0; i < 16; i += 4)
                po[i >> 2] = make_float4(__uint_as_float(ov[0][i]), __uint_as_float(ov[0][i + 1]), __uint_as_float(ov[0][i + 2]), __uint_as_float(ov[0][i + 3]));
            } else if (row < rows) {
              *reinterpret_cast<uint4*>(orow + c) = eight(ov[0], 0);
              *reinterpret_cast<uint4*>(orow + c + 8) = eight(ov[0], 8);
            }
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(o_free);
      plan_done(k);
      if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");      // the buffer may be written again
      __syncwarp();
      give_back(e);
    };
    uint32_t e = 0, k = 0;
    for (;; ++k) {
      if (!(ok = plan_of(k))) break;
      const int n = __shfl_sync(0xffffffffu, plans[k % kWpPlans].blocks, 0);
      if (n < 0) break;
      if (k > 0 && !(ok = wait(qk_done, k - 1))) break;
      for (int j = 0; j < 3; ++j, ++e) {
        if (!(ok = wait(&ring_full[e % NB], e / NB))) break;
        // this row of two Q panels, swizzled shared memory -> packed bf16 pairs in tensor memory
#pragma unroll 1
        for (int hp = 0; hp < (j < 2 ? 4 : 2); ++hp) {
          uint32_t qv[16];
          const uint8_t* src = smem + (e % NB) * kMlaKBytes + (hp >> 1) * kMlaQPanelBytes + row * 128;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const uint4 w = *reinterpret_cast<const uint4*>(src + ((((hp & 1) * 4 + c) ^ (row & 7)) << 4));
            qv[4 * c + 0] = w.x; qv[4 * c + 1] = w.y; qv[4 * c + 2] = w.z; qv[4 * c + 3] = w.w;
          }
          tmem_st16(t_row + kColQ + (4 * j + hp) * 16, qv);
        }
        if (j < 2 || k == 0) give_back(e);
      }
      if (!ok) break;
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_ready);
      if (k == 0) {                                    // nothing remote is ever left to do for this warp
        cluster_wait();
        cluster_arrive();
        left = true;
      }
      if (k > 0) drain(k - 1, e - 1, false);           // the output of the unit before is staged behind the last query panel
      if (!ok) break;
      e += n;
    }
    if (ok && k > 0) drain(k - 1, e, true);
    if (redos > 0 && ok) ok = wait(&plan_free[(k - 1) % kWpPlans], (k - 1) / kWpPlans);      // nobody reads the last job's plan, nor one before it
    if (redos > 0) {                                   // what is written again has been written
      if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
      __syncwarp();
    }
    // Rare: rows key by key over what they see of their job's blocks, this CTA's half of the output from whole scores.  Nobody waits for this warp now (but at the
    // barrier that the pair leaves through, which has no limit).  With more on the list than it holds: every row of the pair's jobs.
    const int redo_jobs = redos > kWpRedo ? (jobs - pair + n_pairs - 1) / n_pairs : redos;
    LiveUnits units;
#pragma unroll 1
    for (int x = 0; ok && x < redo_jobs; ++x) {
      int job = redos > kWpRedo ? pair + x * n_pairs : (int)redo_s[x].x;
      if (DRAFTS && a.live && redos > kWpRedo && (job = units.find(a, job)) < 0) break;
      uint32_t mask = redos > kWpRedo ? 0xffffffffu : redo_s[x].y;
      PromptPlan& p = plans[qd];                       // each warp its own; of the jobs' plans nobody needs more than `blocks` now
      const JobRows j = job_rows<DRAFTS>(a, job);
      if (j.rows < qd * 32 + 32) mask &= low_bits(j.rows - qd * 32);
      __syncwarp();
      if (lane == 0) p.tok0 = j.row0 / a.H;
      __syncwarp();
      const int blocks = build_segs<DRAFTS>(a, (j.row0 + j.rows - 1) / a.H - j.row0 / a.H + 1, p);
      __syncwarp();
      const int per = (blocks + j.n_split - 1) / j.n_split, blk_lo = min(blocks, j.split * per), n_blk = min(blocks, blk_lo + per) - blk_lo;
#pragma unroll 1
      for (; mask; mask &= mask - 1) {
        const int r = qd * 32 + __ffs(mask) - 1, tok = (j.row0 + r) / a.H - p.tok0;
        const int4 sees = p.sees[tok];
        // a lane has values 8 lane .. of either half of the latent and two rope values
        const uint4* qp = reinterpret_cast<const uint4*>(a.q + (int64_t)(j.row0 + r) * kMlaDqk);
        const uint4 q0 = __ldg(qp + lane), q1 = __ldg(qp + 32 + lane);
        const uint32_t qr = __ldg(reinterpret_cast<const uint32_t*>(qp + 64) + lane);
        float rm = -CUDART_INF_F, rl = 0.f, o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        int at = 0;
#pragma unroll 1
        for (int n = 0; n < 2 * n_blk; ++n) {
          const int blk = blk_lo + (n >> 1);
          const int4 s = seg_of(p, at, blk);
          const int k0 = s.x + (blk - s.z) * kMlaBlk + 32 * (n & 1);
          uint32_t todo = range_bits(sees.x, sees.y, k0) | range_bits(sees.z, sees.w, k0);
          if constexpr (DRAFTS) todo = (todo | draft_bits(p.more[tok], p.at, k0)) & a.valid[k0 >> 5];
          todo &= low_bits(s.y - k0);
          if (tok < (s.w & 0xffff) || tok > (s.w >> 16)) todo = 0;
#pragma unroll 1
          for (; todo; todo &= todo - 1) {
            int key = k0 + __ffs(todo) - 1;
            const int2 head = head_of<DRAFTS>(p, s);
            if (key >= s.y - head.y) key += head.x - (s.y - head.y);
            const uint4* kp = reinterpret_cast<const uint4*>(a.kv + (int64_t)key * (kMlaDqk * 2));
            const uint4 v0 = __ldg(kp + lane), v1 = __ldg(kp + 32 + lane);
            float d = dot_bf16x2(qr, __ldg(reinterpret_cast<const uint32_t*>(kp + 64) + lane), 0.f);
            d = dot_bf16x2(q0.x, v0.x, d); d = dot_bf16x2(q0.y, v0.y, d); d = dot_bf16x2(q0.z, v0.z, d); d = dot_bf16x2(q0.w, v0.w, d);
            d = dot_bf16x2(q1.x, v1.x, d); d = dot_bf16x2(q1.y, v1.y, d); d = dot_bf16x2(q1.z, v1.z, d); d = dot_bf16x2(q1.w, v1.w, d);
#pragma unroll
            for (int y = 16; y > 0; y >>= 1) d += __shfl_xor_sync(0xffffffffu, d, y);
            const float sc = d * a.scale_log2e, mx = fmaxf(rm, sc), ref = mx == -CUDART_INF_F ? 0.f : mx;
            const float keep = rm == -CUDART_INF_F ? 0.f : exp2f(rm - ref), pr = exp2f(sc - ref);
            const uint32_t mine[4] = {cta ? v1.x : v0.x, cta ? v1.y : v0.y, cta ? v1.z : v0.z, cta ? v1.w : v0.w};
            rm = mx;
            rl = rl * keep + pr;
#pragma unroll
            for (int i = 0; i < 8; ++i) o[i] = o[i] * keep + pr * __uint_as_float(i & 1 ? mine[i >> 1] & 0xffff0000u : mine[i >> 1] << 16);
          }
        }
        const float ri = rl > 0.f ? 1.f / rl : rl;
        if (j.part >= 0) {
          float4* po = reinterpret_cast<float4*>(a.part_o + ((int64_t)j.part * 128 + r) * kMlaDv + cta * kMlaDvHalf + lane * 8);
          po[0] = make_float4(o[0] * ri, o[1] * ri, o[2] * ri, o[3] * ri);
          po[1] = make_float4(o[4] * ri, o[5] * ri, o[6] * ri, o[7] * ri);
          if (lane == 0) a.part_lse[((int64_t)j.part * 2 + cta) * 128 + r] = rl > 0.f ? rm + log2f(rl) : rl == 0.f ? -CUDART_INF_F : rl;
        } else {
          reinterpret_cast<uint4*>(a.out + (int64_t)(j.row0 + r) * kMlaDv + cta * kMlaDvHalf)[lane] =
              make_uint4(pack_bf16x2(o[0] * ri, o[1] * ri), pack_bf16x2(o[2] * ri, o[3] * ri), pack_bf16x2(o[4] * ri, o[5] * ri), pack_bf16x2(o[6] * ri, o[7] * ri));
        }
      }
    }
  } else {
    regs_dec<kWpRegsRoles>();
    auto load_keys = [&](uint32_t buf, int key0, uint64_t* full) {
      uint8_t* dst = smem + buf * kMlaKBytes;
      if (lane < 4) tma_load_2d(dst + lane * kMlaKPanelBytes, &tmap_lat, (cta * 4 + lane) * 32, key0, full);      // x in 4-byte units
      else if (lane == 4) tma_load_2d(dst + kMlaRopeOff, &tmap_rope, kMlaDv / 2 + cta * 16, key0, full);
      __syncwarp();
    };
    if (warp == kWpMmaWarp) {
      // ------------------------------- MMA issuer -------------------------------
      // Of a unit the scores of a block, then P.V two blocks behind; across units P.V of the last but one, the next unit's first scores, P.V of the last.
      constexpr uint32_t idesc_qk = umma_idesc(1, 1, 0, 0, 128, kMlaBlk);
      constexpr uint32_t idesc_pv = umma_idesc(1, 1, 0, 1, 128, kMlaDvHalf);
      const uint64_t kdesc0 = umma_smem_desc(smem_u32(smem), 16, 1024, kSwz128);
      const uint64_t vdesc0 = umma_smem_desc(smem_u32(smem), kMlaKPanelBytes, 1024, kSwz128);
      const uint64_t rdesc0 = umma_smem_desc(smem_u32(smem + kMlaRopeOff), 16, 512, kSwz64);
      const uint32_t rope_ks = 2 * cta;                  // this CTA's two K-steps of the rope panel
      // What this warp does beside issuing is on the path from block to block (930 cycles of a block are the issue itself), so it counts in steps and walks
      // one loop: three waits, the scores of block i, P.V of block i - 2 -- in a unit's first turn of the last block before it.
      uint32_t gp = 0;                                   // parity of the next block, counted over all units
      uint32_t buf = 0, ring = 0;                        // the next entry's buffer, and the parity of its use
      uint32_t vbuf = 0;                                 // buffer of the next P.V's block
      int n_last = 0;                                    // blocks of the unit before
      bool ok = true;
      auto skip = [&](uint32_t by) {
        buf += by;
        if (buf >= NB) {
          buf -= NB;
          ring ^= 1;
        }
      };
      auto issue_pv = [&](uint32_t parity, bool first, bool last) {
        tc_fence_after();
        if (elect_one()) {
          const uint64_t vd = vdesc0 + uint64_t(vbuf) * (kMlaKBytes >> 4);
#pragma unroll
          for (int ks = 0; ks < kMlaBlk / 16; ++ks)      // 16 keys per step: 16 rows x 128 B further into each panel
            umma_f16_ts(tmem + kColO, tmem + kColP + 8 * ks, vd + ks * (2048 >> 4), idesc_pv, !first || ks != 0);
          asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0], 3;" ::"r"(smem_u32(&ring_free[vbuf])) : "memory");
          umma_commit(&ring_free[vbuf]);
          umma_commit(&pv_done[parity]);
          if (last) umma_commit(o_final);
        }
        __syncwarp();
        vbuf = vbuf == NB - 1 ? 0 : vbuf + 1;
      };
      for (uint32_t k = 0; ok; ++k) {
        if (!(ok = plan_of(k))) break;
        const int n = __reduce_max_sync(0xffffffffu, plans[k % kWpPlans].blocks);      // -1: no more
        plan_done(k);
        // What is left of the unit before: P.V of its last two blocks.  The last one goes behind the first scores of this unit, but for the only block of a
        // unit, which holds the buffer that this unit's first block is to come to.
        if (n_last == 1 && k > 1) ok = wait(o_free, k - 2);
        if (ok && n_last > 0) ok = wait(p_full, n_last > 1 ? gp : gp ^ 1);
        if (!ok) break;
        if (n_last > 0) {
          if (n_last == 2 && k > 1 && !(ok = wait(o_free, k - 2))) break;
          issue_pv(n_last > 1 ? gp : gp ^ 1, n_last <= 2, n_last == 1);
        }
        if (n < 0) {
          if (n_last > 1 && (ok = wait(p_full, gp ^ 1))) issue_pv(gp ^ 1, false, true);
          break;
        }
        skip(3);                                         // Q
        const uint32_t vfirst = buf;
        ok = wait(q_ready, k);
#pragma unroll 1
        for (int i = 0; i < n && ok; ++i) {
          ok = wait(&ring_full[buf], ring);
          if (ok && (k > 0 || i > 0)) ok = wait(s_free, gp ^ 1);
          if (!ok) break;
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
            umma_commit(&s_full[gp]);
            if (i == n - 1) umma_commit(qk_done);
          }
          __syncwarp();
          if (i >= 2 || (i == 0 && n_last > 1)) {
            const uint32_t parity = i >= 2 ? gp : gp ^ 1;
            ok = wait(p_full, parity);
            if (ok && i == 2 && k > 0) ok = wait(o_free, k - 1);       // the first P.V of the unit: the output before has been read
            if (!ok) break;
            issue_pv(parity, i == 2, i == 0);
          }
          if (i == 0) vbuf = vfirst;
          gp ^= 1;
          skip(1);
        }
        n_last = n;
      }
    } else if (warp == kWpLoadWarp) {
      // ------------------------------- loads -------------------------------
      uint32_t e = 0;
      bool ok = true;
      auto claim = [&](uint64_t* full, uint32_t bytes) {      // the next buffer, for a load of so many bytes; 0: to be written by others
        if (e >= NB) ok = wait(&ring_free[e % NB], e / NB - 1);
        if (!ok) return;
        if (lane == 0) {
          if (bytes) mbar_expect_tx(full + e % NB, bytes);
          else mbar_arrive(full + e % NB);
        }
        __syncwarp();
      };
      for (uint32_t k = 0; ok; ++k) {
        if (!(ok = plan_of(k))) break;
        const PromptPlan& p = plans[k % kWpPlans];
        const int n = p.blocks, row0 = p.row0, blk_lo = p.blk_lo;
        if (n < 0) {
          if (k > 0) claim(ring_full, 0);                           // the last unit's output
          break;
        }
        for (int j = 0; j < 3 && ok; ++j) {              // Q: panels 2 j and 2 j + 1
          if (k == 0 && j == 2) {
            ++e;
            break;
          }
          claim(ring_full, j < 2 ? 2 * kMlaQPanelBytes : kMlaQPanelBytes);
          const int lp = 2 * j + lane;                   // x in 4-byte units: 32 per panel
          if (ok && lane < 2 && lp < kMlaPanels)
            tma_load_2d(smem + (e % NB) * kMlaKBytes + lane * kMlaQPanelBytes, &tmap_q, (lp < 4 ? cta * 4 + lp : 8) * 32, row0, &ring_full[e % NB]);
          __syncwarp();
          ++e;
        }
        int at = 0;
        for (int i = 0; i < n && ok; ++i) {
          const int4 s = seg_of(p, at, blk_lo + i);
          const int key0 = s.x + (blk_lo + i - s.z) * kMlaBlk;
          uint64_t* full = s.y - head_of<DRAFTS>(p, s).y - key0 < kMlaBlk ? part_full : ring_full;
          if (k > 0 || i > 0) {
            claim(full, kMlaKBytes);
            if (!ok) break;
            load_keys(e % NB, key0, full + e % NB);
          }
          ++e;
        }
        plan_done(k);
      }
    } else if (warp == kWpFixWarp) {
      // ---- blocks that are not whole: the rows behind the end of the stretch become the sequence's first keys, where they come there, and zeros, whatever they are
      // (P is 0 there, and 0 x NaN is none).  No buffer is loaded again before what this warp does with it is done and used, so it is never two of a barrier's phases behind ----
      uint32_t e = 0, used = 0;                          // parity of each buffer's part_full
      bool ok = true;
      for (uint32_t k = 0; ok; ++k) {
        if (!(ok = plan_of(k))) break;
        const PromptPlan& p = plans[k % kWpPlans];
        const int n = p.blocks, blk_lo = p.blk_lo;
        if (n < 0) break;
        e += 3;
        int at = 0;
        for (int i = 0; i < n && ok; ++i) {
          const int4 s = seg_of(p, at, blk_lo + i);
          const int2 head = head_of<DRAFTS>(p, s);
          const int rows = s.y - head.y - s.x - (blk_lo + i - s.z) * kMlaBlk;
          const uint32_t buf = e % NB;
          if (k == 0 && i == 0) {                        // (the first block's loads: while others see to the queries')
            uint64_t* full = (rows < kMlaBlk ? part_full : ring_full) + buf;
            if (lane == 0) mbar_expect_tx(full, kMlaKBytes);
            __syncwarp();
            load_keys(buf, s.y - head.y - rows, full);
          }
          if (rows < kMlaBlk) {
            uint8_t* dst = smem + buf * kMlaKBytes;
            // a lane has 16 bytes of each of their latent halves, and of every eighth row's rope values; the first loads are under way before the block has landed
            const uint8_t* src = a.kv + (int64_t)head.x * (kMlaDqk * 2);
            uint4 v[4], x;
            auto load = [&](int r0) {
#pragma unroll
              for (int j = 0; j < 4; ++j)
                if (r0 + j < head.y) v[j] = __ldg(reinterpret_cast<const uint4*>(src + (r0 + j) * (kMlaDqk * 2) + cta * kMlaDvHalf * 2) + lane);
              if (r0 + (lane >> 2) < min(head.y, r0 + 4)) x = __ldg(reinterpret_cast<const uint4*>(src + (r0 + (lane >> 2)) * (kMlaDqk * 2) + kMlaDv * 2 + cta * 64) + (lane & 3));
            };
            load(0);
            if (!(ok = wait(&part_full[buf], used >> buf))) break;
            used ^= 1u << buf;
#pragma unroll 1
            for (int r0 = 0; r0 < head.y; r0 += 4) {
              if (r0 > 0) load(r0);
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const int r = rows + r0 + j;
                if (r0 + j < head.y) *reinterpret_cast<uint4*>(dst + (lane >> 3) * kMlaKPanelBytes + r * 128 + (((lane & 7) ^ (r & 7)) << 4)) = v[j];
              }
              const int r = rows + r0 + (lane >> 2);
              if (r0 + (lane >> 2) < min(head.y, r0 + 4)) *reinterpret_cast<uint4*>(dst + kMlaRopeOff + r * 64 + (((lane & 3) ^ (r >> 1 & 3)) << 4)) = x;
            }
            uint8_t* zero = dst + (lane >> 3) * kMlaKPanelBytes + (lane & 7) * 16;
#pragma unroll 4
            for (int r = rows + head.y; r < kMlaBlk; ++r) *reinterpret_cast<uint4*>(zero + r * 128) = make_uint4(0, 0, 0, 0);
            for (int c = 4 * (rows + head.y) + lane; c < 4 * kMlaBlk; c += 32) *reinterpret_cast<uint4*>(dst + kMlaRopeOff + c * 16) = make_uint4(0, 0, 0, 0);
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&ring_full[buf]);
          }
          ++e;
        }
        plan_done(k);
      }
    } else if (warp == kWpPlanWarp) {
      // ------------------------------- plans -------------------------------
      uint32_t k = 0;
      bool ok = true, mine = true;                       // the buffer of plan k is this warp's: the first one from the start
      for (int next = pair; ok && !aborted_warp(abort_flag); next += n_pairs) {
        const int job = next == pair ? job0 : job_at(next);
        if (!mine) ok = wait(&plan_free[k % kWpPlans], (k / kWpPlans) + 1);
        mine = true;
        PromptPlan& p = plans[k % kWpPlans];
        if (!ok) break;
        if (job < 0) {
          if (lane == 0) {
            p.blocks = -1;
            mbar_arrive(&plan_full[k % kWpPlans]);
          }
          break;
        }
        const JobRows j = job_rows<DRAFTS>(a, job);
        const int n = next == pair ? n0 : make_plan(job, j, p);
        if (n == 0) {                                    // nothing seen: zeros (a part: weight zero when they are merged)
          if (j.part < 0) {
            for (int r = 0; r < j.rows; ++r)
              reinterpret_cast<uint4*>(a.out + (int64_t)(j.row0 + r) * kMlaDv + cta * kMlaDvHalf)[lane] = make_uint4(0, 0, 0, 0);
          } else {
            for (int r = lane; r < 128; r += 32) a.part_lse[((int64_t)j.part * 2 + cta) * 128 + r] = -CUDART_INF_F;
          }
          continue;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&plan_full[k % kWpPlans]);
        if (k == 0 && lane == 0) {                       // the third entry of the first job: three warps share what it waits for
          mbar_expect_tx(ring_full + 2, kMlaQPanelBytes);
          tma_load_2d(smem + 2 * kMlaKBytes, &tmap_q, 8 * 32, j.row0, ring_full + 2);
        }
        __syncwarp();
        ++k;
        mine = false;
      }
    }
  }

  __syncwarp();
  if (warp >= 16 && !left) cluster_wait();           // the wait that pairs with the arrive above (softmax: before its first remote access)
  if (!left) cluster_arrive();                       // remote accesses, if any, are behind this warp: the others need not wait for the output
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    // a wait gave up: let the copies that may still be in flight into this CTA land (bounded) before its shared memory goes away
    if (threadIdx.x == 0)
      for (int w = 0; w < 64; ++w) __nanosleep(1000);
    __syncthreads();
  }
  cluster_wait();                 // neither CTA leaves while the other may still copy into it or arrive on its barriers
  if (warp == kWpMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, kMlaTmemCols);
  }
}

// ---- launches --------------------------------------------------------------------------------------------------------
static int prompt_unit_rows(int H) { return H >= 4 ? 128 : 32 * H; }
static int64_t prompt_units(int T, int H) { return ((int64_t)T * H + prompt_unit_rows(H) - 1) / prompt_unit_rows(H); }
size_t window_mla_prefill_workspace(int T, int H, int window, int first) {
  return window_workspace(prompt_units(T, H), window_keys(H, window, first, T, 0x7fffffff));
}

template <bool DRAFTS>
static int launch_prompt(WinArgs a, int64_t units, int64_t keys, void* workspace, size_t workspace_bytes, cudaStream_t stream) {
  window_plan(a, units, keys, workspace, workspace_bytes);
  const int64_t rows = (int64_t)a.T * a.H;
  CUtensorMap tq, to, tl, tr;
  int rc = make_tmap_2d_bytes(&tq, a.q, rows, kMlaDqk * 2, kMlaDqk * 2, 128, 128);
  if (!rc) rc = make_tmap_2d_bytes(&to, a.out, rows, kMlaDv * 2, kMlaDv * 2, 64, 32);
  if (rc) return rc;
  tl = tr = tq;
  if (a.S > 0) {
    rc = make_tmap_2d_bytes(&tl, a.kv, a.S, kMlaDqk * 2, kMlaDqk * 2, 128, kMlaBlk);
    if (!rc) rc = make_tmap_2d_bytes(&tr, a.kv, a.S, kMlaDqk * 2, kMlaDqk * 2, 64, kMlaBlk);
    if (rc) return rc;
  }
  auto kern = window_prompt_kernel<DRAFTS>;
  static uint64_t allowed = 0;
  if (!allow_smem(reinterpret_cast<const void*>(kern), kWpSmem, &allowed))
    return set_error(DSA_ERR_CUDA, "window_mla: cannot raise dynamic shared memory to %d", kWpSmem);
  const int64_t jobs = a.n_full + (units - a.n_full) * a.n_split;
  if (jobs > 0x7ffffff0) return set_error(DSA_ERR_SHAPE, "window_mla: too many work units");
  const int pairs = (int)min(jobs, (int64_t)max(1, sm_count() / 2));
  kern<<<2 * pairs, kWpThreads, kWpSmem, stream>>>(tq, to, tl, tr, a, (int)jobs);
  if (a.n_split > 1) window_combine(a, units, stream);
  return check_launch("window_mla");
}

int window_mla_prefill_launch(const void* q, const void* kv, const int32_t* ks, const int32_t* ke, void* out, int T, int H, int S, int window, int first,
                              float scale, void* workspace, size_t workspace_bytes, int32_t* status, cudaStream_t stream) {
  WinArgs a{};
  a.q = static_cast<const __nv_bfloat16*>(q);
  a.kv = static_cast<const uint8_t*>(kv);
  a.ks = ks; a.ke = ke;
  a.out = static_cast<__nv_bfloat16*>(out);
  a.T = T; a.H = H; a.S = S;
  a.window = window; a.first = first;
  a.scale_log2e = scale * 1.4426950408889634f;
  a.status = status;
  a.unit_rows = prompt_unit_rows(H);
  a.seq_rows = T * H;
  a.seq_units = (int)prompt_units(T, H);
  return launch_prompt<false>(a, a.seq_units, window_keys(H, window, first, T, S), workspace, workspace_bytes, stream);
}

size_t window_prompt_drafts_workspace(int B, int64_t seq_rows, int H, int64_t keys) {
  return window_workspace(B * ((seq_rows + prompt_unit_rows(H) - 1) / prompt_unit_rows(H)), keys);
}
void window_prompt_units(WinArgs& a) {
  a.unit_rows = prompt_unit_rows(a.H);
  a.seq_units = (a.seq_rows + a.unit_rows - 1) / a.unit_rows;
  a.live = (int64_t)(a.T / a.drafts.per_seq) * a.seq_units >= sm_count() / 2;      // fewer are cut into parts
}
int window_prompt_drafts(const WinArgs& a, void* workspace, size_t workspace_bytes, cudaStream_t stream) {
  const int64_t units = (int64_t)(a.T / a.drafts.per_seq) * a.seq_units;
  return launch_prompt<true>(a, units, window_keys(a.H, a.window, a.first, a.drafts.per_seq, a.drafts.max_ctx), workspace, a.live ? 0 : workspace_bytes, stream);
}

}  // namespace dsa
