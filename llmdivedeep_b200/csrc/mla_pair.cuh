// What the kernels that attend over the 576-dim latent with a pair of CTAs have in common (sparse_mla.cu, window_mla.cu): the layout of
// shared and tensor memory, the exchange of partial scores, raw records and their conversion.
#pragma once
#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "dsa_common.cuh"
#include "latent4.cuh"

namespace dsa {

constexpr int kMlaDqk = 576;
constexpr int kMlaDv = 512;
constexpr int kMlaDvHalf = 256;
constexpr int kMlaBlk = 64;                        // keys per block
constexpr int kMlaPanels = 5;                      // panels per CTA: four latent (its V half) + rope
constexpr int kMlaBufs = 5;                        // KV buffers in shared memory
constexpr int kMlaQPanelBytes = 128 * 128;         // 128 heads x 128 B
constexpr int kMlaKPanelBytes = kMlaBlk * 128;     // 64 keys x 128 B
constexpr int kMlaRopeOff = 4 * kMlaKPanelBytes;   // in a buffer: four latent panels, then this CTA's 64 rope bytes of every row
constexpr int kMlaKBytes = kMlaRopeOff + kMlaBlk * 64;        // 36864 per buffer
constexpr int kMlaXBytes = 128 * kMlaBlk * 2;      // one partial score tile, fp16: 16384
constexpr int kMlaXWarp = kMlaXBytes / 8;          // ... a warp's part of it
constexpr int kMlaValidRing = 8;                   // validity bytes (64 per block) for the softmax: >= blocks in flight
// Where the rows come from: bf16 rows (prefill), records of the paged FP8 latent cache, records of the paged 4-bit one (latent4.cuh).
enum MlaSrc : int { kSrcRows = 0, kSrcFp8 = 1, kSrc4 = 2 };
// The registers of the launch (896 threads x 72) are dealt out again: setmaxnreg moves what the issuing and gathering
// warps do not need to the softmax.
template <bool PAGED>
struct MlaRegs {                                   // decode's gather converts in registers
  static constexpr int kSoftmax = PAGED ? 88 : 96, kOther = PAGED ? 48 : 40;
  static_assert(512 * kSoftmax + 384 * kOther <= 896 * 72, "more registers than the launch has");
};
constexpr int kMlaThreads = 896, kMlaSoftmaxWarps = 16, kMlaMmaWarp = 16, kMlaGatherWarp0 = 17, kMlaGatherWarps = 11;
template <int R>
__device__ __forceinline__ void regs_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(R)); }
template <int R>
__device__ __forceinline__ void regs_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(R)); }
// Waits here loop unrolled by four: with the compact loop decode is 7 % slower (batch 64 68.6 us against 64.2, both with the first
// look in front) and prefill the same.
__device__ __forceinline__ bool mla_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* status) {
  return mbar_wait_warp<4>(bar, parity, abort_flag, status);
}
constexpr int kMlaBarBytes = 512;                  // mbarriers and a few words
constexpr int kMlaPairBytes = 4 * 2 * 128 * 2;     // block maxima: [block mod 4][key half][head], bf16
constexpr int kMlaSmemBytes = kMlaBufs * kMlaKBytes + 2 * kMlaXBytes + kMlaBarBytes +
                              kMlaValidRing * kMlaBlk + kMlaPairBytes;
static_assert(kMlaSmemBytes <= 232448, "shared memory budget of one CTA");
constexpr int kLatentTokenBytes = 656;             // 512 e4m3 + 4 fp32 scales + 64 bf16 rope
constexpr int kLatentPage = 64;
// tensor-memory columns: O 256, S 64, P 32, Q 5 x 32
constexpr uint32_t kColO = 0, kColS = 256, kColP = kColS + kMlaBlk, kColQ = kColP + kMlaBlk / 2, kMlaTmemCols = 512;
static_assert(kColQ + kMlaPanels * 32 <= kMlaTmemCols, "tensor memory budget");

// ---- cluster helpers ----------------------------------------------------------------------------
__device__ __forceinline__ uint32_t mapa_u32(uint32_t addr, uint32_t cta) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(cta));
  return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// Arrive on the peer's barrier to say "this warp has READ the tile".  Relaxed: a release at cluster scope costs a memory
// fence of thousands of cycles per block, and nothing written by this thread has to become visible.  But a relaxed arrival
// orders nothing, and straight after the loads it overtakes them -- they queue behind the gather's copies in the load/store
// unit, and the next tile then lands on top of this one before it is read (seen: a few tokens in ten thousand).  So the
// arrival takes the data as its operand: each lane gives a value computed from EVERY word that it loaded, the vote needs all
// lanes' values, and the arrival is predicated on the vote, so that it cannot issue before the loads have returned, whatever
// the compiler does with the code around it.  `x` comes out of fmaxf, which returns numbers or the canonical NaN: it never is
// the bit pattern compared with (a signalling NaN), which the compiler cannot know.  (A register-OR of the loaded words
// as that value, to send the arrival earlier, cost more than it gained: 2228 -> 2280 us.)
__device__ __forceinline__ void mbar_arrive_remote_after(uint32_t cluster_addr, float x, bool leader) {
  const bool seen = __any_sync(0xffffffffu, __float_as_uint(x) != 0x7f812345u);
  if (leader)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.u32 p, %1, 0;\n\t"
        "@p mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];\n\t}"
        ::"r"(cluster_addr), "r"(static_cast<uint32_t>(seen)) : "memory");
}
// this CTA's shared memory -> the peer's, completion counted on the peer's mbarrier
__device__ __forceinline__ void bulk_copy_to_peer(uint32_t dst_cluster, const void* src, uint32_t bytes, uint32_t bar_cluster) {
  asm volatile("cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(dst_cluster), "r"(smem_u32(src)), "r"(bytes), "r"(bar_cluster) : "memory");
}

// one [rows x 128 B] panel, shared memory (128-B swizzle) -> global, tracked by the thread's bulk group
__device__ __forceinline__ void tma_store_2d(const void* tmap, const void* src, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];"
               ::"l"(reinterpret_cast<uint64_t>(tmap)), "r"(x), "r"(y), "r"(smem_u32(src)) : "memory");
}
__device__ __forceinline__ void bulk_commit_and_wait_read() {      // shared memory may be reused / released afterwards
  asm volatile("cp.async.bulk.commit_group;\n\tcp.async.bulk.wait_group.read 0;" ::: "memory");
}

__device__ __forceinline__ uint32_t pack_bf16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float fast_exp2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {      // out-of-range values saturate to +-65504
  uint32_t r;
  asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// a pair of fp16 values plus a pair of fp32 values, one mixed-precision add each
__device__ __forceinline__ void add_f16x2(uint32_t h, float x, float y, float& sx, float& sy) {
  asm("{\n\t.reg .b16 l, u;\n\tmov.b32 {l, u}, %2;\n\tadd.rn.f32.f16 %0, l, %3;\n\tadd.rn.f32.f16 %1, u, %4;\n\t}"
      : "=f"(sx), "=f"(sy) : "r"(h), "f"(x), "f"(y));
}
// A warp's part of a partial score tile is [32 heads][32 keys] fp16, 64 bytes per thread.  The 16-byte chunks c (0..3) of a
// row are rotated by the lane pair, so that the eight lanes of a quarter-warp hit different banks.
__device__ __forceinline__ int xchg_off(int lane, int c) { return lane * 64 + (((c ^ (lane >> 1)) & 3) << 4); }
// fp32 -> bf16 bits, rounded towards +infinity
__device__ __forceinline__ uint32_t bf16_bits_round_up(float x) {
  const uint32_t b = __float_as_uint(x);
  return ((b >> 31) || (b & 0x7fffffffu) >= 0x7f800000u) ? (b >> 16) : ((b + 0xffffu) >> 16);
}

// ---- paged FP8 latent cache (decode) ------------------------------------------------------------
__device__ __forceinline__ void cp_async_16(void* dst, const void* src, int src_bytes) {      // src_bytes 0: zero fill
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(src_bytes) : "memory");
}
__device__ __forceinline__ void cp_async_16_all(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
// counts as this thread's arrival on the barrier when all cp.async it has issued so far have landed
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }
// A gather warp's raw rows of one block: per row this CTA's 256 e4m3 values, the four scales, this CTA's 64 rope bytes; of a 4-bit
// record this CTA's half as it is.
constexpr int kRawRows = (kMlaBlk + kMlaGatherWarps - 1) / kMlaGatherWarps;
template <int SRC>
struct MlaRaw {
  static constexpr int kRow = SRC == kSrc4 ? kLatent4Half : 256 + 16 + 64, kBytes = kRawRows * kRow, kPieces = 2 * kMlaGatherWarps;
  static constexpr int kInBuf = kMlaKBytes / kBytes < kPieces ? kMlaKBytes / kBytes : kPieces;      // pieces in the fifth KV buffer
  static constexpr int kSmem = kMlaSmemBytes + (SRC == kSrcRows ? 0 : (kPieces - kInBuf) * kBytes);
  static_assert(kRawRows % 2 == 0 && kMlaSmemBytes % 16 == 0 && kSmem <= 232448, "raw rows of decode");
};
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Eight e4m3 values times their group scale, rounded to bf16; an empty slot's zeros (values and scale) stay zeros.  bf16 because queries and rope values are: one MMA has
// one type.  (Without the rounding every group of 128 values needs score columns and P of its own, to which the scales are applied, and tensor memory is full.)
// An output is 3.2 to 3.5e-3 off in place of the 2.0 to 2.2e-3 that it is over bf16 rows.
__device__ __forceinline__ uint4 e4m3x8_to_bf16(uint2 raw, float sc) {
  const uint32_t w[2] = {raw.x, raw.y};
  const uint64_t sc2 = pack_f32x2(sc, sc);
  uint32_t o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_fp8x2_storage_t pr = static_cast<__nv_fp8x2_storage_t>((w[i >> 1] >> (16 * (i & 1))) & 0xffffu);
    const __half2_raw h2 = __nv_cvt_fp8x2_to_halfraw2(pr, __NV_E4M3);
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h2));
    float x, y;
    unpack_f32x2(mul_f32x2(pack_f32x2(f.x, f.y), sc2), x, y);
    o[i] = pack_bf16x2(x, y);
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}

}  // namespace dsa
