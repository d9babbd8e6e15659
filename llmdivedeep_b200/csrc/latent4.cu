// Write and read side of the paged 4-bit latent cache (layout: latent4.cuh).
#include <cuda_bf16.h>
#include <cuda_fp4.h>

#include "dsa_common.cuh"
#include "dsa_host.h"
#include "latent4.cuh"

namespace dsa {

// Eight neighbouring values, from 16-byte loads (fp32: two, bf16: one): their magnitudes, and their signs two by two at bits 15 and 31.
struct Eight {
  float v[8];
  uint32_t sign[4];
};
template <typename T>
__device__ __forceinline__ Eight load8(const T* __restrict__ src) {
  Eight x;
  if constexpr (sizeof(T) == 2) {
    const uint4 raw = __ldg(reinterpret_cast<const uint4*>(src));
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {                      // bf16 -> fp32: the value is the upper half of the word
      x.v[2 * i] = __uint_as_float((w[i] << 16) & 0x7fffffffu);
      x.v[2 * i + 1] = __uint_as_float(w[i] & 0x7fff0000u);
      x.sign[i] = w[i] & 0x80008000u;
    }
  } else {
    const uint4 lo = __ldg(reinterpret_cast<const uint4*>(src)), hi = __ldg(reinterpret_cast<const uint4*>(src) + 1);
    const uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) x.v[i] = __uint_as_float(w[i] & 0x7fffffffu);
#pragma unroll
    for (int i = 0; i < 4; ++i) x.sign[i] = ((w[2 * i] >> 16) & 0x8000u) | (w[2 * i + 1] & 0x80000000u);
  }
  return x;
}

// Scale byte of a group from its largest magnitude: a / 6 (IEEE) held to the scales' range, to four significant bits, ties to even.
__device__ __forceinline__ uint32_t latent4_scale_of(float amax) {
  const uint32_t b = __float_as_uint(fminf(fmaxf(__fdiv_rn(amax, 6.f), 0x1p-15f), 61440.f));
  const uint32_t r = (b + 0x7ffffu + ((b >> 20) & 1u)) >> 20;      // exponent and three bits of mantissa; a carry moves the exponent
  return r - (112u << 3);
}

// Eight values -> a word of codes.  The conversion rounds to nearest, ties to even, and saturates; for that it needs value / scale on the
// right side of the halves t between two levels (.25 .75 1.25 1.75 2.5 3.5 5), or on t where it is.  fp32 values are divided (IEEE).  A bf16
// value has eight significant bits, a scale four: their quotient is t or at least 2^-10 from it (all cases counted), so the value times
// the rounded reciprocal, 2^-20 off at most, is put on the nearest multiple of 2^-12 (by adding 3 * 2^10, where that is the last place, and
// taking it away): the same codes.
template <bool FEW_BITS>
__device__ __forceinline__ uint32_t latent4_word(const Eight& x, float scale) {
  const float inv = FEW_BITS ? __frcp_rn(scale) : 0.f;
  auto level = [&](float v) {
    if constexpr (FEW_BITS) return __fsub_rn(__fmaf_rn(v, inv, 0x1.8p11f), 0x1.8p11f);
    else return __fdiv_rn(v, scale);
  };
  constexpr int kSign[4] = {0, 3, 6, 1};
  uint32_t w = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint32_t b = __nv_cvt_float2_to_fp4x2(make_float2(level(x.v[2 * k]), level(x.v[2 * k + 1])), __NV_E2M1, cudaRoundNearest);
    const uint32_t n = b | (b << 12);                  // number of the even value at bit 0, of the odd one at bit 16
    w |= x.sign[k] >> kSign[k];
    if (k < 3) w |= (n & 0x00070007u) << (6 - 3 * k);
    else w |= ((n & 0x00060006u) << 9) | ((n & 0x00010001u) << 13);
  }
  return w;
}

// The tokens' indexer keys, already quantised, on their way into the paged key cache (k8 null: none).
struct KeyRows {
  const uint8_t* k8;                                   // [n, 128] e4m3
  const float* scale;                                  // [n]
  uint8_t* cache;                                      // [cache_rows, 128]
  float* cache_scale;                                  // [cache_rows]
};

// Latent rows -> records at the cache rows `slots` (null: row i -> record i).  A warp per token: 1152 bytes in (bf16), 416 out.  8192 tokens: 7.8 us
// from memory (5.0 out of L2), of which the bytes are 2: a launch, and one wave of warps that, as written, go to memory three times one after the other, for the slot, for
// the token's latents once the slot has been tested, and for its rope values and key behind the codes' stores.  (8.6 with a lane to every group of 16,
// whose loads and stores are pieces of lines, and an IEEE division for every value.)
template <typename T>
__global__ void __launch_bounds__(256) pack_latent4_kernel(const T* __restrict__ kv, int64_t row_stride, int64_t n, uint8_t* __restrict__ cache,
                                                           const int32_t* __restrict__ slots, int64_t cache_rows, const KeyRows keys, int* status) {
  const int lane = threadIdx.x & 31;
  const int64_t warps = (int64_t)gridDim.x * (blockDim.x >> 5);
  for (int64_t t = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); t < n; t += warps) {
    const int64_t slot = slots ? __ldg(slots + t) : t;
    if (slot < 0 || slot >= cache_rows) {              // negative: a token that is not to be written
      if (slot >= 0 && lane == 0 && status) atomicCAS(status, kStatusOk, kStatusBadIndex);
      continue;
    }
    const T* src = kv + t * row_stride;
    uint8_t* dst = cache + slot * kLatent4Bytes;
    // a lane has dims 8 lane .. of either half: two lanes a group, whole lines to every load and store
    Eight x[2];
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) x[hf] = load8(src + hf * 256 + lane * 8);
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      float amax = 0.f, odd = 0.f;                     // odd: 0 x value, NaN where a value is no number
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        amax = fmaxf(amax, x[hf].v[i]);
        odd = fmaf(x[hf].v[i], 0.f, odd);
      }
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      odd += __shfl_xor_sync(0xffffffffu, odd, 1);
      uint32_t byte = latent4_scale_of(amax);
      const float scale = __uint_as_float((byte + (112u << 3)) << 20);
      uint32_t word = latent4_word<sizeof(T) == 2>(x[hf], scale);
      if (odd != 0.f) {
        byte = kLatent4Nan;
        word = 0;
      }
      uint8_t* half = dst + hf * kLatent4Half;
      *reinterpret_cast<uint32_t*>(half + lane * 4) = word;
      if (!(lane & 1)) half[kLatent4Scales + (lane >> 1)] = (uint8_t)byte;
    }
    if (lane < 8) {                                    // eight rope values each
      uint4 rope;
      if constexpr (sizeof(T) == 2) {
        rope = __ldg(reinterpret_cast<const uint4*>(src + 512) + lane);
      } else {
        const float4 a = __ldg(reinterpret_cast<const float4*>(src + 512) + 2 * lane), b = __ldg(reinterpret_cast<const float4*>(src + 512) + 2 * lane + 1);
        const __nv_bfloat162 p[4] = {__floats2bfloat162_rn(a.x, a.y), __floats2bfloat162_rn(a.z, a.w), __floats2bfloat162_rn(b.x, b.y), __floats2bfloat162_rn(b.z, b.w)};
        rope = *reinterpret_cast<const uint4*>(p);
      }
      *reinterpret_cast<uint4*>(dst + (lane >> 2) * kLatent4Half + kLatent4Rope + (lane & 3) * 16) = rope;
    } else if (keys.k8 && lane < 17) {                 // lanes 8 to 15: 16 bytes of the key each, lane 16 its scale
      if (lane < 16) reinterpret_cast<uint4*>(keys.cache + slot * 128)[lane - 8] = __ldg(reinterpret_cast<const uint4*>(keys.k8 + t * 128) + lane - 8);
      else keys.cache_scale[slot] = __ldg(keys.scale + t);
    }
  }
}

// Records of positions 0 .. n-1 -> bf16 rows.  Position p is the record table[p / 64] * 64 + p % 64 (no table: record p); a page that does not
// exist gives a row of zeros.  A warp per token: 416 bytes in, 1152 out.  131072 tokens: 36.1 us = 5.7 TB/s, HBM (38.4 with a lane to every
// group of 16).  Two or four tokens of a warp requested together 37.6, 43.1; a page to a CTA 38.7; one wave of CTAs 37.8; a CTA to every eight
// tokens 36.9.
__global__ void __launch_bounds__(256) unpack_latent4_kernel(const uint8_t* __restrict__ cache, int64_t cache_rows, const int32_t* __restrict__ table, int64_t n,
                                                             __nv_bfloat16* __restrict__ out, int64_t out_stride, int* status) {
  const int lane = threadIdx.x & 31;
  const int64_t warps = (int64_t)gridDim.x * (blockDim.x >> 5);
  for (int64_t t = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); t < n; t += warps) {
    int64_t row = t;
    if (table) {
      const int64_t page = __ldg(table + t / 64);
      row = page < 0 ? -1 : page * 64 + t % 64;
    }
    const bool there = row >= 0 && row < cache_rows;
    if (!there && lane == 0 && status) atomicCAS(status, kStatusOk, kStatusBadIndex);
    const uint8_t* rec = cache + (there ? row : 0) * kLatent4Bytes;
    // a lane has dims 8 lane .. of either half: whole lines to every load and store
    uint32_t w[2] = {0, 0}, byte[2] = {0, 0};
    uint4 rope = make_uint4(0, 0, 0, 0);
    if (there) {
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        w[hf] = __ldg(reinterpret_cast<const uint32_t*>(rec + hf * kLatent4Half) + lane);
        byte[hf] = __ldg(rec + hf * kLatent4Half + kLatent4Scales + (lane >> 1));
      }
      if (lane < 8) rope = __ldg(reinterpret_cast<const uint4*>(rec + (lane >> 2) * kLatent4Half + kLatent4Rope + (lane & 3) * 16));
    }
    __nv_bfloat16* dst = out + t * out_stride;
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      const uint32_t sc = latent4_scale(byte[hf]);
      uint32_t c[4];
      latent4_codes(w[hf], c);
#pragma unroll
      for (int i = 0; i < 4; ++i) c[i] = mul_bf16x2(mul_bf16x2(c[i], sc), kLatent4GainPair);
      reinterpret_cast<uint4*>(dst + hf * 256)[lane] = make_uint4(c[0], c[1], c[2], c[3]);
    }
    if (lane < 8) reinterpret_cast<uint4*>(dst + 512)[lane] = rope;
  }
}

static int latent4_grid(int64_t n) {
  const int64_t want = (n + 7) / 8, most = (int64_t)sm_count() * 16;
  return (int)(want < most ? want : most);
}

int pack_latent4_launch(const void* kv, int kv_is_bf16, int64_t row_stride, int64_t n, void* cache, const int32_t* slots, int64_t cache_rows, const void* k8,
                        const float* k_scale, void* kcache, float* kscale, int32_t* status, cudaStream_t stream) {
  const KeyRows keys{static_cast<const uint8_t*>(k8), k_scale, static_cast<uint8_t*>(kcache), kscale};
  uint8_t* rec = static_cast<uint8_t*>(cache);
  if (kv_is_bf16)
    pack_latent4_kernel<<<latent4_grid(n), 256, 0, stream>>>(static_cast<const __nv_bfloat16*>(kv), row_stride, n, rec, slots, cache_rows, keys, status);
  else
    pack_latent4_kernel<<<latent4_grid(n), 256, 0, stream>>>(static_cast<const float*>(kv), row_stride, n, rec, slots, cache_rows, keys, status);
  return check_launch("pack_latent4");
}

int unpack_latent4_launch(const void* cache, int64_t cache_rows, const int32_t* table, int64_t n, void* out, int64_t out_stride, int32_t* status,
                          cudaStream_t stream) {
  unpack_latent4_kernel<<<latent4_grid(n), 256, 0, stream>>>(static_cast<const uint8_t*>(cache), cache_rows, table, n, static_cast<__nv_bfloat16*>(out), out_stride,
                                                             status);
  return check_launch("unpack_latent4");
}

}  // namespace dsa
