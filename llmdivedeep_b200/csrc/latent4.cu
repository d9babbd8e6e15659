// Write and read side of the paged 4-bit latent cache (layout: latent4.cuh).
#include <cuda_bf16.h>
#include <cuda_fp4.h>

#include "dsa_common.cuh"
#include "dsa_host.h"
#include "latent4.cuh"

namespace dsa {

// A row's 16 values from 16-byte loads (fp32: four, bf16: two).
template <typename T>
__device__ __forceinline__ void load16(const T* __restrict__ src, float (&v)[16]) {
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint4 raw = __ldg(reinterpret_cast<const uint4*>(src) + h);
      const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {                    // bf16 -> fp32: the value is the upper half of the word
        v[8 * h + 2 * i] = __uint_as_float(w[i] << 16);
        v[8 * h + 2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      }
    }
  } else {
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      const float4 raw = __ldg(reinterpret_cast<const float4*>(src) + h);
      v[4 * h] = raw.x; v[4 * h + 1] = raw.y; v[4 * h + 2] = raw.z; v[4 * h + 3] = raw.w;
    }
  }
}

// Scale byte of a group from its largest magnitude: a / 6 (IEEE) held to the scales' range, to four significant bits, ties to even.
__device__ __forceinline__ uint32_t latent4_scale_of(float amax) {
  const uint32_t b = __float_as_uint(fminf(fmaxf(__fdiv_rn(amax, 6.f), 0x1p-15f), 61440.f));
  const uint32_t r = (b + 0x7ffffu + ((b >> 20) & 1u)) >> 20;      // exponent and three bits of mantissa; a carry moves the exponent
  return r - (112u << 3);
}

// Eight values -> a word of codes.  The conversion rounds to nearest, ties to even, and saturates.
__device__ __forceinline__ uint32_t latent4_word(const float* v, float scale) {
  uint32_t w = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint32_t b = __nv_cvt_float2_to_fp4x2(make_float2(__fdiv_rn(v[2 * k], scale), __fdiv_rn(v[2 * k + 1], scale)), __NV_E2M1, cudaRoundNearest);
    const uint32_t n = (b & 15u) | ((b & 0xf0u) << 12);            // sign and number of the even value, of the odd one
    if (k < 3) w |= ((n & 0x00080008u) << (12 - 3 * k)) | ((n & 0x00070007u) << (6 - 3 * k));
    else w |= ((n & 0x00080008u) << 11) | ((n & 0x00060006u) << 9) | ((n & 0x00010001u) << 13);
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

// Latent rows -> records at the cache rows `slots` (null: row i -> record i).  A warp per token: a lane has one group.
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
    float v[16];
    load16(src + lane * 16, v);
    float amax = 0.f, odd = 0.f;                       // odd: 0 x value, NaN where a value is no number
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      amax = fmaxf(amax, fabsf(v[i]));
      odd = fmaf(v[i], 0.f, odd);
    }
    uint32_t byte = latent4_scale_of(amax);
    if (odd != 0.f) {
      byte = kLatent4Nan;
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = 0.f;
    }
    const float scale = __uint_as_float((byte + (112u << 3)) << 20);
    uint8_t* half = dst + (lane >> 4) * kLatent4Half;
    *reinterpret_cast<uint2*>(half + (lane & 15) * 8) = make_uint2(latent4_word(v, scale), latent4_word(v + 8, scale));
    half[kLatent4Scales + (lane & 15)] = (uint8_t)byte;
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
// exist gives a row of zeros.  A warp per token.
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
    const uint8_t* half = cache + (there ? row : 0) * kLatent4Bytes + (lane >> 4) * kLatent4Half;
    uint2 w = make_uint2(0, 0);
    uint32_t byte = 0;
    uint4 rope = make_uint4(0, 0, 0, 0);
    if (there) {
      w = __ldg(reinterpret_cast<const uint2*>(half + (lane & 15) * 8));
      byte = __ldg(half + kLatent4Scales + (lane & 15));
      if (lane < 8)
        rope = __ldg(reinterpret_cast<const uint4*>(cache + row * kLatent4Bytes + (lane >> 2) * kLatent4Half + kLatent4Rope + (lane & 3) * 16));
    }
    const uint32_t sc = latent4_scale(byte);
    uint32_t a[4], b[4];
    latent4_codes(w.x, a);
    latent4_codes(w.y, b);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      a[i] = mul_bf16x2(mul_bf16x2(a[i], sc), kLatent4GainPair);
      b[i] = mul_bf16x2(mul_bf16x2(b[i], sc), kLatent4GainPair);
    }
    __nv_bfloat16* dst = out + t * out_stride;
    reinterpret_cast<uint4*>(dst + lane * 16)[0] = make_uint4(a[0], a[1], a[2], a[3]);
    reinterpret_cast<uint4*>(dst + lane * 16)[1] = make_uint4(b[0], b[1], b[2], b[3]);
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
