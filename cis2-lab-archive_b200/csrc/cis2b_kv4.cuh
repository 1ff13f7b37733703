// cis2b_kv4.cuh -- the 4-bit key/value cache: record format and the small
// device helpers that its kernels share.
//
// A page holds page_size tokens of every KV head.  Per head it is a run of
// records of 16 tokens; one record of head size D is contiguous:
//   16 x D/2 bytes  key codes    (byte b: element 2b low, 2b + 1 high)
//   16 x D/2 bytes  value codes
//   16 x 4 bfloat16 key step, key base, value step, value base
// so 16 tokens are one aligned stretch of 16 (D + 8) bytes: 2,176 for D = 128.
// Code c stands for base + step * c.  Two bfloat16 numbers per group of D
// elements cost 8 (D = 64) or 3 (D = 128) percent of a 16-bit cache's bytes;
// bfloat16 keeps float32's range, so no finite group overflows its parameters.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace cis2b {

constexpr int KV4_REC = 16;  // tokens per record

__host__ __device__ constexpr int kv4_rec_bytes(int hd) { return KV4_REC * (hd + 8); }

// Element types of the caller's tensors (CIS2B_F32, CIS2B_F16, CIS2B_BF16).
enum { KV4_F32 = 0, KV4_F16 = 1, KV4_BF16 = 2 };

__device__ __forceinline__ float bf16_lo(uint32_t x) { return __uint_as_float(x << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t x) { return __uint_as_float(x & 0xffff0000u); }

// The bfloat16 value at or below x (infinities and NaN: unchanged or NaN).
__device__ __forceinline__ uint32_t bf16_down(float x) {
  uint32_t b = __float_as_uint(x);
  uint32_t cut = b & 0xffff0000u;
  if ((b >> 31) && cut != b) cut += 0x10000u;  // a negative value grows in magnitude
  return cut >> 16;
}
// The bfloat16 value at or above x, x >= 0.
__device__ __forceinline__ uint32_t bf16_up(float x) { return (__float_as_uint(x) + 0xffffu) >> 16; }

// Eight consecutive 16-bit elements, zeros where `on` is not set.  `wide`: the
// address is 16-byte aligned (the host checks base and strides once).
__device__ __forceinline__ void load_words(const void *base, int64_t at, bool wide, bool on, uint32_t (&w)[4]) {
  const uint16_t *p = static_cast<const uint16_t *>(base) + at;
  w[0] = w[1] = w[2] = w[3] = 0;
  if (on && wide) {
    const uint4 a = __ldg(reinterpret_cast<const uint4 *>(p));
    w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w;
  } else if (on) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __ldg(p + 2 * i) | (uint32_t)__ldg(p + 2 * i + 1) << 16;
  }
}

// N consecutive elements as float32, zeros where `on` is not set: fp32,
// or 16-bit elements of a type known at run time.  All loads are issued before
// anything is done with them.
template <bool F32, int N>
__device__ __forceinline__ void load_query(const void *base, bool bf16, int64_t at, bool wide, bool on, float (&x)[N]) {
  constexpr int WORDS = F32 ? N : N / 2;
  uint32_t w[WORDS];
#pragma unroll
  for (int i = 0; i < WORDS; ++i) w[i] = 0;
  const uint8_t *p = static_cast<const uint8_t *>(base) + at * (F32 ? 4 : 2);
  if (on && wide) {
#pragma unroll
    for (int i = 0; i < WORDS; i += 4) {
      const uint4 a = __ldg(reinterpret_cast<const uint4 *>(p) + i / 4);
      w[i] = a.x, w[i + 1] = a.y, w[i + 2] = a.z, w[i + 3] = a.w;
    }
  } else if (on) {
#pragma unroll
    for (int i = 0; i < WORDS; ++i) {
      if constexpr (F32) w[i] = __ldg(reinterpret_cast<const uint32_t *>(p) + i);
      else w[i] = __ldg(reinterpret_cast<const uint16_t *>(p) + 2 * i) |
                  (uint32_t)__ldg(reinterpret_cast<const uint16_t *>(p) + 2 * i + 1) << 16;
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if constexpr (F32) {
      x[i] = __uint_as_float(w[i]);
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i / 2]));
      x[i] = (i & 1) ? (bf16 ? bf16_hi(w[i / 2]) : f.y) : (bf16 ? bf16_lo(w[i / 2]) : f.x);
    }
  }
}

__device__ __forceinline__ uint32_t pack_half(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&h);
}

// Eight consecutive elements rounded to nearest into the caller's type.
__device__ __forceinline__ void store8(void *base, int dt, int64_t at, bool wide, const float (&x)[8]) {
  if (dt == KV4_F32) {
    float *p = static_cast<float *>(base) + at;
    if (wide) {
      reinterpret_cast<float4 *>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
      reinterpret_cast<float4 *>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) p[i] = x[i];
    }
    return;
  }
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    w[i] = dt == KV4_F16 ? pack_half(x[2 * i], x[2 * i + 1]) : pack_bf16(x[2 * i], x[2 * i + 1]);
  uint16_t *p = static_cast<uint16_t *>(base) + at;
  if (wide) {
    *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) p[2 * i] = (uint16_t)w[i], p[2 * i + 1] = (uint16_t)(w[i] >> 16);
  }
}

// Four, where an aligned address is one of 8 or 16 bytes.
__device__ __forceinline__ void store4(void *base, int dt, int64_t at, bool wide, float4 x) {
  if (dt == KV4_F32) {
    float *p = static_cast<float *>(base) + at;
    if (wide) *reinterpret_cast<float4 *>(p) = x;
    else p[0] = x.x, p[1] = x.y, p[2] = x.z, p[3] = x.w;
    return;
  }
  const uint32_t a = dt == KV4_F16 ? pack_half(x.x, x.y) : pack_bf16(x.x, x.y);
  const uint32_t b = dt == KV4_F16 ? pack_half(x.z, x.w) : pack_bf16(x.z, x.w);
  uint16_t *p = static_cast<uint16_t *>(base) + at;
  if (wide) *reinterpret_cast<uint2 *>(p) = make_uint2(a, b);
  else p[0] = (uint16_t)a, p[1] = (uint16_t)(a >> 16), p[2] = (uint16_t)b, p[3] = (uint16_t)(b >> 16);
}

}  // namespace cis2b
