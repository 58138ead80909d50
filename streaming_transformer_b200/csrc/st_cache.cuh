// st_cache.cuh -- device helpers of the window-cache operators: rows of 8
// values a lane, 4-bit rows, and the slot a position lives in.
//
// Every kernel that walks rows gives a lane 8 consecutive columns: one 16-byte
// access of a 16-bit row, two of an fp32 row, 4 bytes of codes of a 4-bit row,
// whose groups of 32 columns are then 4 neighbouring lanes. A row of head_dim
// columns takes lanes_per_row(head_dim) lanes (a power of two, so that shuffles
// stay inside the row); lanes past head_dim hold zeros.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "../../include/streaming_b200.h"

namespace st {

__host__ __device__ constexpr int lanes_per_row(int head_dim) {
  int n = 1;
  while (n * 8 < head_dim) n *= 2;
  return n;
}

// ---- 8 columns as floats
__device__ __forceinline__ void load8(const float* p, float (&f)[8]) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
  f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
}
__device__ __forceinline__ void load8(const __half* p, float (&f)[8]) {
  const uint4 u = *reinterpret_cast<const uint4*>(p);
  const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    f[2 * i] = t.x;
    f[2 * i + 1] = t.y;
  }
}
__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&f)[8]) {
  const uint4 u = *reinterpret_cast<const uint4*>(p);
  const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(w[i] << 16);
    f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ void store8(float* p, const float (&f)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
}
__device__ __forceinline__ unsigned pack2(__half*, float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const unsigned*>(&h);
}
__device__ __forceinline__ unsigned pack2(__nv_bfloat16*, float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const unsigned*>(&h);
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&f)[8]) {
  *reinterpret_cast<uint4*>(p) = make_uint4(pack2(p, f[0], f[1]), pack2(p, f[2], f[3]), pack2(p, f[4], f[5]),
                                            pack2(p, f[6], f[7]));
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
// The least of three, NaN if one is.
__device__ __forceinline__ float min3_nan(float a, float b, float c) {
  float y;
  asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}

// ---- 4-bit rows: {scale, lowest} of a group as one word, scale in the low half
__device__ __forceinline__ float group_scale(unsigned pair) { return __uint_as_float(pair << 16); }
__device__ __forceinline__ float group_lowest(unsigned pair) { return __uint_as_float(pair & 0xffff0000u); }

__device__ __forceinline__ void decode8(unsigned codes, unsigned pair, float (&f)[8]) {
  const float s = group_scale(pair), low = group_lowest(pair);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = fmaf((float)((codes >> (4 * i)) & 15u), s, low);
}

// Quantises the 32 values that 4 neighbouring lanes hold: this lane's codes,
// and the group's {scale, lowest}. All 4 lanes of the group call it together;
// `mask` names the lanes of the warp that do.
__device__ __forceinline__ unsigned encode8(const float (&f)[8], unsigned mask, unsigned* pair) {
  float low = min3_nan(f[0], f[1], f[2]), high = max3(f[0], f[1], f[2]);  // a NaN in `low` makes the range one
#pragma unroll
  for (int i = 3; i < 8; i += 2) {
    low = min3_nan(low, f[i], f[i < 7 ? i + 1 : i]);
    high = max3(high, f[i], f[i < 7 ? i + 1 : i]);
  }
#pragma unroll
  for (int o = 1; o < 4; o *= 2) {
    const float other = __shfl_xor_sync(mask, low, o);
    low = min3_nan(low, other, other);
    high = fmaxf(high, __shfl_xor_sync(mask, high, o));
  }
  const float range = __fsub_rn(high, low);
  const __nv_bfloat16 s16 = __float2bfloat16_rn(__fmul_rn(range, 1.0f / 15.0f));
  const __nv_bfloat16 l16 = __float2bfloat16_rn(low);  // below -3.39e38 it rounds to -inf
  if (!(range < INFINITY) || isinf(__bfloat162float(l16))) {
    *pair = 0x7fff7fffu;  // two bf16 NaNs
    return 0;
  }
  const float s = __bfloat162float(s16), l = __bfloat162float(l16);
  unsigned codes = 0;
  if (s > 0.f) {
    // The code is the quotient d / s, correctly rounded, to the nearest integer (ties to even: 1.5 * 2^23 + c has c in
    // its low bits). Half a step is hit often, by rows of 16 bits, so the quotient has to be exact. d times the rounded
    // reciprocal is off by 2^-23 of it at most; what it leaves of d is a multiple of the product of both last places, up
    // to 2^10 of them, so it is exact in fp32, and adding it times the reciprocal leaves an error of 2^-46 before the
    // last rounding (P. Markstein's correction). s has 8 bits, which keeps d / s 2^-33 of itself away from every point
    // where the rounding changes. Below 2^-110 the remainder
    // may leave the fp32 range, above 2^120 the difference. (With a division for the lanes that have a quotient next to
    // a half, as most warps over 16-bit values do: 94.5 us for 16384 rows of 32 and 8 heads of 128, so 92.5.)
    const float inverse = __frcp_rn(s);
    if (s >= 0x1p-110f && s < 0x1p120f) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float d = __fsub_rn(f[i], l), q = __fmul_rn(d, inverse), c = fmaf(fmaf(-s, q, d), inverse, q);
        codes += __float_as_uint(__fadd_rn(fminf(fmaxf(c, 0.f), 15.f), 12582912.f)) << (4 * i);
      }
      codes -= 0x4b400000u * 0x11111111u;  // what 1.5 * 2^23 has of its own
    } else {
      for (int i = 0; i < 8; ++i) {
        const float c = fminf(fmaxf(__fdiv_rn(__fsub_rn(f[i], l), s), 0.f), 15.f);
        codes |= (__float_as_uint(__fadd_rn(c, 12582912.f)) & 15u) << (4 * i);
      }
    }
  }
  *pair = (unsigned)__bfloat16_as_ushort(s16) | ((unsigned)__bfloat16_as_ushort(l16) << 16);
  return codes;
}

// Slots a stream at `position` sees (0 when idle).
__device__ __forceinline__ int slots_seen(long long position, int slots) {
  return position < 0 ? 0 : position >= slots - 1 ? slots : (int)position + 1;
}

__device__ __forceinline__ int clamp_row(int v, int rows) { return v < 0 ? 0 : v > rows ? rows : v; }

}  // namespace st
