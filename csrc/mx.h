// Microscaled floating point (blocks of 32 values that share a power of two): what the quantising and the multiplying kernels have
// in common.
//
// A block's scale is 2^e with the smallest e for which every |v| <= L 2^e, L the largest element (448 in e4m3, 6 in e2m1), so no
// element saturates; stored as the byte e + 127.  Elements are v 2^-e rounded to nearest, ties to even: a product with a power of
// two is exact, so this is the only rounding.  A block with a NaN or an infinity gets the scale byte 255 (NaN) and elements of zero:
// the matrix instruction makes NaN of every product with such a block.
#pragma once
#include "common.h"

typedef uint32_t mx_u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t mx_u32x4 __attribute__((ext_vector_type(4)));
typedef int mx_i32x4 __attribute__((ext_vector_type(4)));
typedef int mx_i32x8 __attribute__((ext_vector_type(8)));

// the scale byte of a block whose largest |v| is `amax` (448 = 1.75 * 2^8, 6 = 1.5 * 2^2).  `amax` as its bits: of non-negative
// floats the order of the bits is the order of the values, infinity and NaN above all
template <int BITS> __device__ __forceinline__ uint32_t mx_scale_byte(uint32_t amax) {
  const int e = (int)(amax >> 23) - (BITS == 8 ? 8 : 2) + ((amax & 0x7fffffu) > (BITS == 8 ? 0x600000u : 0x400000u) ? 1 : 0);
  return amax >= 0x7f800000u ? 255u : (uint32_t)max(e, 0);
}
// 2^-e for a scale byte (0 for 255: elements of a block without a finite scale are zeros; -0 * 0 and 0 * inf are masked below)
__device__ __forceinline__ float mx_inverse(uint32_t byte) {
  return byte == 255u ? 0.f : __uint_as_float((254u - byte) << 23);
}

__device__ __forceinline__ uint32_t mx_abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// the largest bits over a quad of lanes (each holds 8 values of one block of 32)
__device__ __forceinline__ uint32_t mx_quad_max(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, true));     // quad_perm [1, 0, 3, 2]
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xf, 0xf, true));     // quad_perm [2, 3, 0, 1]
  return v;
}

// four values times `inv` as four e4m3 bytes (|v inv| <= 448).  inv = 0: zeros, whatever v is
__device__ __forceinline__ uint32_t mx_pack_fp8(float a, float b, float c, float d, float inv) {
  int r = 0;
  r = __builtin_amdgcn_cvt_pk_fp8_f32(a * inv, b * inv, r, false);
  r = __builtin_amdgcn_cvt_pk_fp8_f32(c * inv, d * inv, r, true);
  return inv == 0.f ? 0u : (uint32_t)r;
}

// eight values times `inv` as eight e2m1 codes, the first in the lowest four bits (|v inv| <= 6)
__device__ __forceinline__ uint32_t mx_pack_fp4(const float (&v)[8], float inv) {
  uint32_t r = 0;
#if defined(__HIP_DEVICE_COMPILE__)
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[0] * inv, v[1] * inv, 1.f, 0);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[2] * inv, v[3] * inv, 1.f, 1);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[4] * inv, v[5] * inv, 1.f, 2);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[6] * inv, v[7] * inv, 1.f, 3);
#endif
  return inv == 0.f ? 0u : r;
}

// eight values of a row (16-bit or 32-bit) as floats
template <typename T> __device__ __forceinline__ void mx_load8(const T* p, float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
    const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
    for (int j = 0; j < 4; ++j) { v[j] = a[j]; v[4 + j] = b[j]; }
  } else {
    const auto a = ld8<T>(p);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = (float)a[j];
  }
}

// A quad's 32 values -> elements and scale.  All four lanes call it; q: this lane's eight bytes, s: the block's scale byte
__device__ __forceinline__ void mx_store8(uint8_t* q, uint8_t* s, const float (&v)[8]) {
  uint32_t a = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) a = max(a, mx_abs_bits(v[j]));
  const uint32_t byte = mx_scale_byte<8>(mx_quad_max(a));
  const float inv = mx_inverse(byte);
  *reinterpret_cast<mx_u32x2*>(q) = mx_u32x2{mx_pack_fp8(v[0], v[1], v[2], v[3], inv), mx_pack_fp8(v[4], v[5], v[6], v[7], inv)};
  if ((threadIdx.x & 3) == 0) *s = (uint8_t)byte;
}
