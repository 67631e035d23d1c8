// Rows to microscaled 8- or 4-bit floating point and back, and the RMS norm that leaves its rows in 8 bits (mx.h has the format).
// All bound by memory.  A thread holds 8 values of a row, four neighbours a block of 32: the block's largest value is found in two
// steps across the quad, without LDS.  Payload rows are padded with zeros to a multiple of 128 columns, the depth of the matrix
// instruction, so that the products read whole tiles.
#include "mx.h"

namespace {

// A thread's groups of 8 columns: row and place in it, a grid apart.  One division in front of the loop (one for each group: 28672 x 4096
// to 4 bits and back 132 us instead of 130)
struct MxWalk {
  long row, rows_on;
  int c, c_on, per_row;
  __device__ __forceinline__ MxWalk(long i, long stride, int per) : row(i / per), rows_on(stride / per), c((int)(i - row * per)),
                                                                    c_on((int)(stride - rows_on * per)), per_row(per) {}
  __device__ __forceinline__ void next() {
    row += rows_on;
    c += c_on;
    if (c >= per_row) { c -= per_row; ++row; }
  }
};

// rows of x [M][K] (src: x[src[row]]) -> q [M][width of BITS], s [M][.]; columns K .. Kp are zeros
template <typename T, int BITS>
__global__ __launch_bounds__(256) void mx_quantize_kernel(uint8_t* __restrict__ q, long ldq, uint8_t* __restrict__ s, long lds,
                                                          const T* __restrict__ x, long ldx, long groups, int per_row, int K,
                                                          const int* __restrict__ src, int x_rows) {
  const long stride = gridDim.x * 256L;
  long i = blockIdx.x * 256L + threadIdx.x;
  for (MxWalk w(i, stride, per_row); i < groups; i += stride, w.next()) {
    const long row = w.row;
    const int c = w.c;
    float v[8];
    if (8 * c < K) {                              // (whole blocks: a quad agrees)
      mx_load8(x + (src != nullptr ? (long)min(max(src[row], 0), x_rows - 1) : row) * ldx + 8 * c, v);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = 0.f;
    }
    if constexpr (BITS == 8) {
      mx_store8(q + row * ldq + 8 * c, s + row * lds + (c >> 2), v);
    } else {
      uint32_t a = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) a = max(a, mx_abs_bits(v[j]));
      const uint32_t byte = mx_scale_byte<4>(mx_quad_max(a));
      *reinterpret_cast<uint32_t*>(q + row * ldq + 4 * c) = mx_pack_fp4(v, mx_inverse(byte));
      if ((c & 3) == 0) s[row * lds + (c >> 2)] = (uint8_t)byte;
    }
  }
}

// An e4m3 byte, an e2m1 code as floats.  Integer arithmetic: exponent and mantissa move to their places in a float, whose exponent
// is then wrong by the difference of the biases - one product with a power of two, exact for subnormal elements too
__device__ __forceinline__ float mx_value8(uint32_t b) {
  const float m = __uint_as_float((b & 0x7fu) << 20) * 0x1p120f;
  return __uint_as_float(__float_as_uint((b & 0x7fu) == 0x7fu ? __uint_as_float(0x7fc00000u) : m) | (b & 0x80u) << 24);
}
__device__ __forceinline__ float mx_value4(uint32_t c) {
  return __uint_as_float(__float_as_uint(__uint_as_float((c & 7u) << 22) * 0x1p126f) | (c & 8u) << 28);
}
// v 2^e for a scale byte: 2^-127 is a subnormal float, so e is applied in two halves
__device__ __forceinline__ float mx_scaled(float v, uint32_t byte) {
  const int e = (int)byte - 127, h = e / 2;
  const float r = v * __uint_as_float((uint32_t)(127 + h) << 23) * __uint_as_float((uint32_t)(127 + e - h) << 23);
  return byte == 255u ? __uint_as_float(0x7fc00000u) : r;
}

template <typename T, int BITS>
__global__ __launch_bounds__(256) void mx_dequantize_kernel(T* __restrict__ out, const uint8_t* __restrict__ q, long ldq,
                                                            const uint8_t* __restrict__ s, long lds, long groups, int per_row) {
  const long stride = gridDim.x * 256L;
  long i = blockIdx.x * 256L + threadIdx.x;
  for (MxWalk at(i, stride, per_row); i < groups; i += stride, at.next()) {
    const long row = at.row;
    const int c = at.c;
    const uint32_t byte = s[row * lds + (c >> 2)];
    float v[8];
    if constexpr (BITS == 8) {
      const mx_u32x2 w = *reinterpret_cast<const mx_u32x2*>(q + row * ldq + 8 * c);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = mx_value8(w[j >> 2] >> (8 * (j & 3)) & 0xffu);
    } else {
      const uint32_t w = *reinterpret_cast<const uint32_t*>(q + row * ldq + 4 * c);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = mx_value4(w >> (4 * j) & 15u);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = mx_scaled(v[j], byte);
    T* const o = out + 8 * i;
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<f32x4*>(o) = f32x4{v[0], v[1], v[2], v[3]};
      *reinterpret_cast<f32x4*>(o + 4) = f32x4{v[4], v[5], v[6], v[7]};
    } else {
      typename Vec8<T>::type r;
#pragma unroll
      for (int j = 0; j < 8; ++j) r[j] = (T)v[j];
      st8<T>(o, r);
    }
  }
}

constexpr int MX_NORM_ITERS = 4;

// v = x (or the sum of ks fp32 slabs of it) + residual, in 32 bits; residual_out = v rounded; rows of v rsqrt(mean v^2 + eps) w.
// The norm is taken of the unrounded sum: its 8 bits follow the numbers, not a 16-bit copy of them.
template <typename T>
__global__ void mx_rms_norm_kernel(uint8_t* __restrict__ q, long ldq, uint8_t* __restrict__ s, long lds, T* __restrict__ residual_out,
                                   const T* __restrict__ x, long ldx, const float* __restrict__ slabs, int ks, long slab_stride,
                                   const T* __restrict__ residual, const T* __restrict__ w, float eps, int H, int Kp) {
  __shared__ float red[17];
  using V = typename Vec8<T>::type;
  const long row = blockIdx.x;
  const int nvec = H >> 3;
  float v[MX_NORM_ITERS][8];
  V gw[MX_NORM_ITERS];
  float ss = 0.f;
#pragma unroll
  for (int it = 0; it < MX_NORM_ITERS; ++it) {
    const int i = threadIdx.x + it * blockDim.x;
    if (i < nvec) {
      gw[it] = ld8<T>(w + 8 * i);
      V r;
      if (residual != nullptr) r = ld8<T>(residual + row * H + 8 * i);
      if (slabs != nullptr) {
        f32x4 a = f32x4{0.f, 0.f, 0.f, 0.f}, b = a;
        const float* p = slabs + row * H + 8 * i;
        for (int k = 0; k < ks; ++k) {
          a += *reinterpret_cast<const f32x4*>(p + k * slab_stride);
          b += *reinterpret_cast<const f32x4*>(p + k * slab_stride + 4);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) { v[it][j] = a[j]; v[it][4 + j] = b[j]; }
      } else {
        mx_load8(x + row * ldx + 8 * i, v[it]);
      }
      if (residual != nullptr) {
        V o;
#pragma unroll
        for (int j = 0; j < 8; ++j) { v[it][j] += (float)r[j]; o[j] = (T)v[it][j]; }
        st8<T>(residual_out + row * H + 8 * i, o);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) ss += v[it][j] * v[it][j];
    }
  }
  ss = block_sum(ss, red);
  const float inv = 1.f / sqrtf(ss / (float)H + eps);
#pragma unroll
  for (int it = 0; it < MX_NORM_ITERS; ++it) {
    const int i = threadIdx.x + it * blockDim.x;
    if (8 * i < Kp) {                                   // (quads agree: H and Kp are multiples of 32)
#pragma unroll
      for (int j = 0; j < 8; ++j) v[it][j] = i < nvec ? v[it][j] * inv * (float)gw[it][j] : 0.f;
      mx_store8(q + row * ldq + 8 * i, s + row * lds + (i >> 2), v[it]);
    }
  }
}

inline unsigned mx_blocks(long groups) {
  const long b = (groups + 255) / 256;
  return (unsigned)(b < 256 * 16 ? b : 256 * 16);
}

}  // namespace

// x [M][K] (row stride ldx, a multiple of 8 elements, 16-byte aligned) -> q, s.  K % 32 == 0; q rows hold Kp >= K columns (a multiple
// of 32; 1 byte each with 8 bits, half with 4), columns from K on zeros; s rows Kp / 32 bytes.
// src [M] or null: row i is that of x [x_rows] that src names.
VDAMD_API int vdamd_mx_quantize(void* q, long ldq, void* s, long lds, const void* x, long ldx, long M, int K, int Kp, int bits,
                                const int* src, int x_rows, int dtype, void* stream) {
  if (M <= 0) return 0;
  if (src != nullptr && x_rows <= 0) return -1;
  if (K <= 0 || K % 32 || Kp < K || Kp % 32 || ldx % 8 || ldx < K || (uintptr_t)x % 16 || (uintptr_t)q % 16 || lds < Kp / 32) return -1;
  if ((bits != 8 && bits != 4) || ldq % 16 || ldq < (bits == 8 ? Kp : Kp / 2)) return -1;
  const int per_row = Kp / 8;
  const long groups = M * per_row;
  hipStream_t st = (hipStream_t)stream;
#define GO(T, B) mx_quantize_kernel<T, B><<<mx_blocks(groups), 256, 0, st>>>((uint8_t*)q, ldq, (uint8_t*)s, lds, (const T*)x, ldx, groups, per_row, K, src, x_rows)
  if (dtype == DT_BF16) { if (bits == 8) GO(bf16_t, 8); else GO(bf16_t, 4); }
  else if (dtype == DT_F16) { if (bits == 8) GO(f16_t, 8); else GO(f16_t, 4); }
  else if (dtype == DT_F32) { if (bits == 8) GO(float, 8); else GO(float, 4); }
  else return -2;
#undef GO
  HIP_LAUNCH_CHECK();
  return 0;
}

// q, s -> out [M][K], contiguous
VDAMD_API int vdamd_mx_dequantize(void* out, const void* q, long ldq, const void* s, long lds, long M, int K, int bits, int dtype,
                                  void* stream) {
  if (M <= 0) return 0;
  if (K <= 0 || K % 32 || (bits != 8 && bits != 4) || ldq % (bits == 8 ? 8 : 4) || (uintptr_t)q % 8 || (uintptr_t)out % 16) return -1;
  if (ldq < (bits == 8 ? K : K / 2) || lds < K / 32) return -1;
  const int per_row = K / 8;
  const long groups = M * per_row;
  hipStream_t st = (hipStream_t)stream;
#define GO(T, B) mx_dequantize_kernel<T, B><<<mx_blocks(groups), 256, 0, st>>>((T*)out, (const uint8_t*)q, ldq, (const uint8_t*)s, lds, groups, per_row)
  if (dtype == DT_BF16) { if (bits == 8) GO(bf16_t, 8); else GO(bf16_t, 4); }
  else if (dtype == DT_F16) { if (bits == 8) GO(f16_t, 8); else GO(f16_t, 4); }
  else if (dtype == DT_F32) { if (bits == 8) GO(float, 8); else GO(float, 4); }
  else return -2;
#undef GO
  HIP_LAUNCH_CHECK();
  return 0;
}

// q, s = RMSNorm(x + residual) w in 8 bits, residual_out = x + residual in 16 (both null: of x alone).  slabs != null: x is the sum of
// ks fp32 slabs [ks][M][H].  H % 32 == 0, Kp as in vdamd_mx_quantize; rows of x ldx elements apart, of the others H.
VDAMD_API int vdamd_mx_rms_norm(void* q, long ldq, void* s, long lds, void* residual_out, const void* x, long ldx, const float* slabs,
                                int ks, const void* residual, const void* w, float eps, int M, int H, int Kp, int dtype, void* stream) {
  if (M <= 0) return 0;
  if (H <= 0 || H % 32 || Kp < H || Kp % 32 || Kp > 8 * 1024 * MX_NORM_ITERS || ldq % 16 || ldq < Kp || lds < Kp / 32) return -1;
  if ((residual == nullptr) != (residual_out == nullptr) || (x == nullptr) == (slabs == nullptr) || (slabs != nullptr && ks < 1)) return -1;
  if (x != nullptr && (ldx % 8 || ldx < H || (uintptr_t)x % 16)) return -1;
  if (((uintptr_t)q | (uintptr_t)residual | (uintptr_t)residual_out | (uintptr_t)w | (uintptr_t)slabs) % 16) return -1;
  hipStream_t st = (hipStream_t)stream;
  int threads = ((Kp / 8 + MX_NORM_ITERS - 1) / MX_NORM_ITERS + 63) / 64 * 64;
  if (dtype == DT_BF16)
    mx_rms_norm_kernel<bf16_t><<<M, threads, 0, st>>>((uint8_t*)q, ldq, (uint8_t*)s, lds, (bf16_t*)residual_out, (const bf16_t*)x, ldx,
                                                      slabs, ks, (long)M * H, (const bf16_t*)residual, (const bf16_t*)w, eps, H, Kp);
  else if (dtype == DT_F16)
    mx_rms_norm_kernel<f16_t><<<M, threads, 0, st>>>((uint8_t*)q, ldq, (uint8_t*)s, lds, (f16_t*)residual_out, (const f16_t*)x, ldx,
                                                     slabs, ks, (long)M * H, (const f16_t*)residual, (const f16_t*)w, eps, H, Kp);
  else
    return -2;
  HIP_LAUNCH_CHECK();
  return 0;
}
