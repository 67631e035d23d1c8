// Products of 8-bit microscaled rows (e4m3) with 4-bit microscaled weights (e2m1) on the scaled matrix instruction of gfx950:
//   y[m][n] = sum_b 2^(xs[m][b] + ws[n][b]) sum_{k in block b} xq[m][k] wq[n][k] (+ bias[n]),   blocks of 32 columns,
// plain, as fp32 slabs of a split K, or as the gated half of a feed-forward whose result leaves in 8 bits again
//   a = silu(g) u,   or  (clamp(u) + 1) g' sigmoid(alpha g'), g' = min(g, limit);   q, s = blocks of a  (mx.h)
// with g, u the products with rows n and N/2 + n of the weight: the activation and its quantisation see the 32-bit sums.
//
// Lane (r, q) = (lane & 15, lane >> 4) of a 16x16x128 instruction holds, of row r of each operand and a 128-column step,
//   4-bit operand: columns 32 q .. 32 q + 31 (16 bytes);   8-bit operand: columns 16 q .. + 15 and 64 + 16 q .. + 15 (two times 16 bytes);
//   scale: one byte, of columns 32 q .. 32 q + 31.
// Weights are laid out for it once: qw [N/16][K/128][64 lanes][16 bytes] (a 16-row tile of a step is one 1 KiB read),
// ws [N/16][K/512][64 lanes][4 bytes], byte i the scale of step 4 j + i.  Rows of x are as the quantising kernels leave them.
// The weights are the instruction's first operand, so a lane ends with four neighbouring columns of one row of y.
#include "mx.h"

namespace {

enum { MX_OUT = 0, MX_SLAB = 1, MX_GLU = 2 };

struct MxArgs {
  const uint8_t* xq; long ldq;
  const uint8_t* xs; long lds;
  const uint8_t* qw;
  const uint8_t* ws;
  void* out; long ldo;              // MX_OUT: rows of y; MX_GLU: rows of 8-bit elements
  uint8_t* os; long ldos;           // MX_GLU: their scales
  float* partial;                   // MX_SLAB: [ksplit][M][N]
  const void* bias;                 // [N] of the model type (MX_GLU: [gate ; up]), or null
  int M, N, KB, ksplit;             // KB: steps of 128 columns
  float limit, alpha;               // MX_GLU: limit 0: SiLU
  // experts: row tiles (matrix, first row, rows) of rows sorted by expert; sorted row r is row src[r] of x (src null: r)
  const int* tiles; int num_tiles; int groups; const int* src; int x_rows;
};

__device__ __forceinline__ f32x4 mx_mfma(mx_u32x4 w, mx_u32x4 x0, mx_u32x4 x1, f32x4 c, uint32_t sw, uint32_t sx) {
#if defined(__HIP_DEVICE_COMPILE__)
  const mx_i32x8 a = {(int)w[0], (int)w[1], (int)w[2], (int)w[3], 0, 0, 0, 0};
  const mx_i32x8 b = {(int)x0[0], (int)x0[1], (int)x0[2], (int)x0[3], (int)x1[0], (int)x1[1], (int)x1[2], (int)x1[3]};
  c = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 4, 0, 0, (int)sw, 0, (int)sx);
#endif
  return c;
}

__device__ __forceinline__ float mx_glu(float g, float u, float limit, float alpha) {
  if (limit > 0.f) {
    g = g > limit ? limit : g;                      // (a NaN stays one)
    u = u > limit ? limit : (u < -limit ? -limit : u);
    return (u + 1.f) * g * fast_sigmoid(alpha * g);
  }
  return g * fast_sigmoid(g) * u;
}

// 16 gated values of a row's block of 32 are with each of four lanes (r, q), 4 columns from 4 q of both 16-column halves: elements and scale
__device__ __forceinline__ void mx_store_block(uint8_t* q, uint8_t* s, const float (&a)[2][4], int lane, bool ok) {
  uint32_t m = 0;
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int r = 0; r < 4; ++r) m = max(m, mx_abs_bits(a[h][r]));
  m = max(m, (uint32_t)__shfl_xor((int)m, 16, 64));
  m = max(m, (uint32_t)__shfl_xor((int)m, 32, 64));
  const uint32_t byte = mx_scale_byte<8>(m);
  const float inv = mx_inverse(byte);
  if (!ok) return;
#pragma unroll
  for (int h = 0; h < 2; ++h)
    *reinterpret_cast<uint32_t*>(q + 16 * h + 4 * (lane >> 4)) = mx_pack_fp8(a[h][0], a[h][1], a[h][2], a[h][3], inv);
  if (lane < 16) *s = (uint8_t)byte;
}

// Few rows: the weights' bytes are the time.  A workgroup has four 16-column tiles (MX_GLU: two of the gate and the two of the same
// columns of the up half); its four waves split K, each streaming its part of the tiles straight into registers; MT row tiles of x
// come from the caches.  grid = (tiles / 4, ksplit, row tiles)
constexpr int MX_NT = 4;
template <typename T, int MT, int EPI>
__global__ __launch_bounds__(256) void mx_stream_kernel(const MxArgs a) {
  __shared__ f32x4 red[4][MX_NT][MT][64];
  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, q = lane >> 4;
  const int KB = a.KB, SS = (KB + 3) >> 2, ntiles = (a.N + 15) >> 4;
  int row0 = blockIdx.z * (16 * MT), rows = min(a.M - row0, 16 * MT), group = 0;
  if (a.tiles != nullptr) {
    const int* d = a.tiles + 3 * blockIdx.z;
    rows = min(d[2], 16 * MT);
    if (rows <= 0) return;
    group = min(max(d[0], 0), a.groups - 1);
    row0 = min(max(d[1], 0), a.M - 1);
    rows = min(rows, a.M - row0);
  }
  const uint8_t* qw = a.qw + (long)group * ntiles * KB * 1024;
  const uint8_t* ws = a.ws + (long)group * ntiles * SS * 256;
  const T* bias = a.bias == nullptr ? nullptr : (const T*)a.bias + (long)group * a.N;

  int nt[MX_NT];
#pragma unroll
  for (int t = 0; t < MX_NT; ++t) {
    if (EPI == MX_GLU) nt[t] = 2 * blockIdx.x + (t & 1) + (t >> 1) * (ntiles >> 1);
    else nt[t] = min(4 * (int)blockIdx.x + t, ntiles - 1);
  }
  const uint8_t *xp[MT], *sp[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    long row = row0 + min(16 * i + r, rows - 1);
    if (a.src != nullptr) row = min(max(a.src[row], 0), a.x_rows - 1);
    xp[i] = a.xq + row * a.ldq + 16 * q;
    sp[i] = a.xs + row * a.lds + q;
  }
  // this wave's steps
  const int part = blockIdx.y * 4 + wid, parts = 4 * a.ksplit;
  const int lo = (int)((long)KB * part / parts), hi = (int)((long)KB * (part + 1) / parts);

  f32x4 acc[MX_NT][MT];
#pragma unroll
  for (int t = 0; t < MX_NT; ++t)
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[t][i] = f32x4{0.f, 0.f, 0.f, 0.f};

  mx_u32x4 w[2][MX_NT], x0[2][MT], x1[2][MT];
  uint32_t sw[2][MX_NT], sx[2][MT];
  auto load = [&](int b, int k) {
#pragma unroll
    for (int t = 0; t < MX_NT; ++t) {
      w[b][t] = *reinterpret_cast<const mx_u32x4*>(qw + ((long)nt[t] * KB + k) * 1024 + lane * 16);
      sw[b][t] = ws[((long)nt[t] * SS + (k >> 2)) * 256 + lane * 4 + (k & 3)];
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      x0[b][i] = *reinterpret_cast<const mx_u32x4*>(xp[i] + 128L * k);
      x1[b][i] = *reinterpret_cast<const mx_u32x4*>(xp[i] + 128L * k + 64);
      sx[b][i] = sp[i][4 * k];
    }
  };
  auto mma = [&](int b) {
#pragma unroll
    for (int t = 0; t < MX_NT; ++t)
#pragma unroll
      for (int i = 0; i < MT; ++i) acc[t][i] = mx_mfma(w[b][t], x0[b][i], x1[b][i], acc[t][i], sw[b][t], sx[b][i]);
  };
  if (lo < hi) load(0, lo);
  for (int k = lo; k < hi; k += 2) {
    if (k + 1 < hi) load(1, k + 1);
    mma(0);
    if (k + 1 < hi) {
      if (k + 2 < hi) load(0, k + 2);
      mma(1);
    }
  }

#pragma unroll
  for (int t = 0; t < MX_NT; ++t)
#pragma unroll
    for (int i = 0; i < MT; ++i) red[wid][t][i][lane] = acc[t][i];
  __syncthreads();
  auto sum = [&](int t, int i) { return (red[0][t][i][lane] + red[1][t][i][lane]) + (red[2][t][i][lane] + red[3][t][i][lane]); };
  if constexpr (EPI == MX_GLU) {
    const int cols = a.N >> 1, n = 32 * blockIdx.x + 4 * q;
    for (int i = wid; i < MT; i += 4) {
      const int m = 16 * i + r;
      float v[2][4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const f32x4 g = sum(h, i), u = sum(2 + h, i);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int c = n + 16 * h + e;
          v[h][e] = mx_glu(g[e] + (bias ? (float)bias[c] : 0.f), u[e] + (bias ? (float)bias[cols + c] : 0.f), a.limit, a.alpha);
        }
      }
      const long row = row0 + min(m, rows - 1);
      mx_store_block((uint8_t*)a.out + row * a.ldo + 32 * blockIdx.x, a.os + row * a.ldos + blockIdx.x, v, lane, m < rows);
    }
  } else {
    const int tile = 4 * blockIdx.x + wid, n = 16 * tile + 4 * q;
    if (n >= a.N) return;
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const int m = 16 * i + r;
      const f32x4 v = sum(wid, i);
      if (m >= rows) continue;
      if constexpr (EPI == MX_SLAB) {
        *reinterpret_cast<f32x4*>(a.partial + ((long)blockIdx.y * a.M + row0 + m) * a.N + n) = v;
      } else {
        typename Vec4<T>::type o;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = (T)(v[e] + (bias ? (float)bias[n + e] : 0.f));
        *reinterpret_cast<typename Vec4<T>::type*>((T*)a.out + (row0 + m) * a.ldo + n) = o;
      }
    }
  }
}

// y = sum of the slabs + bias
template <typename T>
__global__ __launch_bounds__(256) void mx_reduce_kernel(T* __restrict__ out, long ldo, const float* __restrict__ partial,
                                                        const T* __restrict__ bias, int M, int N, int ksplit) {
  const long i = blockIdx.x * 256L + threadIdx.x;
  const int quads = N >> 2;
  if (i >= (long)M * quads) return;
  const int m = (int)(i / quads), n = (int)(i - (long)m * quads) * 4;
  f32x4 s = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int k = 0; k < ksplit; ++k) s += *reinterpret_cast<const f32x4*>(partial + ((long)k * M + m) * N + n);
  typename Vec4<T>::type o;
#pragma unroll
  for (int e = 0; e < 4; ++e) o[e] = (T)(s[e] + (bias ? (float)bias[n + e] : 0.f));
  *reinterpret_cast<typename Vec4<T>::type*>(out + m * ldo + n) = o;
}

template <typename T, int EPI>
int mx_stream(const MxArgs& a, int mt, hipStream_t st) {
  const int ntiles = (a.N + 15) / 16;
  dim3 grid((ntiles + 3) / 4, a.ksplit, a.tiles != nullptr ? a.num_tiles : (a.M + 16 * mt - 1) / (16 * mt));
  if (grid.y > 65535 || grid.z > 65535) return -7;
  switch (mt) {
    case 1: mx_stream_kernel<T, 1, EPI><<<grid, 256, 0, st>>>(a); break;
    case 2: mx_stream_kernel<T, 2, EPI><<<grid, 256, 0, st>>>(a); break;
    case 4: mx_stream_kernel<T, 4, EPI><<<grid, 256, 0, st>>>(a); break;
    default: return -6;
  }
  HIP_LAUNCH_CHECK();
  return 0;
}

template <typename T>
int mx_dispatch(const MxArgs& a, int epi, int mt, hipStream_t st) {
  if (epi == MX_GLU) return mx_stream<T, MX_GLU>(a, mt, st);
  if (epi == MX_SLAB || a.ksplit > 1) {
    const int rc = mx_stream<T, MX_SLAB>(a, mt, st);
    if (rc != 0 || epi == MX_SLAB) return rc;
    const long n = (long)a.M * (a.N / 4);
    mx_reduce_kernel<T><<<(unsigned)((n + 255) / 256), 256, 0, st>>>((T*)a.out, a.ldo, a.partial, (const T*)a.bias, a.M, a.N, a.ksplit);
    HIP_LAUNCH_CHECK();
    return 0;
  }
  return mx_stream<T, MX_OUT>(a, mt, st);
}

}  // namespace

// xq [x_rows][128 KB] bytes (rows ldq apart, a multiple of 16), xs [x_rows][4 KB] scale bytes (rows lds apart, a multiple of 4); qw, ws as
// above for `groups` matrices of N rows (padded to 16), N % 8 == 0.
// epi 0: out [M][N] of the model type, rows ldo elements apart (ksplit > 1: through partial [ksplit][M][N]); 1: partial alone;
// 2: N = [gate ; up], N % 256 == 0: out [M][N / 2] elements, os their scales, ksplit 1; limit 0: SiLU.
// tiles [num_tiles][3] (matrix, first row, rows) or null; src [M] or null: the row of x behind each row.  row_tiles: 16-row tiles a
// workgroup takes (1, 2 or 4; of `tiles` at most 16 row_tiles rows each).
VDAMD_API int vdamd_mx_gemm(void* out, long ldo, void* os, long ldos, float* partial, const void* xq, long ldq, const void* xs, long lds,
                            int x_rows, const void* qw, const void* ws, const void* bias, int M, int N, int KB, int ksplit, int epi,
                            float limit, float alpha, const int* tiles, int num_tiles, int groups, const int* src, int row_tiles,
                            int dtype, void* stream) {
  if (M <= 0 || (tiles != nullptr && num_tiles <= 0)) return 0;
  if (N <= 0 || N % 8 || KB <= 0 || x_rows <= 0 || groups <= 0 || ksplit < 1 || ksplit > KB || (src == nullptr && x_rows < M)) return -1;
  if (ldq % 16 || ldq < 128L * KB || lds < 4L * KB || ((uintptr_t)xq | (uintptr_t)qw) % 16 || (uintptr_t)ws % 4) return -1;
  if (epi == MX_GLU && (N % 256 || ksplit != 1 || ldo % 16 || (uintptr_t)out % 16 || ldo < N / 2 || os == nullptr || ldos < N / 64)) return -1;
  if (epi == MX_OUT && (ldo % 4 || ldo < N || (uintptr_t)out % 8 || (ksplit > 1 && partial == nullptr))) return -1;
  if (epi == MX_SLAB && partial == nullptr) return -1;
  if ((ksplit > 1 || epi == MX_SLAB) && tiles != nullptr) return -1;
  if (epi < 0 || epi > 2) return -1;
  const MxArgs a = {(const uint8_t*)xq, ldq, (const uint8_t*)xs, lds, (const uint8_t*)qw, (const uint8_t*)ws, out, ldo, (uint8_t*)os, ldos,
                    partial, bias, M, N, KB, ksplit, limit, alpha, tiles, num_tiles, groups, src, x_rows};
  hipStream_t st = (hipStream_t)stream;
  if (dtype == DT_BF16) return mx_dispatch<bf16_t>(a, epi, row_tiles, st);
  if (dtype == DT_F16) return mx_dispatch<f16_t>(a, epi, row_tiles, st);
  return -2;
}
