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
  float* partial;                   // MX_SLAB: 32-bit rows [ksplit][M][N]
  const void* bias;                 // [N] of the model type (MX_GLU: [gate ; up]), or null
  int M, N, KB, ksplit;             // KB: steps of 128 columns
  float limit, alpha;               // MX_GLU: limit 0: SiLU
  // experts: row tiles (matrix, first row, rows) of rows sorted by expert; sorted row r is row src[r] of x (src null: r)
  const int* tiles; int num_tiles; int groups; const int* src; int x_rows;
  const void* x16; long ldx; int K; // rows of the model type with K columns, quantised in the kernel (xq null)
};

__device__ __forceinline__ f32x4 mx_mfma(mx_u32x4 w, mx_i32x8 x, f32x4 c, uint32_t sw, uint32_t sx) {
#if defined(__HIP_DEVICE_COMPILE__)
  const mx_i32x8 a = {(int)w[0], (int)w[1], (int)w[2], (int)w[3], 0, 0, 0, 0};      // (the 4-bit form reads four registers)
  c = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, x, c, 4, 0, 0, (int)sw, 0, (int)sx);
#endif
  return c;
}

// the two 16-byte halves of an 8-bit fragment
template <typename P> __device__ __forceinline__ mx_i32x8 mx_fragment(const P* lo, const P* hi) {
  const mx_i32x4 a = *reinterpret_cast<const mx_i32x4*>(lo), b = *reinterpret_cast<const mx_i32x4*>(hi);
  return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

// Both forms as (u' + plus) g' sigmoid(alpha g') with u' = u limited to +-top, g' = g to top: SiLU has no limit.  (A branch for each value
// keeps the next one's exponential from starting under it: 22528 x 5888 x 2944 in 256-row tiles 395 us with limits, 365 without; so 349, 340.)
struct MxGlu {
  float top, plus, alpha;
  __device__ __forceinline__ MxGlu(float limit, float a) : top(limit > 0.f ? limit : __uint_as_float(0x7f800000u)),
                                                           plus(limit > 0.f ? 1.f : 0.f), alpha(limit > 0.f ? a : 1.f) {}
  __device__ __forceinline__ float operator()(float g, float u) const {
    g = g > top ? top : g;                          // (a NaN stays one)
    u = u > top ? top : (u < -top ? -top : u);
    return (u + plus) * g * fast_sigmoid(alpha * g);
  }
};

// A row's block of 32 gated values is with four lanes (r, q), 4 columns from 4 q of both its 16-column halves: elements and scale.  All
// 64 lanes run; ok: the row is stored
__device__ __forceinline__ void mx_store_block(uint8_t* q, uint8_t* s, const float (&a)[2][4], int lane, bool ok) {
#if defined(__HIP_DEVICE_COMPILE__)
  uint32_t m = 0;
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int r = 0; r < 4; ++r) m = max(m, mx_abs_bits(a[h][r]));
  const auto far = __builtin_amdgcn_permlane32_swap(m, m, false, false);
  m = max((uint32_t)far[0], (uint32_t)far[1]);
  const auto near = __builtin_amdgcn_permlane16_swap(m, m, false, false);
  m = max((uint32_t)near[0], (uint32_t)near[1]);
  const uint32_t byte = mx_scale_byte<8>(m);
  const float inv = mx_inverse(byte);
  // lanes of even q trade their second half for the first of the lane after them: eight neighbouring bytes each
  const auto w = __builtin_amdgcn_permlane16_swap(mx_pack_fp8(a[0][0], a[0][1], a[0][2], a[0][3], inv),
                                                  mx_pack_fp8(a[1][0], a[1][1], a[1][2], a[1][3], inv), false, false);
  const int at = lane >> 4;
  if (!ok) return;
  *reinterpret_cast<mx_u32x2*>(q + ((at & 1) ? 16 + 4 * (at - 1) : 4 * at)) = mx_u32x2{(uint32_t)w[0], (uint32_t)w[1]};
  if (lane < 16) *s = (uint8_t)byte;
#endif
}

// Few rows: the weights' bytes are the time.  A workgroup has NT 16-column tiles (MX_GLU: two of the gate and the two of the same columns
// of the up half); its waves split K, each streaming its part of the tiles straight into registers, PF steps ahead; MT row tiles of x
// come from the caches.  QUANT: x holds 16-bit rows, at most 16, which every workgroup quantises for itself into LDS while its first
// weights are on their way: one launch instead of two.  grid = (tiles / NT, ksplit, row tiles)
template <typename T, int MT, int NT, int WAVES, int EPI, bool QUANT, int PF>
__global__ __launch_bounds__(64 * WAVES) void mx_stream_kernel(const MxArgs a) {
  extern __shared__ __attribute__((aligned(16))) unsigned char dyn[];      // QUANT: rows of payload, 16 bytes apart from a multiple of 128; scales
  __shared__ f32x4 red[WAVES][NT][MT][64];
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

  const uint8_t *wp[NT], *wsp[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int nt = EPI == MX_GLU ? 2 * (int)blockIdx.x + (t & 1) + (t >> 1) * (ntiles >> 1) : min(NT * (int)blockIdx.x + t, ntiles - 1);
    wp[t] = qw + (long)nt * KB * 1024 + lane * 16;
    wsp[t] = ws + (long)nt * SS * 256 + lane * 4;
  }
  // this workgroup's steps, this wave's
  const int w_lo = (int)((long)KB * blockIdx.y / a.ksplit), w_n = (int)((long)KB * (blockIdx.y + 1) / a.ksplit) - w_lo;
  const int lo = w_lo + w_n * wid / WAVES, hi = w_lo + w_n * (wid + 1) / WAVES;

  const uint8_t *xp[MT], *sp[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int rr = min(16 * i + r, rows - 1);
    if constexpr (QUANT) {
      xp[i] = dyn + rr * (128 * w_n + 16) + 16 * q - 128 * w_lo;
      sp[i] = dyn + rows * (128 * w_n + 16) + rr * (4 * w_n) + q - 4 * w_lo;
    } else {
      long row = row0 + rr;
      if (a.src != nullptr) row = min(max(a.src[row], 0), a.x_rows - 1);
      xp[i] = a.xq + row * a.ldq + 16 * q;
      sp[i] = a.xs + row * a.lds + q;
    }
  }

  f32x4 acc[NT][MT];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[t][i] = f32x4{0.f, 0.f, 0.f, 0.f};

  mx_u32x4 w[PF][NT];
  mx_i32x8 x[PF][MT];
  uint32_t sw[PF][NT], sx[PF][MT];
  auto load_w = [&](int b, int k) {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const mx_u32x4* const p = reinterpret_cast<const mx_u32x4*>(wp[t] + k * 1024L);
      // One row tile reads a weight once: past the caches (51 experts of 3 x 2880 x 2880 83 + 43 -> 76 + 39 us, 2 x 28672 columns of 8192
      // by 13 rows 53 -> 50)
      if constexpr (MT == 1) w[b][t] = __builtin_nontemporal_load(p);
      else w[b][t] = *p;
      sw[b][t] = wsp[t][(k >> 2) * 256 + (k & 3)];
    }
  };
  auto load_x = [&](int b, int k) {
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      x[b][i] = mx_fragment(xp[i] + 128 * k, xp[i] + 128 * k + 64);
      sx[b][i] = sp[i][4 * k];
    }
  };
#pragma unroll
  for (int u = 0; u < PF; ++u)
    if (lo + u < hi) {
      load_w(u, lo + u);
      if constexpr (!QUANT) load_x(u, lo + u);
    }
  if constexpr (QUANT) {
    const T* src = (const T*)a.x16;
    uint8_t* const scales = dyn + rows * (128 * w_n + 16);
    const int vecs = 16 * w_n;                                   // of 8 values, in a row's part (columns from K on are zeros)
    for (int i = threadIdx.x; i < rows * vecs; i += 64 * WAVES) {
      const int m = i / vecs, c = i - m * vecs, k = 128 * w_lo + 8 * c;
      float v[8];
      if (k < a.K) {
        mx_load8(src + (long)(row0 + m) * a.ldx + k, v);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = 0.f;
      }
      mx_store8(dyn + m * (128 * w_n + 16) + 8 * c, scales + m * (4 * w_n) + (c >> 2), v);
    }
    __syncthreads();
  }
  auto mma = [&](int u, int k) {
    if constexpr (QUANT) load_x(u, k);
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < MT; ++i) acc[t][i] = mx_mfma(w[u][t], x[u][i], acc[t][i], sw[u][t], sx[u][i]);
  };
  auto load = [&](int u, int k) {
    load_w(u, k);
    if constexpr (!QUANT) load_x(u, k);
  };
  int k = lo;
  // (loads under a condition are waited for as if none had been issued behind them: only the last steps have any)
  for (; k + 2 * PF <= hi; k += PF) {
#pragma unroll
    for (int u = 0; u < PF; ++u) {
      mma(u, k + u);
      load(u, k + u + PF);
    }
  }
#pragma unroll
  for (int u = 0; u < PF; ++u)
    if (k + u < hi) {
      mma(u, k + u);
      if (k + u + PF < hi) load(u, k + u + PF);
    }
  k += PF;
#pragma unroll
  for (int u = 0; u < PF; ++u)
    if (k + u < hi) mma(u, k + u);

#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int i = 0; i < MT; ++i) red[wid][t][i][lane] = acc[t][i];
  __syncthreads();
  auto sum = [&](int t, int i) {
    f32x4 v = red[0][t][i][lane];
#pragma unroll
    for (int p = 1; p < WAVES; ++p) v += red[p][t][i][lane];
    return v;
  };
  if constexpr (EPI == MX_GLU) {
    const int cols = a.N >> 1, n = 32 * blockIdx.x + 4 * q;
    const MxGlu glu(a.limit, a.alpha);
    for (int i = wid; i < MT; i += WAVES) {
      const int m = 16 * i + r;
      float v[2][4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const f32x4 g = sum(h, i), u = sum(2 + h, i);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int c = n + 16 * h + e;
          v[h][e] = glu(g[e] + (bias ? (float)bias[c] : 0.f), u[e] + (bias ? (float)bias[cols + c] : 0.f));
        }
      }
      const long row = row0 + min(m, rows - 1);
      mx_store_block((uint8_t*)a.out + row * a.ldo + 32 * blockIdx.x, a.os + row * a.ldos + blockIdx.x, v, lane, m < rows);
    }
  } else {
    for (int j = wid; j < NT * MT; j += WAVES) {
      const int t = j % NT, i = j / NT;
      const int n = 16 * (NT * (int)blockIdx.x + t) + 4 * q, m = 16 * i + r;
      if (n >= a.N || m >= rows) continue;
      f32x4 v = sum(t, i);
      if (bias != nullptr)
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] += (float)bias[n + e];
      if constexpr (EPI == MX_SLAB) {
        *reinterpret_cast<f32x4*>(a.partial + ((long)blockIdx.y * a.M + row0 + m) * a.N + n) = v;
      } else {
        typename Vec4<T>::type o;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = (T)v[e];
        *reinterpret_cast<typename Vec4<T>::type*>((T*)a.out + (row0 + m) * a.ldo + n) = o;
      }
    }
  }
}

// The bias of 32 columns from n0 (the same for the wave) for a lane with columns 16 j + 4 q .. + 3 of them: by scalar loads, since a vector
// load could only be waited for together with everything in flight.  Columns from N on: zeros
template <typename T>
__device__ __forceinline__ void mx_bias(float (&b)[2][4], const void* bias, long group, int n0, int N, int q) {
  typedef const __attribute__((address_space(4))) uint32_t* words;
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) b[j][e] = 0.f;
  if (bias == nullptr) return;
  const T* p = (const T*)bias + group;
  if (n0 + 32 <= N) {
    words w = (words)(uintptr_t)(p + n0);
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t v = w[8 * j + h];
#pragma unroll
        for (int i = 1; i < 4; ++i) v = q == i ? w[8 * j + 2 * i + h] : v;
        typedef T pair __attribute__((ext_vector_type(2)));
        const pair t = __builtin_bit_cast(pair, v);
        b[j][2 * h] = (float)t[0];
        b[j][2 * h + 1] = (float)t[1];
      }
  } else {
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int n = n0 + 16 * j + 4 * q + e;
        if (n < N) b[j][e] = (float)p[n];
      }
  }
}

// Many rows: the matrix cores are the time.  256 x 256 outputs a tile (MX_GLU: 128 columns of the gate and the same of the up half), one
// persistent workgroup of eight waves a compute unit, K in steps of 128.
//  * Both operands go from memory to LDS without passing through registers.  A step is four images: A0, A1 (128 rows x 128 bytes of
//    x; the 16-byte slots of a row XOR-ed with (row >> 1) & 7 at the source, so that the lanes of a fragment read meet no bank twice)
//    and B0, B1 (eight weight tiles of 1 KiB, in the order in which lanes read them).  Two sets of images.
//  * A wave has 128 x 64 outputs as four quadrants of 64 x 32, quadrant (mq, nq) from images A<mq> and B<nq>; a step is four phases of
//    eight matrix instructions, one quadrant each, every fragment read once.  Even steps go A0 B0, A1 B0, A1 B1, A0 B1, odd ones begin
//    with A1: registers of the half that a step begins with are free a phase before it, so the 20 fragment reads of a step spread as
//    6, 6, 4, 4 over its phases and stay below the matrix instructions' time in each (as 8, 8, 2, 2: 2780 TFLOP/s instead of 2880).
//  * The loads are one stream that never drains.  Of step t are issued: B0 in phase 1 of step t - 2, the first A half in 2, the second in
//    3, B1 in phase 0 of step t - 1; each at least two phases after the image before it was read.  A phase waits for what the next one
//    reads, all but the newest six loads of a wave (an A image is two, a B image one).  It runs on through the output tiles.
//  * Scales come 16 bytes a row (four steps) at a time into two further sets, one load of each wave in every other step, at its phase 1:
//    one more in the counts until they are older.  Lanes read their byte from LDS.
//  * Waves 4-7 run one barrier behind waves 0-3: on each SIMD one wave multiplies while the other reads.
//  * An odd number of steps gets one more, whose weights are zeros: loads out of the descriptor's range.
constexpr int MXB_A = 128 * 128, MXB_B = 8 * 1024, MXB_SET = 2 * MXB_A + 2 * MXB_B, MXB_SC = 2 * 4096;
typedef __attribute__((address_space(3))) void mx_lds_void;

template <typename T, int EPI, bool grouped>
__global__ __launch_bounds__(512) void mx_big_kernel(const MxArgs a, int ntm, int ntn) {
#if defined(__HIP_DEVICE_COMPILE__)      // the buffer-descriptor builtins exist in the device pass only
  __shared__ __attribute__((aligned(1024))) unsigned char smem[2 * MXB_SET + 2 * MXB_SC];
  const int lane = threadIdx.x & 63;
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wr = wid >> 2, wc = wid & 3;
  const int r16 = lane & 15, q = lane >> 4;
  const int KB = a.KB, SS = (KB + 3) >> 2, KT = (KB + 1) & ~1, ntiles = (a.N + 15) >> 4;

  // ---- this workgroup's tiles: bands of 8 row tiles, in a band every XCD a range of tile columns, column by column (as the 16-bit
  // product's large tiles: 32 workgroups of an XCD share 12 panels in its L2).  Grouped: two row tiles at a time, column by column, an
  // eighth of all outputs to each XCD - of the entries that hold rows, so that the unused ones leave nobody idle
  const int xcd = blockIdx.x & 7, stride = gridDim.x >> 3;
  const int c0 = (int)((long)ntn * xcd >> 3), c1 = (int)((long)ntn * (xcd + 1) >> 3), ncols = c1 - c0;
  int lo = 0, hi = ntm;                      // the entries with rows (all of them: unused ones are in front and behind)
  if (grouped) {
    lo = ntm, hi = 0;
    for (int i = threadIdx.x; i < ntm; i += 512)
      if (a.tiles[3 * i + 2] > 0) lo = min(lo, i), hi = i + 1;
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) lo = min(lo, __shfl_xor(lo, d)), hi = max(hi, __shfl_xor(hi, d));
    int* const red = reinterpret_cast<int*>(smem);
    if (lane == 0) red[wid] = lo, red[8 + wid] = hi;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) lo = min(lo, red[i]), hi = max(hi, red[8 + i]);
    lo = __builtin_amdgcn_readfirstlane(lo), hi = __builtin_amdgcn_readfirstlane(hi);
    __syncthreads();
  }
  const int pairs = grouped ? max(hi - lo, 0) / 2 * 2 * ntn : 0;      // outputs of whole pairs of row tiles
  const long all = grouped ? (long)max(hi - lo, 0) * ntn : 0;
  const int chunk_end = grouped ? (int)(all * (xcd + 1) >> 3) : ntm * ncols;
  auto row_tile = [&](int tl) { return tl < pairs ? lo + 2 * (tl / (2 * ntn)) + (tl & 1) : hi - 1; };
  auto column = [&](int tl) { return tl < pairs ? tl % (2 * ntn) >> 1 : tl - pairs; };
  auto entry = [&](int rt, int i) { return __builtin_amdgcn_readfirstlane(a.tiles[3 * rt + i]); };
  auto used = [&](int tl) {                  // the first entry with rows from tl on
    if (grouped)
      while (tl < chunk_end) {
        const int rt = row_tile(tl);
        if (entry(rt, 2) > 0) break;
        tl += stride;
      }
    return tl;
  };
  int tile = used((grouped ? (int)(all * xcd >> 3) : 0) + (blockIdx.x >> 3));
  if (tile >= chunk_end) return;
  auto decode = [&](int tl, int& m0, int& end, int& tn, int& g) {      // first row, row limit, tile column, matrix
    if (grouped) {
      const int rt = row_tile(tl);
      g = min(max(entry(rt, 0), 0), a.groups - 1);
      m0 = min(max(entry(rt, 1), 0), a.M - 1);
      end = min(a.M, m0 + min(entry(rt, 2), 256));
      tn = column(tl);
      return;
    }
    const int band = tl / (8 * ncols), rows = min(8, ntm - 8 * band), in = tl - band * 8 * ncols;
    m0 = (8 * band + in % rows) * 256;
    end = a.M;
    tn = c0 + in / rows;
    g = 0;
  };

  // ---- staging.  Everything that depends on the output tile is scalar; rows and weight tiles past the end are out of their
  // descriptors' range and come as zeros
  const auto xr = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(a.xq), 0, (int)(unsigned)((long)a.x_rows * a.ldq), 0x00020000);
  const unsigned wbytes = (unsigned)((long)ntiles * KB * 1024), sbytes = (unsigned)((long)ntiles * SS * 256);
  const unsigned ldq = (unsigned)a.ldq, half_tiles = ntiles >> 1;
  struct Stage { unsigned rows, b0, b1, sc; int g; };        // byte offsets of the tile's rows, weight tiles and scales of this wave
  auto stage_of = [&](int tl) {
    int m0, end, tn, g;
    decode(tl, m0, end, tn, g);
    const unsigned t0 = EPI == MX_GLU ? 8 * tn : 16 * tn, t1 = EPI == MX_GLU ? half_tiles + 8 * tn : 16 * tn + 8;
    const unsigned i = 4 * (wid & 1);
    return Stage{(unsigned)(m0 + 16 * wid) * ldq, (t0 + wid) * (unsigned)(KB * 1024), (t1 + wid) * (unsigned)(KB * 1024),
                 wid < 4 ? (unsigned)(m0 + 64 * wid) * (unsigned)a.lds : ((wid < 6 ? t0 : t1) + i) * (unsigned)(SS * 256), g};
  };
  auto weights = [&](int g) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(a.qw + (long)g * wbytes), 0, (int)wbytes, 0x00020000);
  };
  auto scales = [&](int g) {
    return wid < 4 ? __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(a.xs), 0, (int)(unsigned)((long)a.x_rows * a.lds), 0x00020000)
                   : __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(a.ws + (long)g * sbytes), 0, (int)sbytes, 0x00020000);
  };
  const unsigned lane_a = (unsigned)(lane >> 3) * ldq + 16 * ((lane & 7) ^ (lane >> 4)), lane_b = 16 * lane;
  const unsigned lane_s = wid < 4 ? (unsigned)lane * (unsigned)a.lds : (unsigned)(lane >> 4) * (unsigned)(SS * 256) + 16 * (lane & 15);
  auto wrs = weights(0);
  auto srs = scales(0);
  Stage cur, nxt;                            // of the tile being staged, of the one after it
  // steps past the last address the staging tile's first: by then `cur` is the next output tile's.  The step of zeros takes x from the
  // last one
  auto stage_a = [&](int half, int set, int kt) {
    const int k = min(kt >= KT ? kt - KT : kt, KB - 1);
    const unsigned off = lane_a + (cur.rows + (unsigned)half * 128 * ldq);
    unsigned char* const to = smem + set * MXB_SET + half * MXB_A + 2048 * wid;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(xr, (mx_lds_void*)to, 16, off, k * 128, 0, 0);
    // (eight rows on: the slots' XOR differs by 4; ldq is a multiple of 128)
    __builtin_amdgcn_raw_ptr_buffer_load_lds(xr, (mx_lds_void*)(to + 1024), 16, (off + 8 * ldq) ^ 64, k * 128, 0, 0);
  };
  auto stage_b = [&](int half, int set, int kt) {
    const int k = kt >= KT ? kt - KT : kt;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(wrs, (mx_lds_void*)(smem + set * MXB_SET + 2 * MXB_A + half * MXB_B + wid * 1024), 16,
                                             k < KB ? lane_b + (half ? cur.b1 : cur.b0) : 0xfffffff0u, k < KB ? k * 1024 : 0, 0, 0);
  };
  auto stage_s = [&](int set, int ss) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(srs, (mx_lds_void*)(smem + 2 * MXB_SET + set * MXB_SC + wid * 1024), 16, lane_s + cur.sc,
                                             ss * (wid < 4 ? 16 : 256), 0, 0);
  };

  // ---- fragments
  const int swz = (r16 >> 1) & 7, so0 = (q ^ swz) << 4, so1 = ((4 + q) ^ swz) << 4;
  const int xro = (wr * 64 + r16) * 128, wro = 2 * MXB_A + wc * 2048 + lane * 16;
  const int xso = 2 * MXB_SET + (wr * 64 + r16) * 16 + q, wso = 2 * MXB_SET + 4096 + wc * 512 + lane * 4;
  auto read_x = [&](mx_i32x8 (&f)[4], uint32_t (&s)[4], int from, int to, int set, int half, int sbyte) {
    const unsigned char* b = smem + set * MXB_SET + half * MXB_A + xro;
#pragma unroll
    for (int i = from; i < to; ++i) f[i] = mx_fragment(b + i * 2048 + so0, b + i * 2048 + so1);
#pragma unroll
    for (int i = from; i < to; ++i) s[i] = smem[xso + sbyte + half * 2048 + i * 256];
  };
  auto read_w = [&](mx_u32x4 (&f)[2], uint32_t (&s)[2], int set, int half, int sbyte, int step) {
    const unsigned char* b = smem + set * MXB_SET + half * MXB_B + wro;
#pragma unroll
    for (int j = 0; j < 2; ++j) f[j] = *reinterpret_cast<const mx_u32x4*>(b + j * 1024);
#pragma unroll
    for (int j = 0; j < 2; ++j) s[j] = smem[wso + sbyte + step + half * 2048 + j * 256];
  };
  f32x4 acc00[4][2], acc10[4][2], acc11[4][2], acc01[4][2];
  auto mma = [&](f32x4 (&acc)[4][2], const mx_i32x8 (&xf)[4], const uint32_t (&sx)[4], const mx_u32x4 (&wf)[2], const uint32_t (&sw)[2]) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) acc[i][j] = mx_mfma(wf[j], xf[i], acc[i][j], sw[j], sx[i]);
  };
  mx_i32x8 xf0[4], xf1[4];
  mx_u32x4 wf0[2], wf1[2];
  uint32_t sx0[4], sx1[4], sw0[2], sw1[2];

#define MXB_PHASE(READS, STAGE, WAITN, ACC, XF, SX, WF, SW)                            \
  READS;                                                                               \
  STAGE;                                                                               \
  __builtin_amdgcn_sched_barrier(0);                                                   \
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(WAITN) : "memory");                         \
  __builtin_amdgcn_s_barrier();                                                        \
  __builtin_amdgcn_sched_barrier(0);                                                   \
  __builtin_amdgcn_s_setprio(1);                                                       \
  mma(ACC, XF, SX, WF, SW);                                                            \
  __builtin_amdgcn_s_setprio(0);                                                       \
  __builtin_amdgcn_sched_barrier(0);                                                   \
  __builtin_amdgcn_s_barrier();                                                        \
  __builtin_amdgcn_sched_barrier(0);

  int cm0, cend, ctn, cg;                    // the tile being computed (the staging tile runs ahead)
  decode(tile, cm0, cend, ctn, cg);
  cur = stage_of(tile);
  wrs = weights(cur.g);
  srs = scales(cur.g);
  int par = 0;                               // which set holds the scales of the current four steps
  stage_s(0, 0);
  stage_b(0, 0, 0); stage_a(0, 0, 0); stage_a(1, 0, 0); stage_b(1, 0, 0);
  stage_b(0, 1, 1); stage_a(1, 1, 1); stage_a(0, 1, 1);
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_waitcnt vmcnt(6)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
  if (wr == 1) __builtin_amdgcn_s_barrier();          // waves 4-7 run one barrier behind
  __builtin_amdgcn_sched_barrier(0);
  read_w(wf0, sw0, 0, 0, 0, 0);
  read_x(xf0, sx0, 0, 2, 0, 0, 0);

  for (;;) {
    const int next = used(tile + stride);
    const bool has_next = next < chunk_end;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        acc00[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        acc10[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        acc11[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        acc01[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
      }
    nxt = stage_of(has_next ? next : tile);
    // One body without a branch: the compiler would move a phase's products behind it, past their barriers.  In the last two steps
    // everything staged from the third phase on is the next output tile's.  Scales are loaded in every other step, so twice each; the
    // first time into a set that is free already.
    for (int t = 0; t < KT; t += 2) {
      const int s0 = min(t, KB - 1) & 3, s1 = min(t + 1, KB - 1) & 3;      // (the step of zeros takes its neighbour's scales)
      const bool last = t == KT - 2;
      const int now = par * MXB_SC;
      // the even step: A0 B0, A1 B0, A1 B1, A0 B1
      MXB_PHASE(read_x(xf0, sx0, 2, 4, 0, 0, now + 4 * s0); read_x(xf1, sx1, 0, 1, 0, 1, now + 4 * s0), stage_b(1, 1, t + 1), 7, acc00, xf0, sx0, wf0, sw0)
      cur.rows = last ? nxt.rows : cur.rows;
      cur.b0 = last ? nxt.b0 : cur.b0;
      cur.b1 = last ? nxt.b1 : cur.b1;
      cur.sc = last ? nxt.sc : cur.sc;
      if constexpr (grouped) {
        cur.g = last ? nxt.g : cur.g;
        wrs = weights(cur.g);
        srs = scales(cur.g);
      }
      MXB_PHASE(read_x(xf1, sx1, 1, 4, 0, 1, now + 4 * s0), stage_s(par ^ 1, last ? 0 : (t >> 2) + 1); stage_b(0, 0, t + 2), 7, acc10, xf1, sx1, wf0, sw0)
      MXB_PHASE(read_w(wf1, sw1, 0, 1, now, s0); read_w(wf0, sw0, 1, 0, now, s1), stage_a(0, 0, t + 2), 7, acc11, xf1, sx1, wf1, sw1)
      MXB_PHASE(read_x(xf1, sx1, 0, 2, 1, 1, now + 4 * s1), stage_a(1, 0, t + 2), 7, acc01, xf0, sx0, wf1, sw1)
      // the odd one: A1 B0, A0 B0, A0 B1, A1 B1
      MXB_PHASE(read_x(xf1, sx1, 2, 4, 1, 1, now + 4 * s1); read_x(xf0, sx0, 0, 1, 1, 0, now + 4 * s1), stage_b(1, 0, t + 2), 7, acc10, xf1, sx1, wf0, sw0)
      MXB_PHASE(read_x(xf0, sx0, 1, 4, 1, 0, now + 4 * s1), stage_b(0, 1, t + 3), 6, acc00, xf0, sx0, wf0, sw0)
      par ^= (int)(last || (t & 2));
      const int then = par * MXB_SC, s2 = last ? 0 : (t + 2) & 3;
      MXB_PHASE(read_w(wf1, sw1, 1, 1, now, s1); read_w(wf0, sw0, 0, 0, then, s2), stage_a(1, 1, t + 3), 6, acc01, xf0, sx0, wf1, sw1)
      MXB_PHASE(read_x(xf0, sx0, 0, 2, 0, 0, then + 4 * s2), stage_a(0, 1, t + 3), 6, acc11, xf1, sx1, wf1, sw1)
    }
    // nothing below may be computed before the K loop (it would be live across it)
    asm volatile("" : "+s"(cm0), "+s"(ctn), "+s"(cend), "+s"(cg));

    // ---- lane (r16, q) of fragment (i, j) holds columns 16 j + 4 q .. + 3 of row 16 i + r16 of its quadrant
    int eln = lane;
    asm volatile("" : "+v"(eln));
    const int er = eln & 15, eq = eln >> 4;
    // (MX_OUT: the second group of 32 columns is 128 on, MX_GLU: in the up half)
    const int n0 = EPI == MX_GLU ? 128 * ctn + 32 * wc : 256 * ctn + 32 * wc, n1 = n0 + (EPI == MX_GLU ? a.N >> 1 : 128);
    float b0[2][4], b1[2][4];
    mx_bias<T>(b0, a.bias, (long)cg * a.N, n0, a.N, eq);
    mx_bias<T>(b1, a.bias, (long)cg * a.N, n1, a.N, eq);
    [[maybe_unused]] const MxGlu glu(a.limit, a.alpha);
    auto put = [&](const f32x4 (&a0)[4][2], const f32x4 (&a1)[4][2], int mq) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int m = cm0 + 128 * mq + 64 * wr + 16 * i + er;
        if constexpr (EPI == MX_GLU) {
          float v[2][4];
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) v[j][e] = glu(a0[i][j][e] + b0[j][e], a1[i][j][e] + b1[j][e]);
          mx_store_block((uint8_t*)a.out + (long)m * a.ldo + n0, a.os + (long)m * a.ldos + (n0 >> 5), v, eln, m < cend);
        } else if constexpr (EPI == MX_SLAB) {
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              f32x4 v = h ? a1[i][j] : a0[i][j];
#pragma unroll
              for (int e = 0; e < 4; ++e) v[e] += h ? b1[j][e] : b0[j][e];
              const int n = (h ? n1 : n0) + 16 * j + 4 * eq;
              if (m < cend && n < a.N) *reinterpret_cast<f32x4*>(a.partial + (long)m * a.N + n) = v;
            }
        } else {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            mx_u32x2 pk[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const f32x4 v = h ? a1[i][j] : a0[i][j];
              typename Vec4<T>::type o;
#pragma unroll
              for (int e = 0; e < 4; ++e) o[e] = (T)(v[e] + (h ? b1[j][e] : b0[j][e]));
              pk[j] = __builtin_bit_cast(mx_u32x2, o);
            }
            // lanes of even q trade their second fragment's columns for the next lane's first: 16 bytes each, 64 neighbouring a row
            const auto p0 = __builtin_amdgcn_permlane16_swap(pk[0][0], pk[1][0], false, false);
            const auto p1 = __builtin_amdgcn_permlane16_swap(pk[0][1], pk[1][1], false, false);
            const int n = (h ? n1 : n0) + ((eq & 1) ? 16 + 4 * (eq - 1) : 4 * eq);
            if (m < cend && n < a.N)
              *reinterpret_cast<mx_u32x4*>((T*)a.out + (long)m * a.ldo + n) = mx_u32x4{(uint32_t)p0[0], (uint32_t)p1[0], (uint32_t)p0[1], (uint32_t)p1[1]};
          }
        }
      }
    };
    put(acc00, acc01, 0);
    put(acc10, acc11, 1);
    __builtin_amdgcn_sched_barrier(0);
    if (!has_next) break;
    tile = next;
    decode(tile, cm0, cend, ctn, cg);
  }
#undef MXB_PHASE
  if (wr == 0) __builtin_amdgcn_s_barrier();
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");    // the tail's loads must not outlive the LDS
#endif
}

int mx_num_cus() {
  int dev = 0, n = 0;
  if (hipGetDevice(&dev) != hipSuccess || hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n < 8) return 256;
  return n;
}

// (row_tiles == 16)
template <typename T, int EPI>
int mx_big(const MxArgs& a, hipStream_t st) {
  const long lim = (1L << 32) - 64;
  if ((long)a.x_rows * a.ldq >= lim || a.lds % 16 || ((a.N + 15L) / 16) * a.KB * 1024 >= lim) return -8;
  const int ntn = EPI == MX_GLU ? (a.N / 2 + 127) / 128 : (a.N + 255) / 256;
  const int ntm = a.tiles != nullptr ? a.num_tiles : (a.M + 255) / 256;
  const long per = a.tiles != nullptr ? ((long)ntm * ntn + 7) / 8 : (long)ntm * ((ntn + 7) / 8);
  if (per >= (1L << 27)) return -7;
  const int cus = mx_num_cus() / 8;
  const unsigned grid = 8 * (unsigned)(per < cus ? per : cus);
  if constexpr (EPI != MX_OUT)
    if (a.tiles != nullptr) mx_big_kernel<T, EPI, true><<<grid, 512, 0, st>>>(a, ntm, ntn);
  if constexpr (EPI != MX_SLAB)
    if (a.tiles == nullptr) mx_big_kernel<T, EPI, false><<<grid, 512, 0, st>>>(a, ntm, ntn);
  HIP_LAUNCH_CHECK();
  return 0;
}

// Between: rows enough that x is worth sharing, too few to fill the chip with 256-row tiles.  A workgroup has 16 MT WM rows and 4 NT column
// tiles, a wave NT of them and 16 MT of the rows; K in steps of 128, split over the grid.  x and the weights of S steps are in LDS or on
// their way to it, straight from memory: the loads of the step that is S - 1 ahead go out while one is multiplied, so
// (S - 1) (2 MT WM + 4 NT) KiB a workgroup are in flight, and the bytes of the weights are the time until the matrix cores are.
// WM 1: a step is one barrier; behind it every wave's loads of the step are there and every wave has read the step before.  (Reading the
// next step's fragments while this one's are multiplied takes a step off what is in flight, and was slower at every size: 8192 x 28672 by
// 100 rows 43 -> 53 us.)
// WM 2: 128 rows, two waves to a SIMD; those of the second half of the rows run half a step behind, so that the matrix cores multiply for
// the one while the other reads LDS: a step is two barriers, a wave reads in front of one and multiplies behind it.  Its loads go out
// between its products: the first half's of the step that is S - 1 ahead (the second half still reads this step), the second's of the
// one that is S ahead, into the buffer that both are done with.  256 rows of 28672 into 8192 in four parts: 75 us with both halves in step,
// 68 with the halves apart, 66 with the loads between the products; 1024 of 8192 into 8192 69, 64, 60 (of which 42 are the instructions').
// Scales come 16 bytes a row (four steps) at a time, with the first step of each four, into sets of their own.
// MX_GLU: NT 4, a wave's tiles are two of the gate and the same two of the up half - a block of 32 columns.
template <int MT, int NT, int WM> struct MxRing {
  static constexpr int X = WM * MT * 2048, STEP = X + NT * 4096;          // bytes of a step
  static constexpr int XR = WM * (MT < 4 ? 64 : 16 * MT), SCALES = XR * 16 + NT * 1024;      // rows whose scales are loaded, bytes of a set
  // the sets that S steps under way and the one that is read may touch: S neighbouring steps, for WM 2 one more
  static constexpr int sets(int steps) { return (steps + 1 + WM) / 4 + 1; }
  static constexpr int bytes(int steps) { return steps * STEP + sets(steps) * SCALES; }
  static constexpr int fit(int lds) { int n = 2; while (n < 8 && bytes(n + 1) <= lds) ++n; return n; }
};
template <typename T, int MT, int NT, int WM, int EPI, int S>
__global__ __launch_bounds__(256 * WM) void mx_ring_kernel(const MxArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
  using R = MxRing<MT, NT, WM>;
  constexpr int ROWS = 16 * MT * WM, WP = NT / WM, SCB = R::SCALES, SETS = R::sets(S);
  __shared__ __attribute__((aligned(1024))) unsigned char smem[R::bytes(S)];
  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wn = wid & 3, wm = wid >> 2;                       // this wave's columns, rows
  const int r = lane & 15, q = lane >> 4;
  const int KB = a.KB, SS = (KB + 3) >> 2, ntiles = (a.N + 15) >> 4, half = ntiles >> 1;
  int bx = blockIdx.x, by = blockIdx.y, bz = blockIdx.z;
  if (a.tiles == nullptr && ((gridDim.y * gridDim.z) & 7) == 0) {      // row tiles of the same weights on one of the eight dies, in turn
    const unsigned l = bx + gridDim.x * (by + gridDim.y * bz), u = l / (8 * gridDim.x) * 8 + (l & 7);
    bx = (l >> 3) % gridDim.x;
    by = u % gridDim.y;
    bz = u / gridDim.y;
  }
  int row0 = bx * ROWS, end = a.M, group = 0;
  if (a.tiles != nullptr) {
    const int* d = a.tiles + 3 * bx;
    const int rows = __builtin_amdgcn_readfirstlane(d[2]);
    if (rows <= 0) return;
    group = min(max(__builtin_amdgcn_readfirstlane(d[0]), 0), a.groups - 1);
    row0 = min(max(__builtin_amdgcn_readfirstlane(d[1]), 0), a.M - 1);
    end = min(a.M, row0 + min(rows, ROWS));
  }
  // this workgroup's steps
  const int lo = (int)((long)KB * bz / a.ksplit), hi = (int)((long)KB * (bz + 1) / a.ksplit);
  auto column_tile = [&](int j) {                              // behind tile j of the workgroup's 4 NT: NT of each wave
    if (EPI == MX_GLU) return 2 * (4 * by + j / NT) + (j & 1) + ((j % NT) >> 1) * half;
    return 4 * NT * by + j;
  };
  int ld0[WP];                                                 // those that this wave loads
#pragma unroll
  for (int t = 0; t < WP; ++t) ld0[t] = column_tile(wid * WP + t);

  // ---- staging.  Rows past the end, tiles past the last come as zeros from outside their descriptors
  const unsigned wbytes = (unsigned)((long)ntiles * KB * 1024), sbytes = (unsigned)((long)ntiles * SS * 256);
  const auto xr = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(a.xq), 0, (int)(unsigned)((long)a.x_rows * a.ldq), 0x00020000);
  const auto xsr = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(a.xs), 0, (int)(unsigned)((long)a.x_rows * a.lds), 0x00020000);
  const auto wrs = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(a.qw + (long)group * wbytes), 0, (int)wbytes, 0x00020000);
  const auto wsr = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(a.ws + (long)group * sbytes), 0, (int)sbytes, 0x00020000);
  const unsigned ldq = (unsigned)a.ldq;
  // x: MT / 2 pieces of eight rows a wave (MT 2: one); a row's 16-byte slots XOR-ed with (row >> 1) & 7
  constexpr int XP = MT / 2, XS = R::XR / (64 * WM);
  unsigned xoff[XP], soff[XS];
  auto row_of = [&](int m) {                                   // of x behind row m of this workgroup
    int row = min(row0 + m, end - 1);
    if (a.src != nullptr) row = min(max(a.src[row], 0), a.x_rows - 1);
    return (unsigned)row;
  };
#pragma unroll
  for (int i = 0; i < XP; ++i) {
    const int m = 8 * (XP * wid + i) + (lane >> 3);
    xoff[i] = row_of(m) * ldq + 16 * ((lane & 7) ^ ((m >> 1) & 7));
  }
  // scales of x: 64 lanes x 4 bytes, 16 rows of 16 bytes each; MT < 4: the last rows again
#pragma unroll
  for (int i = 0; i < XS; ++i) soff[i] = row_of(min(16 * (XS * wid + i) + (lane >> 2), ROWS - 1)) * (unsigned)a.lds + 4 * (lane & 3);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");             // (loads of src: nothing of them among the counted ones)
  constexpr int PER = XP + WP;                                 // loads of a wave and step, without scales
  int sbuf = 0, sset = 0;                                      // where the next step's and the next set's loads go
  auto stage = [&](int k, int p) {                             // load p of PER of step k; behind the last step: zeros, read by nobody
    unsigned char* const to = smem + sbuf * R::STEP;
    const unsigned off = __builtin_amdgcn_readfirstlane(k < hi ? 0u : 0xfffffff0u);
    const int at = __builtin_amdgcn_readfirstlane(min(k, hi - 1));
    if (p < XP)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(xr, (mx_lds_void*)(to + (XP * wid + p) * 1024), 16, xoff[p] | off, at * 128, 0, 0);
    else
      __builtin_amdgcn_raw_ptr_buffer_load_lds(wrs, (mx_lds_void*)(to + R::X + (wid * WP + p - XP) * 1024), 16,
                                               (16u * lane + (unsigned)ld0[p - XP] * (unsigned)(KB * 1024)) | off, at * 1024, 0, 0);
  };
  auto stage_scales = [&](int ss, int set) {
    unsigned char* const to = smem + S * R::STEP + set * SCB;
#pragma unroll
    for (int i = 0; i < XS; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(xsr, (mx_lds_void*)(to + (XS * wid + i) * 256), 4, soff[i], ss * 16, 0, 0);
#pragma unroll
    for (int t = 0; t < WP; ++t)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(wsr, (mx_lds_void*)(to + R::XR * 16 + (wid * WP + t) * 256), 4,
                                               4u * lane + (unsigned)ld0[t] * (unsigned)(SS * 256), ss * 256, 0, 0);
  };

  f32x4 acc[NT][MT];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[t][i] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int swz = (r >> 1) & 7, so0 = (q ^ swz) << 4, so1 = ((4 + q) ^ swz) << 4;
  // set of four steps ss: (ss - lo / 4) mod SETS; a step's buffer: (k - lo) mod S
  auto issue_scales = [&](int k) {
    if (k < hi && (k == lo || (k & 3) == 0)) {
      stage_scales(k >> 2, sset);
      sset = sset + 1 == SETS ? 0 : sset + 1;
    }
  };
  // Step k in n parts, this is part i.  (A unit takes a load in 16 cycles: those of all waves in a row, in front of their reads of LDS, hold
  // these up; between the products they do not.)
  auto issue = [&](int k, int i, int n) {
#pragma unroll
    for (int p = 0; p < PER; ++p)
      if (p * n / PER == i) stage(k, p);
    if (i == n - 1) sbuf = sbuf + 1 == S ? 0 : sbuf + 1;
  };
  const int ahead = S - 1 + wm;
  for (int k = lo; k < lo + ahead; ++k) {
    issue_scales(k);
    issue(k, 0, 1);
  }
  int buf = 0, set = 0;
  // at most the S - 2 steps behind the one that is read next are in flight (scales among them make the count stricter)
  auto arrived = []() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"((S - 2) * PER) : "memory"); };
  auto meet = []() {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
  };
  auto next = [&](int k) {
    buf = buf + 1 == S ? 0 : buf + 1;
    if ((k & 3) == 3) set = set + 1 == SETS ? 0 : set + 1;
  };
  mx_u32x4 w[NT];
  uint32_t sw[NT];
  auto read_weights = [&](int k) {
    const unsigned char* const at = smem + buf * R::STEP + R::X + wn * NT * 1024 + lane * 16;
    const unsigned char* const sc = smem + S * R::STEP + set * SCB + R::XR * 16 + wn * NT * 256 + lane * 4 + (k & 3);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      w[t] = *reinterpret_cast<const mx_u32x4*>(at + t * 1024);
      sw[t] = sc[t * 256];
    }
  };
  auto row = [&](int k, int i, mx_i32x8& x, uint32_t& sx) {
    const int m = 16 * (MT * wm + i) + r;
    const unsigned char* const at = smem + buf * R::STEP + m * 128;
    x = mx_fragment(at + so0, at + so1);
    sx = smem[S * R::STEP + set * SCB + m * 16 + 4 * (k & 3) + q];
  };
  mx_i32x8 x[MT];
  uint32_t sx[MT];
  if (wm == 1) {
    arrived();
    meet();
  }
  for (int k = lo; k < hi; ++k) {
    if (wm == 0) arrived();
    meet();
    issue_scales(k + ahead);
    read_weights(k);
#pragma unroll
    for (int i = 0; i < MT; ++i) row(k, i, x[i], sx[i]);
    next(k);
    if constexpr (WM == 2) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      arrived();
      meet();
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      issue(k + ahead, i, MT);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int t = 0; t < NT; ++t) acc[t][i] = mx_mfma(w[t], x[i], acc[t][i], sw[t], sx[i]);
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (WM == 2)
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int t = 0; t < NT; ++t) asm volatile("" : "+v"(acc[t][i]));    // (multiplied here, not behind the next barrier)
  }
  if (WM == 2 && wm == 0) meet();
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");             // (the zeros' loads must not outlive the LDS)

  // ---- lane (r, q): columns 4 q .. + 3 of tile t, row 16 i + r
  if constexpr (EPI == MX_GLU) {
    const int n0 = 32 * (4 * by + wn), n1 = n0 + (a.N >> 1);
    if (n0 >= a.N >> 1) return;
    float b0[2][4], b1[2][4];
    mx_bias<T>(b0, a.bias, (long)group * a.N, n0, a.N, q);
    mx_bias<T>(b1, a.bias, (long)group * a.N, n1, a.N, q);
    const MxGlu glu(a.limit, a.alpha);
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const int m = row0 + 16 * (MT * wm + i) + r;
      float v[2][4];
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) v[j][e] = glu(acc[j][i][e] + b0[j][e], acc[2 + j][i][e] + b1[j][e]);
      mx_store_block((uint8_t*)a.out + (long)m * a.ldo + n0, a.os + (long)m * a.ldos + (n0 >> 5), v, lane, m < end);
    }
  } else {
    const T* bias = a.bias == nullptr ? nullptr : (const T*)a.bias + (long)group * a.N;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int n = 16 * column_tile(wn * NT + t) + 4 * q;
      if (n >= a.N) continue;
      f32x4 b = f32x4{0.f, 0.f, 0.f, 0.f};
      if (bias != nullptr)
#pragma unroll
        for (int e = 0; e < 4; ++e) b[e] = (float)bias[n + e];
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const int m = row0 + 16 * (MT * wm + i) + r;
        if (m >= end) continue;
        if constexpr (EPI == MX_SLAB) {
          *reinterpret_cast<f32x4*>(a.partial + ((long)bz * a.M + m) * a.N + n) = acc[t][i] + b;
        } else {
          typename Vec4<T>::type o;
#pragma unroll
          for (int e = 0; e < 4; ++e) o[e] = (T)(acc[t][i][e] + b[e]);
          *reinterpret_cast<typename Vec4<T>::type*>((T*)a.out + (long)m * a.ldo + n) = o;
        }
      }
    }
  }
#endif
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

// rows of gated activations in 8 bits from the slabs of [gate | up]; a thread has 8 columns, a quad a block
template <typename T>
__global__ __launch_bounds__(256) void mx_reduce_glu_kernel(uint8_t* __restrict__ out, long ldo, uint8_t* __restrict__ os, long ldos,
                                                            const float* __restrict__ partial, const T* __restrict__ bias, int M, int N,
                                                            int ksplit, float limit, float alpha) {
  const long i = blockIdx.x * 256L + threadIdx.x;
  const int half = N >> 1, per_row = half >> 3;
  if (i >= (long)M * per_row) return;                          // (per_row is a multiple of 4: quads agree)
  const int m = (int)(i / per_row), c = (int)(i - (long)m * per_row) * 8;
  float g[8], u[8], v[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    g[e] = bias ? (float)bias[c + e] : 0.f;
    u[e] = bias ? (float)bias[half + c + e] : 0.f;
  }
  for (int k = 0; k < ksplit; ++k) {
    const float* const p = partial + ((long)k * M + m) * N + c;
    float a[8], b[8];
    mx_load8(p, a);
    mx_load8(p + half, b);
#pragma unroll
    for (int e = 0; e < 8; ++e) { g[e] += a[e]; u[e] += b[e]; }
  }
  const MxGlu glu(limit, alpha);
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = glu(g[e], u[e]);
  mx_store8(out + m * ldo + c, os + m * ldos + (c >> 5), v);
}

// out[t] = sum over j of w[t][j] y[at[t k + j]], the 32-bit rows of one token's experts in order, rounded once (the rows in 16 bits would
// add their own rounding to it: 2.4e-3 of a bf16 sum instead of 1.7e-3); slots of experts held elsewhere add nothing
template <typename T>
__global__ __launch_bounds__(256) void mx_combine_kernel(T* __restrict__ out, const float* __restrict__ y, const float* __restrict__ topw,
                                                         const int* __restrict__ topi, const int* __restrict__ at, int tokens, int k,
                                                         int H, int rows, int first, int local) {
  const int quads = H >> 2;
  const long i = blockIdx.x * 256L + threadIdx.x;
  if (i >= (long)tokens * quads) return;
  const int t = (int)(i / quads), c = (int)(i - (long)t * quads) * 4;
  f32x4 s = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int j = 0; j < k; ++j) {
    const int e = topi[t * k + j];
    if (e < first || e >= first + local) continue;
    const int row = min(max(at[t * k + j], 0), rows - 1);
    const float w = topw[t * k + j];
    const f32x4 v = *reinterpret_cast<const f32x4*>(y + (long)row * H + c);
#pragma unroll
    for (int e4 = 0; e4 < 4; ++e4) s[e4] += w * v[e4];
  }
  typename Vec4<T>::type o;
#pragma unroll
  for (int e = 0; e < 4; ++e) o[e] = (T)s[e];
  *reinterpret_cast<typename Vec4<T>::type*>(out + (long)t * H + c) = o;
}

// shapes of a launch of the streaming kernel: one row tile with 1 or 2 column tiles and 8 waves (MX_OUT) or 4 and 8 (not MX_SLAB), and with
// 4 column tiles and 4 waves 1, 2 or 4 row tiles
template <typename T, int EPI>
int mx_stream(const MxArgs& a, int mt, int nt, int waves, hipStream_t st) {
  const int ntiles = (a.N + 15) / 16;
  dim3 grid((ntiles + nt - 1) / nt, a.ksplit, a.tiles != nullptr ? a.num_tiles : (a.M + 16 * mt - 1) / (16 * mt));
  if (grid.y > 65535 || grid.z > 65535) return -7;
#define GO(M_, N_, W_, Q_, P_) mx_stream_kernel<T, M_, N_, W_, EPI, Q_, P_><<<grid, 64 * W_, lds, st>>>(a)
  size_t lds = 0;
  const bool quant = a.x16 != nullptr;
  if (quant) {
    lds = (size_t)a.M * (132 * ((a.KB + a.ksplit - 1) / a.ksplit) + 16);
    if (mt != 1 || a.M > 16 || lds > 49152 || a.tiles != nullptr) return -6;
  }
  if constexpr (EPI == MX_SLAB)
    if (quant || waves != 4) return -6;
  if (nt == 4 && waves == 4) {
    if constexpr (EPI != MX_SLAB)
      if (quant) {
        GO(1, 4, 4, true, 3);
        HIP_LAUNCH_CHECK();
        return 0;
      }
    if (mt == 1) GO(1, 4, 4, false, 3);
    else if (mt == 2) GO(2, 4, 4, false, 2);
    else if (mt == 4) GO(4, 4, 4, false, 2);
    else return -6;
  } else if constexpr (EPI == MX_GLU) {
    if (nt != 4 || waves != 8 || mt != 1) return -6;
    if (quant) GO(1, 4, 8, true, 3);
    else GO(1, 4, 8, false, 3);
  } else if constexpr (EPI == MX_OUT) {
    if (mt != 1 || waves != 8 || (nt != 1 && nt != 2)) return -6;
    if (nt == 1 && quant) GO(1, 1, 8, true, 6);
    else if (nt == 1) GO(1, 1, 8, false, 6);
    else if (quant) GO(1, 2, 8, true, 4);
    else GO(1, 2, 8, false, 4);
  } else {
    return -6;
  }
#undef GO
  HIP_LAUNCH_CHECK();
  return 0;
}

// row_tiles 2 or 4, n_tiles 2 (MX_GLU: 4); 8 and 4.  As many steps as fit half of a unit's LDS: two workgroups a unit hide each other's
// barriers (twice the steps in one workgroup's: 8192 x 28672 by 48 rows 31 -> 35 us, 6144 x 4096 by 411 25.3 -> 25.7); 128 rows: all of it
template <typename T, int EPI, int MT, int NT, int WM>
int mx_ring_go(const MxArgs& a, hipStream_t st) {
  constexpr int S = MxRing<MT, NT, WM>::fit(MT * NT * WM <= 16 ? 80 * 1024 : 158 * 1024), ROWS = 16 * MT * WM;
  const int ntiles = (a.N + 15) / 16, per = 4 * NT;
  dim3 grid(a.tiles != nullptr ? a.num_tiles : (a.M + ROWS - 1) / ROWS, (ntiles + per - 1) / per, a.ksplit);
  if (grid.y > 65535 || grid.z > 65535 || (long)grid.x * grid.y * grid.z >= (1L << 31)) return -7;
  mx_ring_kernel<T, MT, NT, WM, EPI, S><<<grid, 256 * WM, 0, st>>>(a);
  HIP_LAUNCH_CHECK();
  return 0;
}
template <typename T, int EPI>
int mx_ring(const MxArgs& a, int mt, int nt, hipStream_t st) {
  const long lim = (1L << 32) - 64;
  if (a.x16 != nullptr || (long)a.x_rows * a.ldq >= lim || a.lds % 16 || ((a.N + 15L) / 16) * a.KB * 1024 >= lim) return -8;
  constexpr int NT = EPI == MX_GLU ? 4 : 2;
  if (mt == 2 && nt == NT) return mx_ring_go<T, EPI, 2, NT, 1>(a, st);
  if (mt == 4 && nt == NT) return mx_ring_go<T, EPI, 4, NT, 1>(a, st);
  if (mt == 8 && nt == 4) return mx_ring_go<T, EPI, 4, 4, 2>(a, st);
  return -6;
}

template <typename T>
int mx_dispatch(const MxArgs& a, int epi, int mt, int nt, int waves, hipStream_t st) {
  if (mt == 16) {
    if (a.ksplit != 1 || a.src != nullptr || a.x16 != nullptr || (epi == MX_SLAB && a.tiles == nullptr)) return -1;
    return epi == MX_GLU ? mx_big<T, MX_GLU>(a, st) : epi == MX_OUT ? mx_big<T, MX_OUT>(a, st) : mx_big<T, MX_SLAB>(a, st);
  }
  const bool ring = waves == 1;
  MxArgs slabs = a;                                            // (a bias goes in once, where slabs are summed)
  if (a.ksplit > 1) slabs.bias = nullptr;
  if (epi == MX_GLU && a.ksplit > 1) {
    const int rc = ring ? mx_ring<T, MX_SLAB>(slabs, mt, nt, st) : mx_stream<T, MX_SLAB>(slabs, mt, nt, waves, st);
    if (rc != 0) return rc;
    const long n = (long)a.M * (a.N / 16);
    mx_reduce_glu_kernel<T><<<(unsigned)((n + 255) / 256), 256, 0, st>>>((uint8_t*)a.out, a.ldo, a.os, a.ldos, a.partial, (const T*)a.bias,
                                                                        a.M, a.N, a.ksplit, a.limit, a.alpha);
    HIP_LAUNCH_CHECK();
    return 0;
  }
  if (epi == MX_GLU) return ring ? mx_ring<T, MX_GLU>(a, mt, nt, st) : mx_stream<T, MX_GLU>(a, mt, nt, waves, st);
  if (epi == MX_SLAB || a.ksplit > 1) {
    const int rc = ring ? mx_ring<T, MX_SLAB>(slabs, mt, nt, st) : mx_stream<T, MX_SLAB>(slabs, mt, nt, waves, st);
    if (rc != 0 || epi == MX_SLAB) return rc;
    const long n = (long)a.M * (a.N / 4);
    mx_reduce_kernel<T><<<(unsigned)((n + 255) / 256), 256, 0, st>>>((T*)a.out, a.ldo, a.partial, (const T*)a.bias, a.M, a.N, a.ksplit);
    HIP_LAUNCH_CHECK();
    return 0;
  }
  return ring ? mx_ring<T, MX_OUT>(a, mt, nt, st) : mx_stream<T, MX_OUT>(a, mt, nt, waves, st);
}

}  // namespace

// xq [x_rows][128 KB] bytes (rows ldq apart, a multiple of 128), xs [x_rows][4 KB] scale bytes (rows lds apart, a multiple of 4); qw, ws as
// above for `groups` matrices of N rows (padded to 16), N % 8 == 0.
// Or xq null: x16, rows of K columns of the model type (ldx elements apart, a multiple of 8), K % 32 == 0, at most 128 KB, quantised
// inside: at most 16 rows, of which a workgroup's part fits 48 KiB; no tiles.
// epi 0: out [M][N] of the model type, rows ldo elements apart (ksplit > 1: through partial [ksplit][M][N]); 1: partial alone (a bias with
// ksplit 1 only);
// 2: N = [gate ; up], N % 256 == 0: out [M][N / 2] elements, os their scales (ksplit > 1: through partial); limit 0: SiLU.
// tiles [num_tiles][3] (matrix, first row, rows; ksplit 1, epi 1 or 2) or null; src [M] or null: the row of x behind each row.
// shape: 16-row tiles a workgroup takes (of `tiles` at most 16 times as many rows each) + 256 times its 16-column tiles + 65536 times its
// waves for the streaming kernel (mx_stream);  row tiles 2 or 4 + 256 times 2 (4 where epi is 2 and ksplit 1), or 8 + 256 times 4, + 65536:
// the ring of LDS;
// 16: the kernel of 256-row tiles (ksplit 1, src null).  The last two: x_rows ldq and a matrix's bytes below 2^32, lds a multiple of 16.
VDAMD_API int vdamd_mx_gemm(void* out, long ldo, void* os, long ldos, float* partial, const void* xq, long ldq, const void* xs, long lds,
                            int x_rows, const void* x16, long ldx, int K, const void* qw, const void* ws, const void* bias, int M, int N,
                            int KB, int ksplit, int epi, float limit, float alpha, const int* tiles, int num_tiles, int groups,
                            const int* src, int shape, int dtype, void* stream) {
  if (M <= 0 || (tiles != nullptr && num_tiles <= 0)) return 0;
  if (N <= 0 || N % 8 || KB <= 0 || groups <= 0 || ksplit < 1 || ksplit > KB) return -1;
  if (((uintptr_t)qw % 16) || ((uintptr_t)ws | (uintptr_t)bias) % 4) return -1;
  if (x16 != nullptr) {
    if (K <= 0 || K % 32 || K > 128L * KB || ldx % 8 || ldx < K || (uintptr_t)x16 % 16 || src != nullptr) return -1;
  } else if (x_rows <= 0 || (src == nullptr && x_rows < M) || ldq % 128 || ldq < 128L * KB || lds < 4L * KB || (uintptr_t)xq % 16) {
    return -1;
  }
  if (epi == MX_GLU && (N % 256 || (ksplit > 1 && partial == nullptr) || ldo % 16 || (uintptr_t)out % 16 || ldo < N / 2 || os == nullptr || ldos < N / 64)) return -1;
  if (epi == MX_OUT && (ldo % 8 || ldo < N || (uintptr_t)out % 16 || (ksplit > 1 && partial == nullptr))) return -1;
  if (epi == MX_SLAB && partial == nullptr) return -1;
  if (ksplit > 1 && (tiles != nullptr || (epi == MX_SLAB && bias != nullptr))) return -1;
  if (tiles != nullptr && epi == MX_OUT) return -1;
  if (epi < 0 || epi > 2) return -1;
  const MxArgs a = {(const uint8_t*)xq, ldq, (const uint8_t*)xs, lds, (const uint8_t*)qw, (const uint8_t*)ws, out, ldo, (uint8_t*)os, ldos,
                    partial, bias, M, N, KB, ksplit, limit, alpha, tiles, num_tiles, groups, src, x_rows, x16, ldx, K};
  hipStream_t st = (hipStream_t)stream;
  if (dtype == DT_BF16) return mx_dispatch<bf16_t>(a, epi, shape & 255, shape >> 8 & 255, shape >> 16, st);
  if (dtype == DT_F16) return mx_dispatch<f16_t>(a, epi, shape & 255, shape >> 8 & 255, shape >> 16, st);
  return -2;
}

// y [tokens k][H] 32-bit rows (H % 4 == 0), topw and topi [tokens][k], at [tokens k]: the row of each slot -> out [tokens][H], of the slots
// of experts first .. first + local - 1
VDAMD_API int vdamd_mx_combine(void* out, const float* y, const float* topw, const int* topi, const int* at, int tokens, int k, int H,
                               int first, int local, int dtype, void* stream) {
  if (tokens <= 0) return 0;
  if (k <= 0 || H <= 0 || H % 4 || (long)tokens * k >= (1L << 31) || (uintptr_t)y % 16 || (uintptr_t)out % 8) return -1;
  const unsigned blocks = (unsigned)(((long)tokens * (H / 4) + 255) / 256);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == DT_BF16)
    mx_combine_kernel<bf16_t><<<blocks, 256, 0, st>>>((bf16_t*)out, y, topw, topi, at, tokens, k, H, tokens * k, first, local);
  else if (dtype == DT_F16)
    mx_combine_kernel<f16_t><<<blocks, 256, 0, st>>>((f16_t*)out, y, topw, topi, at, tokens, k, H, tokens * k, first, local);
  else
    return -2;
  HIP_LAUNCH_CHECK();
  return 0;
}
