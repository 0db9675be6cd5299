// Newton-Schulz steps towards the orthogonal factor of matrices, and the step of
// the optimizer that goes along it (Muon).
//
//   X = U / |U|_F, along the shorter side m (U^T where there are more rows), then
//   P = X X^T,  Q = b P + c P P,  X <- a X + Q X      (a, b, c: TT_NS_*)
//
// which keeps the singular vectors and moves every singular value s to
// a s + b s^3 + c s^5: after five steps those from about 0.003 on lie within
// [0.68, 1.21].  P and P P are symmetric: half of their tiles are computed.
//
// The products take fp32 results from the fp16 matrix units, which are 16 times as
// fast as the fp32 ones: a value times 2^14 is h + l, two fp16 numbers (l what h
// leaves), 22 bits, and h h' + h l' + l h' has all of the product but l l', 2^-22
// of it.  That is what fp32 sums of these lengths leave too: against 64 bits both
// are off by 1e-6 to 9e-6 (what the steps make of the first rounding).  2^14
// keeps both in the type's range: s stays under 1.21, so the values of X, P and Q
// are within 1.21, 1.46 and 2.81 (46100 of 65504 times 2^14), and l is exact to
// 2^-38.
//
// X, X^T, P and Q are kept as images: rows of blocks of 32 values, a block the 32
// h and then the 32 l, 128 bytes, with zeros behind the last value.  Both operands
// of a product are read along rows: P = X X^T, P P = P P^T, Q X = Q (X^T)^T.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>
#include "tt_rt.h"

namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef f32x4 __attribute__((aligned(4))) f32x4_any;

inline hipStream_t stream() { return (hipStream_t)ttrt_stream(); }
inline int launched() { return hipGetLastError() == hipSuccess ? 0 : -3; }

#ifndef TT_NOBLOCK
#define TT_NOBLOCK 0
#endif
constexpr float UP = 16384.f, DOWN2 = 1.f / (16384.f * 16384.f);
constexpr int MOST = TT_SGD_MAX;   // matrices of different shapes in one run of launches
constexpr int ALIKE = 64;          // of one shape
constexpr int NORM_PARTS = 1024;   // sums of squares of a matrix

struct Matrix {
  const float *g;   // what is orthogonalised, or the gradient (rows x cols)
  float *v, *w;     // momenta and weights; v NULL: the result goes to w
  char *x, *t0, *t1;  // images of X (m rows), X^T (n rows; the steps write one from the other)
  char *p, *q;      // of P and Q
  double *norm;     // NORM_PARTS partial sums of squares
  float keep, rate; // w = keep w + rate X
  int m, n;         // shorter and longer side
  int turned;       // more rows than columns: X is U^T
  int parts;        // of the norm
};
struct Matrices {
  Matrix at[MOST];
  unsigned long first[MOST + 1];  // matrix i has the workgroups, or the units of work, [first[i], first[i + 1])
  int count;
  int alike;       // all are at[0]'s shape: matrix i lies behind it by i times
  long images;     // bytes of the workspace
};

__host__ __device__ inline long blocks_of(int k) { return (k + 31) / 32; }

// which matrix a workgroup or unit belongs to; b becomes its number among that one's
__device__ __forceinline__ Matrix matrix(const Matrices &a, int i) {
  if (!a.alike) return a.at[i];
  Matrix M = a.at[0];
  M.g += (long)i * M.m * M.n, M.w += (long)i * M.m * M.n;
  const long off = i * a.images;
  M.x += off, M.t0 += off, M.t1 += off, M.p += off, M.q += off;
  M.norm += off / (long)sizeof(double);
  return M;
}
template <class N>
__device__ __forceinline__ Matrix matrix_of(const Matrices &a, N &b) {
  int i = 0;
  if (a.alike) {
    i = (int)(b / (N)a.first[1]);
    b -= (N)i * (N)a.first[1];
  } else {
    while (i + 1 < a.count && b >= a.first[i + 1]) i++;
    b -= (N)a.first[i];
  }
  return matrix(a, i);
}

// x 2^14 in two parts
__device__ __forceinline__ void split(float y, _Float16 &h, _Float16 &l) {
  h = (_Float16)y;
  l = (_Float16)(y - (float)h);
}
__device__ __forceinline__ _Float16 *place(char *image, long blocks, long r, long c) {
  return (_Float16 *)(image + (r * blocks + (c >> 5)) * 128) + (c & 31);
}

// ---------------------------------------------------------------- small matrices
//
// A matrix whose image of X and of P or Q (which follow each other in one place) fit
// LDS has a workgroup, which takes it from the gradient to the weights in one
// launch.  A wave has blocks of 32 x 32 of each result, kept in registers until all
// have read what they replace.  X^T is X read by transposing loads.  The products
// are formed transposed: a lane then holds four neighbours of a row, and P and Q
// are symmetric.

constexpr int BLOCK_WAVES = 16, BLOCK_LDS = 160 * 1024 - 256;
constexpr int BLOCK_KEEP = 3;  // blocks of X a wave
// X, P and the partial sums of P (one or four blocks of it: eight or two waves each)
__host__ __device__ inline long block_bytes(int m, int n) {
  const long mb = blocks_of(m), nb = blocks_of(n);
  return 4096 * (mb * nb + mb * mb + (mb == 1 ? 7 : mb == 2 ? 4 : 0));
}
inline bool fits_block(int m, int n) {
  return block_bytes(m, n) <= BLOCK_LDS && blocks_of(m) * blocks_of(n) <= BLOCK_WAVES * BLOCK_KEEP;
}

// Chunk (16 bytes) c of a block's eight in row r lies at c ^ (r / 2 % 8), and odd
// rows begin in the other half of the banks: where a row has an even number of
// blocks, neighbouring ones change places there.  No two of the lanes that LDS
// serves at once meet a bank (128 x 128: 71 us with half of them in one).
__device__ __forceinline__ const char *chunk_of(const char *image, int blocks, int r, int block, int c) {
  block ^= r & ~blocks & 1;
  return image + (r * blocks + block) * 128 + ((c ^ (r >> 1 & 7)) << 4);
}
__device__ __forceinline__ half8 along(const char *image, int blocks, int r0, int block, int half, int part, int lane) {
  return *(const half8 *)chunk_of(image, blocks, r0 + (lane & 31), block, part * 4 + half * 2 + (lane >> 5));
}
// The transposing read: sixteen lanes read four values each of four rows and sixteen
// columns (lane l: row l / 4, columns 4 (l % 4) ..) and get the four rows of column l.
// Eight rows r0 + 8 (lane / 32) .. of column lane % 32 of a block.
__device__ __forceinline__ half8 across(const char *image, int blocks, int r0, int block, int part, int lane) {
  typedef short s16x4 __attribute__((ext_vector_type(4)));
  typedef short s16x8 __attribute__((ext_vector_type(8)));
  s16x8 v;
  const int l = lane & 15, c = (lane >> 4 & 1) * 16 + 4 * (l & 3);
#pragma unroll
  for (int x = 0; x < 2; x++) {
    const char *p = chunk_of(image, blocks, r0 + (lane >> 5) * 8 + x * 4 + l / 4, block, part * 4 + c / 8) + (c & 4) * 2;
    const s16x4 w = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)const_cast<char *>(p));
#pragma unroll
    for (int j = 0; j < 4; j++) v[x * 4 + j] = w[j];
  }
  return __builtin_bit_cast(half8, v);
}
__device__ __forceinline__ void three(f32x16 &acc, half8 ha, half8 la, half8 hb, half8 lb) {
  acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(la, hb, acc, 0, 0, 0);
  acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(ha, lb, acc, 0, 0, 0);
  acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(ha, hb, acc, 0, 0, 0);
}
// four values of row r from column c on, and back
__device__ __forceinline__ f32x4 get4(const char *image, int blocks, int r, int c) {
  typedef _Float16 half4 __attribute__((ext_vector_type(4)));
  const half4 h = *(const half4 *)(chunk_of(image, blocks, r, c >> 5, c >> 3 & 3) + (c & 4) * 2);
  const half4 l = *(const half4 *)(chunk_of(image, blocks, r, c >> 5, 4 + (c >> 3 & 3)) + (c & 4) * 2);
  f32x4 v;
#pragma unroll
  for (int j = 0; j < 4; j++) v[j] = ((float)h[j] + (float)l[j]) * (1.f / UP);
  return v;
}
__device__ __forceinline__ void put4(char *image, int blocks, int r, int c, f32x4 v) {
  typedef _Float16 half4 __attribute__((ext_vector_type(4)));
  half4 h, l;
#pragma unroll
  for (int j = 0; j < 4; j++) {
    _Float16 a, b;
    split(v[j] * UP, a, b);
    h[j] = a, l[j] = b;
  }
  *(half4 *)(chunk_of(image, blocks, r, c >> 5, c >> 3 & 3) + (c & 4) * 2) = h;
  *(half4 *)(chunk_of(image, blocks, r, c >> 5, 4 + (c >> 3 & 3)) + (c & 4) * 2) = l;
}

// v = mu v + g where there are momenta, and u = g + mu v (nesterov) or v; without g
template <class V>
__device__ __forceinline__ V momentum(const float *g, float *v, float mu, int nesterov, bool store) {
  V u = *(const V *)g;
  if (!v) return u;
  V w = *(const V *)v;
  if (store) {
    w = w * mu + u;
    *(V *)v = w;
  }
  return nesterov ? w * mu + u : w;
}

__global__ void __launch_bounds__(BLOCK_WAVES * 64) block_kernel(Matrices a, int steps, float mu, int nesterov) {
  __shared__ __attribute__((aligned(1024))) char lds[BLOCK_LDS];
  __shared__ double sums[BLOCK_WAVES];
  const Matrix M = matrix(a, blockIdx.x);
  int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int mb = (int)blocks_of(M.m), nb = (int)blocks_of(M.n), count = M.m * M.n, cols = M.turned ? M.m : M.n;
  char *const X = lds, *const P = lds + mb * nb * 4096, *const rest = P + mb * mb * 4096;
  constexpr int THREADS = BLOCK_WAVES * 64;
  for (int i = threadIdx.x * 16; i < mb * nb * 4096; i += THREADS * 16) *(f32x4 *)(X + i) = (f32x4){0.f, 0.f, 0.f, 0.f};
  double s = 0.0;
  for (int i = threadIdx.x * 4; i + 4 <= count; i += THREADS * 4) {
    const f32x4 u = momentum<f32x4_any>(M.g + i, M.v ? M.v + i : nullptr, mu, nesterov, true);
#pragma unroll
    for (int j = 0; j < 4; j++) s = fma((double)u[j], (double)u[j], s);
  }
  const int tail = count / 4 * 4 + threadIdx.x;  // up to three more
  if (tail < count) {
    const float u = momentum<float>(M.g + tail, M.v ? M.v + tail : nullptr, mu, nesterov, true);
    s = fma((double)u, (double)u, s);
  }
#pragma unroll
  for (int k = 1; k < 64; k <<= 1) s += __shfl_xor(s, k);
  if (lane == 0) sums[wave] = s;
  __syncthreads();
  s = 0.0;
#pragma unroll
  for (int k = 0; k < BLOCK_WAVES; k++) s += sums[k];
  const double scale = s == 0.0 ? 0.0 : (double)UP / sqrt(s);  // zeros stay zeros
  auto place1 = [&](int i, float u) {
    const int r = i / cols, c = i % cols, row = M.turned ? c : r, col = M.turned ? r : c;
    _Float16 h, l;
    split((float)((double)u * scale), h, l);
    *(_Float16 *)(chunk_of(X, nb, row, col >> 5, col >> 3 & 3) + (col & 7) * 2) = h;
    *(_Float16 *)(chunk_of(X, nb, row, col >> 5, 4 + (col >> 3 & 3)) + (col & 7) * 2) = l;
  };
  for (int i = threadIdx.x * 4; i + 4 <= count; i += THREADS * 4) {  // what this thread wrote itself
    const f32x4 u = momentum<f32x4_any>(M.g + i, M.v ? M.v + i : nullptr, mu, nesterov, false);
#pragma unroll
    for (int j = 0; j < 4; j++) place1(i + j, u[j]);
  }
  if (tail < count) place1(tail, momentum<float>(M.g + tail, M.v ? M.v + tail : nullptr, mu, nesterov, false));

  for (int step = 0;; step++) {
    __syncthreads();
    // the lane as the compiler does not know it from step to step: it would keep every
    // address of the loop in registers, and spill them
    asm volatile("" : "+v"(lane));
    const int low = lane & 31, high = (lane >> 5) * 4;  // result i: values high + 8 (i / 4) + i % 4 of row low
    // P = X X^T: with one block of it (four) eight waves (two) share the sum
    const int pb = mb * mb, ways = mb == 1 ? 8 : mb == 2 ? 2 : 1;
    {
      const int f = wave % pb, way = wave / pb;
      f32x16 acc = {};
      if (way < ways) {
#pragma unroll 1
        for (int k = way; k < nb; k += ways)
#pragma unroll
          for (int h = 0; h < 2; h++)
            three(acc, along(X, nb, f / mb * 32, k, h, 0, lane), along(X, nb, f / mb * 32, k, h, 1, lane),
                  along(X, nb, f % mb * 32, k, h, 0, lane), along(X, nb, f % mb * 32, k, h, 1, lane));
        if (way > 0) {
#pragma unroll
          for (int i = 0; i < 4; i++)
            *(f32x4 *)(rest + (((way - 1) * pb + f) * 4 + i) * 1024 + lane * 16) =
                (f32x4){acc[i * 4], acc[i * 4 + 1], acc[i * 4 + 2], acc[i * 4 + 3]};
        }
      }
      if (ways > 1) __syncthreads();
      if (way == 0) {
#pragma unroll 1
        for (int w = 1; w < ways; w++)
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const f32x4 v = *(const f32x4 *)(rest + (((w - 1) * pb + f) * 4 + i) * 1024 + lane * 16);
#pragma unroll
            for (int j = 0; j < 4; j++) acc[i * 4 + j] += v[j];
          }
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const f32x4 v = {acc[i * 4], acc[i * 4 + 1], acc[i * 4 + 2], acc[i * 4 + 3]};
          put4(P, mb, f % mb * 32 + low, f / mb * 32 + high + 8 * i, v * DOWN2);
        }
      }
    }
    __syncthreads();
    {  // Q = b P + c P P, in P's place
      const bool on = wave < pb;
      const int f = on ? wave : 0;
      f32x16 acc = {};
      f32x4 q[4];
      if (on) {
#pragma unroll 1
        for (int k = 0; k < mb; k++)
#pragma unroll
          for (int h = 0; h < 2; h++)
            three(acc, along(P, mb, f / mb * 32, k, h, 0, lane), along(P, mb, f / mb * 32, k, h, 1, lane),
                  along(P, mb, f % mb * 32, k, h, 0, lane), along(P, mb, f % mb * 32, k, h, 1, lane));
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const f32x4 v = {acc[i * 4], acc[i * 4 + 1], acc[i * 4 + 2], acc[i * 4 + 3]};
          q[i] = get4(P, mb, f % mb * 32 + low, f / mb * 32 + high + 8 * i) * TT_NS_B + v * (TT_NS_C * DOWN2);
        }
      }
      __syncthreads();
      if (on) {
#pragma unroll
        for (int i = 0; i < 4; i++) put4(P, mb, f % mb * 32 + low, f / mb * 32 + high + 8 * i, q[i]);
      }
    }
    __syncthreads();
    asm volatile("" : "+v"(lane));
    // X^T <- a X^T + X^T Q: block f has the columns f % nb of X and its rows f / nb
    f32x16 acc[BLOCK_KEEP] = {};
#pragma unroll
    for (int b = 0; b < BLOCK_KEEP; b++) {
      const int f = wave + b * BLOCK_WAVES, r0 = f / nb * 32, cb = f % nb;
      if (f >= mb * nb) continue;
#pragma unroll 1
      for (int k = 0; k < mb; k++)
#pragma unroll
        for (int h = 0; h < 2; h++)
          three(acc[b], across(X, nb, k * 32 + h * 16, cb, 0, lane), across(X, nb, k * 32 + h * 16, cb, 1, lane),
                along(P, mb, r0, k, h, 0, lane), along(P, mb, r0, k, h, 1, lane));
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const f32x4 v = get4(X, nb, r0 + low, cb * 32 + high + 8 * i) * TT_NS_A;
#pragma unroll
        for (int j = 0; j < 4; j++) acc[b][i * 4 + j] = v[j] + acc[b][i * 4 + j] * DOWN2;
      }
    }
    if (step + 1 == steps) {
#pragma unroll
      for (int b = 0; b < BLOCK_KEEP; b++) {
        const int f = wave + b * BLOCK_WAVES, row = f / nb * 32 + low;
        if (f >= mb * nb || row >= M.m) continue;
#pragma unroll
        for (int i = 0; i < 16; i++) {
          const int col = f % nb * 32 + high + 8 * (i / 4) + i % 4;
          if (col >= M.n) continue;
          float *w = M.w + (M.turned ? col * M.m + row : row * M.n + col);
          *w = M.v ? M.keep * *w + M.rate * acc[b][i] : acc[b][i];
        }
      }
      return;
    }
    __syncthreads();
#pragma unroll
    for (int b = 0; b < BLOCK_KEEP; b++) {
      const int f = wave + b * BLOCK_WAVES;
      if (f >= mb * nb) continue;
#pragma unroll
      for (int i = 0; i < 4; i++)
        put4(X, nb, f / nb * 32 + low, f % nb * 32 + high + 8 * i,
             (f32x4){acc[b][i * 4], acc[b][i * 4 + 1], acc[b][i * 4 + 2], acc[b][i * 4 + 3]});
    }
  }
}

// ---------------------------------------------------------------- before the steps

// v = mu v + g, and the sum of squares of u = g + mu v (nesterov) or v; without
// momenta of g.  In 64 bits: the squares of any fp32 values are within its range.
__global__ void __launch_bounds__(256) momentum_kernel(Matrices a, float mu, int nesterov) {
  __shared__ double sums[4];
  unsigned b = blockIdx.x;
  const Matrix M = matrix_of(a, b);
  const long count = (long)M.m * M.n;
  double s = 0.0;
  for (long i = ((long)b * 256 + threadIdx.x) * 4; i < count; i += (long)M.parts * 1024) {
    if (i + 4 <= count) {
      f32x4 u = *(const f32x4_any *)(M.g + i);
      if (M.v) {
        const f32x4 v = *(const f32x4_any *)(M.v + i) * mu + u;
        *(f32x4_any *)(M.v + i) = v;
        u = nesterov ? v * mu + u : v;
      }
#pragma unroll
      for (int j = 0; j < 4; j++) s = fma((double)u[j], (double)u[j], s);
    } else {
      for (long j = i; j < count; j++) {
        float u = M.g[j];
        if (M.v) {
          const float v = M.v[j] * mu + u;
          M.v[j] = v;
          u = nesterov ? v * mu + u : v;
        }
        s = fma((double)u, (double)u, s);
      }
    }
  }
#pragma unroll
  for (int k = 1; k < 64; k <<= 1) s += __shfl_xor(s, k);
  if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) M.norm[b] = (sums[0] + sums[1]) + (sums[2] + sums[3]);
}

// The images of U / |U|_F and its transpose, a tile of 64 x 64 at a time through
// LDS; both are written along their rows.
__global__ void __launch_bounds__(256) image_kernel(Matrices a, float mu, int nesterov) {
  __shared__ double sums[4];
  __shared__ float tile[64][65];
  unsigned b = blockIdx.x;
  const Matrix M = matrix_of(a, b);
  const int rows = M.turned ? M.n : M.m, cols = M.turned ? M.m : M.n;
  double s = 0.0;
  for (int i = threadIdx.x; i < M.parts; i += 256) s += M.norm[i];
#pragma unroll
  for (int k = 1; k < 64; k <<= 1) s += __shfl_xor(s, k);
  if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = s;
  __syncthreads();
  s = (sums[0] + sums[1]) + (sums[2] + sums[3]);
  const double scale = s == 0.0 ? 0.0 : (double)UP / sqrt(s);  // zeros stay zeros
  const unsigned across = (unsigned)((cols + 63) / 64);
  const long r0 = (long)(b / across) * 64, c0 = (long)(b % across) * 64;
#pragma unroll 4
  for (int k = 0; k < 16; k++) {
    const long r = r0 + k * 4 + (threadIdx.x >> 6), c = c0 + (threadIdx.x & 63);
    float u = 0.f;
    if (r < rows && c < cols) {
      u = M.g[r * cols + c];
      if (M.v) {
        const float v = M.v[r * cols + c];
        u = nesterov ? v * mu + u : v;
      }
    }
    tile[k * 4 + (threadIdx.x >> 6)][threadIdx.x & 63] = (float)((double)u * scale);
  }
  __syncthreads();
  char *along = M.turned ? M.t0 : M.x, *down = M.turned ? M.x : M.t0;
  const long row_blocks = blocks_of(cols), col_blocks = blocks_of(rows);
#pragma unroll 4
  for (int k = 0; k < 16; k++) {
    const int i = k * 4 + (threadIdx.x >> 6), j = threadIdx.x & 63;
    _Float16 h, l;
    if (r0 + i < rows && c0 + j < row_blocks * 32) {
      split(tile[i][j], h, l);
      _Float16 *p = place(along, row_blocks, r0 + i, c0 + j);
      p[0] = h;
      p[32] = l;
    }
    if (c0 + i < cols && r0 + j < col_blocks * 32) {
      split(tile[j][i], h, l);
      _Float16 *p = place(down, col_blocks, c0 + i, r0 + j);
      p[0] = h;
      p[32] = l;
    }
  }
}

// ---------------------------------------------------------------- products

enum { GRAM, SQUARE, STEP, LAST };  // P = X X^T; Q = b P + c P P; X <- a X + Q X; the same, to w

// Tile `b` of a symmetric matrix: those of the lower triangle row by row.
__device__ __forceinline__ void triangle(unsigned b, int &i, int &j) {
  int r = (int)((sqrt(8.0 * b + 1.0) - 1.0) * 0.5);
  while ((unsigned)r * (r + 1u) / 2 > b) r--;
  while ((unsigned)(r + 1) * (r + 2u) / 2 <= b) r++;
  i = r;
  j = (int)(b - (unsigned)r * (r + 1u) / 2);
}

template <int KIND>
struct Operands {
  const char *a, *b;    // images whose rows are multiplied
  const char *add;      // image of the matrix added, times `times` (GRAM: none)
  char *out, *down;     // images of the result and its transpose
  int rows, cols, k;    // of the result; the products' length
  float by, times;
  __device__ __forceinline__ Operands(const Matrix &M, int step) {
    if (KIND == GRAM) {
      a = b = M.x, add = nullptr, out = down = M.p;
      rows = cols = M.m, k = M.n, by = 1.f, times = 0.f;
    } else if (KIND == SQUARE) {
      a = b = add = M.p, out = down = M.q;
      rows = cols = k = M.m, by = TT_NS_C, times = TT_NS_B;
    } else {
      a = M.q, b = step & 1 ? M.t1 : M.t0, add = M.x, out = M.x, down = step & 1 ? M.t0 : M.t1;
      rows = k = M.m, cols = M.n, by = 1.f, times = TT_NS_A;
    }
  }
};

// Tiles of 32 x 32, one a workgroup, the operands read from memory as the matrix
// instructions take them and each wave with a share of the products' length:
// eight sums, joined in LDS.
template <int KIND>
__global__ void __launch_bounds__(512) small_kernel(Matrices a, int step) {
  constexpr int WAVES = 8;
  __shared__ float sums[WAVES][32][33];
  unsigned t = blockIdx.x;
  const Matrix M = matrix_of(a, t);
  const Operands<KIND> o(M, step);
  int ti, tj;
  if (KIND <= SQUARE) {
    triangle(t, ti, tj);
  } else {
    const unsigned across = (unsigned)blocks_of(o.cols);
    ti = (int)(t / across), tj = (int)(t % across);
  }
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const long blocks = blocks_of(o.k);
  // a row behind the last is the last once more: its results are not written
  const int ra = ti * 32 + (lane & 31), rb = tj * 32 + (lane & 31);
  const char *pa = o.a + (ra < o.rows ? ra : o.rows - 1) * blocks * 128 + (lane >> 5) * 16;
  const char *pb = o.b + (rb < o.cols ? rb : o.cols - 1) * blocks * 128 + (lane >> 5) * 16;
  f32x16 acc = {};
#pragma unroll 2
  for (long k = wave; k < blocks; k += WAVES) {
    half8 ha[2], la[2], hb[2], lb[2];
#pragma unroll
    for (int s = 0; s < 2; s++) {
      ha[s] = *(const half8 *)(pa + k * 128 + s * 32);
      la[s] = *(const half8 *)(pa + k * 128 + s * 32 + 64);
      hb[s] = *(const half8 *)(pb + k * 128 + s * 32);
      lb[s] = *(const half8 *)(pb + k * 128 + s * 32 + 64);
    }
#pragma unroll
    for (int s = 0; s < 2; s++) {
      acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(la[s], hb[s], acc, 0, 0, 0);
      acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(ha[s], lb[s], acc, 0, 0, 0);
      acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(ha[s], hb[s], acc, 0, 0, 0);
    }
  }
#pragma unroll
  for (int i = 0; i < 16; i++) sums[wave][8 * (i / 4) + 4 * (lane >> 5) + i % 4][lane & 31] = acc[i];
  __syncthreads();
  const int r = threadIdx.x >> 5, c = threadIdx.x & 31;  // and row r + 16
  float v[2];
#pragma unroll
  for (int e = 0; e < 2; e++) {
    const int i = r + e * 16, row = ti * 32 + i, col = tj * 32 + c;
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; w++) s += sums[w][i][c];
    s *= o.by * DOWN2;
    if (KIND != GRAM && row < o.rows && col < o.cols) {
      const _Float16 *p = place((char *)o.add, blocks_of(o.cols), row, col);
      s += o.times * (1.f / UP) * ((float)p[0] + (float)p[32]);
    }
    v[e] = s;
  }
  __syncthreads();
#pragma unroll
  for (int e = 0; e < 2; e++) {
    const int i = r + e * 16, row = ti * 32 + i, col = tj * 32 + c;
    const bool in = row < o.rows && col < o.cols;
    if (KIND == LAST) {
      if (in && !M.turned) {
        float *w = M.w + (long)row * o.cols + col;
        *w = M.v ? M.keep * *w + M.rate * v[e] : v[e];
      }
    } else if (row < o.rows) {
      _Float16 h, l;
      split(in ? v[e] * UP : 0.f, h, l);
      _Float16 *p = place(o.out, blocks_of(o.cols), row, col);
      p[0] = h;
      p[32] = l;
    }
    sums[0][i][c] = in ? v[e] : 0.f;
  }
  if ((KIND <= SQUARE && ti == tj) || (KIND == LAST && !M.turned)) return;
  __syncthreads();
#pragma unroll
  for (int e = 0; e < 2; e++) {  // the transpose
    const int i = r + e * 16, row = ti * 32 + c, col = tj * 32 + i;
    if (col >= o.cols) continue;
    if (KIND == LAST) {
      if (row < o.rows) {
        float *w = M.w + (long)col * o.rows + row;
        *w = M.v ? M.keep * *w + M.rate * sums[0][c][i] : sums[0][c][i];
      }
    } else {
      _Float16 h, l;
      split(sums[0][c][i] * UP, h, l);
      _Float16 *p = place(o.down, blocks_of(o.rows), col, row);
      p[0] = h;
      p[32] = l;
    }
  }
}

// ---------------------------------------------------------------- large products
//
// Tiles of 128 x 128, four waves with a quarter each, the operands through LDS in
// two buffers of a block (32 of the products' length): while one is multiplied the
// next is on its way by direct loads.  Per block and wave 24 matrix instructions
// stand against 16 KB read from LDS, and two workgroups a CU fill each other's
// waits.  The tiles' blocks are dealt evenly to the workgroups, whatever the
// matrices' shapes: a workgroup has whole tiles and at most two pieces of tiles
// that others have the rest of.  Pieces go to memory, and join_kernel adds them.

#ifndef TT_LARGE
#define TT_LARGE 8e8
#endif
#ifndef TT_HUGE
#define TT_HUGE 1.7e10
#endif
// Tiles of T x T: four waves of 64 x 64 or eight of 128 x 64 values, each FI x 2
// blocks of 32 x 32.
template <int T>
struct Shape {
  static constexpr int WAVES = T == 256 ? 8 : 4, ACROSS = WAVES / 2, FI = T / 64, BLOCKS = 2 * FI;
  static constexpr int GROUPS = T == 256 ? 256 : 512;  // workgroups at most: one or two a CU
  static constexpr int PIECE = T * T;                  // floats
  static constexpr int BUFFER = 2 * T * 128;           // bytes of both operands' block
};

__device__ __forceinline__ unsigned lds_address(const void *p) {
  return (unsigned)(uintptr_t)(__attribute__((address_space(3))) const char *)p;
}
// lane l's 16 bytes at base + off to LDS at lds + 16 l
__device__ __forceinline__ void dma16(const char *base, unsigned off, unsigned lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
               :
               : "s"(lds), "v"(off), "s"(base)
               : "memory", "m0");
}
__device__ __forceinline__ const char *scalar(const char *p) {
  const uint64_t x = (uint64_t)p;
  return (const char *)((uint64_t)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32 |
                        (uint32_t)__builtin_amdgcn_readfirstlane((int)x));
}

// Tiles in bands of eight rows, column by column, so that the workgroups of an XCD
// (consecutive ones) share rows and columns.
constexpr int BAND = 8;
template <int KIND, int T>
__device__ __forceinline__ void tile_of(unsigned long tile, int rows, int cols, int &ti, int &tj) {
  const int nr = (rows + T - 1) / T, nc = (cols + T - 1) / T;
  if (KIND <= SQUARE) {
    // below band b: 32 b^2 + 4 b tiles of the lower triangle
    int b = (int)((sqrt(128.0 * (double)tile + 16.0) - 4.0) / 64.0);
    while (b > 0 && 32ul * b * b + 4ul * b > tile) b--;
    while (32ul * (b + 1) * (b + 1) + 4ul * (b + 1) <= tile) b++;
    const unsigned in = (unsigned)(tile - (32ul * b * b + 4ul * b));
    const unsigned h = nr - b * BAND < BAND ? nr - b * BAND : BAND;
    if (in < (unsigned)b * BAND * h) {
      ti = b * BAND + (int)(in % h), tj = (int)(in / h);
    } else {
      triangle(in - (unsigned)b * BAND * h, ti, tj);
      ti += b * BAND, tj += b * BAND;
    }
  } else {
    const unsigned long band = (unsigned long)BAND * nc;
    const int b = (int)(tile / band);
    const unsigned in = (unsigned)(tile % band), h = nr - b * BAND < BAND ? nr - b * BAND : BAND;
    ti = b * BAND + (int)(in % h), tj = (int)(in / h);
  }
}

// A wave's 32 x 32 values, `acc` as the matrix instructions leave them, to where
// they go: through LDS, so that a lane has 16 of a row (and, for the transpose, of a
// column) and lines are written whole.
template <int KIND>
__device__ __forceinline__ void write32(const Matrix &M, const Operands<KIND> &o, const f32x16 &acc, long r0, long c0,
                                        float (*buf)[33], int lane, bool transpose) {
#pragma unroll
  for (int i = 0; i < 16; i++) buf[8 * (i / 4) + 4 * (lane >> 5) + i % 4][lane & 31] = acc[i];
  __builtin_amdgcn_wave_barrier();
  const int line = lane >> 1, from = (lane & 1) * 16;
  float v[16];
#pragma unroll
  for (int j = 0; j < 16; j++) v[j] = buf[line][from + j] * (o.by * DOWN2);
  const long row = r0 + line, col = c0 + from, blocks = blocks_of(o.cols);
  if (KIND != GRAM && row < o.rows && c0 < o.cols) {
    const half8 *p = (const half8 *)place((char *)o.add, blocks, row, col);
    const half8 h[2] = {p[0], p[1]}, l[2] = {p[4], p[5]};
#pragma unroll
    for (int j = 0; j < 16; j++) v[j] += o.times * (1.f / UP) * ((float)h[j / 8][j % 8] + (float)l[j / 8][j % 8]);
  }
#pragma unroll
  for (int j = 0; j < 16; j++)
    if (row >= o.rows || col + j >= o.cols) v[j] = 0.f;
  if (transpose) {
#pragma unroll
    for (int j = 0; j < 16; j++) buf[line][from + j] = v[j];
  }
  if (KIND == LAST) {
    if (!transpose && row < o.rows) {
      float *w = M.w + row * o.cols + col;
      if (col + 16 <= o.cols) {
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
          f32x4 u = {v[j], v[j + 1], v[j + 2], v[j + 3]};
          if (M.v) u = *(const f32x4_any *)(w + j) * M.keep + u * M.rate;
          *(f32x4_any *)(w + j) = u;
        }
      } else {
#pragma unroll
        for (int j = 0; j < 16; j++)
          if (col + j < o.cols) w[j] = M.v ? M.keep * w[j] + M.rate * v[j] : v[j];
      }
    }
  } else if (row < o.rows && c0 < o.cols) {
    half8 h[2], l[2];
#pragma unroll
    for (int j = 0; j < 16; j++) {
      _Float16 a, b;
      split(v[j] * UP, a, b);
      h[j / 8][j % 8] = a;
      l[j / 8][j % 8] = b;
    }
    half8 *p = (half8 *)place(o.out, blocks, row, col);
    p[0] = h[0], p[1] = h[1], p[4] = l[0], p[5] = l[1];
  }
  if (!transpose) return;
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int j = 0; j < 16; j++) v[j] = buf[from + j][line];
  const long trow = c0 + line, tcol = r0 + from;
  if (trow >= o.cols) return;
  if (KIND == LAST) {
    float *w = M.w + trow * o.rows + tcol;
    if (tcol + 16 <= o.rows) {
#pragma unroll
      for (int j = 0; j < 16; j += 4) {
        f32x4 u = {v[j], v[j + 1], v[j + 2], v[j + 3]};
        if (M.v) u = *(const f32x4_any *)(w + j) * M.keep + u * M.rate;
        *(f32x4_any *)(w + j) = u;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 16; j++)
        if (tcol + j < o.rows) w[j] = M.v ? M.keep * w[j] + M.rate * v[j] : v[j];
    }
  } else if (r0 < o.rows) {
    half8 h[2], l[2];
#pragma unroll
    for (int j = 0; j < 16; j++) {
      _Float16 a, b;
      split(v[j] * UP, a, b);
      h[j / 8][j % 8] = a;
      l[j / 8][j % 8] = b;
    }
    half8 *p = (half8 *)place(o.down, blocks_of(o.rows), trow, tcol);
    p[0] = h[0], p[1] = h[1], p[4] = l[0], p[5] = l[1];
  }
}

// where the 32 x 32 block f of a wave's lies
template <int T>
__device__ __forceinline__ long row_of(int ti, int wave, int f) {
  return (long)ti * T + (wave / Shape<T>::ACROSS) * (T / 2) + f / 2 * 32;
}
template <int T>
__device__ __forceinline__ long col_of(int tj, int wave, int f) {
  return (long)tj * T + (wave % Shape<T>::ACROSS) * 64 + f % 2 * 32;
}
template <int KIND>
__device__ __forceinline__ bool transposed(const Matrix &M, int ti, int tj) {
  return KIND <= SQUARE ? ti != tj : KIND == STEP || M.turned;
}

// How the units (tiles' blocks, tile by tile) are dealt: `rounds` whole tiles to every
// workgroup, then the units from `base` on evenly to the first `sharers`.
struct Deal {
  unsigned rounds, sharers;
  unsigned long base, units;
  // the first of workgroup w's share
  __device__ __forceinline__ unsigned long begins(unsigned w) const {
    return base + (w < sharers ? units * w / sharers : units);
  }
};

template <int KIND, int T>
__global__ void __launch_bounds__(Shape<T>::WAVES * 64, 2) tile_kernel(Matrices a, int step, Deal deal, float *pieces) {
  typedef Shape<T> S;
  __shared__ __attribute__((aligned(1024))) char lds[2 * S::BUFFER];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // consecutive workgroups go to the eight XCDs in turn: give each XCD a run of them
  const unsigned groups = gridDim.x, each = groups / 8, b = blockIdx.x;
  const unsigned w = b < each * 8 ? (b % 8) * each + b / 8 : b;
  const unsigned to = lds_address(lds);
  unsigned round = 0;
  for (unsigned long u = 0, end = 0;;) {
    if (u == end) {
      if (round < deal.rounds) {  // then all tiles have the same number of blocks
        const Operands<KIND> o(a.at[0], step);
        u = ((unsigned long)round * groups + w) * blocks_of(o.k);
        end = u + blocks_of(o.k);
      } else if (round == deal.rounds) {
        u = deal.begins(w), end = deal.begins(w + 1);
        if (u == end) return;
      } else {
        return;
      }
      round++;
    }
    unsigned long in = u;
    const Matrix M = matrix_of(a, in);
    const Operands<KIND> o(M, step);
    const long blocks = blocks_of(o.k);
    int ti, tj;
    tile_of<KIND, T>(in / blocks, o.rows, o.cols, ti, tj);
    const int k0 = (int)(in % blocks), k1 = (int)(end - u < (unsigned long)(blocks - k0) ? k0 + (end - u) : blocks);
    // lane l brings 16 bytes of row r = 8 i + l / 8; where it puts them, l % 8 of the
    // row's eight places, is where its (l % 8) ^ (r / 2 % 8) belong: the 16 lanes that
    // the reads below serve at once then have a bank each.  A row behind the last is
    // the last once more: its results are not written.
    constexpr int EACH = T / 8 / S::WAVES;
    unsigned off[2][EACH];
#pragma unroll
    for (int i = 0; i < EACH; i++) {
      const int r = (wave * EACH + i) * 8 + (lane >> 3), chunk = ((lane & 7) ^ (r >> 1 & 7)) * 16;
      const int ra = ti * T + r < o.rows ? r : o.rows - 1 - ti * T, rb = tj * T + r < o.cols ? r : o.cols - 1 - tj * T;
      off[0][i] = (unsigned)(ra * blocks * 128) + chunk;
      off[1][i] = (unsigned)(rb * blocks * 128) + chunk;
    }
    const char *pa = scalar(o.a + ((long)ti * T * blocks + k0) * 128);
    const char *pb = scalar(o.b + ((long)tj * T * blocks + k0) * 128);
    auto bring = [&](int k, unsigned at) {
#pragma unroll
      for (int i = 0; i < EACH; i++) dma16(pa + (long)k * 128, off[0][i], at + (wave * EACH + i) * 1024);
#pragma unroll
      for (int i = 0; i < EACH; i++) dma16(pb + (long)k * 128, off[1][i], at + T * 128 + (wave * EACH + i) * 1024);
    };
    f32x16 acc[S::FI][2] = {};
    __syncthreads();  // the last tile's LDS is read
    bring(0, to);
    const int n = k1 - k0, row = lane & 31, half = lane >> 5;
    // the wave's rows of either operand in a buffer
    const char *mine[2] = {lds + ((wave / S::ACROSS) * (T / 2) + row) * 128,
                           lds + (T + (wave % S::ACROSS) * 64 + row) * 128};
    for (int k = 0; k < n; k++) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
      const int now = (k & 1) * S::BUFFER;
      if (k + 1 < n) bring(k + 1, to + (S::BUFFER - now));
#pragma unroll
      for (int s = 0; s < 2; s++) {
        const int ph = now + (((s * 2 + half) ^ (row >> 1 & 7)) * 16),
                  pl = now + (((s * 2 + half + 4) ^ (row >> 1 & 7)) * 16);
        half8 ha[S::FI], la[S::FI], hb[2], lb[2];
#pragma unroll
        for (int j = 0; j < 2; j++) {
          hb[j] = *(const half8 *)(mine[1] + ph + j * 4096);
          lb[j] = *(const half8 *)(mine[1] + pl + j * 4096);
        }
#pragma unroll
        for (int i = 0; i < S::FI; i++) {
          ha[i] = *(const half8 *)(mine[0] + ph + i * 4096);
          la[i] = *(const half8 *)(mine[0] + pl + i * 4096);
        }
#pragma unroll
        for (int i = 0; i < S::FI; i++)
#pragma unroll
          for (int j = 0; j < 2; j++)
            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(la[i], hb[j], acc[i][j], 0, 0, 0);
#pragma unroll
        for (int i = 0; i < S::FI; i++)
#pragma unroll
          for (int j = 0; j < 2; j++)
            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ha[i], lb[j], acc[i][j], 0, 0, 0);
#pragma unroll
        for (int i = 0; i < S::FI; i++)
#pragma unroll
          for (int j = 0; j < 2; j++)
            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ha[i], hb[j], acc[i][j], 0, 0, 0);
      }
    }
    if (n == blocks) {
      __syncthreads();  // the operands are read
      const bool transpose = transposed<KIND>(M, ti, tj);
#pragma unroll
      for (int f = 0; f < S::BLOCKS; f++) {
        write32<KIND>(M, o, acc[f / 2][f % 2], row_of<T>(ti, wave, f), col_of<T>(tj, wave, f),
                      (float(*)[33])(lds + wave * 8192), lane, transpose);
        __builtin_amdgcn_wave_barrier();
      }
    } else {
      f32x4 *p = (f32x4 *)(pieces + (2l * w + (k0 == 0)) * S::PIECE) + wave * S::BLOCKS * 256 + lane;
#pragma unroll
      for (int i = 0; i < S::BLOCKS * 4; i++) {
        f32x4 v;
#pragma unroll
        for (int j = 0; j < 4; j++) v[j] = acc[i / 8][i / 4 % 2][i % 4 * 4 + j];
        p[i * 64] = v;
      }
    }
    u += n;
  }
}

// Workgroups (w - 1, .) add the pieces of the tile in which the share of
// tile_kernel's workgroup w begins, where that is the first to begin inside it; a
// wave has 32 x 32 of its values.
template <int KIND, int T>
__global__ void __launch_bounds__(256) join_kernel(Matrices a, int step, Deal deal, const float *pieces) {
  typedef Shape<T> S;
  __shared__ float buf[4][32][33];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned w = blockIdx.x + 1;
  const unsigned long u = deal.begins(w);
  unsigned long in = u;
  const Matrix M = matrix_of(a, in);
  const Operands<KIND> o(M, step);
  const unsigned long blocks = blocks_of(o.k), k0 = in % blocks, first = u - k0, last = first + blocks;
  if (k0 == 0 || deal.begins(w - 1) > first) return;
  int ti, tj;
  tile_of<KIND, T>(in / blocks, o.rows, o.cols, ti, tj);
  const int block = blockIdx.y * 4 + wave;
  unsigned stop = w;  // the first workgroup behind the tile
  while (stop < deal.sharers && deal.begins(stop) < last) stop++;
  f32x16 acc = {};
  const f32x4 *p = (const f32x4 *)pieces + block * 256 + lane;
#pragma unroll 4
  for (unsigned g = w - 1; g < stop; g++) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const f32x4 v = p[(2l * g + (g < w)) * (S::PIECE / 4) + i * 64];
#pragma unroll
      for (int j = 0; j < 4; j++) acc[i * 4 + j] += v[j];
    }
  }
  write32<KIND>(M, o, acc, row_of<T>(ti, block / S::BLOCKS, block % S::BLOCKS),
                col_of<T>(tj, block / S::BLOCKS, block % S::BLOCKS), buf[wave], lane, transposed<KIND>(M, ti, tj));
}

// ---------------------------------------------------------------- host

size_t up(size_t bytes) { return (bytes + 255) & ~(size_t)255; }

bool good_sides(long rows, long cols) {
  return rows > 0 && cols > 0 && rows <= TT_MUON_MAX_SIDE && cols <= TT_MUON_MAX_SIDE && rows * cols <= TT_MUON_MAX_VALUES;
}

size_t images_of(long rows, long cols) {
  const long m = rows < cols ? rows : cols, n = rows < cols ? cols : rows;
  return up((size_t)m * blocks_of((int)n) * 128) + 2 * up((size_t)n * blocks_of((int)m) * 128) +
         2 * up((size_t)m * blocks_of((int)m) * 128) + up(sizeof(double) * NORM_PARTS);
}

void lay(Matrix &M, long rows, long cols, char *&ws) {
  M.turned = rows > cols;
  M.m = (int)(M.turned ? cols : rows);
  M.n = (int)(M.turned ? rows : cols);
  const long parts = ((long)M.m * M.n + 8191) / 8192;
  M.parts = (int)(parts < NORM_PARTS ? parts : NORM_PARTS);
  auto take = [&](size_t bytes) {
    char *p = ws;
    ws += up(bytes);
    return p;
  };
  M.x = take((size_t)M.m * blocks_of(M.n) * 128);
  M.t0 = take((size_t)M.n * blocks_of(M.m) * 128);
  M.t1 = take((size_t)M.n * blocks_of(M.m) * 128);
  M.p = take((size_t)M.m * blocks_of(M.m) * 128);
  M.q = take((size_t)M.m * blocks_of(M.m) * 128);
  M.norm = (double *)take(sizeof(double) * NORM_PARTS);
}

template <class F>
unsigned long number(Matrices &a, F workgroups) {
  unsigned long at = 0;
  const int kinds = a.alike ? 1 : a.count;
  for (int i = 0; i < kinds; i++) {
    a.first[i] = at;
    at += (unsigned long)workgroups(a.at[i]);
  }
  a.first[kinds] = at;
  return a.alike ? at * a.count : at;
}

// Whether every matrix has a workgroup of its own.
bool by_block(const Matrices &a) {
  for (int i = 0; i < (a.alike ? 1 : a.count); i++)
    if (!fits_block(a.at[i].m, a.at[i].n)) return false;
  return !TT_NOBLOCK;
}

// How the products of such matrices go: by tiles of 32 (0), 128 or 256.
int tile_size(const Matrices &a) {
  double work = 0;
  for (int i = 0; i < a.count; i++) {
    const Matrix &M = a.at[a.alike ? 0 : i];
    work += (double)M.m * M.m * M.n;
  }
  return work < TT_LARGE ? 0 : work < TT_HUGE ? 128 : 256;
}

template <int KIND>
void small_product(Matrices &a, int step) {
  const unsigned long grid = number(a, [](const Matrix &M) {
    return KIND <= SQUARE ? blocks_of(M.m) * (blocks_of(M.m) + 1) / 2 : blocks_of(M.m) * blocks_of(M.n);
  });
  hipLaunchKernelGGL(small_kernel<KIND>, dim3((unsigned)grid), dim3(512), 0, stream(), a, step);
}

template <int KIND, int T>
void tile_product(Matrices &a, int step, float *pieces) {
  typedef Shape<T> S;
  bool alike = true;  // in their blocks
  long blocks = 0;
  unsigned long tiles = 0;
  Deal d = {};
  d.units = number(a, [&](const Matrix &M) {
    const long nr = (M.m + T - 1) / T, nc = (M.n + T - 1) / T, k = blocks_of(KIND == GRAM ? M.n : M.m);
    alike = alike && (!blocks || blocks == k);
    blocks = k;
    tiles += (KIND <= SQUARE ? nr * (nr + 1) / 2 : nr * nc) * (a.alike ? a.count : 1);
    return (KIND <= SQUARE ? nr * (nr + 1) / 2 : nr * nc) * k;
  });
  const unsigned groups = (unsigned)(d.units < 8 * S::GROUPS ? (d.units + 7) / 8 : S::GROUPS);
  if (alike) {  // whole tiles side by side read the same blocks at about the same time
    d.rounds = (unsigned)(tiles / groups);
    d.base = (unsigned long)d.rounds * groups * blocks;
    d.units -= d.base;
  }
  d.sharers = (unsigned)(d.units < 8ul * groups ? (d.units + 7) / 8 : groups);
  hipLaunchKernelGGL((tile_kernel<KIND, T>), dim3(groups), dim3(S::WAVES * 64), 0, stream(), a, step, d, pieces);
  if (d.sharers > 1)
    hipLaunchKernelGGL((join_kernel<KIND, T>), dim3(d.sharers - 1, S::PIECE / 4096), dim3(256), 0, stream(), a, step, d,
                       (const float *)pieces);
}

template <int KIND>
void product(Matrices &a, int step, int tile, float *pieces) {
  if (tile == 0) small_product<KIND>(a, step);
  else if (tile == 128) tile_product<KIND, 128>(a, step, pieces);
  else tile_product<KIND, 256>(a, step, pieces);
}

void run(Matrices &a, int steps, float mu, int nesterov, char *rest) {
  if (by_block(a)) {
    hipLaunchKernelGGL(block_kernel, dim3(a.count), dim3(BLOCK_WAVES * 64), 0, stream(), a, steps, mu, nesterov);
    return;
  }
  unsigned long grid = number(a, [](const Matrix &M) { return (long)M.parts; });
  hipLaunchKernelGGL(momentum_kernel, dim3((unsigned)grid), dim3(256), 0, stream(), a, mu, nesterov);
  grid = number(a, [](const Matrix &M) { return (long)((M.m + 63) / 64) * ((M.n + 63) / 64); });
  hipLaunchKernelGGL(image_kernel, dim3((unsigned)grid), dim3(256), 0, stream(), a, mu, nesterov);
  const int tile = tile_size(a);
  for (int s = 0; s < steps; s++) {
    product<GRAM>(a, s, tile, (float *)rest);
    product<SQUARE>(a, s, tile, (float *)rest);
    if (s + 1 < steps) product<STEP>(a, s, tile, (float *)rest);
    else product<LAST>(a, s, tile, (float *)rest);
  }
}

// the images (of a group of matrices), and two pieces a workgroup
size_t ws_of(const Matrices &a, size_t images) {
  if (by_block(a)) return 0;
  const int t = tile_size(a);
  return images + (t == 0 ? 0 : 2 * sizeof(float) * t * t * (t == 128 ? Shape<128>::GROUPS : Shape<256>::GROUPS));
}

// `count` matrices of one shape
void alike(Matrices &a, long count, long rows, long cols, char *ws) {
  a = {};
  a.count = (int)(count < ALIKE ? count : ALIKE);
  a.alike = 1;
  a.images = (long)images_of(rows, cols);
  lay(a.at[0], rows, cols, ws);
}

}  // namespace

extern "C" size_t tt_k_newton_schulz_ws(long count, long rows, long cols) {
  if (count <= 0 || !good_sides(rows, cols)) return 0;
  Matrices a;
  alike(a, count, rows, cols, NULL);
  return ws_of(a, a.count * (size_t)a.images);
}

extern "C" int tt_k_newton_schulz(const float *x, float *y, long count, long rows, long cols, int steps, void *ws) {
  if (!x || !y || count <= 0 || !good_sides(rows, cols) || count > (1L << 40) / (rows * cols) || steps < 1 ||
      steps > TT_NS_MAX_STEPS)
    return -1;
  if (ttrt_init() != 0) return -3;
  const size_t need = tt_k_newton_schulz_ws(count, rows, cols);
  void *own = NULL;
  if (need && !ws) {
    ws = own = ttrt_alloc(need);
    if (!ws) return -2;
  }
  Matrices a;
  alike(a, count, rows, cols, (char *)ws);
  const int most = by_block(a) ? 1 << 20 : a.count;  // without images any number at once
  for (long base = 0; base < count; base += most) {
    a.count = (int)(count - base < most ? count - base : most);
    a.at[0].g = x + base * rows * cols;
    a.at[0].w = y + base * rows * cols;
    run(a, steps, 0.f, 0, (char *)ws + (size_t)(count < ALIKE ? count : ALIKE) * a.images);
  }
  ttrt_free(own);
  return launched();
}

extern "C" size_t tt_k_muon_multi_ws(const long *rows, const long *cols, int count) {
  if (!rows || !cols || count < 1 || count > TT_SGD_MAX) return 0;
  Matrices a = {};
  a.count = count;
  size_t bytes = 0;
  char *at = NULL;
  for (int i = 0; i < count; i++) {
    if (!good_sides(rows[i], cols[i])) return 0;
    lay(a.at[i], rows[i], cols[i], at);
    bytes += images_of(rows[i], cols[i]);
  }
  return ws_of(a, bytes);
}

extern "C" int tt_k_muon_multi(float *const *w, const float *const *g, float *const *v, const long *rows,
                               const long *cols, int count, float lr, float mu, int nesterov, float decay, void *ws) {
  if (!w || !g || !v || !rows || !cols || count < 0 || count > TT_SGD_MAX || !isfinite(lr) || !isfinite(mu) ||
      !isfinite(decay))
    return -1;
  for (int i = 0; i < count; i++) {
    if (!w[i] || !g[i] || !v[i] || !good_sides(rows[i], cols[i])) return -1;
    for (int j = 0; j < i; j++)
      if (w[j] == w[i] || v[j] == v[i]) return -1;
  }
  if (count == 0) return 0;
  if (ttrt_init() != 0) return -3;
  const size_t need = tt_k_muon_multi_ws(rows, cols, count);
  void *own = NULL;
  if (need && !ws) {
    ws = own = ttrt_alloc(need);
    if (!ws) return -2;
  }
  Matrices a = {};
  a.count = count;
  char *at = (char *)ws;
  for (int i = 0; i < count; i++) {
    Matrix &M = a.at[i];
    M.g = g[i], M.v = v[i], M.w = w[i];
    M.keep = (float)(1.0 - (double)lr * decay);
    M.rate = (float)(-(double)lr * TT_MUON_RMS * sqrt((double)(rows[i] > cols[i] ? rows[i] : cols[i])));
    lay(M, rows[i], cols[i], at);
  }
  run(a, TT_MUON_STEPS, mu, nesterov, at);
  ttrt_free(own);
  return launched();
}
