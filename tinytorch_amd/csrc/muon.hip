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
// X, X^T, P and Q are kept as images: blocks of 32 x 32 values as the matrix
// instructions take them, four times 1 KB: h of the columns 0 to 15, where lane l
// has eight of row l % 32 from column 8 (l / 32) on, of the columns 16 to 31, and l
// of both; zeros behind the last row and column.  A wave's load is then 1 KB in one
// piece (rows of 128 bytes, 32 of them a load, take the address unit 40 cycles: three
// times as long a product of 16 x 4000).  Both operands of a product are read along
// rows: P = X X^T, P P = P P^T, Q X = Q (X^T)^T.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>
#include "tt_rt.h"

namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef f32x4 __attribute__((aligned(4))) f32x4_any;

inline hipStream_t stream() { return (hipStream_t)ttrt_stream(); }
inline int launched() { return hipGetLastError() == hipSuccess ? 0 : -3; }

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
// N matrices, or with N = 1 `count` of at[0]'s shape one behind the other.  (A kernel's
// arguments come from afar: of the longer form each line that it needs costs it 0.5 us.)
template <int N>
struct Matrices {
  Matrix at[N];
  unsigned long first[N + 1];  // matrix i has the workgroups, or the units of work, [first[i], first[i + 1])
  int count;
  long images;  // N = 1: bytes of a matrix's workspace
};

__host__ __device__ inline long blocks_of(int k) { return (k + 31) / 32; }

// which matrix a workgroup or unit belongs to; b becomes its number among that one's
template <int N>
__device__ __forceinline__ Matrix matrix(const Matrices<N> &a, int i) {
  if (N > 1) return a.at[i];
  Matrix M = a.at[0];
  M.g += (long)i * M.m * M.n, M.w += (long)i * M.m * M.n;
  const long off = i * a.images;
  M.x += off, M.t0 += off, M.t1 += off, M.p += off, M.q += off;
  M.norm += off / (long)sizeof(double);
  return M;
}
template <int N, class U>
__device__ __forceinline__ Matrix matrix_of(const Matrices<N> &a, U &b) {
  int i = 0;
  if (N > 1) {
    while (i + 1 < a.count && b >= a.first[i + 1]) i++;
    b -= (U)a.first[i];
  } else if (a.count > 1) {
    i = (int)(b / (U)a.first[1]);
    b -= (U)i * (U)a.first[1];
  }
  return matrix(a, i);
}

// x 2^14 in two parts
__device__ __forceinline__ void split(float y, _Float16 &h, _Float16 &l) {
  h = (_Float16)y;
  l = (_Float16)(y - (float)h);
}
// where h of row r and column c of an image lies (l 1024 values further)
__device__ __forceinline__ _Float16 *place(char *image, long blocks, int r, int c) {
  return (_Float16 *)(image + ((r >> 5) * blocks + (c >> 5)) * 4096 + (c >> 4 & 1) * 1024 +
                      ((r & 31) + (c >> 3 & 1) * 32) * 16) +
         (c & 7);
}
// two values of row r from the even column c on
__device__ __forceinline__ void put2(char *image, long blocks, int r, int c, float x, float y) {
  typedef _Float16 half2 __attribute__((ext_vector_type(2)));
  half2 h, l;
  _Float16 a, b;
  split(x * UP, a, b);
  h[0] = a, l[0] = b;
  split(y * UP, a, b);
  h[1] = a, l[1] = b;
  _Float16 *p = place(image, blocks, r, c);
  *(half2 *)p = h;
  *(half2 *)(p + 1024) = l;
}
// 16 values (times 2^14 already) of row r from column c on, a multiple of 16
__device__ __forceinline__ void put16(char *image, long blocks, int r, int c, const float (&v)[16]) {
  half8 h[2], l[2];
#pragma unroll
  for (int j = 0; j < 16; j++) {
    _Float16 a, b;
    split(v[j], a, b);
    h[j / 8][j % 8] = a;
    l[j / 8][j % 8] = b;
  }
  half8 *p = (half8 *)place(image, blocks, r, c);
  p[0] = h[0], p[32] = h[1], p[128] = l[0], p[160] = l[1];
}

// ---------------------------------------------------------------- small matrices
//
// A matrix whose image of X and of P or Q (which follow each other in one place) fit
// LDS has a workgroup, which takes it from the gradient to the weights in one
// launch.  A wave has blocks of 32 x 32 of each result, kept in registers until all
// have read what they replace.  X^T is X read by transposing loads.  The products
// are formed transposed: a lane then holds four neighbours of a row, and P and Q
// are symmetric.  Latency bounds it, of LDS and between the products of a chain: five
// steps of 32 x 32 take 23 us, of 64 x 64 26, of 128 x 128 63, of 64 of these 65.

constexpr int BLOCK_WAVES = 16, BLOCK_LDS = 160 * 1024 - 256;
constexpr int BLOCK_KEEP = 3;  // blocks of X a wave
// X, P and the partial sums of P (one or four blocks of it: eight or two waves each)
__host__ __device__ inline long block_bytes(int m, int n) {
  const long mb = blocks_of(m), nb = blocks_of(n);
  return 4096 * (mb * nb + mb * mb + (mb == 1 ? 7 : mb == 2 ? 4 : 0));
}
// Of a few matrices those whose products have up to 64 blocks (five steps of 128 x 128:
// 63 us, and 72 by launches of a product each; of 128 x 160 72 and 70, of 96 x 300 84
// and 71), of many all that fit (32 of 96 x 300: 85 and 82, 500 of 128 x 128: 145 and 683).
inline bool fits_block(int m, int n, int count) {
  const long mb = blocks_of(m), nb = blocks_of(n);
  return block_bytes(m, n) <= BLOCK_LDS && mb * nb <= BLOCK_WAVES * BLOCK_KEEP && (count >= 32 || mb * mb * nb <= 64);
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
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
__device__ __forceinline__ s16x4 read_transposed(const char *p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)const_cast<char *>(p));
}
// eight rows r0 + 8 (lane / 32) .. of column lane % 32 of a block
__device__ __forceinline__ half8 across(const char *image, int blocks, int r0, int block, int part, int lane) {
  s16x8 v;
  const int l = lane & 15, c = (lane >> 4 & 1) * 16 + 4 * (l & 3);
#pragma unroll
  for (int x = 0; x < 2; x++) {
    const char *p = chunk_of(image, blocks, r0 + (lane >> 5) * 8 + x * 4 + l / 4, block, part * 4 + c / 8) + (c & 4) * 2;
    const s16x4 w = read_transposed(p);
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

template <int N>
__global__ void __launch_bounds__(BLOCK_WAVES * 64) block_kernel(Matrices<N> a, int steps, float mu, int nesterov) {
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
// Bound by memory: 26 us for a block's weights of 12.6 million values (5.8 TB/s).
template <int N>
__global__ void __launch_bounds__(256) momentum_kernel(Matrices<N> a, float mu, int nesterov) {
  __shared__ double sums[4];
  unsigned b = blockIdx.x;
  const Matrix M = matrix_of(a, b);
  const long count = (long)M.m * M.n, groups = count / 4;
  double s = 0.0;
  for (long i = (long)b * 512 + threadIdx.x; i < groups; i += (long)M.parts * 512) {
    f32x4 u[2];
#pragma unroll
    for (int k = 0; k < 2; k++) {
      u[k] = (f32x4){0.f, 0.f, 0.f, 0.f};
      const long at = (i + k * 256) * 4;
      if (i + k * 256 < groups) u[k] = momentum<f32x4_any>(M.g + at, M.v ? M.v + at : nullptr, mu, nesterov, true);
    }
#pragma unroll
    for (int k = 0; k < 2; k++)
#pragma unroll
      for (int j = 0; j < 4; j++) s = fma((double)u[k][j], (double)u[k][j], s);
  }
  const long tail = groups * 4 + threadIdx.x;  // up to three more
  if (b == 0 && tail < count) {
    const float u = momentum<float>(M.g + tail, M.v ? M.v + tail : nullptr, mu, nesterov, true);
    s = fma((double)u, (double)u, s);
  }
#pragma unroll
  for (int k = 1; k < 64; k <<= 1) s += __shfl_xor(s, k);
  if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) M.norm[b] = (sums[0] + sums[1]) + (sums[2] + sums[3]);
}

// The images of U / |U|_F and its transpose, a tile of 64 x 64 at a time through
// LDS; both are written along their rows.  Bound by memory: 36 us for 4096 x 4096
// (5.6 TB/s).
template <int N>
__global__ void __launch_bounds__(256) image_kernel(Matrices<N> a, float mu, int nesterov) {
  __shared__ double sums[4];
  __shared__ float tile[64][65];
  unsigned b = blockIdx.x;
  const Matrix M = matrix_of(a, b);
  const int rows = M.turned ? M.n : M.m, cols = M.turned ? M.m : M.n, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const unsigned across = (unsigned)((cols + 63) / 64);
  const int r0 = (int)(b / across) * 64, c0 = (int)(b % across) * 64;
  float u[16];  // on their way while the norm is added up
#pragma unroll
  for (int k = 0; k < 16; k++) {
    const int r = r0 + k * 4 + wave, c = c0 + lane;
    u[k] = 0.f;
    if (r < rows && c < cols) {
      const long at = (long)r * cols + c;
      u[k] = momentum<float>(M.g + at, M.v ? M.v + at : nullptr, mu, nesterov, false);
    }
  }
  double s = 0.0;
  for (int i = threadIdx.x; i < M.parts; i += 256) s += M.norm[i];
#pragma unroll
  for (int k = 1; k < 64; k <<= 1) s += __shfl_xor(s, k);
  if (lane == 0) sums[wave] = s;
  __syncthreads();
  s = (sums[0] + sums[1]) + (sums[2] + sums[3]);
  const double scale = s == 0.0 ? 0.0 : (double)UP / sqrt(s);  // zeros stay zeros
#pragma unroll
  for (int k = 0; k < 16; k++) tile[k * 4 + wave][lane] = (float)((double)u[k] * scale);
  __syncthreads();
  char *along = M.turned ? M.t0 : M.x, *down = M.turned ? M.x : M.t0;
  const long row_blocks = blocks_of(cols), col_blocks = blocks_of(rows);
  const int line = threadIdx.x >> 2, from = (threadIdx.x & 3) * 16;  // 16 values of a row, then of a column
  float v[16];
  if ((r0 + line) / 32 < col_blocks && (c0 + from) / 32 < row_blocks) {
#pragma unroll
    for (int j = 0; j < 16; j++) v[j] = tile[line][from + j];
    put16(along, row_blocks, r0 + line, c0 + from, v);
  }
  if ((c0 + line) / 32 < row_blocks && (r0 + from) / 32 < col_blocks) {
#pragma unroll
    for (int j = 0; j < 16; j++) v[j] = tile[from + j][line];
    put16(down, col_blocks, c0 + line, r0 + from, v);
  }
}

// ---------------------------------------------------------------- products

enum { GRAM, SQUARE, STEP };  // P = X X^T; Q = b P + c P P; X <- a X + Q X, the last one to w

// Tile `b` of a symmetric matrix: those of the lower triangle row by row.
__device__ __forceinline__ void triangle(unsigned b, int &i, int &j) {
  int r = (int)((sqrtf(8.f * b + 1.f) - 1.f) * 0.5f);
  while ((unsigned)r * (r + 1u) / 2 > b) r--;
  while ((unsigned)(r + 1) * (r + 2u) / 2 <= b) r++;
  i = r;
  j = (int)(b - (unsigned)r * (r + 1u) / 2);
}

template <int KIND>
struct Operands {
  const char *a, *b;    // images whose rows are multiplied
  const char *add;      // image of the transpose of the matrix added, times `times` (GRAM: none)
  const char *plain;    // and of that matrix
  char *out, *down;     // images of the result and its transpose
  int rows, cols, k;    // of the result; the products' length
  float by, times;
  __device__ __forceinline__ Operands(const Matrix &M, int step) {
    if (KIND == GRAM) {
      a = b = M.x, add = plain = nullptr, out = down = M.p;
      rows = cols = M.m, k = M.n, by = 1.f, times = 0.f;
    } else if (KIND == SQUARE) {
      a = b = add = plain = M.p, out = down = M.q;
      rows = cols = k = M.m, by = TT_NS_C, times = TT_NS_B;
    } else {
      a = M.q, b = add = step & 1 ? M.t1 : M.t0, plain = M.x, out = M.x, down = step & 1 ? M.t0 : M.t1;
      rows = k = M.m, cols = M.n, by = 1.f, times = TT_NS_A;
    }
  }
};

// Consecutive workgroups go to the eight XCDs in turn: each XCD gets a run of them,
// and the tiles are in bands of eight rows, column by column, so that what an XCD's
// L2 holds are the rows and columns of a patch.
__device__ __forceinline__ unsigned dealt(unsigned b, unsigned n) {
  const unsigned each = n / 8;
  return b < each * 8 ? (b % 8) * each + b / 8 : b;
}
constexpr int BAND = 8;
template <int KIND, int T, class U>
__device__ __forceinline__ void tile_of(U tile, int rows, int cols, int &ti, int &tj) {
  const int nr = (rows + T - 1) / T, nc = (cols + T - 1) / T;
  if (KIND <= SQUARE) {
    // below band b: 32 b^2 + 4 b tiles of the lower triangle
    int b = (int)((sqrtf(128.f * (float)tile + 16.f) - 4.f) / 64.f);
    while (b > 0 && (U)32 * b * b + (U)4 * b > tile) b--;
    while ((U)32 * (b + 1) * (b + 1) + (U)4 * (b + 1) <= tile) b++;
    const unsigned in = (unsigned)(tile - ((U)32 * b * b + (U)4 * b));
    const unsigned h = nr - b * BAND < BAND ? nr - b * BAND : BAND;
    if (in < (unsigned)b * BAND * h) {
      ti = b * BAND + (int)(in % h), tj = (int)(in / h);
    } else {
      triangle(in - (unsigned)b * BAND * h, ti, tj);
      ti += b * BAND, tj += b * BAND;
    }
  } else {
    const U band = (U)BAND * nc;
    const int b = (int)(tile / band);
    const unsigned in = (unsigned)(tile % band), h = nr - b * BAND < BAND ? nr - b * BAND : BAND;
    ti = b * BAND + (int)(in % h), tj = (int)(in / h);
  }
}

// Tiles of 32 x 32, one a workgroup, the operands read from memory as the matrix
// instructions take them and each wave with a share of the products' length:
// eight sums, joined in LDS.  What bounds these is the way from memory (the L2 of
// another XCD has what the last launch wrote), so the added matrix is on its way
// first, and a tile on the diagonal reads its rows once.  A launch takes 4 us at least;
// 517 x 1003: 6 us for P, 5 for Q, 10 for X; 1300 x 1300: 18, 18 and 29 (450 TFLOP/s
// of fp16 products).  Of few long tiles of P the length is shared by `ways` workgroups,
// whose sums a second launch adds (join): one CU alone reads 80 GB/s.
template <int KIND, bool SHARED, int N>
__global__ void __launch_bounds__(512, 2)
    small_kernel(Matrices<N> a, int step, int to_w, int ways, bool join, float *pieces) {
  typedef _Float16 half2 __attribute__((ext_vector_type(2)));
  constexpr int WAVES = 8;
  __shared__ float sums[WAVES][32][33];
  unsigned t = dealt(blockIdx.x, gridDim.x), way = 0;
  f32x2 *piece = nullptr;
  if (SHARED) {
    piece = (f32x2 *)pieces + (join ? t * ways : t) * 512l + threadIdx.x;
    if (!join) way = t % ways, t /= ways;
  }
  const Matrix M = matrix_of(a, t);
  const Operands<KIND> o(M, step);
  int ti, tj;
  tile_of<KIND, 32>(t, o.rows, o.cols, ti, tj);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = threadIdx.x >> 4, c = (threadIdx.x & 15) * 2;  // this thread's two results
  const int row = ti * 32 + r, col = tj * 32 + c;
  float v[2] = {0.f, 0.f};
  if (KIND != GRAM) {
    const _Float16 *p = place((char *)o.plain, blocks_of(o.cols), row, col);
    const half2 h = *(const half2 *)p, l = *(const half2 *)(p + 1024);
#pragma unroll
    for (int e = 0; e < 2; e++) v[e] = o.times * (1.f / UP) * ((float)h[e] + (float)l[e]);
  }
  float sum[2] = {0.f, 0.f};
  if (SHARED && join) {
#pragma unroll 8
    for (int w = 0; w < ways; w++) {
      const f32x2 p = piece[w * 512l];
      sum[0] += p[0], sum[1] += p[1];
    }
  } else {
    const int blocks = (int)blocks_of(o.k);
    const char *pa = o.a + (long)ti * blocks * 4096 + lane * 16, *pb = o.b + (long)tj * blocks * 4096 + lane * 16;
    f32x16 acc = {};
    const bool same = KIND <= SQUARE && ti == tj;
    for (int k = way * WAVES + wave; k < blocks; k += (SHARED ? ways : 1) * WAVES) {
      half8 x[4], y[4];
#pragma unroll
      for (int s = 0; s < 4; s++) {
        x[s] = *(const half8 *)(pa + k * 4096l + s * 1024);
        y[s] = x[s];
      }
      if (!same) {
#pragma unroll
        for (int s = 0; s < 4; s++) y[s] = *(const half8 *)(pb + k * 4096l + s * 1024);
      }
#pragma unroll
      for (int s = 0; s < 2; s++) three(acc, x[s], x[2 + s], y[s], y[2 + s]);
    }
#pragma unroll
    for (int i = 0; i < 16; i++) sums[wave][8 * (i / 4) + 4 * (lane >> 5) + i % 4][lane & 31] = acc[i];
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 2; e++)
#pragma unroll
      for (int w = 0; w < WAVES; w++) sum[e] += sums[w][r][c + e];
    if (SHARED) {
      *piece = (f32x2){sum[0], sum[1]};
      return;
    }
  }
  bool in[2];
#pragma unroll
  for (int e = 0; e < 2; e++) {
    in[e] = row < o.rows && col + e < o.cols;
    v[e] = in[e] ? v[e] + sum[e] * (o.by * DOWN2) : 0.f;
  }
  if (KIND == STEP && to_w) {
#pragma unroll
    for (int e = 0; e < 2; e++)
      if (in[e] && !M.turned) {
        float *w = M.w + (long)row * o.cols + col + e;
        *w = M.v ? M.keep * *w + M.rate * v[e] : v[e];
      }
  } else {
    put2(o.out, blocks_of(o.cols), row, col, v[0], v[1]);
  }
  if ((KIND <= SQUARE && ti == tj) || (KIND == STEP && to_w && !M.turned)) return;
  __syncthreads();
  sums[0][r][c] = v[0];
  sums[0][r][c + 1] = v[1];
  __syncthreads();
  const int trow = tj * 32 + r, tcol = ti * 32 + c;  // the transpose
  if (KIND == STEP && to_w) {
#pragma unroll
    for (int e = 0; e < 2; e++)
      if (trow < o.cols && tcol + e < o.rows) {
        float *w = M.w + (long)trow * o.rows + tcol + e;
        *w = M.v ? M.keep * *w + M.rate * sums[0][c + e][r] : sums[0][c + e][r];
      }
  } else {
    put2(o.down, blocks_of(o.rows), trow, tcol, sums[0][c][r], sums[0][c + 1][r]);
  }
}

// ---------------------------------------------------------------- large products
//
// The operands come through LDS by direct loads, a block (32 of the products' length)
// at a time, in buffers.  In the 32 cycles of a 32 x 32 x 16 product LDS gives a SIMD one
// of its two operands, so a wave has as large a tile as its registers hold, and what it
// reads goes into several products:
//   tiles of 128  four waves of 64 x 64, one a SIMD, three buffers: a block is on its
//                 way while two are there, and the reads stand between the products
//   tiles of 256  eight waves of 128 x 64, two a SIMD, two buffers: the other wave of
//                 the SIMD fills a wave's waits, and memory gives half as much
// A tile that one workgroup has is finished by it.  The others' parts go to memory,
// and join_kernel adds them.  The matrix units bound these, at the clock that they
// leave: X of 4096 x 4096 takes 343 us, 1200 TFLOP/s of fp16 products, with the units
// 69 % busy at 1.84 GHz; of 2048 x 2048 by tiles of 128 50 us, 1030 TFLOP/s (51 % busy
// at 2 GHz in a transformer block's six matrices).

// Tiles of T x T: four waves of 64 x 64 or eight of 128 x 64 values, each FI x 2
// blocks of 32 x 32.
template <int T, int BUFFERS>
struct Shape {
  static constexpr int WAVES = T == 256 ? 8 : 4, ACROSS = WAVES / 2, FI = T / 64, BLOCKS = 2 * FI;
  static constexpr int BUFFER = 2 * T * 128;  // bytes of both operands' block
  static constexpr int GROUPS = 256;          // workgroups at most: one a CU
  static constexpr int PIECE = T * T;         // floats
  static constexpr int EACH = T / 8 / WAVES;  // loads of either operand's block a wave
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

// A wave's 32 x 32 values from (r0, c0) on as the matrix instructions leave them: a
// lane has of column low = lane % 32 the rows high + 8 i + {0 .. 3}, high = 4 (lane / 32).
// In the image of the transpose those are 8 bytes that with the other lanes' make
// 512, so there they are read (what is added: P is symmetric, X^T has an image) and
// written as they are; the image itself gets its blocks by transposing reads of LDS.
// Behind the last row and column all of it is 0, as the operands are there.
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
struct Added {
  half4 h[4], l[4];
};
__device__ __forceinline__ int part_of(int i, int lane) {  // in the block of the transpose, bytes
  return (i >> 1) * 1024 + ((lane & 31) + 32 * (i & 1)) * 16 + (lane >> 5) * 8;
}
template <int KIND>
__device__ __forceinline__ Added added(const Operands<KIND> &o, int r0, int c0, int lane) {
  Added x = {};
  if (KIND == GRAM || r0 >= o.rows || c0 >= o.cols) return x;
  const char *p = o.add + ((c0 >> 5) * blocks_of(o.rows) + (r0 >> 5)) * 4096;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    x.h[i] = *(const half4 *)(p + part_of(i, lane));
    x.l[i] = *(const half4 *)(p + part_of(i, lane) + 2048);
  }
  return x;
}
// buf: 4 KB of LDS, this wave's; both: the image itself too
template <int KIND>
__device__ __forceinline__ void write32(const Matrix &M, const Operands<KIND> &o, const f32x16 &acc, const Added &x,
                                        int r0, int c0, char *buf, int lane, bool both, bool to_w) {
  if (r0 >= o.rows || c0 >= o.cols) return;
  f32x4 v[4];
#pragma unroll
  for (int i = 0; i < 4; i++)
#pragma unroll
    for (int j = 0; j < 4; j++) {
      v[i][j] = acc[i * 4 + j] * (o.by * DOWN2);
      if (KIND != GRAM) v[i][j] += o.times * (1.f / UP) * ((float)x.h[i][j] + (float)x.l[i][j]);
    }
  if (KIND == STEP && to_w) {
    // (as values of their own: the compiler would read `rate` with its neighbours as a
    // vector, for that put M into LDS, and fetch the launch's packet from the host's
    // memory to find its place there: 10 us a launch)
    float rate = M.rate, keep = M.keep;
    asm("" : "+s"(rate), "+s"(keep));
    // what is read is on its way at once: behind the last row or column, theirs
    const int col = c0 + (lane & 31), row = r0 + (lane >> 5) * 4, c = col < o.cols ? col : o.cols - 1;
    if (M.turned && r0 + 32 <= o.rows) {
      float *w = M.w + (long)c * o.rows + row;
      f32x4 old[4] = {};
#pragma unroll
      for (int i = 0; i < 4; i++)
        if (M.v) old[i] = *(const f32x4_any *)(w + 8 * i) * keep;
#pragma unroll
      for (int i = 0; i < 4; i++)
        if (col < o.cols) *(f32x4_any *)(w + 8 * i) = M.v ? old[i] + v[i] * rate : v[i];
      return;
    }
    const long down = M.turned ? 1 : o.cols, start = M.turned ? (long)c * o.rows : c;
    float old[16] = {};
#pragma unroll
    for (int i = 0; i < 16; i++) {
      const int r = row + 8 * (i / 4) + i % 4;
      if (M.v) old[i] = M.w[start + (r < o.rows ? r : o.rows - 1) * down] * keep;
    }
#pragma unroll
    for (int i = 0; i < 16; i++) {
      const int r = row + 8 * (i / 4) + i % 4;
      if (col < o.cols && r < o.rows) M.w[start + r * down] = M.v ? old[i] + v[i / 4][i % 4] * rate : v[i / 4][i % 4];
    }
    return;
  }
  char *down = o.down + ((c0 >> 5) * blocks_of(o.rows) + (r0 >> 5)) * 4096;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    half4 h, l;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      _Float16 a, b;
      split(v[i][j] * UP, a, b);
      h[j] = a, l[j] = b;
    }
    *(half4 *)(down + part_of(i, lane)) = h;
    *(half4 *)(down + part_of(i, lane) + 2048) = l;
    if (both) {
      *(half4 *)(buf + part_of(i, lane)) = h;
      *(half4 *)(buf + part_of(i, lane) + 2048) = l;
    }
  }
  if (!both) return;
  __builtin_amdgcn_wave_barrier();
  char *out = o.out + ((r0 >> 5) * blocks_of(o.cols) + (c0 >> 5)) * 4096 + lane * 16;
  const int l = lane & 15;
#pragma unroll
  for (int f = 0; f < 4; f++) {  // h and l of either 16 columns: eight rows of the transpose's block
    s16x8 w;
#pragma unroll
    for (int x = 0; x < 2; x++) {
      const int r = (f & 1) * 16 + (lane >> 5) * 8 + x * 4 + l / 4;
      const s16x4 t = read_transposed(buf + (f >> 1) * 2048 + (lane >> 4 & 1) * 1024 + (r + 32 * ((l & 3) / 2)) * 16 +
                                      (l & 1) * 8);
#pragma unroll
      for (int j = 0; j < 4; j++) w[x * 4 + j] = t[j];
    }
    *(s16x8 *)(out + (f >> 1) * 2048 + (f & 1) * 1024) = w;
  }
}

// where the 32 x 32 block f of a wave's lies
template <int T>
__device__ __forceinline__ int row_of(int ti, int wave, int f) {
  return ti * T + (wave / Shape<T, 2>::ACROSS) * (T / 2) + f / 2 * 32;
}
template <int T>
__device__ __forceinline__ int col_of(int tj, int wave, int f) {
  return tj * T + (wave % Shape<T, 2>::ACROSS) * 64 + f % 2 * 32;
}
// How the units (tiles' blocks, tile by tile) are dealt: `rounds` whole tiles to every
// workgroup, then the units from `base` on evenly to the first `sharers`.  A tile has
// `extra` units before those of its blocks, for what it costs besides (with products of
// one block among long ones a workgroup had dozens of them: X of 2375 x 1041 and 1503 x
// 570 32 us, and with 3989 x 5 and three more small ones 94).
struct Deal {
  unsigned rounds, sharers, extra;
  unsigned long base, units;
  // the first of workgroup w's share
  __device__ __forceinline__ unsigned long begins(unsigned w) const {
    return base + (w < sharers ? units * w / sharers : units);  // (no sharers: no units)
  }
};

template <int KIND, int T, int BUFFERS, int N>
__global__ void __launch_bounds__((Shape<T, BUFFERS>::WAVES * 64), (Shape<T, BUFFERS>::WAVES / 4)) tile_kernel(Matrices<N> a, int step, int to_w, Deal deal, float *pieces) {
  typedef Shape<T, BUFFERS> S;
  __shared__ __attribute__((aligned(1024))) char lds[BUFFERS * S::BUFFER];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned groups = gridDim.x, w = dealt(blockIdx.x, groups);
  const unsigned to = lds_address(lds);
  unsigned round = 0;
  for (unsigned long u = 0, end = 0;;) {
    if (u == end) {
      if (round < deal.rounds) {  // then all tiles have the same number of blocks
        const Operands<KIND> o(a.at[0], step);
        u = ((unsigned long)round * groups + w) * blocks_of(o.k);
        end = u + blocks_of(o.k);
        if (u >= deal.base) end = u;  // no tile for this workgroup
      } else if (round == deal.rounds) {
        u = deal.begins(w), end = deal.begins(w + 1);
        if (u == end) return;
      } else {
        return;
      }
      round++;
      if (u == end) continue;
    }
    unsigned long in = u;
    const Matrix M = matrix_of(a, in);
    const Operands<KIND> o(M, step);
    const int extra = N > 1 ? deal.extra : 0;
    const long blocks = blocks_of(o.k), units = blocks + extra;
    int ti, tj;
    tile_of<KIND, T>(in / units, o.rows, o.cols, ti, tj);
    const int r0 = (int)(in % units), r1 = (int)(end - u < (unsigned long)(units - r0) ? r0 + (end - u) : units);
    u += r1 - r0;
    if (r1 <= extra) continue;  // none of its blocks
    const int k0 = r0 < extra ? 0 : r0 - extra, k1 = r1 - extra;
    // a wave brings every WAVES-th KB of the tiles' T / 32 blocks; a block behind the
    // last is the last once more: its results are not written
    constexpr int EACH = S::EACH;
    unsigned off[2][EACH];
#pragma unroll
    for (int i = 0; i < EACH; i++) {
      const int kb = wave * EACH + i, ra = (o.rows - 1) / 32 - ti * (T / 32), rb = (o.cols - 1) / 32 - tj * (T / 32);
      off[0][i] = (unsigned)((kb / 4 < ra ? kb / 4 : ra) * blocks * 4096) + kb % 4 * 1024 + lane * 16;
      off[1][i] = (unsigned)((kb / 4 < rb ? kb / 4 : rb) * blocks * 4096) + kb % 4 * 1024 + lane * 16;
    }
    const char *pa = scalar(o.a + ((long)ti * (T / 32) * blocks + k0) * 4096);
    const char *pb = scalar(o.b + ((long)tj * (T / 32) * blocks + k0) * 4096);
    auto bring = [&](int k, unsigned at) {
#pragma unroll
      for (int i = 0; i < EACH; i++) dma16(pa + (long)k * 4096, off[0][i], at + (wave * EACH + i) * 1024);
#pragma unroll
      for (int i = 0; i < EACH; i++) dma16(pb + (long)k * 4096, off[1][i], at + T * 128 + (wave * EACH + i) * 1024);
    };
    f32x16 acc[S::FI][2] = {};
    __syncthreads();  // the last tile's LDS is read
    const int n = k1 - k0;
    for (int k = 0; k < BUFFERS - 1 && k < n; k++) bring(k, to + k * S::BUFFER);
    // the wave's blocks of either operand in a buffer
    const char *mine[2] = {lds + (wave / S::ACROSS) * (T / 2) * 128 + lane * 16,
                           lds + (T + (wave % S::ACROSS) * 64) * 128 + lane * 16};
    struct Half {  // 16 of a block's 32: the wave's blocks of either operand
      half8 ha[S::FI], la[S::FI], hb[2], lb[2];
    };
    auto read = [&](int at) {  // (compile-time offsets from one address)
      Half x;
#pragma unroll
      for (int j = 0; j < 2; j++) {
        x.hb[j] = *(const half8 *)(mine[1] + at + j * 4096);
        x.lb[j] = *(const half8 *)(mine[1] + at + j * 4096 + 2048);
      }
#pragma unroll
      for (int i = 0; i < S::FI; i++) {
        x.ha[i] = *(const half8 *)(mine[0] + at + i * 4096);
        x.la[i] = *(const half8 *)(mine[0] + at + i * 4096 + 2048);
      }
      return x;
    };
    auto multiply = [&](const Half &x) {
#pragma unroll
      for (int i = 0; i < S::FI; i++)
#pragma unroll
        for (int j = 0; j < 2; j++)
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x.la[i], x.hb[j], acc[i][j], 0, 0, 0);
#pragma unroll
      for (int i = 0; i < S::FI; i++)
#pragma unroll
        for (int j = 0; j < 2; j++)
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x.ha[i], x.lb[j], acc[i][j], 0, 0, 0);
#pragma unroll
      for (int i = 0; i < S::FI; i++)
#pragma unroll
        for (int j = 0; j < 2; j++)
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x.ha[i], x.hb[j], acc[i][j], 0, 0, 0);
    };
    auto arrived = [&](int k) {  // block k, in LDS for every wave
      if (k + BUFFERS - 2 < n)   // with so many behind it still on their way
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"((BUFFERS - 2) * 2 * S::EACH) : "memory");
      else
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
    };
    if constexpr (BUFFERS == 2) {
      for (int k = 0; k < n; k++) {
        arrived(k);
        const int now = (k & 1) * S::BUFFER;
        if (k + 1 < n) bring(k + 1, to + (S::BUFFER - now));
        multiply(read(now));
        multiply(read(now + 1024));
      }
    } else {
      // A wave a SIMD: while it waits to hand over a read or a load it starts no
      // product, so these stand between the products one by one: after each of the
      // first eight a read of the next half, after the others (load) a KB of one
      // operand of the block BUFFERS - 1 further (2048 x 2048: 62 us a product with the
      // reads and loads before the products).
      static_assert(S::FI == 2 && S::EACH == 4, "one wave a SIMD has 64 x 64");
      auto half = [&](const Half &x, Half &y, int at, bool load, const char *from, const unsigned *part, unsigned to) {
#pragma unroll
        for (int m = 0; m < 12; m++) {
          const int i = m >> 1 & 1, j = m & 1;
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(m < 4 ? x.la[i] : x.ha[i], m >= 4 && m < 8 ? x.lb[j] : x.hb[j],
                                                             acc[i][j], 0, 0, 0);
          if (m < 8) {  // in the order in which the products take them
            const int q = m & 1, f = m >> 1 & 1;
            const half8 v = *(const half8 *)(mine[q] + at + f * 4096 + ((m < 4) != (q == 1) ? 2048 : 0));
            if (m < 4) {
              if (q) y.hb[f] = v;
              else y.la[f] = v;
            } else {
              if (q) y.lb[f] = v;
              else y.ha[f] = v;
            }
          } else if (load) {
            dma16(from, part[m - 8], to + (wave * S::EACH + m - 8) * 1024);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      };
      arrived(0);
      Half x = read(0), y;
      int now = 0, k = 0;
      for (; k + BUFFERS - 1 < n; k++) {
        const int next = now == (BUFFERS - 1) * S::BUFFER ? 0 : now + S::BUFFER;
        // into the place of the block before, which all have read by the last barrier
        const unsigned free = to + (now == 0 ? (BUFFERS - 1) * S::BUFFER : now - S::BUFFER);
        half(x, y, now + 1024, true, pa + (long)(k + BUFFERS - 1) * 4096, off[0], free);
        // block k + 1 is there when what follows it may still be on its way
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"((BUFFERS - 3) * 2 * S::EACH + S::EACH) : "memory");
        __syncthreads();
        half(y, x, next, true, pb + (long)(k + BUFFERS - 1) * 4096, off[1], free + T * 128);
        now = next;
      }
      for (; k < n; k++) {
        const int next = now == (BUFFERS - 1) * S::BUFFER ? 0 : now + S::BUFFER;
        half(x, y, now + 1024, false, pa, off[0], 0);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        half(y, x, next, false, pb, off[1], 0);  // (behind the last block nothing takes what it reads)
        now = next;
      }
    }
    if (n == blocks) {
      __syncthreads();  // the operands are read
      Added x = added<KIND>(o, row_of<T>(ti, wave, 0), col_of<T>(tj, wave, 0), lane), next = x;
#pragma unroll
      for (int f = 0; f < S::BLOCKS; f++) {
        if (f + 1 < S::BLOCKS) next = added<KIND>(o, row_of<T>(ti, wave, f + 1), col_of<T>(tj, wave, f + 1), lane);
        write32<KIND>(M, o, acc[f / 2][f % 2], x, row_of<T>(ti, wave, f), col_of<T>(tj, wave, f), lds + wave * 4096, lane,
                      KIND == STEP || ti != tj, to_w);
        x = next;
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
  }
}

// Workgroups (w - 1, .) add the pieces of the tile in which the share of
// tile_kernel's workgroup w begins, where that is the first to begin inside it; a
// wave has 32 x 32 of its values.
// Bound by memory (P of 6000 x 6000, tiles of 256: 20 us) or by its own latency (8 to 12
// us for tiles of 128).
template <int KIND, int T, int N>
__global__ void __launch_bounds__(256) join_kernel(Matrices<N> a, int step, int to_w, Deal deal, const float *pieces) {
  typedef Shape<T, 2> S;
  __shared__ __attribute__((aligned(1024))) char buf[4][4096];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned w = blockIdx.x + 1;
  const unsigned long u = deal.begins(w);
  unsigned long in = u;
  const Matrix M = matrix_of(a, in);
  const Operands<KIND> o(M, step);
  const unsigned extra = N > 1 ? deal.extra : 0;
  const unsigned long units = blocks_of(o.k) + extra, first = u - in % units, last = first + units;
  if (u <= first + extra || deal.begins(w - 1) > first + extra) return;
  int ti, tj;
  tile_of<KIND, T>(in / units, o.rows, o.cols, ti, tj);
  const int block = blockIdx.y * 4 + wave;
  const int r0 = row_of<T>(ti, block / S::BLOCKS, block % S::BLOCKS), c0 = col_of<T>(tj, block / S::BLOCKS, block % S::BLOCKS);
  const Added x = added<KIND>(o, r0, c0, lane);
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
  write32<KIND>(M, o, acc, x, r0, c0, buf[wave], lane, KIND == STEP || ti != tj, to_w);
}

// ---------------------------------------------------------------- host

bool good_sides(long rows, long cols) {
  return rows > 0 && cols > 0 && rows <= TT_MUON_MAX_SIDE && cols <= TT_MUON_MAX_SIDE && rows * cols <= TT_MUON_MAX_VALUES;
}

size_t images_of(long rows, long cols) {
  const long m = rows < cols ? rows : cols, n = rows < cols ? cols : rows;
  const size_t mb = blocks_of((int)m), nb = blocks_of((int)n);
  return 4096 * (3 * mb * nb + 2 * mb * mb) + sizeof(double) * NORM_PARTS;
}

void lay(Matrix &M, long rows, long cols, char *&ws) {
  M.turned = rows > cols;
  M.m = (int)(M.turned ? cols : rows);
  M.n = (int)(M.turned ? rows : cols);
  const long parts = ((long)M.m * M.n + 2047) / 2048;
  M.parts = (int)(parts < NORM_PARTS ? parts : NORM_PARTS);
  const size_t mb = blocks_of(M.m), nb = blocks_of(M.n);
  auto take = [&](size_t bytes) {
    char *p = ws;
    ws += bytes;
    return p;
  };
  M.x = take(4096 * mb * nb);
  M.t0 = take(4096 * mb * nb);
  M.t1 = take(4096 * mb * nb);
  M.p = take(4096 * mb * mb);
  M.q = take(4096 * mb * mb);
  M.norm = (double *)take(sizeof(double) * NORM_PARTS);
}

template <int N, class F>
unsigned long number(Matrices<N> &a, F workgroups) {
  unsigned long at = 0;
  const int kinds = N > 1 ? a.count : 1;
  for (int i = 0; i < kinds; i++) {
    a.first[i] = at;
    at += (unsigned long)workgroups(a.at[i]);
  }
  a.first[kinds] = at;
  return N > 1 ? at : at * a.count;
}

// Whether every matrix has a workgroup of its own.
template <int N>
bool by_block(const Matrices<N> &a) {
  for (int i = 0; i < (N > 1 ? a.count : 1); i++)
    if (!fits_block(a.at[i].m, a.at[i].n, a.count)) return false;
  return true;
}

// blocks of a product's length
long length_of(int kind, const Matrix &M) { return blocks_of(kind == GRAM ? M.n : M.m); }

// How a product of such matrices goes: by tiles of 32 (0), 128 or 256, by its work, m m
// and its length, in all of them.  Of a symmetric result half is computed, and smaller
// tiles are used for longer: they have less to compute twice, and their parts are joined
// sooner.  But few tiles of 128 (136 of 2048 rows), or tiles of different lengths, are
// cut into parts that are not in step, so that each XCD reads all of it from afar (two of
// 4096^2, 1024 x 4096 and its turn: 9137 us with tiles of 256, 9798 with 128).  us of a
// product, with what joins its parts:
//                      P = X X^T            X <- a X + Q X
//   tiles of         32   128   256        32   128   256
//   1024^2           11    19     -        15    20     -
//   700 x 4000       15    21     -        26    24     -
//   2 x 1024^2       17    20     -        27    26     -
//   1400^2           18    22     -        33    28     -
//   1600^2           25    27     -        45    40     -
//   1024 x 4096      37    26     -        56    30     -
//   2048^2            -    41    55         -    54    78
//   2500^2            -    75    75         -   118   115
//   2048 x 4096       -    78    78         -   109   122
//   2200 x 6300       -   108   120         -   194   195
//   3000 x 5000       -   147   159         -   297   251
//   2048 x 8192       -   158   117         -   182   189
//   2100 x 12000      -   205   196         -   370   340
//   4096^2            -   198   219         -   391   348
//   4096 x 8192       -   378   385         -   789   682
//   6000^2            -   610   590         -  1359  1117
//   8192^2            -  1511  1326         -  3459  2533
template <int N>
int tile_size(const Matrices<N> &a, int kind) {
  double work = 0, tiles = 0;  // (of 128)
  int widest = 0;
  bool together = kind != STEP;  // of a symmetric result, and in step
  for (int i = 0; i < a.count; i++) {
    const Matrix &M = a.at[N > 1 ? i : 0];
    const double nr = (M.m + 127) / 128;
    work += (double)M.m * M.m * (kind == SQUARE ? M.m : M.n);
    tiles += nr * (nr + 1) / 2;
    together = together && length_of(kind, M) == length_of(kind, a.at[0]);
    widest = M.m > widest ? M.m : widest;
  }
  if (work < (kind == STEP ? 2e9 : 4e9)) return 0;
  return work < (together && tiles >= 160 ? 1.7e11 : 3e10) || widest < 2048 ? 128 : 256;
}

// Workgroups that share tiles of 32, and blocks of the products' length from which on
// they do (P of 100 x 8000: 21 us by one each, twice 5.5 shared; five steps of 64 x 2000
// 86 and 79, of 256 x 1500 96 and 99, of 256 x 2000 103 both ways, of 256 x 3000 119 and 116)
constexpr int SHARERS = 512, LONG = 60;

template <int KIND, int N>
void small_product(Matrices<N> &a, int step, int to_w, float *pieces) {
  const unsigned grid = (unsigned)number(a, [](const Matrix &M) {
    return KIND <= SQUARE ? blocks_of(M.m) * (blocks_of(M.m) + 1) / 2 : blocks_of(M.m) * blocks_of(M.n);
  });
  if constexpr (KIND == GRAM) {
    long length = 0;
    for (int i = 0; i < (N > 1 ? a.count : 1); i++) length = length < blocks_of(a.at[i].n) ? blocks_of(a.at[i].n) : length;
    const long most = length / 16 < 32 ? length / 16 : 32, ways = SHARERS / grid < most ? SHARERS / grid : most;
    if (length >= LONG && ways > 1) {
      for (int join = 0; join < 2; join++)
        hipLaunchKernelGGL((small_kernel<KIND, true, N>), dim3(join ? grid : grid * (unsigned)ways), dim3(512), 0,
                           stream(), a, step, to_w, (int)ways, join, pieces);
      return;
    }
  }
  hipLaunchKernelGGL((small_kernel<KIND, false, N>), dim3(grid), dim3(512), 0, stream(), a, step, to_w, 1, false, pieces);
}

template <int KIND, int T, int BUFFERS, int N>
void tile_product(Matrices<N> &a, int step, int to_w, float *pieces) {
  typedef Shape<T, BUFFERS> S;
  constexpr int EXTRA = T == 128 ? 12 : 6;  // (2375 x 1041 with five: 598 us with 4, 569 with 8, 559 with 12)
  auto tiles_of = [](const Matrix &M) {
    const long nr = (M.m + T - 1) / T, nc = (M.n + T - 1) / T;
    return KIND <= SQUARE ? nr * (nr + 1) / 2 : nr * nc;
  };
  const long blocks = length_of(KIND, a.at[0]);
  bool alike = true;
  unsigned long tiles = 0;
  for (int i = 0; i < (N > 1 ? a.count : 1); i++) {
    alike = alike && length_of(KIND, a.at[i]) == blocks;
    tiles += tiles_of(a.at[i]) * (N > 1 ? 1 : a.count);
  }
  Deal d = {};
  d.extra = alike ? 0 : EXTRA;
  d.units = number(a, [&](const Matrix &M) { return tiles_of(M) * (length_of(KIND, M) + d.extra); });
  const unsigned groups = (unsigned)(d.units < S::GROUPS ? d.units : S::GROUPS);
  d.sharers = (unsigned)(d.units < 8ul * groups ? (d.units + 7) / 8 : groups);
  if (alike) {
    // In blocks of the busiest workgroup's, a join being worth about 12 (8 where every
    // workgroup has one piece, and all of them the same parts of the length): whole
    // tiles as often as they go round, and the rest whole as well, each tile among as
    // many workgroups as there are for it, or evenly.
    d.rounds = (unsigned)(tiles / groups);
    const unsigned long rest = tiles % groups, most = rest ? groups / rest : 1,
                        ways = most < (unsigned long)blocks ? most : blocks;  // no part is empty
    const double whole = rest ? (double)blocks : 0, shared = (double)((blocks + ways - 1) / ways) + 8,
                 even = (double)(rest * blocks) / groups + 12;
    if (rest && whole <= shared && whole <= even) d.rounds++;
    d.base = (unsigned long)d.rounds * groups < tiles ? (unsigned long)d.rounds * groups * blocks : d.units;
    d.units -= d.base;
    if (!d.units) d.sharers = 0;
    else if (shared <= even) d.sharers = (unsigned)(rest * ways);
  }
  hipLaunchKernelGGL((tile_kernel<KIND, T, BUFFERS, N>), dim3(groups), dim3(S::WAVES * 64), 0, stream(), a, step, to_w, d, pieces);
  if (d.sharers > 1)
    hipLaunchKernelGGL((join_kernel<KIND, T, N>), dim3(d.sharers - 1, S::PIECE / 4096), dim3(256), 0, stream(), a, step, to_w, d,
                       (const float *)pieces);
}

template <int KIND, int N>
void product(Matrices<N> &a, int step, float *pieces, int to_w = 0) {
  const int tile = tile_size(a, KIND);
  if (tile == 0) small_product<KIND, N>(a, step, to_w, pieces);
  else if (tile == 128) tile_product<KIND, 128, 3, N>(a, step, to_w, pieces);
  else tile_product<KIND, 256, 2, N>(a, step, to_w, pieces);
}

template <int N>
void run(Matrices<N> &a, bool blocks, int steps, float mu, int nesterov, char *rest) {
  if (blocks) {
    hipLaunchKernelGGL(block_kernel<N>, dim3(a.count), dim3(BLOCK_WAVES * 64), 0, stream(), a, steps, mu, nesterov);
    return;
  }
  unsigned long grid = number(a, [](const Matrix &M) { return (long)M.parts; });
  hipLaunchKernelGGL(momentum_kernel<N>, dim3((unsigned)grid), dim3(256), 0, stream(), a, mu, nesterov);
  grid = number(a, [](const Matrix &M) { return (long)((M.m + 63) / 64) * ((M.n + 63) / 64); });
  hipLaunchKernelGGL(image_kernel<N>, dim3((unsigned)grid), dim3(256), 0, stream(), a, mu, nesterov);
  for (int s = 0; s < steps; s++) {
    product<GRAM, N>(a, s, (float *)rest);
    product<SQUARE, N>(a, s, (float *)rest);
    product<STEP, N>(a, s, (float *)rest, s + 1 == steps);
  }
}

// the images (of a group of matrices), and two pieces a workgroup, or one of a small tile
template <int N>
size_t ws_of(const Matrices<N> &a, size_t images) {
  if (by_block(a)) return 0;
  const int g = tile_size(a, GRAM), s = tile_size(a, STEP), t = g > s ? g : s;  // (SQUARE's: no larger than these)
  return images + sizeof(float) * (t == 0 ? 1024 * SHARERS : 2 * t * t * 256);
}

// `count` matrices of one shape
Matrices<1> alike(long count, long rows, long cols, char *ws) {
  Matrices<1> a = {};
  a.count = (int)(count < ALIKE ? count : ALIKE);
  a.images = (long)images_of(rows, cols);
  lay(a.at[0], rows, cols, ws);
  return a;
}

}  // namespace

extern "C" size_t tt_k_newton_schulz_ws(long count, long rows, long cols) {
  if (count <= 0 || !good_sides(rows, cols)) return 0;
  const Matrices<1> a = alike(count, rows, cols, NULL);
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
  Matrices<1> a = alike(count, rows, cols, (char *)ws);
  const bool blocks = by_block(a);  // (of the last group too, however few are left for it)
  const int most = blocks ? 1 << 20 : a.count;  // without images any number at once
  for (long base = 0; base < count; base += most) {
    a.count = (int)(count - base < most ? count - base : most);
    a.at[0].g = x + base * rows * cols;
    a.at[0].w = y + base * rows * cols;
    run(a, blocks, steps, 0.f, 0, (char *)ws + (size_t)(count < ALIKE ? count : ALIKE) * a.images);
  }
  ttrt_free(own);
  return launched();
}

extern "C" size_t tt_k_muon_multi_ws(const long *rows, const long *cols, int count) {
  if (!rows || !cols || count < 1 || count > TT_SGD_MAX) return 0;
  Matrices<MOST> a = {};
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
  Matrices<MOST> a = {};
  a.count = count;
  char *at = (char *)ws;
  for (int i = 0; i < count; i++) {
    Matrix &M = a.at[i];
    M.g = g[i], M.v = v[i], M.w = w[i];
    M.keep = (float)(1.0 - (double)lr * decay);
    M.rate = (float)(-(double)lr * TT_MUON_RMS * sqrt((double)(rows[i] > cols[i] ? rows[i] : cols[i])));
    lay(M, rows[i], cols[i], at);
  }
  run(a, by_block(a), TT_MUON_STEPS, mu, nesterov, at);
  ttrt_free(own);
  return launched();
}
