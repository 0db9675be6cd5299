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
// fast as the fp32 ones: a value is h + l, two fp16 numbers (l what h leaves), 22
// bits, and h h' + h l' + l h' has all of the product but l l', 2^-22 of it.  The
// rounding of the operands so is 4 times fp32's, and what the sums of these lengths
// leave is of the same size.
//
// fp16 has few exponents: under 2^-17 of the largest value the parts lose bits.  So
// each row of an operand has a scale of its own, a power of two D_i over the norm of
// X's row i, or F_j over its column j's (without them a row 1e7 times weaker than the
// others was off by 2e-3 of itself, and is by 1e-6):
//   G = D^-1 X,  T = F^-1 X^T,  C = G G^T
//   image of P:  C D               (D^-1 P; what the rows of P P are made of)
//   image of Q:  (b C + c (C D)(C D)^T) D     (D^-1 Q)
//   X <- a X + D (image of Q) T^T F
// The polynomial divided by s lies within [0.64, 3.4445], so a row or column grows by
// no more than that a step, and to no more than 1.21: the scales are measured once,
// with `room` for that, 2 at most.  Then the rows of the images have norms under 1,
// 1.21 and 2.82, and times 2^14 their values (46200) are within the type.  After
// MOST_STEPS such steps X begins anew from its fp32 values.
//
// X, X^T, P and Q are kept as images: blocks of 32 x 32 values as the matrix
// instructions take them, four times 1 KB: h of the columns 0 to 15, where lane l
// has eight of row l % 32 from column 8 (l / 32) on, of the columns 16 to 31, and l
// of both; zeros behind the last row and column.  A wave's load is then 1 KB in one
// piece (rows of 128 bytes, 32 of them a load, take the address unit 40 cycles: a
// product of few long rows three times as long).  Both operands of a product are read
// along rows: P = X X^T, P P = P P^T, Q X = Q (X^T)^T.
//
// Matrices of up to 32 rows or columns go another way, in 64 bits (FEW).
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
typedef unsigned short Scale;  // the upper half of a power of two
typedef Scale scale2 __attribute__((ext_vector_type(2)));
typedef Scale scale4 __attribute__((ext_vector_type(4)));

inline hipStream_t stream() { return (hipStream_t)ttrt_stream(); }
inline int launched() { return hipGetLastError() == hipSuccess ? 0 : -3; }

constexpr float UP = 16384.f, DOWN2 = 1.f / (16384.f * 16384.f);
constexpr int MOST = TT_SGD_MAX;   // matrices of different shapes in one run of launches
constexpr int ALIKE = 64;          // of one shape, of up to
constexpr long ALIKE_BYTES = 1L << 32;  // of images
constexpr int NORM_PARTS = 1024;   // sums of squares of a matrix
constexpr int MOST_STEPS = 6;      // with the scales measured before the first
constexpr int FEW = 32;            // up to so many rows
constexpr int FEW_SHORT = 1024, FEW_ALONE = 16384, FEW_PARTS = 64;

__host__ __device__ inline long blocks_of(int k) { return (k + 31) / 32; }

struct Matrix {
  const float *g;   // what is orthogonalised, or the gradient (rows x cols)
  float *v, *w;     // momenta (or NULL) and weights
  char *base;       // the matrix's workspace
  long side, square;  // bytes of an image of X, and of P
  float keep, rate; // w = keep w + rate X where `onto`, else X
  int m, n;         // shorter and longer side
  short turned;     // more rows than columns: X is U^T
  short onto;
  int parts;        // of the norm; of few rows' P
  // Images of G (m rows), of T (n rows; the steps write one from the other), of P and Q.
  __device__ char *x() const { return base; }
  __device__ char *t(int odd) const { return base + side + (odd ? side : 0); }
  __device__ char *p() const { return base + side * 3; }
  __device__ char *q() const { return p() + square; }
  // D and F, of whole blocks
  __device__ Scale *d() const { return (Scale *)(q() + square); }
  __device__ Scale *f() const { return d() + blocks_of(m) * 32; }
  // partial sums of squares, and behind them what X = U times
  __device__ double *norm() const { return (double *)(f() + blocks_of(n) * 32); }
  // and of rows and columns, in 64 of the other: where the second T comes to lie
  __device__ double *of_rows() const { return (double *)t(1); }
  __device__ double *of_cols() const { return of_rows() + (long)(turned ? n : m) * (((turned ? m : n) + 63) / 64); }
  // Of few long rows: parts of P, and behind them T and what X = U times.
  __device__ double *few() const { return (double *)base; }
  __host__ long bytes() const {
    const long all = 3 * side + 2 * square + 64 * (blocks_of(m) + blocks_of(n)) + 8 * (NORM_PARTS + 1);
    return (all + 255) / 256 * 256;
  }
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

// which matrix a workgroup or unit belongs to; b becomes its number among that one's
template <int N>
__device__ __forceinline__ Matrix matrix(const Matrices<N> &a, int i) {
  if (N > 1) return a.at[i];
  Matrix M = a.at[0];
  M.g += (long)i * M.m * M.n, M.w += (long)i * M.m * M.n;
  M.base += i * a.images;
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

// The scales: powers of two, at or over the norms.  (A row of zeros has one that
// sends none to its column's scale, a column of zeros one that sends none to its rows'.)
constexpr float OF_NO_ROW = 2.f, OF_NO_COLUMN = 0x1p-100f;
__device__ __forceinline__ Scale scale_over(float norm, unsigned room, float of_none) {
  const unsigned up = (__float_as_uint(norm) + 0x7fffffu) & 0x7f800000u;
  const float x = norm > 0.f ? fminf(fmaxf(__uint_as_float(up), 0x1p-100f) * __uint_as_float(0x3f800000u + room), 2.f) : of_none;
  return (Scale)(__float_as_uint(x) >> 16);
}
// what a row or column may grow by before the last of such steps, in a float's exponent
inline unsigned room_for(int steps) { return (steps < 6 ? 2u * (steps - 1) : 9u) << 23; }
__device__ __forceinline__ float value_of(Scale scale) { return __uint_as_float((unsigned)scale << 16); }
// 1 / x and 2^14 / x of a power of two
__device__ __forceinline__ float inverse(float x) { return __uint_as_float(0x7f000000u - __float_as_uint(x)); }
__device__ __forceinline__ float inverse_up(float x) { return __uint_as_float(0x86000000u - __float_as_uint(x)); }
// y times a power of two in two parts (multiply-adds, whose results are halves)
__device__ __forceinline__ void split(float y, float scale, _Float16 &h, _Float16 &l) {
  h = (_Float16)fmaf(y, scale, 0.f);
  l = (_Float16)fmaf(y, scale, -(float)h);
}
// where h of row r and column c of a block lies, in bytes (l 2048 further), and of an image
__host__ __device__ __forceinline__ unsigned inner(unsigned r, unsigned c) {
  return (c >> 4) * 1024 + (r + (c >> 3 & 1) * 32) * 16 + (c & 7) * 2;
}
__device__ __forceinline__ _Float16 *place(char *image, long blocks, int r, int c) {
  return (_Float16 *)(image + ((r >> 5) * blocks + (c >> 5)) * 4096 + inner(r & 31, c & 31));
}
// two neighbours of a row, times these
__device__ __forceinline__ void put2(char *p, float x, float y, float sx, float sy) {
  typedef _Float16 half2 __attribute__((ext_vector_type(2)));
  half2 h, l;
  _Float16 a, b;
  split(x, sx, a, b);
  h[0] = a, l[0] = b;
  split(y, sy, a, b);
  h[1] = a, l[1] = b;
  *(half2 *)p = h;
  *(half2 *)(p + 2048) = l;
}
// 16 values, times scale, of row r from column c on, a multiple of 16
__device__ __forceinline__ void put16(char *image, long blocks, int r, int c, const float (&v)[16], float scale) {
  half8 h[2], l[2];
#pragma unroll
  for (int j = 0; j < 16; j++) {
    _Float16 a, b;
    split(v[j], scale, a, b);
    h[j / 8][j % 8] = a;
    l[j / 8][j % 8] = b;
  }
  half8 *p = (half8 *)place(image, blocks, r, c);
  p[0] = h[0], p[32] = h[1], p[128] = l[0], p[160] = l[1];
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

// ---------------------------------------------------------------- few rows
//
// All steps together are a product from the left, X <- T X, and T is made of P alone:
//   P = X X^T;  M = a I + b P + c P P,  T <- M T,  P <- M P M
// (P, M and T have the same eigenvectors, so they are symmetric and their products in
// any order).  With up to FEW rows these are small, and X is read twice, for P and for
// T X.  P has squares of X's values, so it is formed in 64 bits, as are the steps; entries
// of weak rows are as near as any, since P = D C D keeps its form.  What the rounding
// leaves in place of an eigenvalue of 0, of either sign, grows by a a = 12 a step, and
// once negative and large without bounds: after MOST_STEPS (of 2^-36, the most for the
// longest rows, 2^-18) X begins anew from its fp32 values.  (In images a single row
// would have blocks of 32 x 32, and where sums are as short as these the parts' 22 bits
// show: up to 5 times as far off as fp32 products.)
// A workgroup has a matrix of up to FEW_SHORT columns, bound by latency: five steps of 32 x
// 32 take 23 us (1.1 us a step of up to 16 rows, 1.8 of more), of 10 x 785 29, of 32 x
// 1024 49.  Longer ones are cut: parts of P, then one workgroup for the steps, then T X:
// 16 x 100000 48 us, 32 x 2^20 335 (through images 155 and 1150).

typedef double f64x4 __attribute__((ext_vector_type(4)));
constexpr double NS_A = 3.4445, NS_B = -4.7750, NS_C = 2.0315;  // not as fp32 rounds them
static_assert((float)NS_A == TT_NS_A && (float)NS_B == TT_NS_B && (float)NS_C == TT_NS_C, "one polynomial");
constexpr int FEW_COLS = 256, FEW_THREADS = 1024;
struct Few {
  float tile[FEW][FEW_COLS + 1];  // columns of X
  double a[4][FEW][FEW + 2];      // P, M, T, M P; parts of P before
};
// f(k, i, c, at) for this thread's k-th value, row i and column c of X's columns from c0
// on, at `at` of the matrix as it is given; one behind the last column has at < 0.
// Along the memory's rows.
template <class F>
__device__ __forceinline__ void few_values(const Matrix &M, long c0, const F &f) {
#pragma unroll
  for (int k = 0; k < FEW * FEW_COLS / FEW_THREADS; k++) {
    const unsigned x = threadIdx.x + k * FEW_THREADS, m = (unsigned)M.m;
    if (x >= m * FEW_COLS) break;
    const unsigned c = M.turned ? x / m : x % FEW_COLS, i = M.turned ? x - c * m : x / FEW_COLS;
    f(k, i, c, c0 + c < M.n ? (M.turned ? c0 * m + x : (long)i * M.n + c0 + c) : -1l);
  }
}
// U's columns from `from` to `to` (FEW_COLS, or fewer at the end) in the tile for f(c0),
// one after the other, the next on their way meanwhile; `store`: with the momenta.
template <class F>
__device__ __forceinline__ void few_tiles(const Matrix &M, Few &s, long from, long to, float mu, int nesterov, bool store,
                                          const F &f) {
  float u[FEW * FEW_COLS / FEW_THREADS];
  auto load = [&](long c0) {
    few_values(M, c0, [&](int k, unsigned, unsigned, long at) {
      u[k] = at < 0 ? 0.f : momentum<float>(M.g + at, M.v ? M.v + at : nullptr, mu, nesterov, store);
    });
  };
  load(from);
  for (int i = M.m * FEW_COLS + threadIdx.x; i < FEW * FEW_COLS; i += FEW_THREADS) s.tile[i / FEW_COLS][i % FEW_COLS] = 0.f;
  for (long c0 = from; c0 < to; c0 += FEW_COLS) {
    __syncthreads();  // the last columns are read
    few_values(M, c0, [&](int k, unsigned i, unsigned c, long) { s.tile[i][c] = u[k]; });
    __syncthreads();
    if (c0 + FEW_COLS < to) load(c0 + FEW_COLS);
    f(c0);
  }
}
// a[0] = U U^T of the columns from `from` to `to`.  Of 16 waves four have the same 64 of
// the columns, a quarter of the result each (but that above the diagonal).  The
// instruction's lane l holds row l % 16 of either operand and column l / 16 of four, and
// of the result the rows l / 16 + 4 i of column l % 16.
__device__ __forceinline__ void few_gram(const Matrix &M, Few &s, long from, long to, float mu, int nesterov) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, low = lane & 15, high = lane >> 4;
  const int qi = (wave >> 1 & 1) * 16, qj = (wave & 1) * 16, part = wave >> 2;
  const bool on = qj <= qi && qi < M.m;
  f64x4 acc = {};
  few_tiles(M, s, from, to, mu, nesterov, true, [&](long) {
    if (!on) return;
#pragma unroll 4
    for (int k = 0; k < 16; k++) {
      const int c = part * 64 + k * 4 + high;
      acc = __builtin_amdgcn_mfma_f64_16x16x4f64(s.tile[qi + low][c], s.tile[qj + low][c], acc, 0, 0, 0);
    }
  });
#pragma unroll
  for (int i = 0; i < 4; i++) s.a[part][qi + 4 * i + high][qj + low] = acc[i];
  __syncthreads();
  const int r = threadIdx.x >> 5, c = threadIdx.x & 31, i = r < 16 && c >= 16 ? c : r, j = i == r ? c : r;
  const double v = (s.a[0][i][j] + s.a[1][i][j]) + (s.a[2][i][j] + s.a[3][i][j]);
  __syncthreads();
  s.a[0][r][c] = v;
  __syncthreads();
}
// From U U^T in a[0]: T of so many steps to a[2]; what X = U times is returned (`again`:
// 1).  Four waves have a quarter each (one where a quarter is all).
__device__ __forceinline__ double few_steps(const Matrix &M, Few &s, int steps, int again) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, low = lane & 15, high = lane >> 4;
  const int qi = (wave >> 1 & 1) * 16, qj = (wave & 1) * 16, k4 = M.m > 16 ? 8 : 4;
  const bool on = wave < 4 && qi < M.m && qj < M.m;
  double norm = 0.0;
#pragma unroll 8
  for (int i = 0; i < M.m; i++) norm += s.a[0][i][i];
  // zeros stay zeros; an infinity or a NaN makes all of it NaN
  const double over = again ? 1.0 : norm == 0.0 ? 0.0 : norm < __builtin_inf() ? 1.0 / norm : __builtin_nan("");
  __syncthreads();
  s.a[0][threadIdx.x >> 5][threadIdx.x & 31] *= over;
  __syncthreads();
  auto times = [&](int x, int y) {  // (the right one is symmetric)
    f64x4 acc = {};
    if (!on) return acc;
#pragma unroll 4
    for (int k = 0; k < k4; k++)
      acc = __builtin_amdgcn_mfma_f64_16x16x4f64(s.a[x][qi + low][4 * k + high], s.a[y][qj + low][4 * k + high], acc, 0, 0, 0);
    return acc;
  };
  auto put = [&](int x, f64x4 v) {
    if (!on) return;
#pragma unroll
    for (int i = 0; i < 4; i++) s.a[x][qi + 4 * i + high][qj + low] = v[i];
  };
  for (int step = 0; step < steps; step++) {
    f64x4 m = times(0, 0);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int r = qi + 4 * i + high, c = qj + low;
      m[i] = (r == c && r < M.m ? NS_A : 0.0) + NS_B * s.a[0][r][c] + NS_C * m[i];
    }
    put(1, m);
    __syncthreads();
    const bool last = step + 1 == steps;
    const f64x4 t = step ? times(1, 2) : m;
    f64x4 r = {};
    if (!last) r = times(1, 0);
    __syncthreads();
    put(2, t);
    put(3, r);
    __syncthreads();
    if (!last) put(0, times(1, 3));
    __syncthreads();
  }
  return sqrt(over);
}
// w = T X, or onto w, of the columns from `from` to `to`: a wave has 16 of each 256.
__device__ __forceinline__ void few_apply(const Matrix &M, Few &s, long from, long to, double scale, float mu, int nesterov) {
  const int lane = threadIdx.x & 63, low = lane & 15, high = lane >> 4, col = (threadIdx.x >> 6) * 16 + low;
  const int k4 = M.m > 16 ? 8 : 4;
  few_tiles(M, s, from, to, mu, nesterov, false, [&](long c0) {
    f64x4 x[2] = {};
#pragma unroll 4
    for (int k = 0; k < k4; k++) {
      const double u = s.tile[4 * k + high][col];
      x[0] = __builtin_amdgcn_mfma_f64_16x16x4f64(s.a[2][low][4 * k + high], u, x[0], 0, 0, 0);
      if (M.m > 16) x[1] = __builtin_amdgcn_mfma_f64_16x16x4f64(s.a[2][16 + low][4 * k + high], u, x[1], 0, 0, 0);
    }
    // (these columns are this wave's)
#pragma unroll
    for (int i = 0; i < 4; i++) {
      s.tile[4 * i + high][col] = (float)(x[0][i] * scale);
      if (M.m > 16) s.tile[16 + 4 * i + high][col] = (float)(x[1][i] * scale);
    }
    __syncthreads();
    few_values(M, c0, [&](int, unsigned i, unsigned c, long at) {
      if (at >= 0) M.w[at] = M.onto ? M.keep * M.w[at] + M.rate * s.tile[i][c] : s.tile[i][c];
    });
  });
}

template <int N>
__global__ void __launch_bounds__(FEW_THREADS) few_gram_kernel(Matrices<N> a, float mu, int nesterov) {
  __shared__ Few s;
  unsigned b = blockIdx.x;
  const Matrix M = matrix_of(a, b);
  const long tiles = (M.n + FEW_COLS - 1) / FEW_COLS, to = tiles * (b + 1) / M.parts * FEW_COLS;
  few_gram(M, s, tiles * b / M.parts * FEW_COLS, to < M.n ? to : M.n, mu, nesterov);
  M.few()[(long)b * FEW * FEW + threadIdx.x] = s.a[0][threadIdx.x >> 5][threadIdx.x & 31];
}
template <int N>
__global__ void __launch_bounds__(FEW_THREADS) few_steps_kernel(Matrices<N> a, int steps, int again) {
  __shared__ Few s;
  const Matrix M = matrix(a, blockIdx.x);
  double v = 0.0, *at = M.few() + threadIdx.x;
#pragma unroll 16
  for (int b = 0; b < M.parts; b++, at += FEW * FEW) v += *at;
  s.a[0][threadIdx.x >> 5][threadIdx.x & 31] = v;
  __syncthreads();
  const double scale = few_steps(M, s, steps, again);
  *at = s.a[2][threadIdx.x >> 5][threadIdx.x & 31];
  if (threadIdx.x == 0) at[FEW * FEW] = scale;
}
template <int N>
__global__ void __launch_bounds__(FEW_THREADS) few_apply_kernel(Matrices<N> a, float mu, int nesterov) {
  __shared__ Few s;
  unsigned b = blockIdx.x;
  const Matrix M = matrix_of(a, b);
  const double *in = M.few() + (long)M.parts * FEW * FEW;
  s.a[2][threadIdx.x >> 5][threadIdx.x & 31] = in[threadIdx.x];  // (few_tiles waits for it)
  const long from = (long)b * FEW_COLS, to = from + FEW_COLS;
  few_apply(M, s, from, to < M.n ? to : M.n, in[FEW * FEW], mu, nesterov);
}

// ---------------------------------------------------------------- small matrices
//
// A matrix that fits LDS, X and the image of P or Q (which follow each other in one
// place), has a workgroup, which takes it from the gradient to the weights in one
// launch.  A wave has blocks of 32 x 32 of each result, kept in registers until all
// have read what they replace.  X^T is X read by transposing loads.  The products are
// formed transposed: a lane then holds four neighbours of a row, and P and Q are
// symmetric.
// X is an image without scales where it is even: the largest values of its weakest row
// and of its weakest column (zeros aside) have a product of EVEN or more.  The values
// where these two meet are then off by 2^-17 of themselves at most, whole rows and
// columns by less than the sums leave.  Else X are fp32 values, whose parts are made as
// they are read, by rows with their scales for C and by columns with theirs for the
// step; the scales come from the largest value of a row and its length (five steps of
// 64 x 64: 26 us and 32, 500 of 128 x 128 157 and 214).
// Latency bounds it, of LDS and between the products of a chain: five steps of 64 x 64
// take 26 us, of 96 x 96 46, of 64 of 64 x 64 27.

constexpr int BLOCK_WAVES = 16, BLOCK_LDS = 39 * 4096;
constexpr int BLOCK_KEEP = 3;  // blocks of X a wave
constexpr float EVEN = 0x1p-22f;
// X, P and the partial sums of P (four blocks of it: two waves each)
__host__ __device__ inline long block_bytes(int m, int n) {
  const long mb = blocks_of(m), nb = blocks_of(n);
  return 4096 * (mb * nb + mb * mb + (mb == 2 ? 4 : 0));
}
// Of a few matrices those whose products have up to 48 blocks (five steps of 96 x 96:
// 46 us, and 59 by launches of a product each; of 128 x 128 66 and 60), of many all that
// fit (32 of 96 x 300: 86 and 79, 500 of 128 x 128: 157 and 739).
inline bool fits_block(int m, int n, int count) {
  const long mb = blocks_of(m), nb = blocks_of(n);
  return block_bytes(m, n) <= BLOCK_LDS && mb * nb <= BLOCK_WAVES * BLOCK_KEEP && (count >= 32 || mb * mb * nb <= 48);
}

// Chunk (16 bytes) c of a block's eight in row r lies at c ^ (r / 2 % 8), and odd
// rows begin in the other half of the banks: where a row has an even number of
// blocks, neighbouring ones change places there.  No two of the lanes that LDS
// serves at once meet a bank (128 x 128: 71 us with half of them in one).  X has four
// values a chunk, an image in the first four h and in the others l.
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
struct Parts {
  half8 h, l;
};
// eight rows r0 + 8 (lane / 32) .. of column lane % 32 of an image's block
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
__device__ __forceinline__ Parts parts_of(const float (&v)[8], float scale) {
  Parts x;
#pragma unroll
  for (int j = 0; j < 8; j++) {
    _Float16 a, b;
    split(v[j], scale, a, b);
    x.h[j] = a, x.l[j] = b;
  }
  return x;
}
// of X's values: eight columns of row r0 + lane % 32, times scale
__device__ __forceinline__ Parts row_parts(const char *X, int blocks, int r0, int block, int half, float scale, int lane) {
  float v[8];
#pragma unroll
  for (int x = 0; x < 2; x++) {
    const f32x4 w = *(const f32x4 *)chunk_of(X, blocks, r0 + (lane & 31), block, half * 4 + (lane >> 5) * 2 + x);
#pragma unroll
    for (int j = 0; j < 4; j++) v[x * 4 + j] = w[j];
  }
  return parts_of(v, scale);
}
// eight rows r0 + 8 (lane / 32) .. of column lane % 32 of a block, times scale
__device__ __forceinline__ Parts column_parts(const char *X, int blocks, int r0, int block, float scale, int lane) {
  float v[8];
#pragma unroll
  for (int x = 0; x < 8; x++)
    v[x] = *(const float *)(chunk_of(X, blocks, r0 + (lane >> 5) * 8 + x, block, lane >> 2 & 7) + (lane & 3) * 4);
  return parts_of(v, scale);
}
__device__ __forceinline__ void three(f32x16 &acc, half8 ha, half8 la, half8 hb, half8 lb) {
  acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(la, hb, acc, 0, 0, 0);
  acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(ha, lb, acc, 0, 0, 0);
  acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(ha, hb, acc, 0, 0, 0);
}
// four values of row r from column c on: of X's values, and of an image (times 2^-14) and
// back, times these
__device__ __forceinline__ f32x4 *x4(char *X, int blocks, int r, int c) {
  return (f32x4 *)const_cast<char *>(chunk_of(X, blocks, r, c >> 5, c >> 2 & 7));
}
__device__ __forceinline__ f32x4 get4(const char *image, int blocks, int r, int c) {
  typedef _Float16 half4 __attribute__((ext_vector_type(4)));
  const half4 h = *(const half4 *)(chunk_of(image, blocks, r, c >> 5, c >> 3 & 3) + (c & 4) * 2);
  const half4 l = *(const half4 *)(chunk_of(image, blocks, r, c >> 5, 4 + (c >> 3 & 3)) + (c & 4) * 2);
  f32x4 v;
#pragma unroll
  for (int j = 0; j < 4; j++) v[j] = ((float)h[j] + (float)l[j]) * (1.f / UP);
  return v;
}
__device__ __forceinline__ void put4(char *image, int blocks, int r, int c, f32x4 v, f32x4 scale) {
  typedef _Float16 half4 __attribute__((ext_vector_type(4)));
  half4 h, l;
#pragma unroll
  for (int j = 0; j < 4; j++) {
    _Float16 a, b;
    split(v[j], scale[j], a, b);
    h[j] = a, l[j] = b;
  }
  *(half4 *)(chunk_of(image, blocks, r, c >> 5, c >> 3 & 3) + (c & 4) * 2) = h;
  *(half4 *)(chunk_of(image, blocks, r, c >> 5, 4 + (c >> 3 & 3)) + (c & 4) * 2) = l;
}

// The steps of X in LDS and the result to w; VALUES: X are fp32 values, else an image.
template <bool VALUES>
__device__ __forceinline__ void steps_in_lds(const Matrix &M, int steps, char *lds, const Scale *scales, int lane, int wave) {
  const int mb = (int)blocks_of(M.m), nb = (int)blocks_of(M.n);
  char *const X = lds, *const P = lds + mb * nb * 4096, *const rest = P + mb * mb * 4096;
  for (int step = 0;; step++) {
    __syncthreads();
    // the lane as the compiler does not know it from step to step: it would keep every
    // address of the loop in registers, and spill them
    asm volatile("" : "+v"(lane));
    auto of_row = [&](int r) { return VALUES ? value_of(scales[r]) : 1.f; };
    auto of_rows = [&](int r) {  // four of them
      if (!VALUES) return (f32x4){1.f, 1.f, 1.f, 1.f};
      const scale4 x = *(const scale4 *)(scales + r);
      return (f32x4){value_of(x[0]), value_of(x[1]), value_of(x[2]), value_of(x[3])};
    };
    const int low = lane & 31, high = (lane >> 5) * 4;  // result i: values high + 8 (i / 4) + i % 4 of row low
    // C = G G^T: with four blocks of it two waves share the sum
    const int pb = mb * mb, ways = mb == 2 ? 2 : 1;
    f32x4 c4[4];
    {
      const int f = wave % pb, way = wave / pb, ra = f / mb * 32, rb = f % mb * 32;
      f32x16 acc = {};
      if (way < ways) {
        const float da = inverse_up(of_row(ra + low)), db = inverse_up(of_row(rb + low));
#pragma unroll 1
        for (int k = way; k < nb; k += ways)
#pragma unroll
          for (int h = 0; h < 2; h++) {
            if constexpr (VALUES) {
              const Parts x = row_parts(X, nb, ra, k, h, da, lane);
              Parts y = x;
              if (ra != rb) y = row_parts(X, nb, rb, k, h, db, lane);
              three(acc, x.h, x.l, y.h, y.l);
            } else {
              three(acc, along(X, nb, ra, k, h, 0, lane), along(X, nb, ra, k, h, 1, lane), along(X, nb, rb, k, h, 0, lane),
                    along(X, nb, rb, k, h, 1, lane));
            }
          }
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
          c4[i] = (f32x4){acc[i * 4], acc[i * 4 + 1], acc[i * 4 + 2], acc[i * 4 + 3]} * DOWN2;
          put4(P, mb, rb + low, ra + high + 8 * i, c4[i], of_rows(ra + high + 8 * i) * UP);
        }
      }
    }
    __syncthreads();
    {  // the image of Q, in P's place
      const bool on = wave < pb;
      const int f = on ? wave : 0, ra = f / mb * 32, rb = f % mb * 32;
      f32x16 acc = {};
      if (on) {
#pragma unroll 1
        for (int k = 0; k < mb; k++)
#pragma unroll
          for (int h = 0; h < 2; h++)
            three(acc, along(P, mb, ra, k, h, 0, lane), along(P, mb, ra, k, h, 1, lane), along(P, mb, rb, k, h, 0, lane),
                  along(P, mb, rb, k, h, 1, lane));
      }
      __syncthreads();
      if (on) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const f32x4 v = {acc[i * 4], acc[i * 4 + 1], acc[i * 4 + 2], acc[i * 4 + 3]};
          const f32x4 q = c4[i] * TT_NS_B + v * (TT_NS_C * DOWN2);
          put4(P, mb, rb + low, ra + high + 8 * i, q, of_rows(ra + high + 8 * i) * UP);
        }
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
      const float column = inverse_up(of_row(mb * 32 + cb * 32 + low)), row = of_row(r0 + low) * DOWN2;
#pragma unroll 1
      for (int k = 0; k < mb; k++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
          Parts x;
          if constexpr (VALUES) x = column_parts(X, nb, k * 32 + h * 16, cb, column, lane);
          else x.h = across(X, nb, k * 32 + h * 16, cb, 0, lane), x.l = across(X, nb, k * 32 + h * 16, cb, 1, lane);
          three(acc[b], x.h, x.l, along(P, mb, r0, k, h, 0, lane), along(P, mb, r0, k, h, 1, lane));
        }
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int c = cb * 32 + high + 8 * i;
        const f32x4 v = (VALUES ? *x4(X, nb, r0 + low, c) : get4(X, nb, r0 + low, c)) * TT_NS_A;
        const f32x4 columns = of_rows(mb * 32 + c);
#pragma unroll
        for (int j = 0; j < 4; j++) acc[b][i * 4 + j] = v[j] + acc[b][i * 4 + j] * row * columns[j];
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
          *w = M.onto ? M.keep * *w + M.rate * acc[b][i] : acc[b][i];
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
      for (int i = 0; i < 4; i++) {
        const f32x4 v = {acc[b][i * 4], acc[b][i * 4 + 1], acc[b][i * 4 + 2], acc[b][i * 4 + 3]};
        const int r = f / nb * 32 + low, c = f % nb * 32 + high + 8 * i;
        if (VALUES) *x4(X, nb, r, c) = v;
        else put4(X, nb, r, c, v, (f32x4){UP, UP, UP, UP});
      }
    }
  }
}

// `again`: X is what is given, without its norm.
template <int N>
__global__ void __launch_bounds__(BLOCK_WAVES * 64)
    block_kernel(Matrices<N> a, int steps, float mu, int nesterov, int again, unsigned room) {
  __shared__ __attribute__((aligned(1024))) char lds[BLOCK_LDS];
  __shared__ Scale scales[(4 + 15) * 32];  // of 4 blocks of rows and 15 of columns
  __shared__ double sums[BLOCK_WAVES];
  __shared__ float least[2][BLOCK_WAVES];
  const Matrix M = matrix(a, blockIdx.x);
  if (M.m <= FEW) {
    Few &few = *(Few *)lds;
    few_gram(M, few, 0, M.n, mu, nesterov);
    const double times = few_steps(M, few, steps, again);
    few_apply(M, few, 0, M.n, times, mu, nesterov);
    return;
  }
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int mb = (int)blocks_of(M.m), nb = (int)blocks_of(M.n), count = M.m * M.n, cols = M.turned ? M.m : M.n;
  char *const X = lds;
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
  const double scale = again ? 1.0 : s == 0.0 ? 0.0 : 1.0 / sqrt(s);  // zeros stay zeros
  auto place1 = [&](int i, float u) {
    const int r = i / cols, c = i % cols, row = M.turned ? c : r, col = M.turned ? r : c;
    ((float *)x4(X, nb, row, col & ~3))[col & 3] = (float)((double)u * scale);
  };
  for (int i = threadIdx.x * 4; i + 4 <= count; i += THREADS * 4) {  // what this thread wrote itself
    const f32x4 u = momentum<f32x4_any>(M.g + i, M.v ? M.v + i : nullptr, mu, nesterov, false);
#pragma unroll
    for (int j = 0; j < 4; j++) place1(i + j, u[j]);
  }
  if (tail < count) place1(tail, momentum<float>(M.g + tail, M.v ? M.v + tail : nullptr, mu, nesterov, false));
  __syncthreads();
  // the scales, a wave a row, then a thread a column, and the least value of either
  // (zeros aside)
  {
    const float long_row = sqrtf((float)M.n), long_column = sqrtf((float)M.m);
    float less[2] = {1.f, 1.f};
    for (int r = wave; r < mb * 32; r += BLOCK_WAVES) {
      float most = 0.f;
      for (int c = lane; c < nb * 8; c += 64) {
        const f32x4 v = *x4(X, nb, r, c * 4);
#pragma unroll
        for (int j = 0; j < 4; j++) most = fmaxf(most, fabsf(v[j]));
      }
#pragma unroll
      for (int k = 1; k < 64; k <<= 1) most = fmaxf(most, __shfl_xor(most, k));
      if (lane == 0) scales[r] = scale_over(most * long_row, room, OF_NO_ROW);
      if (most > 0.f) less[0] = fminf(less[0], most);
    }
    if ((int)threadIdx.x < nb * 32) {
      float most = 0.f;
#pragma unroll 8
      for (int r = 0; r < mb * 32; r++) most = fmaxf(most, fabsf(((const float *)x4(X, nb, r, threadIdx.x & ~3))[threadIdx.x & 3]));
      scales[mb * 32 + threadIdx.x] = scale_over(most * long_column, room, OF_NO_COLUMN);
      if (most > 0.f) less[1] = fminf(less[1], most);
    }
#pragma unroll
    for (int k = 1; k < 64; k <<= 1) less[1] = fminf(less[1], __shfl_xor(less[1], k));
    if (lane == 0) least[0][wave] = less[0], least[1][wave] = less[1];
  }
  f32x4 x[BLOCK_KEEP][4];  // of this wave's blocks
  const int low = lane & 31, high = (lane >> 5) * 4;
#pragma unroll
  for (int b = 0; b < BLOCK_KEEP; b++) {
    const int f = wave + b * BLOCK_WAVES;
    if (f >= mb * nb) continue;
#pragma unroll
    for (int i = 0; i < 4; i++) x[b][i] = *x4(X, nb, f / nb * 32 + low, f % nb * 32 + high + 8 * i);
  }
  __syncthreads();
  float row = 1.f, column = 1.f;
#pragma unroll
  for (int k = 0; k < BLOCK_WAVES; k++) row = fminf(row, least[0][k]), column = fminf(column, least[1][k]);
  if (row * column < EVEN) {
    steps_in_lds<true>(M, steps, lds, scales, lane, wave);
    return;
  }
#pragma unroll
  for (int b = 0; b < BLOCK_KEEP; b++) {
    const int f = wave + b * BLOCK_WAVES;
    if (f >= mb * nb) continue;
#pragma unroll
    for (int i = 0; i < 4; i++)
      put4(X, nb, f / nb * 32 + low, f % nb * 32 + high + 8 * i, x[b][i], (f32x4){UP, UP, UP, UP});
  }
  steps_in_lds<false>(M, steps, lds, scales, lane, wave);
}

// ---------------------------------------------------------------- before the steps

// x of the lane N further on, round its sixteen
template <int N>
__device__ __forceinline__ double turned_by(double x) {
  union {
    double d;
    int i[2];
  } v = {x};
#pragma unroll
  for (int k = 0; k < 2; k++) v.i[k] = __builtin_amdgcn_update_dpp(0, v.i[k], 0x120 + N, 15, 15, false);
  return v.d;
}

// v = mu v + g, and the sums of squares of u = g + mu v (nesterov) or v (without
// momenta of g), in all and of the rows and columns of each tile of 64 x 64.  In 64
// bits: the squares of any fp32 values are within its range.  Bound by memory: 29 us for
// a block's weights of 12.6 million values (5.2 TB/s).
template <int N>
__global__ void __launch_bounds__(256) momentum_kernel(Matrices<N> a, float mu, int nesterov) {
  __shared__ double down[16][64];
  unsigned b = blockIdx.x;
  const Matrix M = matrix_of(a, b);
  const int rows = M.turned ? M.n : M.m, cols = M.turned ? M.m : M.n, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const unsigned nc = (unsigned)((cols + 63) / 64), tiles = (unsigned)((rows + 63) / 64) * nc;
  double all = 0.0;
  for (unsigned tile = b; tile < tiles; tile += M.parts) {
    // lane l has four columns from 4 (l % 16) on of every fourth row
    const int ti = (int)(tile / nc), tj = (int)(tile % nc), c = tj * 64 + (lane & 15) * 4;
    f32x4 u[4];
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const int r = ti * 64 + wave * 16 + k * 4 + (lane >> 4);
      u[k] = (f32x4){0.f, 0.f, 0.f, 0.f};
      const long at = (long)r * cols + c;
      if (r < rows && c + 4 <= cols) {
        u[k] = momentum<f32x4_any>(M.g + at, M.v ? M.v + at : nullptr, mu, nesterov, true);
      } else if (r < rows) {
#pragma unroll
        for (int j = 0; j < 3; j++)
          if (c + j < cols) u[k][j] = momentum<float>(M.g + at + j, M.v ? M.v + at + j : nullptr, mu, nesterov, true);
      }
    }
    double column[4] = {};
#pragma unroll
    for (int k = 0; k < 4; k++) {
      double row = 0.0;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const double q = (double)u[k][j] * (double)u[k][j];
        row += q;
        column[j] += q;
      }
      row += turned_by<8>(row);
      row += turned_by<4>(row);
      row += turned_by<2>(row);
      row += turned_by<1>(row);
      const int r = ti * 64 + wave * 16 + k * 4 + (lane >> 4);
      if ((lane & 15) == 0 && r < rows) M.of_rows()[(long)tj * rows + r] = row;
    }
    __syncthreads();  // the last tile's are read
#pragma unroll
    for (int j = 0; j < 4; j++) down[wave * 4 + (lane >> 4)][(lane & 15) * 4 + j] = column[j];
    __syncthreads();
    if (threadIdx.x < 64) {
      double q = 0.0;
#pragma unroll
      for (int k = 0; k < 16; k++) q += down[k][lane];
      if (tj * 64 + lane < cols) M.of_cols()[(long)ti * cols + tj * 64 + lane] = q;
      all += q;
    }
  }
  if (wave == 0) {
#pragma unroll
    for (int k = 1; k < 64; k <<= 1) all += __shfl_xor(all, k);
    if (lane == 0) M.norm()[b] = all;
  }
}

// Up to this length the scales are formed with the images (785 x 256 with two smaller
// ones: a launch of 4 us less; for 40 x 70001 the launch takes 5).
constexpr int MEASURE = 1024;

// X = U times this; `again`: X is what is given
__device__ __forceinline__ double scale_of(double norm, int again) {
  return again ? 1.0 : norm == 0.0 ? 0.0 : 1.0 / sqrt(norm);  // zeros stay zeros
}

// The scales of X's rows, and of its columns, where they are formed from more than
// MEASURE / 64 parts: 16 of them a workgroup, 16 or 64 threads each, in a fixed order.
// 7 us for a block's weights, 5 for 4096 x 4096.
template <int N>
__global__ void __launch_bounds__(1024) scale_kernel(Matrices<N> a, int again, unsigned room) {
  __shared__ double sums[16][16], norms[16];
  unsigned b = blockIdx.x;
  const Matrix M = matrix_of(a, b);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const unsigned of_x = 2 * (unsigned)blocks_of(M.m);  // workgroups for X's rows; the others have its columns
  const bool down = b >= of_x;
  const int i = (int)(down ? b - of_x : b) * 16 + (lane & 15), many = down ? M.n : M.m, other = down ? M.m : M.n;
  const double *part = down != (bool)M.turned ? M.of_cols() : M.of_rows();
  double norm = 0.0, s = 0.0;
  for (int k = threadIdx.x; k < M.parts; k += blockDim.x) norm += M.norm()[k];
  if (i < many) {
#pragma unroll 8
    for (int k = threadIdx.x >> 4; k < (other + 63) / 64; k += blockDim.x >> 4) s += part[(long)k * many + i];
  }
#pragma unroll
  for (int k = 1; k < 64; k <<= 1) norm += __shfl_xor(norm, k);
  s += __shfl_xor(s, 16);
  s += __shfl_xor(s, 32);
  if (lane == 0) norms[wave] = norm;
  if (lane < 16) sums[wave][lane] = s;
  __syncthreads();
  if (threadIdx.x >= 16) return;
  norm = s = 0.0;
  for (unsigned k = 0; k < blockDim.x >> 6; k++) norm += norms[k], s += sums[k][lane];
  const double scale = scale_of(norm, again);
  (down ? M.f() : M.d())[i] = scale_over(i < many ? (float)(sqrt(s) * scale) : 0.f, room, down ? OF_NO_COLUMN : OF_NO_ROW);
  if (b == 0 && lane == 0) M.norm()[NORM_PARTS] = scale;
}

// The images of G and T, a tile of 64 x 64 at a time through LDS; both are written
// along their rows.  `keep`: X goes to w as well.  The other scales are formed here, by
// every tile of the same rows or columns again, and written by the first.  Bound by
// memory: 35 us for 4096 x 4096 (5.7 TB/s).
template <int N>
__global__ void __launch_bounds__(256) image_kernel(Matrices<N> a, float mu, int nesterov, int again, int keep, unsigned room) {
  __shared__ float tile[64][65];
  __shared__ double norms[2];
  __shared__ Scale scales[2][64];
  unsigned b = blockIdx.x;
  const Matrix M = matrix_of(a, b);
  const int rows = M.turned ? M.n : M.m, cols = M.turned ? M.m : M.n, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const unsigned across = (unsigned)((cols + 63) / 64);
  const int r0 = (int)(b / across) * 64, c0 = (int)(b % across) * 64;
  Scale *of_rows = M.turned ? M.f() : M.d(), *of_cols = M.turned ? M.d() : M.f();
  float u[16];  // on their way while the scales are formed
#pragma unroll
  for (int k = 0; k < 16; k++) {
    const int r = r0 + k * 4 + wave, c = c0 + lane;
    u[k] = 0.f;
    if (r < rows && c < cols) {
      const long at = (long)r * cols + c;
      u[k] = momentum<float>(M.g + at, M.v ? M.v + at : nullptr, mu, nesterov, false);
    }
  }
  // waves 0 and 1: the rows' and the columns' sums of squares; 2 and 3: that of all
  const int i = (wave ? c0 : r0) + lane, many = wave ? cols : rows, other = wave ? rows : cols;
  const bool total = M.n <= MEASURE, here = wave < 2 && other <= MEASURE;
  double s = 0.0;
  if (here && i < many) {
    const double *part = (wave ? M.of_cols() : M.of_rows()) + i;
    double q[MEASURE / 64];  // on their way at once
#pragma unroll
    for (int k = 0; k < MEASURE / 64; k++) q[k] = k < (other + 63) / 64 ? part[(long)k * many] : 0.0;
#pragma unroll
    for (int k = 0; k < MEASURE / 64; k++) s += q[k];
  } else if (wave >= 2 && total) {
#pragma unroll 2
    for (int k = threadIdx.x - 128; k < M.parts; k += 128) s += M.norm()[k];
#pragma unroll
    for (int k = 1; k < 64; k <<= 1) s += __shfl_xor(s, k);
    if (lane == 0) norms[wave - 2] = s;
  }
  if (total) __syncthreads();
  const double scale = total ? scale_of(norms[0] + norms[1], again) : M.norm()[NORM_PARTS];
  if (wave < 2 && i < blocks_of(many) * 32) {
    Scale *of = wave ? of_cols : of_rows;
    Scale x = 0;
    if (here) {
      x = scale_over((float)(sqrt(s) * scale), room, (bool)wave != (bool)M.turned ? OF_NO_COLUMN : OF_NO_ROW);
      if ((wave ? r0 : c0) == 0) of[i] = x;
    } else {
      x = of[i];
    }
    scales[wave][lane] = x;
  }
#pragma unroll
  for (int k = 0; k < 16; k++) {
    const int r = r0 + k * 4 + wave, c = c0 + lane;
    u[k] = (float)((double)u[k] * scale);
    if (keep && r < rows && c < cols) M.w[(long)r * cols + c] = u[k];
    tile[k * 4 + wave][lane] = u[k];
  }
  __syncthreads();
  char *along = M.turned ? M.t(0) : M.x(), *down = M.turned ? M.x() : M.t(0);
  const long row_blocks = blocks_of(cols), col_blocks = blocks_of(rows);
  const int line = threadIdx.x >> 2, from = (threadIdx.x & 3) * 16;  // 16 values of a row, then of a column
  float v[16];
  if ((r0 + line) / 32 < col_blocks && (c0 + from) / 32 < row_blocks) {
    const float by = inverse_up(value_of(scales[0][line]));
#pragma unroll
    for (int j = 0; j < 16; j++) v[j] = tile[line][from + j];
    put16(along, row_blocks, r0 + line, c0 + from, v, by);
  }
  if ((c0 + line) / 32 < row_blocks && (r0 + from) / 32 < col_blocks) {
    const float by = inverse_up(value_of(scales[1][line]));
#pragma unroll
    for (int j = 0; j < 16; j++) v[j] = tile[from + j][line];
    put16(down, col_blocks, c0 + line, r0 + from, v, by);
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

// A step's parity, and whether what X adds comes from w (`onto`, of the last)
struct Phase {
  int odd, from_w;
};

template <int KIND>
struct Operands {
  const char *a, *b;    // images whose rows are multiplied
  const char *add;      // what is added, in the image of the transpose (GRAM: none)
  const char *plain;    // and in its own
  char *out, *down;     // images of the result and its transpose
  const Scale *d, *f;   // scales of the result's rows and columns
  int rows, cols, k;    // of the result; the products' length
  float by, times;
  __device__ __forceinline__ Operands(const Matrix &M, const Phase &phase) {
    d = M.d(), f = KIND <= SQUARE ? M.d() : M.f();
    if (KIND == GRAM) {
      a = b = M.x(), add = plain = nullptr, out = down = M.p();
      rows = cols = M.m, k = M.n, by = DOWN2, times = 0.f;
    } else if (KIND == SQUARE) {
      a = b = add = plain = M.p(), out = down = M.q();
      rows = cols = k = M.m, by = TT_NS_C * DOWN2, times = TT_NS_B;
    } else {
      a = M.q(), b = add = M.t(phase.odd), plain = M.x(), out = M.x(), down = M.t(!phase.odd);
      rows = k = M.m, cols = M.n, by = DOWN2, times = TT_NS_A;
    }
  }
  // What is added, of values h + l of its own image or the transpose's: X is in the
  // image of its rows without d and in that of its columns without f, C in both with the
  // other's.  Either way a row weaker than the column has it finer in its own image, and
  // a column weaker than the row in the transpose's.  One of them is read as it comes;
  // X, whose weak values grow, from the other where that is finer by more than 4 (a
  // column's of rows longer than 200000 beside 2, the most a scale may be), C by 32.
  static constexpr float FAR = KIND == STEP ? 4.f : 32.f;
  __device__ __forceinline__ float plain_scale(float d, float f) const { return times / UP * (KIND == STEP ? d : inverse(f)); }
  __device__ __forceinline__ float add_scale(float d, float f) const { return times / UP * (KIND == STEP ? f : inverse(d)); }
  // The products' sum (C, and Q without its scales, are as the sums are), and what is
  // added.  (Multiply-adds take the halves as they are.)
  __device__ __forceinline__ float of_sum(float sum, float d, float f) const {
    return KIND == STEP ? sum * (by * f) * d : sum * by;
  }
  __device__ __forceinline__ static float add_to(float sum, _Float16 h, _Float16 l, float scale) {
    return fmaf((float)h, scale, fmaf((float)l, scale, sum));
  }
  // what the images have it times
  __device__ __forceinline__ static float out_scale(float d, float f) { return KIND == STEP ? inverse_up(d) : UP * f; }
  __device__ __forceinline__ static float down_scale(float d, float f) { return KIND == STEP ? inverse_up(f) : UP * d; }
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
// 517 x 1003: 6 us for P, 5 for Q, 11 for X; 1024 x 1024: 11, 12 and 16 (400 TFLOP/s
// of fp16 products).  Of few long tiles of P the length is shared by `ways` workgroups,
// whose sums a second launch adds (join): one CU alone reads 80 GB/s.
template <int KIND, bool SHARED, int N>
__global__ void __launch_bounds__(512, 2)
    small_kernel(Matrices<N> a, Phase phase, int to_w, int ways, bool join, float *pieces) {
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
  const Operands<KIND> o(M, phase);
  int ti, tj;
  tile_of<KIND, 32>(t, o.rows, o.cols, ti, tj);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = threadIdx.x >> 4, c = (threadIdx.x & 15) * 2;  // this thread's two results
  // where these lie in the tile's block of an image, and (their transposes') in the
  // transpose's; their scales, and the transposes'
  const unsigned at = inner(r, c);
  const long block = ((long)ti * blocks_of(o.cols) + tj) * 4096, across = ((long)tj * blocks_of(o.rows) + ti) * 4096;
  const Scale *rows = o.d + ti * 32, *cols = o.f + tj * 32;
  const Scale d = rows[(unsigned)r], df = cols[(unsigned)r];
  const scale2 f = *(const scale2 *)(cols + (unsigned)c), dd = *(const scale2 *)(rows + (unsigned)c);
  half2 h = {}, l = {};
  if (KIND != GRAM && !(KIND == STEP && phase.from_w)) {
    const char *p = o.plain + block;
    h = *(const half2 *)(p + at), l = *(const half2 *)(p + 2048 + at);
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
  float v[2];
#pragma unroll
  for (int e = 0; e < 2; e++) {
    const float x = value_of(d), y = value_of(f[e]);
    in[e] = ti * 32 + r < o.rows && tj * 32 + c + e < o.cols;
    const float product = o.of_sum(sum[e], x, y);
    v[e] = KIND == GRAM ? product : o.add_to(product, h[e], l[e], o.plain_scale(x, y));
    if (KIND != GRAM && !phase.from_w && in[e] && x > o.FAR * y) {
      const _Float16 *p = (const _Float16 *)(o.add + across + inner(c + e, r));
      v[e] = o.add_to(product, p[0], p[1024], o.add_scale(x, y));
    }
    if (!in[e]) v[e] = 0.f;
  }
  if (KIND == STEP && to_w) {
#pragma unroll
    for (int e = 0; e < 2; e++)
      if (in[e] && !M.turned) {
        float *w = M.w + (long)(ti * 32 + r) * o.cols + tj * 32 + c + e;
        *w = M.onto ? M.keep * *w + M.rate * v[e] : v[e];
      }
  } else {
    char *p = o.out + block;
    put2(p + at, v[0], v[1], o.out_scale(value_of(d), value_of(f[0])), o.out_scale(value_of(d), value_of(f[1])));
  }
  if ((KIND <= SQUARE && ti == tj) || (KIND == STEP && to_w && !M.turned)) return;
  __syncthreads();
  sums[0][r][c] = v[0];
  sums[0][r][c + 1] = v[1];
  __syncthreads();
  if (KIND == STEP && to_w) {
#pragma unroll
    for (int e = 0; e < 2; e++)
      if (tj * 32 + r < o.cols && ti * 32 + c + e < o.rows) {
        float *w = M.w + (long)(tj * 32 + r) * o.rows + ti * 32 + c + e;
        *w = M.onto ? M.keep * *w + M.rate * sums[0][c + e][r] : sums[0][c + e][r];
      }
  } else {
    char *p = o.down + across;
    put2(p + at, sums[0][c][r], sums[0][c + 1][r], o.down_scale(value_of(dd[0]), value_of(df)),
         o.down_scale(value_of(dd[1]), value_of(df)));
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
// leave: X of 4096 x 4096 takes 351 us, 1170 TFLOP/s of fp16 products, with the units
// 68 % busy at 1.82 GHz; of 2048 x 2048 by tiles of 128 54 us, 950 TFLOP/s (46 % busy
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
  scale4 d[4];  // scales of the rows and of the column
  Scale f;
};
__device__ __forceinline__ int part_of(int i, int lane) {  // in the block of the transpose, bytes
  return (i >> 1) * 1024 + ((lane & 31) + 32 * (i & 1)) * 16 + (lane >> 5) * 8;
}
template <int KIND>
__device__ __forceinline__ Added added(const Operands<KIND> &o, int r0, int c0, int lane, bool from_w,
                                       const Added *of_rows = nullptr) {  // (what has the same rows)
  Added x = {};
  if (of_rows) {
#pragma unroll
    for (int i = 0; i < 4; i++) x.d[i] = of_rows->d[i];
  }
  if (r0 >= o.rows || c0 >= o.cols || (KIND <= SQUARE && r0 < c0)) return x;
#pragma unroll
  for (int i = 0; i < 4; i++)
    if (!of_rows) x.d[i] = *(const scale4 *)(o.d + r0 + (lane >> 5) * 4 + 8 * i);
  x.f = o.f[c0 + (lane & 31)];
  if (KIND == GRAM || (KIND == STEP && from_w)) return x;
  const char *p = o.add + ((c0 >> 5) * blocks_of(o.rows) + (r0 >> 5)) * 4096;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    x.h[i] = *(const half4 *)(p + part_of(i, lane));
    x.l[i] = *(const half4 *)(p + part_of(i, lane) + 2048);
  }
  return x;
}
// buf: 4 KB of LDS, this wave's.  Of a symmetric result the blocks behind the diagonal
// are left to those before it.
template <int KIND>
__device__ __forceinline__ void write32(const Matrix &M, const Operands<KIND> &o, const f32x16 &acc, const Added &x,
                                        int r0, int c0, char *buf, int lane, const Phase &phase, bool to_w) {
  if (r0 >= o.rows || c0 >= o.cols || (KIND <= SQUARE && r0 < c0)) return;
  const bool both = KIND == STEP || r0 != c0;
  const int col = c0 + (lane & 31), row = r0 + (lane >> 5) * 4;
  f32x4 v[4];
  const float f = value_of(x.f);
  Scale least = x.d[0][0];
#pragma unroll
  for (int i = 0; i < 16; i++) {
    const float d = value_of(x.d[i / 4][i % 4]);
    const float product = o.of_sum(acc[i], d, f);
    v[i / 4][i % 4] = KIND == GRAM ? product : o.add_to(product, x.h[i / 4][i % 4], x.l[i / 4][i % 4], o.add_scale(d, f));
    least = x.d[i / 4][i % 4] < least ? x.d[i / 4][i % 4] : least;
  }
  if (KIND != GRAM && !phase.from_w && __any(col < o.cols && f > o.FAR * value_of(least))) {
    // by way of LDS, each lane its own: sixteen reads in line were a third of the kernel's code
    typedef _Float16 half2 __attribute__((ext_vector_type(2)));
    half2 *mine = (half2 *)buf + lane;
#pragma unroll 1
    for (int i = 0; i < 16; i++) {
      const _Float16 *p = place((char *)o.plain, blocks_of(o.cols), row + 8 * (i >> 2) + (i & 3), col);
      half2 w = {};
      if (col < o.cols) w[0] = p[0], w[1] = p[1024];
      mine[i * 64] = w;
    }
#pragma unroll
    for (int i = 0; i < 16; i++) {
      const float d = value_of(x.d[i / 4][i % 4]);
      const half2 w = mine[i * 64];
      if (f > o.FAR * d) v[i / 4][i % 4] = o.add_to(o.of_sum(acc[i], d, f), w[0], w[1], o.plain_scale(d, f));
    }
  }
  if (KIND == STEP && to_w) {
    // (as values of their own: the compiler would read `rate` with its neighbours as a
    // vector, for that put M into LDS, and fetch the launch's packet from the host's
    // memory to find its place there: 10 us a launch)
    float rate = M.rate, keep = M.keep;
    asm("" : "+s"(rate), "+s"(keep));
    // what is read is on its way at once: behind the last row or column, theirs
    const int c = col < o.cols ? col : o.cols - 1;
    if (M.turned && r0 + 32 <= o.rows) {
      float *w = M.w + (long)c * o.rows + row;
      f32x4 old[4] = {};
#pragma unroll
      for (int i = 0; i < 4; i++)
        if (M.onto) old[i] = *(const f32x4_any *)(w + 8 * i) * keep;
#pragma unroll
      for (int i = 0; i < 4; i++)
        if (col < o.cols) *(f32x4_any *)(w + 8 * i) = M.onto ? old[i] + v[i] * rate : v[i];
      return;
    }
    const long down = M.turned ? 1 : o.cols, start = M.turned ? (long)c * o.rows : c;
    float old[16] = {};
#pragma unroll
    for (int i = 0; i < 16; i++) {
      const int r = row + 8 * (i / 4) + i % 4;
      if (M.onto) old[i] = M.w[start + (r < o.rows ? r : o.rows - 1) * down] * keep;
    }
#pragma unroll
    for (int i = 0; i < 16; i++) {
      const int r = row + 8 * (i / 4) + i % 4;
      if (col < o.cols && r < o.rows) M.w[start + r * down] = M.onto ? old[i] + v[i / 4][i % 4] * rate : v[i / 4][i % 4];
    }
    return;
  }
  char *down = o.down + ((c0 >> 5) * blocks_of(o.rows) + (r0 >> 5)) * 4096;
  auto put = [&](char *at, int i, bool out) {
    half4 h, l;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const float d = value_of(x.d[i][j]);
      _Float16 a, b;
      split(v[i][j], out ? o.out_scale(d, f) : o.down_scale(d, f), a, b);
      h[j] = a, l[j] = b;
    }
    *(half4 *)(at + part_of(i, lane)) = h;
    *(half4 *)(at + part_of(i, lane) + 2048) = l;
  };
#pragma unroll
  for (int i = 0; i < 4; i++) {
    put(down, i, false);
    if (both) put(buf, i, true);
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

// g of every number from F on (a loop of this length the compiler does not unroll, and
// registers have no other numbers)
template <int F>
struct Number {
  static constexpr int value = F;
};
template <int F, int END, class G>
__device__ __forceinline__ void each(const G &g) {
  if constexpr (F < END) {
    g(Number<F>());
    each<F + 1, END>(g);
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
__global__ void __launch_bounds__((Shape<T, BUFFERS>::WAVES * 64), (Shape<T, BUFFERS>::WAVES / 4)) tile_kernel(Matrices<N> a, Phase phase, int to_w, Deal deal, float *pieces) {
  typedef Shape<T, BUFFERS> S;
  __shared__ __attribute__((aligned(1024))) char lds[BUFFERS * S::BUFFER];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned groups = gridDim.x, w = dealt(blockIdx.x, groups);
  const unsigned to = lds_address(lds);
  unsigned round = 0;
  for (unsigned long u = 0, end = 0;;) {
    if (u == end) {
      if (round < deal.rounds) {  // then all tiles have the same number of blocks
        const Operands<KIND> o(a.at[0], phase);
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
    const Operands<KIND> o(M, phase);
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
      Added x = added<KIND>(o, row_of<T>(ti, wave, 0), col_of<T>(tj, wave, 0), lane, phase.from_w), next = x;
      each<0, S::BLOCKS>([&](auto number) __attribute__((always_inline)) {
        constexpr int f = decltype(number)::value;
        if constexpr (f + 1 < S::BLOCKS)
          next = added<KIND>(o, row_of<T>(ti, wave, f + 1), col_of<T>(tj, wave, f + 1), lane, phase.from_w,
                             f % 2 == 0 ? &x : nullptr);
        write32<KIND>(M, o, acc[f / 2][f % 2], x, row_of<T>(ti, wave, f), col_of<T>(tj, wave, f), lds + wave * 4096, lane,
                      phase, to_w);
        x = next;
      });
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
__global__ void __launch_bounds__(256) join_kernel(Matrices<N> a, Phase phase, int to_w, Deal deal, const float *pieces) {
  typedef Shape<T, 2> S;
  __shared__ __attribute__((aligned(1024))) char buf[4][4096];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned w = blockIdx.x + 1;
  const unsigned long u = deal.begins(w);
  unsigned long in = u;
  const Matrix M = matrix_of(a, in);
  const Operands<KIND> o(M, phase);
  const unsigned extra = N > 1 ? deal.extra : 0;
  const unsigned long units = blocks_of(o.k) + extra, first = u - in % units, last = first + units;
  if (u <= first + extra || deal.begins(w - 1) > first + extra) return;
  int ti, tj;
  tile_of<KIND, T>(in / units, o.rows, o.cols, ti, tj);
  const int block = blockIdx.y * 4 + wave;
  const int r0 = row_of<T>(ti, block / S::BLOCKS, block % S::BLOCKS), c0 = col_of<T>(tj, block / S::BLOCKS, block % S::BLOCKS);
  const Added x = added<KIND>(o, r0, c0, lane, phase.from_w);
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
  write32<KIND>(M, o, acc, x, r0, c0, buf[wave], lane, phase, to_w);
}

// ---------------------------------------------------------------- host

bool good_sides(long rows, long cols) {
  return rows > 0 && cols > 0 && rows <= TT_MUON_MAX_SIDE && cols <= TT_MUON_MAX_SIDE && rows * cols <= TT_MUON_MAX_VALUES;
}

void lay(Matrix &M, long rows, long cols, bool few, char *&ws) {
  M.turned = rows > cols;
  M.m = (int)(M.turned ? cols : rows);
  M.n = (int)(M.turned ? rows : cols);
  const long tiles = (long)((M.m + 63) / 64) * ((M.n + 63) / 64);
  M.parts = (int)(tiles < NORM_PARTS ? tiles : NORM_PARTS);
  if (few) {
    const long few_tiles = (M.n + FEW_COLS - 1) / FEW_COLS;
    M.parts = (int)(few_tiles < FEW_PARTS ? few_tiles : FEW_PARTS);
  }
  M.side = 4096 * blocks_of(M.m) * blocks_of(M.n);
  M.square = 4096 * blocks_of(M.m) * blocks_of(M.m);
  M.base = ws;
  ws += few ? 8l * FEW * FEW * (M.parts + 1) + 256 : M.bytes();
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

// How a matrix goes: by itself in a workgroup, as one of few long rows, or by products.
enum Way { IN_LDS, FEW_LONG, PRODUCTS };
// those of one way; `ways` of each
Matrices<MOST> of_way(const Matrices<MOST> &a, const Way *ways, Way way) {
  Matrices<MOST> some = {};
  for (int i = 0; i < a.count; i++)
    if (ways[i] == way) some.at[some.count++] = a.at[i];
  return some;
}
// of many of one shape
Way way_of(int m, int n, int count) {
  if (m <= FEW) return n <= FEW_SHORT ? IN_LDS : FEW_LONG;
  return fits_block(m, n, count) ? IN_LDS : PRODUCTS;
}
// Of a list's: matrices of few rows cost next to nothing in the launches that others
// need anyway (129 x 10 beside 785 x 256 and 257 x 128: 99 us, 115 by itself), but for the
// longest, whose blocks are mostly empty (1 x 2^20: 196 us, 1020 by products).
void ways_of(const Matrices<MOST> &a, Way *ways) {
  bool products = false;
  for (int i = 0; i < a.count; i++) {
    ways[i] = way_of(a.at[i].m, a.at[i].n, a.count);
    products = products || ways[i] == PRODUCTS;
  }
  for (int i = 0; i < a.count && products; i++)
    if (a.at[i].m > FEW || a.at[i].n <= FEW_ALONE) ways[i] = PRODUCTS;
}

// blocks of a product's length
long length_of(int kind, const Matrix &M) { return blocks_of(kind == GRAM ? M.n : M.m); }

// How a product of such matrices goes: by tiles of 32 (0), 128 or 256, by its work, m m
// and its length, in all of them.  Of a symmetric result half is computed, and smaller
// tiles are used for longer: they have less to compute twice, and their parts are joined
// sooner.  But few tiles of 128 (136 of 2048 rows), or tiles of different lengths, are
// cut into parts that are not in step, so that each XCD reads all of it from afar (two of
// 4096^2, 1024 x 4096 and its turn: 9590 us with tiles of 256, 10080 with 128).  us of a
// product, with what joins its parts:
//                      P = X X^T            X <- a X + Q X
//   tiles of         32   128   256        32   128   256
//   1024^2           11    18     -        16    24     -
//   700 x 4000       20    21     -        28    25     -
//   2 x 1024^2       18    20     -        29    30     -
//   1400^2           20    23     -        38    30     -
//   1600^2           27    28     -        50    45     -
//   1024 x 4096      34    31     -        51    32     -
//   2048^2            -    41    56         -    54    78
//   2500^2            -    76    83         -   124   126
//   2048 x 4096       -    75    75         -   103   120
//   2200 x 6300       -   110   122         -   209   202
//   3000 x 5000       -   152   160         -   313   262
//   2048 x 8192       -   156   120         -   202   197
//   2100 x 12000      -   204   201         -   387   354
//   4096^2            -   203   218         -   394   353
//   4096 x 8192       -   386   392         -   804   693
//   6000^2            -   615   591         -  1377  1113
//   8192^2            -  1542  1379         -  3573  2619
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
void small_product(Matrices<N> &a, const Phase &phase, int to_w, float *pieces) {
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
                           stream(), a, phase, to_w, (int)ways, join, pieces);
      return;
    }
  }
  hipLaunchKernelGGL((small_kernel<KIND, false, N>), dim3(grid), dim3(512), 0, stream(), a, phase, to_w, 1, false, pieces);
}

template <int KIND, int T, int BUFFERS, int N>
void tile_product(Matrices<N> &a, const Phase &phase, int to_w, float *pieces) {
  typedef Shape<T, BUFFERS> S;
  constexpr int EXTRA = T == 128 ? 12 : 6;  // (2375 x 1041 with five: 651 us with 4, 603 with 8, 590 with 12)
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
  hipLaunchKernelGGL((tile_kernel<KIND, T, BUFFERS, N>), dim3(groups), dim3(S::WAVES * 64), 0, stream(), a, phase, to_w, d, pieces);
  if (d.sharers > 1)
    hipLaunchKernelGGL((join_kernel<KIND, T, N>), dim3(d.sharers - 1, S::PIECE / 4096), dim3(256), 0, stream(), a, phase, to_w, d,
                       (const float *)pieces);
}

template <int KIND, int N>
void product(Matrices<N> &a, const Phase &phase, float *pieces, int to_w = 0) {
  const int tile = tile_size(a, KIND);
  if (tile == 0) small_product<KIND, N>(a, phase, to_w, pieces);
  else if (tile == 128) tile_product<KIND, 128, 3, N>(a, phase, to_w, pieces);
  else tile_product<KIND, 256, 2, N>(a, phase, to_w, pieces);
}

// Steps of matrices that a workgroup has, MOST_STEPS at most; `again`: of X that is given.
template <int N>
void run_in_lds(const Matrices<N> &a, int steps, float mu, int nesterov, int again = 0) {
  if (a.count)
    hipLaunchKernelGGL(block_kernel<N>, dim3(a.count), dim3(BLOCK_WAVES * 64), 0, stream(), a, steps, mu, nesterov, again,
                       room_for(steps));
}

// The same of matrices of few long rows.
template <int N>
void run_few(Matrices<N> &a, int steps, float mu, int nesterov, int again = 0) {
  if (!a.count) return;
  unsigned long grid = number(a, [](const Matrix &M) { return (long)M.parts; });
  hipLaunchKernelGGL(few_gram_kernel<N>, dim3((unsigned)grid), dim3(FEW_THREADS), 0, stream(), a, mu, nesterov);
  hipLaunchKernelGGL(few_steps_kernel<N>, dim3(a.count), dim3(FEW_THREADS), 0, stream(), a, steps, again);
  grid = number(a, [](const Matrix &M) { return (long)((M.n + FEW_COLS - 1) / FEW_COLS); });
  hipLaunchKernelGGL(few_apply_kernel<N>, dim3((unsigned)grid), dim3(FEW_THREADS), 0, stream(), a, mu, nesterov);
}

// Steps with the scales measured before the first, MOST_STEPS at most; `again`: of X
// that is given.  `keep`: X goes to w, and the last step takes a X from there.
template <int N>
void run(Matrices<N> &a, int steps, float mu, int nesterov, char *rest, int again = 0, int keep = 0) {
  unsigned long grid = number(a, [](const Matrix &M) { return (long)M.parts; });
  hipLaunchKernelGGL(momentum_kernel<N>, dim3((unsigned)grid), dim3(256), 0, stream(), a, mu, nesterov);
  grid = number(a, [](const Matrix &M) {
    return (M.n > MEASURE ? 2 * blocks_of(M.m) : 0) + (M.m > MEASURE ? 2 * blocks_of(M.n) : 0);
  });
  if (grid) {
    int longest = 0;
    for (int i = 0; i < (N > 1 ? a.count : 1); i++) longest = a.at[i].n > longest ? a.at[i].n : longest;
    // (64 threads a row and 16: 40 x 70001 5 us and 9, four of 4096 x 4096 16 us and 9)
    hipLaunchKernelGGL(scale_kernel<N>, dim3((unsigned)grid), dim3(longest > 16384 ? 1024 : 256), 0, stream(), a, again,
                       room_for(steps));
  }
  grid = number(a, [](const Matrix &M) { return (long)((M.m + 63) / 64) * ((M.n + 63) / 64); });
  hipLaunchKernelGGL(image_kernel<N>, dim3((unsigned)grid), dim3(256), 0, stream(), a, mu, nesterov, again, keep && !again,
                     room_for(steps));
  for (int s = 0; s < steps; s++) {
    const bool last = s + 1 == steps;
    Phase phase = {s & 1, 0};
    product<GRAM, N>(a, phase, (float *)rest);
    product<SQUARE, N>(a, phase, (float *)rest);
    phase.from_w = last && keep;
    product<STEP, N>(a, phase, (float *)rest, last);
  }
}

// two pieces a workgroup, or one of a small tile
template <int N>
size_t pieces_of(const Matrices<N> &a) {
  const int g = tile_size(a, GRAM), s = tile_size(a, STEP), t = g > s ? g : s;  // (SQUARE's: no larger than these)
  return sizeof(float) * (t == 0 ? 1024 * SHARERS : 2 * t * t * 256);
}

// A list's matrices and their ways, laid into a workspace but for those that need none;
// what follows them (pieces) is left at ws.  The bytes of all.
size_t lay_all(Matrices<MOST> &a, Way *ways, const long *rows, const long *cols, int count, char *&ws) {
  char *const start = ws;
  a.count = count;
  for (int i = 0; i < count; i++) {
    char *none = NULL;
    lay(a.at[i], rows[i], cols[i], false, none);
  }
  ways_of(a, ways);
  bool products = false;
  for (int i = 0; i < count; i++) {
    if (ways[i] != IN_LDS) lay(a.at[i], rows[i], cols[i], ways[i] == FEW_LONG, ws);
    products = products || ways[i] == PRODUCTS;
  }
  return (size_t)(ws - start) + (products ? pieces_of(of_way(a, ways, PRODUCTS)) : 0);
}

// As many of `count` matrices of one shape as go together (blocks are of 32 x 32, so a
// flat matrix's images are many times as large as it: 33 x 2^20 has 8 GB)
Matrices<1> alike(long count, long rows, long cols, char *ws, Way &way) {
  Matrices<1> a = {};
  const int m = (int)(rows < cols ? rows : cols), n = (int)(rows < cols ? cols : rows);
  way = way_of(m, n, (int)(count < ALIKE ? count : ALIKE));
  char *end = ws;
  lay(a.at[0], rows, cols, way == FEW_LONG, end);
  a.images = end - ws;
  const long fit = ALIKE_BYTES / a.images < 1 ? 1 : ALIKE_BYTES / a.images;
  const long most = way == IN_LDS ? 1 << 20 : fit < ALIKE ? fit : ALIKE;  // (in LDS any number at once)
  a.count = (int)(count < most ? count : most);
  return a;
}

}  // namespace

extern "C" size_t tt_k_newton_schulz_ws(long count, long rows, long cols) {
  if (count <= 0 || !good_sides(rows, cols)) return 0;
  Way way;
  const Matrices<1> a = alike(count, rows, cols, NULL, way);
  return way == IN_LDS ? 0 : a.count * (size_t)a.images + (way == PRODUCTS ? pieces_of(a) : 0);
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
  Way way;  // (of the last group too, however few are left for it)
  Matrices<1> a = alike(count, rows, cols, (char *)ws, way);
  const int most = a.count;
  char *const rest = way == PRODUCTS ? (char *)ws + most * a.images : NULL;
  // More steps than the scales or few rows' 64 bits hold for go on from y.  By products then each begins anew
  // and adds to y: what is weak by its row and its column, and so in every image, is
  // carried in fp32 (60 x 500 with 1e-7 of half of both: a column's 3e-6 after 16 steps,
  // 2e-4 from images of six).  In LDS such an X is fp32 throughout.
  const int keep = way == PRODUCTS && steps > MOST_STEPS;
  const int each = keep ? 1 : MOST_STEPS;
  a.at[0].onto = keep, a.at[0].keep = TT_NS_A, a.at[0].rate = 1.f;
  for (long base = 0; base < count; base += most) {
    a.count = (int)(count - base < most ? count - base : most);
    a.at[0].g = x + base * rows * cols;
    a.at[0].w = y + base * rows * cols;
    for (int done = 0; done < steps; done += each) {
      const int n = steps - done < each ? steps - done : each;
      if (way == IN_LDS) run_in_lds(a, n, 0.f, 0, done > 0);
      else if (way == FEW_LONG) run_few(a, n, 0.f, 0, done > 0);
      else run(a, n, 0.f, 0, rest, done > 0, keep);
      a.at[0].g = a.at[0].w;
    }
  }
  ttrt_free(own);
  return launched();
}

extern "C" size_t tt_k_muon_multi_ws(const long *rows, const long *cols, int count) {
  if (!rows || !cols || count < 1 || count > TT_SGD_MAX) return 0;
  for (int i = 0; i < count; i++)
    if (!good_sides(rows[i], cols[i])) return 0;
  Matrices<MOST> a = {};
  Way ways[MOST];
  char *at = NULL;
  return lay_all(a, ways, rows, cols, count, at);
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
  Way ways[MOST];
  char *at = (char *)ws;
  lay_all(a, ways, rows, cols, count, at);
  for (int i = 0; i < count; i++) {
    Matrix &M = a.at[i];
    M.g = g[i], M.v = v[i], M.w = w[i], M.onto = 1;
    M.keep = (float)(1.0 - (double)lr * decay);
    M.rate = (float)(-(double)lr * TT_MUON_RMS * sqrt((double)(rows[i] > cols[i] ? rows[i] : cols[i])));
  }
  Matrices<MOST> few = of_way(a, ways, FEW_LONG), products = of_way(a, ways, PRODUCTS);
  run_in_lds(of_way(a, ways, IN_LDS), TT_MUON_STEPS, mu, nesterov);
  run_few(few, TT_MUON_STEPS, mu, nesterov);
  if (products.count) run(products, TT_MUON_STEPS, mu, nesterov, at);
  ttrt_free(own);
  return launched();
}
