// Layer norm over the last axis, forward and backward (HBM roofline: the
// forward pass reads x and writes y, the backward pass reads x and dy and
// writes dx).
//
//   y = h w + b, h = (x - mean) rstd;  with g = dy w over a row of C values
//   dx = rstd (g - mean(g) - h mean(g h));  dw = sum_rows dy h, db = sum_rows dy
//
// A row is held in registers by the NT threads that share it, so memory sees
// each value once and the variance is that of the deviations (two sums over
// the registers; one pass with sums of squares would cancel).  All sums are
// fp32, over a thread's values and then in a fixed tree.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>
#include "tt_rt.h"

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
// in memory: 16-byte accesses need no more than a float's alignment here, so
// rows of any length and place take them
typedef f32x4 __attribute__((aligned(4))) f32x4_any;

inline hipStream_t stream() { return (hipStream_t)ttrt_stream(); }
inline int launched() { return hipGetLastError() == hipSuccess ? 0 : -3; }

__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) x += __shfl_xor(x, s);
  return x;
}

// sums of two values over the NT threads of a row; every thread gets them
template <int NT>
__device__ __forceinline__ void row_sum2(float &x, float &y, float (*part)[2]) {
  x = wave_sum(x);
  y = wave_sum(y);
  if (NT == 64) return;
  const int wave = threadIdx.x >> 6;
  __syncthreads();  // the last sums are read
  if ((threadIdx.x & 63) == 0) {
    part[wave][0] = x;
    part[wave][1] = y;
  }
  __syncthreads();
  x = y = 0.f;
#pragma unroll
  for (int w = 0; w < NT / 64; w++) {
    x += part[w][0];
    y += part[w][1];
  }
}

// Group n of a thread's values: the four columns from this one on.
template <int NT>
__device__ __forceinline__ int col_of(int n, int t) {
  return (n * NT + t) * 4;
}

// With TAIL (cols not a multiple of 4, and more than 4) the groups at and behind
// the row's end are its last four columns, of which a thread's own are those that
// no other has: every load is one instruction with no branch around it, so none
// waits for the one before (4725 rows of 2555 columns, backward with the sums:
// 75 us with the last columns loaded one by one, 38 so, 35 for 2556 columns).
template <int NT, int NV, bool TAIL>
struct Groups {
  int at[NV], cols, t;
  __device__ __forceinline__ Groups(int cols_, int t_) : cols(cols_), t(t_) {
#pragma unroll
    for (int n = 0; n < NV; n++) {
      const int c = col_of<NT>(n, t);
      at[n] = TAIL && c > cols - 4 ? cols - 4 : c;
    }
  }
  __device__ __forceinline__ bool own(int n, int j) const {
    return TAIL ? j >= col_of<NT>(n, t) - at[n] : col_of<NT>(n, t) < cols;
  }
  __device__ __forceinline__ void load(f32x4 (&v)[NV], const float *p) const {
#pragma unroll
    for (int n = 0; n < NV; n++) {
      v[n] = (f32x4){0.f, 0.f, 0.f, 0.f};
      if (TAIL || col_of<NT>(n, t) < cols) v[n] = *(const f32x4_any *)(p + at[n]);
    }
  }
  __device__ __forceinline__ void mask(f32x4 (&v)[NV]) const {
    if (!TAIL) return;
#pragma unroll
    for (int n = 0; n < NV; n++)
#pragma unroll
      for (int j = 0; j < 4; j++) v[n][j] = own(n, j) ? v[n][j] : 0.f;
  }
  __device__ __forceinline__ void store(const f32x4 (&v)[NV], float *p) const {
#pragma unroll
    for (int n = 0; n < NV; n++) {
      if (own(n, 0)) {
        *(f32x4_any *)(p + at[n]) = v[n];
      } else if (TAIL) {
#pragma unroll
        for (int j = 1; j < 4; j++)
          if (own(n, j)) p[at[n] + j] = v[n][j];
      }
    }
  }
};

constexpr int threads_of(int nt) { return nt < 256 ? 256 : nt; }

template <int NT, int NV, bool TAIL>
__global__ void __launch_bounds__(threads_of(NT))
    ln_fwd_kernel(const float *__restrict__ x, const float *__restrict__ w, const float *__restrict__ b,
                  float *__restrict__ y, float *__restrict__ mean, float *__restrict__ rstd, long rows, int cols,
                  float eps) {
  constexpr int RB = threads_of(NT) / NT;  // rows a workgroup
  __shared__ float part[NT / 64][2];
  const int t = threadIdx.x % NT, sub = __builtin_amdgcn_readfirstlane(threadIdx.x / NT);
  const Groups<NT, NV, TAIL> gr(cols, t);
  for (long row = (long)blockIdx.x * RB + sub; row < rows; row += (long)gridDim.x * RB) {
    f32x4 v[NV];
    gr.load(v, x + row * cols);
    gr.mask(v);
    float s = 0.f, z = 0.f;
#pragma unroll
    for (int n = 0; n < NV; n++) s += (v[n][0] + v[n][1]) + (v[n][2] + v[n][3]);
    row_sum2<NT>(s, z, part);
    const float mu = s / (float)cols;
    float q = 0.f;
#pragma unroll
    for (int n = 0; n < NV; n++)
#pragma unroll
      for (int j = 0; j < 4; j++) {
        v[n][j] -= mu;
        if (gr.own(n, j)) q = fmaf(v[n][j], v[n][j], q);
      }
    z = 0.f;
    row_sum2<NT>(q, z, part);
    const float r = 1.f / sqrtf(q / (float)cols + eps);
    f32x4 g[NV], o[NV];
    if (w) gr.load(g, w);
    if (b) gr.load(o, b);
#pragma unroll
    for (int n = 0; n < NV; n++)
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const float h = v[n][j] * r;
        v[n][j] = fmaf(h, w ? g[n][j] : 1.f, b ? o[n][j] : 0.f);
      }
    gr.store(v, y + row * cols);
    if (t == 0) {
      if (mean) mean[row] = mu;
      if (rstd) rstd[row] = r;
    }
  }
}

// dx, and (part) this workgroup's sums over its rows for dw and db: part[block][2][cols]
template <int NT, int NV, bool TAIL>
__global__ void __launch_bounds__(threads_of(NT))
    ln_bwd_kernel(const float *__restrict__ x, const float *__restrict__ w, const float *__restrict__ dy,
                  const float *__restrict__ mean, const float *__restrict__ rstd, float *__restrict__ dx,
                  float *__restrict__ part, long rows, int cols) {
  constexpr int RB = threads_of(NT) / NT;
  __shared__ float red[NT / 64][2];
  __shared__ __attribute__((aligned(16))) float join[RB > 1 ? RB * NT * 4 : 4];
  const int t = threadIdx.x % NT, sub = __builtin_amdgcn_readfirstlane(threadIdx.x / NT);
  const Groups<NT, NV, TAIL> gr(cols, t);
  f32x4 aw[NV], ab[NV];
#pragma unroll
  for (int n = 0; n < NV; n++) aw[n] = ab[n] = (f32x4){0.f, 0.f, 0.f, 0.f};
  for (long row = (long)blockIdx.x * RB + sub; row < rows; row += (long)gridDim.x * RB) {
    f32x4 v[NV], d[NV];
    gr.load(v, x + row * cols);
    gr.load(d, dy + row * cols);
    const float mu = mean[row], r = rstd[row];
    f32x4 g[NV];
    if (w) gr.load(g, w);
    gr.mask(v);
    gr.mask(d);
    if (w) gr.mask(g);  // an infinite weight times 0 would count
    float s = 0.f, q = 0.f;
#pragma unroll
    for (int n = 0; n < NV; n++)
#pragma unroll
      for (int j = 0; j < 4; j++) {
        v[n][j] = (v[n][j] - mu) * r;  // where not its own: dy is 0, so nothing counts
        aw[n][j] = fmaf(d[n][j], v[n][j], aw[n][j]);
        ab[n][j] += d[n][j];
        if (w) d[n][j] *= g[n][j];
        s += d[n][j];
        q = fmaf(d[n][j], v[n][j], q);
      }
    row_sum2<NT>(s, q, red);
    s /= (float)cols;
    q /= (float)cols;
    if (dx) {
#pragma unroll
      for (int n = 0; n < NV; n++)
#pragma unroll
        for (int j = 0; j < 4; j++) v[n][j] = r * (d[n][j] - s - v[n][j] * q);
      gr.store(v, dx + row * cols);
    }
  }
  if (!part) return;
  float *out = part + (long)blockIdx.x * 2 * cols;
#pragma unroll
  for (int n = 0; n < NV; n++) {
#pragma unroll
    for (int p = 0; p < 2; p++) {
      f32x4 a = p ? ab[n] : aw[n];
      if (RB > 1) {  // the workgroup's rows, in order
        __syncthreads();
        *(f32x4 *)(join + threadIdx.x * 4) = a;
        __syncthreads();
        if (threadIdx.x >= NT) continue;
#pragma unroll
        for (int k = 1; k < RB; k++) a += *(const f32x4 *)(join + (k * NT + t) * 4);
      }
#pragma unroll
      for (int j = 0; j < 4; j++)
        if (gr.own(n, j)) out[(long)p * cols + gr.at[n] + j] = a[j];
    }
  }
}

// dw / db from the workgroups' sums: 16 columns a workgroup, 64 threads a
// column, each every 64th of them, then in a fixed tree.  Latency-bound (4 MB
// at 1024 columns): a thread's reads do not wait for each other.
__global__ void __launch_bounds__(1024)
    ln_join_kernel(const float *__restrict__ part, float *__restrict__ dw, float *__restrict__ db, int blocks,
                   long cols) {
  __shared__ float sum[16][16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  float *out = blockIdx.y ? db : dw;
  if (!out) return;
  for (long c0 = (long)blockIdx.x * 16; c0 < cols; c0 += (long)gridDim.x * 16) {
    const long c = c0 + (lane & 15);
    float s = 0.f;
    if (c < cols) {
#pragma unroll 8
      for (int k = threadIdx.x >> 4; k < blocks; k += 64) s += part[((long)k * 2 + blockIdx.y) * cols + c];
    }
    s += __shfl_xor(s, 16);
    s += __shfl_xor(s, 32);
    if (lane < 16) sum[wave][lane] = s;
    __syncthreads();
    if (threadIdx.x < 16 && c < cols) {
      s = 0.f;
#pragma unroll
      for (int k = 0; k < 16; k++) s += sum[k][lane];
      out[c] = s;
    }
    __syncthreads();
  }
}

// rows too long for registers (or shorter than a group): read again for each sum
__global__ void __launch_bounds__(1024)
    ln_fwd_long_kernel(const float *__restrict__ x, const float *__restrict__ w, const float *__restrict__ b,
                       float *__restrict__ y, float *__restrict__ mean, float *__restrict__ rstd, long rows,
                       long cols, float eps) {
  __shared__ float part[16][2];
  for (long row = blockIdx.x; row < rows; row += gridDim.x) {
    const float *p = x + row * cols;
    float s = 0.f, z = 0.f;
    for (long c = threadIdx.x; c < cols; c += 1024) s += p[c];
    row_sum2<1024>(s, z, part);
    const float mu = s / (float)cols;
    float q = 0.f;
    for (long c = threadIdx.x; c < cols; c += 1024) q = fmaf(p[c] - mu, p[c] - mu, q);
    z = 0.f;
    row_sum2<1024>(q, z, part);
    const float r = 1.f / sqrtf(q / (float)cols + eps);
    for (long c = threadIdx.x; c < cols; c += 1024)
      y[row * cols + c] = fmaf((p[c] - mu) * r, w ? w[c] : 1.f, b ? b[c] : 0.f);
    if (threadIdx.x == 0) {
      if (mean) mean[row] = mu;
      if (rstd) rstd[row] = r;
    }
  }
}

__global__ void __launch_bounds__(1024)
    ln_dx_long_kernel(const float *__restrict__ x, const float *__restrict__ w, const float *__restrict__ dy,
                      const float *__restrict__ mean, const float *__restrict__ rstd, float *__restrict__ dx,
                      long rows, long cols) {
  __shared__ float part[16][2];
  for (long row = blockIdx.x; row < rows; row += gridDim.x) {
    const float *p = x + row * cols, *d = dy + row * cols;
    const float mu = mean[row], r = rstd[row];
    float s = 0.f, q = 0.f;
    for (long c = threadIdx.x; c < cols; c += 1024) {
      const float g = w ? d[c] * w[c] : d[c];
      s += g;
      q = fmaf(g, (p[c] - mu) * r, q);
    }
    row_sum2<1024>(s, q, part);
    s /= (float)cols;
    q /= (float)cols;
    for (long c = threadIdx.x; c < cols; c += 1024) {
      const float g = w ? d[c] * w[c] : d[c];
      dx[row * cols + c] = r * (g - s - (p[c] - mu) * r * q);
    }
  }
}

// part[blockIdx.y][2][cols]: the sums for dw and db over a run of rows
__global__ void __launch_bounds__(256)
    ln_cols_long_kernel(const float *__restrict__ x, const float *__restrict__ dy, const float *__restrict__ mean,
                        const float *__restrict__ rstd, float *__restrict__ part, long rows, long cols) {
  const long c = (long)blockIdx.x * 256 + threadIdx.x;
  if (c >= cols) return;
  float sw = 0.f, sb = 0.f;
  for (long row = blockIdx.y; row < rows; row += gridDim.y) {
    const float d = dy[row * cols + c];
    sw = fmaf(d, (x[row * cols + c] - mean[row]) * rstd[row], sw);
    sb += d;
  }
  part[((long)blockIdx.y * 2) * cols + c] = sw;
  part[((long)blockIdx.y * 2 + 1) * cols + c] = sb;
}

// columns that 1024 threads hold 16 each of; and rows without a whole group
bool long_rows(long cols) { return cols > 16384 || cols < 4; }

// threads of a row and float4 a thread
#define BY_COLS(RUN)              \
  if (cols <= 256) {              \
    RUN(64, 1);                   \
  } else if (cols <= 512) {       \
    RUN(64, 2);                   \
  } else if (cols <= 1024) {      \
    RUN(64, 4);                   \
  } else if (cols <= 2048) {      \
    RUN(256, 2);                  \
  } else if (cols <= 4096) {      \
    RUN(256, 4);                  \
  } else if (cols <= 8192) {      \
    RUN(1024, 2);                 \
  } else {                        \
    RUN(1024, 4);                 \
  }

int rows_a_group(long cols) { return cols <= 1024 ? 4 : 1; }

// Workgroups of the backward pass, each with sums of its own: two a CU of 256
// threads, one of 1024, and two row groups at least for each; a few more of them
// where that saves a pass (4099 rows of 1003 columns: 20.1 -> 19.0 us).
int bwd_blocks(long rows, long cols) {
  if (long_rows(cols)) {  // few columns leave few threads, so more runs of rows
    const long runs = cols < 4 ? 2048 : 64;
    return (int)(rows < runs ? rows : runs);
  }
  const long groups = (rows + rows_a_group(cols) - 1) / rows_a_group(cols), most = cols <= 4096 ? 512 : 256;
  const long each = groups < 2 * most ? 2 : groups / most;
  return (int)((groups + each - 1) / each);
}

bool good(long rows, long cols) { return rows > 0 && cols > 0 && cols <= 1L << 30 && rows <= (1L << 40) / cols; }

}  // namespace

extern "C" int tt_k_layernorm_fwd(const float *x, const float *w, const float *b, float *y, float *mean,
                                  float *rstd, long rows, long cols, float eps) {
  if (!x || !y || !good(rows, cols) || !(eps >= 0.f) || isinf(eps)) return -1;
  if (ttrt_init() != 0) return -3;
  if (long_rows(cols)) {
    hipLaunchKernelGGL(ln_fwd_long_kernel, dim3((unsigned)(rows < 65536 ? rows : 65536)), dim3(1024), 0, stream(),
                       x, w, b, y, mean, rstd, rows, cols, eps);
    return launched();
  }
  const long groups = (rows + rows_a_group(cols) - 1) / rows_a_group(cols);
  const unsigned grid = (unsigned)(groups < 1 << 20 ? groups : 1 << 20);
#define RUN(NT, NV)                                                                                            \
  if (cols % 4 == 0)                                                                                                    \
    hipLaunchKernelGGL((ln_fwd_kernel<NT, NV, false>), dim3(grid), dim3(threads_of(NT)), 0, stream(), x, w, b, y, \
                       mean, rstd, rows, (int)cols, eps);                                                      \
  else                                                                                                         \
    hipLaunchKernelGGL((ln_fwd_kernel<NT, NV, true>), dim3(grid), dim3(threads_of(NT)), 0, stream(), x, w, b, y, \
                       mean, rstd, rows, (int)cols, eps)
  BY_COLS(RUN)
#undef RUN
  return launched();
}

extern "C" size_t tt_k_layernorm_bwd_ws(long rows, long cols) {
  return good(rows, cols) ? sizeof(float) * 2 * (size_t)cols * bwd_blocks(rows, cols) : 0;
}

extern "C" int tt_k_layernorm_bwd(const float *x, const float *w, const float *dy, const float *mean,
                                  const float *rstd, float *dx, float *dw, float *db, long rows, long cols,
                                  void *ws) {
  if (!x || !dy || !mean || !rstd || !good(rows, cols)) return -1;
  if (!dx && !dw && !db) return 0;
  if (ttrt_init() != 0) return -3;
  const int blocks = bwd_blocks(rows, cols);
  float *own = NULL, *part = NULL;
  if (dw || db) {
    part = (float *)ws;
    if (!part) part = own = (float *)ttrt_alloc(tt_k_layernorm_bwd_ws(rows, cols));
    if (!part) return -2;
  }
  if (long_rows(cols)) {
    if (dx)
      hipLaunchKernelGGL(ln_dx_long_kernel, dim3((unsigned)(rows < 65536 ? rows : 65536)), dim3(1024), 0, stream(),
                         x, w, dy, mean, rstd, dx, rows, cols);
    if (part)
      hipLaunchKernelGGL(ln_cols_long_kernel, dim3((unsigned)((cols + 255) / 256), (unsigned)blocks), dim3(256), 0,
                         stream(), x, dy, mean, rstd, part, rows, cols);
  } else {
    // without sums every row group has a workgroup of its own
    const long groups = (rows + rows_a_group(cols) - 1) / rows_a_group(cols);
    const unsigned grid = part ? (unsigned)blocks : (unsigned)(groups < 1 << 20 ? groups : 1 << 20);
#define RUN(NT, NV)                                                                                           \
  if (cols % 4 == 0)                                                                                                   \
    hipLaunchKernelGGL((ln_bwd_kernel<NT, NV, false>), dim3(grid), dim3(threads_of(NT)), 0, stream(), x, w, dy, \
                       mean, rstd, dx, part, rows, (int)cols);                                                \
  else                                                                                                        \
    hipLaunchKernelGGL((ln_bwd_kernel<NT, NV, true>), dim3(grid), dim3(threads_of(NT)), 0, stream(), x, w, dy, \
                       mean, rstd, dx, part, rows, (int)cols)
    BY_COLS(RUN)
#undef RUN
  }
  if (part) {
    // a grid axis has less than 2^32 threads (with more, columns stay unwritten)
    const long groups = (cols + 15) / 16;
    hipLaunchKernelGGL(ln_join_kernel, dim3((unsigned)(groups < 1 << 20 ? groups : 1 << 20), 2), dim3(1024), 0,
                       stream(), part, dw, db, blocks, cols);
  }
  ttrt_free(own);
  return launched();
}
