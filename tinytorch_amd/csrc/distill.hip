// Distillation from a teacher's top logits: loss and gradient of a row of
// student logits in one pass (HBM roofline: logits read, gradient written).
//
//   p = softmax over the row's `top` entries of teacher / T,
//   q = softmax over all columns of logits / T,
//   rowloss = T^2 sum_e p_e (log p_e - log q[ids_e]),
//   dlogits = scale T (q - sum of the p_e at their columns).
//
// A workgroup holds a row in registers: its maximum, the exponentials and
// their sum, and the gradient come from one read.  The entries (a wave's work)
// are done while the row is on its way; their columns are written once more
// behind the row.  Maxima, sums and exponentials are fp32.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>
#include "tt_rt.h"

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef f32x4 __attribute__((aligned(4))) f32x4_any;  // in memory, at any float

inline hipStream_t stream() { return (hipStream_t)ttrt_stream(); }
inline int launched() { return hipGetLastError() == hipSuccess ? 0 : -3; }

constexpr float LOG2E = 1.44269504088896340736f;
constexpr float LN2 = 0.69314718055994530942f;

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

struct Max {
  __device__ float operator()(float a, float b) const { return fmaxf(a, b); }
};
struct Add {
  __device__ float operator()(float a, float b) const { return a + b; }
};

template <class OP>
__device__ __forceinline__ float wave_all(float x, OP op) {
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) x = op(x, __shfl_xor(x, s));
  return x;
}

template <int NT, class OP>
__device__ __forceinline__ float group_all(float x, float *part, OP op) {
  x = wave_all(x, op);
  if (NT == 64) return x;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = x;
  __syncthreads();
  x = part[0];
#pragma unroll
  for (int w = 1; w < NT / 64; w++) x = op(x, part[w]);
  return x;
}

struct Call {
  const float *z;
  const int32_t *ids;
  const float *teacher;
  float *rowloss, *dz;
  long rows;
  int cols, top;
  float c;     // log2(e) / T
  float t2;    // T^2
  float coef;  // scale T
};

struct Entries {
  int4 id[TT_DISTILL_MAX_TOP / 4];  // -1: none
  float z[TT_DISTILL_MAX_TOP];  // the student's logits at them
  float p[TT_DISTILL_MAX_TOP];  // the teacher's logit, then log2 of the probability
  int left_out;                 // a row without entries, or with -inf for all: loss and gradient 0
};

// wave 0: the row's entries to LDS as probabilities
__device__ __forceinline__ void read_entries(const Call &a, long row, Entries &e, int lane) {
  float most = -INFINITY;
  int *ids = (int *)e.id;
  for (int k = a.top + lane; k < (a.top + 3 & ~3); k += 64) ids[k] = -1;
  for (int k = lane; k < a.top; k += 64) {
    const int id = a.ids[row * a.top + k];
    const bool ok = id >= 0 && id < a.cols;
    const float t = ok ? a.teacher[row * a.top + k] : -INFINITY;
    ids[k] = ok ? id : -1;
    if (ok) e.z[k] = a.z[row * a.cols + id];
    e.p[k] = t;
    most = t != t || most != most ? NAN : fmaxf(most, t);  // a NaN is the row's
  }
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) {
    const float o = __shfl_xor(most, s);
    most = most != most || o != o ? NAN : fmaxf(most, o);
  }
  const bool none = most == -INFINITY;
  float sum = 0.f;
  // differences before the factor and the logarithm: next to the type's lowest
  // values either would be lost
  for (int k = lane; k < a.top; k += 64) {
    e.p[k] = none ? -INFINITY : (e.p[k] - most) * a.c;
    sum += exp2_fast(e.p[k]);
  }
  sum = wave_all(sum, Add());
  const float off = none ? 0.f : log2f(sum);
  for (int k = lane; k < a.top; k += 64) e.p[k] -= off;
  if (lane == 0) e.left_out = none;
}

// wave 0: the loss, and the gradient at the entries' columns
__device__ __forceinline__ void finish(const Call &a, long row, const Entries &e, float most, bool flat,
                                       float lse2, int lane, bool gradient) {
  float loss = 0.f;
  const int *ids = (const int *)e.id;
  for (int k = lane; k < a.top; k += 64) {
    const int id = ids[k];
    const float lp = e.p[k];
    if (id < 0) continue;
    const float lq = (flat ? 0.f : (e.z[k] - most) * a.c) - lse2;
    const float p = exp2_fast(lp);
    if (p != 0.f) loss = fmaf(p, (lp - lq) * LN2, loss);
    if (!gradient || e.left_out) continue;
    // entries of one column: the first writes the sum of all
    int same = 0, first = k;
    for (int o = (a.top + 3) / 4 - 1; o >= 0; o--) {
      const int4 t = e.id[o];
      same += (t.x == id) + (t.y == id) + (t.z == id) + (t.w == id);
      if (t.w == id) first = 4 * o + 3;
      if (t.z == id) first = 4 * o + 2;
      if (t.y == id) first = 4 * o + 1;
      if (t.x == id) first = 4 * o;
    }
    if (first != k) continue;
    float sum = p;
    for (int o = k + 1; same > 1; o++)
      if (ids[o] == id) {
        sum += exp2_fast(e.p[o]);
        same--;
      }
    a.dz[row * a.cols + id] = a.coef * (exp2_fast(lq) - sum);
  }
  loss = wave_all(loss, Add());
  if (lane == 0) a.rowloss[row] = e.left_out ? 0.f : loss * a.t2;
}

// A thread's groups of four columns, from column c on.  With TAIL (cols not a
// multiple of 4, and more than 4) the groups at and behind the row's end are its
// last four columns, of which a thread's own are those that no other has: every
// load is one instruction with no branch around it, and none waits for the one
// before.
template <bool TAIL>
struct Group {
  int at, by;  // where it is loaded from; its first value that is the thread's own (TAIL: 4 and more: none)
  __device__ __forceinline__ Group(int c, int cols) {
    at = TAIL && c > cols - 4 ? cols - 4 : c;
    by = TAIL ? c - at : c < cols ? 0 : 4;
  }
  __device__ __forceinline__ f32x4 load(const float *p) const {
    f32x4 v = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
    if (TAIL || by == 0) v = *(const f32x4_any *)(p + at);
    return v;
  }
  __device__ __forceinline__ void mask(f32x4 &v) const {
    if (!TAIL) return;
#pragma unroll
    for (int j = 0; j < 4; j++) v[j] = j >= by ? v[j] : -INFINITY;
  }
  __device__ __forceinline__ void store(float *p, f32x4 v) const {
    if (by == 0) {
      *(f32x4_any *)(p + at) = v;
    } else if (TAIL) {
#pragma unroll
      for (int j = 1; j < 4; j++)
        if (j >= by) p[at + j] = v[j];
    }
  }
};

// a row of up to 4 NT NV columns; TAIL: their number is no multiple of 4
template <int NT, int NV, bool TAIL>
__global__ void __launch_bounds__(NT) distill_kernel(Call a) {
  __shared__ float part[NT / 64];
  __shared__ Entries e;
  const int t = threadIdx.x;
  for (long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const float *z = a.z + row * a.cols;
    f32x4 v[NV];
#pragma unroll
    for (int n = 0; n < NV; n++) v[n] = Group<TAIL>((n * NT + t) * 4, a.cols).load(z);
    if (t < 64) read_entries(a, row, e, t);
#pragma unroll
    for (int n = 0; n < NV; n++) Group<TAIL>((n * NT + t) * 4, a.cols).mask(v[n]);
    float most = -INFINITY;
#pragma unroll
    for (int n = 0; n < NV; n++) most = fmaxf(most, fmaxf(fmaxf(v[n][0], v[n][1]), fmaxf(v[n][2], v[n][3])));
    most = group_all<NT>(most, part, Max());
    // a flat row holds -inf, which count as equal, or NaN, which the maximum
    // passed over and the sum takes to the loss and the gradient
    const bool flat = most == -INFINITY;
    const float base = flat ? 0.f : most, equal = flat ? 1.f : 0.f;
    float sum = 0.f;
#pragma unroll
    for (int n = 0; n < NV; n++)
#pragma unroll
      for (int j = 0; j < 4; j++) {
        float x = exp2_fast((v[n][j] - base) * a.c) + equal;
        if (j < Group<TAIL>((n * NT + t) * 4, a.cols).by) x = 0.f;
        v[n][j] = x;
        sum += x;
      }
    sum = group_all<NT>(sum, part, Add());
    const float lse2 = log2f(sum);
    if (a.dz) {
      float f = a.coef / sum;
      float *dz = a.dz + row * a.cols;
      // a row that is left out may hold infinities and NaN, so f = 0 alone is not
      // enough (a store of its own for it: 2048 x 8192 28.6 us, so 25.1)
      if (__builtin_amdgcn_readfirstlane(e.left_out)) {
        f = 0.f;
#pragma unroll
        for (int n = 0; n < NV; n++) v[n] = (f32x4){0.f, 0.f, 0.f, 0.f};
      }
#pragma unroll
      for (int n = 0; n < NV; n++) {
        v[n] *= f;
        Group<TAIL>((n * NT + t) * 4, a.cols).store(dz, v[n]);
      }
    }
    __syncthreads();  // the row is written: its entries' columns may be
    if (t < 64) finish(a, row, e, most, flat, lse2, t, a.dz != NULL);
    __syncthreads();  // the entries are read
  }
}

// Longer rows: running maximum and sum in a first pass, the gradient in a second
// that finds most of the row in a cache.  TINY: rows of up to 3 columns.
template <bool TINY>
__global__ void __launch_bounds__(1024) distill_long_kernel(Call a) {
  constexpr int U = 4, STEP = U * 4096;  // groups of four on their way at once
  __shared__ float part[16];
  __shared__ Entries e;
  const int t = threadIdx.x;
  for (long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const float *z = a.z + row * a.cols;
    // groups past the end take its last columns, and none of them as their own
    auto group = [&](long c) { return Group<true>((int)(c < a.cols ? c : a.cols), a.cols); };
    auto load = [&](f32x4(&v)[U], long c0) {
      if (TINY) {
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
          for (int j = 0; j < 4; j++) v[u][j] = u == 0 && c0 + j < a.cols ? z[c0 + j] : -INFINITY;
        return;
      }
#pragma unroll
      for (int u = 0; u < U; u++) v[u] = group(c0 + u * 4096).load(z);
#pragma unroll
      for (int u = 0; u < U; u++) group(c0 + u * 4096).mask(v[u]);
    };
    if (t < 64) read_entries(a, row, e, t);
    float most = -INFINITY, sum = 0.f;
    for (long c0 = 4 * t; c0 < a.cols; c0 += STEP) {
      f32x4 v[U];
      load(v, c0);
      float top = most;
#pragma unroll
      for (int u = 0; u < U; u++) top = fmaxf(top, fmaxf(fmaxf(v[u][0], v[u][1]), fmaxf(v[u][2], v[u][3])));
      const float base = top == -INFINITY ? 0.f : top;
      sum *= exp2_fast((most - base) * a.c);
      most = top;
#pragma unroll
      for (int u = 0; u < U; u++)
#pragma unroll
        for (int j = 0; j < 4; j++) sum += exp2_fast((v[u][j] - base) * a.c);
    }
    const float mine = most;
    most = group_all<1024>(most, part, Max());
    const bool flat = most == -INFINITY;
    sum *= flat ? 0.f : exp2_fast((mine - most) * a.c);
    sum = group_all<1024>(sum, part, Add());
    if (flat) sum += (float)a.cols;  // equal logits; a NaN stays
    if (__builtin_amdgcn_readfirstlane(e.left_out)) {
      if (a.dz)
        for (long c = t; c < a.cols; c += 1024) a.dz[row * a.cols + c] = 0.f;
    } else if (a.dz) {
      const float f = a.coef / sum;
      float *dz = a.dz + row * a.cols;
      for (long c0 = 4 * t; c0 < a.cols; c0 += STEP) {
        f32x4 v[U];
        load(v, c0);
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
          for (int j = 0; j < 4; j++) {
            v[u][j] = (flat ? 1.f : exp2_fast((v[u][j] - most) * a.c)) * f;
            if (TINY && u == 0 && c0 + j < a.cols) dz[c0 + j] = v[u][j];
          }
#pragma unroll
        for (int u = 0; u < U; u++)
          if (!TINY) group(c0 + u * 4096).store(dz, v[u]);
      }
    }
    __syncthreads();
    if (t < 64) finish(a, row, e, most, flat, log2f(sum), t, a.dz != NULL);
    __syncthreads();
  }
}

}  // namespace

extern "C" int tt_k_distill(const float *logits, const int32_t *ids, const float *teacher, int top,
                            float temperature, float *rowloss, float *dlogits, long rows, int cols, float scale) {
  if (!logits || !ids || !teacher || !rowloss || rows <= 0 || cols <= 0 || top <= 0 || top > TT_DISTILL_MAX_TOP ||
      !(temperature > 0.f) || isinf(temperature) || !(scale == scale) || isinf(scale) || rows > (1L << 40) / cols ||
      dlogits == logits)
    return -1;
  // factors in 32 bits: T^2 and scale T, and 1 / T with them, within its normal numbers
  if (!(temperature * temperature >= 0x1p-126f) || isinf(temperature * temperature) || isinf(scale * temperature))
    return -1;
  if (ttrt_init() != 0) return -3;
  const Call a = {logits, ids, teacher, rowloss, dlogits, rows, cols, top, LOG2E / temperature,
                  temperature * temperature, scale * temperature};
  const dim3 grid((unsigned)(rows < 1 << 20 ? rows : 1 << 20));
#define RUN(NT, NV)                                                                          \
  if (cols % 4 == 0)                                                                                  \
    hipLaunchKernelGGL((distill_kernel<NT, NV, false>), grid, dim3(NT), 0, stream(), a);      \
  else                                                                                       \
    hipLaunchKernelGGL((distill_kernel<NT, NV, true>), grid, dim3(NT), 0, stream(), a)
  // rows of up to 32768 columns leave room for two workgroups a CU, so that one
  // reads while the other reduces or writes (with a tail past 16384 columns for
  // one, of 136 registers: 2048 x 20001 108 us, x 20000 67).  Past that a row's 1024
  // threads have 128 registers each, which a tail overruns: in two passes 2048 x
  // 32769 / 50257 / 65535 take 141 / 211 / 254 us, in registers that spill 185 / 229
  // / 262; without a tail 50256 columns take 172 in registers.
  if (cols < 4) {
    hipLaunchKernelGGL(distill_long_kernel<true>, grid, dim3(1024), 0, stream(), a);
  } else if (cols <= 1024) {
    RUN(256, 1);
  } else if (cols <= 4096) {
    RUN(256, 4);
  } else if (cols <= 8192) {
    RUN(512, 4);
  } else if (cols <= 16384) {
    RUN(512, 8);
  } else if (cols <= 32768) {
    RUN(512, 16);
  } else if (cols <= 65536 && cols % 4 == 0) {
    hipLaunchKernelGGL((distill_kernel<1024, 16, false>), grid, dim3(1024), 0, stream(), a);
  } else {
    // the second pass reads from the last cache (256 MB) while the rows at work
    // take no more than half of it; a workgroup a CU at least
    long most = (128L << 20) / (4L * cols);
    if (most < 256) most = 256;
    hipLaunchKernelGGL(distill_long_kernel<false>, dim3((unsigned)(rows < most ? rows : most)), dim3(1024), 0, stream(), a);
  }
#undef RUN
  return launched();
}
