// Rotary positions (HBM roofline: each value read and written once).
//
// The pair (a, b) of a head turns by t = position * f_j:
//   (a cos t - b sin t, a sin t + b cos t);  its gradient turns by -t.
// Far positions make t large, and an fp32 angle would lose it (position 2^17
// at f = 1 leaves 2^-7 of a radian): t is formed in turns, position * (f_j /
// 2 pi) in 64 bits, its whole part dropped there, and only the fraction goes
// to fp32, whose sine and cosine are then good to about 2^-24.
//
// A workgroup takes some rows: their sines and cosines go to LDS once and
// serve all heads.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>
#include "tt_rt.h"

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef f32x4 __attribute__((aligned(4))) f32x4_any;  // in memory, at any float

inline hipStream_t stream() { return (hipStream_t)ttrt_stream(); }
inline int launched() { return hipGetLastError() == hipSuccess ? 0 : -3; }

constexpr int MAX_PAIRS = TT_ROPE_MAX_DIM / 2;

struct Turns {
  double f[MAX_PAIRS];  // turns a position
};

template <int V>
struct Vals {
  float v[V];
};

template <int V>
__device__ __forceinline__ Vals<V> get(const float *p) {
  Vals<V> x;
  if (V == 4) {
    const f32x4 t = *(const f32x4_any *)p;
#pragma unroll
    for (int j = 0; j < V; j++) x.v[j] = t[j];
  } else {
#pragma unroll
    for (int j = 0; j < V; j++) x.v[j] = p[j];
  }
  return x;
}

template <int V>
__device__ __forceinline__ void put(float *p, const Vals<V> &x) {
  if (V == 4) {
    const f32x4 t = {x.v[0], x.v[V > 1], x.v[V > 2 ? 2 : 0], x.v[V > 3 ? 3 : 0]};
    *(f32x4_any *)p = t;
  } else {
#pragma unroll
    for (int j = 0; j < V; j++) p[j] = x.v[j];
  }
}

// V pairs, or V values behind them, a thread
template <int V>
__global__ void __launch_bounds__(256)
    rope_kernel(Turns turns, const float *x, float *y, const int32_t *__restrict__ positions, long rows,
                long seq_len, int heads, int head_dim, int pairs, int interleaved, long ldx, long ldy, float sign,
                float magnitude, int rows_a_group) {
  extern __shared__ float2 cs[];  // [row][pair]
  const long row0 = (long)blockIdx.x * rows_a_group;
  const int nr = rows - row0 < rows_a_group ? (int)(rows - row0) : rows_a_group;
  for (int e = threadIdx.x; e < nr * pairs; e += 256) {
    const int r = e / pairs, j = e - r * pairs;
    const long row = row0 + r;
    const double t = (double)(positions ? (long)positions[row] : row % seq_len) * turns.f[j];
    float s, c;
    sincospif((float)(2.0 * (t - rint(t))), &s, &c);
    cs[e] = make_float2(c * magnitude, s * sign * magnitude);
  }
  __syncthreads();
  const int up = pairs / V, units = up + (head_dim - 2 * pairs) / V, all = nr * heads * units;
  for (int e = threadIdx.x; e < all; e += 256) {
    const int hr = e / units, u = e - hr * units, r = hr / heads, h = hr - r * heads;
    const float *p = x + (row0 + r) * ldx + (long)h * head_dim;
    float *o = y + (row0 + r) * ldy + (long)h * head_dim;
    if (u >= up) {
      const int d = 2 * pairs + (u - up) * V;
      put<V>(o + d, get<V>(p + d));
      continue;
    }
    const float2 *t = cs + r * pairs + u * V;
    if (interleaved) {
      float v[2 * V];
#pragma unroll
      for (int k = 0; k < 2; k++) {
        const Vals<V> w = get<V>(p + u * 2 * V + k * V);
#pragma unroll
        for (int j = 0; j < V; j++) v[k * V + j] = w.v[j];
      }
#pragma unroll
      for (int j = 0; j < V; j++) {
        const float a = v[2 * j], b = v[2 * j + 1];
        v[2 * j] = fmaf(a, t[j].x, -(b * t[j].y));
        v[2 * j + 1] = fmaf(a, t[j].y, b * t[j].x);
      }
#pragma unroll
      for (int k = 0; k < 2; k++) {
        Vals<V> w;
#pragma unroll
        for (int j = 0; j < V; j++) w.v[j] = v[k * V + j];
        put<V>(o + u * 2 * V + k * V, w);
      }
    } else {
      Vals<V> a = get<V>(p + u * V), b = get<V>(p + pairs + u * V);
#pragma unroll
      for (int j = 0; j < V; j++) {
        const float av = a.v[j], bv = b.v[j];
        a.v[j] = fmaf(av, t[j].x, -(bv * t[j].y));
        b.v[j] = fmaf(av, t[j].y, bv * t[j].x);
      }
      put<V>(o + u * V, a);
      put<V>(o + pairs + u * V, b);
    }
  }
}

bool positive(double x) { return x > 0 && x < INFINITY; }

bool good(const TTRope *r) {
  if (!r || r->head_dim <= 0 || r->rot_dim <= 0 || r->rot_dim % 2 != 0 || r->rot_dim > r->head_dim ||
      r->rot_dim > TT_ROPE_MAX_DIM || !positive(r->base) || !(r->magnitude >= 0 && r->magnitude < INFINITY))
    return false;
  switch (r->scaling) {
    case TT_ROPE_PLAIN: return true;
    case TT_ROPE_LINEAR:
    case TT_ROPE_NTK: return positive(r->factor);
    case TT_ROPE_PARTS: return positive(r->factor) && positive(r->trained) && r->high > r->low;
    default: return false;
  }
}

}  // namespace

extern "C" int tt_rope_frequencies(const TTRope *r, double *f) {
  if (!good(r) || !f) return -1;
  const int R = r->rot_dim;
  double base = r->base;
  if (r->scaling == TT_ROPE_NTK && R > 2) base *= pow(r->factor, (double)R / (R - 2));
  // one power in 64, and products between them (off by at most 126 roundings of
  // 2^-53), so that a token's 64 frequencies do not take the host as long as the launch
  const double ratio = pow(base, -2.0 / R), per = 1 / r->factor, turns = r->trained / (2 * M_PI),
               range = 1 / (r->high - r->low);
  double g = 1;
  for (int j = 0; j < R / 2; j++) {
    g = j % 64 ? g * ratio : pow(base, -2.0 * j / R);
    f[j] = g;
    if (r->scaling == TT_ROPE_LINEAR) f[j] *= per;
    if (r->scaling == TT_ROPE_PARTS) {
      double keep = (turns * f[j] - r->low) * range;
      keep = keep < 0 ? 0 : keep > 1 ? 1 : keep;
      f[j] = (1 - keep) * f[j] * per + keep * f[j];
    }
    if (!(fabs(f[j]) < INFINITY)) return -1;  // low = -infinity, or past the range: NaN at every position
  }
  return 0;
}

extern "C" int tt_k_rope(const TTRope *r, const float *x, float *y, const int32_t *positions, long rows,
                         long seq_len, int heads, long ldx, long ldy, int transpose) {
  if (!good(r) || !x || !y || rows <= 0 || heads <= 0 || (!positions && seq_len <= 0) ||
      r->head_dim > (1L << 20) / heads)
    return -1;
  const long width = (long)heads * r->head_dim;
  if (ldx == 0) ldx = width;
  if (ldy == 0) ldy = width;
  if (ldx < width || ldy < width || rows > (1L << 40) / (ldx > ldy ? ldx : ldy)) return -1;
  if (x == y && ldx != ldy) return -1;
  const int pairs = r->rot_dim / 2;
  // rows for four float4 a thread, within 32 KB of sines and cosines
  long n = 4096 / width;
  if (n > 4096 / pairs) n = 4096 / pairs;
  if (n < 1) n = 1;
  if ((rows + n - 1) / n > (1L << 24) - 1) n = (rows + (1L << 24) - 2) / ((1L << 24) - 1);
  if (n > 4096 / pairs || n * width > 0x7fffffffL) return -1;
  Turns t;
  if (tt_rope_frequencies(r, t.f) != 0) return -1;
  if (ttrt_init() != 0) return -3;
  for (int j = 0; j < r->rot_dim / 2; j++) t.f[j] *= 1 / (2 * M_PI);
  const float sign = transpose ? -1.f : 1.f, mag = r->magnitude != 0 ? (float)r->magnitude : 1.f;
  const dim3 grid((unsigned)((rows + n - 1) / n));
  const size_t lds = sizeof(float2) * n * pairs;
  if (pairs % 4 == 0 && r->head_dim % 4 == 0)
    hipLaunchKernelGGL(rope_kernel<4>, grid, dim3(256), lds, stream(), t, x, y, positions, rows, seq_len, heads,
                       r->head_dim, pairs, r->interleaved != 0, ldx, ldy, sign, mag, (int)n);
  else
    hipLaunchKernelGGL(rope_kernel<1>, grid, dim3(256), lds, stream(), t, x, y, positions, rows, seq_len, heads,
                       r->head_dim, pairs, r->interleaved != 0, ldx, ldy, sign, mag, (int)n);
  return launched();
}
