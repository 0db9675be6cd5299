// Attention on the matrix units: forward, the form for few query rows, and the
// backward pass, which recomputes the probabilities.
//
//   o_i = sum_j p_ij v_j,  p_ij = exp(s_ij - lse_i),  s_ij = scale q_i . k_j
//   over the keys lo_i <= j < hi_i that the masks leave query i, with
//   lse_i = log sum_j exp(s_ij); no key: o_i = 0, lse_i = -inf.
//   delta_i = do_i . o_i,  dv_j = sum_i p_ij do_i,  dp_ij = do_i . v_j,
//   ds_ij = p_ij (dp_ij - delta_i),  dq_i = scale sum_j ds_ij k_j,
//   dk_j = scale sum_i ds_ij q_i  (both sums over the heads that share a key).
//
// The matrix units multiply fp32 at 1/16 the rate of bf16.  A float is the sum of
// three bf16 values, exactly (three times 8 bits of its 24), and a product of two
// such sums is their nine products; six of them, all but 2^-21 of it (below), come
// out of v_mfma_f32_16x16x32_bf16, which adds in fp32.  The fp32 products,
// v_mfma_f32_16x16x4_f32, are left to the form for few rows, which waits for
// memory.  In both A holds rows lane % 16 and B columns lane % 16, each the summed
// indexes of its group lane / 16, and C holds column lane % 16, rows
// 4 (lane / 16) + r in register r.  Two consequences carry all kernels here:
//   * a summed index may be dealt to lanes in any order that A and B share;
//   * a product's C registers are the B operand of the next one as they
//     stand, so probabilities go from the scores to the second product without
//     leaving their registers.
// Scores and probabilities are therefore formed transposed, a query (or in the
// key gradients a key) a column: its running maximum and sum are one value a
// lane, and rescaling is one multiplication by it.
//
// The query rows of the heads that share a key head are packed into one row
// axis r = i * group + member, so shared keys are loaded once for all of them.
//
// All sums and statistics are fp32; scores are formed in units of log2 (q or k is
// multiplied by scale * log2(e) once, a rounding of 2^-24).  An infinity that the
// masks leave makes NaN: its parts are it and NaN, and the forms without parts do
// the same.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>
#include "tt_rt.h"

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef f32x4 __attribute__((aligned(4))) f32x4_any;  // in memory, at any float

inline hipStream_t stream() { return (hipStream_t)ttrt_stream(); }
inline int launched() { return hipGetLastError() == hipSuccess ? 0 : -3; }

constexpr float LOG2E = 1.44269504088896340736f;
constexpr float LN2 = 0.69314718055994530942f;
constexpr int MAX_SPLITS = 1024;  // parts that a join takes
constexpr int KT = 32;  // rows of the streamed operand a tile

struct Strides {
  long b, r, h;  // elements from a sequence / row / head to the next
};

struct Args {
  int B, Lq, Lk, Hkv, G, D;
  int R;              // Lq * G packed rows
  int causal;
  long window;
  float scale;
  const int32_t *q_start, *q_len, *k_len;
  Strides q, k, v, o;
  int vec;            // D is a multiple of 4: rows are read four values at a time
  int chunk;          // keys a workgroup takes of a row tile's (splits > 1)
  int splits;
};

struct Range {
  int lo, hi;
};

// Sequence b, read once by a workgroup: its keys, the queries of it that hold
// anything and the position of its first query, whatever the lengths in device
// memory hold.
struct Seq {
  int keys, queries;
  long start;
};
__device__ __forceinline__ Seq seq_of(const Args &a, int b) {
  const int n = a.k_len ? a.k_len[b] : a.Lk, nq = a.q_len ? a.q_len[b] : a.Lq;
  Seq s;
  s.keys = n < 0 ? 0 : n > a.Lk ? a.Lk : n;
  s.queries = nq < 0 ? 0 : nq > a.Lq ? a.Lq : nq;
  s.start = a.q_start ? (long)a.q_start[b] : (long)a.Lk - a.Lq;
  return s;
}

// first key, and the end of the keys, that a query at position `at` sees: both
// grow with `at`
__device__ __forceinline__ int low_of(const Args &a, long at) {
  const long lo = a.window > 0 ? at - a.window + 1 : 0;
  return lo < 0 ? 0 : lo > a.Lk ? a.Lk : (int)lo;
}
__device__ __forceinline__ int high_of(const Args &a, const Seq &s, long at) {
  const long hi = a.causal ? at + 1 : a.window > 0 ? at + a.window : s.keys;
  return hi < 0 ? 0 : hi > s.keys ? s.keys : (int)hi;
}

// the keys lo <= j < hi of [0, Lk) that query i of the sequence sees
__device__ __forceinline__ Range range_of(const Args &a, const Seq &s, int i) {
  const long at = s.start + i;
  Range g = {low_of(a, at), high_of(a, s, at)};
  if (g.hi <= g.lo || i >= s.queries) g.lo = g.hi = 0;
  return g;
}

// what the queries [i0, i1] of a sequence see: no query a key outside
// [lo, hi), every row all keys of [ilo, ihi)
struct Span {
  int lo, hi, ilo, ihi;
};

__device__ __forceinline__ Span span_of(const Args &a, const Seq &q, int i0, int i1) {
  Span s = {0, 0, 0, 0};
  const bool whole = i1 < q.queries;
  if (!whole) i1 = q.queries - 1;
  if (i0 > i1) return s;
  s.lo = low_of(a, q.start + i0);
  s.hi = high_of(a, q, q.start + i1);
  if (s.hi <= s.lo) s.lo = s.hi = 0;
  if (whole) {
    s.ilo = low_of(a, q.start + i1);
    s.ihi = high_of(a, q, q.start + i0);
    if (s.ihi <= s.ilo) s.ilo = s.ihi = 0;
  }
  return s;
}

// the same for the 16 packed rows of a wave from r0 on
__device__ __forceinline__ Span wave_span(const Args &a, const Seq &q, int r0, int r1) {
  if (r0 >= r1) return Span{0, 0, 0, 0};
  return span_of(a, q, r0 / a.G, ((r0 + 16 < r1 ? r0 + 16 : r1) - 1) / a.G);
}

// Workgroups start in the order of blockIdx, 256 CUs at a time, and under a
// causal mask the first have the most to do: every other round goes backwards,
// so that a CU that holds several is not given the heaviest of each.  Eight
// neighbours keep their order, and with it their XCD and its L2.
__device__ __forceinline__ int snake(int p, int all) {
  const int round = p & ~255;
  return (p & 256) && round + 256 <= all ? round + ((p & 255) ^ 248) : p;
}

// What workgroup `block` of T tiles of `per` a (sequence, key head) takes.  Plain: tile
// by tile, the last (which see the most keys under a causal mask) first.  Where
// the sequences' lengths are given and few enough for a wave, tile by tile of
// those that reach so far, so that the heaviest come first and tiles behind a
// sequence's end last: 64 heads in a batch of 1024 to 600 rows otherwise leave
// the CUs idle for 40 % of the time.  from_end: tile T - 1 is a sequence's first
// (key tiles, the first of which meet the most queries).
struct Item {
  int b, h, tile;
};
__device__ __forceinline__ Item item_of(const Args &a, int block, int blocks, const int32_t *len, int rows, int G,
                                        int per, bool from_end) {
  int p = snake(block, blocks);
  const int T = blocks / (a.B * a.Hkv);
  Item it;
  if (!len || a.B > 64 || a.B == 1 || T > 256) {
    const int nbh = a.B * a.Hkv, bh = p % nbh;
    it.b = bh / a.Hkv;
    it.h = bh % a.Hkv;
    it.tile = from_end ? p / nbh : T - 1 - p / nbh;
    return it;
  }
  const int lane = threadIdx.x & 63;
  int n = -1;
  if (lane < a.B) {
    const int v = len[lane];
    n = (int)(((long)(v < 0 ? 0 : v > rows ? rows : v) * G + per - 1) / per);
  }
  unsigned long long m = 0;
  int t = T - 1;
  bool empty = false;
  for (; t >= 0; t--) {
    m = __ballot(n > t);
    const int c = __popcll(m) * a.Hkv;
    if (p < c) break;
    p -= c;
  }
  if (t < 0) {
    empty = true;
    for (t = 0; t < T - 1; t++) {
      m = __ballot(n >= 0 && n <= t);
      const int c = __popcll(m) * a.Hkv;
      if (p < c) break;
      p -= c;
    }
    if (t == T - 1) m = __ballot(n >= 0 && n <= t);
  }
  for (int k = p / a.Hkv; k > 0; k--) m &= m - 1;
  it.b = __ffsll(m) - 1;
  it.h = p % a.Hkv;
  it.tile = from_end && !empty ? __builtin_amdgcn_readlane(n, it.b) - 1 - t : t;
  return it;
}

// four values of a row from column c on; 0 behind the row's end
__device__ __forceinline__ f32x4 load4(const float *p, int c, int D, int vec) {
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  if (vec) {
    if (c < D) v = *(const f32x4_any *)(p + c);
  } else {
#pragma unroll
    for (int j = 0; j < 4; j++)
      if (c + j < D) v[j] = p[c + j];
  }
  return v;
}

template <int VW>
struct Vec;
template <>
struct Vec<1> {
  typedef float T;
  static __device__ __forceinline__ float at(const T &v, int) { return v; }
};
template <>
struct Vec<2> {
  typedef f32x2 T;
  static __device__ __forceinline__ float at(const T &v, int c) { return v[c]; }
};
template <>
struct Vec<4> {
  typedef f32x4 T;
  static __device__ __forceinline__ float at(const T &v, int c) { return v[c]; }
};

// Output columns of a product over rows of the streamed tile: the 16-row
// blocks of the transposed result take columns d = 16 VW t + VW m + c, so
// that one read of VW values a lane feeds VW blocks.
template <int DB>
struct Cols {
  static constexpr int VW = DB % 4 == 0 ? 4 : DB % 2 == 0 ? 2 : 1;
  static constexpr int T = DB / VW;
};

__device__ __forceinline__ f32x4 mfma(float a, float b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

// One query (or key) at a time, its values over the lanes (two each): what a
// workgroup falls back to when a tile holds an infinity or NaN that a mask
// hides from some of its columns (in the matrix units 0 * inf would reach
// them).  Nothing hidden is read here.  Rare, so small rather than fast: kept
// apart from the loops that run, whose registers it must not take.  A pass whose
// tiles on the masks' edges all hold NaN takes about a hundred times as long (8 x
// 600 to 1024 rows, 8 heads of 64, forward and backward: 0.2 -> 23 ms).
struct Pair {
  float x, y;
};
// x, and NaN for an infinity: what the products of parts make of one
__device__ __forceinline__ float finite(float x) { return fmaf(x, 0.f, x); }
__device__ __forceinline__ Pair load2(const float *p, int D, int lane) {
  Pair r = {0.f, 0.f};
  if (lane < D) r.x = finite(p[lane]);
  if (lane + 64 < D) r.y = finite(p[lane + 64]);
  return r;
}
__device__ __forceinline__ void store2(float *p, Pair v, float f, int D, int lane) {
  if (lane < D) p[lane] = v.x * f;
  if (lane + 64 < D) p[lane + 64] = v.y * f;
}
__device__ __forceinline__ float dot2(Pair a, Pair b) {
  float s = fmaf(a.x, b.x, a.y * b.y);
#pragma unroll
  for (int n = 1; n < 64; n <<= 1) s += __shfl_xor(s, n);
  return s;
}
__device__ __forceinline__ void add2(Pair &a, float f, Pair b) {
  a.x = fmaf(f, b.x, a.x);
  a.y = fmaf(f, b.y, a.y);
}

// row p[0 .. D) = f * the columns d that acc holds of this lane's row
template <int DB>
__device__ __forceinline__ void store_row(float *p, const f32x4 (&acc)[DB], float f, int D, int vec, int lane) {
  constexpr int VW = Cols<DB>::VW, T = Cols<DB>::T;
  const int g = lane >> 4;
#pragma unroll
  for (int t = 0; t < T; t++)
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const int d = 16 * VW * t + VW * (4 * g + e);
      if (VW == 4 && vec) {
        if (d < D) {
          const f32x4 v = {acc[t * VW][e] * f, acc[t * VW + (VW > 1)][e] * f, acc[t * VW + (VW > 2 ? 2 : 0)][e] * f,
                           acc[t * VW + (VW > 2 ? 3 : 0)][e] * f};
          *(f32x4_any *)(p + d) = v;
        }
      } else {
#pragma unroll
        for (int c = 0; c < VW; c++)
          if (d + c < D) p[d + c] = acc[t * VW + c][e] * f;
      }
    }
}

// row p[0 .. D) = f * the columns that acc holds of this lane's row, block by block
template <int DB>
__device__ __forceinline__ void store_columns(float *p, const f32x4 (&acc)[DB], float f, int D, int vec, int lane) {
#pragma unroll
  for (int o = 0; o < DB; o++) {
    const int d = 16 * o + 4 * (lane >> 4);
    const f32x4 v = acc[o] * f;
    if (vec) {
      if (d < D) *(f32x4_any *)(p + d) = v;
    } else {
#pragma unroll
      for (int e = 0; e < 4; e++)
        if (d + e < D) p[d + e] = v[e];
    }
  }
}

// Loads through a buffer descriptor: an offset past its length gives zeros, so
// that rows and columns outside an operand cost a select and no branch.
constexpr unsigned OUTSIDE = 0x80000000u;
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(const float *p, int bytes = 0x7fffffff) {
  return __builtin_amdgcn_make_buffer_rsrc((void *)p, 0, bytes, 0x00020000);
}

__device__ __forceinline__ float get1(__amdgpu_buffer_rsrc_t r, int off, int c, bool in, int D) {
  return __builtin_bit_cast(
      float, __builtin_amdgcn_raw_buffer_load_b32(r, in && c < D ? (unsigned)(off + c) * 4u : OUTSIDE, 0, 0));
}
__device__ __forceinline__ f32x4 get4(__amdgpu_buffer_rsrc_t r, int off, int c, bool in, int D, int vec) {
  f32x4 v;
  if (vec) {
    v = __builtin_bit_cast(
        f32x4, __builtin_amdgcn_raw_buffer_load_b128(r, in && c < D ? (unsigned)(off + c) * 4u : OUTSIDE, 0, 0));
  } else {
#pragma unroll
    for (int j = 0; j < 4; j++) v[j] = get1(r, off, c + j, in, D);
  }
  return v;
}

// x / G for x < G + KT: at most 1 from KT heads a key on
__device__ __forceinline__ int small_div(int x, int G, unsigned magic) {
  return G >= KT ? x >= G : (int)((unsigned)x * magic >> 16);
}

// ---------------------------------------------------------------- fp32 products in bf16 parts
//
// The fp32 matrix instructions run at 1/16 of the bf16 ones.  An fp32 value is
// the sum of three bf16 values, x = x1 + x2 + x3, cut from its 24 significant
// bits eight at a time (each difference is exact), and of the nine products of
// two such values the six
//   x1 y1 + x1 y2 + x2 y1 + x2 y2 + x1 y3 + x3 y1
// leave out at most 2^-21 of |x y|, 2^-24 on average and in proportion to x y
// itself: less than the roundings of an fp32 sum of a few terms.  Each bf16
// product is exact and added in fp32.  So the matrix units do an fp32 product in
// 6/16 of their time.  An infinity has no such parts: it comes out as NaN.

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
                                                 0);
}

// the leading parts of two values, the first in the low half
__device__ __forceinline__ unsigned lead(float a, float b) {
  return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
}
// what the leading part leaves
__device__ __forceinline__ float rest(float x) { return x - __uint_as_float(__float_as_uint(x) & 0xffff0000u); }

struct Parts {
  u32x4 p[3];  // eight values: part 1, 2 and 3
};
__device__ __forceinline__ Parts parts_of(float (&x)[8]) {
  Parts r;
#pragma unroll
  for (int n = 0; n < 3; n++) {
#pragma unroll
    for (int j = 0; j < 4; j++) r.p[n][j] = lead(x[2 * j], x[2 * j + 1]);
    if (n < 2) {
#pragma unroll
      for (int j = 0; j < 8; j++) x[j] = rest(x[j]);
    }
  }
  return r;
}

// The 16x16x32 product: A holds row m = lane % 16 and B column m, both at the
// eight summed indices of their group g = lane / 16; C holds column m, rows 4 g +
// r in register r.  A wave has 16 query rows (or keys), so that two to four of
// them fit a SIMD's registers and cover each other's waits (32 a wave, with half
// the reads of LDS: 671 against 658 us for the forward pass of 4096 rows and 128
// columns, 76 against 59 for 1024 rows and 64 columns).  DB: blocks of 16 columns of a head, DK: steps of 32.
//
// A tile of KT rows lies in LDS as its parts, a row RC chunks of eight values,
// chunk c of row r at place c ^ f(r): the lanes that LDS serves at once (of a read
// of 16 bytes: 0-3, 12-15, 20-23, 24-27 and so on: rows of two groups; of a
// transposing read, two chunks of eight rows) meet every bank once.  With an odd
// number of fours of chunks the rows' starts already differ in these.
template <int DB>
struct Dim {
  static constexpr int DK = (DB + 1) / 2;
  static constexpr int RC = 4 * DK;
  static constexpr int PART = KT * RC * 16, SIZE = 3 * PART;  // bytes of a part, of a tile
  static __device__ __forceinline__ int f(int r) {
    const int quad = ((r >> 2 ^ r >> 3) & 1) << 1 | (r >> 3 & 1);
    return RC == 16 ? (r & 3) << 2 | quad : RC == 8 ? (r >> 1 & 1) << 2 | quad : quad;
  }
  // the place of chunk x (0 or 2) of the u-th four, where a lane's place in the first is `at`
  static __device__ __forceinline__ int four(int at, int u, int x = 0) {
    return RC % 8 == 4 ? (at ^ x << 4) + u * 64 : at ^ (4 * u + x) << 4;
  }
  static constexpr int TASKS = KT * RC;  // chunks of a tile
};

// a chunk of a tile on its way from memory to LDS
template <int DU>
struct Chunk {
  f32x4 v[2];
  // the eight values at byte `off` of the buffer, of which D - c are the row's:
  // VEC, all of a group of four or none, and where none `off` is OUTSIDE
  template <bool VEC>
  __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t r, unsigned off, int c, int D) {
    if (VEC) {
      v[0] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0));
      v[1] = __builtin_bit_cast(f32x4,
                                __builtin_amdgcn_raw_buffer_load_b128(r, c + 4 < D ? off + 16 : OUTSIDE, 0, 0));
    } else {
#pragma unroll
      for (int j = 0; j < 8; j++)
        v[j / 4][j % 4] = __builtin_bit_cast(
            float, __builtin_amdgcn_raw_buffer_load_b32(r, c + j < D ? off + 4 * j : OUTSIDE, 0, 0));
    }
  }
  // to LDS as parts; NaN for an infinity or NaN among them, else 0
  __device__ __forceinline__ float store(char *tile, int task) const {
    typedef Dim<DU> M;
    const int row = task / M::RC, c = task % M::RC;
    float x[8], t = 0.f;
#pragma unroll
    for (int j = 0; j < 8; j++) {
      x[j] = v[j / 4][j % 4];
      t = fmaf(x[j], 0.f, t);
    }
    const Parts p = parts_of(x);
    char *to = tile + row * M::RC * 16 + ((c ^ M::f(row)) << 4);
#pragma unroll
    for (int n = 0; n < 3; n++) *(u32x4 *)(to + n * M::PART) = p.p[n];
    return t;
  }
};

// A step: the reads of the next one's operands, six products, and some of the
// work of `side`, whose instructions go between the products.  Nothing moves from
// step to step: left alone, the compiler moves every read of an unrolled loop to its front
// and runs out of registers.
__device__ __forceinline__ void step_end() {
#pragma unroll
  for (int n = 0; n < 6; n++) {
    __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);  // a product
    __builtin_amdgcn_sched_group_barrier(0x2, 4, 0);  // vector instructions
  }
  __builtin_amdgcn_sched_barrier(0);
}

__device__ __forceinline__ Parts read_rows(const char *p, int part) {
  Parts r;
#pragma unroll
  for (int n = 0; n < 3; n++) r.p[n] = *(const u32x4 *)(p + n * part);
  return r;
}

__device__ __forceinline__ void six(const Parts &a, const Parts &b, f32x4 &c) {
  c = mma(a.p[0], b.p[0], c);
  c = mma(a.p[0], b.p[1], c);
  c = mma(a.p[1], b.p[0], c);
  c = mma(a.p[1], b.p[1], c);
  c = mma(a.p[0], b.p[2], c);
  c = mma(a.p[2], b.p[0], c);
}

// s[n] = the tile's rows 16 n + .. times this lane's row, columns 32 u + 8 g + ..
template <int DU>
__device__ __forceinline__ void dots(f32x4 (&s)[2], const char *tile, const Parts (&b)[Dim<DU>::DK], int lane) {
  typedef Dim<DU> M;
  const int r = lane & 15, at = r * M::RC * 16 + ((M::f(r) ^ (lane >> 4)) << 4);
  s[0] = s[1] = (f32x4){0.f, 0.f, 0.f, 0.f};
  Parts a = read_rows(tile + at, M::PART), next = a;
#pragma unroll
  for (int n = 0; n < 2 * M::DK; n++) {
    if (n + 1 < 2 * M::DK)
      next = read_rows(tile + M::four(at, (n + 1) / 2) + (n + 1) % 2 * 16 * M::RC * 16, M::PART);
    six(a, b[n / 2], s[n % 2]);
    step_end();
    a = next;
  }
}

// The transposing read: sixteen lanes read four values each of four rows and
// sixteen columns (lane l: row l / 4, columns 4 (l % 4) ..) and get the four
// rows of column l.  Two of them are the eight summed indices of a lane's group
// g, rows 4 g + {0 .. 3, 16 .. 19}: what it holds of a product's two blocks.
typedef short s16x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ u32x2 read_transposed(const char *p) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                       (__attribute__((address_space(3))) s16x4 *)const_cast<char *>(p)));
}
template <int DU>
__device__ __forceinline__ Parts read_columns(const char *tile, int at, int o) {
  typedef Dim<DU> M;
  Parts r;
#pragma unroll
  for (int n = 0; n < 3; n++)
#pragma unroll
    for (int x = 0; x < 2; x++) {
      const u32x2 w = read_transposed(tile + n * M::PART + M::four(at, o / 2, o % 2 * 2) + 16 * x * M::RC * 16);
      r.p[n][2 * x] = w[0];
      r.p[n][2 * x + 1] = w[1];
    }
  return r;
}

template <int DU>
__device__ __forceinline__ int columns_at(int lane) {
  typedef Dim<DU> M;
  const int l = lane & 15, r = 4 * (lane >> 4) + l / 4;
  return r * M::RC * 16 + ((l % 4 / 2 ^ M::f(r)) << 4) + l % 2 * 8;
}
// acc (columns 16 o + .. of block o) += sum over the tile's rows k of
// x[k][column] w[k][l % 16], w the registers of a product with these rows; `a`:
// read_columns of block 0, which the caller has on its way by now
template <int DU, class SIDE>
__device__ __forceinline__ void product(f32x4 (&acc)[DU], const f32x4 (&w)[2], Parts a, const char *tile, int lane,
                                        SIDE side) {
  const int at = columns_at<DU>(lane);
  float x[8];
#pragma unroll
  for (int e = 0; e < 8; e++) x[e] = w[e / 4][e % 4];
  const Parts b = parts_of(x);
  Parts next = a;
#pragma unroll
  for (int n = 0; n < DU; n++) {
    if (n + 1 < DU) next = read_columns<DU>(tile, at, n + 1);
    six(a, b, acc[n]);
    side(n);
    step_end();
    a = next;
  }
}

// this lane's row p[0 .. D) times f as parts, columns 32 u + 8 g + ..
template <int DU>
__device__ __forceinline__ void load_parts(Parts (&b)[Dim<DU>::DK], const float *p, bool in, float f, int D, int vec,
                                           int lane) {
#pragma unroll
  for (int u = 0; u < Dim<DU>::DK; u++) {
    float x[8];
#pragma unroll
    for (int k = 0; k < 2; k++) {
      f32x4 v = {0.f, 0.f, 0.f, 0.f};
      if (in) v = load4(p, 32 * u + 8 * (lane >> 4) + 4 * k, D, vec);
#pragma unroll
      for (int j = 0; j < 4; j++) x[4 * k + j] = v[j] * f;
    }
    b[u] = parts_of(x);
  }
}

// Two tiles (keys and values, or the packed rows of q and do) in turn through
// two buffers: a thread's chunks of the next one are loaded, and go to LDS as
// side work of the products with the present one.
template <int DU, int NT>
struct Stream {
  typedef Dim<DU> M;
  static constexpr int N = (2 * M::TASKS + NT - 1) / NT;
  Chunk<DU> c[N];
  unsigned at[N];  // keys: byte offsets within a tile
  float odd;
  static __device__ __forceinline__ bool has(int t) { return 2 * M::TASKS % NT == 0 || t < 2 * M::TASKS; }
  // a wave's chunks are of one tile of the two
  static __device__ __forceinline__ bool second(int t) { return __builtin_amdgcn_readfirstlane(t) >= M::TASKS; }
  static __device__ __forceinline__ int row_of(int t) { return t % M::TASKS / M::RC; }
  static __device__ __forceinline__ int col_of(int t) { return t % M::TASKS % M::RC * 8; }

  __device__ __forceinline__ void init(int s0, int s1, int D, int tid) {
#pragma unroll
    for (int n = 0; n < N; n++) {
      const int t = tid + n * NT;
      at[n] = col_of(t) < D ? (unsigned)(row_of(t) * (second(t) ? s1 : s0) + col_of(t)) * 4u : OUTSIDE;
    }
  }
  template <bool VEC>
  __device__ __forceinline__ void load_some(__amdgpu_buffer_rsrc_t r0, __amdgpu_buffer_rsrc_t r1, int D, int tid) {
#pragma unroll
    for (int n = 0; n < N; n++) {
      const int t = tid + n * NT;
      if (has(t)) c[n].template load<VEC>(second(t) ? r1 : r0, at[n], col_of(t), D);
    }
  }
  // the rows from p0 (p1) on, s0 (s1) floats apart, zeros from `left` on: past
  // the buffer's length
  __device__ __forceinline__ void load(const float *p0, const float *p1, int s0, int s1, int left, int D, int vec,
                                       int tid) {
    left = left < 0 ? 0 : left < KT ? left : KT;
    const __amdgpu_buffer_rsrc_t r0 = buffer_of(p0, 4 * left * s0), r1 = buffer_of(p1, 4 * left * s1);
    if (vec)
      load_some<true>(r0, r1, D, tid);
    else
      load_some<false>(r0, r1, D, tid);
    odd = 0.f;
  }
  // the same for packed query rows, r = i * G + member, from member m0 of the
  // query at p0 (p1) on
  __device__ __forceinline__ void load_rows(const float *p0, const float *p1, const Strides &s0, const Strides &s1, int G,
                                            unsigned magic, int m0, int left, int D, int vec, int tid) {
#pragma unroll
    for (int n = 0; n < N; n++) {
      const int t = tid + n * NT, row = row_of(t), i = small_div(m0 + row, G, magic), m = m0 + row - i * G;
      const int rs = second(t) ? (int)s1.r : (int)s0.r, hs = second(t) ? (int)s1.h : (int)s0.h;
      at[n] = (row < left && col_of(t) < D) ? (unsigned)(i * rs + m * hs + col_of(t)) * 4u : OUTSIDE;
    }
    const __amdgpu_buffer_rsrc_t r0 = buffer_of(p0), r1 = buffer_of(p1);
    if (vec)
      load_some<true>(r0, r1, D, tid);
    else
      load_some<false>(r0, r1, D, tid);
    odd = 0.f;
  }
  // chunk n to the pair of tiles at `to`; the tiles of `look` (bits) are looked
  // through for infinities and NaN
  __device__ __forceinline__ void store(int n, char *to, int look, int tid) {
    const int t = tid + n * NT;
    if (has(t)) {
      const float z = c[n].store(to + (second(t) ? M::SIZE : 0), t % M::TASKS);
      if (look == 3 || (look == 1) != second(t)) odd += z;
    }
  }
  // at step n of `steps`: the chunks whose turn it is
  __device__ __forceinline__ void side(int n, int steps, char *to, int look, int tid) {
#pragma unroll
    for (int k = 0; k < N; k++)
      if (n == (2 * k + 1) * steps / (2 * N)) store(k, to, look, tid);
  }
  __device__ __forceinline__ void all(char *to, int look, int tid) {
#pragma unroll
    for (int k = 0; k < N; k++) store(k, to, look, tid);
  }
};

// ---- tiles split beforehand
//
// Where a tile is used by many workgroups, a kernel before them writes its parts
// to memory once, as the image of a pair of tiles in LDS, and direct loads bring
// it there: no registers hold it on the way and no vector work cuts it up (2 x
// 4096 causal rows, 16 heads on 4, 128 columns: forward 768 -> 640 us, dq 1021 ->
// 953, dk and dv, which spilled, 2247 -> 1410).  Rows outside an operand are zeros
// in the image.

__device__ __forceinline__ unsigned lds_address(const void *p) {
  return (unsigned)(uintptr_t)(__attribute__((address_space(3))) const char *)p;
}
// lane l's 16 bytes at base + off to LDS at lds + 16 l
__device__ __forceinline__ void dma16(const char *base, int off, unsigned lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
               :
               : "s"(lds), "v"(off), "s"(base)
               : "memory", "m0");
}
// a pointer that is the same for all lanes, in scalar registers
__device__ __forceinline__ const char *scalar(const char *p) {
  const uint64_t x = (uint64_t)p;
  return (const char *)((uint64_t)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32 |
                        (uint32_t)__builtin_amdgcn_readfirstlane((int)x));
}
template <int DU, int NW>
__device__ __forceinline__ void feed(const char *image_, const char *lds, int wave, int lane) {
  constexpr int N = 2 * Dim<DU>::SIZE / 1024;  // what a wave's load moves
  const unsigned to = lds_address(lds);
  const char *image = scalar(image_);
#pragma unroll
  for (int n = 0; n < N; n += NW)
    if (N % NW == 0 || n + wave < N) dma16(image, (n + wave) * 1024 + lane * 16, to + (n + wave) * 1024);
}
// what is on its way to LDS has arrived, for every wave
__device__ __forceinline__ void arrived() {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
}

constexpr int STATS = 4 * KT * 4;  // bytes of a row tile's statistics: lse / ln 2, delta, first key, end of keys

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// over the four lanes that hold a column: exchanges of 16 and 32 lanes between
// registers, without a trip through LDS
__device__ __forceinline__ float col_max(float x) {
  const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1]));
  const auto q = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(q[0]), __uint_as_float(q[1]));
}
__device__ __forceinline__ float col_sum(float x) {
  const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(p[0]) + __uint_as_float(p[1]);
  const auto q = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(q[0]) + __uint_as_float(q[1]);
}

// Waves of a workgroup.  Up to 64 columns three workgroups of four fit a CU (two of
// eight: 8 x 600 to 1024 rows, 8 heads of 64 columns, forward 65 against 60 us, dq
// 87 - 83, dk and dv 108 - 94).  Past 96 columns LDS holds one, of eight.  Between,
// two: of four where they split the tiles themselves forward (8 x 900 rows, 8 heads
// of 80 columns: 104 -> 81 us, 8 x 48 rows of 2048 keys 48 -> 33) and in the backward
// pass over images (8 x 1024 rows, 8 heads on 2: 271 -> 243), of eight in the forward
// pass over images, whose registers are fewer; the backward pass that splits tiles
// itself loses by four (8 x 900 rows: 263 -> 277).
constexpr int waves(int DU) { return DU <= 4 ? 4 : 8; }
constexpr int fwd_waves(int DU, bool pre) { return !pre && DU <= 6 ? 4 : waves(DU); }
constexpr int bwd_waves(int DU, bool pre) { return pre && DU <= 6 ? 4 : waves(DU); }
// waves a SIMD that the registers have to allow
constexpr int bwd_lives(int DU, bool pre) { return DU <= 4 && pre ? 3 : 2; }
constexpr int fwd_lives(int DU, bool pre) { return DU <= 4 ? 3 : DU <= 6 && pre ? 4 : 2; }

// ---------------------------------------------------------------- images

// where the images and flags lie in a workspace
struct Images {
  char *kv, *rows;
  int *kv_flags, *row_flags;
  size_t bytes;
};

// eight values from column c of a row on; 0 behind its end and where not `in`
__device__ __forceinline__ void load8(float (&x)[8], const float *p, int c, bool in, int D, int vec) {
#pragma unroll
  for (int k = 0; k < 2; k++) {
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (in) v = load4(p, c + 4 * k, D, vec);
#pragma unroll
    for (int j = 0; j < 4; j++) x[4 * k + j] = v[j];
  }
}
template <int DU>
__device__ __forceinline__ bool put8(char *tile, float (&x)[8], int row, int c) {
  typedef Dim<DU> M;
  float t = 0.f;
#pragma unroll
  for (int j = 0; j < 8; j++) t = fmaf(x[j], 0.f, t);
  const Parts p = parts_of(x);
  char *to = tile + row * M::RC * 16 + ((c ^ M::f(row)) << 4);
#pragma unroll
  for (int n = 0; n < 3; n++) *(u32x4 *)(to + n * M::PART) = p.p[n];
  return t != t;
}

// The image of a pair of key tiles; flags: 1 where the keys hold an infinity or
// NaN, 2 where the values do.
template <int DU>
__global__ void __launch_bounds__(256)
    attn_kv_images_kernel(Args a, const float *__restrict__ k, const float *__restrict__ v, char *__restrict__ images,
                          int *__restrict__ flags) {
  typedef Dim<DU> M;
  const int tiles = (a.Lk + KT - 1) / KT, bh = blockIdx.x / tiles, tile = blockIdx.x % tiles, b = bh / a.Hkv,
            h = bh % a.Hkv;
  const int keys = seq_of(a, b).keys;
  char *image = images + (long)blockIdx.x * 2 * M::SIZE;
  if (tile * KT >= keys) return;  // behind the sequence: never read
  bool ok = false, ov = false;
  for (int t = threadIdx.x; t < KT * M::RC; t += 256) {
    const int row = t / M::RC, c = t % M::RC, key = tile * KT + row;
    const bool in = key < keys;
    float x[8];
    load8(x, k + (long)b * a.k.b + (long)h * a.k.h + (long)key * a.k.r, 8 * c, in, a.D, a.vec);
    ok |= put8<DU>(image, x, row, c);
    load8(x, v + (long)b * a.v.b + (long)h * a.v.h + (long)key * a.v.r, 8 * c, in, a.D, a.vec);
    ov |= put8<DU>(image + M::SIZE, x, row, c);
  }
  const int f = (__syncthreads_or(ok) ? 1 : 0) | (__syncthreads_or(ov) ? 2 : 0);
  if (threadIdx.x == 0) flags[blockIdx.x] = f;
}

// The image of a pair of tiles of packed rows, q and do, with the rows'
// statistics behind them; delta = do . o on the way.  flags: not 0 where they
// hold an infinity or NaN.
template <int DU>
__global__ void __launch_bounds__(256)
    attn_row_images_kernel(Args a, const float *__restrict__ q, const float *__restrict__ dout,
                           const float *__restrict__ o, const float *__restrict__ lse, float *__restrict__ delta,
                           char *__restrict__ images, int *__restrict__ flags) {
  typedef Dim<DU> M;
  const int tiles = (a.R + KT - 1) / KT, bh = blockIdx.x / tiles, tile = blockIdx.x % tiles, b = bh / a.Hkv,
            h = bh % a.Hkv;
  const Seq sq = seq_of(a, b);
  char *image = images + (long)blockIdx.x * (2 * M::SIZE + STATS);
  float *st = (float *)(image + 2 * M::SIZE);
  bool odd = false;
  constexpr int W = M::RC <= 4 ? 4 : M::RC <= 8 ? 8 : 16;  // lanes of a row
  for (int t = threadIdx.x; t < KT * W; t += 256) {
    const int row = t / W, c = t % W, r = tile * KT + row, i = r / a.G, hq = h * a.G + r - i * a.G;
    const bool in = r < a.R && i < sq.queries;
    const long oo = (long)b * a.o.b + (long)i * a.o.r + (long)hq * a.o.h;
    float x[8], y[8], dl = 0.f;
    load8(x, dout + oo, 8 * c, in, a.D, a.vec);
    load8(y, o + oo, 8 * c, in, a.D, a.vec);
#pragma unroll
    for (int j = 0; j < 8; j++) dl = fmaf(x[j], y[j], dl);
#pragma unroll
    for (int n = 1; n < W; n <<= 1) dl += __shfl_xor(dl, n);
    if (c < M::RC) odd |= put8<DU>(image + M::SIZE, x, row, c);
    load8(x, q + (long)b * a.q.b + (long)i * a.q.r + (long)hq * a.q.h, 8 * c, in, a.D, a.vec);
    if (c < M::RC) odd |= put8<DU>(image, x, row, c);
    if (c == 0) {
      Range rg = {0, 0};
      float l2 = 0.f;
      if (in) {
        rg = range_of(a, sq, i);
        const long at = ((long)b * a.Hkv * a.G + hq) * a.Lq + i;
        l2 = lse[at] * LOG2E;
        if (l2 == -INFINITY) l2 = 0.f;
        delta[at] = dl;
      }
      st[row] = l2;
      st[KT + row] = dl;
      ((int *)st)[2 * KT + row] = rg.lo;
      ((int *)st)[3 * KT + row] = rg.hi;
    }
  }
  odd = __syncthreads_or(odd);
  if (threadIdx.x == 0) flags[blockIdx.x] = odd;
}

// ---------------------------------------------------------------- forward

// 16 packed rows from `first` on, for attn_fwd_kernel's keys [k0, k1)
__device__ __forceinline__ void fwd_one_by_one(const Args &a, const Seq &sq, int b, int h, int first, int r1, int k0, int k1,
                                               const float *q, const float *k, const float *v, float *o, float *lse,
                                               float *ws_ml, float *ws_o, int width, int lane) {
#pragma unroll 1
  for (int row = first; row < first + 16 && row < r1; row++) {
    const int i = row / a.G, hm = row - i * a.G;
    Range rg = range_of(a, sq, i);
    if (rg.lo < k0) rg.lo = k0;
    if (rg.hi > k1) rg.hi = k1;
    Pair qv = {0.f, 0.f}, acc = qv;
    if (rg.lo < rg.hi) qv = load2(q + (long)i * a.q.r + (long)hm * a.q.h, a.D, lane);
    qv.x *= a.scale * LOG2E;
    qv.y *= a.scale * LOG2E;
    float mx = -INFINITY, sum = 0.f;
#pragma unroll 1
    for (int j = rg.lo; j < rg.hi; j++) {
      const float s = dot2(qv, load2(k + (long)j * a.k.r, a.D, lane)), t = fmaxf(s, mx);
      const float base = t == -INFINITY ? 0.f : t, f = exp2_fast(mx - base), p = exp2_fast(s - base);
      mx = t;
      sum = fmaf(sum, f, p);
      acc.x *= f;
      acc.y *= f;
      add2(acc, p, load2(v + (long)j * a.v.r, a.D, lane));
    }
    const int hq = h * a.G + hm;
    if (a.splits > 1) {
      const long at = ((long)blockIdx.y * a.B * a.Hkv + (long)b * a.Hkv + h) * a.R + row;
      if (lane == 0) {
        ws_ml[2 * at] = mx;
        ws_ml[2 * at + 1] = sum;
      }
      store2(ws_o + at * width, acc, 1.f, a.D, lane);
      continue;
    }
    if (lse && lane == 0)
      lse[((long)b * a.Hkv * a.G + hq) * a.Lq + i] = sum == 0.f ? -INFINITY : (mx + log2f(sum)) * LN2;
    store2(o + (long)b * a.o.b + (long)i * a.o.r + (long)hq * a.o.h, acc, sum == 0.f ? 0.f : 1.f / sum, a.D, lane);
  }
}

// One workgroup of NW waves: 16 packed rows a wave of one key head against
// the keys they see, KT at a time through LDS, from memory or (PRE) from images.
// Bound by the matrix units and by what lies between their products (2 x 4096
// causal rows, 16 heads on 4, 128 columns: 640 us, 215 TFLOP/s of fp32, matrix
// units 62 % busy at 1.8 GHz, LDS without conflicts).
// With splits > 1 it takes `chunk` keys of them and leaves maximum, sum and the
// unscaled result to the join.
template <int DU, int NW, bool PRE>
__global__ void __launch_bounds__(64 * NW, fwd_lives(DU, PRE))
    attn_fwd_kernel(Args a, const float *__restrict__ q, const float *__restrict__ k,
                    const float *__restrict__ v, float *__restrict__ o, float *__restrict__ lse,
                    float *__restrict__ ws_ml, float *__restrict__ ws_o, const char *__restrict__ images,
                    const int *__restrict__ flags) {
  typedef Dim<DU> M;
  __shared__ __attribute__((aligned(16))) char lds[2][2 * M::SIZE];
  constexpr int ROWS = 16 * NW;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4;
  const int nbh = a.B * a.Hkv;
  const Item it = item_of(a, blockIdx.x, gridDim.x, a.q_len, a.Lq, a.G, ROWS, false);
  const int b = it.b, h = it.h, tile = it.tile, bh = b * a.Hkv + h;
  const int r0 = tile * ROWS, r1 = r0 + ROWS < a.R ? r0 + ROWS : a.R;
  const Seq sq = seq_of(a, b);
  const Span sp = span_of(a, sq, r0 / a.G, (r1 - 1) / a.G);
  const Span mine = wave_span(a, sq, r0 + wave * 16, r1);
  int k_first = sp.lo / KT * KT, k_end = sp.hi;
  if (a.splits > 1) {
    const long c0 = (long)blockIdx.y * a.chunk, c1 = c0 + a.chunk;
    if (c0 > k_first) k_first = c0 < sp.hi ? (int)c0 : sp.hi;
    if (c1 < k_end) k_end = (int)c1;
  }
  const float *qp = q + (long)b * a.q.b + (long)h * a.G * a.q.h;
  const float *kp = k + (long)b * a.k.b + (long)h * a.k.h, *vp = v + (long)b * a.v.b + (long)h * a.v.h;
  const long tile0 = (long)bh * ((a.Lk + KT - 1) / KT);  // of the images
  Stream<DU, 64 * NW> next;
  if constexpr (!PRE) next.init((int)a.k.r, (int)a.v.r, a.D, tid);
  auto load = [&](int k0, int buf) {
    if constexpr (PRE)
      feed<DU, NW>(images + (tile0 + k0 / KT) * 2 * M::SIZE, lds[buf], wave, lane);
    else
      next.load(kp + (long)k0 * a.k.r, vp + (long)k0 * a.v.r, (int)a.k.r, (int)a.v.r, k_end - k0, a.D, a.vec, tid);
  };
  auto is_mixed = [&](int k0) { return k0 < sp.ilo || k0 + KT > sp.ihi; };
  bool odd = false;
  if (k_first < k_end) load(k_first, 0);
  Parts qf[M::DK];
  f32x4 acc[DU];
  float mx = -INFINITY, sum = 0.f;
  const int row = r0 + wave * 16 + (lane & 15), i = row / a.G;
  const bool in = row < a.R, live = in && i < sq.queries;  // q holds nothing behind the sequence's queries
  Range rg = {0, 0};
  if (live) rg = range_of(a, sq, i);
  load_parts<DU>(qf, qp + (long)i * a.q.r + (long)(row - i * a.G) * a.q.h, live, a.scale * LOG2E, a.D, a.vec, lane);
#pragma unroll
  for (int n = 0; n < DU; n++) acc[n] = (f32x4){0.f, 0.f, 0.f, 0.f};
  if (k_first < k_end) {
    if constexpr (PRE) {
      arrived();
    } else {
      next.all(lds[0], 2, tid);
      odd = __syncthreads_or(next.odd != next.odd) && is_mixed(k_first);
    }
  }
  int buf = 0;
  for (int k0 = k_first; k0 < k_end; k0 += KT, buf ^= 1) {
    if (PRE && is_mixed(k0)) odd = flags[tile0 + k0 / KT] & 2;
    if (odd) break;
    const char *lk = lds[buf], *lv = lk + M::SIZE;
    char *to = lds[buf ^ 1];
    if (!PRE || k0 + KT < k_end) load(k0 + KT, buf ^ 1);  // from memory: zeros behind the last
    if (k0 < mine.hi && k0 + KT > mine.lo) {  // this wave's rows see some of the tile
      f32x4 s[2];
      dots<DU>(s, lk, qf, lane);
      const Parts first = read_columns<DU>(lv, columns_at<DU>(lane), 0);
      if (is_mixed(k0)) {
#pragma unroll
        for (int r = 0; r < 8; r++) {
          const int key = k0 + 16 * (r / 4) + 4 * g + r % 4;
          s[r / 4][r % 4] = ((key < rg.lo) | (key >= rg.hi)) ? -INFINITY : s[r / 4][r % 4];
        }
      }
      float t = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                      fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
      t = fmaxf(col_max(t), mx);
      const float base = t == -INFINITY ? 0.f : t;
      if (__any(t > mx)) {
        const float f = exp2_fast(mx - base);
        sum *= f;
#pragma unroll
        for (int n = 0; n < DU; n++) acc[n] *= f;
        mx = t;
      }
#pragma unroll
      for (int r = 0; r < 8; r++) s[r / 4][r % 4] = exp2_fast(s[r / 4][r % 4] - base);
      sum += ((s[0][0] + s[0][1]) + (s[0][2] + s[0][3])) + ((s[1][0] + s[1][1]) + (s[1][2] + s[1][3]));
      product<DU>(acc, s, first, lv, lane, [&](int n) {
        if constexpr (!PRE) next.side(n, DU, to, 2, tid);
      });
    } else if constexpr (!PRE) {
      next.all(to, 2, tid);
    }
    if constexpr (PRE) {
      arrived();
    } else {
      if (is_mixed(k0 + KT))
        odd = __syncthreads_or(next.odd != next.odd);
      else
        __syncthreads();
    }
  }
  if (odd) {
    fwd_one_by_one(a, sq, b, h, r0 + wave * 16, r1, k_first, k_end, qp, kp, vp, o, lse, ws_ml, ws_o, 16 * DU, lane);
    return;
  }

  const float total = col_sum(sum);
  if (!in) return;
  if (a.splits > 1) {
    const long at = ((long)blockIdx.y * nbh + bh) * a.R + row;
    if (g == 0) {
      ws_ml[2 * at] = mx;
      ws_ml[2 * at + 1] = total;
    }
    store_columns<DU>(ws_o + at * 16 * DU, acc, 1.f, 16 * DU, 1, lane);
    return;
  }
  const int hq = h * a.G + row - i * a.G;
  if (lse && g == 0)
    lse[((long)b * a.Hkv * a.G + hq) * a.Lq + i] = total == 0.f ? -INFINITY : (mx + log2f(total)) * LN2;
  store_columns<DU>(o + (long)b * a.o.b + (long)i * a.o.r + (long)hq * a.o.h, acc, total == 0.f ? 0.f : 1.f / total,
                    a.D, a.vec, lane);
}

// Few packed rows, 16 a workgroup: the keys pass once, from memory to registers in
// the operand layouts, 16 a wave at a time.  Bandwidth-bound, so the keys are
// split over workgroups; a wave's next keys are on their way as soon as its
// scores are done, its next values as soon as these are used.  32 sequences of
// 100 to 8192 keys, 32 heads on 8, 128 columns: 226 us, 4.8 TB/s.
template <int DB>
struct FewTile {
  static constexpr int VW = Cols<DB>::VW, T = Cols<DB>::T;
  typedef typename Vec<VW>::T V;
  f32x4 k[DB];
  V v[4][T];
  // keys [0, 16) from `base` on, those of [from, left)
  __device__ __forceinline__ void load_k(const float *base, int stride, int from, int left, int D, int vec, int lane) {
    const __amdgpu_buffer_rsrc_t r = buffer_of(base);
    const int g = lane >> 4, m = lane & 15;
    const bool in = m >= from && m < left;
#pragma unroll
    for (int u = 0; u < DB; u++) k[u] = get4(r, m * stride, 16 * u + 4 * g, in, D, vec);
  }
  __device__ __forceinline__ void load_v(const float *base, int stride, int from, int left, int D, int vec, int lane) {
    const __amdgpu_buffer_rsrc_t rs = buffer_of(base);
    const int g = lane >> 4, m = lane & 15;
#pragma unroll
    for (int r = 0; r < 4; r++) {
      const int key = 4 * g + r;
      const bool in = key >= from && key < left;
#pragma unroll
      for (int t = 0; t < T; t++) {
        const int d = 16 * VW * t + VW * m;
        if constexpr (VW == 4) {
          v[r][t] = get4(rs, key * stride, d, in, D, vec);
        } else if constexpr (VW == 2) {
          if (vec)
            v[r][t] = __builtin_bit_cast(
                V, __builtin_amdgcn_raw_buffer_load_b64(rs, in && d < D ? (unsigned)(key * stride + d) * 4u : OUTSIDE,
                                                        0, 0));
          else
            v[r][t] = (V){get1(rs, key * stride, d, in, D), get1(rs, key * stride, d + 1, in, D)};
        } else {
          v[r][t] = get1(rs, key * stride, d, in, D);
        }
      }
    }
  }
};

template <int DB, int NW>
__global__ void __launch_bounds__(64 * NW, 2)
    attn_few_kernel(Args a, const float *__restrict__ q, const float *__restrict__ k,
                    const float *__restrict__ v, float *__restrict__ o, float *__restrict__ lse,
                    float *__restrict__ ws_ml, float *__restrict__ ws_o) {
  constexpr int VW = Cols<DB>::VW, T = Cols<DB>::T, LD = DB * 16 + 4;
  __shared__ __attribute__((aligned(16))) float part[NW][16 * LD];
  __shared__ float pml[NW][2][16];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, m = lane & 15;
  const int nbh = a.B * a.Hkv, bh = blockIdx.x % nbh, b = bh / a.Hkv, h = bh % a.Hkv;
  const int r0 = blockIdx.x / nbh * 16, r1 = r0 + 16 < a.R ? r0 + 16 : a.R;
  const Seq sq = seq_of(a, b);
  const Span sp = span_of(a, sq, r0 / a.G, (r1 - 1) / a.G);
  int k_first = sp.lo / 16 * 16, k_end = sp.hi;
  if (a.splits > 1) {
    const long c0 = (long)blockIdx.y * a.chunk, c1 = c0 + a.chunk;
    if (c0 > k_first) k_first = c0 < sp.hi ? (int)c0 : sp.hi;
    if (c1 < k_end) k_end = (int)c1;
  }
  const int row = r0 + m, i = row / a.G, hq = h * a.G + row - i * a.G;
  const bool live = row < a.R && i < sq.queries;  // q holds nothing behind the sequence's queries
  Range rg = {0, 0};
  if (live) rg = range_of(a, sq, i);
  f32x4 qf[DB], acc[DB];
  float mx = -INFINITY, sum = 0.f;
  const float *qp = q + (long)b * a.q.b + (long)i * a.q.r + (long)hq * a.q.h;
#pragma unroll
  for (int u = 0; u < DB; u++) {
    qf[u] = (f32x4){0.f, 0.f, 0.f, 0.f};
    acc[u] = (f32x4){0.f, 0.f, 0.f, 0.f};
    if (live) qf[u] = load4(qp, 16 * u + 4 * g, a.D, a.vec) * (a.scale * LOG2E);
  }
  const float *kp = k + (long)b * a.k.b + (long)h * a.k.h, *vp = v + (long)b * a.v.b + (long)h * a.v.h;
  FewTile<DB> cur;
  auto load_k = [&](int k0) {
    cur.load_k(kp + (long)k0 * a.k.r, (int)a.k.r, sp.lo - k0, k_end - k0, a.D, a.vec, lane);
  };
  auto load_v = [&](int k0) {
    cur.load_v(vp + (long)k0 * a.v.r, (int)a.v.r, sp.lo - k0, k_end - k0, a.D, a.vec, lane);
  };
  int k0 = k_first + wave * 16;
  if (k0 < k_end) {
    load_k(k0);
    load_v(k0);
  }
  for (; k0 < k_end; k0 += 16 * NW) {
    f32x4 s = {0.f, 0.f, 0.f, 0.f}, s2 = s;  // two chains: one waits for each product's result
#pragma unroll
    for (int u = 0; u < DB; u++)
#pragma unroll
      for (int c = 0; c < 4; c += 2) {
        s = mfma(cur.k[u][c], qf[u][c], s);
        s2 = mfma(cur.k[u][c + 1], qf[u][c + 1], s2);
      }
    s += s2;
    if (k0 + 16 * NW < k_end) load_k(k0 + 16 * NW);
    // an infinite score that a row sees (one in q or k, or a sum past the type's
    // range) is NaN, not a key without weight
    float t = -INFINITY;
#pragma unroll
    for (int r = 0; r < 4; r++) {
      const int key = k0 + 4 * g + r;
      s[r] = key < rg.lo || key >= rg.hi ? -INFINITY : finite(s[r]);
      t = fmaxf(t, s[r]);
    }
    t = fmaxf(col_max(t), mx);
    const float base = t == -INFINITY ? 0.f : t;
    if (__any(t > mx)) {
      const float f = exp2_fast(mx - base);
      sum *= f;
#pragma unroll
      for (int u = 0; u < DB; u++) acc[u] *= f;
    }
    mx = t;
#pragma unroll
    for (int r = 0; r < 4; r++) {
      s[r] = exp2_fast(s[r] - base);
      sum += s[r];
    }
    bool odd = false;
    if (k0 < sp.ilo || k0 + 16 > sp.ihi) {
      float z = 0.f;
#pragma unroll
      for (int r = 0; r < 4; r++)
#pragma unroll
        for (int t2 = 0; t2 < T; t2++)
#pragma unroll
          for (int c = 0; c < VW; c++) z = fmaf(Vec<VW>::at(cur.v[r][t2], c), 0.f, z);
      odd = __any(z != z);
    }
    if (odd) {
      // a mask hides an infinity or NaN of these: the values that a row sees, from memory
      float *mine = part[wave];
#pragma unroll
      for (int r = 0; r < 4; r++) mine[(4 * g + r) * 16 + m] = s[r];
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll 1
      for (int kk = 0; kk < 16; kk++) {
        const int key = k0 + kk;
        if (key < rg.lo || key >= rg.hi || key >= k_end) continue;
        const float p = mine[kk * 16 + m];
        const float *x = vp + (long)key * a.v.r;
#pragma unroll
        for (int t2 = 0; t2 < T; t2++)
#pragma unroll
          for (int c = 0; c < VW; c++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
              const int d = 16 * VW * t2 + VW * (4 * g + e) + c;
              if (d < a.D) acc[t2 * VW + c][e] = fmaf(p, x[d], acc[t2 * VW + c][e]);
            }
      }
      __builtin_amdgcn_wave_barrier();
    } else {
#pragma unroll
      for (int r = 0; r < 4; r++)
#pragma unroll
        for (int t2 = 0; t2 < T; t2++)
#pragma unroll
          for (int c = 0; c < VW; c++)
            acc[t2 * VW + c] = mfma(Vec<VW>::at(cur.v[r][t2], c), s[r], acc[t2 * VW + c]);
    }
    if (k0 + 16 * NW < k_end) load_v(k0 + 16 * NW);
  }
  sum = col_sum(sum);
  // An infinity in v comes out as NaN here too.  Scores and results looked at
  // cost nothing that shows; the values of k and v as they are used 4 % (20 rows
  // of 32 x 8 heads of 4096 keys of 80 columns 194 -> 202 us).
#pragma unroll
  for (int u = 0; u < DB; u++)
#pragma unroll
    for (int e = 0; e < 4; e++) acc[u][e] = finite(acc[u][e]);
  // the waves' parts, joined in wave order
  if (g == 0) {
    pml[wave][0][m] = mx;
    pml[wave][1][m] = sum;
  }
  store_row<DB>(&part[wave][m * LD], acc, 1.f, DB * 16, 1, lane);
  __syncthreads();
  for (int e = tid; e < 16 * DB * 16; e += 64 * NW) {
    const int rr = e / (DB * 16), d = e % (DB * 16), r = r0 + rr;
    if (r >= a.R) continue;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < NW; w++) top = fmaxf(top, pml[w][0][rr]);
    const float base = top == -INFINITY ? 0.f : top;
    float total = 0.f, x = 0.f;
#pragma unroll
    for (int w = 0; w < NW; w++) {
      const float f = exp2_fast(pml[w][0][rr] - base);
      total = fmaf(f, pml[w][1][rr], total);
      x = fmaf(f, part[w][rr * LD + d], x);
    }
    if (a.splits > 1) {
      const long at = ((long)blockIdx.y * nbh + bh) * a.R + r;
      if (d == 0) {
        ws_ml[2 * at] = top;
        ws_ml[2 * at + 1] = total;
      }
      ws_o[at * (DB * 16) + d] = x;
      continue;
    }
    const int qi = r / a.G, hh = h * a.G + r - qi * a.G;
    if (lse && d == 0)
      lse[((long)b * a.Hkv * a.G + hh) * a.Lq + qi] = total == 0.f ? -INFINITY : (top + log2f(total)) * LN2;
    if (d < a.D)
      o[(long)b * a.o.b + (long)qi * a.o.r + (long)hh * a.o.h + d] = total == 0.f ? 0.f : x / total;
  }
}

// The parts of a row that several workgroups took, joined in a fixed order.  A
// part without keys has sum 0 and values 0; one without weight next to the others
// counts times 0, so that a NaN that the row sees in it stays.
__device__ __forceinline__ void join_store(const Args &a, long at, float top, float total, float2 x, int lane,
                                           float *o, float *lse) {
  const int bh = (int)(at / a.R), r = (int)(at % a.R), b = bh / a.Hkv, i = r / a.G;
  const int hq = bh % a.Hkv * a.G + r - i * a.G;
  if (lse && lane == 0)
    lse[((long)b * a.Hkv * a.G + hq) * a.Lq + i] = total == 0.f ? -INFINITY : (top + log2f(total)) * LN2;
  float *q = o + (long)b * a.o.b + (long)i * a.o.r + (long)hq * a.o.h + 2 * lane;
  const float f = total == 0.f ? 0.f : 1.f / total;
  if (2 * lane < a.D) q[0] = x.x * f;
  if (2 * lane + 1 < a.D) q[1] = x.y * f;
}

// Up to FEW_PARTS parts: four columns a thread, which forms its row's weights itself
// (16000 rows of four parts of 80 columns: 10.4 us with a wave a row, 7.7 so).
constexpr int FEW_PARTS = 8;
__global__ void __launch_bounds__(256)
    attn_join_few_kernel(Args a, int width, const float *__restrict__ ws_ml, const float *__restrict__ ws_o,
                         float *__restrict__ o, float *__restrict__ lse) {
  const int lanes = width / 4, per = 256 / lanes, c = threadIdx.x % lanes * 4;
  const long rows = (long)a.B * a.Hkv * a.R;
  if ((int)threadIdx.x >= per * lanes) return;
  for (long at = (long)blockIdx.x * per + threadIdx.x / lanes; at < rows; at += (long)gridDim.x * per) {
    f32x4 v[FEW_PARTS], x = {0.f, 0.f, 0.f, 0.f};
    float2 ml[FEW_PARTS];
    const float *p = ws_o + at * width + c;
#pragma unroll
    for (int s = 0; s < FEW_PARTS; s++) {
      ml[s] = make_float2(-INFINITY, 0.f);
      v[s] = x;
      if (s < a.splits) {
        ml[s] = *(const float2 *)(ws_ml + 2 * (s * rows + at));
        v[s] = *(const f32x4 *)(p + s * rows * width);
      }
    }
    float top = -INFINITY, total = 0.f;
#pragma unroll
    for (int s = 0; s < FEW_PARTS; s++) top = fmaxf(top, ml[s].x);
    const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int s = 0; s < FEW_PARTS; s++) {
      const float f = ml[s].y == 0.f ? 0.f : exp2_fast(ml[s].x - base);
      total = fmaf(f, ml[s].y, total);
#pragma unroll
      for (int j = 0; j < 4; j++) x[j] = fmaf(f, v[s][j], x[j]);
    }
    const int bh = (int)(at / a.R), r = (int)(at % a.R), b = bh / a.Hkv, i = r / a.G;
    const int hq = bh % a.Hkv * a.G + r - i * a.G;
    if (lse && c == 0)
      lse[((long)b * a.Hkv * a.G + hq) * a.Lq + i] = total == 0.f ? -INFINITY : (top + log2f(total)) * LN2;
    float *q = o + (long)b * a.o.b + (long)i * a.o.r + (long)hq * a.o.h + c;
    x *= total == 0.f ? 0.f : 1.f / total;
    if (a.vec) {
      if (c < a.D) *(f32x4_any *)q = x;
    } else {
#pragma unroll
      for (int j = 0; j < 4; j++)
        if (c + j < a.D) q[j] = x[j];
    }
  }
}

// More parts: a workgroup a row.  The weights of all parts first; then the
// values, four columns a thread and as many parts at once as threads allow, so
// that few loads wait for each other (256 parts of 64 columns: 28 us with a wave
// for every fourth part, 5.4 so).
constexpr int JOIN = 512;
__global__ void __launch_bounds__(JOIN)
    attn_join_kernel(Args a, int width, const float *__restrict__ ws_ml, const float *__restrict__ ws_o,
                     float *__restrict__ o, float *__restrict__ lse) {
  __shared__ float weight[MAX_SPLITS];
  __shared__ float red[2][JOIN / 64];
  __shared__ __attribute__((aligned(16))) float sums[JOIN * 4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int lanes = width / 4, groups = JOIN / lanes, group = tid / lanes, c = tid % lanes * 4;
  const long rows = (long)a.B * a.Hkv * a.R;
  for (long at = blockIdx.x; at < rows; at += gridDim.x) {
    float2 ml[MAX_SPLITS / JOIN];
    float top = -INFINITY, total = 0.f;
#pragma unroll
    for (int n = 0; n < MAX_SPLITS / JOIN; n++) {
      const int s = n * JOIN + tid;
      ml[n] = make_float2(-INFINITY, 0.f);
      if (s < a.splits) ml[n] = *(const float2 *)(ws_ml + 2 * (s * rows + at));
      top = fmaxf(top, ml[n].x);
    }
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) top = fmaxf(top, __shfl_xor(top, x));
    if (lane == 0) red[0][wave] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < JOIN / 64; w++) top = fmaxf(top, red[0][w]);
    const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int n = 0; n < MAX_SPLITS / JOIN; n++) {
      const float f = ml[n].y == 0.f ? 0.f : exp2_fast(ml[n].x - base);
      weight[n * JOIN + tid] = f;
      total = fmaf(f, ml[n].y, total);
    }
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) total += __shfl_xor(total, x);
    if (lane == 0) red[1][wave] = total;
    __syncthreads();
    f32x4 x = {0.f, 0.f, 0.f, 0.f};
    if (group < groups) {
      const float *p = ws_o + at * width + c;
#pragma unroll 8
      for (int s = group; s < a.splits; s += groups) {
        const float f = weight[s];
        const f32x4 v = *(const f32x4 *)(p + s * rows * width);
#pragma unroll
        for (int j = 0; j < 4; j++) x[j] = fmaf(f, v[j], x[j]);
      }
      *(f32x4 *)(sums + group * width + c) = x;
    }
    total = 0.f;
#pragma unroll
    for (int w = 0; w < JOIN / 64; w++) total += red[1][w];
    __syncthreads();
    if (wave == 0) {
      float2 y = make_float2(0.f, 0.f);
      if (2 * lane < width)
        for (int g = 0; g < groups && g < a.splits; g++) {
          const float2 v = *(const float2 *)(sums + g * width + 2 * lane);
          y.x += v.x;
          y.y += v.y;
        }
      join_store(a, at, top, total, y, lane, o, lse);
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------- backward

// delta[b][h][i] = do . o, 16 lanes a row
__global__ void __launch_bounds__(256)
    attn_delta_kernel(Args a, const float *__restrict__ o, const float *__restrict__ dout,
                      float *__restrict__ delta) {
  const long rows = (long)a.B * a.Hkv * a.G * a.Lq;
  const int m = threadIdx.x & 15;
  // 16 lanes share `at`: whole groups leave the loop together
  for (long at = ((long)blockIdx.x * 256 + threadIdx.x) >> 4; at < rows; at += (long)gridDim.x * 16) {
    float s = 0.f;
    const int i = (int)(at % a.Lq), Hq = a.Hkv * a.G;
    const long bh = at / a.Lq;
    const int b = (int)(bh / Hq), h = (int)(bh % Hq);
    if (i < seq_of(a, b).queries) {
      const long off = (long)b * a.o.b + (long)i * a.o.r + (long)h * a.o.h;
      for (int c = 4 * m; c < a.D; c += 64) {
        const f32x4 x = load4(o + off, c, a.D, a.vec), y = load4(dout + off, c, a.D, a.vec);
#pragma unroll
        for (int j = 0; j < 4; j++) s = fmaf(x[j], y[j], s);
      }
    }
#pragma unroll
    for (int x = 1; x < 16; x <<= 1) s += __shfl_xor(s, x);
    if (m == 0) delta[at] = s;
  }
}

// dq of 16 packed rows from `first` on
__device__ __forceinline__ void dq_one_by_one(const Args &a, const Seq &sq, int b, int h, int first, int r1, const float *q,
                                              const float *k, const float *v, const float *dout, const float *lse,
                                              const float *delta, float *dq, int lane) {
#pragma unroll 1
  for (int row = first; row < first + 16 && row < r1; row++) {
    const int i = row / a.G, hq = h * a.G + row - i * a.G;
    const Range rg = range_of(a, sq, i);
    Pair acc = {0.f, 0.f};
    const long at = ((long)b * a.Hkv * a.G + hq) * a.Lq + i, qo = (long)b * a.q.b + (long)i * a.q.r + (long)hq * a.q.h;
    if (rg.lo < rg.hi) {
      Pair qv = load2(q + qo, a.D, lane);
      const Pair dv = load2(dout + (long)b * a.o.b + (long)i * a.o.r + (long)hq * a.o.h, a.D, lane);
      qv.x *= a.scale * LOG2E;
      qv.y *= a.scale * LOG2E;
      float l2 = lse[at] * LOG2E;
      if (l2 == -INFINITY) l2 = 0.f;
      const float dl = delta[at];
#pragma unroll 1
      for (int j = rg.lo; j < rg.hi; j++) {
        const Pair kv = load2(k + (long)j * a.k.r, a.D, lane);
        const float p = exp2_fast(dot2(qv, kv) - l2);
        add2(acc, p * (dot2(dv, load2(v + (long)j * a.v.r, a.D, lane)) - dl), kv);
      }
    }
    store2(dq + qo, acc, a.scale, a.D, lane);
  }
}

// dq of 16 NW packed rows (16 a wave): keys and values through LDS as in the
// forward pass
template <int DU, int NW, bool PRE>
__device__ __forceinline__ void dq_tile(const Args &a, char (*lds)[2 * Dim<DU>::SIZE + STATS], int block, int blocks,
                                        const float *__restrict__ q, const float *__restrict__ k,
                                        const float *__restrict__ v, const float *__restrict__ dout,
                                        const float *__restrict__ lse, const float *__restrict__ delta,
                                        float *__restrict__ dq, const char *__restrict__ images,
                                        const int *__restrict__ flags) {
  typedef Dim<DU> M;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4;
  const Item it = item_of(a, block, blocks, a.q_len, a.Lq, a.G, 16 * NW, false);
  const int b = it.b, h = it.h, tile = it.tile;
  const int r0 = tile * 16 * NW, r1 = r0 + 16 * NW < a.R ? r0 + 16 * NW : a.R;
  const Seq sq = seq_of(a, b);
  const Span sp = span_of(a, sq, r0 / a.G, (r1 - 1) / a.G);
  const Span mine = wave_span(a, sq, r0 + wave * 16, r1);
  const int row = r0 + wave * 16 + (lane & 15), i = row / a.G, hq = h * a.G + row - i * a.G;
  const bool in = row < a.R, live = in && i < sq.queries;
  Range rg = {0, 0};
  float l2 = 0.f, dl = 0.f;
  if (live) {
    rg = range_of(a, sq, i);
    const long at = ((long)b * a.Hkv * a.G + hq) * a.Lq + i;
    l2 = lse[at] * LOG2E;
    if (l2 == -INFINITY) l2 = 0.f;  // no key has weight: exp2(-inf - 0) = 0
    dl = delta[at];
  }
  const float *kp = k + (long)b * a.k.b + (long)h * a.k.h, *vp = v + (long)b * a.v.b + (long)h * a.v.h;
  const int k_first = sp.lo / KT * KT, k_end = sp.hi;
  const long tile0 = (long)(b * a.Hkv + h) * ((a.Lk + KT - 1) / KT);
  Stream<DU, 64 * NW> next;
  if constexpr (!PRE) next.init((int)a.k.r, (int)a.v.r, a.D, tid);
  auto load = [&](int k0, int buf) {
    if constexpr (PRE)
      feed<DU, NW>(images + (tile0 + k0 / KT) * 2 * M::SIZE, lds[buf], wave, lane);
    else
      next.load(kp + (long)k0 * a.k.r, vp + (long)k0 * a.v.r, (int)a.k.r, (int)a.v.r, k_end - k0, a.D, a.vec, tid);
  };
  auto is_mixed = [&](int k0) { return k0 < sp.ilo || k0 + KT > sp.ihi; };
  bool odd = false;
  if (k_first < k_end) load(k_first, 0);
  Parts qf[M::DK], df[M::DK];
  f32x4 acc[DU];
  load_parts<DU>(qf, q + (long)b * a.q.b + (long)i * a.q.r + (long)hq * a.q.h, live, a.scale * LOG2E, a.D, a.vec, lane);
  load_parts<DU>(df, dout + (long)b * a.o.b + (long)i * a.o.r + (long)hq * a.o.h, live, 1.f, a.D, a.vec, lane);
#pragma unroll
  for (int n = 0; n < DU; n++) acc[n] = (f32x4){0.f, 0.f, 0.f, 0.f};
  if (k_first < k_end) {
    if constexpr (PRE) {
      arrived();
    } else {
      next.all(lds[0], 1, tid);
      odd = __syncthreads_or(next.odd != next.odd) && is_mixed(k_first);
    }
  }
  int buf = 0;
  for (int k0 = k_first; k0 < k_end; k0 += KT, buf ^= 1) {
    if (PRE && is_mixed(k0)) odd = flags[tile0 + k0 / KT] & 1;
    if (odd) break;
    const char *lk = lds[buf], *lv = lk + M::SIZE;
    char *to = lds[buf ^ 1];
    if (!PRE || k0 + KT < k_end) load(k0 + KT, buf ^ 1);
    if (k0 < mine.hi && k0 + KT > mine.lo) {
      f32x4 s[2], dp[2];
      dots<DU>(s, lk, qf, lane);
      dots<DU>(dp, lv, df, lane);
      const Parts first = read_columns<DU>(lk, columns_at<DU>(lane), 0);
#pragma unroll
      for (int r = 0; r < 8; r++)
        s[r / 4][r % 4] = exp2_fast(s[r / 4][r % 4] - l2) * (dp[r / 4][r % 4] - dl);
      if (is_mixed(k0)) {
#pragma unroll
        for (int r = 0; r < 8; r++) {
          const int key = k0 + 16 * (r / 4) + 4 * g + r % 4;
          s[r / 4][r % 4] = ((key < rg.lo) | (key >= rg.hi)) ? 0.f : s[r / 4][r % 4];
        }
      }
      product<DU>(acc, s, first, lk, lane, [&](int n) {
        if constexpr (!PRE) next.side(n, DU, to, 1, tid);
      });
    } else if constexpr (!PRE) {
      next.all(to, 1, tid);
    }
    if constexpr (PRE) {
      arrived();
    } else {
      if (is_mixed(k0 + KT))
        odd = __syncthreads_or(next.odd != next.odd);
      else
        __syncthreads();
    }
  }
  if (odd) {
    dq_one_by_one(a, sq, b, h, r0 + wave * 16, r1, q, kp, vp, dout, lse, delta, dq, lane);
    return;
  }
  if (in)
    store_columns<DU>(dq + (long)b * a.q.b + (long)i * a.q.r + (long)hq * a.q.h, acc, a.scale, a.D, a.vec, lane);
}

// the packed rows that see a key of [k0, k1), from the start of their tile on
struct Rows {
  int first, end;
};
__device__ __forceinline__ Rows rows_of(const Args &a, const Seq &s, int k0, int k1) {
  long i0 = 0, i1 = s.queries;
  if (a.causal) {
    if (k0 - s.start > i0) i0 = k0 - s.start;
  } else if (a.window > 0 && k0 - a.window - s.start + 1 > i0) {
    i0 = k0 - a.window - s.start + 1;
  }
  if (a.window > 0 && k1 - 1 + a.window - s.start < i1) i1 = k1 - 1 + a.window - s.start;
  Rows r = {0, 0};
  if (k0 >= s.keys || i0 >= i1) return r;
  r.first = (int)i0 * a.G / KT * KT;
  r.end = (int)i1 * a.G;
  return r;
}

// dk and dv of 16 keys from `first` on, from the packed rows [r0, r1)
__device__ __forceinline__ void dkv_one_by_one(const Args &a, const Seq &seq, int b, int h, int first, int r0, int r1,
                                               const float *q, const float *k, const float *v, const float *dout,
                                               const float *lse, const float *delta, float *dk, float *dv, float *ws,
                                               int split, int width, int lane) {
  const int keys = seq.keys;
#pragma unroll 1
  for (int key = first; key < first + 16 && key < a.Lk; key++) {
    Pair ak = {0.f, 0.f}, av = {0.f, 0.f};
    const long ko = (long)b * a.k.b + (long)h * a.k.h + (long)key * a.k.r;
    const long vo = (long)b * a.v.b + (long)h * a.v.h + (long)key * a.v.r;
    if (key < keys) {
      Pair kv = load2(k + ko, a.D, lane);
      const Pair vv = load2(v + vo, a.D, lane);
      kv.x *= a.scale * LOG2E;
      kv.y *= a.scale * LOG2E;
#pragma unroll 1
      for (int row = r0; row < r1; row++) {
        const int i = row / a.G, hq = h * a.G + row - i * a.G;
        const Range rg = range_of(a, seq, i);
        if (key < rg.lo || key >= rg.hi) continue;
        const long at = ((long)b * a.Hkv * a.G + hq) * a.Lq + i;
        float l2 = lse[at] * LOG2E;
        if (l2 == -INFINITY) l2 = 0.f;
        const Pair qv = load2(q + (long)b * a.q.b + (long)i * a.q.r + (long)hq * a.q.h, a.D, lane);
        const Pair dw = load2(dout + (long)b * a.o.b + (long)i * a.o.r + (long)hq * a.o.h, a.D, lane);
        const float p = exp2_fast(dot2(qv, kv) - l2);
        add2(av, p, dw);
        add2(ak, p * (dot2(dw, vv) - delta[at]), qv);
      }
    }
    if (a.splits > 1) {
      const long nbh = (long)a.B * a.Hkv, at = ((long)split * nbh + (long)b * a.Hkv + h) * a.Lk + key;
      store2(ws + at * width, ak, a.scale, a.D, lane);
      store2(ws + ((long)a.splits * nbh * a.Lk + at) * width, av, 1.f, a.D, lane);
    } else {
      store2(dk + ko, ak, a.scale, a.D, lane);
      store2(dv + vo, av, 1.f, a.D, lane);
    }
  }
}

// dk and dv of 16 NW keys (16 a wave): the packed query rows that see any of
// them through LDS, q and do.  With splits > 1 a workgroup takes `chunk` of the
// rows and leaves its sums to the join: where many rows meet few keys, and so
// that no fp32 sum runs over more rows than that.
template <int DU, int NW, bool PRE>
__device__ __forceinline__ void dkv_tile(const Args &a, char (*lds)[2 * Dim<DU>::SIZE + STATS], int block, int blocks,
                                         int split, const float *__restrict__ q, const float *__restrict__ k,
                                         const float *__restrict__ v, const float *__restrict__ dout,
                                         const float *__restrict__ lse, const float *__restrict__ delta,
                                         float *__restrict__ dk, float *__restrict__ dv, float *__restrict__ ws,
                                         const char *__restrict__ images, const int *__restrict__ flags) {
  typedef Dim<DU> M;
  constexpr int KEYS = 16 * NW;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4;
  const int nbh = a.B * a.Hkv;
  const Item it = item_of(a, block, blocks, a.k_len, a.Lk, 1, KEYS, true);
  const int b = it.b, h = it.h, bh = b * a.Hkv + h, k0 = it.tile * KEYS, kw = k0 + wave * 16, key = kw + (lane & 15);
  const Seq seq = seq_of(a, b);
  Rows rows = rows_of(a, seq, k0, k0 + KEYS);
  if (a.splits > 1) {
    const long c0 = rows.first + (long)split * a.chunk;
    if (c0 >= rows.end && split > 0) return;  // the join leaves it out
    if (c0 + a.chunk < rows.end) rows.end = (int)c0 + a.chunk;
    rows.first = (int)c0;
  }
  const bool in = key < a.Lk, live = key < seq.keys;
  const float *qp = q + (long)b * a.q.b + (long)h * a.G * a.q.h;
  const float *op = dout + (long)b * a.o.b + (long)h * a.G * a.o.h;
  const long tile0 = (long)bh * ((a.R + KT - 1) / KT);
  Stream<DU, 64 * NW> next;
  // row statistics of a tile, by the first KT threads
  float l2_ = 0.f, dl_ = 0.f;
  Range rg_ = {0, 0};
  int i_next = 0, m_next = 0;  // the next tile's first row: query and member
  const int step_i = KT / a.G, step_m = KT % a.G;
  const unsigned magic = 65536u / a.G + 1;  // of small_div: exact for x < 2 KT and G < KT
  // mixed: a mask hides some of the tile's rows from some of the keys; touched:
  // some of the rows see some of this wave's keys
  bool next_mixed = true, next_touched = false;
  auto load = [&](int r0, int buf) {
    const Span sp = span_of(a, seq, i_next, i_next + small_div(m_next + KT - 1, a.G, magic));
    next_touched = kw < sp.hi && kw + 16 > sp.lo;
    next_mixed = r0 + KT > rows.end || k0 < sp.ilo || k0 + KEYS > sp.ihi;
    if constexpr (PRE) {
      const char *from = images + (tile0 + r0 / KT) * (2 * M::SIZE + STATS);
      if (r0 < rows.end) {
        feed<DU, NW>(from, lds[buf], wave, lane);
        if (wave == 0 && lane < STATS / 16) dma16(scalar(from), 2 * M::SIZE + lane * 16, lds_address(lds[buf]) + 2 * M::SIZE);
      }
    } else {
      const float *q0 = qp + (long)i_next * a.q.r, *d0 = op + (long)i_next * a.o.r;
      next.load_rows(q0, d0, a.q, a.o, a.G, magic, m_next, rows.end - r0, a.D, a.vec, tid);
      if (tid < KT) {
        const int e = m_next + tid, di = small_div(e, a.G, magic), i = i_next + di;
        l2_ = dl_ = 0.f;
        rg_.lo = rg_.hi = 0;
        if (r0 + tid < rows.end) {
          rg_ = range_of(a, seq, i);
          const long at = ((long)b * a.Hkv * a.G + h * a.G + e - di * a.G) * a.Lq + i;
          l2_ = lse[at] * LOG2E;
          if (l2_ == -INFINITY) l2_ = 0.f;
          dl_ = delta[at];
        }
      }
    }
    i_next += step_i;
    m_next += step_m;
    if (m_next >= a.G) {
      m_next -= a.G;
      i_next++;
    }
  };
  auto store_statistics = [&](int to) {
    if (tid < KT) {
      float *st = (float *)(lds[to] + 2 * M::SIZE);
      st[tid] = l2_;
      st[KT + tid] = dl_;
      ((int *)st)[2 * KT + tid] = rg_.lo;
      ((int *)st)[3 * KT + tid] = rg_.hi;
    }
  };
  if (rows.first < rows.end) {
    i_next = rows.first / a.G;
    m_next = rows.first - i_next * a.G;
    load(rows.first, 0);
  }
  Parts kf[M::DK], vf[M::DK];
  f32x4 ak[DU], av[DU];
  load_parts<DU>(kf, k + (long)b * a.k.b + (long)h * a.k.h + (long)key * a.k.r, live, a.scale * LOG2E, a.D, a.vec, lane);
  load_parts<DU>(vf, v + (long)b * a.v.b + (long)h * a.v.h + (long)key * a.v.r, live, 1.f, a.D, a.vec, lane);
#pragma unroll
  for (int n = 0; n < DU; n++) ak[n] = av[n] = (f32x4){0.f, 0.f, 0.f, 0.f};
  bool odd = false;
  if (rows.first < rows.end) {
    if constexpr (PRE) {
      arrived();
    } else {
      next.all(lds[0], 3, tid);
      store_statistics(0);
      odd = __syncthreads_or(next.odd != next.odd) && next_mixed;
    }
  }
  int buf = 0;
  for (int r0 = rows.first; r0 < rows.end; r0 += KT, buf ^= 1) {
    const bool mixed = next_mixed, touched = next_touched;
    if (PRE && mixed) odd = flags[tile0 + r0 / KT];
    if (odd) break;
    const char *lq = lds[buf], *ld = lq + M::SIZE;
    const float *st = (const float *)(lq + 2 * M::SIZE);
    char *to = lds[buf ^ 1];
    load(r0 + KT, buf ^ 1);
    if (touched) {
      f32x4 s[2], dp[2];
      dots<DU>(s, lq, kf, lane);
      dots<DU>(dp, ld, vf, lane);
      const Parts first = read_columns<DU>(ld, columns_at<DU>(lane), 0);
#pragma unroll
      for (int n = 0; n < 2; n++) {
        const f32x4 l2 = *(const f32x4 *)(st + 16 * n + 4 * g), dl = *(const f32x4 *)(st + KT + 16 * n + 4 * g);
#pragma unroll
        for (int j = 0; j < 4; j++) {
          s[n][j] = exp2_fast(s[n][j] - l2[j]);
          dp[n][j] = s[n][j] * (dp[n][j] - dl[j]);
        }
      }
      if (mixed) {
#pragma unroll
        for (int n = 0; n < 2; n++) {
          const i32x4 lo = *(const i32x4 *)(st + 2 * KT + 16 * n + 4 * g);
          const i32x4 hi = *(const i32x4 *)(st + 3 * KT + 16 * n + 4 * g);
#pragma unroll
          for (int j = 0; j < 4; j++) {
            const bool hidden = (key < lo[j]) | (key >= hi[j]);
            s[n][j] = hidden ? 0.f : s[n][j];
            dp[n][j] = hidden ? 0.f : dp[n][j];
          }
        }
      }
      product<DU>(av, s, first, ld, lane, [&](int n) {
        if constexpr (!PRE) next.side(n, 2 * DU, to, 3, tid);
      });
      product<DU>(ak, dp, read_columns<DU>(lq, columns_at<DU>(lane), 0), lq, lane, [&](int n) {
        if constexpr (!PRE) next.side(DU + n, 2 * DU, to, 3, tid);
      });
    } else if constexpr (!PRE) {
      next.all(to, 3, tid);
    }
    if constexpr (PRE) {
      arrived();
    } else {
      store_statistics(buf ^ 1);
      if (next_mixed)
        odd = __syncthreads_or(next.odd != next.odd);
      else
        __syncthreads();
    }
  }
  if (odd) {
    dkv_one_by_one(a, seq, b, h, kw, rows.first, rows.end, q, k, v, dout, lse, delta, dk, dv, ws, split,
                   16 * DU, lane);
    return;
  }
  if (!in) return;
  if (a.splits > 1) {
    const long at = ((long)split * nbh + bh) * a.Lk + key, half = (long)a.splits * nbh * a.Lk;
    store_columns<DU>(ws + at * 16 * DU, ak, a.scale, 16 * DU, 1, lane);
    store_columns<DU>(ws + (half + at) * 16 * DU, av, 1.f, 16 * DU, 1, lane);
    return;
  }
  store_columns<DU>(dk + (long)b * a.k.b + (long)h * a.k.h + (long)key * a.k.r, ak, a.scale, a.D, a.vec, lane);
  store_columns<DU>(dv + (long)b * a.v.b + (long)h * a.v.h + (long)key * a.v.r, av, 1.f, a.D, a.vec, lane);
}

// Both gradients in one launch, the keys' tiles first (they take the longest): where
// either leaves CUs idle, or at its end, the other fills them (10 x 203 rows, 8
// heads of 64 columns, with the forward pass: 66 -> 49 us).  Bound like the forward
// pass; both gradients form scores and do . v for themselves, seven products a pair
// for the five that a pass needs (2 x 4096 causal rows, 16 heads on 4, 128 columns:
// 2.25 ms with the images and the join, 153 TFLOP/s of the five, matrix units 66 %
// busy at 1.8 GHz).  dkv_blocks: the tiles of dk and dv times their splits.
template <int DU, int NW, bool PRE>
__global__ void __launch_bounds__(64 * NW, bwd_lives(DU, PRE))
    attn_bwd_kernel(Args a, int dkv_blocks, const float *__restrict__ q, const float *__restrict__ k,
                    const float *__restrict__ v, const float *__restrict__ dout, const float *__restrict__ lse,
                    const float *__restrict__ delta, float *__restrict__ dq, float *__restrict__ dk,
                    float *__restrict__ dv, float *__restrict__ ws, Images m) {
  __shared__ __attribute__((aligned(16))) char lds[2][2 * Dim<DU>::SIZE + STATS];
  const int p = blockIdx.x;
  if (p < dkv_blocks) {
    // splits outermost: the tiles at work at once share rows in the caches (side by
    // side: 2 x 4096 rows, 16 heads on 4, 128 columns 2757 against 2200 us)
    const int n = __builtin_amdgcn_readfirstlane(dkv_blocks / a.splits), split = __builtin_amdgcn_readfirstlane(p / n);
    dkv_tile<DU, NW, PRE>(a, lds, p - split * n, n, split, q, k, v, dout, lse, delta, dk, dv, ws, m.rows, m.row_flags);
  } else {
    dq_tile<DU, NW, PRE>(a, lds, p - dkv_blocks, gridDim.x - dkv_blocks, q, k, v, dout, lse, delta, dq, m.kv,
                         m.kv_flags);
  }
}

// the workgroups' sums of a key, added in their order; 32 lanes a key
__global__ void __launch_bounds__(256)
    attn_dkv_join_kernel(Args a, int width, int keys_a_group, const float *__restrict__ ws, float *__restrict__ dk,
                         float *__restrict__ dv) {
  const long nbh = (long)a.B * a.Hkv, all = nbh * a.Lk;
  const int lane = threadIdx.x & 31;
  for (long e = (long)blockIdx.x * 8 + (threadIdx.x >> 5); e < all; e += (long)gridDim.x * 8) {
    const int bh = (int)(e / a.Lk), key = (int)(e % a.Lk), b = bh / a.Hkv, h = bh % a.Hkv;
    const int k0 = key / keys_a_group * keys_a_group;
    const Rows rows = rows_of(a, seq_of(a, b), k0, k0 + keys_a_group);
    int parts = (rows.end - rows.first + a.chunk - 1) / a.chunk;
    if (parts < 1) parts = 1;
    if (4 * lane >= width) continue;
    f32x4 sk = {0.f, 0.f, 0.f, 0.f}, sv = sk;
    for (int p = 0; p < parts; p++) {
      const float *x = ws + ((p * nbh + bh) * a.Lk + key) * width + 4 * lane;
      sk += *(const f32x4 *)x;
      sv += *(const f32x4 *)(x + (long)a.splits * all * width);
    }
    float *ok = dk + (long)b * a.k.b + (long)h * a.k.h + (long)key * a.k.r;
    float *ov = dv + (long)b * a.v.b + (long)h * a.v.h + (long)key * a.v.r;
#pragma unroll
    for (int j = 0; j < 4; j++)
      if (4 * lane + j < a.D) {
        ok[4 * lane + j] = sk[j];
        ov[4 * lane + j] = sv[j];
      }
  }
}

// ---------------------------------------------------------------- host side

Strides packed(const TTStrides &s, long rows, int heads, int dim) {
  Strides p;
  p.h = s.head ? s.head : dim;
  p.r = s.row ? s.row : (long)heads * dim;
  p.b = s.batch ? s.batch : rows * p.r;
  return p;
}

// 16-column blocks that the kernel of few rows holds for a head dimension
int blocks(int dim) {
  const int n = (dim + 15) / 16;
  return n == 7 ? 8 : n;
}

struct Plan {
  bool few;
  int rows;    // of a workgroup
  int tiles;   // row (key gradients: key) tiles
  int splits, chunk;
  int width;   // floats a row of the parts takes
};

// 0: the arguments describe an attention that the kernels' 32-bit row and
// grid arithmetic covers
int check(const TTAttention *t) {
  if (!t || t->batch <= 0 || t->q_rows <= 0 || t->k_rows <= 0 || t->q_heads <= 0 || t->kv_heads <= 0 ||
      t->head_dim <= 0 || t->head_dim > TT_ATTENTION_MAX_DIM || t->q_heads % t->kv_heads != 0 || t->window < 0 ||
      !(t->scale == t->scale) || isinf(t->scale))
    return -1;
  const TTStrides *all[4] = {&t->q, &t->k, &t->v, &t->o};
  const long G = t->q_heads / t->kv_heads;
  for (const TTStrides *s : all) {
    if (s->batch < 0 || (s->row != 0 && s->row < t->head_dim) || (s->head != 0 && s->head < t->head_dim)) return -1;
    // a tile's rows and a group's heads lie within 2^31 bytes
    if (s->row > (1L << 28) / KT || s->head > (1L << 28) / G || s->batch > 1L << 50) return -1;
  }
  if ((long)t->q_heads * t->head_dim > (1L << 28) / KT) return -1;
  const long lim = 1L << 30, grid = (1L << 23) - 1;
  if (t->q_rows > lim / G || t->k_rows > lim || t->batch > grid / t->kv_heads) return -1;
  const long nbh = t->batch * t->kv_heads;  // the two parts of a grid axis have less than 2^32 threads
  if ((t->q_rows * G + 63) / 64 > grid / nbh || (t->k_rows + 63) / 64 > grid / nbh) return -1;
  return 0;
}

// n in parts of `least` or more, about `want` of them and a multiple of `step`
void split(Plan &p, long n, long want, long least, long step) {
  long parts = want < 1 ? 1 : want;
  if (parts > n / least) parts = n / least;
  if (parts < 1) parts = 1;
  if (parts > MAX_SPLITS) parts = MAX_SPLITS;
  const long c = ((n + parts - 1) / parts + step - 1) / step * step;
  p.chunk = (int)c;
  p.splits = (int)((n + c - 1) / c);
}

// bytes of a pair of tiles' image
size_t pair_bytes(int head_dim) {
  return (size_t)2 * 3 * KT * 16 * 4 * ((blocks(head_dim) + 1) / 2);
}
// Tiles are split beforehand where enough workgroups use each: forward from 1024
// packed rows on, backward (whose products spill registers otherwise, and whose
// rows' images hold delta too) from 384.  us with and without, causal, 8 heads,
// batches of 384 / 512 / 1024 rows, 8192 in all:
//   forward   64 columns   43 - 36,   49 - 43,    70 - 73
//            128 columns   88 - 77,   96 - 87,   135 - 137
//   backward  64 columns  107 - 113, 125 - 132,  190 - 219
//             80 columns  161 - 160, 184 - 189,  260 - 297
//            128 columns  239 - 278, 270 - 326,  398 - 547
// and, backward, there have to be 256 keys to use the rows' for.  At most 4 GiB
// each: past that the tiles are split where they are used.
constexpr long IMAGE_ROWS = 1024, IMAGE_ROWS_BWD = 384, IMAGE_KEYS = 256;
bool fits_images(const TTAttention *t, long rows) {
  return (double)t->batch * t->kv_heads * ((rows + KT - 1) / KT) * (pair_bytes(t->head_dim) + STATS) < 4294967296.;
}
bool images_for_rows(const TTAttention *t) {
  return t->q_rows * (t->q_heads / t->kv_heads) >= IMAGE_ROWS && fits_images(t, t->k_rows);
}
bool images_for_keys(const TTAttention *t) {
  const long rows = t->q_rows * (t->q_heads / t->kv_heads);
  return rows >= IMAGE_ROWS_BWD && t->k_rows >= IMAGE_KEYS && fits_images(t, t->k_rows) && fits_images(t, rows);
}

Plan plan_of(const TTAttention *t) {
  Plan p = {};
  const long G = t->q_heads / t->kv_heads, R = t->q_rows * G, nbh = t->batch * t->kv_heads;
  p.width = 16 * blocks(t->head_dim);
  // Two tiles of few rows, each reading the keys, the second from a cache: 20 rows
  // of 32 x 8 heads of 4096 keys 64 / 80 / 128 columns 161 / 194 / 280 us against
  // 151 / 297 / 311 through LDS, of 8 heads of 32768 keys 38 / 46 / 68 against 41 /
  // 77 / 89; three lose (48 rows: 204 / 317 / 471 against 156 / 304 / 320), and two
  // of 96 columns, which come 8 bytes at a time (235 against 195, 56 against 52)
  p.few = R <= (p.width == 96 ? 16 : 32);
  if (p.few) {
    p.tiles = (int)((R + 15) / 16);
    // parts of 64 to 1024 keys, about two workgroups a CU (eight: 8 heads of 32768
    // keys of 128 columns 71 us, so 51; 64 of 2048 keys 44 and 30; half as many: 52
    // and 29)
    long c = (p.tiles * nbh * t->k_rows / 512 + 63) / 64 * 64;
    c = c < 64 ? 64 : c > 1024 ? 1024 : c;
    split(p, t->k_rows, (t->k_rows + c - 1) / c, 1, 64);
  } else {
    p.rows = 16 * fwd_waves(blocks(t->head_dim), images_for_rows(t));
    p.tiles = (int)((R + p.rows - 1) / p.rows);
    // two workgroups a CU, of 128 keys or more (256: 2 x 141 rows of 698 keys, 2
    // heads, 24.5 against 15.9 us; 64: 3 x 78 rows of 974 keys, 13 heads of 128
    // columns, 50 against 37)
    split(p, t->k_rows, 512 / (p.tiles * nbh), 128, KT);
  }
  return p;
}

Plan dkv_plan(const TTAttention *t) {
  Plan p = {};
  const long G = t->q_heads / t->kv_heads, R = t->q_rows * G, nbh = t->batch * t->kv_heads;
  p.width = 16 * blocks(t->head_dim);
  p.few = false;
  p.rows = 16 * bwd_waves(blocks(t->head_dim), images_for_keys(t));
  p.tiles = (int)((t->k_rows + p.rows - 1) / p.rows);
  // As many workgroups as the CUs hold (512 for three of them: 7 x 152 rows, 40
  // heads on 5, 65 against 54 us; 768 for two: 8 x 524 rows, 8 on 2 of 128
  // columns, 183 against 177); fp32 sums over at most 4096 rows
  const long fill = (p.width <= 64 ? 768 : 512) / (p.tiles * nbh), sums = (R + 4095) / 4096;
  // within 4 GiB of parts (4096 rows a part up to 65536 x 65536 rows and keys of 4
  // heads of 128 columns; sums of more rows past that) and the grid's axis
  const long part = 8L * nbh * t->k_rows * p.width, room = (1L << 32) / part, axis = (1L << 22) / (p.tiles * nbh);
  long want = fill > sums ? fill : sums;
  if (want > room) want = room;
  split(p, R, want < axis ? want : axis, 128, KT);
  return p;
}

Args args_of(const TTAttention *t) {
  Args a;
  a.B = (int)t->batch;
  a.Lq = (int)t->q_rows;
  a.Lk = (int)t->k_rows;
  a.Hkv = t->kv_heads;
  a.G = t->q_heads / t->kv_heads;
  a.D = t->head_dim;
  a.R = a.Lq * a.G;
  a.causal = t->causal != 0;
  a.window = t->window < 1L << 40 ? t->window : 1L << 40;
  a.scale = t->scale != 0.f ? t->scale : 1.f / sqrtf((float)t->head_dim);
  a.q_start = t->q_start;
  a.q_len = t->q_len;
  a.k_len = t->k_len;
  a.q = packed(t->q, t->q_rows, t->q_heads, t->head_dim);
  a.k = packed(t->k, t->k_rows, t->kv_heads, t->head_dim);
  a.v = packed(t->v, t->k_rows, t->kv_heads, t->head_dim);
  a.o = packed(t->o, t->q_rows, t->q_heads, t->head_dim);
  a.vec = a.D % 4 == 0;
  a.chunk = 0;
  a.splits = 1;
  return a;
}

template <int DB>
void run_few(const Plan &p, const Args &a, const float *q, const float *k, const float *v, float *o, float *lse,
             float *ml, float *wo) {
  hipLaunchKernelGGL((attn_few_kernel<DB, 4>), dim3((unsigned)(p.tiles * (long)a.B * a.Hkv), (unsigned)p.splits),
                     dim3(256), 0, stream(), a, q, k, v, o, lse, ml, wo);
}

size_t up(size_t n) { return (n + 255) / 256 * 256; }
Images images_of(const TTAttention *t, bool kv, bool rows, void *base) {
  const long nbh = t->batch * t->kv_heads, kt = (t->k_rows + KT - 1) / KT,
             rt = (t->q_rows * (t->q_heads / t->kv_heads) + KT - 1) / KT;
  const size_t pair = pair_bytes(t->head_dim);
  const size_t n[4] = {kv ? up(nbh * kt * pair) : 0, rows ? up(nbh * rt * (pair + STATS)) : 0,
                       kv ? up(nbh * kt * sizeof(int)) : 0, rows ? up(nbh * rt * sizeof(int)) : 0};
  char *p = (char *)base;
  Images m;
  m.kv = p;
  m.rows = p + n[0];
  m.kv_flags = (int *)(p + n[0] + n[1]);
  m.row_flags = (int *)(p + n[0] + n[1] + n[2]);
  m.bytes = n[0] + n[1] + n[2] + n[3];
  return m;
}

template <int DU>
void run_kv_images(const Args &a, const float *k, const float *v, const Images &m) {
  const long tiles = (long)a.B * a.Hkv * ((a.Lk + KT - 1) / KT);
  hipLaunchKernelGGL(attn_kv_images_kernel<DU>, dim3((unsigned)tiles), dim3(256), 0, stream(), a, k, v, m.kv,
                     m.kv_flags);
}
template <int DU>
void run_row_images(const Args &a, const float *q, const float *dout, const float *o, const float *lse, float *delta,
                    const Images &m) {
  const long tiles = (long)a.B * a.Hkv * ((a.R + KT - 1) / KT);
  hipLaunchKernelGGL(attn_row_images_kernel<DU>, dim3((unsigned)tiles), dim3(256), 0, stream(), a, q, dout, o, lse,
                     delta, m.rows, m.row_flags);
}

template <int DU>
void run_fwd(const Plan &p, const Args &a, const float *q, const float *k, const float *v, float *o, float *lse,
             float *ml, float *wo, const Images *m) {
  constexpr int NW = fwd_waves(DU, false), NP = fwd_waves(DU, true);
  const dim3 grid((unsigned)(p.tiles * (long)a.B * a.Hkv), (unsigned)p.splits);
  if (m)
    hipLaunchKernelGGL((attn_fwd_kernel<DU, NP, true>), grid, dim3(64 * NP), 0, stream(), a, q, k, v, o, lse,
                       ml, wo, m->kv, m->kv_flags);
  else
    hipLaunchKernelGGL((attn_fwd_kernel<DU, NW, false>), grid, dim3(64 * NW), 0, stream(), a, q, k, v, o, lse, ml,
                       wo, NULL, NULL);
}

template <int DU>
void run_bwd(const Plan &p, const Args &a, const float *q, const float *k, const float *v, const float *dout,
             const float *lse, const float *delta, float *dq, float *dk, float *dv, float *ws, bool pre,
             const Images &m) {
  constexpr int NW = bwd_waves(DU, false), NP = bwd_waves(DU, true);
  const int rows = 16 * (pre ? NP : NW);
  const long nbh = (long)a.B * a.Hkv, nk = dk ? p.tiles * nbh * p.splits : 0,
             nq = dq ? ((long)a.R + rows - 1) / rows * nbh : 0;
  if (pre)
    hipLaunchKernelGGL((attn_bwd_kernel<DU, NP, true>), dim3((unsigned)(nk + nq)), dim3(64 * NP), 0, stream(), a,
                       (int)nk, q, k, v, dout, lse, delta, dq, dk, dv, ws, m);
  else
    hipLaunchKernelGGL((attn_bwd_kernel<DU, NW, false>), dim3((unsigned)(nk + nq)), dim3(64 * NW), 0, stream(), a,
                       (int)nk, q, k, v, dout, lse, delta, dq, dk, dv, ws, m);
}

#define BY_STEPS(N, F, ...)            \
  switch (N) {                         \
    case 1: F<1>(__VA_ARGS__); break;  \
    case 2: F<2>(__VA_ARGS__); break;  \
    case 3: F<3>(__VA_ARGS__); break;  \
    case 4: F<4>(__VA_ARGS__); break;  \
    case 5: F<5>(__VA_ARGS__); break;  \
    case 6: F<6>(__VA_ARGS__); break;  \
    default: F<8>(__VA_ARGS__); break; \
  }

// maxima and sums of the parts of a row, and the results behind them
size_t ml_bytes(const TTAttention *t, const Plan &p) {
  return up(sizeof(float) * 2 * p.splits * t->batch * t->q_heads * t->q_rows);
}
size_t fwd_parts(const TTAttention *t, const Plan &p) {
  const size_t rows = (size_t)t->batch * t->q_heads * t->q_rows;
  return p.splits > 1 ? ml_bytes(t, p) + up(sizeof(float) * rows * p.splits * p.width) : 0;
}
size_t fwd_bytes(const TTAttention *t, const Plan &p) {
  return fwd_parts(t, p) + images_of(t, !p.few && images_for_rows(t), false, NULL).bytes;
}

// delta of every query row, and the parts of dk and dv
size_t delta_bytes(const TTAttention *t) { return up(sizeof(float) * t->batch * t->q_heads * t->q_rows); }
size_t dkv_parts(const TTAttention *t, const Plan &p) {
  return p.splits > 1 ? up(sizeof(float) * 2 * p.splits * t->batch * t->kv_heads * t->k_rows * p.width) : 0;
}

}  // namespace

extern "C" size_t tt_k_attention_fwd_ws(const TTAttention *t) {
  if (check(t)) return 0;
  return fwd_bytes(t, plan_of(t));
}

extern "C" int tt_k_attention_fwd(const TTAttention *t, const float *q, const float *k, const float *v, float *o,
                                  float *lse, void *ws) {
  if (check(t) || !q || !k || !v || !o || ((uintptr_t)ws & 15)) return -1;
  if (ttrt_init() != 0) return -3;
  const Plan p = plan_of(t);
  Args a = args_of(t);
  a.splits = p.splits;
  a.chunk = p.chunk;
  const size_t need = fwd_bytes(t, p);
  void *own = NULL;
  if (need && !ws) {
    ws = own = ttrt_alloc(need);
    if (!own) return -2;
  }
  float *ml = (float *)ws, *wo = (float *)((char *)ws + ml_bytes(t, p));
  if (p.few) {
    BY_STEPS(blocks(a.D), run_few, p, a, q, k, v, o, lse, ml, wo);
  } else {
    const bool pre = images_for_rows(t);
    const Images m = images_of(t, pre, false, (char *)ws + fwd_parts(t, p));
    if (pre) {
      BY_STEPS(blocks(a.D), run_kv_images, a, k, v, m);
    }
    BY_STEPS(blocks(a.D), run_fwd, p, a, q, k, v, o, lse, ml, wo, pre ? &m : NULL);
  }
  if (p.splits > 1) {
    const long rows = (long)a.B * a.Hkv * a.R;
    if (p.splits <= FEW_PARTS) {
      const long per = 256 / (p.width / 4), groups = (rows + per - 1) / per;
      hipLaunchKernelGGL(attn_join_few_kernel, dim3((unsigned)(groups < 65536 ? groups : 65536)), dim3(256), 0,
                         stream(), a, p.width, ml, wo, o, lse);
    } else {
      hipLaunchKernelGGL(attn_join_kernel, dim3((unsigned)(rows < 65536 ? rows : 65536)), dim3(JOIN), 0, stream(), a,
                         p.width, ml, wo, o, lse);
    }
  }
  ttrt_free(own);
  return launched();
}

extern "C" size_t tt_k_attention_bwd_ws(const TTAttention *t) {
  if (check(t)) return 0;
  const bool pre = images_for_keys(t);
  return delta_bytes(t) + dkv_parts(t, dkv_plan(t)) + images_of(t, pre, pre, NULL).bytes;
}

extern "C" int tt_k_attention_bwd(const TTAttention *t, const float *q, const float *k, const float *v,
                                  const float *o, const float *dout, const float *lse, float *dq, float *dk,
                                  float *dv, void *ws) {
  if (check(t) || !q || !k || !v || !o || !dout || !lse || (dk == NULL) != (dv == NULL) || ((uintptr_t)ws & 15))
    return -1;
  if (!dq && !dk) return 0;
  if (ttrt_init() != 0) return -3;
  Args a = args_of(t);
  void *own = NULL;
  if (!ws) {
    ws = own = ttrt_alloc(tt_k_attention_bwd_ws(t));
    if (!own) return -2;
  }
  const Plan p = dkv_plan(t);
  const bool pre = images_for_keys(t);
  float *delta = (float *)ws, *parts = (float *)((char *)ws + delta_bytes(t));
  const Images m = images_of(t, pre, pre, (char *)ws + delta_bytes(t) + dkv_parts(t, p));
  if (pre) {
    BY_STEPS(blocks(a.D), run_row_images, a, q, dout, o, lse, delta, m);
  } else {
    const long rows = (long)a.B * a.Hkv * a.R;
    hipLaunchKernelGGL(attn_delta_kernel, dim3((unsigned)((rows + 15) / 16 < 8192 ? (rows + 15) / 16 : 8192)),
                       dim3(256), 0, stream(), a, o, dout, delta);
  }
  if (dq && pre) {
    BY_STEPS(blocks(a.D), run_kv_images, a, k, v, m);
  }
  a.splits = p.splits;
  a.chunk = p.chunk;
  BY_STEPS(blocks(a.D), run_bwd, p, a, q, k, v, dout, lse, delta, dq, dk, dv, parts, pre, m);
  if (dk) {
    if (p.splits > 1) {
      const long keys = (long)a.B * a.Hkv * a.Lk;
      hipLaunchKernelGGL(attn_dkv_join_kernel, dim3((unsigned)((keys + 7) / 8 < 8192 ? (keys + 7) / 8 : 8192)),
                         dim3(256), 0, stream(), a, p.width, p.rows, parts, dk, dv);
    }
  }
  ttrt_free(own);
  return launched();
}
