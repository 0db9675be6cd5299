// Rows of a table at a batch's tokens, and the table's gradient.
//
//   y[r] = scale w[ids[r]];  dw[v] = scale sum_{r: ids[r] = v} dy[r]
//
// A token outside the table has a row of zeros and no gradient.  Both are bound
// by memory.  The gradient sums over sorted tokens: a workgroup then has the same
// number of rows whatever the tokens are (in a text one word in fifteen is the
// same one), nothing is added atomically, and the sums have one order, that of
// the rows.
//
//   1. Blocks of SORT tokens are sorted by counting: a token's place is the
//      number of the block's tokens that are smaller, or equal and before it.
//      Every pair is compared, 64 tokens a workgroup, so the work spreads over
//      the GPU where a sort by exchanges has one workgroup a block.
//   2. Up to WAYS sorted blocks at a time are merged: a token's place is the sum
//      of its ranks in all of them, each by bisection.  (Not for one block.)
//   3. Each group of lanes adds the rows of TILE tokens in sorted order.  A run of
//      one token that lies inside is written; one that passes an end of the tile
//      is left as a part.
//   4. The parts of such runs are added by the tile that the run begins in.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include "tt_rt.h"

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef f32x4 __attribute__((aligned(4))) f32x4_any;  // any float's alignment

inline hipStream_t stream() { return (hipStream_t)ttrt_stream(); }
inline int launched() { return hipGetLastError() == hipSuccess ? 0 : -3; }

constexpr unsigned NONE = 0xfffffffeu;  // a token outside the table: behind all others
constexpr int SORT = 2048, WAYS = 32, TILE = 32;

__device__ __forceinline__ unsigned key_of(int id, long vocab) {
  return id >= 0 && id < vocab ? (unsigned)id : NONE;
}

// ---------------------------------------------------------------- forward

// TX threads a row, 256 / TX rows at once, R rows a thread: the loads of all R
// are on their way before the first is written.
template <int TX, int R, bool VEC>
__global__ void __launch_bounds__(256)
    embed_kernel(const float *__restrict__ w, const int32_t *__restrict__ ids, float *__restrict__ y, long rows,
                 long vocab, long cols, float scale) {
  constexpr int TY = 256 / TX;
  const long groups = VEC ? (cols + 3) / 4 : cols;
  for (long r0 = (long)blockIdx.x * (TY * R) + threadIdx.x / TX; r0 < rows; r0 += (long)gridDim.x * (TY * R)) {
    int id[R];
#pragma unroll
    for (int k = 0; k < R; k++) id[k] = r0 + k * TY < rows ? ids[r0 + k * TY] : -1;
    for (long n = (long)blockIdx.y * TX + threadIdx.x % TX; n < groups; n += (long)gridDim.y * TX) {
      if (VEC) {
        // the last group is the last four columns: what two groups have is the same in both
        const long c = n * 4 > cols - 4 ? cols - 4 : n * 4;
        f32x4 v[R];
#pragma unroll
        for (int k = 0; k < R; k++) {
          v[k] = (f32x4){0.f, 0.f, 0.f, 0.f};
          if (id[k] >= 0 && id[k] < vocab) v[k] = *(const f32x4_any *)(w + id[k] * cols + c) * scale;
        }
#pragma unroll
        for (int k = 0; k < R; k++)
          if (r0 + k * TY < rows) *(f32x4_any *)(y + (r0 + k * TY) * cols + c) = v[k];
      } else {
#pragma unroll
        for (int k = 0; k < R; k++)
          if (r0 + k * TY < rows)
            y[(r0 + k * TY) * cols + n] = id[k] >= 0 && id[k] < vocab ? w[id[k] * cols + n] * scale : 0.f;
      }
    }
  }
}

// ---------------------------------------------------------------- sorting

// Workgroup q of a block places its tokens [64 q, 64 q + 64): wave s counts
// those of the block's [256 s, 256 s + 256).  Equal tokens before one count too:
// all that are below its successor.  The workgroups behind the last block clear
// the table's gradient meanwhile.
__global__ void __launch_bounds__(512)
    sort_kernel(const int32_t *__restrict__ ids, unsigned *__restrict__ key, int32_t *__restrict__ row, long n,
                long vocab, unsigned sorters, float *__restrict__ clear, long values) {
  if (blockIdx.x >= sorters) {
    const long step = (long)(gridDim.x - sorters) * 512 * 4;
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
    for (long i = ((long)(blockIdx.x - sorters) * 512 + threadIdx.x) * 4; i < values; i += step) {
      if (i + 4 <= values) {
        *(f32x4_any *)(clear + i) = zero;
      } else {
        for (long j = i; j < values; j++) clear[j] = 0.f;
      }
    }
    return;
  }
  __shared__ __attribute__((aligned(16))) unsigned id[SORT];
  __shared__ int below[8][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const long base = (long)(blockIdx.x / (SORT / 64)) * SORT;
  const int q = blockIdx.x % (SORT / 64);
  if (base + q * 64 >= n) return;
  for (int i = threadIdx.x; i < SORT; i += 512) id[i] = base + i < n ? key_of(ids[base + i], vocab) : 0xffffffffu;
  __syncthreads();
  const unsigned mine = id[q * 64 + lane];
  int count = 0;
  for (int g = wave * 4; g < wave * 4 + 4; g++) {
    const unsigned limit = g < q ? mine + 1 : mine;
#pragma unroll
    for (int j = 0; j < 64; j++) count += id[g * 64 + j] < limit;
    if (g == q) {
#pragma unroll 1
      for (int j = 0; j < lane; j++) count += id[g * 64 + j] == mine;
    }
  }
  below[wave][lane] = count;
  __syncthreads();
  if (wave != 0 || base + q * 64 + lane >= n) return;
#pragma unroll
  for (int s = 1; s < 8; s++) count += below[s][lane];
  // fewer than the block's tokens are before a token of it
  key[base + count] = mine;
  row[base + count] = (int32_t)(base + q * 64 + lane);
}

// A token's place among `ways` sorted blocks of `size` tokens: eight threads a
// token, each with the ranks in every eighth block.
__global__ void __launch_bounds__(256)
    merge_kernel(const unsigned *__restrict__ key, const int32_t *__restrict__ row, unsigned *__restrict__ key2,
                 int32_t *__restrict__ row2, long n, long size, int ways) {
  const long i = (long)blockIdx.x * 32 + threadIdx.x / 8;
  const int part = threadIdx.x & 7;
  long place = 0, first = 0;
  unsigned mine = 0;
  if (i < n) {
    mine = key[i];
    const long block = i / size;
    first = block / ways * ways;
    for (long b = first + part; b < first + ways && b * size < n; b += 8) {
      if (b == block) {
        place += i - b * size;
        continue;
      }
      const unsigned limit = b < block ? mine + 1 : mine;  // equal ones of earlier blocks come first
      const unsigned *p = key + b * size;
      const long end = n - b * size < size ? n - b * size : size;
      long lo = 0, hi = end;  // the first that is not below the limit
      while (lo < hi) {
        const long mid = (lo + hi) >> 1;
        if (p[mid] < limit) lo = mid + 1;
        else hi = mid;
      }
      place += lo;
    }
  }
  place += __shfl_xor(place, 1);
  place += __shfl_xor(place, 2);
  place += __shfl_xor(place, 4);
  if (i < n && part == 0) {
    key2[first * size + place] = mine;
    row2[first * size + place] = row[i];
  }
}

// ---------------------------------------------------------------- sums

// The columns of a lane: four, or of the last group those that no other has; with
// V = float (rows under four columns) one.
template <class V>
struct Columns;
template <>
struct Columns<f32x4> {
  long at;
  int from;  // the first of its own; 4: none
  __device__ __forceinline__ Columns(long n, long cols) {
    const long c = n * 4;
    at = c > cols - 4 ? cols - 4 : c;
    from = c >= cols ? 4 : (int)(c - at);
  }
  __device__ __forceinline__ f32x4 load(const float *p) const { return *(const f32x4_any *)(p + at); }
  template <bool ADD>
  __device__ __forceinline__ void store(float *p, f32x4 v) const {
    p += at;
    if (from == 0) {
      if (ADD) v += *(const f32x4_any *)p;
      *(f32x4_any *)p = v;
    } else {
#pragma unroll
      for (int j = 1; j < 4; j++)
        if (j >= from) p[j] = ADD ? p[j] + v[j] : v[j];
    }
  }
};
template <>
struct Columns<float> {
  long at;
  int from;
  __device__ __forceinline__ Columns(long n, long cols) : at(n), from(n < cols ? 0 : 4) {}
  __device__ __forceinline__ float load(const float *p) const { return p[at]; }
  template <bool ADD>
  __device__ __forceinline__ void store(float *p, float v) const {
    p[at] = ADD ? p[at] + v : v;
  }
};

// part[tile][0]: of the run that comes from the tile before; [1]: of the one that
// begins here and goes on into the next.
template <class V, int LANES, bool ADD>
__global__ void __launch_bounds__(256)
    sum_kernel(const unsigned *__restrict__ key, const int32_t *__restrict__ row, const float *__restrict__ dy,
               float *__restrict__ dw, float *__restrict__ part, long n, long tiles, long cols, float scale) {
  constexpr int GROUPS = 256 / LANES, AT_ONCE = 8;
  __shared__ unsigned ids[GROUPS][TILE + 2];
  __shared__ int32_t rows[GROUPS][TILE];
  const long t0 = (long)blockIdx.x * GROUPS;
  for (int i = threadIdx.x; i < GROUPS * (TILE + 2); i += 256) {
    const int g = i / (TILE + 2), k = i % (TILE + 2);
    const long at = (t0 + g) * TILE + k - 1;
    // outside: a token that none is equal to (no run passes the ends)
    ids[g][k] = at >= 0 && at < n ? key[at] : 0xffffffffu;
    if (k > 0 && k <= TILE) rows[g][k - 1] = at < n ? row[at] : 0;
  }
  __syncthreads();
  const int g = threadIdx.x / LANES;
  const long tile = t0 + g;
  const Columns<V> col((long)blockIdx.y * LANES + threadIdx.x % LANES, cols);
  if (tile >= tiles || col.from == 4) return;
  V sum = {};
  bool inside = ids[g][0] != ids[g][1];  // the run began in this tile
#pragma unroll 1
  for (int k0 = 0; k0 < TILE; k0 += AT_ONCE) {
    if (ids[g][k0 + 1] >= NONE) return;  // none of the table's from here on
    V v[AT_ONCE];
#pragma unroll
    for (int k = 0; k < AT_ONCE; k++) v[k] = col.load(dy + (long)rows[g][k0 + k] * cols);
#pragma unroll
    for (int k = 0; k < AT_ONCE; k++) {
      const unsigned id = ids[g][k0 + k + 1];
      if (id >= NONE) return;
      sum += v[k];
      const bool ends = ids[g][k0 + k + 2] != id;
      if (ends || k0 + k == TILE - 1) {
        if (ends && inside)
          col.template store<ADD>(dw + (long)id * cols, sum * scale);
        else
          col.template store<false>(part + (tile * 2 + (inside ? 1 : 0)) * cols, sum);
        sum = V{};
        inside = true;
      }
    }
  }
}

// The tile that a run begins in and does not end in adds its parts: the
// workgroup's groups of lanes take shares of consecutive tiles, joined in order.
template <class V, int LANES, bool ADD>
__global__ void __launch_bounds__(256)
    sum_parts_kernel(const unsigned *__restrict__ key, const float *__restrict__ part, float *__restrict__ dw,
                     long n, long cols, float scale) {
  constexpr int GROUPS = 256 / LANES;
  __shared__ V sums[GROUPS][LANES];
  const long tile = blockIdx.x, last = tile * TILE + TILE - 1;
  if (last + 1 >= n) return;
  const unsigned id = key[last];
  if (id >= NONE || key[last + 1] != id) return;                      // no run goes on from here
  if (tile > 0 && key[tile * TILE] == id && key[tile * TILE - 1] == id) return;  // it began before
  long lo = last + 1, hi = n;
  while (lo < hi) {  // its end
    const long mid = (lo + hi) >> 1;
    if (key[mid] <= id) lo = mid + 1;
    else hi = mid;
  }
  const long more = (lo - 1) / TILE - tile;  // tiles that it goes on in
  const int g = threadIdx.x / LANES;
  const Columns<V> col((long)blockIdx.y * LANES + threadIdx.x % LANES, cols);
  V sum = {};
  if (col.from < 4) {
    if (g == 0) sum = col.load(part + (tile * 2 + 1) * cols);
    const long each = (more + GROUPS - 1) / GROUPS, from = g * each, to = from + each < more ? from + each : more;
#pragma unroll 8
    for (long k = from; k < to; k++) sum += col.load(part + (tile + 1 + k) * 2 * cols);
  }
  sums[g][threadIdx.x % LANES] = sum;
  __syncthreads();
  if (g || col.from == 4) return;
#pragma unroll
  for (int k = 1; k < GROUPS; k++) sum += sums[k][threadIdx.x % LANES];
  col.template store<ADD>(dw + (long)id * cols, sum * scale);
}

bool good(long rows, long vocab, long cols) {
  // grid axes: 8 threads a row, 65535 groups of 64 lanes with 4 columns each
  return rows > 0 && vocab > 0 && cols > 0 && rows <= 1L << 28 && vocab <= 1L << 30 && cols <= 1L << 22;
}

long tiles_of(long rows) { return (rows + TILE - 1) / TILE; }

// Lanes that share a row: those that leave the fewest idle (of long rows, at
// most one wave in sixteen).
int lanes_of(long cols) {
  const long groups = (cols + 3) / 4;
  if (groups > 1024) return 64;
  int best = 64;
  for (int l = 32; l >= 8; l /= 2)
    if ((groups + l - 1) / l * l < (groups + best - 1) / best * best) best = l;
  return best;
}

}  // namespace

extern "C" int tt_k_embedding_fwd(const float *w, const int32_t *ids, float *y, long rows, long vocab, long cols,
                                  float scale) {
  if (!w || !ids || !y || !good(rows, vocab, cols)) return -1;
  if (ttrt_init() != 0) return -3;
  const long groups = (cols + 3) / 4;
#define RUN(TX, R, VEC)                                                                                             \
  {                                                                                                                 \
    const long gx = (rows + 256 / TX * R - 1) / (256 / TX * R), gy = ((VEC ? groups : cols) + TX - 1) / TX;         \
    hipLaunchKernelGGL((embed_kernel<TX, R, VEC>), dim3((unsigned)(gx < 1 << 20 ? gx : 1 << 20), (unsigned)(gy < 1024 ? gy : 1024)), \
                       dim3(256), 0, stream(), w, ids, y, rows, vocab, cols, scale);                                \
  }
  if (cols < 4) RUN(4, 1, false)
  else if (groups <= 16) RUN(16, 1, true)
  else if (groups <= 64) RUN(64, 1, true)
  else RUN(256, 1, true)
#undef RUN
  return launched();
}

// the sorted tokens and their rows, twice (a merge reads one and writes the
// other), and two parts a tile
extern "C" size_t tt_k_embedding_bwd_ws(long rows, long vocab, long cols) {
  if (!good(rows, vocab, cols)) return 0;
  return 16 * (size_t)((rows + 3) / 4 * 4) + 8 * (size_t)tiles_of(rows) * (size_t)cols;
}

extern "C" int tt_k_embedding_bwd(const int32_t *ids, const float *dy, float *dw, long rows, long vocab, long cols,
                                  float scale, int accumulate, void *ws) {
  if (!ids || !dy || !dw || !good(rows, vocab, cols)) return -1;
  if (ttrt_init() != 0) return -3;
  void *own = NULL;
  if (!ws) ws = own = ttrt_alloc(tt_k_embedding_bwd_ws(rows, vocab, cols));
  if (!ws) return -2;
  const long padded = (rows + 3) / 4 * 4, tiles = tiles_of(rows);
  unsigned *key = (unsigned *)ws, *key2 = key + 2 * padded;
  int32_t *row = (int32_t *)(key + padded), *row2 = row + 2 * padded;
  float *part = (float *)(key + 4 * padded);
  const unsigned sorters = (unsigned)((rows + SORT - 1) / SORT * (SORT / 64));
  const long values = accumulate ? 0 : vocab * cols, clearers = (values + 8191) / 8192;
  hipLaunchKernelGGL(sort_kernel, dim3(sorters + (unsigned)(clearers < 4096 ? clearers : 4096)), dim3(512), 0,
                     stream(), ids, key, row, rows, vocab, sorters, dw, values);
  for (long size = SORT; size < rows; size *= WAYS) {
    hipLaunchKernelGGL(merge_kernel, dim3((unsigned)((rows + 31) / 32)), dim3(256), 0, stream(), key, row, key2,
                       row2, rows, size, WAYS);
    unsigned *k = key;
    int32_t *r = row;
    key = key2, row = row2, key2 = k, row2 = r;
  }
  const long groups = cols < 4 ? cols : (cols + 3) / 4;
#define RUN(V, LANES, ADD)                                                                                          \
  {                                                                                                                 \
    const unsigned chunks = (unsigned)((groups + LANES - 1) / LANES);                                               \
    const long wide = 256 / LANES;                                                                                  \
    hipLaunchKernelGGL((sum_kernel<V, LANES, ADD>), dim3((unsigned)((tiles + wide - 1) / wide), chunks), dim3(256), \
                       0, stream(), key, row, dy, dw, part, rows, tiles, cols, scale);                              \
    if (tiles > 1)                                                                                                  \
      hipLaunchKernelGGL((sum_parts_kernel<V, LANES, ADD>), dim3((unsigned)(tiles - 1), chunks), dim3(256), 0,      \
                         stream(), key, part, dw, rows, cols, scale);                                               \
    break;                                                                                                          \
  }
#define BY_LANES(ADD)                      \
  switch (cols < 4 ? 0 : lanes_of(cols)) { \
    case 0: RUN(float, 8, ADD)             \
    case 8: RUN(f32x4, 8, ADD)             \
    case 16: RUN(f32x4, 16, ADD)           \
    case 32: RUN(f32x4, 32, ADD)           \
    default: RUN(f32x4, 64, ADD)           \
  }
  if (accumulate) {
    BY_LANES(true)
  } else {
    BY_LANES(false)
  }
#undef BY_LANES
#undef RUN
  ttrt_free(own);
  return launched();
}
