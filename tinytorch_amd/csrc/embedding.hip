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
//   1. Blocks of tokens are sorted by counting: a token's place is the number of
//      the block's tokens that are smaller, or equal and before it.  Every pair is
//      compared, 16 to 64 tokens a workgroup, so the work spreads over the GPU where
//      a sort by exchanges has one workgroup a block.  Beside it the table's gradient
//      is cleared.
//   2. Up to WAYS sorted blocks at a time are merged: a token's place is the sum
//      of its ranks in all of them, each by bisection.  (Not for one block.)
//   3. Each group of lanes adds the rows of TILE tokens in sorted order.  A run of
//      one token that lies inside is written; one that passes an end of the tile
//      is left as a part.
//   4. The parts of such runs are added by the tile that the run begins in.
//
// A few tokens (up to FEW) are not sorted: a wave for each looks for its equals in
// LDS and adds their rows if it is the first of them, all in one launch.
//
// us a launch (tokens as often as words are):
//   tokens x columns, rows of the table   1    sort, clear    merge    sum    parts
//   8192 x 1024 of 32000                 11         18           -      10      6
//   4099 x 259 of 1003                  3.6        5.4           -     5.2    5.8
//   32768 x 1024 of 131072               42         83           9      66      7
// The first is 6.3 TB/s of the rows read and written (some from the last cache), the
// clearing of 537 MB 6.5; the sums read 134 MB behind it, 2.8 TB/s of reads and
// writes whatever the tile is (8, 16 or 32 tokens, all loads at once or two groups).
#include <hip/hip_runtime.h>
#include <stdint.h>
#include "tt_rt.h"

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef f32x4 __attribute__((aligned(4))) f32x4_any;  // any float's alignment

inline hipStream_t stream() { return (hipStream_t)ttrt_stream(); }
inline int launched() { return hipGetLastError() == hipSuccess ? 0 : -3; }

constexpr unsigned NONE = 0xfffffffeu;  // a token outside the table: behind all others
constexpr int WAYS = 32, FEW = 512;

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

// zeros from `clear` on, by workgroup b of n
template <int THREADS>
__device__ __forceinline__ void clear_all(float *clear, long values, unsigned b, unsigned n) {
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  for (long i = ((long)b * THREADS + threadIdx.x) * 4; i < values; i += (long)n * THREADS * 4) {
    if (i + 4 <= values) {
      *(f32x4_any *)(clear + i) = zero;
    } else {
      for (long j = i; j < values; j++) clear[j] = 0.f;
    }
  }
}

// Workgroup q of a block of BLOCK tokens places E of them, from E q on.  A wave
// counts in its share of the block, every E lanes in a part of that: equal tokens
// before one count too, so of the groups of E before its own all that are below its
// successor.  The fewer tokens, the fewer a workgroup: what it takes is E times the
// block's comparisons.  The workgroups
// behind the sorters clear the table's gradient.
template <int BLOCK, int WAVES, int E>
__global__ void __launch_bounds__(WAVES * 64)
    sort_kernel(const int32_t *__restrict__ ids, unsigned *__restrict__ key, int32_t *__restrict__ row, long n,
                long vocab, unsigned sorters, float *__restrict__ clear, long values) {
  if (blockIdx.x >= sorters) {
    clear_all<WAVES * 64>(clear, values, blockIdx.x - sorters, gridDim.x - sorters);
    return;
  }
  typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
  constexpr int PARTS = WAVES * 64 / E;
  __shared__ __attribute__((aligned(16))) unsigned id[BLOCK];
  __shared__ int below[WAVES][E];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), e = lane % E;
  const long base = (long)(blockIdx.x / (BLOCK / E)) * BLOCK;
  const int q = blockIdx.x % (BLOCK / E), have = (int)(n - base < BLOCK ? n - base : BLOCK);
  if (q * E >= have) return;
  for (int i = threadIdx.x; i < BLOCK; i += WAVES * 64) id[i] = i < have ? key_of(ids[base + i], vocab) : 0xffffffffu;
  __syncthreads();
  const unsigned mine = id[q * E + e];
  int count = 0;
  const int part = ((have + PARTS - 1) / PARTS + E - 1) / E * E,  // tokens that a lane looks at
      from = (wave * (64 / E) + lane / E) * part, to = from + part < BLOCK ? from + part : BLOCK;
  for (int c = from; c < to; c += E) {
    const unsigned limit = c < q * E ? mine + 1 : mine;
#pragma unroll
    for (int j = 0; j < E; j += 4) {
      const u32x4 other = *(const u32x4 *)(id + c + j);
#pragma unroll
      for (int x = 0; x < 4; x++) count += other[x] < limit;
    }
  }
  if (wave == 0 && lane < E) {
#pragma unroll 8
    for (int j = 0; j < E; j++) count += id[q * E + j] == mine && j < e;
  }
#pragma unroll
  for (int s = E; s < 64; s <<= 1) count += __shfl_xor(count, s);
  if (lane < E) below[wave][e] = count;
  __syncthreads();
  if (wave != 0 || lane >= E || q * E + e >= have) return;
#pragma unroll
  for (int s = 1; s < WAVES; s++) count += below[s][e];
  // fewer than the block's tokens are before a token of it
  key[base + count] = mine;
  row[base + count] = (int32_t)(base + q * E + e);
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
template <class V, int LANES, int TILE, bool ADD>
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
  if (ids[g][1] >= NONE) return;
  V v[AT_ONCE], next[AT_ONCE];
#pragma unroll
  for (int k = 0; k < AT_ONCE; k++) next[k] = col.load(dy + (long)rows[g][k] * cols);
#pragma unroll 1
  for (int k0 = 0; k0 < TILE; k0 += AT_ONCE) {
#pragma unroll
    for (int k = 0; k < AT_ONCE; k++) v[k] = next[k];
    // the rows behind are on their way while these are added (tokens of none: row 0
    // or their own, not added)
    if (k0 + AT_ONCE < TILE) {
#pragma unroll
      for (int k = 0; k < AT_ONCE; k++) next[k] = col.load(dy + (long)rows[g][k0 + AT_ONCE + k] * cols);
    }
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
template <class V, int LANES, int TILE, bool ADD>
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
  long more = 0;  // tiles that it goes on in: those that begin with it
  for (int here = 256; here == 256; more += here) {
    const long at = (tile + 1 + more + threadIdx.x) * TILE;
    here = __syncthreads_count(at < n && key[at] == id);
  }
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

// ---------------------------------------------------------------- a few tokens

// Wave w of workgroup b has token 4 b + w; the workgroups behind those clear rows,
// but for the batch's, each a share of the table.
template <class V, bool ADD>
__global__ void __launch_bounds__(256)
    few_kernel(const int32_t *__restrict__ ids, const float *__restrict__ dy, float *__restrict__ dw, int n, long vocab,
               long cols, float scale, unsigned adders) {
  __shared__ unsigned id[FEW];
  __shared__ unsigned short equal[4][FEW];
  for (int i = threadIdx.x; i < n; i += 256) id[i] = key_of(ids[i], vocab);
  __syncthreads();
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (blockIdx.x >= adders) {
    const unsigned wgs = gridDim.x - adders;
    if (blockIdx.y != 0) return;
    // a wave a row
    for (long r = (long)(blockIdx.x - adders) * 4 + wave; r < vocab; r += (long)wgs * 4) {
      bool taken = false;
      for (int c = 0; c < n; c += 64) taken |= c + lane < n && id[c + lane] == (unsigned)r;
      if (__any(taken)) continue;
      float *p = dw + r * cols;
      for (long i = lane * 4; i < cols; i += 256) {
        if (i + 4 <= cols) {
          *(f32x4_any *)(p + i) = (f32x4){0.f, 0.f, 0.f, 0.f};
        } else {
          for (long j = i; j < cols; j++) p[j] = 0.f;
        }
      }
    }
    return;
  }
  const int r = (int)blockIdx.x * 4 + wave;
  if (r >= n || id[r] >= NONE) return;
  const unsigned mine = id[r];
  int count = 0;
  for (int c = 0; c < n; c += 64) {
    const bool is = c + lane < n && id[c + lane] == mine;
    const unsigned long long found = __ballot(is);
    if (c <= r && found & (r - c >= 64 ? ~0ull : (1ull << (r - c)) - 1)) return;  // not the first of them
    if (is) equal[wave][count + __popcll(found & ((1ull << lane) - 1))] = (unsigned short)(c + lane);
    count += __popcll(found);
  }
  __builtin_amdgcn_wave_barrier();
  const Columns<V> col((long)blockIdx.y * 64 + lane, cols);
  if (col.from == 4) return;
  V sum = {};
  constexpr int AT_ONCE = 8;
  for (int k = 0; k < count; k += AT_ONCE) {
    V v[AT_ONCE];
#pragma unroll
    for (int j = 0; j < AT_ONCE; j++) v[j] = col.load(dy + equal[wave][k + j < count ? k + j : k] * cols);
#pragma unroll
    for (int j = 0; j < AT_ONCE; j++)
      if (k + j < count) sum += v[j];
  }
  col.template store<ADD>(dw + (long)mine * cols, sum * scale);
}

bool good(long rows, long vocab, long cols) {
  // grid axes: 8 threads a row, 65535 groups of 64 lanes with 4 columns each
  return rows > 0 && vocab > 0 && cols > 0 && rows <= 1L << 28 && vocab <= 1L << 30 && cols <= 1L << 22;
}

// Tokens a tile: few where waves are (8192 x 1024: 13 us by tiles of 32, 9 of 8),
// many where parts would be.
int tile_of(long rows, long cols) { return rows * ((cols + 255) / 256) <= 65536 ? 8 : 32; }
long tiles_of(long rows, long cols) { return (rows + tile_of(rows, cols) - 1) / tile_of(rows, cols); }

// Lanes that share a row: those that leave the fewest idle (of long rows, at
// most one wave in sixteen).
int lanes_of(long cols) {
  const long groups = (cols + 3) / 4;
  if (groups > 192) return 256;  // a workgroup's waves read a row side by side
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
  else if (rows < 4096) RUN(256, 1, true)
  else RUN(256, 4, true)  // 32768 rows of 1024 columns: 45 us with one row a thread, 42 with four
#undef RUN
  return launched();
}

// the sorted tokens and their rows, twice (a merge reads one and writes the
// other), and two parts a tile
extern "C" size_t tt_k_embedding_bwd_ws(long rows, long vocab, long cols) {
  if (!good(rows, vocab, cols) || rows <= FEW) return 0;
  return 16 * (size_t)((rows + 3) / 4 * 4) + 8 * (size_t)tiles_of(rows, cols) * (size_t)cols;
}

extern "C" int tt_k_embedding_bwd(const int32_t *ids, const float *dy, float *dw, long rows, long vocab, long cols,
                                  float scale, int accumulate, void *ws) {
  if (!ids || !dy || !dw || !good(rows, vocab, cols)) return -1;
  if (ttrt_init() != 0) return -3;
  const long groups = cols < 4 ? cols : (cols + 3) / 4, values = accumulate ? 0 : vocab * cols;
  if (rows <= FEW) {
    const unsigned adders = (unsigned)((rows + 3) / 4), chunks = (unsigned)((groups + 63) / 64);
    const long clearers = accumulate ? 0 : (vocab + 15) / 16;
    const dim3 grid(adders + (unsigned)(clearers < 4096 ? clearers : 4096), chunks);
#define RUN(V, ADD)                                                                                                   \
  hipLaunchKernelGGL((few_kernel<V, ADD>), grid, dim3(256), 0, stream(), ids, dy, dw, (int)rows, vocab, cols, scale, \
                     adders)
    if (accumulate) {
      if (cols < 4) RUN(float, true);
      else RUN(f32x4, true);
    } else {
      if (cols < 4) RUN(float, false);
      else RUN(f32x4, false);
    }
#undef RUN
    return launched();
  }
  void *own = NULL;
  if (!ws) ws = own = ttrt_alloc(tt_k_embedding_bwd_ws(rows, vocab, cols));
  if (!ws) return -2;
  const long padded = (rows + 3) / 4 * 4, tiles = tiles_of(rows, cols);
  unsigned *key = (unsigned *)ws, *key2 = key + 2 * padded;
  int32_t *row = (int32_t *)(key + padded), *row2 = row + 2 * padded;
  float *part = (float *)(key + 4 * padded);
  // one block is sorted without a merge; of more tokens every pair would cost too much
  const bool whole = rows <= 8192;
  const long block = whole ? 8192 : 2048, clearers = (values + 8191) / 8192;
  const unsigned extra = (unsigned)(clearers < 4096 ? clearers : 4096);
#define SORT(BLOCK, WAVES, E)                                                                                     \
  {                                                                                                               \
    const unsigned sorters = (unsigned)((rows + BLOCK - 1) / BLOCK * (BLOCK / E)),                                \
                   some = (unsigned)(whole ? (rows + E - 1) / E : sorters);                                       \
    hipLaunchKernelGGL((sort_kernel<BLOCK, WAVES, E>), dim3(some + extra), dim3(WAVES * 64), 0, stream(), ids,    \
                       key, row, rows, vocab, some, dw, values);                                                  \
  }
  // beside a long clearing the sort is on half of the CUs (8192 tokens, 131 MB: 18 us, on all 22)
  if (whole && values > 1 << 24) SORT(8192, 16, 64)
  else if (rows <= 5000) SORT(8192, 16, 16)
  else if (whole) SORT(8192, 16, 32)
  else SORT(2048, 8, 64)
#undef SORT
  for (long size = block; size < rows; size *= WAYS) {
    hipLaunchKernelGGL(merge_kernel, dim3((unsigned)((rows + 31) / 32)), dim3(256), 0, stream(), key, row, key2,
                       row2, rows, size, WAYS);
    unsigned *k = key;
    int32_t *r = row;
    key = key2, row = row2, key2 = k, row2 = r;
  }
#define RUN(V, LANES, TILE, ADD)                                                                                     \
  {                                                                                                                  \
    const unsigned chunks = (unsigned)((groups + LANES - 1) / LANES);                                                \
    const long wide = 256 / LANES;                                                                                   \
    hipLaunchKernelGGL((sum_kernel<V, LANES, TILE, ADD>), dim3((unsigned)((tiles + wide - 1) / wide), chunks),       \
                       dim3(256), 0, stream(), key, row, dy, dw, part, rows, tiles, cols, scale);                    \
    if (tiles > 1)                                                                                                   \
      hipLaunchKernelGGL((sum_parts_kernel<V, LANES == 256 ? 64 : LANES, TILE, ADD>),                                \
                         dim3((unsigned)(tiles - 1), LANES == 256 ? (unsigned)((groups + 63) / 64) : chunks),        \
                         dim3(256), 0, stream(), key, part, dw, rows, cols, scale);                                  \
    break;                                                                                                           \
  }
#define BY_LANES(TILE, ADD)                \
  switch (cols < 4 ? 0 : lanes_of(cols)) { \
    case 0: RUN(float, 8, TILE, ADD)       \
    case 8: RUN(f32x4, 8, TILE, ADD)       \
    case 16: RUN(f32x4, 16, TILE, ADD)     \
    case 32: RUN(f32x4, 32, TILE, ADD)     \
    case 64: RUN(f32x4, 64, TILE, ADD)     \
    default: RUN(f32x4, 256, TILE, ADD)    \
  }
  if (tile_of(rows, cols) == 8) {
    if (accumulate) {
      BY_LANES(8, true)
    } else {
      BY_LANES(8, false)
    }
  } else if (accumulate) {
    BY_LANES(32, true)
  } else {
    BY_LANES(32, false)
  }
#undef BY_LANES
#undef RUN
  ttrt_free(own);
  return launched();
}
