// Lookup of table rows by token (atomic number, species pair, ..) with a scale, and its gradient: the sum of the rows'
// gradients by token.  Replaces the indexing of the training step's first convolution and of the expert readout's
// table of scores, whose gradient was an atomic addition into a handful of rows
// (models/pure_cartesian_sparse_layers.py:258-259 embeds the species of every atom).
//   out_i = scale table[index_i], a given value (zeros) where index_i lies outside the table
//   dtable_v = scale sum over i with index_i = v, in 32 bits and an order that the sizes alone give
//
// Bound by memory: rows x width values written forward, read backward.  Measured (a fill of 400 MB takes 59 us, torch's sum of it
// 106 us): 520,000 x 192 fp32 into 9 rows 58 us forward (6.9 TB/s; 95 us in a pass with its gradient, which reads what is not yet
// written back) and 81 us backward (4.9 TB/s), into 100 rows by the sort 111 us (3.6 TB/s), into 1,000 rows 137 us; 8,125 x
// 12,288 into 16 rows 59 and 79 us; 65,536 x 331 bf16 into 30,011 rows 13 and 53 us, 28 us of those the sort; 32 x 16 a launch each.
#include <algorithm>

#include "common.h"
#include "expert_types.h"
#include "fsctep.h"

namespace fsc {
namespace embed {

constexpr int NT = 256;

// runs the statement with FULL whether the condition holds
#define FSC_EMBED_FULL(condition, ...)                           \
  {                                                              \
    if (condition) { constexpr bool FULL = true; __VA_ARGS__; }  \
    else { constexpr bool FULL = false; __VA_ARGS__; }           \
  }

struct Args {
  int64_t rows, stride;        // row stride of the table (forward) or of dy (backward), in elements
  int64_t table_rows;
  int width;
  float scale;
  const void *in, *index;
  void* out;
  float outside;               // forward: what stands where a token has no row
};

template <typename T>
struct Vec {
  static constexpr int N = 16 / sizeof(T);     // values of a vector
};
// A vector of M values from p on, by one load; not FULL: a row shorter than a vector, n values and zeros behind them.  FULL is known
// when the kernel is compiled: a branch at every load would have each wait for the one before.
template <bool FULL, int M, typename T>
__device__ __forceinline__ void load_some(const T* p, int n, float (&v)[M]) {
  if constexpr (FULL) {
    struct alignas(sizeof(T)) Pack { T t[M]; };
    const Pack k = *reinterpret_cast<const Pack*>(p);
#pragma unroll
    for (int j = 0; j < M; ++j) v[j] = to_f(k.t[j]);
  } else {
#pragma unroll
    for (int j = 0; j < M; ++j) v[j] = j < n ? to_f(p[j < n ? j : 0]) : 0.f;
  }
}
template <bool FULL, int M, typename T>
__device__ __forceinline__ void store_some(T* p, int n, const float (&v)[M]) {
  if constexpr (FULL) {
    struct alignas(sizeof(T)) Pack { T t[M]; };
    Pack k;
#pragma unroll
    for (int j = 0; j < M; ++j) k.t[j] = from_f<T>(v[j]);
    *reinterpret_cast<Pack*>(p) = k;
  } else {
#pragma unroll
    for (int j = 0; j < M; ++j)
      if (j < n) p[j] = from_f<T>(v[j]);
  }
}

// ---------------------------------------------------------------- lookup
// A row's vector a thread.  Where no vector divides the width, a row's last one lies at its end and writes some of the values
// before it once more (the same ones); rows shorter than a vector are one vector that is not full.  Bound by the stores,
// which go past the caches: what they write is read by other kernels, on other XCDs (520,000 x 192: 58 us, a fill of that
// size 59 us; ordinary stores 95 us; four vectors a thread 69 and 86 us).
template <typename T, typename I, bool FULL>
__global__ __launch_bounds__(NT) void lookup_kernel(Args a, int64_t first, uint32_t vectors) {
  constexpr int N = Vec<T>::N;
  const int64_t f0 = first + (int64_t)blockIdx.x * NT, r0 = f0 / vectors;     // the block's first vector, in row r0
  if (f0 + threadIdx.x >= a.rows * vectors) return;
  const uint32_t local = (uint32_t)(f0 - r0 * vectors) + threadIdx.x, up = local / vectors;
  const int n = FULL ? N : a.width, col = std::min((int)(local - up * vectors) * N, a.width - n);
  const int64_t row = r0 + up, t = ((const I*)a.index)[row];
  const bool there = t >= 0 && t < a.table_rows;
  float v[N];
  load_some<FULL, N>((const T*)a.in + (there ? t : 0) * a.stride + col, n, v);
#pragma unroll
  for (int j = 0; j < N; ++j) v[j] = there ? a.scale * v[j] : a.outside;
  T* out = (T*)a.out + row * a.width + col;
  if constexpr (FULL) {
    typedef unsigned u4s __attribute__((ext_vector_type(4), aligned(2)));
    struct Pack { T t[N]; } k;
#pragma unroll
    for (int j = 0; j < N; ++j) k.t[j] = from_f<T>(v[j]);
    __builtin_nontemporal_store(__builtin_bit_cast(u4s, k), reinterpret_cast<u4s*>(out));
  } else {
    store_some<false, N>(out, n, v);
  }
}

// ---------------------------------------------------------------- gradient, few tokens
// A block owns a row of the table and a vector a lane of its columns, its waves look through a share of the tokens each, 64 at a
// time, and add the rows they find, AHEAD on their way; one launch, no sort.  Eight waves a block where the chip holds all blocks at
// once, four where it does not (1,024 tokens by four and eight: 64 columns of 100 rows, all of one token, 17.7 and 11.0 us; 640
// columns of 5,000 rows 13.7 and 19.1 us).  For up to 2,048 tokens and 2^23 pairs of token and row to look at (by it and by the
// sort: 2,048 tokens, 640 columns of 100 rows 5.8 and 21.0 us, all of one token 28.7 and 18.7 us; 1,024 of 5,000 rows 13.7 and 29.4
// us; 256 of 30,000 rows x 331 24.6 and 33.5 us, 1,024 40.2 and 35.6 us), and 2^25 for those pairs times the blocks of columns,
// each of which looks through the tokens again (fp32: 1,024 tokens of 1,600 rows x 4,096 29.3 and 35.5 us, 2,048 tokens 47.9 and
// 37.9 us, of 1,600 rows x 12,288 156 and 70 us, of 4,000 rows 331 and 95 us; bf16: 256 of 30,000 rows x 2,048 54.9 and 55.4 us,
// 1,024 of 1,600 rows x 12,288 48.6 and 45.8 us).  512 tokens where the table is small (192 columns of 9 rows, all of one token: 512 tokens 6.3
// and 7.6 us, 1,024 tokens 11.1 and 7.9 us; 12,288 columns of 24 rows 6.6 and 27.1 us).
inline bool few(int64_t rows, int64_t table_rows, int width, int size);
template <int WAVES, typename T, typename I, bool FULL>
__global__ __launch_bounds__(64 * WAVES) void few_kernel(Args a) {
  constexpr int N = Vec<T>::N, AHEAD = 8;
  __shared__ float red[WAVES][64 * N];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int n = FULL ? N : a.width, first = (blockIdx.y * 64 + lane) * N, col = std::min(first, a.width - n);
  const int per = (int)((a.rows + 64 * WAVES - 1) / (64 * WAVES)) * 64;
  const int i0 = std::min<int>(a.rows, wave * per), i1 = std::min<int>(a.rows, i0 + per);
  for (int64_t v = blockIdx.x; v < a.table_rows; v += gridDim.x) {
    float s[N];
#pragma unroll
    for (int j = 0; j < N; ++j) s[j] = 0.f;
    for (int b = i0; b < i1; b += 64) {
      const int i = b + lane;
      uint64_t hits = __ballot(i < i1 && (int64_t)((const I*)a.index)[std::min(i, i1 - 1)] == v);
      while (hits) {                     // AHEAD rows on their way together, the last one again where there are fewer
        int at = 0, m = 0;
        float u[AHEAD][N];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
          at = hits ? b + __ffsll((unsigned long long)hits) - 1 : at;
          m += hits != 0;
          hits &= hits - 1;
          load_some<FULL, N>((const T*)a.in + at * a.stride + col, n, u[k]);
        }
#pragma unroll
        for (int k = 0; k < AHEAD; ++k)
#pragma unroll
          for (int j = 0; j < N; ++j) s[j] = k < m ? s[j] + u[k][j] : s[j];
      }
    }
#pragma unroll
    for (int j = 0; j < N; ++j) red[wave][lane * N + j] = s[j];
    __syncthreads();
    if (wave == 0 && first < a.width) {
#pragma unroll
      for (int j = 0; j < N; ++j) {
#pragma unroll
        for (int w = 1; w < WAVES; ++w) s[j] += red[w][lane * N + j];
        s[j] *= a.scale;
      }
      store_some<FULL, N>((T*)a.out + v * a.width + col, n, s);
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------- gradient, small tables
// Up to SMALL table rows: no sort.  Every group of lanes adds the rows it streams through, in order and AHEAD on their way, to its
// own copy of 256 columns of the table in LDS; a block's copies are added to a partial table, and those by small_join_kernel.
// More rows leave too few copies for the chip (520,000 x 192 by copies and by the sort: 9 rows 81 and 116 us, 24 rows 105 and
// 111 us, 32 rows 123 and 110 us).
constexpr int SMALL = 24;
inline bool few(int64_t rows, int64_t table_rows, int width, int size) {
  if (table_rows <= SMALL) return rows <= 512;
  if (rows > 2048 || rows * table_rows > 1 << 23) return false;
  const int columns = 64 * (16 / size);                                   // of a block
  return rows * table_rows * ((width + columns - 1) / columns) <= 1 << 25;
}
inline int small_waves(int64_t table_rows) { return table_rows <= 16 ? 4 : 2; }       // at most 64 KB of copies a block
struct Stream {
  int lanes;                             // of a row's columns: four values each, 256 at most for the group
  int64_t range;                         // rows of a block
  float* part;                           // [gridDim.x][table_rows][width]
};

template <typename T, typename I, bool FULL>
__global__ __launch_bounds__(NT) void small_kernel(Args a, Stream s) {
  extern __shared__ __align__(16) float copies[];
  constexpr int AHEAD = 8;
  const int lane = threadIdx.x & 63, L = s.lanes, rows = (int)a.table_rows;
  const int group = threadIdx.x / L, groups = blockDim.x / L;
  const int n = FULL ? 4 : a.width, first = 4 * (lane & (L - 1)), c0 = blockIdx.y * 256;
  const int col = std::min(c0 + first, a.width - n);                     // a row's last vector lies at its end
  float* mine = copies + (int64_t)group * rows * L * 4 + first;          // a row of a copy: L vectors
  for (int i = threadIdx.x; i < groups * rows * L * 4; i += blockDim.x) copies[i] = 0.f;
  __syncthreads();
  const int64_t r0 = blockIdx.x * s.range, r1 = std::min<int64_t>(r0 + s.range, a.rows);
  const T* in = (const T*)a.in + col;
  for (int64_t r = r0 + group; r < r1; r += groups * AHEAD) {
    int64_t t[AHEAD];
    float v[AHEAD][4];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {    // rows past the last one: the last one again, not added
      const int64_t q = std::min<int64_t>(r + k * groups, r1 - 1);
      t[k] = (int64_t)((const I*)a.index)[q];
      load_some<FULL, 4>(in + q * a.stride, n, v[k]);
    }
#pragma unroll
    for (int k = 0; k < AHEAD; ++k)
      if (r + k * groups < r1 && t[k] >= 0 && t[k] < rows) {
        f4* at = reinterpret_cast<f4*>(mine + (int)t[k] * (L * 4));
        *at = *at + f4{v[k][0], v[k][1], v[k][2], v[k][3]};
      }
  }
  __syncthreads();
  float* part = s.part + (int64_t)blockIdx.x * rows * a.width;
  const int vectors = std::min(64, (a.width - c0 + 3) / 4);
  for (int i = threadIdx.x; i < rows * L; i += blockDim.x) {
    const int row = i / L, k = i - row * L;
    if (k >= vectors) continue;
    f4 x = {0.f, 0.f, 0.f, 0.f};
    for (int g = 0; g < groups; ++g) x += *reinterpret_cast<const f4*>(copies + ((int64_t)(g * rows + row) * L + k) * 4);
    const float o[4] = {x.x, x.y, x.z, x.w};
    store_some<FULL, 4>(part + (int64_t)row * a.width + std::min(c0 + 4 * k, a.width - n), n, o);
  }
}

// Adds the partial tables: 64 values a block, 16 waves over the tables, in a fixed order.
template <typename T>
__global__ __launch_bounds__(1024) void small_join_kernel(Args a, const float* __restrict__ part, int n) {
  __shared__ float red[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t values = a.table_rows * a.width, at = (int64_t)blockIdx.x * 64 + lane;
  float x = 0.f;
  if (at < values)
#pragma unroll 8
    for (int i = wave; i < n; i += 16) x += part[i * values + at];
  red[wave][lane] = x;
  __syncthreads();
  if (wave == 0 && at < values) {
    x = 0.f;
#pragma unroll
    for (int w = 0; w < 16; ++w) x += red[w][lane];
    ((T*)a.out)[at] = from_f<T>(a.scale * x);
  }
}

// ---------------------------------------------------------------- gradient, many tokens: sort
// The tokens' numbers sorted by token (a stable radix sort, 8 bits a pass, tokens outside the table last), so that
// sums are over runs of the sorted list.  A pass has counts by digit and block, each digit's counts added up over the blocks, and
// the places: a digit's first place (all smaller digits' totals), the blocks before, the waves before, the lanes before.  Bound
// by its launches (65,536 tokens: 14 us a pass).  A block takes PER tokens a thread: 16 where that leaves a block for every CU,
// 4 otherwise (the whole gradient of 64 columns of 100 rows: 100,000 tokens 35 and 26 us, 2,000,000 tokens 160 and 170 us).
// Up to FEW_BLOCKS blocks each block of the places adds the counts itself, one launch less (BY_DIGIT false: counts [block][digit];
// by themselves and by a scan: 2,000 tokens of 5,000 rows x 331 30.6 and 34.5 us, 32,768 of 5,000 x 64 34.3 and 37.0 us, 65,536 of
// 30,011 x 331 in bf16 53.1 and 53.4 us); more are scanned (counts [digit][block]; 130,000 of 5,000 x 64 52.1 and 49.7 us).
constexpr int DIGITS = 256, FEW_BLOCKS = 64;
inline int per_thread(int64_t rows) { return rows >= (int64_t)256 * 16 * NT ? 16 : 4; }

// key of token i for the sort, from the index (first pass) or the pass before
template <typename I>
struct Source {
  const I* index;
  const int32_t *key, *pos;
  int64_t rows, table_rows;
  __device__ __forceinline__ int32_t key_of(int64_t i) const {
    if (key) return key[i];
    const int64_t t = index[i];
    return (int32_t)(t >= 0 && t < table_rows ? t : table_rows);
  }
  __device__ __forceinline__ int32_t pos_of(int64_t i) const { return key ? pos[i] : (int32_t)i; }
};

// Blocks from `blocks` on fill the table's gradient with zeros (rows that no token names).
template <int PER, bool BY_DIGIT, typename I, typename T>
__global__ __launch_bounds__(NT) void count_kernel(Source<I> src, int shift, int blocks, int32_t* __restrict__ counts,
                                                   T* __restrict__ table, int64_t values) {
  if ((int)blockIdx.x >= blocks) {
    constexpr int N = Vec<T>::N;
    const float zero[N] = {};
    const int64_t step = (int64_t)(gridDim.x - blocks) * NT * N;
    for (int64_t f = ((int64_t)(blockIdx.x - blocks) * NT + threadIdx.x) * N; f < values; f += step)
      if (f + N <= values) store_some<true, N>(table + f, N, zero);
      else store_some<false, N>(table + f, (int)(values - f), zero);
    return;
  }
  __shared__ int cnt[DIGITS];
  cnt[threadIdx.x] = 0;
  __syncthreads();
  const int64_t b0 = (int64_t)blockIdx.x * (NT * PER);
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int64_t i = b0 + k * NT + threadIdx.x;
    if (i < src.rows) atomicAdd(&cnt[src.key_of(i) >> shift & (DIGITS - 1)], 1);   // counts: any order
  }
  __syncthreads();
  counts[BY_DIGIT ? (int64_t)threadIdx.x * blocks + blockIdx.x : (int64_t)blockIdx.x * DIGITS + threadIdx.x] = cnt[threadIdx.x];
}

__device__ __forceinline__ int wave_scan(int v, int lane) {       // inclusive
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int u = __shfl_up(v, off, 64);
    if (lane >= off) v += u;
  }
  return v;
}

// One wave a digit: its counts become the numbers before each block, its total stands behind them.
__global__ __launch_bounds__(64) void scan_kernel(int blocks, int32_t* __restrict__ counts, int32_t* __restrict__ totals) {
  int32_t* c = counts + (int64_t)blockIdx.x * blocks;
  const int lane = threadIdx.x;
  int before = 0;
  for (int b = 0; b < blocks; b += 64) {
    const int v = b + lane < blocks ? c[b + lane] : 0;
    const int s = wave_scan(v, lane);
    if (b + lane < blocks) c[b + lane] = before + s - v;
    before += __shfl(s, 63, 64);
  }
  if (lane == 0) totals[blockIdx.x] = before;
}

// Lanes of the wave with the same digit (lanes that are not `ok` have none).
__device__ __forceinline__ uint64_t peers(int digit, bool ok) {
  uint64_t m = __ballot(ok);
#pragma unroll
  for (int b = 0; b < 8; ++b) {
    const uint64_t v = __ballot(digit >> b & 1);
    m &= (digit >> b & 1) ? v : ~v;
  }
  return m;
}

template <int PER, bool BY_DIGIT, typename I>
__global__ __launch_bounds__(NT) void place_kernel(Source<I> src, int shift, int blocks, const int32_t* __restrict__ counts,
                                                   const int32_t* __restrict__ totals, int32_t* __restrict__ key,
                                                   int32_t* __restrict__ pos) {
  __shared__ int cnt[NT / 64][DIGITS], sums[NT / 64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, d = threadIdx.x;
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) cnt[w][d] = 0;
  // the digit's first place
  int total = 0, blocks_before = 0;
  if (BY_DIGIT) {
    total = totals[d];
    blocks_before = counts[(int64_t)d * blocks + blockIdx.x];
  } else {
#pragma unroll
    for (int b0 = 0; b0 < FEW_BLOCKS; b0 += 16) {
      if (b0 >= blocks) break;
      int v[16];
#pragma unroll
      for (int b = 0; b < 16; ++b) v[b] = counts[std::min(b0 + b, blocks - 1) * DIGITS + d];
#pragma unroll
      for (int b = 0; b < 16; ++b) {
        total += b0 + b < blocks ? v[b] : 0;
        blocks_before += b0 + b < (int)blockIdx.x ? v[b] : 0;
      }
    }
  }
  const int run = wave_scan(total, lane);
  if (lane == 63) sums[wave] = run;
  __syncthreads();
  int base = run - total + blocks_before;
  for (int w = 0; w < wave; ++w) base += sums[w];
  const int64_t w0 = ((int64_t)blockIdx.x * NT + wave * 64) * PER;
  int32_t k[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int64_t i = w0 + j * 64 + lane;
    k[j] = i < src.rows ? src.key_of(i) : -1;
    if (k[j] >= 0) atomicAdd(&cnt[wave][k[j] >> shift & (DIGITS - 1)], 1);
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) {
    const int c = cnt[w][d];
    cnt[w][d] = base;
    base += c;
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const bool ok = k[j] >= 0;
    const int digit = k[j] >> shift & (DIGITS - 1);
    const uint64_t m = peers(digit, ok);
    int at = 0;
    if (ok) at = cnt[wave][digit] + __popcll(m & ((1ull << lane) - 1));
    wave_sync();
    if (ok && (m >> lane) == 1ull) cnt[wave][digit] += __popcll(m);     // the last lane of each digit
    wave_sync();
    if (ok) {
      key[at] = k[j];
      pos[at] = src.pos_of(w0 + j * 64 + lane);
    }
  }
}

// ---------------------------------------------------------------- gradient, many tokens: sums
// The sorted list is cut into shares of `share` tokens.  A group of `lanes` lanes adds a share's rows in order, a vector a lane,
// AHEAD rows on their way; a run of one token that lies within the share goes to the table, one that began
// before it or goes on behind it leaves a partial row (first or second of the share's two), which join_kernel adds.  Bound by the
// gather: a token's rows lie far apart (65,536 x 331 bf16: 15 us, 43 MB).
struct Sums {
  const int32_t *key, *pos;
  int64_t rows, shares;
  int share, lanes, columns;             // columns: groups of lanes that a row's vectors take
  float* part;                           // [shares][2][width]
};

template <typename T, bool FULL>
__global__ __launch_bounds__(NT) void sum_kernel(Args a, Sums s) {
  constexpr int N = Vec<T>::N, AHEAD = 8;
  const int64_t g = ((int64_t)blockIdx.x * NT + threadIdx.x) / s.lanes;
  const int64_t share = g / s.columns;
  if (share >= s.shares) return;
  const int first_col = ((int)(g - share * s.columns) * s.lanes + (threadIdx.x & (s.lanes - 1))) * N;
  if (first_col >= a.width) return;
  const int n = FULL ? N : a.width, col = std::min(first_col, a.width - n);     // a row's last vector lies at its end
  const int64_t p0 = share * s.share, p1 = std::min<int64_t>(p0 + s.share, s.rows);
  const T* in = (const T*)a.in + col;
  float acc[N];
#pragma unroll
  for (int j = 0; j < N; ++j) acc[j] = 0.f;
  int32_t now = s.key[p0];
  const bool before = p0 > 0 && s.key[p0 - 1] == now;
  const int32_t behind = p1 < s.rows ? s.key[p1] : -1;
  bool first = true;
  auto flush = [&](bool end) {
    if (now >= a.table_rows) return;
    const bool head = first && before, tail = end && behind == now;
    if (head || tail) {
      float* out = s.part + (2 * share + (head ? 0 : 1)) * a.width + col;
      store_some<FULL, N>(out, n, acc);
    } else {
      float o[N];
#pragma unroll
      for (int j = 0; j < N; ++j) o[j] = a.scale * acc[j];
      store_some<FULL, N>((T*)a.out + now * (int64_t)a.width + col, n, o);
    }
  };
  for (int64_t p = p0; p < p1; p += AHEAD) {
    int32_t k[AHEAD];
    float v[AHEAD][N];
    const int64_t last = p1 - 1;
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int64_t q = std::min<int64_t>(p + i, last);
      k[i] = s.key[q];
      load_some<FULL, N>(in + s.pos[q] * a.stride, n, v[i]);
    }
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      if (p + i > last) break;
      if (k[i] != now) {
        flush(false);
        first = false;
        now = k[i];
#pragma unroll
        for (int j = 0; j < N; ++j) acc[j] = 0.f;
      }
#pragma unroll
      for (int j = 0; j < N; ++j) acc[j] += v[i][j];
    }
  }
  flush(true);
}

// The number of places from `from` on, `step` apart and below `n`, that hold keys below `v` (OR_EQUAL: or v itself): a
// search by 64 lanes at once.
template <bool OR_EQUAL>
__device__ __forceinline__ int64_t count_below(const int32_t* key, int64_t n, int32_t v, int lane) {
  int64_t lo = 0, hi = n;                // the answer lies in [lo, hi]
  while (hi > lo) {
    const int64_t step = (hi - lo + 63) / 64, at = lo + lane * step;
    const bool below = at < hi && (OR_EQUAL ? key[at] <= v : key[at] < v);
    const int c = __popcll(__ballot(below));
    if (c == 0) return lo;               // the first place looked at is above
    lo += (int64_t)(c - 1) * step + 1;   // one behind the last place that is below
    hi = std::min<int64_t>(hi, lo + step - 1);
  }
  return lo;
}

// Adds the partial rows of one token: 256 columns a block, four a lane, eight waves over the rows, narrow rows several
// to a wave.  BY_TOKEN: a block a token, which writes the zeros of one that is not there; otherwise a block a share, which does
// nothing unless a token's run begins in it and goes on.
constexpr int JT = 512, JW = JT / 64;
template <typename T, bool BY_TOKEN, bool FULL>
__global__ __launch_bounds__(JT) void join_kernel(Args a, Sums s) {
  __shared__ float red[JW][256];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int c0 = blockIdx.y * 256, wide = std::min(256, a.width - c0);
  T* out = (T*)a.out + c0;
  int32_t v;
  int64_t s0, s1;                        // the shares it lies in
  if (BY_TOKEN) {
    v = (int32_t)blockIdx.x;
    const int64_t b = count_below<false>(s.key, s.rows, v, lane);
    if (b >= s.rows || s.key[b] != v) {
      if ((int)threadIdx.x < wide) out[v * (int64_t)a.width + threadIdx.x] = from_f<T>(0.f);
      return;
    }
    s0 = b / s.share;
    const int64_t p1 = (s0 + 1) * s.share;
    if (p1 >= s.rows || s.key[p1] != v) return;
    s1 = (p1 + count_below<true>(s.key + p1, s.rows - p1, v, lane) - 1) / s.share;
  } else {
    s0 = blockIdx.x;
    const int64_t p0 = s0 * s.share, p1 = p0 + s.share;
    if (p1 >= s.rows) return;
    v = s.key[p1 - 1];
    if (v >= a.table_rows || s.key[p1] != v || (p0 > 0 && s.key[p0 - 1] == v)) return;
    s1 = (p1 + count_below<true>(s.key + p1, s.rows - p1, v, lane) - 1) / s.share;
  }
  const int vectors = (wide + 3) / 4;
  int cols = 1;                          // lanes of a row: a power of two
  while (cols < vectors) cols <<= 1;
  const int per = 64 / cols, sub = lane / cols, n = FULL ? 4 : a.width;
  const int col = std::min(c0 + 4 * (lane & (cols - 1)), a.width - n);   // a row's last vector lies at its end
  const int64_t m = s1 - s0 + 1;         // partial rows: the second of s0, the first of the others
  float x[4] = {0.f, 0.f, 0.f, 0.f};
  const float* part = s.part + col;
  for (int64_t i = (int64_t)wave * per + sub; i < m; i += 8 * JW * per) {
    float u[8][4];
#pragma unroll
    for (int k = 0; k < 8; ++k) {        // rows past the last one: the last one again, not added
      const int64_t r = std::min<int64_t>(i + k * JW * per, m - 1);
      load_some<FULL, 4>(part + (2 * (s0 + r) + (r == 0 ? 1 : 0)) * a.width, n, u[k]);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (i + k * JW * per < m)
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] += u[k][j];
  }
  for (int off = cols; off < 64; off <<= 1)
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] += __shfl_xor(x[j], off, 64);
  if (sub == 0)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < n && col + j >= c0) red[wave][col + j - c0] = x[j];
  __syncthreads();
  if ((int)threadIdx.x < wide) {
    float y = 0.f;
    for (int w = 0; w < JW; ++w) y += red[w][threadIdx.x];
    out[v * (int64_t)a.width + threadIdx.x] = from_f<T>(a.scale * y);
  }
}

// Workspace of the gradient: the sorted tokens and their numbers, twice, the counts, and the partial rows.
struct Layout {
  int passes, share, lanes, columns;
  int64_t blocks, shares, key[2], pos[2], counts, totals, part, bytes;
};
Layout layout_of(int64_t rows, int width, int64_t table_rows, int size) {
  Layout l{};
  const int64_t vectors = (width + 16 / size - 1) / (16 / size);
  // a row's vectors go to groups of 16, 32 or 64 lanes, whichever leaves the fewest lanes idle; short rows take fewer lanes
  l.lanes = 4;
  while (l.lanes < 64 && l.lanes < vectors) l.lanes *= 2;
  for (int k = l.lanes / 2; k >= 16; k /= 2)
    if ((vectors + k - 1) / k * k < (vectors + l.lanes - 1) / l.lanes * l.lanes) l.lanes = k;
  l.columns = (int)((vectors + l.lanes - 1) / l.lanes);
  l.passes = 1;
  while (l.passes < 4 && (table_rows >> (8 * l.passes))) ++l.passes;
  l.blocks = (rows + NT * per_thread(rows) - 1) / (NT * per_thread(rows));
  // shares of 32 tokens, more where there would be more than 8,192 shares, whose partial rows take long to join (65,536 x 331 in
  // bf16 by 16, 32, 64 tokens: 58, 54, 57 us)
  l.share = (int)std::min<int64_t>(1024, std::max<int64_t>(32, rows / 8192));
  l.shares = (rows + l.share - 1) / l.share;
  int64_t at = 0;
  auto take = [&](int64_t n) {
    const int64_t was = at;
    at += (4 * n + 63) / 64 * 64;
    return was;
  };
  for (int i = 0; i < 2; ++i) {
    l.key[i] = take(rows);
    l.pos[i] = take(rows);
  }
  l.counts = take(DIGITS * l.blocks);
  l.totals = take(DIGITS);
  l.part = take(2 * l.shares * width);
  l.bytes = at;
  return l;
}

// Blocks of a small table's sums: as many as the copies let the chip hold, four waves a SIMD at most.
struct SmallLayout {
  int lanes, chunks, waves, blocks;
  int64_t range, bytes;
};
SmallLayout small_layout(int64_t rows, int width, int64_t table_rows) {
  SmallLayout l{};
  l.chunks = (width + 255) / 256;
  l.lanes = 1;
  while (l.lanes < 64 && 4 * l.lanes < width) l.lanes *= 2;
  l.waves = small_waves(table_rows);
  const int64_t fit = std::max<int64_t>(1, std::min<int64_t>(16 / l.waves, 160 / (l.waves * table_rows)));
  const int64_t most = std::max<int64_t>(1, 256 * fit / l.chunks);
  const int64_t least = (int64_t)l.waves * 64 / l.lanes * 8;               // rows that a block has on their way
  l.range = std::max(least, (rows + most - 1) / most);
  l.blocks = (int)((rows + l.range - 1) / l.range);
  l.bytes = (int64_t)l.blocks * table_rows * width * 4;
  return l;
}

template <typename T, typename I>
void launch_lookup(const Args& a, hipStream_t st) {
  constexpr int64_t BLOCK = NT, MOST = BLOCK << 23;                      // fewer than 2^32 threads a launch
  const int64_t vectors = (a.width + Vec<T>::N - 1) / Vec<T>::N, total = a.rows * vectors;
  for (int64_t f = 0; f < total; f += MOST)
    FSC_EMBED_FULL(a.width >= Vec<T>::N, (lookup_kernel<T, I, FULL><<<(unsigned)((std::min(total - f, MOST) + BLOCK - 1) / BLOCK),
                                                                      NT, 0, st>>>(a, f, (uint32_t)vectors)));
}

template <typename T, typename I>
void launch_backward(const Args& a, char* ws, hipStream_t st) {
  constexpr int N = Vec<T>::N;
  if (few(a.rows, a.table_rows, a.width, sizeof(T))) {
    const dim3 grid((unsigned)std::min<int64_t>(a.table_rows, 1 << 16), (a.width + 64 * N - 1) / (64 * N));
    if ((int64_t)grid.x * grid.y <= 2048) FSC_EMBED_FULL(a.width >= N, (few_kernel<8, T, I, FULL><<<grid, 512, 0, st>>>(a)))
    else FSC_EMBED_FULL(a.width >= N, (few_kernel<4, T, I, FULL><<<grid, 256, 0, st>>>(a)))
    return;
  }
  if (a.table_rows <= SMALL) {
    const SmallLayout l = small_layout(a.rows, a.width, a.table_rows);
    const Stream s{l.lanes, l.range, (float*)ws};
    FSC_EMBED_FULL(a.width >= 4, (small_kernel<T, I, FULL><<<dim3(l.blocks, l.chunks), 64 * l.waves,
                                                             l.waves * a.table_rows * 1024, st>>>(a, s)));
    small_join_kernel<T><<<(unsigned)((a.table_rows * a.width + 63) / 64), 1024, 0, st>>>(a, s.part, l.blocks);
    return;
  }
  const Layout l = layout_of(a.rows, a.width, a.table_rows, sizeof(T));
  int32_t *key[2], *pos[2], *counts = (int32_t*)(ws + l.counts), *totals = (int32_t*)(ws + l.totals);
  for (int i = 0; i < 2; ++i) {
    key[i] = (int32_t*)(ws + l.key[i]);
    pos[i] = (int32_t*)(ws + l.pos[i]);
  }
  // few table rows: a block a row joins them, and writes the zeros; many: a block a share, zeros written first (65,536 x 331 in
  // bf16, 2,048 shares: 100 rows 36 and 37 us, 1,000 rows 54 and 51 us, 30,000 rows 188 and 65 us)
  const bool by_token = a.table_rows <= l.shares / 4;
  Source<I> src{(const I*)a.index, nullptr, nullptr, a.rows, a.table_rows};
  for (int p = 0; p < l.passes; ++p) {
    const int64_t values = p == 0 && !by_token ? a.table_rows * a.width : 0;
    const unsigned fill = (unsigned)std::min<int64_t>((values + NT * N - 1) / (NT * N), 2048);
    auto sort = [&](auto per, auto by_digit) {
      constexpr int PER = decltype(per)::value;
      constexpr bool BY_DIGIT = decltype(by_digit)::value;
      count_kernel<PER, BY_DIGIT, I, T><<<(unsigned)l.blocks + fill, NT, 0, st>>>(src, 8 * p, (int)l.blocks, counts, (T*)a.out,
                                                                                  values);
      if (BY_DIGIT) scan_kernel<<<DIGITS, 64, 0, st>>>((int)l.blocks, counts, totals);
      place_kernel<PER, BY_DIGIT, I><<<(unsigned)l.blocks, NT, 0, st>>>(src, 8 * p, (int)l.blocks, counts, totals, key[p & 1],
                                                                        pos[p & 1]);
    };
    if (l.blocks <= FEW_BLOCKS) sort(std::integral_constant<int, 4>{}, std::false_type{});
    else if (per_thread(a.rows) == 4) sort(std::integral_constant<int, 4>{}, std::true_type{});
    else sort(std::integral_constant<int, 16>{}, std::true_type{});
    src.key = key[p & 1];
    src.pos = pos[p & 1];
  }
  const Sums s{src.key, src.pos, a.rows, l.shares, l.share, l.lanes, l.columns, (float*)(ws + l.part)};
  const int64_t threads = l.shares * l.columns * l.lanes;
  FSC_EMBED_FULL(a.width >= N, (sum_kernel<T, FULL><<<(unsigned)((threads + NT - 1) / NT), NT, 0, st>>>(a, s)));
  const dim3 grid((unsigned)(by_token ? a.table_rows : l.shares), (a.width + 255) / 256);
  if (by_token) FSC_EMBED_FULL(a.width >= 4, (join_kernel<T, true, FULL><<<grid, JT, 0, st>>>(a, s)))
  else FSC_EMBED_FULL(a.width >= 4, (join_kernel<T, false, FULL><<<grid, JT, 0, st>>>(a, s)))
}

int check_sizes(int64_t rows, int32_t width, int64_t table_rows, int32_t dtype, int32_t index_bits) {
  FSC_CHECK_ARG(rows >= 0 && rows < (1ll << 31), "embedding: rows must be below 2^31");
  FSC_CHECK_ARG(width >= 1 && width <= (1 << 20), "embedding: width must be 1 to 2^20");
  FSC_CHECK_ARG(table_rows >= 0 && table_rows < (1ll << 31), "embedding: the table's rows must be below 2^31");
  FSC_CHECK_ARG(dtype == FSC_F32 || dtype == FSC_BF16, "embedding: the table is float32 or bfloat16");
  FSC_CHECK_ARG(index_bits == 32 || index_bits == 64, "embedding: the index is int32 or int64");
  return 0;
}

// runs the statement with (T, I)
#define FSC_EMBED_INDEX(...)                                     \
  if (index_bits == 32) { using I = int32_t; __VA_ARGS__; }      \
  else { using I = int64_t; __VA_ARGS__; }
#define FSC_EMBED_TYPES(...)                                     \
  if (dtype == FSC_F32) { using T = float; FSC_EMBED_INDEX(__VA_ARGS__) } \
  else { using T = __bf16; FSC_EMBED_INDEX(__VA_ARGS__) }

}  // namespace embed
}  // namespace fsc

extern "C" {

int fsc_embedding_forward_or(int64_t rows, int32_t width, int64_t table_rows, int32_t dtype, int32_t index_bits,
                             int64_t table_stride, const void* table, const void* index, float scale, float outside, void* out,
                             hipStream_t stream) {
  using namespace fsc;
  using namespace fsc::embed;
  if (int rc = check_sizes(rows, width, table_rows, dtype, index_bits)) return rc;
  if (rows == 0) return 0;
  FSC_CHECK_ARG(index && out && (table || table_rows == 0), "embedding: null array");
  FSC_CHECK_ARG(table_stride >= 0, "embedding: negative row stride");
  // without a table no row is read for its values: any array does
  const Args a{rows, table_rows ? table_stride : 0, table_rows, width, scale, table_rows ? table : out, index, out, outside};
  FSC_EMBED_TYPES((launch_lookup<T, I>(a, stream)));
  return check_launch("embedding") ? 2 : 0;
}

int fsc_embedding_forward(int64_t rows, int32_t width, int64_t table_rows, int32_t dtype, int32_t index_bits,
                          int64_t table_stride, const void* table, const void* index, float scale, void* out,
                          hipStream_t stream) {
  return fsc_embedding_forward_or(rows, width, table_rows, dtype, index_bits, table_stride, table, index, scale, 0.f, out, stream);
}

int fsc_embedding_workspace(int64_t rows, int32_t width, int64_t table_rows, int64_t* bytes) {
  FSC_CHECK_ARG(bytes != nullptr, "embedding: null output");
  if (int rc = fsc::embed::check_sizes(rows, width, table_rows, FSC_F32, 32)) return rc;
  *bytes = 0;
  if (table_rows == 0) return 0;
  for (int size : {2, 4}) {              // path and layout depend on the type: room for either
    if (fsc::embed::few(rows, table_rows, width, size)) continue;
    if (table_rows <= fsc::embed::SMALL) *bytes = std::max(*bytes, fsc::embed::small_layout(rows, width, table_rows).bytes);
    else *bytes = std::max(*bytes, fsc::embed::layout_of(rows, width, table_rows, size).bytes);
  }
  return 0;
}

int fsc_embedding_backward(int64_t rows, int32_t width, int64_t table_rows, int32_t dtype, int32_t index_bits,
                           int64_t dy_stride, const void* dy, const void* index, float scale, void* dtable,
                           void* workspace, hipStream_t stream) {
  using namespace fsc;
  using namespace fsc::embed;
  if (int rc = check_sizes(rows, width, table_rows, dtype, index_bits)) return rc;
  if (table_rows == 0) return 0;
  FSC_CHECK_ARG(dtable && (rows == 0 || (dy && index)), "embedding_backward: null array");
  FSC_CHECK_ARG(dy_stride >= 0, "embedding_backward: negative row stride");
  FSC_CHECK_ARG(rows * (int64_t)width <= 1ll << 41, "embedding_backward: dy has more than 2^41 values");   // grids of 32 bits
  const Args a{rows, dy_stride, table_rows, width, scale, dy, index, dtable, 0.f};
  FSC_CHECK_ARG(few(rows, table_rows, width, dtype == FSC_F32 ? 4 : 2) || workspace, "embedding_backward: null workspace");
  FSC_EMBED_TYPES((launch_backward<T, I>(a, (char*)workspace, stream)));
  return check_launch("embedding_backward") ? 2 : 0;
}

}  // extern "C"
