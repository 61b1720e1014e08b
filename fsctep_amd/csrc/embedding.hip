// Lookup of table rows by token (atomic number, species pair, ..) with a scale, and its gradient: the sum of the rows'
// gradients by token.  Replaces the indexing of the training step's first convolution and of the expert readout's
// table of scores, whose gradient was an atomic addition into a handful of rows
// (models/pure_cartesian_sparse_layers.py:258-259 embeds the species of every atom).
//   out_i = scale table[index_i], zeros where index_i lies outside the table
//   dtable_v = scale sum over i with index_i = v, in ascending order of i in 32 bits
#include <algorithm>

#include "common.h"
#include "expert_types.h"
#include "fsctep.h"

namespace fsc {
namespace embed {

constexpr int NT = 256;

struct Args {
  int64_t rows, stride;        // row stride of the table (forward) or of dy (backward), in elements
  int64_t table_rows;
  int width;
  float scale;
  const void *in, *index;
  void* out;
};

// A vector of 16 bytes at any address a value may lie at.
template <typename T>
struct alignas(sizeof(T)) Vec {
  static constexpr int N = 16 / sizeof(T);
  T t[N];
};
// n values from p on (all of them by one load where n is a vector's), zeros behind them
template <typename T>
__device__ __forceinline__ void load_some(const T* p, int n, float (&v)[Vec<T>::N]) {
  constexpr int N = Vec<T>::N;
  if (n >= N) {
    const Vec<T> k = *reinterpret_cast<const Vec<T>*>(p);
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = to_f(k.t[j]);
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = j < n ? to_f(p[j]) : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void store_some(T* p, int n, const float (&v)[Vec<T>::N]) {
  constexpr int N = Vec<T>::N;
  if (n >= N) {
    Vec<T> k;
#pragma unroll
    for (int j = 0; j < N; ++j) k.t[j] = from_f<T>(v[j]);
    *reinterpret_cast<Vec<T>*>(p) = k;
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (j < n) p[j] = from_f<T>(v[j]);
  }
}

// ---------------------------------------------------------------- lookup
// The output is written as one array, 16 bytes a thread and store whatever the width: a thread's values lie in one row
// and come by one load, but for those that a row's end parts.  STEPS stores a thread, a block's width apart.
constexpr int STEPS = 4;
template <typename T, typename I>
__global__ __launch_bounds__(NT) void lookup_kernel(Args a, int64_t first) {
  constexpr int N = Vec<T>::N;
  const int64_t total = a.rows * a.width;
  const int64_t f0 = first + (int64_t)blockIdx.x * (NT * N * STEPS);      // the block's first value, in row r0
  const int64_t r0 = f0 / a.width;
  const uint32_t c0 = (uint32_t)(f0 - r0 * a.width), width = a.width;
#pragma unroll
  for (int s = 0; s < STEPS; ++s) {
    const uint32_t local = c0 + (s * NT + threadIdx.x) * N;
    const int64_t f = f0 + (s * NT + threadIdx.x) * N;
    if (f >= total) return;
    const uint32_t up = local / width;
    int64_t row = r0 + up;
    uint32_t col = local - up * width;
    const int n = (int)std::min<int64_t>(N, total - f);
    float v[N];
    if (col + n <= width) {
      const int64_t t = ((const I*)a.index)[row];
      if (t >= 0 && t < a.table_rows) {
        load_some((const T*)a.in + t * a.stride + col, n, v);
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] *= a.scale;
      } else {
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = 0.f;
      }
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        v[j] = 0.f;
        if (j >= n) continue;
        const int64_t t = ((const I*)a.index)[row];
        if (t >= 0 && t < a.table_rows) v[j] = a.scale * to_f(((const T*)a.in)[t * a.stride + col]);
        if (++col == width) {
          col = 0;
          ++row;
        }
      }
    }
    store_some((T*)a.out + f, n, v);
  }
}

// ---------------------------------------------------------------- gradient, few tokens
// Up to FEW tokens: a block owns a row of the table and a vector a lane of its columns, its four waves look through a
// quarter of the tokens each, 64 at a time, and add the rows they find; one launch, no sort.
constexpr int FEW = 1024;
template <typename T, typename I>
__global__ __launch_bounds__(NT) void few_kernel(Args a) {
  constexpr int N = Vec<T>::N, AHEAD = 4;
  __shared__ float red[NT / 64][64 * N];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int col = (blockIdx.y * 64 + lane) * N, n = std::max(0, std::min(N, a.width - col));
  const int per = (int)((a.rows + 255) / 256) * 64;
  const int i0 = std::min<int>(a.rows, wave * per), i1 = std::min<int>(a.rows, i0 + per);
  for (int64_t v = blockIdx.x; v < a.table_rows; v += gridDim.x) {
    float s[N];
#pragma unroll
    for (int j = 0; j < N; ++j) s[j] = 0.f;
    for (int b = i0; b < i1; b += 64) {
      const int i = b + lane;
      uint64_t hits = __ballot(i < i1 && (int64_t)((const I*)a.index)[std::min(i, i1 - 1)] == v);
      while (hits) {                     // AHEAD rows on their way together
        int at[AHEAD], m = 0;
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
          at[k] = hits ? b + __ffsll((unsigned long long)hits) - 1 : -1;
          m += hits != 0;
          hits &= hits - 1;
        }
        float u[AHEAD][N];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k)
          if (at[k] >= 0) load_some((const T*)a.in + at[k] * a.stride + col, n, u[k]);
#pragma unroll
        for (int k = 0; k < AHEAD; ++k)
          if (k < m)
#pragma unroll
            for (int j = 0; j < N; ++j) s[j] += u[k][j];
      }
    }
#pragma unroll
    for (int j = 0; j < N; ++j) red[wave][lane * N + j] = s[j];
    __syncthreads();
    if (wave == 0 && n > 0) {
#pragma unroll
      for (int j = 0; j < N; ++j)
        s[j] = a.scale * ((red[0][lane * N + j] + red[1][lane * N + j]) + (red[2][lane * N + j] + red[3][lane * N + j]));
      store_some((T*)a.out + v * a.width + col, n, s);
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------- gradient, many tokens: sort
// The tokens' numbers sorted by token (a stable radix sort, 8 bits a pass, tokens outside the table last), so that
// sums are over runs of the sorted list.  A pass: counts by digit and block, each digit's counts scanned over the blocks, and
// the places: a digit's first place (all smaller digits' totals), the blocks before, the waves before, the lanes before.
constexpr int TILE = 4096, PER = TILE / NT;       // tokens of a block, and of a thread
constexpr int DIGITS = 256;

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
template <typename I, typename T>
__global__ __launch_bounds__(NT) void count_kernel(Source<I> src, int shift, int blocks, int32_t* __restrict__ counts,
                                                   T* __restrict__ table, int64_t values) {
  if ((int)blockIdx.x >= blocks) {
    constexpr int N = Vec<T>::N;
    const float zero[N] = {};
    const int64_t step = (int64_t)(gridDim.x - blocks) * NT * N;
    for (int64_t f = ((int64_t)(blockIdx.x - blocks) * NT + threadIdx.x) * N; f < values; f += step)
      store_some(table + f, (int)std::min<int64_t>(N, values - f), zero);
    return;
  }
  __shared__ int cnt[DIGITS];
  cnt[threadIdx.x] = 0;
  __syncthreads();
  const int64_t b0 = (int64_t)blockIdx.x * TILE;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int64_t i = b0 + k * NT + threadIdx.x;
    if (i < src.rows) atomicAdd(&cnt[src.key_of(i) >> shift & (DIGITS - 1)], 1);   // counts: any order
  }
  __syncthreads();
  counts[(int64_t)threadIdx.x * blocks + blockIdx.x] = cnt[threadIdx.x];
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

template <typename I>
__global__ __launch_bounds__(NT) void place_kernel(Source<I> src, int shift, int blocks, const int32_t* __restrict__ counts,
                                                   const int32_t* __restrict__ totals, int32_t* __restrict__ key,
                                                   int32_t* __restrict__ pos) {
  __shared__ int cnt[NT / 64][DIGITS], sums[NT / 64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, d = threadIdx.x;
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) cnt[w][d] = 0;
  // the digit's first place
  const int total = totals[d];
  const int run = wave_scan(total, lane);
  if (lane == 63) sums[wave] = run;
  __syncthreads();
  int base = run - total + counts[(int64_t)d * blocks + blockIdx.x];
  for (int w = 0; w < wave; ++w) base += sums[w];
  const int64_t w0 = (int64_t)blockIdx.x * TILE + wave * (TILE / (NT / 64));
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
// before it or goes on behind it leaves a partial row (first or second of the share's two), which join_kernel adds.
struct Sums {
  const int32_t *key, *pos;
  int64_t rows, shares;
  int share, lanes, columns;             // columns: groups of lanes that a row's vectors take
  float* part;                           // [shares][2][width]
};

template <typename T>
__global__ __launch_bounds__(NT) void sum_kernel(Args a, Sums s) {
  constexpr int N = Vec<T>::N, AHEAD = 8;
  const int64_t g = ((int64_t)blockIdx.x * NT + threadIdx.x) / s.lanes;
  const int64_t share = g / s.columns;
  if (share >= s.shares) return;
  const int col = ((int)(g - share * s.columns) * s.lanes + (threadIdx.x & (s.lanes - 1))) * N;
  const int n = std::min(N, a.width - col);
  if (n <= 0) return;
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
      store_some(out, std::min(n, 4), *(float(*)[4])&acc[0]);
      if constexpr (N == 8) {
        if (n > 4) store_some(out + 4, n - 4, *(float(*)[4])&acc[4]);
      }
    } else {
      float o[N];
#pragma unroll
      for (int j = 0; j < N; ++j) o[j] = a.scale * acc[j];
      store_some((T*)a.out + now * (int64_t)a.width + col, n, o);
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
      load_some(in + s.pos[q] * a.stride, n, v[i]);
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

// Adds the partial rows of one token: 64 columns a block, 16 waves over the rows, narrow rows several to a wave.  BY_TOKEN: a
// block a token, which writes the zeros of one that is not there; otherwise a block a share, which does nothing unless a
// token's run begins in it and goes on.
constexpr int JT = 1024;
template <typename T, bool BY_TOKEN>
__global__ __launch_bounds__(JT) void join_kernel(Args a, Sums s) {
  __shared__ float red[JT / 64][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int c0 = blockIdx.y * 64, wide = std::min(64, a.width - c0);
  int32_t v;
  int64_t s0, s1;                        // the shares it lies in
  if (BY_TOKEN) {
    v = (int32_t)blockIdx.x;
    const int64_t b = count_below<false>(s.key, s.rows, v, lane);
    if (b >= s.rows || s.key[b] != v) {
      if ((int)threadIdx.x < wide) ((T*)a.out)[v * (int64_t)a.width + c0 + threadIdx.x] = from_f<T>(0.f);
      return;
    }
    const int64_t e = b + count_below<true>(s.key + b, s.rows - b, v, lane);
    s0 = b / s.share;
    s1 = (e - 1) / s.share;
    if (s0 == s1) return;
  } else {
    s0 = blockIdx.x;
    const int64_t p0 = s0 * s.share, p1 = p0 + s.share;
    if (p1 >= s.rows) return;
    v = s.key[p1 - 1];
    if (v >= a.table_rows || s.key[p1] != v || (p0 > 0 && s.key[p0 - 1] == v)) return;
    const int64_t e = p1 + count_below<true>(s.key + p1, s.rows - p1, v, lane);
    s1 = (e - 1) / s.share;
  }
  int cols = 1;                          // lanes of a row: a power of two
  while (cols < wide) cols <<= 1;
  const int per = 64 / cols, sub = lane / cols, c = lane & (cols - 1);
  const int64_t m = s1 - s0 + 1;         // partial rows: the second of s0, the first of the others
  float x = 0.f;
  if (c < wide) {
    const float* part = s.part + c0 + c;
    // a run that goes on from the share's first token on has its partial row in the first share's second place as well
#pragma unroll 8
    for (int64_t i = (int64_t)wave * per + sub; i < m; i += (JT / 64) * per)
      x += part[(2 * (s0 + i) + (i == 0 ? 1 : 0)) * a.width];
  }
  for (int off = cols; off < 64; off <<= 1) x += __shfl_xor(x, off, 64);
  red[wave][lane] = x;
  __syncthreads();
  if (wave == 0 && lane < wide) {
    x = 0.f;
    for (int w = 0; w < JT / 64; ++w) x += red[w][lane];
    ((T*)a.out)[v * (int64_t)a.width + c0 + lane] = from_f<T>(a.scale * x);
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
  l.lanes = 4;
  while (l.lanes < 64 && l.lanes < vectors) l.lanes *= 2;
  l.columns = (int)((vectors + l.lanes - 1) / l.lanes);
  l.passes = 1;
  while (l.passes < 4 && (table_rows >> (8 * l.passes))) ++l.passes;
  l.blocks = (rows + TILE - 1) / TILE;
  // enough shares to fill the chip with waves, not so many that a token's partial rows take long to join
  const int64_t waves = rows * l.columns * l.lanes / 64;
  l.share = (int)std::min<int64_t>(1024, std::max<int64_t>({16, waves / 8192, rows / 8192}));
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

template <typename T, typename I>
void launch_lookup(const Args& a, hipStream_t st) {
  constexpr int64_t BLOCK = (int64_t)NT * Vec<T>::N * STEPS, MOST = BLOCK << 23;    // fewer than 2^32 threads a launch
  const int64_t total = a.rows * a.width;
  for (int64_t f = 0; f < total; f += MOST)
    lookup_kernel<T, I><<<(unsigned)((std::min(total - f, MOST) + BLOCK - 1) / BLOCK), NT, 0, st>>>(a, f);
}

template <typename T, typename I>
void launch_backward(const Args& a, char* ws, hipStream_t st) {
  constexpr int N = Vec<T>::N;
  if (a.rows <= FEW) {
    const dim3 grid((unsigned)std::min<int64_t>(a.table_rows, 1 << 16), (a.width + 64 * N - 1) / (64 * N));
    few_kernel<T, I><<<grid, NT, 0, st>>>(a);
    return;
  }
  const Layout l = layout_of(a.rows, a.width, a.table_rows, sizeof(T));
  int32_t *key[2], *pos[2], *counts = (int32_t*)(ws + l.counts), *totals = (int32_t*)(ws + l.totals);
  for (int i = 0; i < 2; ++i) {
    key[i] = (int32_t*)(ws + l.key[i]);
    pos[i] = (int32_t*)(ws + l.pos[i]);
  }
  // few table rows: a block a row joins them, and writes the zeros; many: a block a share, zeros written first
  const bool by_token = a.table_rows <= l.shares;
  Source<I> src{(const I*)a.index, nullptr, nullptr, a.rows, a.table_rows};
  for (int p = 0; p < l.passes; ++p) {
    const int64_t values = p == 0 && !by_token ? a.table_rows * a.width : 0;
    const unsigned fill = (unsigned)std::min<int64_t>((values + NT * N - 1) / (NT * N), 2048);
    count_kernel<I, T><<<(unsigned)l.blocks + fill, NT, 0, st>>>(src, 8 * p, (int)l.blocks, counts, (T*)a.out, values);
    scan_kernel<<<DIGITS, 64, 0, st>>>((int)l.blocks, counts, totals);
    place_kernel<I><<<(unsigned)l.blocks, NT, 0, st>>>(src, 8 * p, (int)l.blocks, counts, totals, key[p & 1], pos[p & 1]);
    src.key = key[p & 1];
    src.pos = pos[p & 1];
  }
  const Sums s{src.key, src.pos, a.rows, l.shares, l.share, l.lanes, l.columns, (float*)(ws + l.part)};
  const int64_t threads = l.shares * l.columns * l.lanes;
  sum_kernel<T><<<(unsigned)((threads + NT - 1) / NT), NT, 0, st>>>(a, s);
  const dim3 grid((unsigned)(by_token ? a.table_rows : l.shares), (a.width + 63) / 64);
  if (by_token) join_kernel<T, true><<<grid, JT, 0, st>>>(a, s);
  else join_kernel<T, false><<<grid, JT, 0, st>>>(a, s);
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

int fsc_embedding_forward(int64_t rows, int32_t width, int64_t table_rows, int32_t dtype, int32_t index_bits,
                          int64_t table_stride, const void* table, const void* index, float scale, void* out,
                          hipStream_t stream) {
  using namespace fsc;
  using namespace fsc::embed;
  if (int rc = check_sizes(rows, width, table_rows, dtype, index_bits)) return rc;
  if (rows == 0) return 0;
  FSC_CHECK_ARG(index && out && (table || table_rows == 0), "embedding: null array");
  FSC_CHECK_ARG(table_stride >= 0, "embedding: negative row stride");
  const Args a{rows, table_stride, table_rows, width, scale, table, index, out};
  FSC_EMBED_TYPES((launch_lookup<T, I>(a, stream)));
  return check_launch("embedding") ? 2 : 0;
}

int fsc_embedding_workspace(int64_t rows, int32_t width, int64_t table_rows, int64_t* bytes) {
  FSC_CHECK_ARG(bytes != nullptr, "embedding: null output");
  if (int rc = fsc::embed::check_sizes(rows, width, table_rows, FSC_F32, 32)) return rc;
  // the layout depends on the type: room for either
  *bytes = rows <= fsc::embed::FEW || table_rows == 0
               ? 0
               : std::max(fsc::embed::layout_of(rows, width, table_rows, 4).bytes,
                          fsc::embed::layout_of(rows, width, table_rows, 2).bytes);
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
  const Args a{rows, dy_stride, table_rows, width, scale, dy, index, dtable};
  FSC_CHECK_ARG(rows <= FEW || workspace, "embedding_backward: null workspace");
  FSC_EMBED_TYPES((launch_backward<T, I>(a, (char*)workspace, stream)));
  return check_launch("embedding_backward") ? 2 : 0;
}

}  // extern "C"
