// Layer norm of per-atom rows with an optional SiLU, its backward pass and the backward of that (a force loss
// differentiates the energy twice).  Replaces LayerNorm and SiLU of the energy head in the training step
// (models/mlp.py:8-66).  With zh = (x - mean) r, r = 1 / sqrt(mean (x - mean)^2 + eps), u = zh w + b:
//   forward    y = act(u)
//   backward   du = dy act'(u), g = du w:  dx = r (g - mean g - zh mean(g zh)), dw = sum du zh, db = sum du
//   twice      for cotangents V, Vw, Vb of dx, dw, db, with q = r (V - mean V - zh mean(V zh)):
//              a = w q + Vw zh + Vb,  e = dy act''(u) a
//              d/d dy = act'(u) a,  d/d w = sum du q + e zh,  d/d b = sum e
//              k = e w + du Vw - r (g mean(V zh) + V mean(g zh))
//              d/d x = r (k - mean k - zh (mean(k zh) + r (mean(g V) - mean g mean V - mean(g zh) mean(V zh))))
// (the last term is r's own dependence on x, dr / dx_j = -r^2 zh_j / width).
//
// Bound by memory: forward 2 arrays of the rows' size, backward 3 (4 with plus), twice 5.  A row is read once and kept in registers
// between its passes; rows shorter than a vector and rows past the registers take a block that reads them again (wide_kernel).
//
// Measured alone, without an activation (large copies and fills on this card: 5.2 and 6.8 TB/s): 10,000 x 1,600 fp32 forward 20.7 us
// (128 MB, 6.2 TB/s), backward 38 us (192 MB, 5.0 TB/s) with 5 us for the sums, twice 59 us (320 MB, 5.5 TB/s); 100,000 x 640 bf16 50 us
// (256 MB, 5.1 TB/s), 76 us (384 MB, 5.1 TB/s) and 227 us; 10,000 x 3,200 fp32 46, 80 and 135 us; 4,000 x 8,192 fp32 49, 84 and 135 us (131
// MB an array).  With SiLU 29, 45 and 75 us; 70, 135 and 318 us; 54, 95 and 232 us; 54, 95 and 212 us: its second pass is bound by
// registers, 512 x 4 in fp32 keeps 188 bytes a lane in scratch there and 256 x 4 in bf16 128.
#include <algorithm>

#include "common.h"
#include "expert_types.h"
#include "fsctep.h"

namespace fsc {
namespace lnorm {

constexpr int NT = 256;        // threads of a block: four waves
constexpr int NW = NT / 64;

struct Args {
  int64_t rows, xs, ys, vs;    // row strides of x, dy and v, in elements
  int width;
  float eps;
  const void *x, *w, *b;       // w, b null: 1 and 0
  double* mean;
  float* rstd;
  // forward
  void* y;
  // backward: dx null: not wanted
  const void* dy;
  const void* plus;            // added to dx, or null
  int64_t ps;                  // its row stride
  void* dx;
  void *dw, *db;               // null: not wanted
  float* part;                 // [gridDim.x][2][width] partial sums of the two
  // twice: v, vw, vb null: 0; gx, gdy null: not wanted
  const void *v, *vw, *vb;
  void *gx, *gdy;
};

// act and its derivatives at u.  The sigmoid's argument never overflows to a NaN: exp(-u) is at most inf.
template <bool SILU, typename F>
__device__ __forceinline__ F act0(F u) {
  if constexpr (!SILU) return u;
  else return u / (F(1) + exp(-u));
}
template <bool SILU, typename F>
__device__ __forceinline__ void act12(F u, F& d1, F& d2) {
  if constexpr (!SILU) {
    d1 = F(1);
    d2 = F(0);
  } else {
    const F s = F(1) / (F(1) + exp(-u)), t = s * (F(1) - s);
    d1 = s + u * t;
    d2 = t * (F(2) + u * (F(1) - F(2) * s));
  }
}

template <typename F>
__device__ __forceinline__ F wave_add(F v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}
// Sums of N values over the block, the same in every thread.
template <int N, typename F>
__device__ __forceinline__ void block_add(F (&v)[N], F* red) {
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    v[i] = wave_add(v[i]);
    if ((threadIdx.x & 63) == 0) red[i * NW + (threadIdx.x >> 6)] = v[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = (red[i * NW] + red[i * NW + 1]) + (red[i * NW + 2] + red[i * NW + 3]);
}

template <typename W>
__device__ __forceinline__ float at_or(const W* p, int i, float other) { return p ? to_f(p[i]) : other; }

// ---------------------------------------------------------------- one block a row
// Any width and alignment; the row is read again from the caches for each pass over it (figures: top of the file).  Sums for the
// statistics run in 64 bits: a mean far from zero would lose the deviations otherwise.
template <typename T, typename W, bool SILU>
__global__ __launch_bounds__(NT) void wide_kernel(Args a) {
  __shared__ double red[NW];
  const int64_t row = blockIdx.x;
  const T* x = (const T*)a.x + row * a.xs;
  const W *w = (const W*)a.w, *b = (const W*)a.b;
  T* y = (T*)a.y + row * a.width;
  double s[1] = {0.0};
  for (int i = threadIdx.x; i < a.width; i += NT) s[0] += (double)to_f(x[i]);
  block_add(s, red);
  const double mean = s[0] / a.width;
  s[0] = 0.0;
  for (int i = threadIdx.x; i < a.width; i += NT) {
    const double c = (double)to_f(x[i]) - mean;
    s[0] += c * c;
  }
  block_add(s, red);
  const float rstd = (float)(1.0 / sqrt(s[0] / a.width + (double)a.eps));
  for (int i = threadIdx.x; i < a.width; i += NT) {
    const float zh = (float)((double)to_f(x[i]) - mean) * rstd;
    y[i] = from_f<T>(act0<SILU>(zh * at_or(w, i, 1.f) + at_or(b, i, 0.f)));
  }
  if (threadIdx.x == 0 && a.mean) {
    a.mean[row] = mean;
    a.rstd[row] = rstd;
  }
}

// F: the type that dx is formed in, 64 bits for rows of at most 64 values, where it is what is left of nearly equal
// numbers (nothing at all in a row of one); the mean and the root are taken again there.
template <typename T, typename F>
__device__ __forceinline__ void statistics(const Args& a, int64_t row, const T* x, double* red, double& mean, F& r) {
  mean = a.mean[row];
  if constexpr (sizeof(F) == 4) {
    r = a.rstd[row];
  } else {
    double s[1] = {0.0};
    for (int i = threadIdx.x; i < a.width; i += NT) {
      const double c = (double)to_f(x[i]) - mean;
      s[0] += c * c;
    }
    block_add(s, red);
    r = 1.0 / sqrt(s[0] / a.width + (double)a.eps);
  }
}

template <typename T, typename W, bool SILU, typename F>
__global__ __launch_bounds__(NT) void wide_back_kernel(Args a) {
  __shared__ double red[2 * NW];
  const W *w = (const W*)a.w, *b = (const W*)a.b;
  float* part = a.dw || a.db ? a.part + (int64_t)blockIdx.x * 2 * a.width : nullptr;
  if (part)                              // a thread's own columns from here on
    for (int i = threadIdx.x; i < a.width; i += NT) part[i] = part[a.width + i] = 0.f;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = (const T*)a.x + row * a.xs;
    const T* dy = (const T*)a.dy + row * a.ys;
    double mean;
    F r;
    statistics<T, F>(a, row, x, red, mean, r);
    auto terms = [&](int i, F& zh, F& du) {
      F d1, d2;
      zh = (F)((double)to_f(x[i]) - mean) * r;
      act12<SILU>(zh * (F)at_or(w, i, 1.f) + (F)at_or(b, i, 0.f), d1, d2);
      du = (F)to_f(dy[i]) * d1;
    };
    F s[2] = {F(0), F(0)};
    for (int i = threadIdx.x; i < a.width; i += NT) {
      F zh, du;
      terms(i, zh, du);
      const F g = du * (F)at_or(w, i, 1.f);
      s[0] += g;
      s[1] += g * zh;
      if (part) {
        part[i] += (float)(du * zh);
        part[a.width + i] += (float)du;
      }
    }
    if (!a.dx) continue;
    block_add(s, (F*)red);
    const F mg = s[0] / a.width, mgz = s[1] / a.width;
    T* dx = (T*)a.dx + row * a.width;
    const T* plus = a.plus ? (const T*)a.plus + row * a.ps : nullptr;
    for (int i = threadIdx.x; i < a.width; i += NT) {
      F zh, du;
      terms(i, zh, du);
      dx[i] = from_f<T>((float)((F)at_or(plus, i, 0.f) + r * (du * (F)at_or(w, i, 1.f) - mg - zh * mgz)));
    }
  }
}

template <typename T, typename W, bool SILU, typename F>
__global__ __launch_bounds__(NT) void wide_twice_kernel(Args a) {
  __shared__ double red[5 * NW];
  const W *w = (const W*)a.w, *b = (const W*)a.b, *vw = (const W*)a.vw, *vb = (const W*)a.vb;
  float* part = a.dw || a.db ? a.part + (int64_t)blockIdx.x * 2 * a.width : nullptr;
  if (part)
    for (int i = threadIdx.x; i < a.width; i += NT) part[i] = part[a.width + i] = 0.f;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = (const T*)a.x + row * a.xs;
    const T* dy = (const T*)a.dy + row * a.ys;
    const T* v = a.v ? (const T*)a.v + row * a.vs : nullptr;
    double mean;
    F r;
    statistics<T, F>(a, row, x, red, mean, r);
    auto terms = [&](int i, F& zh, F& d1, F& d2) {
      zh = (F)((double)to_f(x[i]) - mean) * r;
      act12<SILU>(zh * (F)at_or(w, i, 1.f) + (F)at_or(b, i, 0.f), d1, d2);
    };
    F s[5] = {F(0), F(0), F(0), F(0), F(0)};
    for (int i = threadIdx.x; i < a.width; i += NT) {
      F zh, d1, d2;
      terms(i, zh, d1, d2);
      const F g = (F)to_f(dy[i]) * d1 * (F)at_or(w, i, 1.f), c = v ? (F)to_f(v[i]) : F(0);
      s[0] += g;
      s[1] += g * zh;
      s[2] += c;
      s[3] += c * zh;
      s[4] += g * c;
    }
    block_add(s, (F*)red);
    const F n = (F)a.width, mg = s[0] / n, mgz = s[1] / n, mv = s[2] / n, mvz = s[3] / n;
    const F turn = r * (s[4] / n - mg * mv - mgz * mvz);
    // what the row's value i gives: its k, its du, and its share of the other gradients
    auto second = [&](int i, F& zh, F& k, F& gdy, F& gw, F& gb) {
      F d1, d2;
      terms(i, zh, d1, d2);
      const F wi = (F)at_or(w, i, 1.f), c = v ? (F)to_f(v[i]) : F(0), d = (F)to_f(dy[i]), du = d * d1;
      const F q = r * (c - mv - zh * mvz), vwi = (F)at_or(vw, i, 0.f);
      const F aa = wi * q + vwi * zh + (F)at_or(vb, i, 0.f), e = d * d2 * aa;
      gdy = d1 * aa;
      gw = du * q + e * zh;
      gb = e;
      k = e * wi + du * vwi - r * (du * wi * mvz + c * mgz);
    };
    F t[2] = {F(0), F(0)};
    for (int i = threadIdx.x; i < a.width; i += NT) {
      F zh, k, gdy, gw, gb;
      second(i, zh, k, gdy, gw, gb);
      t[0] += k;
      t[1] += k * zh;
      if (part) {
        part[i] += (float)gw;
        part[a.width + i] += (float)gb;
      }
      if (a.gdy) ((T*)a.gdy)[row * a.width + i] = from_f<T>((float)gdy);
    }
    if (!a.gx) continue;
    block_add(t, (F*)red);
    const F mk = t[0] / n, mkz = t[1] / n + turn;
    for (int i = threadIdx.x; i < a.width; i += NT) {
      F zh, k, gdy, gw, gb;
      second(i, zh, k, gdy, gw, gb);
      ((T*)a.gx)[row * a.width + i] = from_f<T>((float)(r * (k - mk - zh * mkz)));
    }
  }
}

// ---------------------------------------------------------------- a row in the registers of L lanes
// Lane l of a row's L holds the vectors of 16 bytes c L + l, c < CH; a row is read once.  The last vector of a row whose
// width no vector divides is read from the row's end back, and its lane takes the values from `skip` on as its own; lanes
// past the end own none.  Values that are not a lane's own are zeros in every sum.
//
// Bound by memory with the vector units behind it, which issue in 42 to 56 % of the cycles at the large cases (a wave's instruction
// takes four): shapes leave few lanes idle, sums within 16 lanes are DPP additions, and a value takes about a dozen instructions in
// each pass.
template <typename T>
struct alignas(sizeof(T)) Vec {          // at any address a value may lie at
  static constexpr int N = 16 / sizeof(T);
  T t[N];
};

// threads of a block whose rows take L lanes
constexpr int threads_of(int L) { return L > NT ? L : NT; }

template <typename T, int L, int CH>
struct Row {
  static constexpr int V = Vec<T>::N;
  int width, lane;
  bool ragged;                           // some lane owns less than CH vectors
  __device__ __forceinline__ Row(int w) : width(w), lane(threadIdx.x & (L - 1)), ragged(w != L * CH * V) {}
  __device__ __forceinline__ int base(int c) const { return std::min((c * L + lane) * V, width - V); }
  __device__ __forceinline__ int skip(int c) const { return (c * L + lane) * V - base(c); }

  template <typename S>
  __device__ __forceinline__ void load_one(const S* p, int c, float (&v)[V]) const {
    if constexpr (sizeof(S) == sizeof(T)) {
      const Vec<S> k = *reinterpret_cast<const Vec<S>*>(p + base(c));
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = to_f(k.t[j]);
    } else {                             // float32 weights of bfloat16 rows
#pragma unroll
      for (int h = 0; h < V; h += 4) {
        const Vec<float> k = *reinterpret_cast<const Vec<float>*>(p + base(c) + h);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[h + j] = k.t[j];
      }
    }
  }
  template <typename S>
  __device__ __forceinline__ void load(const S* p, float (&v)[CH][V]) const {
#pragma unroll
    for (int c = 0; c < CH; ++c) load_one(p, c, v[c]);
  }
  template <typename S>
  __device__ __forceinline__ void load_or(const S* p, float other, float (&v)[CH][V]) const {
    if (p) {
      load(p, v);
      return;
    }
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int j = 0; j < V; ++j) v[c][j] = other;
  }
  // zeros for what is not the lane's own
  template <typename F>
  __device__ __forceinline__ void own(F (&v)[CH][V]) const {
    if (!ragged) return;
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int j = 0; j < V; ++j) v[c][j] = j >= skip(c) ? v[c][j] : F(0);
  }
  // Past the caches' own keeping: what a pass writes is read by another kernel, on other XCDs (10,000 x 1,600: 34 -> 27 us
  // forward, 39 -> 37 us backward).
  template <typename F>
  __device__ __forceinline__ void store(T* p, int c, const F (&v)[V]) const {
    typedef unsigned u4s __attribute__((ext_vector_type(4), aligned(2)));
    const int s = skip(c);
    if (s == 0) {
      Vec<T> k;
#pragma unroll
      for (int j = 0; j < V; ++j) k.t[j] = from_f<T>((float)v[j]);
      __builtin_nontemporal_store(__builtin_bit_cast(u4s, k), reinterpret_cast<u4s*>(p + base(c)));
    } else if (s < V) {
#pragma unroll
      for (int j = 1; j < V; ++j)
        if (j >= s) p[base(c) + j] = from_f<T>((float)v[j]);
    }
  }
};

// v of the lane that DPP's CTRL names
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
template <int CTRL>
__device__ __forceinline__ double dpp(double v) {
  const int2 u = __builtin_bit_cast(int2, v);
  const int2 w = {__builtin_amdgcn_update_dpp(0, u.x, CTRL, 0xf, 0xf, true),
                  __builtin_amdgcn_update_dpp(0, u.y, CTRL, 0xf, 0xf, true)};
  return __builtin_bit_cast(double, w);
}

// Sums of N values over a row's lanes, the same in each.  A row of a whole block's lanes meets in LDS, in two places by
// turns: who still reads the one has not passed the barrier before the next but one sum.
template <int L, typename F>
struct RowAdd {
  static constexpr int WAVES = L / 64;
  F* red;                                // [2][5][WAVES] where a row takes the block
  int turn = 0;
  __device__ __forceinline__ explicit RowAdd(F* r) : red(r) {}
  template <int N>
  __device__ __forceinline__ void operator()(F (&v)[N]) {
    static_assert(L >= 16, "whole DPP rows");
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] += dpp<0xB1>(v[i]);           // neighbours, then pairs, then (both halves alike) mirrored in 8 and in 16
      v[i] += dpp<0x4E>(v[i]);
      v[i] += dpp<0x141>(v[i]);
      v[i] += dpp<0x140>(v[i]);
    }
#pragma unroll
    for (int off = 16; off < (L < 64 ? L : 64); off <<= 1)
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] += __shfl_xor(v[i], off, 64);
    if constexpr (L >= NT) {
      F* at = red + turn * 5 * WAVES;
      turn ^= 1;
      if ((threadIdx.x & 63) == 0)
#pragma unroll
        for (int i = 0; i < N; ++i) at[i * WAVES + (threadIdx.x >> 6)] = v[i];
      __syncthreads();
#pragma unroll
      for (int i = 0; i < N; ++i) {
        v[i] = F(0);
#pragma unroll
        for (int k = 0; k < WAVES; k += 4)
          v[i] += (at[i * WAVES + k] + at[i * WAVES + k + 1]) + (at[i * WAVES + k + 2] + at[i * WAVES + k + 3]);
      }
    }
  }
};

// A 64-bit mean in two 32-bit parts: deviations keep their own accuracy, far from zero and next to the mean.
__device__ __forceinline__ void parts_of(double mean, float& hi, float& lo) {
  hi = (float)mean;
  lo = (float)(mean - (double)hi);
}

template <typename T, typename W, bool SILU, int L, int CH>
__global__ __launch_bounds__(threads_of(L)) void row_kernel(Args a) {
  using R = Row<T, L, CH>;
  constexpr int V = R::V;
  __shared__ double red64[L >= NT ? 2 * 5 * L / 64 : 1];
  __shared__ float red32[L >= NT ? 2 * 5 * L / 64 : 1];
  RowAdd<L, double> add64(red64);
  RowAdd<L, float> add32(red32);
  const int64_t row = ((int64_t)blockIdx.x * threads_of(L) + threadIdx.x) / L;
  if (row >= a.rows) return;
  const R at(a.width);
  float x[CH][V], w[CH][V], b[CH][V];
  at.load((const T*)a.x + row * a.xs, x);
  at.load_or((const W*)a.w, 1.f, w);
  at.load_or((const W*)a.b, 0.f, b);
  double s[1] = {0.0};
  float t[1] = {0.f}, hi, lo;
  at.own(x);
#pragma unroll
  for (int c = 0; c < CH; ++c)
#pragma unroll
    for (int j = 0; j < V; ++j) s[0] += (double)x[c][j];
  add64(s);
  const double mean = s[0] / a.width;
  parts_of(mean, hi, lo);
#pragma unroll
  for (int c = 0; c < CH; ++c)
#pragma unroll
    for (int j = 0; j < V; ++j) x[c][j] = (x[c][j] - hi) - lo;
  at.own(x);
#pragma unroll
  for (int c = 0; c < CH; ++c)
#pragma unroll
    for (int j = 0; j < V; ++j) t[0] += x[c][j] * x[c][j];
  add32(t);
  const float var = t[0] / a.width + a.eps;
  float rstd = 1.f / sqrtf(var);
  if (!(var > 0x1p-110f && var < 0x1p126f)) {
    // squares past 32 bits' range (deviations from 2^63 on, or below 2^-55 with an eps as small): again in 64 bits.  The whole row
    // comes here: every lane of it has the same sum.
    s[0] = 0.0;
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int j = 0; j < V; ++j) s[0] += (double)x[c][j] * (double)x[c][j];
    add64(s);
    rstd = (float)(1.0 / sqrt(s[0] / a.width + (double)a.eps));
  }
  T* y = (T*)a.y + row * a.width;
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    float o[V];
#pragma unroll
    for (int j = 0; j < V; ++j) o[j] = act0<SILU>(x[c][j] * rstd * w[c][j] + b[c][j]);
    at.store(y, c, o);
  }
  if (at.lane == 0 && a.mean) {
    a.mean[row] = mean;
    a.rstd[row] = rstd;
  }
}

// zh of the row in x: zeros where a value is not the lane's own.  Returns the root's factor.
template <typename T, typename F, int L, int CH, int V>
__device__ __forceinline__ F normalised(const Args& a, const Row<T, L, CH>& at, RowAdd<L, F>& row_add, double mean, float rstd,
                                        const float (&x)[CH][V], F (&z)[CH][V]) {
  if constexpr (sizeof(F) == 4) {
    float hi, lo;
    parts_of(mean, hi, lo);
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int j = 0; j < V; ++j) z[c][j] = ((x[c][j] - hi) - lo) * rstd;
    at.own(z);
    return rstd;
  } else {
    double s[1] = {0.0};
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int j = 0; j < V; ++j) z[c][j] = (double)x[c][j] - mean;
    at.own(z);
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int j = 0; j < V; ++j) s[0] += z[c][j] * z[c][j];
    row_add(s);
    const F r = 1.0 / sqrt(s[0] / a.width + (double)a.eps);
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int j = 0; j < V; ++j) z[c][j] *= r;
    return r;
  }
}

// Adds a lane's sums of the weight's and the bias' gradients over the wave's rows and the block's waves: a partial row
// for the block, or the gradients themselves where there is one block.  buf: [2][width] unless a row takes the block's lanes, where
// every column is one thread's own.
template <typename T, typename W, int L, int CH, int V>
__device__ __forceinline__ void put_part(const Args& a, const Row<T, L, CH>& at, float (&gw)[CH][V], float (&gb)[CH][V],
                                         float* buf) {
  float* part = a.part + (int64_t)blockIdx.x * 2 * a.width;
  auto put = [&](int i, float w, float b) {
    if (gridDim.x > 1) {
      part[i] = w;
      part[a.width + i] = b;
    } else {
      if (a.dw) ((W*)a.dw)[i] = from_f<W>(w);
      if (a.db) ((W*)a.db)[i] = from_f<W>(b);
    }
  };
  if constexpr (L >= NT) {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int i = at.base(c), skip = at.skip(c);
      if (skip == 0 && gridDim.x > 1) {
#pragma unroll
        for (int h = 0; h < V; h += 4) {
          *reinterpret_cast<Vec<float>*>(part + i + h) = Vec<float>{gw[c][h], gw[c][h + 1], gw[c][h + 2], gw[c][h + 3]};
          *reinterpret_cast<Vec<float>*>(part + a.width + i + h) = Vec<float>{gb[c][h], gb[c][h + 1], gb[c][h + 2], gb[c][h + 3]};
        }
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (j >= skip) put(i + j, gw[c][j], gb[c][j]);
      }
    }
  } else {
    const int wave = threadIdx.x >> 6;
#pragma unroll
    for (int off = L; off < 64; off <<= 1)
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          gw[c][j] += __shfl_xor(gw[c][j], off, 64);
          gb[c][j] += __shfl_xor(gb[c][j], off, 64);
        }
#pragma unroll 1
    for (int k = 0; k < NW; ++k) {
      if (wave == k && (threadIdx.x & 63) < L) {
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
          for (int j = 0; j < V; ++j)
            if (j >= at.skip(c)) {
              const int i = at.base(c) + j;
              buf[i] = k ? buf[i] + gw[c][j] : gw[c][j];
              buf[a.width + i] = k ? buf[a.width + i] + gb[c][j] : gb[c][j];
            }
      }
      __syncthreads();
    }
    for (int i = threadIdx.x; i < a.width; i += NT) put(i, buf[i], buf[a.width + i]);
  }
}

template <typename T, typename W, bool SILU, typename F, int L, int CH>
__global__ __launch_bounds__(threads_of(L)) void row_back_kernel(Args a) {
  using R = Row<T, L, CH>;
  constexpr int V = R::V, ROWS = threads_of(L) / L;
  __shared__ float buf[L >= NT ? 1 : 2 * L * CH * V];
  __shared__ F red[L >= NT ? 2 * 5 * L / 64 : 1];
  RowAdd<L, F> row_add(red);
  const R at(a.width);
  float w[CH][V], b[CH][V], gw[CH][V] = {}, gb[CH][V] = {};
  at.load_or((const W*)a.w, 1.f, w);
  if (SILU) at.load_or((const W*)a.b, 0.f, b);
  const F n = (F)a.width;
  // every lane goes round as often: rows past the last one are the last one again, with zeros for what is added and stored nowhere
  for (int64_t r0 = (int64_t)blockIdx.x * ROWS; r0 < a.rows; r0 += (int64_t)gridDim.x * ROWS) {
    const int64_t mine = r0 + threadIdx.x / L, row = std::min<int64_t>(mine, a.rows - 1);
    const bool there = mine < a.rows;
    float x[CH][V], d[CH][V];
    at.load((const T*)a.x + row * a.xs, x);
    at.load((const T*)a.dy + row * a.ys, d);
    F z[CH][V], g[CH][V];
    const F r = normalised<T, F, L, CH, V>(a, at, row_add, a.mean[row], a.rstd[row], x, z);
    at.own(d);
    if (r0 + ROWS > a.rows && !there)
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int j = 0; j < V; ++j) z[c][j] = F(0), d[c][j] = 0.f;
    F s[2] = {F(0), F(0)};
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        F d1, d2, du = (F)d[c][j];
        if (SILU) {
          act12<SILU>(z[c][j] * (F)w[c][j] + (F)b[c][j], d1, d2);
          du *= d1;
        }
        gw[c][j] += (float)(du * z[c][j]);
        gb[c][j] += (float)du;
        g[c][j] = du * (F)w[c][j];
        s[0] += g[c][j];
        s[1] += g[c][j] * z[c][j];
      }
    if (!a.dx) continue;
    at.load_or(a.plus ? (const T*)a.plus + row * a.ps : nullptr, 0.f, d);
    row_add(s);
    const F mg = s[0] / n, mgz = s[1] / n;
    if (there)
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        F o[V];
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] = (F)d[c][j] + r * ((g[c][j] - mg) - z[c][j] * mgz);
        at.store((T*)a.dx + row * a.width, c, o);
      }
  }
  if (a.dw || a.db) put_part<T, W, L, CH, V>(a, at, gw, gb, buf);
}

template <typename T, typename W, bool SILU, typename F, int L, int CH>
__global__ __launch_bounds__(threads_of(L)) void row_twice_kernel(Args a) {
  using R = Row<T, L, CH>;
  constexpr int V = R::V, ROWS = threads_of(L) / L;
  __shared__ float buf[L >= NT ? 1 : 2 * L * CH * V];
  __shared__ F red[L >= NT ? 2 * 5 * L / 64 : 1];
  RowAdd<L, F> row_add(red);
  const R at(a.width);
  float w[CH][V], b[CH][V], gw[CH][V] = {}, gb[CH][V] = {};
  at.load_or((const W*)a.w, 1.f, w);
  if (SILU) at.load_or((const W*)a.b, 0.f, b);
  const F n = (F)a.width;
  for (int64_t r0 = (int64_t)blockIdx.x * ROWS; r0 < a.rows; r0 += (int64_t)gridDim.x * ROWS) {
    const int64_t mine = r0 + threadIdx.x / L, row = std::min<int64_t>(mine, a.rows - 1);
    const bool there = mine < a.rows;
    float x[CH][V], d[CH][V], v[CH][V];
    at.load((const T*)a.x + row * a.xs, x);
    at.load((const T*)a.dy + row * a.ys, d);
    at.load_or(a.v ? (const T*)a.v + row * a.vs : nullptr, 0.f, v);
    F z[CH][V];
    const F r = normalised<T, F, L, CH, V>(a, at, row_add, a.mean[row], a.rstd[row], x, z);
    at.own(d);
    at.own(v);
    if (r0 + ROWS > a.rows && !there)
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int j = 0; j < V; ++j) z[c][j] = F(0), d[c][j] = v[c][j] = 0.f;
    F s[5] = {F(0), F(0), F(0), F(0), F(0)};
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        F d1, d2, g = (F)d[c][j] * (F)w[c][j];
        if (SILU) {
          act12<SILU>(z[c][j] * (F)w[c][j] + (F)b[c][j], d1, d2);
          g *= d1;
        }
        const F q = (F)v[c][j];
        s[0] += g;
        s[1] += g * z[c][j];
        s[2] += q;
        s[3] += q * z[c][j];
        s[4] += g * q;
      }
    row_add(s);
    const F mg = s[0] / n, mgz = s[1] / n, mv = s[2] / n, mvz = s[3] / n;
    const F turn = r * (s[4] / n - mg * mv - mgz * mvz);
    F k[CH][V], t[2] = {F(0), F(0)};
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      F gdy[V];
      float vw[V] = {}, vb[V] = {};
      if (a.vw) at.load_one((const W*)a.vw, c, vw);
      if (a.vb) at.load_one((const W*)a.vb, c, vb);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        F d1 = F(1), d2 = F(0);
        const F wi = (F)w[c][j], dj = (F)d[c][j], zj = z[c][j];
        if (SILU) act12<SILU>(zj * wi + (F)b[c][j], d1, d2);
        // a value that is not the lane's own has d 0: nothing of it reaches a sum
        const F du = dj * d1, q = r * (((F)v[c][j] - mv) - zj * mvz);
        const F aa = wi * q + (F)vw[j] * zj + (F)vb[j], e = dj * d2 * aa;
        gdy[j] = d1 * aa;
        gw[c][j] += (float)(du * q + e * zj);
        gb[c][j] += (float)e;
        k[c][j] = e * wi + du * (F)vw[j] - r * (du * wi * mvz + (F)v[c][j] * mgz);
        t[0] += k[c][j];
        t[1] += k[c][j] * zj;
      }
      if (a.gdy && there) at.store((T*)a.gdy + row * a.width, c, gdy);
    }
    if (!a.gx) continue;
    row_add(t);
    const F mk = t[0] / n, mkz = t[1] / n + turn;
    if (there)
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        F o[V];
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] = r * ((k[c][j] - mk) - z[c][j] * mkz);
        at.store((T*)a.gx + row * a.width, c, o);
      }
  }
  if (a.dw || a.db) put_part<T, W, L, CH, V>(a, at, gw, gb, buf);
}

// Column sums of the blocks' partial rows, the weight's gradient and the bias': 32 columns a block, 32 threads a column,
// then a fixed tree (the same sum every time).  blockIdx.y: which of the two.  1,024 x 1,600 partial sums: 5 us, in part the
// launch.
template <typename W>
__global__ __launch_bounds__(1024) void sum_kernel(const float* __restrict__ part, int n, int width, W* __restrict__ dw,
                                                   W* __restrict__ db) {
  __shared__ float red[32][33];
  W* out = blockIdx.y ? db : dw;
  if (!out) return;
  const int c = threadIdx.x & 31, k = threadIdx.x >> 5, col = blockIdx.x * 32 + c;
  float s = 0.f;
  if (col < width)
#pragma unroll 8
    for (int i = k; i < n; i += 32) s += part[((int64_t)i * 2 + blockIdx.y) * width + col];
  red[k][c] = s;
  __syncthreads();
  s = group_sum(red[c][k], 32);          // column k of the block in lanes c = 0..31
  if (c == 0 && blockIdx.x * 32 + k < width) out[blockIdx.x * 32 + k] = from_f<W>(s);
}

// Calls f(L, CH) for the fewest vectors of L lanes that hold a row; false where none do (a row shorter than a vector, or too
// wide).  FORWARD shapes may have the registers of five vectors of 16 bits a lane, the backward passes three (100,000 x 640 in
// bf16 backward, five vectors of 16 lanes: 130 us, three of 32: 88 us), the second one three of either type.  Rows of 4,097 to 8,192
// float32 values take 512 lanes (4,000 x 8,192 without an activation by 512 lanes, 1,024 lanes of two vectors and wide_kernel: forward
// 49, 50 and 105 us, backward 84, 86 and 344 us, twice 136, 269 and 439 us; the same vectors of bfloat16 have no room for the second
// pass).
enum Pass { FORWARD, BACK, TWICE };
template <typename T, Pass P, typename F>
bool by_shape(int width, F&& f) {
  constexpr int V = Vec<T>::N;
  constexpr bool FIVE = P == FORWARD || (P == BACK && V == 4);
#define FSC_LN_SHAPE(L_, CH_)                                                               \
  if (width <= L_ * CH_ * V) {                                                              \
    f(std::integral_constant<int, L_>{}, std::integral_constant<int, CH_>{});               \
    return true;                                                                            \
  }
  if (width < V) return false;
  FSC_LN_SHAPE(16, 1)
  FSC_LN_SHAPE(16, 2)
  FSC_LN_SHAPE(16, 3)
  if constexpr (FIVE) {
    FSC_LN_SHAPE(16, 5)
  }
  FSC_LN_SHAPE(32, 3)
  FSC_LN_SHAPE(64, 2)
  if constexpr (FIVE) {
    FSC_LN_SHAPE(32, 5)
  }
  FSC_LN_SHAPE(64, 3)
  FSC_LN_SHAPE(256, 1)
  FSC_LN_SHAPE(256, 2)
  FSC_LN_SHAPE(256, 4)
  if constexpr (V == 4) {
    FSC_LN_SHAPE(512, 4)
  }
#undef FSC_LN_SHAPE
  return false;
}

// Blocks of the two backward passes on rows of L lanes.  Two rounds of rows are left to one block, which needs no partial rows
// (32 x 128: 7.5 us, by two blocks 8.9 us; 64 x 128: 9.6 us by one, 9.0 us by four).  At most 512, 1,024 where a row takes a
// block's four waves (100,000 x 640 in bf16 by 512 and 1,024: 80 and 90 us; 10,000 x 1,600: 47 and 44 us).
inline int back_blocks(int64_t rows, int L) {
  const int64_t at_once = threads_of(L) / L;
  if (rows <= 2 * at_once) return 1;
  return (int)std::min<int64_t>((rows + at_once - 1) / at_once, L == NT ? 1024 : 512);
}

template <typename T, typename W, bool SILU>
void launch_forward(const Args& all, hipStream_t st) {
  constexpr int64_t MOST = 1ll << 22;    // rows of a launch: a grid has fewer than 2^32 threads
  for (int64_t r0 = 0; r0 < all.rows; r0 += MOST) {
    Args a = all;
    a.rows = std::min(all.rows - r0, MOST);
    a.x = (const T*)all.x + r0 * all.xs;
    a.y = (T*)all.y + r0 * all.width;
    if (all.mean) {
      a.mean = all.mean + r0;
      a.rstd = all.rstd + r0;
    }
    if (!by_shape<T, FORWARD>(a.width, [&](auto L, auto CH) {
          constexpr int l = decltype(L)::value, ch = decltype(CH)::value;
          row_kernel<T, W, SILU, l, ch><<<(unsigned)((a.rows * l + threads_of(l) - 1) / threads_of(l)), threads_of(l), 0, st>>>(a);
        }))
      wide_kernel<T, W, SILU><<<(unsigned)a.rows, NT, 0, st>>>(a);
  }
}

template <typename T, typename W, bool SILU, Pass P>
void launch_backward(const Args& a, hipStream_t st) {
  int blocks = 0;
  const bool done = by_shape<T, P>(a.width, [&](auto L, auto CH) {
    constexpr int l = decltype(L)::value, ch = decltype(CH)::value;
    blocks = back_blocks(a.rows, l);
    if constexpr (l * ch <= 16) {
      if (a.width <= 64) {
        if constexpr (P == TWICE) row_twice_kernel<T, W, SILU, double, l, ch><<<blocks, NT, 0, st>>>(a);
        else row_back_kernel<T, W, SILU, double, l, ch><<<blocks, NT, 0, st>>>(a);
        return;
      }
    }
    if constexpr (l * ch > 16 || sizeof(T) == 2) {
      if constexpr (P == TWICE) row_twice_kernel<T, W, SILU, float, l, ch><<<blocks, threads_of(l), 0, st>>>(a);
      else row_back_kernel<T, W, SILU, float, l, ch><<<blocks, threads_of(l), 0, st>>>(a);
    }
  });
  if (!done) {
    blocks = back_blocks(a.rows, NT);
    if (a.width <= 64) {
      if constexpr (P == TWICE) wide_twice_kernel<T, W, SILU, double><<<blocks, NT, 0, st>>>(a);
      else wide_back_kernel<T, W, SILU, double><<<blocks, NT, 0, st>>>(a);
    } else {
      if constexpr (P == TWICE) wide_twice_kernel<T, W, SILU, float><<<blocks, NT, 0, st>>>(a);
      else wide_back_kernel<T, W, SILU, float><<<blocks, NT, 0, st>>>(a);
    }
  }
  if ((a.dw || a.db) && (blocks > 1 || !done))
    sum_kernel<W><<<dim3((a.width + 31) / 32, 2), 1024, 0, st>>>(a.part, blocks, a.width, (W*)a.dw, (W*)a.db);
}

// runs the statement with (T, W, SILU)
#define FSC_LN_ACT(...)                                        \
  if (act) { constexpr bool SILU = true; __VA_ARGS__; }        \
  else { constexpr bool SILU = false; __VA_ARGS__; }
#define FSC_LN_TYPES(...)                                                                    \
  if (dtype == FSC_F32) { using T = float; using W = float; FSC_LN_ACT(__VA_ARGS__) }        \
  else if (wtype == FSC_F32) { using T = __bf16; using W = float; FSC_LN_ACT(__VA_ARGS__) }  \
  else { using T = __bf16; using W = __bf16; FSC_LN_ACT(__VA_ARGS__) }

int check_types(int64_t rows, int32_t width, int32_t dtype, int32_t wtype, int32_t act) {
  FSC_CHECK_ARG(rows >= 0 && rows < (1ll << 31), "layer_norm: rows must be below 2^31");
  FSC_CHECK_ARG(width >= 1 && width <= (1 << 20), "layer_norm: width must be 1 to 2^20");
  FSC_CHECK_ARG(dtype == FSC_F32 || dtype == FSC_BF16, "layer_norm: rows are float32 or bfloat16");
  FSC_CHECK_ARG(wtype == FSC_F32 || wtype == dtype, "layer_norm: weight and bias are float32 or of the rows' type");
  FSC_CHECK_ARG(act == FSC_ACT_NONE || act == FSC_ACT_SILU, "layer_norm: unknown activation");
  return 0;
}

int backward(const Args& a, int32_t dtype, int32_t wtype, int32_t act, bool twice, hipStream_t st) {
  if (int rc = check_types(a.rows, a.width, dtype, wtype, act)) return rc;
  FSC_CHECK_ARG(a.rows == 0 || (a.x && a.mean && a.rstd && a.dy), "layer_norm_backward: null array");
  FSC_CHECK_ARG(a.xs >= 0 && a.ys >= 0 && a.vs >= 0 && a.ps >= 0, "layer_norm_backward: negative row stride");
  FSC_CHECK_ARG(!(a.dw || a.db) || a.part, "layer_norm_backward: the weight's and the bias' gradients need a workspace");
  if (!a.dw && !a.db && (a.rows == 0 || !(a.dx || a.gx || a.gdy))) return 0;
  if (twice) {
    FSC_LN_TYPES((launch_backward<T, W, SILU, TWICE>(a, st)));
  } else {
    FSC_LN_TYPES((launch_backward<T, W, SILU, BACK>(a, st)));
  }
  return check_launch("layer_norm_backward") ? 2 : 0;
}

}  // namespace lnorm
}  // namespace fsc

extern "C" {

int fsc_layer_norm_forward(int64_t rows, int32_t width, int32_t dtype, int32_t weight_dtype, int32_t activation,
                           int64_t x_stride, const void* x, const void* weight, const void* bias, float eps, void* y,
                           double* mean, float* rstd, hipStream_t stream) {
  using namespace fsc;
  using namespace fsc::lnorm;
  const int32_t wtype = weight_dtype, act = activation;
  if (int rc = check_types(rows, width, dtype, wtype, act)) return rc;
  if (rows == 0) return 0;
  FSC_CHECK_ARG(x && y && !mean == !rstd, "layer_norm: null array");
  FSC_CHECK_ARG(x_stride >= 0, "layer_norm: negative row stride");
  Args a{};
  a.rows = rows; a.xs = x_stride; a.width = width; a.eps = eps;
  a.x = x; a.w = weight; a.b = bias; a.y = y; a.mean = mean; a.rstd = rstd;
  FSC_LN_TYPES(launch_forward<T, W, SILU>(a, stream));
  return check_launch("layer_norm") ? 2 : 0;
}

int fsc_layer_norm_workspace(int64_t rows, int32_t width, int64_t* floats) {
  FSC_CHECK_ARG(floats != nullptr, "layer_norm: null output");
  FSC_CHECK_ARG(rows >= 0 && width >= 1, "layer_norm: negative size");
  *floats = (int64_t)fsc::lnorm::back_blocks(rows, fsc::lnorm::NT) * 2 * width;   // no shape takes more blocks
  return 0;
}

int fsc_layer_norm_backward(int64_t rows, int32_t width, int32_t dtype, int32_t weight_dtype, int32_t activation,
                            int64_t x_stride, int64_t dy_stride, int64_t plus_stride, const void* x, const void* weight,
                            const void* bias, float eps, const double* mean, const float* rstd, const void* dy,
                            const void* plus, void* dx, void* dweight, void* dbias, float* workspace, hipStream_t stream) {
  fsc::lnorm::Args a{};
  a.rows = rows; a.xs = x_stride; a.ys = dy_stride; a.width = width; a.eps = eps;
  a.x = x; a.w = weight; a.b = bias; a.mean = const_cast<double*>(mean); a.rstd = const_cast<float*>(rstd);
  a.dy = dy; a.plus = plus; a.ps = plus_stride; a.dx = dx; a.dw = dweight; a.db = dbias; a.part = workspace;
  return fsc::lnorm::backward(a, dtype, weight_dtype, activation, false, stream);
}

int fsc_layer_norm_backward_twice(int64_t rows, int32_t width, int32_t dtype, int32_t weight_dtype, int32_t activation,
                                  int64_t x_stride, int64_t dy_stride, int64_t v_stride, const void* x,
                                  const void* weight, const void* bias, float eps, const double* mean,
                                  const float* rstd, const void* dy, const void* v, const void* v_weight,
                                  const void* v_bias, void* grad_x, void* grad_dy, void* grad_weight, void* grad_bias,
                                  float* workspace, hipStream_t stream) {
  fsc::lnorm::Args a{};
  a.rows = rows; a.xs = x_stride; a.ys = dy_stride; a.vs = v_stride; a.width = width; a.eps = eps;
  a.x = x; a.w = weight; a.b = bias; a.mean = const_cast<double*>(mean); a.rstd = const_cast<float*>(rstd);
  a.dy = dy; a.v = v; a.vw = v_weight; a.vb = v_bias; a.gx = grad_x; a.gdy = grad_dy;
  a.dw = grad_weight; a.db = grad_bias; a.part = workspace;
  return fsc::lnorm::backward(a, dtype, weight_dtype, activation, true, stream);
}

}  // extern "C"
