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
  void* dx;
  float* part;                 // [gridDim.x][2][width] partial sums of the weight's and the bias' gradients, or null
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
// Any width and alignment; the row is read again from the caches for each pass over it.  Sums for the statistics run
// in 64 bits: a mean far from zero would lose the deviations otherwise.
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
  float* part = a.part ? a.part + (int64_t)blockIdx.x * 2 * a.width : nullptr;
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
    for (int i = threadIdx.x; i < a.width; i += NT) {
      F zh, du;
      terms(i, zh, du);
      dx[i] = from_f<T>((float)(r * (du * (F)at_or(w, i, 1.f) - mg - zh * mgz)));
    }
  }
}

template <typename T, typename W, bool SILU, typename F>
__global__ __launch_bounds__(NT) void wide_twice_kernel(Args a) {
  __shared__ double red[5 * NW];
  const W *w = (const W*)a.w, *b = (const W*)a.b, *vw = (const W*)a.vw, *vb = (const W*)a.vb;
  float* part = a.part ? a.part + (int64_t)blockIdx.x * 2 * a.width : nullptr;
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

// Column sums of the blocks' partial rows, the weight's gradient and the bias': 32 columns a block, 32 threads a column,
// then a fixed tree (the same sum every time).  blockIdx.y: which of the two.
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

// Blocks of the two backward passes.
inline int back_blocks(int64_t rows) { return (int)std::max<int64_t>(1, std::min<int64_t>((rows + 3) / 4, 1024)); }

template <typename T, typename W, bool SILU>
void launch_forward(const Args& all, hipStream_t st) {
  constexpr int64_t MOST = 1ll << 23;    // rows of a launch: a grid has fewer than 2^32 threads
  for (int64_t r0 = 0; r0 < all.rows; r0 += MOST) {
    Args a = all;
    a.rows = std::min(all.rows - r0, MOST);
    a.x = (const T*)all.x + r0 * all.xs;
    a.y = (T*)all.y + r0 * all.width;
    if (all.mean) {
      a.mean = all.mean + r0;
      a.rstd = all.rstd + r0;
    }
    wide_kernel<T, W, SILU><<<(unsigned)a.rows, NT, 0, st>>>(a);
  }
}

template <typename T, typename W, bool SILU>
void launch_backward(const Args& a, bool twice, W* dw, W* db, hipStream_t st) {
  const int blocks = back_blocks(a.rows);
  if (a.width <= 64) {
    if (twice) wide_twice_kernel<T, W, SILU, double><<<blocks, NT, 0, st>>>(a);
    else wide_back_kernel<T, W, SILU, double><<<blocks, NT, 0, st>>>(a);
  } else {
    if (twice) wide_twice_kernel<T, W, SILU, float><<<blocks, NT, 0, st>>>(a);
    else wide_back_kernel<T, W, SILU, float><<<blocks, NT, 0, st>>>(a);
  }
  if (a.part) sum_kernel<W><<<dim3((a.width + 31) / 32, 2), 1024, 0, st>>>(a.part, blocks, a.width, dw, db);
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

int backward(const Args& a, int32_t dtype, int32_t wtype, int32_t act, bool twice, void* dw, void* db, hipStream_t st) {
  if (int rc = check_types(a.rows, a.width, dtype, wtype, act)) return rc;
  FSC_CHECK_ARG(a.rows == 0 || (a.x && a.mean && a.rstd && a.dy), "layer_norm_backward: null array");
  FSC_CHECK_ARG(a.xs >= 0 && a.ys >= 0 && a.vs >= 0, "layer_norm_backward: negative row stride");
  FSC_CHECK_ARG(!(dw || db) || a.part, "layer_norm_backward: the weight's and the bias' gradients need a workspace");
  Args k = a;
  if (!dw && !db) k.part = nullptr;
  if (!k.part && (a.rows == 0 || !(a.dx || a.gx || a.gdy))) return 0;
  FSC_LN_TYPES(launch_backward<T, W, SILU>(k, twice, (W*)dw, (W*)db, st));
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
  *floats = (int64_t)fsc::lnorm::back_blocks(rows) * 2 * width;
  return 0;
}

int fsc_layer_norm_backward(int64_t rows, int32_t width, int32_t dtype, int32_t weight_dtype, int32_t activation,
                            int64_t x_stride, int64_t dy_stride, const void* x, const void* weight, const void* bias,
                            float eps, const double* mean, const float* rstd, const void* dy, void* dx, void* dweight,
                            void* dbias, float* workspace, hipStream_t stream) {
  fsc::lnorm::Args a{};
  a.rows = rows; a.xs = x_stride; a.ys = dy_stride; a.width = width; a.eps = eps;
  a.x = x; a.w = weight; a.b = bias; a.mean = const_cast<double*>(mean); a.rstd = const_cast<float*>(rstd);
  a.dy = dy; a.dx = dx; a.part = workspace;
  return fsc::lnorm::backward(a, dtype, weight_dtype, activation, false, dweight, dbias, stream);
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
  a.dy = dy; a.v = v; a.vw = v_weight; a.vb = v_bias; a.gx = grad_x; a.gdy = grad_dy; a.part = workspace;
  return fsc::lnorm::backward(a, dtype, weight_dtype, activation, true, grad_weight, grad_bias, stream);
}

}  // extern "C"
