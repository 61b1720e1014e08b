// Root-mean-square norm of per-atom rows with the residual's addition: z = x + r (held in the rows' type),
// rstd = 1 / sqrt(mean z^2 + eps), y = (z rstd) w; its gradients; and the same with y in 8-bit codes and a scale
// for each row.  No counterpart in the reference (its readout norms are LayerNorms, models/mlp.py:8-66).
//
// Bound by memory: forward T H (2 in + 2 out) values with a residual, backward T H (3 in + 1 out).  A row is read
// once: a wave owns it and keeps it in registers between the sum of squares and the scaling (row_kernel); rows
// wider than that take a block and are read again from the caches (wide_kernel).
//
// The sum of squares runs in 64 bits (a square of a float is exact there) and the root is rounded to 32 bits once,
// so rstd, and with it every 8-bit code, is the same for any order of the sum.  At the sizes here the 64-bit
// operations hide behind the loads.
//
// Measured (a copy of this size moves 4.4 TB/s; smaller arrays come in part from the last-level cache): 100,000 x 640
// bf16 with a residual 91 us forward (512 MB, 5.6 TB/s) and 108 us backward (512 MB, 4.7 TB/s) with 5 us for the
// weight's gradient; 10,007 x 1,600 bf16 to codes 25 us (112 MB, 4.4 TB/s); 32 x 640 3.7 us, a launch.
#include <algorithm>

#include "common.h"
#include "expert_types.h"
#include "fsctep.h"

namespace fsc {
namespace norm {

constexpr int NT = 256;        // threads of a block: four waves

struct Args {
  int64_t rows, xs, rs;        // row strides of x and the residual, in elements
  int width;
  float eps;
  const void *x, *r, *w;
  void *y, *z;
  float* rstd;                 // y's row factors (forward) or the rows' code scales (8-bit codes)
};

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v = max_nan(v, __shfl_xor(v, off, 64));
  return v;
}

__device__ __forceinline__ float row_factor(double ss, int width, float eps) {
  return (float)(1.0 / sqrt(ss / width + (double)eps));
}

// The code of y in a row whose largest |y| is top: rint(y * (127 / top)), 0 in a row of zeros.  |y| <= top keeps
// the product within 127 after rounding; a row with a NaN has NaN for its scale and codes of 0.
__device__ __forceinline__ int8_t code_of(float y, float inv) {
  const float c = rintf(y * inv);
  return c >= -127.f && c <= 127.f ? (int8_t)c : (int8_t)0;
}

// One wave a row; lane l holds the chunks l, l + 64, .. of V values each (CH of them): 16 bytes a lane and load, a row
// read once.  Figures: top of the file.
template <typename T, typename W, int V, int CH, bool Q8>
__global__ __launch_bounds__(NT) void row_kernel(Args a) {
  const int64_t row = (int64_t)blockIdx.x * (NT / 64) + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (row >= a.rows) return;
  const T* x = (const T*)a.x + row * a.xs;
  float v[CH][V];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int at = (c * 64 + lane) * V;
    if (at < a.width) load_vec<V>(x + at, v[c]);
    else
#pragma unroll
      for (int j = 0; j < V; ++j) v[c][j] = 0.f;
  }
  if (a.r) {
    const T* r = (const T*)a.r + row * a.rs;
    T* z = (T*)a.z + row * a.width;
    float u[CH][V];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int at = (c * 64 + lane) * V;
      if (at < a.width) load_vec<V>(r + at, u[c]);
      else
#pragma unroll
        for (int j = 0; j < V; ++j) u[c][j] = 0.f;
    }
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int at = (c * 64 + lane) * V;
#pragma unroll
      for (int j = 0; j < V; ++j) v[c][j] = held<T>(v[c][j] + u[c][j]);
      if (at < a.width) store_vec<V>(z + at, v[c]);
    }
  }
  double ss = 0.0;
#pragma unroll
  for (int c = 0; c < CH; ++c)
#pragma unroll
    for (int j = 0; j < V; ++j) ss += (double)v[c][j] * (double)v[c][j];
  const float rstd = row_factor(wave_sum64(ss), a.width, a.eps);
  const W* w = (const W*)a.w;
  float top = 0.f;
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int at = (c * 64 + lane) * V;
    if (at < a.width) {
      float g[V];
      load_vec<V>(w + at, g);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        v[c][j] = v[c][j] * rstd * g[j];
        top = max_nan(top, fabsf(v[c][j]));
      }
      if (!Q8) store_vec<V>((T*)a.y + row * a.width + at, v[c]);
    }
  }
  if (!Q8) {
    if (lane == 0) a.rstd[row] = rstd;
    return;
  }
  top = wave_max(top);
  const float inv = top > 0.f ? 127.f / top : 0.f;
  int8_t* q = (int8_t*)a.y + row * a.width;
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int at = (c * 64 + lane) * V;
    if (at < a.width) {
      int8_t b[V];
#pragma unroll
      for (int j = 0; j < V; ++j) b[j] = code_of(v[c][j], inv);
      store_bytes<V>(q + at, b);
    }
  }
  if (lane == 0) a.rstd[row] = top / 127.f;
}

__device__ __forceinline__ double block_sum64(double v, double* red) {
  v = wave_sum64(v);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return (red[0] + red[1]) + (red[2] + red[3]);
}

// One block a row, any width and alignment: the row is read from memory once and from the caches again.  For rows that
// a wave's registers do not hold (above 2,048 values, unaligned rows too): 2 x 5,000 takes a launch's time.
template <typename T, typename W, bool Q8>
__global__ __launch_bounds__(NT) void wide_kernel(Args a) {
  __shared__ double red[NT / 64];
  __shared__ float redf[NT / 64];
  const int64_t row = blockIdx.x;
  const T* x = (const T*)a.x + row * a.xs;
  const T* r = a.r ? (const T*)a.r + row * a.rs : nullptr;
  T* z = a.r ? (T*)a.z + row * a.width : nullptr;
  const W* w = (const W*)a.w;
  auto value = [&](int i) { return r ? held<T>(to_f(x[i]) + to_f(r[i])) : to_f(x[i]); };
  double ss = 0.0;
  for (int i = threadIdx.x; i < a.width; i += NT) {
    const float v = value(i);
    if (z) z[i] = from_f<T>(v);
    ss += (double)v * (double)v;
  }
  const float rstd = row_factor(block_sum64(ss, red), a.width, a.eps);
  if (!Q8) {
    T* y = (T*)a.y + row * a.width;
    for (int i = threadIdx.x; i < a.width; i += NT) y[i] = from_f<T>(value(i) * rstd * to_f(w[i]));
    if (threadIdx.x == 0) a.rstd[row] = rstd;
    return;
  }
  float top = 0.f;
  for (int i = threadIdx.x; i < a.width; i += NT) top = max_nan(top, fabsf(value(i) * rstd * to_f(w[i])));
  top = wave_max(top);
  if ((threadIdx.x & 63) == 0) redf[threadIdx.x >> 6] = top;
  __syncthreads();
  top = max_nan(max_nan(redf[0], redf[1]), max_nan(redf[2], redf[3]));
  const float inv = top > 0.f ? 127.f / top : 0.f;
  int8_t* q = (int8_t*)a.y + row * a.width;
  for (int i = threadIdx.x; i < a.width; i += NT) q[i] = code_of(value(i) * rstd * to_f(w[i]), inv);
  if (threadIdx.x == 0) a.rstd[row] = top / 127.f;
}

// ---------------------------------------------------------------- backward
// With zn = z rstd and g = dy w: dx = rstd (g - zn mean(g zn)) + dz, dw = sum over rows of dy zn.  dw is added in
// two fixed-order steps (a partial row for each block, then over the blocks), so repeats give the same bits.
struct BackArgs {
  int64_t rows, zs, ys, ds;      // row strides of z, dy and dz, in elements
  int width;
  float eps;
  const void *z, *w, *dy, *dz;   // dz null: no gradient of the sum
  const float* rstd;
  void* dx;                      // null: the weight's gradient alone
  float* part;                   // [gridDim.x][width] partial dw, or null
};

// dx = rstd (w dy - zhat mean(w dy zhat)) + dz, dweight = sum over rows of dy zhat (zhat = z rstd).  A wave takes every
// gridDim.x * 4-th row and keeps its part of dweight in registers, so that a block writes one partial row.  NARROW: at most 64 columns, where dx is a
// difference of nearly equal numbers (exactly zero at one column) and is formed in 64 bits; the other instance does not
// carry those registers.
template <typename T, typename W, int V, int CH, bool NARROW>
__global__ __launch_bounds__(NT) void row_back_kernel(BackArgs a) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  __shared__ float buf[64 * V * CH];
  const W* w = (const W*)a.w;
  float g[CH][V], acc[CH][V];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int at = (c * 64 + lane) * V;
#pragma unroll
    for (int j = 0; j < V; ++j) g[c][j] = acc[c][j] = 0.f;
    if (at < a.width) load_vec<V>(w + at, g[c]);
  }
  for (int64_t row = (int64_t)blockIdx.x * (NT / 64) + wave; row < a.rows; row += (int64_t)gridDim.x * (NT / 64)) {
    const float rstd = a.rstd[row];
    float z[CH][V], d[CH][V];
    float dot = 0.f;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int at = (c * 64 + lane) * V;
      if (at < a.width) {
        load_vec<V>((const T*)a.z + row * a.zs + at, z[c]);
        load_vec<V>((const T*)a.dy + row * a.ys + at, d[c]);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) z[c][j] = d[c][j] = 0.f;
      }
    }
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        z[c][j] *= rstd;
        acc[c][j] += d[c][j] * z[c][j];
        d[c][j] *= g[c][j];
        dot += d[c][j] * z[c][j];
      }
    if (!a.dx) continue;
    const float mean = wave_sum(dot) / (float)a.width;
    // In a narrow row g can lie along zn, and dx is what is left of their difference (nearly nothing at width 1):
    // there the difference is formed in 64 bits, from z and a 64-bit root.
    double zr = 1.0, fine = 0.0;
    if constexpr (NARROW) {
      double ss = 0.0, gz = 0.0;
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const int at = (c * 64 + lane) * V + j;
          const double v = at < a.width ? (double)to_f(((const T*)a.z)[row * a.zs + at]) : 0.0;
          ss += v * v;
          gz += (double)g[c][j] * (at < a.width ? (double)to_f(((const T*)a.dy)[row * a.ys + at]) : 0.0) * v;
        }
      zr = 1.0 / sqrt(wave_sum64(ss) / a.width + (double)a.eps);
      fine = wave_sum64(gz) * zr / a.width;          // mean(g zn)
    }
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int at = (c * 64 + lane) * V;
      if (at < a.width) {
        float o[V];
        if (a.dz) load_vec<V>((const T*)a.dz + row * a.ds + at, o);
        else
#pragma unroll
          for (int j = 0; j < V; ++j) o[j] = 0.f;
        if constexpr (NARROW) {
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const double zn = (double)to_f(((const T*)a.z)[row * a.zs + at + j]) * zr;
            const double gd = (double)g[c][j] * (double)to_f(((const T*)a.dy)[row * a.ys + at + j]);
            o[j] += (float)(zr * (gd - zn * fine));
          }
        } else {
#pragma unroll
          for (int j = 0; j < V; ++j) o[j] += rstd * (d[c][j] - z[c][j] * mean);
        }
        store_vec<V>((T*)a.dx + row * a.width + at, o);
      }
    }
  }
  if (!a.part) return;
  // the four waves' sums, one wave after the other
#pragma unroll 1
  for (int k = 0; k < NT / 64; ++k) {
    if (wave == k) {
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const int at = (c * 64 + lane) * V + j;
          const float s = k ? buf[at] + acc[c][j] : acc[c][j];
          buf[at] = s;
        }
    }
    __syncthreads();
  }
  for (int i = threadIdx.x; i < a.width; i += NT) a.part[(int64_t)blockIdx.x * a.width + i] = buf[i];
}

template <typename T, typename W>
__global__ __launch_bounds__(NT) void wide_back_kernel(BackArgs a) {
  __shared__ float red[NT / 64];
  const W* w = (const W*)a.w;
  float* part = a.part ? a.part + (int64_t)blockIdx.x * a.width : nullptr;
  bool first = true;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const float rstd = a.rstd[row];
    const T* z = (const T*)a.z + row * a.zs;
    const T* dy = (const T*)a.dy + row * a.ys;
    const T* dz = a.dz ? (const T*)a.dz + row * a.ds : nullptr;
    float dot = 0.f;
    for (int i = threadIdx.x; i < a.width; i += NT) {
      const float zn = to_f(z[i]) * rstd, d = to_f(dy[i]);
      dot += d * to_f(w[i]) * zn;
      if (part) part[i] = first ? d * zn : part[i] + d * zn;   // this thread's columns in every row
    }
    first = false;
    if (!a.dx) continue;
    dot = wave_sum(dot);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = dot;
    __syncthreads();
    const float mean = ((red[0] + red[1]) + (red[2] + red[3])) / (float)a.width;
    T* dx = (T*)a.dx + row * a.width;
    for (int i = threadIdx.x; i < a.width; i += NT) {
      const float zn = to_f(z[i]) * rstd, d = to_f(dy[i]) * to_f(w[i]);
      dx[i] = from_f<T>((dz ? to_f(dz[i]) : 0.f) + rstd * (d - zn * mean));
    }
  }
  if (part && first)
    for (int i = threadIdx.x; i < a.width; i += NT) part[i] = 0.f;
}

// dw[c] = sum over the blocks' partial rows: 32 columns a block, 32 threads a column, then a fixed tree (the same sum
// every time).  1,024 x 640 partial sums: 5 us, in part the launch.
template <typename W>
__global__ __launch_bounds__(1024) void sum_kernel(const float* __restrict__ part, int n, int width, W* __restrict__ dw) {
  __shared__ float red[32][33];
  const int c = threadIdx.x & 31, k = threadIdx.x >> 5, col = blockIdx.x * 32 + c;
  float s = 0.f;
  if (col < width)
#pragma unroll 8
    for (int i = k; i < n; i += 32) s += part[(int64_t)i * width + col];
  red[k][c] = s;
  __syncthreads();
  s = group_sum(red[c][k], 32);          // column k of the block in lanes c = 0..31
  if (c == 0 && blockIdx.x * 32 + k < width) dw[blockIdx.x * 32 + k] = from_f<W>(s);
}

// Blocks of the backward: enough waves to fill the chip, few enough that the partial rows stay small beside the
// rows themselves (100,000 x 640 bf16, forward and backward with 512, 1,024, 2,048, 4,096 blocks: 252, 199, 208, 223 us).
inline int back_blocks(int64_t rows) { return (int)std::max<int64_t>(1, std::min<int64_t>((rows + 3) / 4, 1024)); }

inline bool aligned(const void* p, int64_t stride, int size, int vec) {
  return !p || ((uintptr_t)p % (size * vec) == 0 && stride % vec == 0);
}

// Calls f with (T, W, V, CH) where a wave can hold a row, V values a load: 16 bytes where every array allows it,
// single values for other strides and widths.  Returns false where the row is too wide.
template <typename T, typename W, typename F>
bool by_width(int width, bool vec, F&& f) {
  constexpr int V = 16 / sizeof(T);
  if (vec) {
    if (width <= 64 * V) f(std::integral_constant<int, V>{}, std::integral_constant<int, 1>{});
    else if (width <= 128 * V) f(std::integral_constant<int, V>{}, std::integral_constant<int, 2>{});
    else if (width <= 256 * V) f(std::integral_constant<int, V>{}, std::integral_constant<int, 4>{});
    else if (sizeof(T) == 4 && width <= 512 * V) f(std::integral_constant<int, V>{}, std::integral_constant<int, 8>{});
    else return false;
    return true;
  }
  if (width <= 128) f(std::integral_constant<int, 1>{}, std::integral_constant<int, 2>{});
  else if (width <= 512) f(std::integral_constant<int, 1>{}, std::integral_constant<int, 8>{});
  else if (width <= 2048) f(std::integral_constant<int, 1>{}, std::integral_constant<int, 32>{});
  else return false;
  return true;
}

template <typename T, typename W>
void launch_rows(const Args& a, bool q8, bool vec, hipStream_t st) {
  const unsigned grid = (unsigned)((a.rows + 3) / 4);
  const bool done = by_width<T, W>(a.width, vec, [&](auto V, auto CH) {
    constexpr int v = decltype(V)::value, ch = decltype(CH)::value;
    if (q8) row_kernel<T, W, v, ch, true><<<grid, NT, 0, st>>>(a);
    else row_kernel<T, W, v, ch, false><<<grid, NT, 0, st>>>(a);
  });
  if (done) return;
  if (q8) wide_kernel<T, W, true><<<(unsigned)a.rows, NT, 0, st>>>(a);
  else wide_kernel<T, W, false><<<(unsigned)a.rows, NT, 0, st>>>(a);
}

// At most 2^23 rows a launch: a grid has fewer than 2^32 threads, and a wide row takes 256.
template <typename T, typename W>
void launch_forward(const Args& all, bool q8, bool vec, hipStream_t st) {
  constexpr int64_t MOST = 1ll << 23;
  for (int64_t r0 = 0; r0 < all.rows; r0 += MOST) {
    Args a = all;
    a.rows = std::min(all.rows - r0, MOST);
    a.x = (const T*)all.x + r0 * all.xs;
    a.r = all.r ? (const T*)all.r + r0 * all.rs : nullptr;
    a.y = (char*)all.y + r0 * all.width * (int64_t)(q8 ? 1 : sizeof(T));
    a.z = all.z ? (T*)all.z + r0 * all.width : nullptr;
    a.rstd = all.rstd + r0;
    launch_rows<T, W>(a, q8, vec, st);
  }
}

template <typename T, typename W>
void launch_backward(const BackArgs& a, bool vec, W* dw, hipStream_t st) {
  const int blocks = back_blocks(a.rows);
  const bool done = by_width<T, W>(a.width, vec, [&](auto V, auto CH) {
    constexpr int v = decltype(V)::value, ch = decltype(CH)::value;
    if constexpr (v * ch <= 8) {
      if (a.width <= 64) {
        row_back_kernel<T, W, v, ch, true><<<blocks, NT, 0, st>>>(a);
        return;
      }
    }
    row_back_kernel<T, W, v, ch, false><<<blocks, NT, 0, st>>>(a);
  });
  if (!done) wide_back_kernel<T, W><<<blocks, NT, 0, st>>>(a);
  if (dw) sum_kernel<W><<<(a.width + 31) / 32, 1024, 0, st>>>(a.part, blocks, a.width, dw);
}

// runs the statements with (T, W) the element types of rows and weight
#define FSC_NORM_TYPES(...)                                                  \
  if (dtype == FSC_F32) { using T = float; using W = float; __VA_ARGS__; }   \
  else if (wtype == FSC_F32) { using T = __bf16; using W = float; __VA_ARGS__; } \
  else { using T = __bf16; using W = __bf16; __VA_ARGS__; }

int check_types(int64_t rows, int32_t width, int32_t dtype, int32_t wtype) {
  FSC_CHECK_ARG(rows >= 0 && rows < (1ll << 31), "rms_norm: rows must be below 2^31");
  FSC_CHECK_ARG(width >= 1 && width <= (1 << 20), "rms_norm: width must be 1 to 2^20");
  FSC_CHECK_ARG(dtype == FSC_F32 || dtype == FSC_BF16, "rms_norm: rows are float32 or bfloat16");
  FSC_CHECK_ARG(wtype == FSC_F32 || wtype == dtype, "rms_norm: the weight is float32 or of the rows' type");
  return 0;
}

int forward(int64_t rows, int32_t width, int32_t dtype, int32_t wtype, int64_t xs, int64_t rs, const void* x,
            const void* r, const void* w, float eps, void* y, void* z, float* row_out, bool q8, hipStream_t st) {
  if (int rc = check_types(rows, width, dtype, wtype)) return rc;
  if (rows == 0) return 0;
  FSC_CHECK_ARG(x && w && y && row_out && (!r || z), "rms_norm: null array");
  FSC_CHECK_ARG(xs >= 0 && (!r || rs >= 0), "rms_norm: negative row stride");
  const int size = dtype == FSC_F32 ? 4 : 2, vec = 16 / size, wsize = wtype == FSC_F32 ? 4 : 2;
  const bool wide = width % vec == 0 && aligned(x, xs, size, vec) && aligned(r, rs, size, vec) &&
                    aligned(w, 0, wsize, vec) && aligned(y, width, q8 ? 1 : size, vec) && aligned(z, width, size, vec);
  const Args a{rows, xs, rs, width, eps, x, r, w, y, z, row_out};
  FSC_NORM_TYPES(launch_forward<T, W>(a, q8, wide, st));
  return check_launch("rms_norm") ? 2 : 0;
}

}  // namespace norm
}  // namespace fsc

extern "C" {

int fsc_rms_norm_forward(int64_t rows, int32_t width, int32_t dtype, int32_t weight_dtype, int64_t x_stride,
                         int64_t residual_stride, const void* x, const void* residual, const void* weight, float eps,
                         void* y, void* z, float* rstd, hipStream_t stream) {
  return fsc::norm::forward(rows, width, dtype, weight_dtype, x_stride, residual_stride, x, residual, weight, eps, y,
                            z, rstd, false, stream);
}

int fsc_rms_norm_q8(int64_t rows, int32_t width, int32_t dtype, int32_t weight_dtype, int64_t x_stride,
                    int64_t residual_stride, const void* x, const void* residual, const void* weight, float eps,
                    int8_t* codes, float* scales, void* z, hipStream_t stream) {
  return fsc::norm::forward(rows, width, dtype, weight_dtype, x_stride, residual_stride, x, residual, weight, eps,
                            codes, z, scales, true, stream);
}

int fsc_rms_norm_workspace(int64_t rows, int32_t width, int64_t* floats) {
  FSC_CHECK_ARG(floats != nullptr, "rms_norm: null output");
  FSC_CHECK_ARG(rows >= 0 && width >= 1, "rms_norm: negative size");
  *floats = (int64_t)fsc::norm::back_blocks(rows) * width;
  return 0;
}

int fsc_rms_norm_backward(int64_t rows, int32_t width, int32_t dtype, int32_t weight_dtype, int64_t z_stride,
                          int64_t dy_stride, int64_t dz_stride, const void* z, const void* weight, const float* rstd,
                          float eps, const void* dy, const void* dz, void* dx, void* dweight, float* workspace,
                          hipStream_t stream) {
  using namespace fsc;
  using namespace fsc::norm;
  const int32_t dtype_ = dtype, wtype = weight_dtype;
  if (int rc = check_types(rows, width, dtype_, wtype)) return rc;
  FSC_CHECK_ARG(weight && (rows == 0 || (z && rstd && dy)), "rms_norm_backward: null array");
  FSC_CHECK_ARG(z_stride >= 0 && dy_stride >= 0 && (!dz || dz_stride >= 0), "rms_norm_backward: negative row stride");
  FSC_CHECK_ARG(!dweight || workspace, "rms_norm_backward: the weight's gradient needs a workspace");
  if (!dx && !dweight) return 0;
  if (rows == 0 && !dweight) return 0;
  const int size = dtype == FSC_F32 ? 4 : 2, vec = 16 / size, wsize = wtype == FSC_F32 ? 4 : 2;
  const bool wide = width % vec == 0 && aligned(z, z_stride, size, vec) && aligned(dy, dy_stride, size, vec) &&
                    aligned(dz, dz_stride, size, vec) && aligned(weight, 0, wsize, vec) && aligned(dx, width, size, vec);
  const BackArgs a{rows, z_stride, dy_stride, dz_stride, width, eps, z, weight, dy, dz, rstd, dx,
                   dweight ? workspace : nullptr};
  FSC_NORM_TYPES(launch_backward<T, W>(a, wide, (W*)dweight, stream));
  return check_launch("rms_norm_backward") ? 2 : 0;
}

}  // extern "C"
