// The AdamW step over many tensors at once, with the gradients clipped by their common norm, and states in 32 bits or in
// 8-bit floats with a scale for each 256 values.  The reference trains with torch's optimiser (training/trainer.py);
// formulas and formats: include/fsctep.h.
//
// Bound by memory: 28 bytes a value with states in 32 bits (parameter, two states in and out, gradient in), 16 with
// states in 8.  A launch takes a table of tensors in its arguments, and a block a share of one tensor.
#include <algorithm>
#include <cstring>

#include "common.h"
#include "expert_types.h"
#include "fsctep.h"

namespace fsc {
namespace adamw {

constexpr int NT = 256;
constexpr int SHARE = 2048;          // values of a block
constexpr int GROUP = 256;           // values that share a scale: a wave's, four a lane
constexpr int MOST = 48;             // tensors of a launch: their table has to fit 4 KB of arguments

struct Entry {
  int64_t n;
  void* p;
  const void* g;
  void *m, *v;
  float *m_scale, *v_scale, *master;
};
struct Table {
  int count;
  int32_t first[MOST + 1];           // first block of each tensor
  uint8_t bf16[MOST], wide[MOST];    // type of p and g; whether every array is aligned for four values a load
  Entry t[MOST];
};
static_assert(sizeof(Table) <= 3800, "kernel arguments");

struct Steps {
  int count;
  float* step[MOST];
};
// What the elements need, made on the GPU for each step: decay and clip, then for each tensor its step size, the root's
// factor and the number of the step.
struct Factors {
  float decay, clip, pad0, pad1;
  struct { float size, over, step, pad; } of[MOST];
};

struct Rule {
  float b1, b2, a1, a2, eps;         // a = 1 - b
};

__device__ __forceinline__ int tensor_of(const Table& tab, int block) {
  int lo = 0, hi = tab.count;        // first[lo] <= block < first[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (tab.first[mid] <= block) lo = mid;
    else hi = mid;
  }
  return lo;
}

// One value.  Every operation rounds by itself, root and quotient correctly (the compiler's default; no fused
// multiply-add): the codes of the 8-bit states then depend on
// nothing but the formula.
__device__ __forceinline__ void update(const Rule& k, float decay, float size, float over, float g, float& p, float& m,
                                       float& v, float& root) {
#pragma clang fp contract(off)
  m = k.b1 * m + k.a1 * g;
  v = k.b2 * v + (k.a2 * g) * g;
  root = sqrtf(v);
  p = p * decay - size * (m / (root * over + k.eps));
}

// 32 bits from a value's number and the step: two rounds of multiplying and folding.
__device__ __forceinline__ uint32_t hash(uint32_t place, uint32_t step) {
  uint32_t h = place * 0x9E3779B1u + step * 0x6A09E667u;
  h ^= h >> 16;
  h *= 0xBB67AE85u;
  h ^= h >> 15;
  h *= 0x3C6EF373u;
  return h ^ (h >> 16);
}

// 8-bit floats: the upper bits of a float in [0, 1], counted down from those of 1.
template <bool ROOT>
struct Code {
  static constexpr int SHIFT = ROOT ? 19 : 20, TOP = ROOT ? 255 : 127, BASE = (0x3F800000 >> SHIFT) - TOP;
};
template <bool ROOT>
__device__ __forceinline__ float decode(uint32_t c, float scale) {
  using K = Code<ROOT>;
  const uint32_t size = c & K::TOP;
  float y = size ? __uint_as_float((size + K::BASE) << K::SHIFT) : 0.f;
  if (!ROOT && c >= 128u) y = -y;
  return y * scale;
}
// over: 1 / the block's largest (0 where the block is zeros); bits: what the rounding adds below the last bit kept
template <bool ROOT>
__device__ __forceinline__ uint32_t encode(float x, float over, uint32_t bits) {
  using K = Code<ROOT>;
  const float y = fminf(fabsf(x) * over, 1.f);
  const uint32_t add = ROOT ? bits >> 13 : bits & 0xFFFFFu;
  const int c = min((int)((__float_as_uint(y) + add) >> K::SHIFT) - K::BASE, K::TOP);
  if (ROOT) return y > 0.f ? (uint32_t)max(c, 1) : 0u;
  return (uint32_t)max(c, 0) | (x < 0.f ? 128u : 0u);
}

__device__ __forceinline__ float wave_top(float v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v = max_nan(v, __shfl_xor(v, off, 64));
  return v;
}

// The step counts go up by one; decay, clip and each tensor's factors from them, in 64 bits.  One block.
__global__ __launch_bounds__(64) void prepare_kernel(Steps s, FscAdamSettings k, Factors* __restrict__ out) {
  const double lr = k.lr_tensor ? (double)*k.lr_tensor : k.lr;
  if (threadIdx.x == 0) {
    out->decay = (float)(1.0 - lr * k.weight_decay);
    double c = 1.0;
    if (k.norm) {
      c = k.max_norm / ((double)*k.norm + 1e-6);
      if (c > 1.0) c = 1.0;              // a norm that is NaN stays one
    }
    out->clip = (float)c;
  }
  const int i = threadIdx.x;
  if (i < s.count) {
    const float t = *s.step[i] + 1.f;
    *s.step[i] = t;
    out->of[i].size = (float)(lr / (1.0 - pow(k.beta1, (double)t)));
    out->of[i].over = (float)(1.0 / sqrt(1.0 - pow(k.beta2, (double)t)));
    out->of[i].step = t;
  }
}

// N values from `at` on, those past n zeros; V: by one load (N * size aligned)
template <int N, typename T>
__device__ __forceinline__ void read(const T* p, int64_t at, int64_t n, bool wide, float (&v)[N]) {
  if (wide && at + N <= n) {
    struct alignas(N * sizeof(T)) Pack { T t[N]; };
    const Pack k = *reinterpret_cast<const Pack*>(p + at);
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = to_f(k.t[j]);
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = at + j < n ? to_f(p[at + j]) : 0.f;
  }
}
template <int N, typename T>
__device__ __forceinline__ void write(T* p, int64_t at, int64_t n, bool wide, const float (&v)[N]) {
  if (wide && at + N <= n) {
    struct alignas(N * sizeof(T)) Pack { T t[N]; };
    Pack k;
#pragma unroll
    for (int j = 0; j < N; ++j) k.t[j] = from_f<T>(v[j]);
    *reinterpret_cast<Pack*>(p + at) = k;
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (at + j < n) p[at + j] = from_f<T>(v[j]);
  }
}

// Four values a lane, 256 a wave: the values that share a scale.
template <bool Q8>
__global__ __launch_bounds__(NT) void step_kernel(Table tab, Rule rule, const Factors* __restrict__ f) {
  const int i = tensor_of(tab, blockIdx.x);
  const Entry& e = tab.t[i];
  const int lane = threadIdx.x & 63;
  const bool wide = tab.wide[i], bf16 = tab.bf16[i];
  const float decay = f->decay, clip = f->clip, size = f->of[i].size, over = f->of[i].over;
  const uint32_t step = (uint32_t)(int64_t)f->of[i].step;
  const int64_t base = (int64_t)(blockIdx.x - tab.first[i]) * SHARE;
  for (int part = threadIdx.x >> 6; part < SHARE / GROUP; part += NT / 64) {
    const int64_t b0 = base + part * GROUP, at = b0 + lane * 4;
    if (b0 >= e.n) break;
    float p[4], g[4], m[4], v[4], root[4];
    if (bf16) {
      read<4>((const __bf16*)e.g, at, e.n, wide, g);
      read<4>(e.master, at, e.n, wide, p);
    } else {
      read<4>((const float*)e.g, at, e.n, wide, g);
      read<4>((const float*)e.p, at, e.n, wide, p);
    }
    const int64_t group = b0 / GROUP;
    if (Q8) {
      const float ms = e.m_scale[group], vs = e.v_scale[group];
      uint32_t mc = 0, vc = 0;
      if (wide && at + 4 <= e.n) {
        mc = *reinterpret_cast<const uint32_t*>((const uint8_t*)e.m + at);
        vc = *reinterpret_cast<const uint32_t*>((const uint8_t*)e.v + at);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (at + j < e.n) {
            mc |= (uint32_t)((const uint8_t*)e.m)[at + j] << (8 * j);
            vc |= (uint32_t)((const uint8_t*)e.v)[at + j] << (8 * j);
          }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        m[j] = decode<false>(mc >> (8 * j) & 255u, ms);
        const float r = decode<true>(vc >> (8 * j) & 255u, vs);
        v[j] = r * r;
      }
    } else {
      read<4>((const float*)e.m, at, e.n, wide, m);
      read<4>((const float*)e.v, at, e.n, wide, v);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) update(rule, decay, size, over, g[j] * clip, p[j], m[j], v[j], root[j]);
    if (bf16) {
      write<4>(e.master, at, e.n, wide, p);
      write<4>((__bf16*)e.p, at, e.n, wide, p);
    } else {
      write<4>((float*)e.p, at, e.n, wide, p);
    }
    if (Q8) {
      float mt = 0.f, vt = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        mt = max_nan(mt, fabsf(m[j]));
        vt = max_nan(vt, root[j]);
      }
      mt = wave_top(mt);
      vt = wave_top(vt);
      if (mt < 0x1p-100f) mt = 0.f;
      if (vt < 0x1p-100f) vt = 0.f;
      const float mo = mt > 0.f ? 1.f / mt : 0.f, vo = vt > 0.f ? 1.f / vt : 0.f;
      uint32_t mc = 0, vc = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t bits = hash((uint32_t)(at + j), step);
        mc |= encode<false>(m[j], mo, bits) << (8 * j);
        vc |= encode<true>(root[j], vo, bits) << (8 * j);
      }
      if (wide && at + 4 <= e.n) {
        *reinterpret_cast<uint32_t*>((uint8_t*)e.m + at) = mc;
        *reinterpret_cast<uint32_t*>((uint8_t*)e.v + at) = vc;
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (at + j < e.n) {
            ((uint8_t*)e.m)[at + j] = (uint8_t)(mc >> (8 * j));
            ((uint8_t*)e.v)[at + j] = (uint8_t)(vc >> (8 * j));
          }
      }
      if (lane == 0) {
        e.m_scale[group] = mt;
        e.v_scale[group] = vt;
      }
    } else {
      write<4>((float*)e.m, at, e.n, wide, m);
      write<4>((float*)e.v, at, e.n, wide, v);
    }
  }
}

// ---------------------------------------------------------------- the gradients' norm
constexpr int NORM_SHARE = 8192;

// Sum of squares of a block's share, in 64 bits (a square of a float is exact there).
__global__ __launch_bounds__(NT) void square_kernel(Table tab, double* __restrict__ part) {
  __shared__ double red[NT / 64];
  const int i = tensor_of(tab, blockIdx.x);
  const Entry& e = tab.t[i];
  const int64_t base = (int64_t)(blockIdx.x - tab.first[i]) * NORM_SHARE;
  double s = 0.0;
  for (int64_t at = base + threadIdx.x * 4; at < std::min<int64_t>(base + NORM_SHARE, e.n); at += NT * 4) {
    float g[4];
    if (tab.bf16[i]) read<4>((const __bf16*)e.g, at, e.n, tab.wide[i], g);
    else read<4>((const float*)e.g, at, e.n, tab.wide[i], g);
#pragma unroll
    for (int j = 0; j < 4; ++j) s += (double)g[j] * (double)g[j];
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) part[blockIdx.x] = (red[0] + red[1]) + (red[2] + red[3]);
}
__global__ __launch_bounds__(1024) void norm_kernel(const double* __restrict__ part, int64_t n, float* __restrict__ norm) {
  __shared__ double red[16];
  double s = 0.0;
  for (int64_t i = threadIdx.x; i < n; i += 1024) s += part[i];
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    s = 0.0;
    for (int w = 0; w < 16; ++w) s += red[w];
    *norm = (float)sqrt(s);
  }
}

template <bool ROOT>
__global__ __launch_bounds__(NT) void values_kernel(int64_t n, const uint8_t* __restrict__ c,
                                                    const float* __restrict__ scale, float* __restrict__ v) {
  for (int64_t i = (int64_t)blockIdx.x * NT + threadIdx.x; i < n; i += (int64_t)gridDim.x * NT)
    v[i] = decode<ROOT>(c[i], scale[i / GROUP]);
}

inline int64_t blocks_of(int64_t n, int share) { return (n + share - 1) / share; }

// Calls f(table, its blocks, its first tensor) for runs of at most MOST tensors whose blocks a grid can have.
template <typename F>
int by_tables(int32_t count, const FscAdamTensor* t, int share, F&& f) {
  constexpr int64_t GRID = 1ll << 23;          // blocks of 256 threads: fewer than 2^32 threads
  for (int32_t i = 0; i < count;) {
    Table tab{};
    int64_t blocks = 0;
    const int32_t i0 = i;
    for (; i < count && tab.count < MOST; ++i) {
      const FscAdamTensor& s = t[i];
      const int64_t b = blocks_of(s.n, share);
      FSC_CHECK_ARG(b <= GRID, "adamw: a tensor has more than 2^34 values");
      if (blocks + b > GRID) break;
      const int k = tab.count++;
      tab.first[k] = (int32_t)blocks;
      blocks += b;
      tab.bf16[k] = s.dtype == FSC_BF16;
      const uintptr_t half = (uintptr_t)s.g | (uintptr_t)s.p, full = (uintptr_t)s.master | (uintptr_t)s.m | (uintptr_t)s.v;
      tab.wide[k] = half % (s.dtype == FSC_BF16 ? 8 : 16) == 0 && full % 16 == 0;
      tab.t[k] = Entry{s.n, s.p, s.g, s.m, s.v, s.m_scale, s.v_scale, s.master};
    }
    tab.first[tab.count] = (int32_t)blocks;
    if (int rc = f(tab, blocks, i0)) return rc;
  }
  return 0;
}

int check_tensors(int32_t count, const FscAdamTensor* t, const char* what) {
  FSC_CHECK_ARG(count >= 0 && (count == 0 || t), std::string(what) + ": no tensors");
  for (int32_t i = 0; i < count; ++i) {
    FSC_CHECK_ARG(t[i].n >= 0 && (t[i].n == 0 || t[i].g), std::string(what) + ": a gradient is null");
    FSC_CHECK_ARG(t[i].dtype == FSC_F32 || t[i].dtype == FSC_BF16, std::string(what) + ": tensors are float32 or bfloat16");
  }
  return 0;
}

}  // namespace adamw
}  // namespace fsc

extern "C" {

int fsc_adamw_workspace(int32_t count, const FscAdamTensor* tensors, int64_t* step_bytes, int64_t* norm_bytes) {
  using namespace fsc::adamw;
  FSC_CHECK_ARG(step_bytes && norm_bytes && count >= 0 && (count == 0 || tensors), "adamw: null output");
  int64_t blocks = 0;
  for (int32_t i = 0; i < count; ++i) {
    FSC_CHECK_ARG(tensors[i].n >= 0, "adamw: negative size");
    blocks += blocks_of(tensors[i].n, NORM_SHARE);
  }
  *step_bytes = (int64_t)sizeof(Factors) * (count + 1);   // a launch takes at least one tensor
  *norm_bytes = 8 * std::max<int64_t>(1, blocks);
  return 0;
}

int fsc_grad_norm(int32_t count, const FscAdamTensor* tensors, void* workspace, float* norm, hipStream_t stream) {
  using namespace fsc;
  using namespace fsc::adamw;
  if (int rc = check_tensors(count, tensors, "grad_norm")) return rc;
  FSC_CHECK_ARG(workspace && norm, "grad_norm: null array");
  double* part = (double*)workspace;
  int64_t n = 0;
  if (int rc = by_tables(count, tensors, NORM_SHARE, [&](const Table& tab, int64_t blocks, int32_t) {
        if (blocks) square_kernel<<<(unsigned)blocks, NT, 0, stream>>>(tab, part + n);
        n += blocks;
        return 0;
      }))
    return rc;
  norm_kernel<<<1, 1024, 0, stream>>>(part, n, norm);
  return check_launch("grad_norm") ? 2 : 0;
}

int fsc_adamw_step(int32_t count, const FscAdamTensor* tensors, const FscAdamSettings* settings, void* workspace,
                   hipStream_t stream) {
  using namespace fsc;
  using namespace fsc::adamw;
  if (int rc = check_tensors(count, tensors, "adamw")) return rc;
  FSC_CHECK_ARG(settings, "adamw: no settings");
  const FscAdamSettings k = *settings;
  FSC_CHECK_ARG(k.bits == 32 || k.bits == 8, "adamw: states have 32 or 8 bits");
  FSC_CHECK_ARG(k.beta1 >= 0 && k.beta1 < 1 && k.beta2 >= 0 && k.beta2 < 1, "adamw: betas must be in [0, 1)");
  FSC_CHECK_ARG(k.eps >= 0 && k.weight_decay >= 0 && (k.lr_tensor || k.lr >= 0), "adamw: negative lr, eps or weight_decay");
  FSC_CHECK_ARG(!k.norm || k.max_norm > 0, "adamw: max_norm must be positive");
  if (count == 0) return 0;
  FSC_CHECK_ARG(workspace, "adamw: null workspace");
  for (int32_t i = 0; i < count; ++i) {
    const FscAdamTensor& t = tensors[i];
    FSC_CHECK_ARG(t.step, "adamw: a step count is null");
    FSC_CHECK_ARG(t.n == 0 || (t.p && t.m && t.v), "adamw: a parameter or a state is null");
    FSC_CHECK_ARG(t.n == 0 || t.dtype == FSC_F32 || t.master, "adamw: a bfloat16 parameter needs its float32 copy");
    FSC_CHECK_ARG(t.n == 0 || k.bits == 32 || (t.m_scale && t.v_scale), "adamw: a scale is null");
  }
  const Rule rule{(float)k.beta1, (float)k.beta2, (float)(1.0 - k.beta1), (float)(1.0 - k.beta2), (float)k.eps};
  Factors* f = (Factors*)workspace;
  if (int rc = by_tables(count, tensors, SHARE, [&](const Table& tab, int64_t blocks, int32_t i0) {
        Steps s{};
        s.count = tab.count;
        for (int j = 0; j < tab.count; ++j) s.step[j] = tensors[i0 + j].step;
        prepare_kernel<<<1, 64, 0, stream>>>(s, k, f);
        if (blocks && k.bits == 8) step_kernel<true><<<(unsigned)blocks, NT, 0, stream>>>(tab, rule, f);
        else if (blocks) step_kernel<false><<<(unsigned)blocks, NT, 0, stream>>>(tab, rule, f);
        ++f;
        return 0;
      }))
    return rc;
  return check_launch("adamw") ? 2 : 0;
}

int fsc_adamw_values(int64_t n, int32_t root, const uint8_t* codes, const float* scale, float* values,
                     hipStream_t stream) {
  using namespace fsc;
  using namespace fsc::adamw;
  FSC_CHECK_ARG(n >= 0, "adamw_values: negative size");
  if (n == 0) return 0;
  FSC_CHECK_ARG(codes && scale && values, "adamw_values: null array");
  const unsigned grid = (unsigned)std::min<int64_t>((n + NT - 1) / NT, 1 << 16);
  if (root) values_kernel<true><<<grid, NT, 0, stream>>>(n, codes, scale, values);
  else values_kernel<false><<<grid, NT, 0, stream>>>(n, codes, scale, values);
  return check_launch("adamw_values") ? 2 : 0;
}

}  // extern "C"
