// The AdamW step over many tensors at once, with the gradients clipped by their common norm, and states in 32 bits or in
// 8-bit floats with a scale for each 256 values.  The reference trains with torch's optimiser (training/trainer.py);
// formulas and formats: include/fsctep.h.
//
// Bound by memory: 28 bytes a value with states in 32 bits (parameter, two states in and out, gradient in), 16 with
// states in 8.  A launch takes a table of tensors in its arguments, and a block a share of one tensor.
//
// Measured (additions over large arrays move 6.1 TB/s here): 43 tensors of 44.5 M fp32 values 214 us (1,246 MB, 5.8 TB/s) and 57 us
// for the norm (178 MB); 39 M bf16 values with fp32 copies 192 and 28 us (1,101 MB, 5.7 TB/s); 79 M fp32 values with states in 8
// bits 234 us (1,258 MB, 5.4 TB/s, and vector instructions issued in 98 % of the cycles: 120 M of four cycles each on 1,024 SIMDs of
// 478,000; states in 32 bits 18 %) and 73 us for the norm (314 MB), their values 65 us for each state (393 MB, 6.0 TB/s); 1.7 M
// values 10 us.  prepare_kernel and norm_kernel are launches (3 us).
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
  uint8_t bf16[MOST];                // type of p and g
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

// One value.  Every operation that reaches a state rounds by itself, the root correctly (the compiler's default; no fused
// multiply-add): the codes of the 8-bit states then depend on
// nothing but the formula.
__device__ __forceinline__ void update(const Rule& k, float decay, float size, float over, float g, float& p, float& m,
                                       float& v, float& root) {
#pragma clang fp contract(off)
  m = k.b1 * m + k.a1 * g;
  v = k.b2 * v + (k.a2 * g) * g;
  root = sqrtf(v);
  // the parameter alone takes the hardware's reciprocal, off by 2^-23: of the step, which is far below the parameter
  p = p * decay - size * (m * __builtin_amdgcn_rcpf(root * over + k.eps));
}

// 32 bits from place * 0x9E3779B1 + step * 0x6A09E667, place the value's number: two rounds of folding and multiplying.
__device__ __forceinline__ uint32_t hash(uint32_t h) {
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
// over: 1 / the block's largest (0 where the block is zeros); bits: what the rounding adds below the last bit kept.  The mean of
// the roundings is the value from code 1 on (1.25 2^-16 of the largest, ROOT: 1.125 2^-16).  Below it there is no neighbour at a
// float's spacing: a root above zero becomes code 1, whose step is smaller than the value's own, others 0 from one
// spacing below code 1 on.
template <bool ROOT>
__device__ __forceinline__ uint32_t encode(float x, float over, uint32_t bits) {
  using K = Code<ROOT>;
  const float y = fminf(fabsf(x) * over, 1.f);
  const uint32_t add = ROOT ? bits >> 13 : bits & 0xFFFFFu;
  const int c = min((int)((__float_as_uint(y) + add) >> K::SHIFT) - K::BASE, K::TOP);
  if (ROOT) return y > 0.f ? (uint32_t)max(c, 1) : 0u;
  return (uint32_t)max(c, 0) | (x < 0.f ? 128u : 0u);
}

// The wave's largest of values at and above zero, by their bits, which order as they do, NaN last; 0 below 2^-100.
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}
__device__ __forceinline__ float wave_top(uint32_t v) {
  v = max(v, dpp<0xB1>(v));              // neighbours, pairs, then mirrored in 8 and in 16 lanes
  v = max(v, dpp<0x4E>(v));
  v = max(v, dpp<0x141>(v));
  v = max(v, dpp<0x140>(v));
  v = max(v, (uint32_t)__shfl_xor((int)v, 16, 64));
  v = max(v, (uint32_t)__shfl_xor((int)v, 32, 64));
  const float top = __uint_as_float(v);
  return top < 0x1p-100f ? 0.f : top;
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

// Four values at any address; `last`: the tensor ends among them, those past n are zeros and not written.
template <typename T>
struct alignas(sizeof(T)) Four { T t[4]; };
template <typename T>
__device__ __forceinline__ void read(const T* p, int64_t at, int64_t n, bool last, float (&v)[4]) {
  if (!last) {
    const Four<T> k = *reinterpret_cast<const Four<T>*>(p + at);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = to_f(k.t[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = at + j < n ? to_f(p[at + j]) : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void write(T* p, int64_t at, int64_t n, bool last, const float (&v)[4]) {
  if (!last) {
    Four<T> k;
#pragma unroll
    for (int j = 0; j < 4; ++j) k.t[j] = from_f<T>(v[j]);
    *reinterpret_cast<Four<T>*>(p + at) = k;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (at + j < n) p[at + j] = from_f<T>(v[j]);
  }
}
__device__ __forceinline__ uint32_t read_codes(const uint8_t* p, int64_t at, int64_t n, bool last) {
  uint32_t c = 0;
  if (!last) {
    const Four<uint8_t> k = *reinterpret_cast<const Four<uint8_t>*>(p + at);
    c = __builtin_bit_cast(uint32_t, k);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (at + j < n) c |= (uint32_t)p[at + j] << (8 * j);
  }
  return c;
}
__device__ __forceinline__ void write_codes(uint8_t* p, int64_t at, int64_t n, bool last, uint32_t c) {
  if (!last) {
    *reinterpret_cast<Four<uint8_t>*>(p + at) = __builtin_bit_cast(Four<uint8_t>, c);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (at + j < n) p[at + j] = (uint8_t)(c >> (8 * j));
  }
}

// Four values a lane, 256 a wave: the values that share a scale.  LAST: the group that the tensor ends in.
template <bool Q8, typename T, bool LAST>
__device__ __forceinline__ void step_group(const Entry& e, int64_t group, int lane, const Rule& rule, const Factors& f, int i) {
  const int64_t at = group * GROUP + lane * 4;
  const bool last = LAST && at + 4 > e.n;
  T* const p_ = (T*)e.p;
  float* const own = sizeof(T) == 2 ? e.master : (float*)e.p;   // the value that is stepped
  float p[4], g[4], m[4], v[4], root[4];
  read((const T*)e.g, at, e.n, last, g);
  read(own, at, e.n, last, p);
  if (Q8) {
    const float ms = e.m_scale[group], vs = e.v_scale[group];
    const uint32_t mc = read_codes((const uint8_t*)e.m, at, e.n, last), vc = read_codes((const uint8_t*)e.v, at, e.n, last);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      m[j] = decode<false>(mc >> (8 * j) & 255u, ms);
      const float r = decode<true>(vc >> (8 * j) & 255u, vs);
      v[j] = r * r;
    }
  } else {
    read((const float*)e.m, at, e.n, last, m);
    read((const float*)e.v, at, e.n, last, v);
  }
  const float clip = f.clip, size = f.of[i].size, over = f.of[i].over;
#pragma unroll
  for (int j = 0; j < 4; ++j) update(rule, f.decay, size, over, g[j] * clip, p[j], m[j], v[j], root[j]);
  write(own, at, e.n, last, p);
  if (sizeof(T) == 2) write(p_, at, e.n, last, p);
  if (Q8) {
    uint32_t mt = 0, vt = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      mt = max(mt, __float_as_uint(fabsf(m[j])));
      vt = max(vt, __float_as_uint(root[j]));
    }
    const float ml = wave_top(mt), vl = wave_top(vt);
    const float mo = ml > 0.f ? 1.f / ml : 0.f, vo = vl > 0.f ? 1.f / vl : 0.f;
    const uint32_t step = (uint32_t)(int64_t)f.of[i].step, salt = (uint32_t)at * 0x9E3779B1u + step * 0x6A09E667u;
    uint32_t mc = 0, vc = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t bits = hash(salt + j * 0x9E3779B1u);
      mc |= encode<false>(m[j], mo, bits) << (8 * j);
      vc |= encode<true>(root[j], vo, bits) << (8 * j);
    }
    write_codes((uint8_t*)e.m, at, e.n, last, mc);
    write_codes((uint8_t*)e.v, at, e.n, last, vc);
    if (lane == 0) {
      e.m_scale[group] = ml;
      e.v_scale[group] = vl;
    }
  } else {
    write((float*)e.m, at, e.n, last, m);
    write((float*)e.v, at, e.n, last, v);
  }
}

template <bool Q8>
__global__ __launch_bounds__(NT) void step_kernel(Table tab, Rule rule, const Factors* __restrict__ f) {
  const int i = tensor_of(tab, blockIdx.x);
  const Entry& e = tab.t[i];
  const int lane = threadIdx.x & 63;
  const int64_t g0 = (int64_t)(blockIdx.x - tab.first[i]) * (SHARE / GROUP) + (threadIdx.x >> 6);
#pragma unroll
  for (int k = 0; k < SHARE / GROUP; k += NT / 64) {
    const int64_t group = g0 + k;
    if (group * GROUP >= e.n) break;
    const bool whole = (group + 1) * GROUP <= e.n;
    if (tab.bf16[i]) {
      if (whole) step_group<Q8, __bf16, false>(e, group, lane, rule, *f, i);
      else step_group<Q8, __bf16, true>(e, group, lane, rule, *f, i);
    } else {
      if (whole) step_group<Q8, float, false>(e, group, lane, rule, *f, i);
      else step_group<Q8, float, true>(e, group, lane, rule, *f, i);
    }
  }
}

// ---------------------------------------------------------------- the gradients' norm
constexpr int NORM_SHARE = 8192, NORM_STEPS = NORM_SHARE / (NT * 4);

// Sum of squares of a block's share, in 64 bits (a square of a float is exact there).  A whole share's loads are on their way
// together (314 MB: one at a time 95 us, eight 72 us).
template <typename T>
__device__ __forceinline__ double squares(const T* g, int64_t base, int64_t n) {
  double s = 0.0;
  if (n >= 4) {
    // vectors past the end: the last four values again, those that are not a lane's own left out
    Four<T> v[NORM_STEPS];
#pragma unroll
    for (int k = 0; k < NORM_STEPS; ++k)
      v[k] = *reinterpret_cast<const Four<T>*>(g + std::min<int64_t>(base + (k * NT + threadIdx.x) * 4, n - 4));
#pragma unroll
    for (int k = 0; k < NORM_STEPS; ++k) {
      const int64_t at = base + (k * NT + threadIdx.x) * 4, skip = at - std::min<int64_t>(at, n - 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const double x = j >= skip ? (double)to_f(v[k].t[j]) : 0.0;
        s += x * x;
      }
    }
  } else if (threadIdx.x < n) {
    const double x = (double)to_f(g[threadIdx.x]);
    s = x * x;
  }
  return s;
}
__global__ __launch_bounds__(NT) void square_kernel(Table tab, double* __restrict__ part) {
  __shared__ double red[NT / 64];
  const int i = tensor_of(tab, blockIdx.x);
  const Entry& e = tab.t[i];
  const int64_t base = (int64_t)(blockIdx.x - tab.first[i]) * NORM_SHARE;
  double s = tab.bf16[i] ? squares((const __bf16*)e.g, base, e.n) : squares((const float*)e.g, base, e.n);
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

// Four codes a thread, which share a scale, VALUE_STEPS times a block's width apart; stored past the caches.
constexpr int VALUE_STEPS = 4, VALUE_SHARE = NT * 4 * VALUE_STEPS;
template <bool ROOT>
__global__ __launch_bounds__(NT) void values_kernel(int64_t n, const uint8_t* __restrict__ c,
                                                    const float* __restrict__ scale, float* __restrict__ v, int64_t first) {
  const int64_t base = first + (int64_t)blockIdx.x * VALUE_SHARE;
  if (base + VALUE_SHARE <= n) {
    struct alignas(1) Pack { uint8_t t[4]; };
    Pack k[VALUE_STEPS];
    float s[VALUE_STEPS];
#pragma unroll
    for (int j = 0; j < VALUE_STEPS; ++j) {
      const int64_t at = base + (j * NT + threadIdx.x) * 4;
      k[j] = *reinterpret_cast<const Pack*>(c + at);
      s[j] = scale[at / GROUP];
    }
#pragma unroll
    for (int j = 0; j < VALUE_STEPS; ++j) {
      typedef float f4s __attribute__((ext_vector_type(4), aligned(4)));
      f4s x;
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = decode<ROOT>(k[j].t[i], s[j]);
      __builtin_nontemporal_store(x, reinterpret_cast<f4s*>(v + base + (j * NT + threadIdx.x) * 4));
    }
  } else {
    for (int64_t i = base + threadIdx.x; i < n; i += NT) v[i] = decode<ROOT>(c[i], scale[i / GROUP]);
  }
}

inline int64_t blocks_of(int64_t n, int share) { return (n + share - 1) / share; }

// Calls f(table, its blocks, its first tensor) for runs of at most MOST tensors whose blocks a grid can have (check_tensors: each
// tensor's by itself fits one).
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
      if (blocks + b > GRID) break;
      const int k = tab.count++;
      tab.first[k] = (int32_t)blocks;
      blocks += b;
      tab.bf16[k] = s.dtype == FSC_BF16;
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
    FSC_CHECK_ARG(t[i].n <= (int64_t)SHARE << 23, std::string(what) + ": a tensor has more than 2^34 values");
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
  constexpr int64_t MOST_VALUES = (int64_t)VALUE_SHARE << 23;             // fewer than 2^32 threads a launch
  for (int64_t f = 0; f < n; f += MOST_VALUES) {
    const unsigned grid = (unsigned)((std::min(n - f, MOST_VALUES) + VALUE_SHARE - 1) / VALUE_SHARE);
    if (root) values_kernel<true><<<grid, NT, 0, stream>>>(n, codes, scale, values, f);
    else values_kernel<false><<<grid, NT, 0, stream>>>(n, codes, scale, values, f);
  }
  return check_launch("adamw_values") ? 2 : 0;
}

}  // extern "C"
