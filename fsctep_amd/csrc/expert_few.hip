// The experts' products where an expert has few rows (an MD step of a molecule, one changed atom): what counts is
// the time to read the weights once.
//
// A block takes one expert and one strip of output columns.  It finds the expert's slots itself (a ballot over at
// most 1,024 indices: no sort, no plan launch) and keeps h, a, o and da by slot.  Its eight waves split the
// reduction and meet in LDS in a fixed order; every weight goes from memory into a register and from there into
// v_mfma_f32_16x16x4_f32 once for 16 rows (fp32 products throughout, at 9.8 TB/s of bf16 and 19 TB/s of fp32
// weights: more than memory gives).
//   up, down (weights contiguous along the reduction): lane (r, q) holds column r, four (bf16: eight) neighbouring
//     k from 4 q (8 q); a strip is 16 columns (up: their gate and up rows).
//   dh, dx (weights contiguous along the output): lane (r, q) holds four (eight) neighbouring columns of one k; a
//     strip is 64 (128) columns, product c of a load covering the columns 4 m + c (8 m + c).
#include <type_traits>

#include "common.h"
#include "expert_types.h"
#include "expert_args.h"

namespace fsc {
namespace experts {

constexpr int FT = 512;             // eight waves
constexpr int FW = FT / 64;

// N values from p (all of them if n > 0 with VEC, the first n otherwise), widened
template <int N, bool VEC, typename T>
__device__ __forceinline__ void get(const T* p, int n, float (&v)[N]) {
  if (VEC) {
    if (n > 0) load_vec<N>(p, v);
    else
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = 0.f;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = i < n ? to_f(p[i]) : 0.f;
  }
}

template <typename S, int MODE, bool VEC>
__global__ __launch_bounds__(FT) void few_kernel(Args g) {
  constexpr int CE = 16 / sizeof(S);                   // weights of a load
  constexpr bool ALONG = MODE == UP || MODE == DOWN;   // weights contiguous along the reduction
  constexpr int NA = MODE == UP ? 2 : MODE == DOWN ? 1 : CE;   // accumulators of 16 rows
  constexpr int NC = ALONG ? 16 : 16 * CE;             // output columns of a strip
  using R = std::conditional_t<MODE == DOWN || MODE == DX, float, S>;
  __shared__ f4 red[FW][NA][64];
  __shared__ int16_t list[FEW_SLOTS];
  __shared__ float dred[NA][16];
  const int cols = MODE == UP || MODE == DH ? g.F : g.H;
  const int strips = (cols + NC - 1) / NC;
  const int e = few_expert(g, blockIdx.x / strips);
  if (e < 0) return;
  const int n0 = (blockIdx.x % strips) * NC;
  const int cnt = few_slots(g, e, list);
  if (cnt == 0) return;
  __syncthreads();
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
  const int K = MODE == UP || MODE == DH ? g.H : MODE == DOWN ? g.F : 2 * g.ldf;

  for (int t0 = 0; t0 < cnt; t0 += 16) {
    const int slot = t0 + r < cnt ? list[t0 + r] : -1;
    const R* x = nullptr;
    if (slot >= 0) {
      if (MODE == UP) x = (const R*)g.x + (int64_t)(slot / g.k) * g.xs;
      if (MODE == DH) x = (const R*)g.dy + (int64_t)(slot / g.k) * g.ds;
      if (MODE == DOWN) x = (const R*)g.h + (int64_t)slot * g.ldf;
      if (MODE == DX) x = (const R*)g.da + (int64_t)slot * 2 * g.ldf;
    }
    f4 acc[NA];
#pragma unroll
    for (int c = 0; c < NA; ++c) acc[c] = f4{0.f, 0.f, 0.f, 0.f};
    if constexpr (ALONG) {
      const int n = n0 + r;
      const S* w = nullptr;
      if (n < cols)
        w = MODE == UP ? (const S*)g.w_in + ((int64_t)e * 2 * g.F + n) * g.H : (const S*)g.w_out + ((int64_t)e * g.H + n) * g.F;
      const int64_t up = (int64_t)g.F * g.H;           // from a column's gate row to its up row
      constexpr int STEP = 4 * CE;
#pragma unroll 5
      for (int k0 = wave * STEP; k0 < K; k0 += FW * STEP) {
        const int k = k0 + CE * q;
        float wv[NA][CE], xv[CE];
#pragma unroll
        for (int c = 0; c < NA; ++c) get<CE, VEC>(w + c * up + k, w ? K - k : 0, wv[c]);
        get<CE, VEC>(x + k, x ? K - k : 0, xv);
#pragma unroll
        for (int i = 0; i < CE; ++i)
#pragma unroll
          for (int c = 0; c < NA; ++c) acc[c] = mfma16x16x4(wv[c][i], xv[i], acc[c]);
      }
    } else {
      const int n = n0 + CE * r;
#pragma unroll 2
      for (int k0 = wave * 16; k0 < K; k0 += FW * 16) {
        const int k = k0 + 4 * q;
        float wv[4][CE], xv[4];
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          const S* w = nullptr;
          if (MODE == DH) {
            if (k + s < g.H) w = (const S*)g.w_out + ((int64_t)e * g.H + k + s) * g.F + n;
          } else {
            const int half = k + s >= g.ldf, f = k + s - half * g.ldf;
            if (k + s < K && f < g.F) w = (const S*)g.w_in + ((int64_t)e * 2 * g.F + half * g.F + f) * g.H + n;
          }
          get<CE, VEC>(w, w ? cols - n : 0, wv[s]);
        }
        if constexpr (MODE == DX) {
          get<4, true>(x + k, x ? K - k : 0, xv);      // K is a multiple of 16, da's rows are aligned
        } else {
          get<4, false>(x + k, x ? K - k : 0, xv);
        }
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
          for (int c = 0; c < NA; ++c) acc[c] = mfma16x16x4(wv[s][c], xv[s], acc[c]);
      }
    }
    __syncthreads();                                   // the last tile's sums have been read
#pragma unroll
    for (int c = 0; c < NA; ++c) red[wave][c][lane] = acc[c];
    __syncthreads();
    // thread (c, lane) of the first NA waves: the eight waves' sums of one accumulator, in order
    if (wave < (MODE == UP ? 1 : NA)) {
      f4 v[MODE == UP ? 2 : 1];
#pragma unroll
      for (int c = 0; c < (MODE == UP ? 2 : 1); ++c) {
        v[c] = red[0][MODE == UP ? c : wave][lane];
#pragma unroll
        for (int u = 1; u < FW; ++u) v[c] += red[u][MODE == UP ? c : wave][lane];
      }
      if constexpr (MODE == UP) {
        const int n = n0 + 4 * q;
        if (slot >= 0 && n < g.ldf) {
          f4 h;
#pragma unroll
          for (int j = 0; j < 4; ++j) h[j] = v[0][j] * sigmoid(v[0][j]) * v[1][j];
          if (g.a) {
            float* a = g.a + (int64_t)slot * 2 * g.ldf + n;
            st4(a, v[0]);
            st4(a + g.ldf, v[1]);
          }
          st4((float*)g.h + (int64_t)slot * g.ldf + n, h);
        }
      } else if constexpr (MODE == DOWN) {
        const int n = n0 + 4 * q;
        if (slot >= 0) store4(g.o + (int64_t)slot * g.ldo + n, v[0], g.H - n);
      } else if constexpr (MODE == DX) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int n = n0 + CE * (4 * q + j) + wave;
          if (slot >= 0 && n < g.H) g.o[(int64_t)slot * g.ldo + n] = v[0][j];
        }
      } else {
        float part = 0.f;
        const float wt = slot >= 0 ? g.weight[slot] : 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int n = n0 + CE * (4 * q + j) + wave;
          if (slot < 0 || n >= g.ldf) continue;
          const float* a = g.a + (int64_t)slot * 2 * g.ldf + n;
          const float ga = a[0], up = a[g.ldf], s = sigmoid(ga), act = ga * s, h = act * up, p = v[0][j], dh = p * wt;
          part += h * p;
          float* d = (float*)g.da + (int64_t)slot * 2 * g.ldf + n;
          d[0] = dh * up * (s * (1.f + ga * (1.f - s)));
          d[g.ldf] = dh * act;
          if (g.hw) ((float*)g.hw)[(int64_t)slot * g.ldf + n] = h * wt;
        }
        part += __shfl_xor(part, 16, 64);
        part += __shfl_xor(part, 32, 64);
        if (q == 0) dred[wave][r] = part;
      }
    }
    if constexpr (MODE == DH) {
      __syncthreads();
      if (g.dwpart && threadIdx.x < 16 && slot >= 0) {
        float t = dred[0][r];
#pragma unroll
        for (int c = 1; c < NA; ++c) t += dred[c][r];
        g.dwpart[(int64_t)(blockIdx.x % strips) * g.M + slot] = t;
      }
    }
  }
}

template <typename S, int MODE>
void launch_mode(const Args& g, bool vec, hipStream_t st) {
  constexpr int NC = MODE == UP || MODE == DOWN ? 16 : 16 * (16 / sizeof(S));
  const int cols = MODE == UP || MODE == DH ? g.F : g.H;
  const unsigned grid = (unsigned)few_blocks(g) * ((cols + NC - 1) / NC);
  if (vec) few_kernel<S, MODE, true><<<grid, FT, 0, st>>>(g);
  else few_kernel<S, MODE, false><<<grid, FT, 0, st>>>(g);
}

template <typename S>
void few_launch(int mode, const Args& g, bool vec, hipStream_t st) {
  if (mode == UP) launch_mode<S, UP>(g, vec, st);
  else if (mode == DOWN) launch_mode<S, DOWN>(g, vec, st);
  else if (mode == DH) launch_mode<S, DH>(g, vec, st);
  else launch_mode<S, DX>(g, vec, st);
}
template void few_launch<float>(int, const Args&, bool, hipStream_t);
template void few_launch<__bf16>(int, const Args&, bool, hipStream_t);

int few_parts(int F, int size) { return (F + 16 * (16 / size) - 1) / (16 * (16 / size)); }

// ---------------------------------------------------------------- 8 bits
typedef int i4v __attribute__((ext_vector_type(4)));

template <bool VEC>
__device__ __forceinline__ i4v get16(const int8_t* p, int n) {
  if (VEC) return n > 0 ? *reinterpret_cast<const i4v*>(p) : i4v{0, 0, 0, 0};
  alignas(16) int8_t b[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) b[i] = i < n ? p[i] : (int8_t)0;
  i4v v;
  __builtin_memcpy(&v, b, 16);
  return v;
}

// up: a block an expert and a group of 128 hidden columns, a wave 16 of them (gate and up rows over all of K), so
// the group's largest value is known in the block and h leaves it as codes.
template <bool VEC>
__global__ __launch_bounds__(FT) void few_up_q8_kernel(Args g) {
  __shared__ int16_t list[FEW_SLOTS];
  __shared__ float tops[FW][16];
  const int ng = g.ldf / QG, grp = blockIdx.x % ng;
  const int e = few_expert(g, blockIdx.x / ng);
  if (e < 0) return;
  const int cnt = few_slots(g, e, list);
  if (cnt == 0) return;
  __syncthreads();
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
  const int nr = grp * QG + wave * 16 + r, n = grp * QG + wave * 16 + 4 * q;
  const int8_t* wg = nr < g.F ? (const int8_t*)g.w_in + ((int64_t)e * 2 * g.F + nr) * g.H : nullptr;
  const int64_t up = (int64_t)g.F * g.H;
  f4 sg, su;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float* s = g.in_scale + (int64_t)e * 2 * g.F + n + j;
    sg[j] = n + j < g.F ? s[0] : 0.f;
    su[j] = n + j < g.F ? s[g.F] : 0.f;
  }
  for (int t0 = 0; t0 < cnt; t0 += 16) {
    const int slot = t0 + r < cnt ? list[t0 + r] : -1;
    const int8_t* x = slot >= 0 ? (const int8_t*)g.x + (int64_t)(slot / g.k) * g.xs : nullptr;
    i4v ag = {0, 0, 0, 0}, au = {0, 0, 0, 0};
#pragma unroll 5
    for (int k0 = 0; k0 < g.H; k0 += 64) {
      const int k = k0 + 16 * q;
      const i4v a = get16<VEC>(wg + k, wg ? g.H - k : 0), b = get16<VEC>(wg + up + k, wg ? g.H - k : 0);
      const i4v xv = get16<VEC>(x + k, x ? g.H - k : 0);
      ag = __builtin_amdgcn_mfma_i32_16x16x64_i8(a, xv, ag, 0, 0, 0);
      au = __builtin_amdgcn_mfma_i32_16x16x64_i8(b, xv, au, 0, 0, 0);
    }
    const float xs = slot >= 0 ? g.xscale[slot / g.k] : 0.f;
    float h[4], top = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float ga = n + j < g.F ? (float)ag[j] * (xs * sg[j]) : 0.f;
      const float u = n + j < g.F ? (float)au[j] * (xs * su[j]) : 0.f;
      h[j] = ga * sigmoid(ga) * u;
      top = max_nan(top, fabsf(h[j]));
    }
    top = max_nan(top, __shfl_xor(top, 16, 64));
    top = max_nan(top, __shfl_xor(top, 32, 64));
    __syncthreads();                                   // the last tile's maxima have been read
    if (q == 0) tops[wave][r] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < FW; ++w) top = max_nan(top, tops[w][r]);
    const float inv = top > 0.f ? 127.f / top : 0.f;
    if (slot >= 0) {
      int8_t b[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float c = rintf(h[j] * inv);
        b[j] = c >= -127.f && c <= 127.f ? (int8_t)c : (int8_t)0;
      }
      store_bytes<4>((int8_t*)g.h + (int64_t)slot * g.ldf + n, b);
      if (wave == 0 && q == 0) g.hscale[(int64_t)slot * ng + grp] = top / 127.f;
    }
  }
}

// down: a block an expert and 16 columns, the groups of h dealt to its waves.
template <bool VEC>
__global__ __launch_bounds__(256) void few_down_q8_kernel(Args g) {
  __shared__ int16_t list[FEW_SLOTS];
  __shared__ f4 red[4][64];
  const int strips = (g.H + 15) / 16, n0 = (blockIdx.x % strips) * 16, ng = g.ldf / QG;
  const int e = few_expert(g, blockIdx.x / strips);
  if (e < 0) return;
  const int cnt = few_slots(g, e, list);
  if (cnt == 0) return;
  __syncthreads();
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
  const int8_t* w = n0 + r < g.H ? (const int8_t*)g.w_out + ((int64_t)e * g.H + n0 + r) * g.F : nullptr;
  const int n = n0 + 4 * q;
  for (int t0 = 0; t0 < cnt; t0 += 16) {
    const int slot = t0 + r < cnt ? list[t0 + r] : -1;
    const int8_t* h = slot >= 0 ? (const int8_t*)g.h + (int64_t)slot * g.ldf : nullptr;
    f4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 2
    for (int grp = wave; grp < ng; grp += 4) {
      i4v acc = {0, 0, 0, 0};
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const int k = grp * QG + 64 * s + 16 * q;
        const i4v a = get16<VEC>(w + k, w ? g.F - k : 0), b = get16<true>(h + k, h ? 16 : 0);
        acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, acc, 0, 0, 0);
      }
      const float u = slot >= 0 ? g.hscale[(int64_t)slot * ng + grp] : 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) sum[j] += (float)acc[j] * u;
    }
    __syncthreads();
    red[wave][lane] = sum;
    __syncthreads();
    if (wave == 0 && slot >= 0) {
      sum = (red[0][lane] + red[1][lane]) + (red[2][lane] + red[3][lane]);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (n + j < g.H) sum[j] *= g.out_scale[(int64_t)e * g.H + n + j];
      store4(g.o + (int64_t)slot * g.ldo + n, sum, g.H - n);
    }
  }
}

void few_launch_q8(const Args& g, bool vin, bool vout, hipStream_t st) {
  const unsigned up = (unsigned)few_blocks(g) * (g.ldf / QG), down = (unsigned)few_blocks(g) * ((g.H + 15) / 16);
  if (vin) few_up_q8_kernel<true><<<up, FT, 0, st>>>(g);
  else few_up_q8_kernel<false><<<up, FT, 0, st>>>(g);
  if (vout) few_down_q8_kernel<true><<<down, 256, 0, st>>>(g);
  else few_down_q8_kernel<false><<<down, 256, 0, st>>>(g);
}

}  // namespace experts
}  // namespace fsc
