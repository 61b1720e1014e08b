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
//   dh, dx (weights contiguous along the output): lane (r, q) holds two (four) neighbouring columns of one k; a
//     strip is 32 (64) columns, 128 bytes of a weight row, product c of a load covering the columns 2 m + c (4 m + c).
#include <type_traits>

#include "common.h"
#include "expert_tiles.h"

namespace fsc {
namespace experts {

constexpr int FT = 512;             // eight waves
constexpr int FW = FT / 64;

// B bytes from p, by 16- or 8-byte loads where ALIGNED (to four bytes)
typedef unsigned u4w __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned u2w __attribute__((ext_vector_type(2), aligned(4)));
template <int B, bool ALIGNED>
struct Raw {
  uint32_t v[B / 4];
  template <typename T>
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (ALIGNED && B % 16 == 0) {
#pragma unroll
      for (int i = 0; i < B / 16; ++i) {
        const u4w t = *(reinterpret_cast<const u4w*>(p) + i);
        v[4 * i] = t.x; v[4 * i + 1] = t.y; v[4 * i + 2] = t.z; v[4 * i + 3] = t.w;
      }
    } else if constexpr (ALIGNED) {
      const u2w t = *reinterpret_cast<const u2w*>(p);
      v[0] = t.x; v[1] = t.y;
    } else {
      T t[B / sizeof(T)];
#pragma unroll
      for (int i = 0; i < (int)(B / sizeof(T)); ++i) t[i] = p[i];
      __builtin_memcpy(v, t, B);
    }
  }
  // the first n values of p, zeros after them
  template <typename T>
  __device__ __forceinline__ void load(const T* p, int n) {
    T t[B / sizeof(T)];
#pragma unroll
    for (int i = 0; i < (int)(B / sizeof(T)); ++i) t[i] = i < n ? p[i] : (T)0;
    __builtin_memcpy(v, t, B);
  }
  // value i as a float
  template <typename T>
  __device__ __forceinline__ float at(int i) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(v[i]);
    else return __uint_as_float(i & 1 ? v[i >> 1] & 0xffff0000u : v[i >> 1] << 16);
  }
};

// 32 rows of 640, hidden 640, two of eight experts, fp32 (39 MB of weights, 9 us at a copy's rate, read once forward and once
// backward): up 11.2, down 7.1, dh 11.8, dx 15.0 us (bf16: 9.4, 6.4, 16.6, 20.6, whose dh and dx strips of 64 columns make 80
// blocks where fp32's make 160); what bounds them is the chain index, weights, rows, LDS of a block.
//
// Whole steps of the reduction run without conditions: a lane past the last column or row reads the last one's
// values, and what it computes is not stored.  The weights of a wave's first U steps are on their way before the
// expert's slots are known.  Only the last, partial step looks at the bounds.
template <typename S, int MODE, bool VEC>
__global__ __launch_bounds__(FT, MODE == UP || MODE == DOWN ? 4 : 2) void few_kernel(Args g) {
  constexpr bool ALONG = MODE == UP || MODE == DOWN;   // weights contiguous along the reduction
  constexpr int NW = FW;                               // waves
  constexpr int WB = ALONG ? 16 : 8;                   // bytes of a load of weights
  constexpr int CE = WB / sizeof(S);                   // its weights
  constexpr int NL = ALONG ? (MODE == UP ? 2 : 1) : 4; // loads of weights in a step
  constexpr int NA = MODE == UP ? 2 : MODE == DOWN ? 1 : CE;   // accumulators of 16 rows
  constexpr int NC = ALONG ? 16 : 16 * CE;             // output columns of a strip
  constexpr int STEP = ALONG ? 4 * CE : 16;            // reduction entries of a step
  constexpr int U = 5;                                 // steps in flight
  using R = std::conditional_t<MODE == DOWN || MODE == DX, float, S>;
  constexpr int XE = ALONG ? CE : 4;                   // values of x of a step
  __shared__ f4 red[NW][NA][64];
  __shared__ int16_t list[FEW_SLOTS];
  __shared__ float dred[NA][16];
  const int cols = MODE == UP || MODE == DH ? g.F : g.H;
  const int e = few_expert(g, blockIdx.y);
  if (e < 0) return;
  const int first = few_first(g);
  const int n0 = blockIdx.x * NC;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;

  // The reduction: PARTS runs of K entries (dx: the gate and the up half of da), each of `whole` whole steps.
  constexpr int PARTS = MODE == DX ? 2 : 1;
  const int K = MODE == UP || MODE == DH ? g.H : g.F;
  const int whole = K / STEP, steps = PARTS * whole;
  const int n = n0 + (ALONG ? r : CE * r);
  // (a lane whose columns reach past the last one reads on into the next row, zeros past the matrix: not stored)
  const int nc = ALONG ? min(n, cols - 1) : VEC && n >= cols ? cols - CE : n;
  const S* wbase = MODE == UP ? (const S*)g.w_in + ((int64_t)e * 2 * g.F + nc) * g.H
                   : MODE == DOWN ? (const S*)g.w_out + ((int64_t)e * g.H + nc) * g.F
                   : MODE == DH ? (const S*)g.w_out + (int64_t)e * g.H * g.F
                                : (const S*)g.w_in + (int64_t)e * 2 * g.F * g.H;
  const int64_t up = (int64_t)g.F * g.H;               // from a column's gate row to its up row
  // A whole step's weights: the matrix of an expert (below 2^31 bytes) through a buffer descriptor, whose scalar
  // offset carries the step, so that a load takes no address arithmetic.
  const int64_t msize = (MODE == UP || MODE == DX ? 2 : 1) * up;
  const S* const mbase = (MODE == UP || MODE == DX ? (const S*)g.w_in : (const S*)g.w_out) + e * msize;
  const __amdgpu_buffer_rsrc_t rsrc = buffer_rsrc_bytes(const_cast<S*>(mbase), (uint32_t)(msize * sizeof(S)));
  const int voff = (ALONG ? nc * K + CE * q : 4 * q * cols + nc) * (int)sizeof(S);
  auto load_step = [&](Raw<WB, VEC> (&w)[NL], int part, int k) {
    const int soff = (ALONG ? k : (part * K + k) * cols) * (int)sizeof(S);
#pragma unroll
    for (int c = 0; c < NL; ++c) {
      const int so = soff + c * (int)(ALONG ? up : (int64_t)cols) * (int)sizeof(S);
      if constexpr (WB == 16) {
        const u4v t = __builtin_bit_cast(u4v, __builtin_amdgcn_raw_buffer_load_b128(rsrc, voff, so, 0));
        w[c].v[0] = t.x; w[c].v[1] = t.y; w[c].v[2] = t.z; w[c].v[3] = t.w;
      } else {
        const u2v t = __builtin_bit_cast(u2v, __builtin_amdgcn_raw_buffer_load_b64(rsrc, voff, so, 0));
        w[c].v[0] = t.x; w[c].v[1] = t.y;
      }
    }
  };
  // a step's weights from entry k of a part on, `left` of them
  auto load_w = [&](Raw<WB, VEC> (&w)[NL], int part, int k, int left) {
    if constexpr (ALONG) {
#pragma unroll
      for (int c = 0; c < NL; ++c) {
        const S* p = wbase + c * up + k + CE * q;
        if (left >= STEP) w[c].load(p);
        else w[c].load(p, left - CE * q);
      }
    } else {
#pragma unroll
      for (int c = 0; c < NL; ++c) {
        const int kk = 4 * q + c;
        const int row = part * K + k + (kk < left ? kk : left - 1);
        const S* p = wbase + (int64_t)row * cols + nc;
        if (VEC && cols % CE == 0) w[c].load(p);
        else w[c].load(p, cols - nc);
      }
    }
  };
  auto load_x = [&](Raw<XE * sizeof(R), VEC>& v, const R* x, int part, int k, int left) {
    const R* p = x + (MODE == DX ? part * g.ldf : 0) + k + XE * q;
    if (left >= STEP) v.load(p);
    else v.load(p, left - XE * q);
  };
  f4 acc[NA];
  auto mul = [&](const Raw<WB, VEC> (&w)[NL], const Raw<XE * sizeof(R), VEC>& v) {
    if constexpr (ALONG) {
#pragma unroll
      for (int i = 0; i < CE; ++i)
#pragma unroll
        for (int c = 0; c < NA; ++c) acc[c] = mfma16x16x4(w[c].template at<S>(i), v.template at<R>(i), acc[c]);
    } else {
#pragma unroll
      for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int c = 0; c < NA; ++c) acc[c] = mfma16x16x4(w[s].template at<S>(c), v.template at<R>(s), acc[c]);
    }
  };

  Raw<WB, VEC> w[U][NL];
  auto load_chunk = [&](int i0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int s = wave + (i0 + u) * NW;              // the same for the whole wave
      if (s >= steps) continue;
      const int part = PARTS == 2 && s >= whole, k = (s - part * whole) * STEP;
      if constexpr (VEC) load_step(w[u], part, k);
      else load_w(w[u], part, k, STEP);
    }
  };
  load_chunk(0);
  const int cnt = few_slots(g, e, first, list);
  if (cnt == 0) return;
  __syncthreads();

  for (int t0 = 0; t0 < cnt; t0 += 16) {
    const bool live = t0 + r < cnt;
    const int slot = list[live ? t0 + r : 0];
    const R* x = MODE == UP     ? (const R*)g.x + few_row(g, slot) * g.xs
                 : MODE == DH   ? (const R*)g.dy + few_row(g, slot) * g.ds
                 : MODE == DOWN ? (const R*)g.h + (int64_t)slot * g.ldf
                                : (const R*)g.da + (int64_t)slot * 2 * g.ldf;
#pragma unroll
    for (int c = 0; c < NA; ++c) acc[c] = f4{0.f, 0.f, 0.f, 0.f};
    // dh: what the epilogue needs of the forward, on its way during the products (columns past the padding: the last)
    float av[2][4], wt = 0.f;
    if (MODE == DH && wave < NA) {
      wt = g.weight[slot];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float* a = g.a + (int64_t)slot * 2 * g.ldf + min(n0 + CE * (4 * q + j) + wave, g.ldf - 1);
        av[0][j] = a[0];
        av[1][j] = a[g.ldf];
      }
    }
    for (int i0 = 0; wave + i0 * NW < steps; i0 += U) {
      Raw<XE * sizeof(R), VEC> xv[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int s = wave + (i0 + u) * NW;
        const int part = PARTS == 2 && s >= whole;
        if (s < steps) load_x(xv[u], x, part, (s - part * whole) * STEP, STEP);
      }
      if (i0 > 0 || (t0 > 0 && wave + U * NW < steps)) load_chunk(i0);   // else the first chunk is still there
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (wave + (i0 + u) * NW < steps) mul(w[u], xv[u]);
    }
    if (K % STEP != 0 && wave < PARTS) {               // the partial step of part `wave`
      Raw<WB, VEC> wt[NL];
      Raw<XE * sizeof(R), VEC> xt;
      load_w(wt, wave, whole * STEP, K - whole * STEP);
      load_x(xt, x, wave, whole * STEP, K - whole * STEP);
      mul(wt, xt);
    }
    __syncthreads();                                   // the last tile's sums have been read
#pragma unroll
    for (int c = 0; c < NA; ++c) red[wave][c][lane] = acc[c];
    __syncthreads();
    // thread (c, lane) of the first NA waves: the waves' sums of one accumulator, in order
    if (wave < (MODE == UP ? 1 : NA)) {
      f4 v[MODE == UP ? 2 : 1];
#pragma unroll
      for (int c = 0; c < (MODE == UP ? 2 : 1); ++c) {
        f4 t[NW];
#pragma unroll
        for (int u = 0; u < NW; ++u) t[u] = red[u][MODE == UP ? c : wave][lane];
        v[c] = ((t[0] + t[1]) + (t[2] + t[3])) + ((t[4] + t[5]) + (t[6] + t[7]));
      }
      if constexpr (MODE == UP) {
        const int m = n0 + 4 * q;
        if (live && m < g.ldf) {
          f4 h;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (m + j >= g.F) v[0][j] = v[1][j] = 0.f;   // the padding
            h[j] = v[0][j] * sigmoid(v[0][j]) * v[1][j];
          }
          if (g.a) {
            float* a = g.a + (int64_t)slot * 2 * g.ldf + m;
            st4(a, v[0]);
            st4(a + g.ldf, v[1]);
          }
          st4((float*)g.h + (int64_t)slot * g.ldf + m, h);
        }
      } else if constexpr (MODE == DOWN) {
        const int m = n0 + 4 * q;
        if (live) store4(g.o + (int64_t)slot * g.ldo + m, v[0], g.H - m);
      } else if constexpr (MODE == DX) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int m = n0 + CE * (4 * q + j) + wave;
          if (live && m < g.H) g.o[(int64_t)slot * g.ldo + m] = v[0][j];
        }
      } else {
        float part = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int m = n0 + CE * (4 * q + j) + wave;
          if (!live || m >= g.ldf) continue;
          const float ga = av[0][j], ua = av[1][j], s = sigmoid(ga), act = ga * s, h = act * ua;
          const float p = m < g.F ? v[0][j] : 0.f, dh = p * wt;
          part += h * p;
          float* d = (float*)g.da + (int64_t)slot * 2 * g.ldf + m;
          d[0] = dh * ua * (s * (1.f + ga * (1.f - s)));
          d[g.ldf] = dh * act;
          if (g.hw) ((float*)g.hw)[(int64_t)slot * g.ldf + m] = h * wt;
        }
        part += __shfl_xor(part, 16, 64);
        part += __shfl_xor(part, 32, 64);
        if (q == 0) dred[wave][r] = part;
      }
    }
    if constexpr (MODE == DH) {
      __syncthreads();
      if (g.dwpart && threadIdx.x < 16 && live) {
        float t = dred[0][r];
#pragma unroll
        for (int c = 1; c < NA; ++c) t += dred[c][r];
        g.dwpart[(int64_t)blockIdx.x * g.M + slot] = t;
      }
    }
  }
}

constexpr int strip_cols(int mode, int size) { return mode == UP || mode == DOWN ? 16 : 16 * (8 / size); }

template <typename S, int MODE>
void launch_mode(const Args& g, bool vec, hipStream_t st) {
  constexpr int NC = strip_cols(MODE, sizeof(S));
  const int cols = MODE == UP || MODE == DH ? g.F : g.H;
  const dim3 grid((cols + NC - 1) / NC, few_blocks(g));
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

int few_parts(int F, int size) { return (F + strip_cols(DH, size) - 1) / strip_cols(DH, size); }

// ---------------------------------------------------------------- 8 bits
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

// up: a block an expert and 16 hidden columns, gate and up rows; its waves split the reduction and meet in LDS as whole
// numbers.  h stays in 32 bits here: its codes need the largest value of 128 columns, which no block holds (blocks of whole
// groups, a tenth as many, took 12 us where this takes 4.9 at 32 rows of 640, hidden 640, two of eight experts).
template <bool VEC>
__global__ __launch_bounds__(256) void few_up_q8_kernel(Args g) {
  __shared__ int16_t list[FEW_SLOTS];
  __shared__ i4v red[4][2][64];
  const int e = few_expert(g, blockIdx.y), n0 = blockIdx.x * 16;
  if (e < 0) return;
  const int first = few_first(g);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
  const int n = n0 + 4 * q;
  const int8_t* wg = (const int8_t*)g.w_in + ((int64_t)e * 2 * g.F + min(n0 + r, g.F - 1)) * g.H;
  const int64_t up = (int64_t)g.F * g.H;
  // the first U steps' weights and the columns' scales (a column past the last: the last one's), before the slots
  // are known
  constexpr int U = VEC ? 4 : 1;
  const int whole = g.H / 64;
  Raw<16, VEC> a[U], b[U];
  auto load_chunk = [&](int s0) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (wave + 4 * (s0 + u) < whole) {
        const int k = (wave + 4 * (s0 + u)) * 64 + 16 * q;
        a[u].load(wg + k);
        b[u].load(wg + up + k);
      }
  };
  load_chunk(0);
  f4 sg, su;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float* s = g.in_scale + (int64_t)e * 2 * g.F + min(n + j, g.F - 1);
    sg[j] = s[0];
    su[j] = s[g.F];
  }
  const int cnt = few_slots(g, e, first, list);
  if (cnt == 0) return;
  __syncthreads();
  for (int t0 = 0; t0 < cnt; t0 += 16) {
    const bool live = t0 + r < cnt;
    const int slot = list[live ? t0 + r : 0];
    const int8_t* x = (const int8_t*)g.x + few_row(g, slot) * g.xs;
    const float xs = g.xscale[few_row(g, slot)];
    i4v ag = {0, 0, 0, 0}, au = {0, 0, 0, 0};
    auto mul = [&](const i4v& a, const i4v& b, const i4v& xv) {
      ag = __builtin_amdgcn_mfma_i32_16x16x64_i8(a, xv, ag, 0, 0, 0);
      au = __builtin_amdgcn_mfma_i32_16x16x64_i8(b, xv, au, 0, 0, 0);
    };
    for (int s0 = 0; wave + 4 * s0 < whole; s0 += U) {
      Raw<16, VEC> xv[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (wave + 4 * (s0 + u) < whole) xv[u].load(x + (wave + 4 * (s0 + u)) * 64 + 16 * q);
      if (s0 > 0 || (t0 > 0 && wave + 4 * U < whole)) load_chunk(s0);
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (wave + 4 * (s0 + u) < whole)
          mul(__builtin_bit_cast(i4v, a[u]), __builtin_bit_cast(i4v, b[u]), __builtin_bit_cast(i4v, xv[u]));
    }
    if (wave == 3 && whole * 64 < g.H) {
      const int k = whole * 64 + 16 * q, n16 = g.H - k;
      mul(get16<VEC>(wg + k, n16), get16<VEC>(wg + up + k, n16), get16<VEC>(x + k, n16));
    }
    __syncthreads();                                   // the last tile's sums have been read
    red[wave][0][lane] = ag;
    red[wave][1][lane] = au;
    __syncthreads();
    if (wave == 0 && live) {
      ag = (red[0][0][lane] + red[1][0][lane]) + (red[2][0][lane] + red[3][0][lane]);
      au = (red[0][1][lane] + red[1][1][lane]) + (red[2][1][lane] + red[3][1][lane]);
      f4 h;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float ga = (float)ag[j] * (xs * sg[j]), u = (float)au[j] * (xs * su[j]);
        h[j] = n + j < g.F ? ga * sigmoid(ga) * u : 0.f;
      }
      st4((float*)g.h + (int64_t)slot * g.ldf + n, h);
    }
  }
}

// down: a block an expert and 16 columns, the groups of h dealt to its waves.  Lane (r, q) makes the codes of its 32 values
// of slot r's group, which are its part of the matrix operand.  32 rows of 640, hidden 640: 6.2 us.
template <bool VEC>
__global__ __launch_bounds__(FT) void few_down_q8_kernel(Args g) {
  __shared__ int16_t list[FEW_SLOTS];
  __shared__ f4 red[FW][64];
  const int n0 = blockIdx.x * 16, ng = g.ldf / QG;
  const int e = few_expert(g, blockIdx.y);
  if (e < 0) return;
  const int first = few_first(g);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
  const int8_t* w = (const int8_t*)g.w_out + ((int64_t)e * g.H + min(n0 + r, g.H - 1)) * g.F;
  const int n = n0 + 4 * q;
  // the first group's weights and the columns' scales, before the slots are known
  i4v a[2];
  auto weights = [&](int grp) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int k = grp * QG + 64 * s + 16 * q;
      a[s] = get16<VEC>(w + k, g.F - k);
    }
  };
  weights(wave);
  f4 scale;
#pragma unroll
  for (int j = 0; j < 4; ++j) scale[j] = g.out_scale[(int64_t)e * g.H + min(n + j, g.H - 1)];
  const int cnt = few_slots(g, e, first, list);
  if (cnt == 0) return;
  __syncthreads();
  for (int t0 = 0; t0 < cnt; t0 += 16) {
    const bool live = t0 + r < cnt;
    const int slot = list[live ? t0 + r : 0];
    const float* h = (const float*)g.h + (int64_t)slot * g.ldf;
    f4 sum = {0.f, 0.f, 0.f, 0.f};
    for (int grp = wave; grp < ng; grp += FW) {
      f4 v[2][4];
      uint32_t top = 0;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const int k = grp * QG + 64 * s + 16 * q;
#pragma unroll
        for (int j = 0; j < 4; ++j) v[s][j] = ld4(h + k + 4 * j);
      }
      if (grp != wave || (t0 > 0 && ng > FW)) weights(grp);   // else the first group's are still there
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int j = 0; j < 4; ++j) top = max(top, most4(v[s][j]));
      top = max(top, (uint32_t)__shfl_xor((int)top, 16, 64));
      top = max(top, (uint32_t)__shfl_xor((int)top, 32, 64));
      const float most = __uint_as_float(top), inv = most > 0.f ? 127.f / most : 0.f;
      i4v acc = {0, 0, 0, 0};
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        i4v b;
#pragma unroll
        for (int j = 0; j < 4; ++j) b[j] = (int)codes4(v[s][j], inv);
        acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[s], b, acc, 0, 0, 0);
      }
      const float u = most / 127.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) sum[j] += (float)acc[j] * u;
    }
    __syncthreads();
    red[wave][lane] = sum;
    __syncthreads();
    if (wave == 0 && live) {
      f4 t[FW];
#pragma unroll
      for (int u = 0; u < FW; ++u) t[u] = red[u][lane];
      sum = (((t[0] + t[1]) + (t[2] + t[3])) + ((t[4] + t[5]) + (t[6] + t[7]))) * scale;
      store4(g.o + (int64_t)slot * g.ldo + n, sum, g.H - n);
    }
  }
}

void few_launch_q8(const Args& g, bool vin, bool vout, hipStream_t st) {
  const dim3 up(g.ldf / 16, few_blocks(g)), down((g.H + 15) / 16, few_blocks(g));
  if (vin) few_up_q8_kernel<true><<<up, 256, 0, st>>>(g);
  else few_up_q8_kernel<false><<<up, 256, 0, st>>>(g);
  if (vout) few_down_q8_kernel<true><<<down, FT, 0, st>>>(g);
  else few_down_q8_kernel<false><<<down, FT, 0, st>>>(g);
}

}  // namespace experts
}  // namespace fsc
