// Pieces of the tile kernels of the experts' products (expert_mlp.hip).
#pragma once

#include "common.h"
#include "expert_types.h"
#include "expert_args.h"

namespace fsc {
namespace experts {

typedef int i4v __attribute__((ext_vector_type(4)));

// F32: fp32 products from two scaled fp16 parts an operand (mfma_x3); X6: from three bf16 parts (mfma_x6); FINE: bf16
// operands as they are, fp32 ones in three bf16 parts (one product, or three where the other operand is fp32)
enum Kind { F32 = 0, BF16 = 1, I8 = 2, X6 = 3, FINE = 4 };

// T: the type between the kernels; BK: reduction entries of a step; CE: those of a 16-byte LDS chunk; planes<O>: LDS
// planes of an operand that is an O in memory
template <int KIND> struct El;
template <> struct El<F32> {
  using T = float;
  static constexpr int BK = 32, CE = 8;
  template <typename O> static constexpr int planes = 2;
};
template <> struct El<X6> {
  using T = float;
  static constexpr int BK = 32, CE = 8;
  template <typename O> static constexpr int planes = 3;
};
template <> struct El<FINE> {
  using T = float;
  static constexpr int BK = 32, CE = 8;
  template <typename O> static constexpr int planes = sizeof(O) == 4 ? 3 : 1;
};
template <> struct El<BF16> {
  using T = __bf16;
  static constexpr int BK = 64, CE = 8;
  template <typename O> static constexpr int planes = 1;
};
template <> struct El<I8> {
  using T = int8_t;
  static constexpr int BK = 128, CE = 16;
  template <typename O> static constexpr int planes = 1;
};

template <int KIND> struct Acc { using V = f4; };
template <> struct Acc<I8> { using V = i4v; };

// The power of two k that brings values up to `most` (bits of a non-negative float) below 2^14, for their two fp16
// parts: 0 where there is nothing to bring (zero, infinity, NaN); within the exponents of normal floats.
__device__ __forceinline__ int part_exp(uint32_t most) {
  if (most == 0 || most >= 0x7f800000u) return 0;
  return min(max(14 - __builtin_amdgcn_frexp_expf(__uint_as_float(most)), -126), 126);
}
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// Workgroup -> (row tile, column tile).  Workgroup w runs on XCD w % 8: each XCD takes a contiguous run of row
// tiles with all their column tiles, so that a tile's rows and an expert's weights meet in one L2.
__device__ __forceinline__ bool tile_of(int n_tiles, int n_cols, int& t, int& c) {
  const int per = (n_tiles * n_cols + 7) / 8;
  const int i = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  t = i / n_cols;
  c = i - t * n_cols;
  return t < n_tiles && (int)(blockIdx.x >> 3) < per;
}
inline unsigned tile_grid(int64_t n_tiles, int64_t n_cols) { return (unsigned)((n_tiles * n_cols + 7) / 8 * 8); }

// A row tile of an expert: sorted positions p0 .. p0 + rows - 1, their slots and rows in LDS.
struct RowTile {
  int e, rows;
  int64_t p0;
  const int32_t *slots, *rws;
};

// Sixteen rows of a wave's sums, NI weight tiles wide, through LDS (TURN floats a wave) into rows: lane l holds the
// columns 4 (l % L) .. + 3 of the rows l / L + s (64 / L), L = 4 NI lanes a row, so that stores and loads of a row
// cover whole 128-byte lines where lane (r, q) of the products would touch 64 bytes of sixteen rows.  The wave reads
// only what it wrote itself.
template <int NI> struct Turned {
  static constexpr int L = 4 * NI, R = 64 / L, S = 16 / R, LD = 16 * NI + 4;
  f4 v[S];
};
template <int NI, typename F>
__device__ __forceinline__ void turn_rows(F&& sums, float* buf, Turned<NI>& t) {
  const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
  using U = Turned<NI>;
#pragma unroll
  for (int i = 0; i < NI; ++i) st4(buf + r * U::LD + 16 * i + 4 * q, sums(i));
  wave_sync();
#pragma unroll
  for (int s = 0; s < U::S; ++s) t.v[s] = ld4(buf + (s * U::R + lane / U::L) * U::LD + 4 * (lane % U::L));
  wave_sync();
}
constexpr int TURN = 16 * 68;

// Raises a row's largest magnitude so far (bits; a NaN is above all numbers) by the values of `width` neighbouring
// lanes, all of which call it with the same row.  Maxima do not depend on their order.
__device__ __forceinline__ uint32_t most4(const f4& v) {
  return max(max(abs_bits(v.x), abs_bits(v.y)), max(abs_bits(v.z), abs_bits(v.w)));
}
__device__ __forceinline__ void raise(uint32_t* most, uint32_t m, int width, bool in) {
#pragma unroll
  for (int off = width >> 1; off > 0; off >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, off, 64));
  if (in && (threadIdx.x & (width - 1)) == 0) atomicMax(most, m);
}

// Four codes rint(h inv), |h inv| <= 127: the sum with 1.5 * 2^23 has the whole number in its low bits.  (A NaN or an
// infinity has some code: its group's unit is one too.)
__device__ __forceinline__ uint32_t codes4(const f4& h, float inv) {
  uint32_t w[4];
#pragma unroll
  for (int v = 0; v < 4; ++v) w[v] = __float_as_uint(__fadd_rn(__fmul_rn(h[v], inv), 12582912.f));
  return __builtin_amdgcn_perm(__builtin_amdgcn_perm(w[3], w[2], 0x0c0c0400u), __builtin_amdgcn_perm(w[1], w[0], 0x0c0c0400u), 0x05040100u);
}

// What becomes of a tile's sums.  acc[i][j]: weight tile w0 + i (16 rows of the weight operand), row tile x0 + j; lane
// (r, q) holds the weight rows 4 q .. 4 q + 3 of row r.  n0: the tile's first output column (up: a weight tile pair
// is 16 hidden columns, gate then up).  buf: LDS that nobody reads any more, TURN floats for each wave, then WW * BM
// floats (dh, 8-bit up); WW waves side by side along the weights, this one the wn-th.
template <int KIND, int MODE, int NI, int NJ, int WW, int BM, typename V>
__device__ __forceinline__ void finish(const Args& g, const RowTile& t, int n0, int ci, int wn, int w0, int x0,
                                       V (&acc)[NI][NJ], float* buf) {
  using T = typename El<KIND>::T;
  const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
  float* const mine = buf + (threadIdx.x >> 6) * TURN;
  float* const red = buf + (blockDim.x >> 6) * TURN;
  if constexpr (MODE == DOWN || MODE == DX) {
    using U = Turned<NI>;
    const int n = n0 + w0 * 16 + 4 * (lane % U::L);
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      U u;
      turn_rows<NI>([&](int i) { return acc[i][j]; }, mine, u);
#pragma unroll
      for (int s = 0; s < U::S; ++s) {
        const int row = 16 * (x0 + j) + s * U::R + lane / U::L;
        if (row < t.rows) store4(g.o + (t.p0 + row) * g.ldo + n, u.v[s], g.H - n);
      }
    }
  } else if constexpr (MODE == UP && KIND == I8) {
    // the block holds whole groups of 128 columns: their largest values, then the codes
    static_assert(WW * NI == 16, "8-bit up: 128 hidden columns a tile");
    f4 h[NI / 2][NJ], sg[NI / 2], su[NI / 2];
    uint32_t top[NJ];
#pragma unroll
    for (int i = 0; i < NI / 2; ++i)
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const float* s = g.in_scale + (int64_t)t.e * 2 * g.F + min(n0 + (w0 / 2 + i) * 16 + 4 * q + v, g.F - 1);
        sg[i][v] = s[0];
        su[i][v] = s[g.F];
      }
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const int row = 16 * (x0 + j) + r;
      const float xs = g.xscale[t.rws[row]];               // a row past the tile: any row's, not stored
      top[j] = 0;
#pragma unroll
      for (int i = 0; i < NI / 2; ++i) {
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const float ga = (float)acc[2 * i][j][v] * (xs * sg[i][v]), up = (float)acc[2 * i + 1][j][v] * (xs * su[i][v]);
          h[i][j][v] = ga * sigmoid(ga) * up;              // columns past the last have sums of zero
        }
        top[j] = max(top[j], most4(h[i][j]));
      }
      top[j] = max(top[j], (uint32_t)__shfl_xor((int)top[j], 16, 64));
      top[j] = max(top[j], (uint32_t)__shfl_xor((int)top[j], 32, 64));
      if (q == 0) reinterpret_cast<uint32_t*>(red)[wn * BM + row] = top[j];
    }
    __syncthreads();
    // a row's 128 codes are one line: through LDS, so that eight lanes store it
    constexpr int LD = QG + 16;
    int8_t* const line = reinterpret_cast<int8_t*>(buf);
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const int row = 16 * (x0 + j) + r;
#pragma unroll
      for (int w = 0; w < WW; ++w) top[j] = max(top[j], reinterpret_cast<const uint32_t*>(red)[w * BM + row]);
      const float most = __uint_as_float(top[j]), inv = most > 0.f ? 127.f / most : 0.f;
#pragma unroll
      for (int i = 0; i < NI / 2; ++i)
        *reinterpret_cast<uint32_t*>(line + row * LD + (w0 / 2 + i) * 16 + 4 * q) = codes4(h[i][j], inv);
      if (wn == 0 && q == 0 && row < t.rows) g.hscale[(t.p0 + row) * (g.ldf / QG) + n0 / QG] = most / 127.f;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < t.rows * (QG / 16); i += blockDim.x) {
      const int row = i / (QG / 16), c = i % (QG / 16) * 16;
      *reinterpret_cast<u4v*>((int8_t*)g.h + (t.p0 + row) * g.ldf + n0 + c) = *reinterpret_cast<const u4v*>(line + row * LD + c);
    }
  } else if constexpr (MODE == UP) {
    using U = Turned<NI / 2>;
    const int n = n0 + w0 / 2 * 16 + 4 * (lane % U::L);
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      U ga, up;
      turn_rows<NI / 2>([&](int i) { return acc[2 * i][j]; }, mine, ga);
      turn_rows<NI / 2>([&](int i) { return acc[2 * i + 1][j]; }, mine, up);
#pragma unroll
      for (int s = 0; s < U::S; ++s) {
        const int row = 16 * (x0 + j) + s * U::R + lane / U::L;
        f4 h;
#pragma unroll
        for (int v = 0; v < 4; ++v) h[v] = ga.v[s][v] * sigmoid(ga.v[s][v]) * up.v[s][v];
        // columns past the last have sums of zero
        if constexpr (KIND == F32) raise(g.hmost + t.p0 + row, most4(h), U::L, row < t.rows);
        if (row >= t.rows || n >= g.ldf) continue;
        if (g.a) {
          float* a = g.a + (t.p0 + row) * 2 * g.ldf + n;
          st4(a, ga.v[s]);
          st4(a + g.ldf, up.v[s]);
        }
        store4((T*)g.h + (t.p0 + row) * g.ldf + n, h, 4);
      }
    }
  } else if constexpr (MODE == DH) {
    using U = Turned<NI>;
    const int n = n0 + w0 * 16 + 4 * (lane % U::L);
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      U p;
      turn_rows<NI>([&](int i) { return acc[i][j]; }, mine, p);
      f4 ga[U::S], up[U::S];
      float w[U::S];
#pragma unroll
      for (int s = 0; s < U::S; ++s) {                     // rows and columns past the tile: the last ones, not stored
        const int row = min(16 * (x0 + j) + s * U::R + lane / U::L, t.rows - 1);
        const float* a = g.a + (t.p0 + row) * 2 * g.ldf + min(n, g.ldf - 4);
        ga[s] = ld4(a);
        up[s] = ld4(a + g.ldf);
        w[s] = g.weight[t.slots[row]];
      }
#pragma unroll
      for (int s = 0; s < U::S; ++s) {
        const int row = 16 * (x0 + j) + s * U::R + lane / U::L;
        const bool in = row < t.rows && n < g.ldf;
        f4 dg, du, hw;
        float part = 0.f;
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const float sg = sigmoid(ga[s][v]), act = ga[s][v] * sg, h = act * up[s][v];
          const float pv = n + v < g.F ? p.v[s][v] : 0.f, dh = pv * w[s];
          part += h * pv;
          hw[v] = h * w[s];
          du[v] = dh * act;
          dg[v] = dh * up[s][v] * (sg * (1.f + ga[s][v] * (1.f - sg)));
        }
        if (in) {
          T* d = (T*)g.da + (t.p0 + row) * 2 * g.ldf + n;
          store4(d, dg, 4);
          store4(d + g.ldf, du, 4);
          if (g.hw) store4((T*)g.hw + (t.p0 + row) * g.ldf + n, hw, 4);
        }
        if constexpr (KIND == F32) raise(g.damost + t.p0 + row, in ? max(most4(dg), most4(du)) : 0, U::L, row < t.rows);
        if (g.dwpart) {                                    // the row's sum over the wave's columns
          part = group_sum(in ? part : 0.f, U::L);
          if (lane % U::L == 0) red[wn * BM + row] = part;
        }
      }
    }
    if (g.dwpart) {
      __syncthreads();
      for (int i = threadIdx.x; i < t.rows; i += blockDim.x) {
        float s = red[i];
#pragma unroll
        for (int w = 1; w < WW; ++w) s += red[w * BM + i];
        g.dwpart[(int64_t)ci * g.M + t.p0 + i] = s;
      }
    }
  }
}

}  // namespace experts
}  // namespace fsc
