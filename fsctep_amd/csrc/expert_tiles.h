// Pieces of the tile kernels of the experts' products (expert_mlp.hip).
#pragma once

#include "common.h"
#include "expert_types.h"
#include "expert_args.h"

namespace fsc {
namespace experts {

typedef int i4v __attribute__((ext_vector_type(4)));

enum Kind { F32 = 0, BF16 = 1, I8 = 2 };

// T: the type between the kernels; BK: reduction entries of a step; CE: those of a 16-byte LDS chunk; PL: LDS planes
template <int KIND> struct El;
template <> struct El<F32> { using T = float; static constexpr int BK = 32, CE = 8, PL = 3; };
template <> struct El<BF16> { using T = __bf16; static constexpr int BK = 64, CE = 8, PL = 1; };
template <> struct El<I8> { using T = int8_t; static constexpr int BK = 128, CE = 16, PL = 1; };

template <int KIND> struct Acc { using V = f4; };
template <> struct Acc<I8> { using V = i4v; };

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

// What becomes of a tile's sums.  acc[i][j]: weight tile w0 + i (16 rows of the weight operand), row tile x0 + j; lane
// (r, q) holds the weight rows 4 q .. 4 q + 3 of row r.  n0: the tile's first output column (up: a weight tile pair
// is 16 hidden columns, gate then up).  red: WW * BM floats of LDS that nobody reads any more (dh, 8-bit up), WW waves
// side by side along the weights, this one the wn-th.
template <int KIND, int MODE, int NI, int NJ, int WW, int BM>
__device__ __forceinline__ void finish(const Args& g, const RowTile& t, int n0, int ci, int wn, int w0, int x0,
                                       typename Acc<KIND>::V (&acc)[NI][NJ], float* red) {
  using T = typename El<KIND>::T;
  const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
  if constexpr (MODE == DOWN || MODE == DX) {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int n = n0 + (w0 + i) * 16 + 4 * q;
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const int row = 16 * (x0 + j) + r;
        if constexpr (KIND != I8)
          if (row < t.rows) store4(g.o + (t.p0 + row) * g.ldo + n, acc[i][j], g.H - n);
      }
    }
  } else if constexpr (MODE == UP && KIND == I8) {
    // the block holds whole groups of 128 columns: their largest values, then the codes
    static_assert(WW * NI == 16, "8-bit up: 128 hidden columns a tile");
    f4 h[NI / 2][NJ];
    float top[NJ];
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const int row = 16 * (x0 + j) + r;
      const float xs = g.xscale[t.rws[row]];               // a row past the tile: any row's, not stored
      top[j] = 0.f;
#pragma unroll
      for (int i = 0; i < NI / 2; ++i) {
        const int n = n0 + (w0 / 2 + i) * 16 + 4 * q;
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const float* s = g.in_scale + (int64_t)t.e * 2 * g.F + min(n + v, g.F - 1);
          const float ga = (float)acc[2 * i][j][v] * (xs * s[0]), up = (float)acc[2 * i + 1][j][v] * (xs * s[g.F]);
          h[i][j][v] = ga * sigmoid(ga) * up;              // columns past the last have sums of zero
          top[j] = max_nan(top[j], fabsf(h[i][j][v]));
        }
      }
      top[j] = max_nan(top[j], __shfl_xor(top[j], 16, 64));
      top[j] = max_nan(top[j], __shfl_xor(top[j], 32, 64));
      if (q == 0) red[wn * BM + row] = top[j];
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const int row = 16 * (x0 + j) + r;
#pragma unroll
      for (int w = 0; w < WW; ++w) top[j] = max_nan(top[j], red[w * BM + row]);
      if (row >= t.rows) continue;
      const float inv = top[j] > 0.f ? 127.f / top[j] : 0.f;
#pragma unroll
      for (int i = 0; i < NI / 2; ++i) {
        const int n = n0 + (w0 / 2 + i) * 16 + 4 * q;
        int8_t b[4];
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const float c = rintf(h[i][j][v] * inv);
          b[v] = c >= -127.f && c <= 127.f ? (int8_t)c : (int8_t)0;
        }
        store_bytes<4>((int8_t*)g.h + (t.p0 + row) * g.ldf + n, b);
      }
      if (wn == 0 && q == 0) g.hscale[(t.p0 + row) * (g.ldf / QG) + n0 / QG] = top[j] / 127.f;
    }
  } else if constexpr (MODE == UP) {
#pragma unroll
    for (int i = 0; i < NI / 2; ++i) {
      const int n = n0 + (w0 / 2 + i) * 16 + 4 * q;
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const int row = 16 * (x0 + j) + r;
        if (row >= t.rows || n >= g.ldf) continue;
        const f4 ga = acc[2 * i][j], up = acc[2 * i + 1][j];
        f4 h;
#pragma unroll
        for (int v = 0; v < 4; ++v) h[v] = ga[v] * sigmoid(ga[v]) * up[v];
        if (g.a) {
          float* a = g.a + (t.p0 + row) * 2 * g.ldf + n;
          st4(a, ga);
          st4(a + g.ldf, up);
        }
        store4((T*)g.h + (t.p0 + row) * g.ldf + n, h, 4);
      }
    }
  } else if constexpr (MODE == DH) {
    float part[NJ];
#pragma unroll
    for (int j = 0; j < NJ; ++j) part[j] = 0.f;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int n = n0 + (w0 + i) * 16 + 4 * q;
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const int row = 16 * (x0 + j) + r;
        if (row >= t.rows || n >= g.ldf) continue;
        const float w = g.weight[t.slots[row]];
        const float* a = g.a + (t.p0 + row) * 2 * g.ldf + n;
        const f4 ga = ld4(a), up = ld4(a + g.ldf);
        f4 dg, du, hw;
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const float s = sigmoid(ga[v]), act = ga[v] * s, h = act * up[v], p = acc[i][j][v], dh = p * w;
          part[j] += h * p;
          hw[v] = h * w;
          du[v] = dh * act;
          dg[v] = dh * up[v] * (s * (1.f + ga[v] * (1.f - s)));
        }
        T* d = (T*)g.da + (t.p0 + row) * 2 * g.ldf + n;
        store4(d, dg, 4);
        store4(d + g.ldf, du, 4);
        if (g.hw) store4((T*)g.hw + (t.p0 + row) * g.ldf + n, hw, 4);
      }
    }
    if (g.dwpart) {
      // rows' sums over this tile's columns: the four lanes of a row, then the waves along the columns
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        part[j] += __shfl_xor(part[j], 16, 64);
        part[j] += __shfl_xor(part[j], 32, 64);
        if (q == 0) red[wn * BM + 16 * (x0 + j) + r] = part[j];
      }
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
