// Products of the expert readout.  For the rows by expert (expert_plan.hip), expert e's rows x:
//   up      a = W_in[e] x (gate and up halves), h = silu(a_gate) a_up
//   down    o = W_out[e] h;  y_t = sum_j weight_tj o_tj                       (combine_kernel, fixed order)
//   dh      p = W_out[e]^T dy; dweight = h . p; dh = weight p; da_up = dh silu(a_gate), da_gate = dh a_up silu'(a_gate)
//   dx      W_in[e]^T da, summed over a row's experts                          (combine_kernel)
//   dw_in   sum over rows of da x^T;  dw_out  sum over rows of dy (weight h)^T
// All are products over tiles of 128 x (32, 64 or 128) entries on the matrix cores, 32-bit accumulators:
//   bf16 rows: v_mfma_f32_16x16x32_bf16;  fp32 rows: three bf16 parts an operand and six such products (split3,
//   mfma_x6: as accurate as fp32 at any scale);  8-bit rows: v_mfma_i32_16x16x64_i8.
// The weights are the MFMA's A operand, the rows its B operand: a lane's four results are four neighbouring
// columns of one row, stored by one access.
//
// Rounding of what is held between the kernels: bf16 rows hold h, da and weight h in bf16 (each output passes one
// such rounding and its own), or in fp32 where an expert has few rows; a, p and o stay in fp32.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "common.h"
#include "expert_types.h"
#include "expert_args.h"
#include "expert_plan.h"
#include "fsctep.h"

namespace fsc {
namespace experts {

typedef int i4v __attribute__((ext_vector_type(4)));

enum Kind { F32 = 0, BF16 = 1, I8 = 2 };

constexpr int NT = 256;          // four waves, two by two
constexpr int BN = 128;          // rows of the tile's weight operand

template <int KIND> struct El;
template <> struct El<F32> { using T = float; static constexpr int BK = 32, CE = 8, PL = 3; };
template <> struct El<BF16> { using T = __bf16; static constexpr int BK = 64, CE = 8, PL = 1; };
template <> struct El<I8> { using T = int8_t; static constexpr int BK = 128, CE = 16, PL = 1; };

// ---------------------------------------------------------------- tiles of the operands
// A chunk is 16 bytes of an LDS plane: 8 values (16 in 8 bits) along the row.  Straight operands (rows of the tile
// = rows of memory) lie as [row][chunk], the chunk's place XORed with the row so that 16 lanes reading one chunk
// column of 16 rows meet no bank twice; turned operands (rows of memory along K) lie as [k][column] with 16
// columns of padding and are read by ds_read_b64_tr_b16.
constexpr int TRP = BN + 16;

template <int KIND, int ROWS, bool TR, typename T>
struct Tile {                                                        // T: the type in memory
  using E = El<KIND>;
  static constexpr int CPR = E::BK / E::CE;                          // chunks of a straight row
  static constexpr int NCH = TR ? E::BK * ROWS / 8 : ROWS * CPR;     // chunks of the tile
  static constexpr int PER = (NCH + NT - 1) / NT;                    // chunks of a thread
  static constexpr int PLANE = TR ? E::BK * TRP * 2 : ROWS * CPR * 16;   // bytes
  static constexpr int BYTES = PLANE * E::PL;

  static constexpr int NV = E::CE * sizeof(T) / 16;                  // 16-byte parts of a chunk in memory

  struct Reg { u4v v[NV]; };
  Reg reg[PER];

  __device__ static constexpr int row_of(int c) { return TR ? c / (ROWS / 8) : c / CPR; }
  __device__ static constexpr int chunk_of(int c) { return TR ? c % (ROWS / 8) : c % CPR; }
  __device__ static constexpr int swz(int row) { return CPR == 4 ? (row >> 1) & 3 : row & 7; }

  // chunk c of the thread from p (n values of it exist, the rest are zeros; VEC: all or none, aligned)
  template <bool VEC>
  __device__ __forceinline__ void fetch(int c, const T* p, int n) {
    Reg& g = reg[c];
    if (VEC) {
      const bool in = n > 0;
      const u4v* q = reinterpret_cast<const u4v*>(p);
#pragma unroll
      for (int i = 0; i < NV; ++i) g.v[i] = in ? q[i] : u4v{0, 0, 0, 0};
    } else {
      alignas(16) T t[E::CE];
#pragma unroll
      for (int i = 0; i < E::CE; ++i) t[i] = i < n ? p[i] : (T)0;
      __builtin_memcpy(&g, t, sizeof(t));
    }
  }
  // the thread's chunks into LDS
  __device__ __forceinline__ void put(char* lds) const {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int c = threadIdx.x + i * NT;
      if (NCH % NT && c >= NCH) break;
      const int row = row_of(c), kc = chunk_of(c);
      const int at = TR ? row * TRP * 2 + kc * 16 : (row * CPR + (kc ^ swz(row))) * 16;
      if constexpr (KIND == F32) {
        bf8 h, m, l;
        if constexpr (sizeof(T) == 4) {
          float v[8];
          __builtin_memcpy(v, &reg[i], 32);
          split3(v, h, m, l);
        } else {                                                     // a bf16 value is its own first part
          h = __builtin_bit_cast(bf8, reg[i].v[0]);
          m = l = __builtin_bit_cast(bf8, u4v{0, 0, 0, 0});
        }
        *reinterpret_cast<bf8*>(lds + at) = h;
        *reinterpret_cast<bf8*>(lds + PLANE + at) = m;
        *reinterpret_cast<bf8*>(lds + 2 * PLANE + at) = l;
      } else {
        *reinterpret_cast<u4v*>(lds + at) = reg[i].v[0];
      }
    }
  }
  // lane (r, q)'s part of the MFMA operand: tile row 16 t + r, chunk 4 ks + q of the K step
  __device__ __forceinline__ static u4v frag(const char* lds, int plane, int t, int ks) {
    const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
    if constexpr (TR) {
      typedef short s4 __attribute__((__vector_size__(8)));
      typedef __attribute__((address_space(3))) s4* lp;
      const char* p = lds + plane * PLANE + ((32 * ks + 8 * q + (r >> 2)) * TRP + 16 * t + 4 * (r & 3)) * 2;
      const u2v lo = __builtin_bit_cast(u2v, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(const_cast<char*>(p))));
      const u2v hi = __builtin_bit_cast(u2v, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(const_cast<char*>(p + 4 * TRP * 2))));
      return u4v{lo.x, lo.y, hi.x, hi.y};
    } else {
      const int row = 16 * t + r;
      return *reinterpret_cast<const u4v*>(lds + plane * PLANE + (row * CPR + ((4 * ks + q) ^ swz(row))) * 16);
    }
  }
};

template <int KIND> struct Acc { using V = f4; };
template <> struct Acc<I8> { using V = i4v; };

// acc[i][j] += (weight tiles w0 + i) (row tiles x0 + j) over one K step in LDS.
template <int KIND, int NI, int NJ, typename TW, typename TX>
__device__ __forceinline__ void step(const char* lw, const char* lx, int w0, int x0,
                                     typename Acc<KIND>::V (&acc)[NI][NJ]) {
  using E = El<KIND>;
  constexpr int KS = E::BK / (4 * E::CE);
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    u4v x[NJ][E::PL];
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int p = 0; p < E::PL; ++p) x[j][p] = TX::frag(lx, p, x0 + j, ks);
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      u4v w[E::PL];
#pragma unroll
      for (int p = 0; p < E::PL; ++p) w[p] = TW::frag(lw, p, w0 + i, ks);
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        if constexpr (KIND == F32)
          acc[i][j] = mfma_x6(__builtin_bit_cast(bf8, w[0]), __builtin_bit_cast(bf8, w[1]),
                              __builtin_bit_cast(bf8, w[2]), __builtin_bit_cast(bf8, x[j][0]),
                              __builtin_bit_cast(bf8, x[j][1]), __builtin_bit_cast(bf8, x[j][2]), acc[i][j]);
        else if constexpr (KIND == BF16)
          acc[i][j] = mfma_bf16(__builtin_bit_cast(bf8, w[0]), __builtin_bit_cast(bf8, x[j][0]), acc[i][j]);
        else
          acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i4v, w[0]),
                                                            __builtin_bit_cast(i4v, x[j][0]), acc[i][j], 0, 0, 0);
      }
    }
  }
}

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

// ---------------------------------------------------------------- the products by row tiles
// up: 64 hidden columns a tile, their gate and up rows in turn by 16, so that a wave holds both of a column.
template <int KIND, typename S, int MODE, int NJ, bool VEC>
__global__ __launch_bounds__(NT) void rows_kernel(Args g) {
  using E = El<KIND>;
  using T = typename E::T;                                   // of the arrays between the kernels; S: the caller's
  using R = std::conditional_t<MODE == DOWN || MODE == DX, T, S>;
  constexpr int BM = 32 * NJ;
  constexpr bool TR = MODE == DH || MODE == DX;
  using TW = Tile<KIND, BN, TR, S>;
  using TX = Tile<KIND, BM, false, R>;
  __shared__ __align__(16) char lds[TW::BYTES + TX::BYTES];
  __shared__ int32_t slots[BM], rws[BM];
  char* lw = lds;
  char* lx = lds + TW::BYTES;

  const int NC = MODE == UP ? 64 : BN;                       // output columns of a tile
  // output columns (8 bits: the last group of h is whole)
  const int cols = KIND == I8 && MODE == UP ? g.ldf : MODE == UP || MODE == DH ? g.F : g.H;
  const int K = MODE == UP || MODE == DH ? g.H : MODE == DOWN ? g.F : 2 * g.ldf;
  int ti, ci;
  if (!tile_of(g.n_tiles, (cols + NC - 1) / NC, ti, ci)) return;
  const int e = g.tiles[2 * ti];
  if (e < 0) return;
  const int64_t p0 = g.tiles[2 * ti + 1];                    // first sorted position
  const int64_t left = g.offsets[e + 1] - p0;
  const int rows = left < BM ? (int)left : BM;
  const int n0 = ci * NC;
  for (int i = threadIdx.x; i < BM; i += NT) {
    slots[i] = i < rows ? g.slot_of[p0 + i] : -1;
    rws[i] = i < rows ? g.row_of[p0 + i] : 0;
  }
  __syncthreads();

  // row pointers of this thread's chunks (straight operands); null where there is none
  const R* xp[TX::PER];
#pragma unroll
  for (int i = 0; i < TX::PER; ++i) {
    const int c = threadIdx.x + i * NT, row = TX::row_of(c);
    xp[i] = nullptr;
    if (c < TX::NCH && row < rows) {
      if (MODE == UP) xp[i] = (const R*)g.x + (int64_t)rws[row] * g.xs;
      if (MODE == DH) xp[i] = (const R*)g.dy + (int64_t)rws[row] * g.ds;
      if (MODE == DOWN) xp[i] = (const R*)g.h + (p0 + row) * g.ldf;
      if (MODE == DX) xp[i] = (const R*)g.da + (p0 + row) * 2 * g.ldf;
    }
  }
  const S* wp[TW::PER];
  if (!TR) {
#pragma unroll
    for (int i = 0; i < TW::PER; ++i) {
      const int row = TW::row_of(threadIdx.x + i * NT);
      if (MODE == UP) {
        const int n = n0 + (row >> 5) * 16 + (row & 15);
        wp[i] = n < g.F ? (const S*)g.w_in + ((int64_t)e * 2 * g.F + (row & 16 ? g.F : 0) + n) * g.H : nullptr;
      } else {
        const int n = n0 + row;
        wp[i] = n < g.H ? (const S*)g.w_out + ((int64_t)e * g.H + n) * g.F : nullptr;
      }
    }
  }
  TW tw;
  TX tx;
  // the arrays between the kernels are padded with zeros to ldf, a multiple of a chunk
  const int KX = MODE == DOWN ? g.ldf : K;
  auto fetch = [&](int k0) {
#pragma unroll
    for (int i = 0; i < TX::PER; ++i) {
      const int k = k0 + TX::chunk_of(threadIdx.x + i * NT) * E::CE;
      tx.template fetch<VEC>(i, xp[i] + k, xp[i] ? KX - k : 0);
    }
#pragma unroll
    for (int i = 0; i < TW::PER; ++i) {
      const int c = threadIdx.x + i * NT;
      if (!TR) {
        const int k = k0 + TW::chunk_of(c) * E::CE;
        tw.template fetch<VEC>(i, wp[i] + k, wp[i] ? K - k : 0);
      } else {
        const int k = k0 + TW::row_of(c), n = n0 + TW::chunk_of(c) * 8;
        const S* p = nullptr;
        if (MODE == DH) {
          if (k < g.H) p = (const S*)g.w_out + ((int64_t)e * g.H + k) * g.F + n;
        } else {
          const int half = k >= g.ldf, f = k - half * g.ldf;
          if (k < K && f < g.F) p = (const S*)g.w_in + ((int64_t)e * 2 * g.F + half * g.F + f) * g.H + n;
        }
        tw.template fetch<VEC>(i, p, p ? cols - n : 0);
      }
    }
  };

  typename Acc<KIND>::V acc[4][NJ];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j) acc[i][j] = {0, 0, 0, 0};
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
  const int w0 = (wave & 1) * 4, x0 = (wave >> 1) * NJ;      // first tiles of the wave

  if constexpr (KIND == I8 && MODE == DOWN) {
    // a K step is one group of h: its sums are whole numbers, scaled by the group's unit into 32-bit floats
    f4 sum[4][NJ];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < NJ; ++j) sum[i][j] = f4{0.f, 0.f, 0.f, 0.f};
    const int ng = g.ldf / QG;
    fetch(0);
    for (int k0 = 0; k0 < K; k0 += E::BK) {
      __syncthreads();
      tw.put(lw);
      tx.put(lx);
      __syncthreads();
      if (k0 + E::BK < K) fetch(k0 + E::BK);
      float u[NJ];
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const int row = 16 * (x0 + j) + r;
        u[j] = row < rows ? g.hscale[(p0 + row) * ng + k0 / QG] : 0.f;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j) acc[i][j] = {0, 0, 0, 0};
      step<KIND, 4, NJ, TW, TX>(lw, lx, w0, x0, acc);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
          for (int v = 0; v < 4; ++v) sum[i][j][v] += (float)acc[i][j][v] * u[j];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int n = n0 + (w0 + i) * 16 + 4 * q;
      f4 sc;
#pragma unroll
      for (int v = 0; v < 4; ++v) sc[v] = n + v < g.H ? g.out_scale[(int64_t)e * g.H + n + v] : 0.f;
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const int row = 16 * (x0 + j) + r;
        if (row < rows) store4(g.o + (p0 + row) * g.ldo + n, sum[i][j] * sc, g.H - n);
      }
    }
    return;
  } else {
    fetch(0);
    for (int k0 = 0; k0 < K; k0 += E::BK) {
      __syncthreads();
      tw.put(lw);
      tx.put(lx);
      __syncthreads();
      if (k0 + E::BK < K) fetch(k0 + E::BK);
      step<KIND, 4, NJ, TW, TX>(lw, lx, w0, x0, acc);
    }
  }

  if constexpr (MODE == DOWN || MODE == DX) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int n = n0 + (w0 + i) * 16 + 4 * q;
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const int row = 16 * (x0 + j) + r;
        if constexpr (KIND != I8)
          if (row < rows) store4(g.o + (p0 + row) * g.ldo + n, acc[i][j], g.H - n);
      }
    }
  } else if constexpr (MODE == UP) {
    f4 hv[2][NJ];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int n = n0 + ((wave & 1) * 2 + i) * 16 + 4 * q;
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const int row = 16 * (x0 + j) + r;
        f4 ga, up;
        if constexpr (KIND == I8) {
          const float xs = row < rows ? g.xscale[rws[row]] : 0.f;
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            const float* s = g.in_scale + (int64_t)e * 2 * g.F + n + v;
            ga[v] = n + v < g.F ? (float)acc[2 * i][j][v] * (xs * s[0]) : 0.f;
            up[v] = n + v < g.F ? (float)acc[2 * i + 1][j][v] * (xs * s[g.F]) : 0.f;
          }
        } else {
          ga = acc[2 * i][j];
          up = acc[2 * i + 1][j];
        }
#pragma unroll
        for (int v = 0; v < 4; ++v) hv[i][j][v] = ga[v] * sigmoid(ga[v]) * up[v];
        if constexpr (KIND != I8) {
          if (row < rows && n < g.ldf) {
            if (g.a) {
              float* a = g.a + (p0 + row) * 2 * g.ldf + n;
              st4(a, ga);
              st4(a + g.ldf, up);
            }
            store4((T*)g.h + (p0 + row) * g.ldf + n, hv[i][j], 4);
          }
        }
      }
    }
    if constexpr (KIND == I8) {
      // the block holds half a group of 128 columns: h goes out in 32 bits, quant_kernel makes the codes
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int n = n0 + ((wave & 1) * 2 + i) * 16 + 4 * q;
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          const int row = 16 * (x0 + j) + r;
          if (row < rows && n < g.ldf) st4(g.a + (p0 + row) * g.ldf + n, hv[i][j]);
        }
      }
    }
  } else if constexpr (MODE == DH) {
    float part[NJ];
#pragma unroll
    for (int j = 0; j < NJ; ++j) part[j] = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int n = n0 + (w0 + i) * 16 + 4 * q;
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const int row = 16 * (x0 + j) + r;
        if (row >= rows || n >= g.ldf) continue;
        const float w = g.weight[slots[row]];
        const float* a = g.a + (p0 + row) * 2 * g.ldf + n;
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
        T* d = (T*)g.da + (p0 + row) * 2 * g.ldf + n;
        store4(d, dg, 4);
        store4(d + g.ldf, du, 4);
        if (g.hw) store4((T*)g.hw + (p0 + row) * g.ldf + n, hw, 4);
      }
    }
    if (g.dwpart) {
      // rows' sums over this tile's columns: the four lanes of a row, then the two waves of the columns
      __syncthreads();
      float* red = reinterpret_cast<float*>(lds);
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        part[j] += __shfl_xor(part[j], 16, 64);
        part[j] += __shfl_xor(part[j], 32, 64);
        if (q == 0) red[(wave & 1) * BM + 16 * (x0 + j) + r] = part[j];
      }
      __syncthreads();
      for (int i = threadIdx.x; i < rows; i += NT) g.dwpart[(int64_t)ci * g.M + p0 + i] = red[i] + red[BM + i];
    }
  }
}

// ---------------------------------------------------------------- weight gradients
// dw_in[e][m][n] = sum over expert e's positions of da[.][m] x[.][n]; dw_out[e][m][n] = that of dy[.][m] hw[.][n].
// The matrix of the contiguous output index n is the MFMA's A operand; both are turned.
// FEW: h's arrays lie by slot and the block finds the expert's slots itself.
template <int KIND, typename S, int MODE, bool VEC, bool FEW>
__global__ __launch_bounds__(NT) void weights_kernel(Args g) {
  using E = El<KIND>;
  using T = typename E::T;
  using RA = std::conditional_t<MODE == DWIN, S, T>;
  using RB = std::conditional_t<MODE == DWIN, T, S>;
  using TT = Tile<KIND, BN, true, RA>;
  using TB = Tile<KIND, BN, true, RB>;
  __shared__ __align__(16) char lds[2 * TT::BYTES];
  char* la = lds;
  char* lb = lds + TT::BYTES;
  const int na = MODE == DWIN ? g.H : g.ldf, nb = MODE == DWIN ? 2 * g.ldf : g.H;   // columns of the operands
  const int ta = (na + BN - 1) / BN, tb = (nb + BN - 1) / BN;
  int e, c;
  if (!tile_of(g.E, ta * tb, e, c)) return;
  const int b0 = (c / ta) * BN, a0 = (c % ta) * BN;
  __shared__ int16_t list[FEW ? FEW_SLOTS : 1];
  int64_t p0 = 0, cnt;
  if constexpr (FEW) {
    cnt = few_slots(g, e, few_first(g), list);
    __syncthreads();
  } else {
    p0 = g.offsets[e];
    cnt = g.offsets[e + 1] - p0;
  }
  TT A;
  TB B;
  // rows of x or dy of a step's positions, loaded a step ahead of the rows themselves
  int tok[TT::PER];
  auto find = [&](int64_t k0) {
#pragma unroll
    for (int i = 0; i < TT::PER; ++i) {
      const int64_t k = k0 + TT::row_of(threadIdx.x + i * NT);
      if constexpr (FEW) tok[i] = k < cnt ? (int)few_row(g, list[k]) : 0;
      else tok[i] = g.row_of[p0 + (k < cnt ? k : cnt - 1)];
    }
  };
  auto fetch = [&](int64_t k0) {
#pragma unroll
    for (int i = 0; i < TT::PER; ++i) {
      const int cc = threadIdx.x + i * NT;
      const int64_t k = k0 + TT::row_of(cc);
      const int n = TT::chunk_of(cc) * 8;
      const RA* pa = nullptr;
      const RB* pb = nullptr;
      if (k < cnt) {
        const int64_t pos = FEW ? list[k] : p0 + k;
        if (MODE == DWIN) {
          pa = (const RA*)g.x + (int64_t)tok[i] * g.xs + a0 + n;
          pb = (const RB*)g.da + pos * 2 * g.ldf + b0 + n;
        } else {
          pa = (const RA*)g.hw + pos * g.ldf + a0 + n;
          pb = (const RB*)g.dy + (int64_t)tok[i] * g.ds + b0 + n;
        }
      }
      A.template fetch<VEC>(i, pa, pa ? na - a0 - n : 0);
      B.template fetch<VEC>(i, pb, pb ? nb - b0 - n : 0);
    }
  };
  f4 acc[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = f4{0.f, 0.f, 0.f, 0.f};
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
  const int w0 = (wave & 1) * 4, x0 = (wave >> 1) * 4;
  if (cnt > 0) {
    find(0);
    fetch(0);
    find(E::BK);
  }
  for (int64_t k0 = 0; k0 < cnt; k0 += E::BK) {
    __syncthreads();
    A.put(la);
    B.put(lb);
    __syncthreads();
    if (k0 + E::BK < cnt) {
      fetch(k0 + E::BK);
      find(k0 + 2 * E::BK);
    }
    step<KIND, 4, 4, TT, TB>(la, lb, w0, x0, acc);
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    int m = b0 + (x0 + j) * 16 + r;
    int64_t out = -1;
    if (MODE == DWIN) {
      const int half = m >= g.ldf, f = m - half * g.ldf;
      if (m < nb && f < g.F) out = ((int64_t)e * 2 * g.F + half * g.F + f) * g.H;
    } else if (m < g.H) {
      out = ((int64_t)e * g.H + m) * g.F;
    }
    if (out < 0) continue;
    const int len = MODE == DWIN ? g.H : g.F;
    S* dw = (S*)(MODE == DWIN ? g.dw_in : g.dw_out) + out;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int n = a0 + (w0 + i) * 16 + 4 * q;
      if (n < len) store4(dw + n, acc[i][j], len - n);
    }
  }
}

// ---------------------------------------------------------------- rows from their experts, in slot order
// The row of a slot in the arrays between the kernels, -1 for a slot with no expert.
__device__ __forceinline__ int place_of(const int32_t* place, const int32_t* index, int E, int64_t s) {
  if (place) return place[s];
  const int e = index[s];
  return e >= 0 && e < E ? (int)s : -1;
}

template <typename T>
__global__ __launch_bounds__(NT) void combine_kernel(int64_t rows, int H, int ldo, int k,
                                                     const int32_t* __restrict__ place,
                                                     const int32_t* __restrict__ index, int E,
                                                     const float* __restrict__ weight, const float* __restrict__ o,
                                                     T* __restrict__ y) {
  const int nv = (H + 3) / 4;
  const int64_t n = rows * nv;
  for (int64_t i = (int64_t)blockIdx.x * NT + threadIdx.x; i < n; i += (int64_t)gridDim.x * NT) {
    const int64_t t = i / nv;
    const int c = (int)(i - t * nv) * 4;
    f4 s = {0.f, 0.f, 0.f, 0.f};
    for (int j = 0; j < k; ++j) {
      const int p = place_of(place, index, E, t * k + j);
      if (p < 0) continue;
      const float w = weight ? weight[t * k + j] : 1.f;
      s += w * ld4(o + (int64_t)p * ldo + c);
    }
    store4(y + t * H + c, s, H - c);
  }
}

// dweight by slot: the partial sums over the column tiles, in order; 0 for a slot with no expert.
__global__ __launch_bounds__(NT) void dweight_kernel(int64_t M, int parts, const int32_t* __restrict__ place,
                                                     const int32_t* __restrict__ index, int E, const float* __restrict__ part, float* __restrict__ dweight) {
  const int64_t s = (int64_t)blockIdx.x * NT + threadIdx.x;
  if (s >= M) return;
  const int p = place_of(place, index, E, s);
  float t = 0.f;
  if (p >= 0)
    for (int i = 0; i < parts; ++i) t += part[(int64_t)i * M + p];
  dweight[s] = t;
}

// 8 bits: codes and units of h by groups of 128 columns; a wave a group, two columns a lane.
__global__ __launch_bounds__(NT) void quant_kernel(Args g) {
  const int ng = g.ldf / QG;
  const int64_t i = (int64_t)blockIdx.x * (NT / 64) + (threadIdx.x >> 6);
  if (i >= (int64_t)g.offsets[g.E] * ng) return;
  const int64_t p = i / ng;
  const int grp = (int)(i - p * ng), lane = threadIdx.x & 63;
  const float* h = g.a + p * g.ldf + grp * QG + 2 * lane;
  const float v0 = h[0], v1 = h[1];
  float top = max_nan(fabsf(v0), fabsf(v1));
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) top = max_nan(top, __shfl_xor(top, off, 64));
  const float inv = top > 0.f ? 127.f / top : 0.f;
  auto code = [&](float v) {
    const float c = rintf(v * inv);
    return c >= -127.f && c <= 127.f ? (int)c : 0;
  };
  *(uint16_t*)((int8_t*)g.h + p * g.ldf + grp * QG + 2 * lane) =
      (uint16_t)((code(v0) & 0xff) | (code(v1) & 0xff) << 8);
  if (lane == 0) g.hscale[i] = top / 127.f;
}

// ---------------------------------------------------------------- host
inline int up8(int v) { return (v + 7) / 8 * 8; }
inline int64_t align64(int64_t b) { return (b + 63) / 64 * 64; }

// Few rows: at most 16 for each expert on average, and few enough slots for a block to look through.  The few-rows
// kernels read an expert's weights once for 16 rows, the tiles once for up to 128.
inline bool few(int64_t M, int E) { return M <= FEW_SLOTS && M <= 16 * (int64_t)E; }

// Rows of a tile by the rows that an expert has on average: the weights are read once for each tile of an expert,
// and rows that a tile lacks are still computed.
inline int tile_rows(int64_t M, int E) {
  const int64_t avg = M / std::max(1, E);
  return avg > 64 ? 128 : avg > 32 ? 64 : 32;
}

inline bool vec_ok(const void* p, int64_t stride, int size, int n) {
  return !p || ((uintptr_t)p % 16 == 0 && (stride * size) % 16 == 0 && n % (size == 1 ? 16 : 8) == 0);
}

template <int KIND, typename S, int MODE>
void launch_rows(const Args& g, int tile, bool vec, hipStream_t st) {
  const int NC = MODE == UP ? 64 : BN;
  const int cols = KIND == I8 && MODE == UP ? g.ldf : MODE == UP || MODE == DH ? g.F : g.H;
  const unsigned grid = tile_grid(g.n_tiles, (cols + NC - 1) / NC);
  auto go = [&](auto NJ) {
    constexpr int nj = decltype(NJ)::value;
    if (vec) rows_kernel<KIND, S, MODE, nj, true><<<grid, NT, 0, st>>>(g);
    else rows_kernel<KIND, S, MODE, nj, false><<<grid, NT, 0, st>>>(g);
  };
  if (tile == 128) go(std::integral_constant<int, 4>{});
  else if (tile == 64) go(std::integral_constant<int, 2>{});
  else go(std::integral_constant<int, 1>{});
}

template <int KIND, typename S, int MODE, bool FEW = false>
void launch_weights(const Args& g, bool vec, hipStream_t st) {
  const int64_t na = MODE == DWIN ? g.H : g.ldf, nb = MODE == DWIN ? 2 * g.ldf : g.H;
  const unsigned grid = tile_grid(g.E, ((na + BN - 1) / BN) * ((nb + BN - 1) / BN));
  if (vec) weights_kernel<KIND, S, MODE, true, FEW><<<grid, NT, 0, st>>>(g);
  else weights_kernel<KIND, S, MODE, false, FEW><<<grid, NT, 0, st>>>(g);
}

template <typename T>
void launch_combine(const Args& g, const float* weight, T* y, hipStream_t st) {
  const int64_t n = g.T * ((g.H + 3) / 4);
  const unsigned grid = (unsigned)std::min<int64_t>((n + NT - 1) / NT, 1 << 20);
  combine_kernel<T><<<grid, NT, 0, st>>>(g.T, g.H, g.ldo, g.k, g.place, g.index, g.E, weight, g.o, y);
}

int check_dims(const FscExpertDims* d, bool q8) {
  FSC_CHECK_ARG(d != nullptr, "expert_mlp: null dims");
  FSC_CHECK_ARG(d->rows >= 0 && d->rows < (1ll << 31), "expert_mlp: rows must be below 2^31");
  FSC_CHECK_ARG(d->n_experts >= 1 && d->n_experts <= MAX_EXPERTS, "expert_mlp: 1 to 512 experts");
  FSC_CHECK_ARG(d->k >= 1 && d->k <= 64 && d->rows * d->k < (1ll << 31), "expert_mlp: 1 to 64 slots a row, fewer than 2^31 in all");
  FSC_CHECK_ARG(d->width >= 1 && d->width <= (1 << 20) && d->hidden >= 1 && d->hidden <= (1 << 20),
                "expert_mlp: width and hidden must be 1 to 2^20");
  if (q8) FSC_CHECK_ARG(d->dtype == FSC_I8, "expert_mlp_q8: rows and weights are int8");
  else FSC_CHECK_ARG(d->dtype == FSC_F32 || d->dtype == FSC_BF16, "expert_mlp: rows are float32 or bfloat16");
  return 0;
}

inline int ldf_of(const FscExpertDims& d) {
  return d.dtype == FSC_I8 ? (d.hidden + QG - 1) / QG * QG : up8(d.hidden);
}
inline int ldo_of(const FscExpertDims& d) { return (d.width + 3) / 4 * 4; }

// bf16 rows, few for each expert: the products wait for the weights from memory, so what is held between the
// kernels stays in fp32 and the products run as those of fp32 rows do.
inline bool fine(const FscExpertDims& d) {
  const int64_t M = d.rows * d.k;
  return d.dtype == FSC_BF16 && (few(M, d.n_experts) || tile_rows(M, d.n_experts) == 32);
}
// bytes of a value of the arrays between the kernels
inline int64_t held_size(const FscExpertDims& d) { return d.dtype == FSC_I8 ? 1 : d.dtype == FSC_F32 || fine(d) ? 4 : 2; }

// Parts of a workspace, in bytes.
struct Space {
  int64_t h, o, da, hw, part, hs, total;
};
inline Space forward_space(const FscExpertDims& d) {
  const int64_t M = d.rows * d.k, ldf = ldf_of(d), size = held_size(d);
  Space s{};
  int64_t at = 0;
  s.h = at; at += align64(M * ldf * size);
  s.o = at; at += align64(M * ldo_of(d) * 4);
  if (d.dtype == FSC_I8) {
    s.da = at; at += align64(M * ldf * 4);          // h in 32 bits
    s.hs = at; at += align64(M * (ldf / QG) * 4);
  }
  s.total = at;
  return s;
}
inline Space backward_space(const FscExpertDims& d) {
  const int64_t M = d.rows * d.k, ldf = ldf_of(d), size = held_size(d);
  Space s{};
  int64_t at = 0;
  s.o = at; at += align64(M * ldo_of(d) * 4);
  s.da = at; at += align64(M * 2 * ldf * size);
  s.hw = at; at += align64(M * ldf * size);
  s.part = at; at += align64(M * ((d.hidden + 31) / 32) * 4);
  s.total = at;
  return s;
}

Args args_of(const FscExpertDims& d, const Plan& p) {
  Args g{};
  g.T = d.rows;
  g.M = d.rows * d.k;
  g.H = d.width;
  g.F = d.hidden;
  g.ldf = ldf_of(d);
  g.ldo = ldo_of(d);
  g.E = d.n_experts;
  g.k = d.k;
  g.k_inv = ((1u << 20) + d.k - 1) / d.k;
  if (!few(g.M, g.E)) {
    g.n_tiles = p.n_tiles;
    g.offsets = p.offsets;
    g.slot_of = p.slot_of;
    g.row_of = p.row_of;
    g.tiles = p.tiles;
    g.place = p.place;
  }
  return g;
}

template <int KIND, typename S>
void forward(Args g, int tile, void* y, hipStream_t st) {
  const bool vin = vec_ok(g.x, g.xs, sizeof(S), g.H) && vec_ok(g.w_in, g.H, sizeof(S), g.H);
  const bool vout = vec_ok(g.w_out, g.F, sizeof(S), g.F);
  if (!g.place) {
    if constexpr (KIND == I8) {
      few_launch_q8(g, vin, vout, st);
    } else {
      few_launch<S>(UP, g, vin, st);
      few_launch<S>(DOWN, g, vout, st);
    }
  } else {
    launch_rows<KIND, S, UP>(g, tile, vin, st);
    if constexpr (KIND == I8) quant_kernel<<<(unsigned)((g.M * (g.ldf / QG) + 3) / 4), NT, 0, st>>>(g);
    launch_rows<KIND, S, DOWN>(g, tile, vout, st);
  }
  using Y = std::conditional_t<KIND == I8, __bf16, S>;
  launch_combine<Y>(g, g.weight, (Y*)y, st);
}

template <int KIND, typename S>
void backward(Args g, int tile, void* dx, float* dweight, hipStream_t st) {
  const bool vdy = vec_ok(g.dy, g.ds, sizeof(S), g.H), vx = vec_ok(g.x, g.xs, sizeof(S), g.H);
  const bool vin = vec_ok(g.w_in, g.H, sizeof(S), g.H), vout = vec_ok(g.w_out, g.F, sizeof(S), g.F);
  const bool by_slot = !g.place;
  if (by_slot) few_launch<S>(DH, g, vdy && vout, st);
  else launch_rows<KIND, S, DH>(g, tile, vdy && vout, st);
  if (dweight)
    dweight_kernel<<<(unsigned)((g.M + NT - 1) / NT), NT, 0, st>>>(
        g.M, by_slot ? few_parts(g.F, sizeof(S)) : (g.F + BN - 1) / BN, g.place, g.index, g.E, g.dwpart, dweight);
  if (dx) {
    if (by_slot) few_launch<S>(DX, g, vin, st);
    else launch_rows<KIND, S, DX>(g, tile, vin, st);
    launch_combine<S>(g, nullptr, (S*)dx, st);
  }
  if (by_slot) {
    if constexpr (KIND == F32) {
      if (g.dw_in) launch_weights<F32, S, DWIN, true>(g, vx, st);
      if (g.dw_out) launch_weights<F32, S, DWOUT, true>(g, vdy, st);
    }
  } else {
    if (g.dw_in) launch_weights<KIND, S, DWIN>(g, vx, st);
    if (g.dw_out) launch_weights<KIND, S, DWOUT>(g, vdy, st);
  }
}

}  // namespace experts
}  // namespace fsc

extern "C" {

int fsc_expert_sizes(const FscExpertDims* dims, int64_t* plan_ints, int64_t* saved_floats, int64_t* forward_bytes,
                     int64_t* backward_bytes) {
  using namespace fsc::experts;
  if (int rc = check_dims(dims, dims && dims->dtype == FSC_I8)) return rc;
  FSC_CHECK_ARG(plan_ints && saved_floats && forward_bytes && backward_bytes, "expert_sizes: null output");
  const int64_t M = dims->rows * dims->k;
  *plan_ints = few(M, dims->n_experts) ? 0 : fsc::experts::plan_ints(M, dims->n_experts, tile_rows(M, dims->n_experts));
  *saved_floats = dims->dtype == FSC_I8 ? 0 : M * 2 * ldf_of(*dims);
  *forward_bytes = forward_space(*dims).total;
  *backward_bytes = dims->dtype == FSC_I8 ? 0 : backward_space(*dims).total;
  return 0;
}

int fsc_expert_plan(const FscExpertDims* dims, const int32_t* index, int32_t* plan, hipStream_t stream) {
  using namespace fsc::experts;
  if (int rc = check_dims(dims, dims && dims->dtype == FSC_I8)) return rc;
  const int64_t M = dims->rows * dims->k;
  if (few(M, dims->n_experts)) return 0;       // the products find their rows themselves
  FSC_CHECK_ARG(plan && index, "expert_plan: null array");
  const int tile = tile_rows(M, dims->n_experts);
  launch_plan(plan_of(plan, M, dims->n_experts, tile), M, dims->n_experts, dims->k, tile, index, stream);
  return fsc::check_launch("expert_plan") ? 2 : 0;
}

int fsc_expert_mlp_forward(const FscExpertDims* dims, int64_t x_stride, const void* x, const int32_t* index,
                           const int32_t* plan, const float* weight, const void* w_in, const void* w_out, float* saved,
                           void* workspace, void* y, hipStream_t stream) {
  using namespace fsc::experts;
  if (int rc = check_dims(dims, false)) return rc;
  if (dims->rows == 0) return 0;
  const int64_t M = dims->rows * dims->k;
  FSC_CHECK_ARG(x && index && (plan || few(M, dims->n_experts)) && weight && w_in && w_out && workspace && y,
                "expert_mlp_forward: null array");
  FSC_CHECK_ARG(x_stride >= 0, "expert_mlp_forward: negative row stride");
  const int tile = tile_rows(M, dims->n_experts);
  const Plan p = plan_of(const_cast<int32_t*>(plan), M, dims->n_experts, tile);
  Args g = args_of(*dims, p);
  const Space s = forward_space(*dims);
  char* ws = (char*)workspace;
  g.index = index;
  g.x = x; g.xs = x_stride; g.weight = weight; g.w_in = w_in; g.w_out = w_out; g.a = saved;
  g.h = ws + s.h;
  g.o = (float*)(ws + s.o);
  if (dims->dtype == FSC_F32) forward<F32, float>(g, tile, y, stream);
  else if (fine(*dims)) forward<F32, __bf16>(g, tile, y, stream);
  else forward<BF16, __bf16>(g, tile, y, stream);
  return fsc::check_launch("expert_mlp_forward") ? 2 : 0;
}

int fsc_expert_mlp_backward(const FscExpertDims* dims, int64_t x_stride, int64_t dy_stride, const void* dy,
                            const void* x, const int32_t* index, const int32_t* plan, const float* weight,
                            const void* w_in, const void* w_out, const float* saved, void* workspace, void* dx, float* dweight,
                            void* dw_in, void* dw_out, hipStream_t stream) {
  using namespace fsc::experts;
  if (int rc = check_dims(dims, false)) return rc;
  const int64_t M = dims->rows * dims->k;
  FSC_CHECK_ARG((plan || few(M, dims->n_experts)) && w_in && w_out, "expert_mlp_backward: null array");
  FSC_CHECK_ARG(M == 0 || (dy && x && index && weight && saved && workspace), "expert_mlp_backward: null array");
  FSC_CHECK_ARG(x_stride >= 0 && dy_stride >= 0, "expert_mlp_backward: negative row stride");
  const int tile = tile_rows(M, dims->n_experts);
  const Plan p = plan_of(const_cast<int32_t*>(plan), M, dims->n_experts, tile);
  Args g = args_of(*dims, p);
  const Space s = backward_space(*dims);
  char* ws = (char*)workspace;
  g.index = index;
  g.x = x; g.xs = x_stride; g.dy = dy; g.ds = dy_stride; g.weight = weight; g.w_in = w_in; g.w_out = w_out;
  g.a = const_cast<float*>(saved);
  g.o = (float*)(ws + s.o);
  g.da = ws + s.da;
  g.hw = dw_out ? ws + s.hw : nullptr;
  g.dwpart = dweight ? (float*)(ws + s.part) : nullptr;
  g.dw_in = dw_in;
  g.dw_out = dw_out;
  if (M == 0) {              // no rows: zero weight gradients, written by the products' empty sums
    if (dims->dtype == FSC_F32) {
      if (dw_in) launch_weights<F32, float, DWIN, true>(g, false, stream);
      if (dw_out) launch_weights<F32, float, DWOUT, true>(g, false, stream);
    } else {
      if (dw_in) launch_weights<F32, __bf16, DWIN, true>(g, false, stream);
      if (dw_out) launch_weights<F32, __bf16, DWOUT, true>(g, false, stream);
    }
  } else if (dims->dtype == FSC_F32) {
    backward<F32, float>(g, tile, dx, dweight, stream);
  } else if (fine(*dims)) {
    backward<F32, __bf16>(g, tile, dx, dweight, stream);
  } else {
    backward<BF16, __bf16>(g, tile, dx, dweight, stream);
  }
  return fsc::check_launch("expert_mlp_backward") ? 2 : 0;
}

int fsc_expert_mlp_q8(const FscExpertDims* dims, int64_t x_stride, const int8_t* x, const float* x_scale,
                      const int32_t* index, const int32_t* plan, const float* weight, const int8_t* w_in, const float* w_in_scale,
                      const int8_t* w_out, const float* w_out_scale, void* workspace, void* y, hipStream_t stream) {
  using namespace fsc::experts;
  if (int rc = check_dims(dims, true)) return rc;
  if (dims->rows == 0) return 0;
  const int64_t M = dims->rows * dims->k;
  FSC_CHECK_ARG(x && x_scale && index && (plan || few(M, dims->n_experts)) && weight && w_in && w_in_scale && w_out && w_out_scale && workspace && y,
                "expert_mlp_q8: null array");
  FSC_CHECK_ARG(x_stride >= 0, "expert_mlp_q8: negative row stride");
  const int tile = tile_rows(M, dims->n_experts);
  const Plan p = plan_of(const_cast<int32_t*>(plan), M, dims->n_experts, tile);
  Args g = args_of(*dims, p);
  const Space s = forward_space(*dims);
  char* ws = (char*)workspace;
  g.index = index;
  g.x = x; g.xs = x_stride; g.weight = weight; g.w_in = w_in; g.w_out = w_out;
  g.xscale = x_scale; g.in_scale = w_in_scale; g.out_scale = w_out_scale;
  g.h = ws + s.h;
  g.o = (float*)(ws + s.o);
  g.a = (float*)(ws + s.da);
  g.hscale = (float*)(ws + s.hs);
  forward<I8, int8_t>(g, tile, y, stream);
  return fsc::check_launch("expert_mlp_q8") ? 2 : 0;
}

}  // extern "C"
