// Products of the expert readout.  For the rows by expert (expert_plan.hip), expert e's rows x:
//   up      a = W_in[e] x (gate and up halves), h = silu(a_gate) a_up
//   down    o = W_out[e] h;  y_t = sum_j weight_tj o_tj                       (combine_kernel, fixed order)
//   dh      p = W_out[e]^T dy; dweight = h . p; dh = weight p; da_up = dh silu(a_gate), da_gate = dh a_up silu'(a_gate)
//   dx      W_in[e]^T da, summed over a row's experts                          (combine_kernel)
//   dw_in   sum over rows of da x^T;  dw_out  sum over rows of dy (weight h)^T
// All are products over tiles of 128 x (32, 64 or 128) entries on the matrix cores, 32-bit accumulators:
//   bf16 rows: v_mfma_f32_16x16x32_bf16;  8-bit rows: v_mfma_i32_16x16x64_i8;
//   fp32 rows: two fp16 parts an operand and three products (split2h_pk, mfma_x3), each row of the rows' operand and
//     each output column's weights brought below 2^14 by a power of two of their own (from their largest magnitude,
//     one pass before the products; h's and da's come from the products that make them) and the sums brought back
//     exactly: 22 bits of every value down to 2^-17 of its row's largest, 2^-39 of that below;
//   fp32 weight gradients, and all fp32 products where an expert has few rows: three bf16 parts and six products (split3,
//     mfma_x6), 24 bits at any scale, since there the sum runs over rows of different scales, or a pass over the weights
//     for their scales costs more than three products;
//   bf16 rows where an expert has few: what is held between the kernels in fp32, its three bf16 parts against the weights
//     as they are (three products; one where both operands are bf16).
// The weights are the MFMA's A operand, the rows its B operand: a lane's four results are four neighbouring
// columns of one row, stored by one access.
//
// Measured, us for all kernels of a call and what the products alone would take at a large library product's rate (1,125
// TFLOP/s of 16-bit products): 10,000 x 640 fp32, hidden 640, two of eight experts, forward and rows' gradient 589 (262);
// 16,384 x 1,600 bf16, hidden 800, two of 16, forward and all gradients 1,408 (671); 50,000 x 640 in 8 bits, hidden 1,280,
// two of 16: 590 (219).  What bounds them is the step itself, a chain of loads, barrier, LDS and products in every block:
// counters show the matrix units 18 to 34% busy, LDS as much, no unit above 50%, a third to a half of a wave's time waiting
// for issue and a quarter for loads.  Larger tiles (128 x 256; 256 x 256 with two LDS buffers), operands copied to LDS without registers or loaded
// into them two or three steps ahead, four waves a SIMD, raised priorities in the products, and other orders of the tiles
// took the same time or more.
//
// Rounding of what is held between the kernels: bf16 rows hold h, da and weight h in bf16 (each output passes one
// such rounding and its own), or in fp32 where an expert has few rows; a, p and o stay in fp32.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "common.h"
#include "expert_plan.h"
#include "expert_room.h"
#include "expert_shares.h"
#include "expert_tiles.h"
#include "fsctep.h"

namespace fsc {
namespace experts {

constexpr int NT = 256;          // four waves, two by two
constexpr int BN = 128;          // rows of the tile's weight operand
static_assert(BN == WEIGHT_TILE, "the weight gradients' tiles");

// ---------------------------------------------------------------- tiles of the operands
// A chunk is 16 bytes of an LDS plane: 8 values (16 in 8 bits) along the row.  Straight operands (rows of the tile
// = rows of memory) lie as [row][chunk], the chunk's place XORed with the row so that 16 lanes reading one chunk
// column of 16 rows meet no bank twice; turned operands (rows of memory along K) lie as [k][column] with 16
// columns of padding and are read by ds_read_b64_tr_b16.
constexpr int TRP = 128 + 16;

template <int KIND, int ROWS, bool TR, typename T, int NT>
struct Tile {                                                        // T: the type in memory
  using E = El<KIND>;
  static constexpr int CPR = E::BK / E::CE;                          // chunks of a straight row
  static constexpr int NCH = TR ? E::BK * ROWS / 8 : ROWS * CPR;     // chunks of the tile
  static constexpr int PER = (NCH + NT - 1) / NT;                    // chunks of a thread
  static constexpr int PLANE = TR ? E::BK * TRP * 2 : ROWS * CPR * 16;   // bytes
  static constexpr int PL = E::template planes<T>;
  static constexpr int BYTES = PLANE * PL;

  static constexpr int NV = E::CE * sizeof(T) / 16;                  // 16-byte parts of a chunk in memory

  struct Reg { u4v v[NV]; };
  Reg reg[PER];
  // F32: what the values are multiplied by, for each chunk (straight) or column of the thread's chunks (turned)
  static constexpr int NSC = KIND == F32 ? (TR ? 8 : PER) : 1;
  float scale[NSC];

  __device__ static constexpr int row_of(int c) { return TR ? c / (ROWS / 8) : c / CPR; }
  __device__ static constexpr int chunk_of(int c) { return TR ? c % (ROWS / 8) : c % CPR; }
  __device__ static constexpr int swz(int row) { return CPR == 4 ? (row >> 1) & 3 : row & 7; }

  // chunk c of the thread at byte off + more of a buffer (more the same for the wave), zeros outside it or with drop
  __device__ __forceinline__ void fetch(int c, __amdgpu_buffer_rsrc_t rsrc, uint32_t off, int more = 0, bool drop = false) {
    const int o = (int)(drop ? kDropOffset : off);
#pragma unroll
    for (int i = 0; i < NV; ++i)
      reg[c].v[i] = __builtin_bit_cast(u4v, __builtin_amdgcn_raw_buffer_load_b128(rsrc, o + 16 * i, more, 0));
  }
  // chunk c of the thread from p (n values of it exist, the rest are zeros), of any alignment
  __device__ __forceinline__ void fetch(int c, const T* p, int n) {
    alignas(16) T t[E::CE];
#pragma unroll
    for (int i = 0; i < E::CE; ++i) t[i] = i < n ? p[i] : (T)0;
    __builtin_memcpy(&reg[c], t, sizeof(t));
  }
  // of the step's chunks, entries from `left` of the step's on become zeros (straight: along the reduction, where a row
  // ends inside a chunk and the loads have gone on into the next one)
  __device__ __forceinline__ void cut(int left) {
    static_assert(!TR);
    constexpr int EW = 4 / sizeof(T);                                // entries of a 32-bit word
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int l = left - chunk_of(threadIdx.x + i * NT) * E::CE;
#pragma unroll
      for (int w = 0; w < 4 * NV; ++w) reg[i].v[w / 4][w % 4] = w * EW < l ? reg[i].v[w / 4][w % 4] : 0;
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
      if constexpr (KIND == F32 || KIND == X6 || PL == 3) {
        float v[8];
        if constexpr (sizeof(T) == 4) {
          __builtin_memcpy(v, &reg[i], 32);
        } else {
          const bf8 b = __builtin_bit_cast(bf8, reg[i].v[0]);
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] = (float)b[j];
        }
        if constexpr (KIND == F32) {
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] *= scale[TR ? j : i];
          h8 h, l;
          split2h_pk(v, h, l);
          *reinterpret_cast<h8*>(lds + at) = h;
          *reinterpret_cast<h8*>(lds + PLANE + at) = l;
        } else {
          bf8 h, m, l;
          split3(v, h, m, l);
          *reinterpret_cast<bf8*>(lds + at) = h;
          *reinterpret_cast<bf8*>(lds + PLANE + at) = m;
          *reinterpret_cast<bf8*>(lds + 2 * PLANE + at) = l;
        }
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

// acc[i][j] += (weight tiles w0 + i) (row tiles x0 + j) over one K step in LDS.
template <int KIND, int NI, int NJ, typename TW, typename TX>
__device__ __forceinline__ void step(const char* lw, const char* lx, int w0, int x0,
                                     typename Acc<KIND>::V (&acc)[NI][NJ]) {
  using E = El<KIND>;
  constexpr int KS = E::BK / (4 * E::CE);
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    u4v x[NJ][TX::PL];
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int p = 0; p < TX::PL; ++p) x[j][p] = TX::frag(lx, p, x0 + j, ks);
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      u4v w[TW::PL];
#pragma unroll
      for (int p = 0; p < TW::PL; ++p) w[p] = TW::frag(lw, p, w0 + i, ks);
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        if constexpr (KIND == F32)
          acc[i][j] = mfma_x3(__builtin_bit_cast(h8, w[0]), __builtin_bit_cast(h8, w[1]),
                              __builtin_bit_cast(h8, x[j][0]), __builtin_bit_cast(h8, x[j][1]), acc[i][j]);
        else if constexpr (KIND == X6)
          acc[i][j] = mfma_x6(__builtin_bit_cast(bf8, w[0]), __builtin_bit_cast(bf8, w[1]),
                              __builtin_bit_cast(bf8, w[2]), __builtin_bit_cast(bf8, x[j][0]),
                              __builtin_bit_cast(bf8, x[j][1]), __builtin_bit_cast(bf8, x[j][2]), acc[i][j]);
        else if constexpr (KIND == BF16 || KIND == FINE)
#pragma unroll
          for (int p = TW::PL * TX::PL - 1; p >= 0; --p)     // small terms first
            acc[i][j] = mfma_bf16(__builtin_bit_cast(bf8, w[p % TW::PL]), __builtin_bit_cast(bf8, x[j][p / TW::PL]), acc[i][j]);
        else
          acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i4v, w[0]),
                                                            __builtin_bit_cast(i4v, x[j][0]), acc[i][j], 0, 0, 0);
      }
    }
  }
}

// n entries in whole 32-bit words (rows that end inside one are read from padded copies)
template <typename T>
__device__ __forceinline__ int64_t whole_words(int n) { constexpr int w = 4 / sizeof(T); return (n + w - 1) / w * w; }

// ---------------------------------------------------------------- the products by row tiles
// A block takes one tile: rows of one expert, read by their numbers (up, dh: the gather is the load), by columns.  Two
// operands meet in LDS, double-buffered in registers, swizzled so that no read meets a bank twice; W_out and W_in of the
// backward are turned by the transposing LDS reads.  The epilogues make h, da, dweight's parts and the codes from the sums in
// registers, through LDS once into whole lines.  us at the sizes above (up, down, dh, dx): fp32 141, 86, 123, 158 (98, 49,
// 49, 98 GFLOP of 16-bit products: 560 to 700 TFLOP/s, dh with 204 MB of a and da besides); bf16 233, 151, 191, 248 (168, 84,
// 84, 168 GFLOP: 560 to 720 TFLOP/s, up with 210 MB of a, down and dx with 210 MB of o besides); 8 bits 311 and 200 (328
// and 164 Gop; up's issue is half vector instructions: sigmoid, codes).
//
// up: 64 hidden columns a tile, their gate and up rows in turn by 16, so that a wave holds both of a column.
// WW waves side by side along the weight operand, four (8-bit up: so many that 128 hidden columns make a tile)
// 16-row tiles each, two along the rows.  Registers of 8-bit up are held to 128, so that two of its blocks of eight waves
// share a CU (424 -> 333 us at 50,000 rows); those of fp32 dh to 168, three waves a SIMD (124 -> 118 us).
template <int KIND, int MODE>
constexpr int waves_w() { return KIND == I8 && MODE == UP ? 4 : 2; }
template <int KIND, int MODE, bool VEC>                    // waves a SIMD that the registers leave room for
constexpr int rows_waves() { return VEC && KIND == I8 && MODE == UP ? 4 : VEC && KIND == F32 && MODE == DH ? 3 : 2; }

template <int KIND, typename S, int MODE, int NJ, bool VEC>
__global__ __launch_bounds__((128 * waves_w<KIND, MODE>()), (rows_waves<KIND, MODE, VEC>())) void rows_kernel(Args g) {
  using E = El<KIND>;
  using T = typename E::T;                                   // of the arrays between the kernels; S: the caller's
  using R = std::conditional_t<MODE == DOWN || MODE == DX, T, S>;
  constexpr int BM = 32 * NJ, NI = 4, WW = waves_w<KIND, MODE>(), BN = 64 * WW, NT = 128 * WW;
  constexpr bool TR = MODE == DH || MODE == DX;
  using TW = Tile<KIND, BN, TR, S, NT>;
  using TX = Tile<KIND, BM, false, R, NT>;
  // the operands; after the products the waves' rows and the sums across waves
  constexpr int OPERANDS = TW::BYTES + TX::BYTES, AFTER = (2 * WW * TURN + WW * BM) * 4;
  __shared__ __align__(16) char lds[OPERANDS > AFTER ? OPERANDS : AFTER];
  __shared__ int32_t slots[BM], rws[BM];
  char* lw = lds;
  char* lx = lds + TW::BYTES;

  const int NC = MODE == UP ? BN / 2 : BN;                   // output columns of a tile
  // output columns (8 bits: the last group of h is whole)
  const int cols = KIND == I8 && MODE == UP ? g.ldf : MODE == UP || MODE == DH ? g.F : g.H;
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

  // The reduction: SEG segments of K entries (dx: the gate half of da and W_in, then the up half).  h and da are padded
  // with zeros to ldf.
  constexpr bool GATHER = MODE == UP || MODE == DH;
  constexpr int SEG = MODE == DX ? 2 : 1;
  const int K = GATHER ? g.H : g.F, KX = GATHER ? g.H : g.ldf;
  const int64_t xld = MODE == UP ? g.xs : MODE == DH ? g.ds : MODE == DOWN ? g.ldf : 2 * (int64_t)g.ldf;
  const R* const xbase = MODE == UP     ? (const R*)g.x
                         : MODE == DH   ? (const R*)g.dy
                         : MODE == DOWN ? (const R*)g.h + p0 * g.ldf
                                        : (const R*)g.da + p0 * 2 * g.ldf;
  const int64_t wld = MODE == UP || MODE == DX ? g.li : g.lo;
  const int64_t wseg = (MODE == UP ? 2 * g.F : MODE == DX ? g.F : g.H) * wld;   // entries of the weights of a segment
  const S* const wbase = (MODE == UP || MODE == DX ? (const S*)g.w_in : (const S*)g.w_out) + e * wseg * SEG;
  // Where the thread's chunks lie in the first step, in entries (OFF: a 32-bit byte offset for VEC, where buffers over
  // x or dy, the tile's rows and a segment's weights give zeros outside: loads without branches, at any multiple of
  // four bytes; a chunk that goes on past its row's end is cut along the reduction, and past an output's last column
  // it is not stored); kNoChunk: nowhere.
  using Off = std::conditional_t<VEC, uint32_t, int64_t>;
  constexpr Off kNoChunk = VEC ? (Off)kDropOffset : (Off)-1;
  Off xo[TX::PER], wo[TW::PER];
#pragma unroll
  for (int i = 0; i < TX::PER; ++i) {
    const int c = threadIdx.x + i * NT, row = TX::row_of(c);
    xo[i] = c < TX::NCH && row < rows
                ? (Off)(((GATHER ? rws[row] : row) * xld + TX::chunk_of(c) * E::CE) * (VEC ? sizeof(R) : 1))
                : kNoChunk;
  }
#pragma unroll
  for (int i = 0; i < TW::PER; ++i) {
    const int c = threadIdx.x + i * NT, row = TW::row_of(c);
    int64_t at = -1;
    if (TR) {
      const int n = n0 + TW::chunk_of(c) * 8;
      if (n < cols) at = row * wld + n;
    } else if (MODE == UP) {
      const int n = n0 + (row >> 5) * 16 + (row & 15);
      if (n < g.F) at = ((row & 16 ? g.F : 0) + n) * wld + TW::chunk_of(c) * E::CE;
    } else if (n0 + row < g.H) {
      at = (n0 + row) * wld + TW::chunk_of(c) * E::CE;
    }
    wo[i] = at >= 0 ? (Off)(at * (VEC ? sizeof(S) : 1)) : kNoChunk;
  }
  const __amdgpu_buffer_rsrc_t xr = buffer_rsrc_bytes(
      const_cast<R*>(xbase), (uint32_t)((((GATHER ? g.T : rows) - 1) * xld + (GATHER ? whole_words<R>(g.H) : xld)) * sizeof(R)));
  TW tw;
  TX tx;
  // fp32: the powers of two of this tile's rows and of the output columns' weights
  const uint32_t* const xm = MODE == UP ? g.xmost : MODE == DH ? g.dymost : MODE == DOWN ? g.hmost + p0 : g.damost + p0;
  const uint32_t* const wm = MODE == UP     ? g.in_row + (int64_t)e * 2 * g.F
                             : MODE == DOWN ? g.out_row + (int64_t)e * g.H
                             : MODE == DH   ? g.out_col + (int64_t)e * g.F
                                            : g.in_col + (int64_t)e * g.H;
  auto row_exp = [&](int row) { return part_exp(xm[GATHER ? rws[row < rows ? row : 0] : row < rows ? row : 0]); };
  // weight row (straight) or column (turned) i of the tile; past the last: any
  auto weight_exp = [&](int i) {
    const int n = MODE == UP ? (i & 16 ? g.F : 0) + min(n0 + (i >> 5) * 16 + (i & 15), g.F - 1) : min(n0 + i, cols - 1);
    return part_exp(wm[n]);
  };
  if constexpr (KIND == F32) {
#pragma unroll
    for (int i = 0; i < TX::PER; ++i) tx.scale[i] = ldexpf(1.f, row_exp(TX::row_of(threadIdx.x + i * NT) % BM));
#pragma unroll
    for (int i = 0; i < TW::NSC; ++i)
      tw.scale[i] = ldexpf(1.f, weight_exp(TR ? TW::chunk_of(threadIdx.x) * 8 + i : TW::row_of(threadIdx.x + i * NT)));
  }
  const int per_seg = (K + E::BK - 1) / E::BK, steps = SEG * per_seg;
  auto fetch = [&](int s) {
    const int seg = SEG == 2 && s >= per_seg, k0 = (s - seg * per_seg) * E::BK;
    const bool last = k0 + E::BK > K;                        // the same for the whole block
    const int64_t xat = seg * g.ldf + k0;
#pragma unroll
    for (int i = 0; i < TX::PER; ++i) {
      const int left = KX - k0 - TX::chunk_of(threadIdx.x + i * NT) * E::CE;
      if constexpr (VEC) {
        tx.fetch(i, xr, xo[i], (int)(xat * sizeof(R)), last && left <= 0);
      } else {
        tx.fetch(i, xbase + xo[i] + xat, xo[i] < 0 ? 0 : left);
      }
    }
    // turned: the buffer begins at row k0 of the segment and ends with it, rows past K are outside
    const int64_t wat = TR ? k0 * wld : k0;
    const __amdgpu_buffer_rsrc_t wr = buffer_rsrc_bytes(const_cast<S*>(wbase + seg * wseg + (TR ? wat : 0)),
                                                        (uint32_t)((wseg - (TR ? wat : 0)) * sizeof(S)));
#pragma unroll
    for (int i = 0; i < TW::PER; ++i) {
      const int c = threadIdx.x + i * NT;
      const int left = TR ? K - k0 - TW::row_of(c) : K - k0 - TW::chunk_of(c) * E::CE;
      if constexpr (VEC) {
        tw.fetch(i, wr, wo[i], TR ? 0 : (int)(wat * sizeof(S)), !TR && last && left <= 0);
      } else {
        const int n = TR ? cols - n0 - TW::chunk_of(c) * 8 : left;
        tw.fetch(i, wbase + seg * wseg + wo[i] + wat, wo[i] < 0 || left <= 0 ? 0 : n);
      }
    }
  };

  // (dx: da is padded and its reduction runs over W_in's rows)
  auto trim = [&](int s) {
    if constexpr (VEC && MODE != DX) {
      if (K % E::CE == 0 || s + 1 < steps) return;
      if constexpr (!TR) tw.cut(K - s * E::BK);
      if constexpr (GATHER) tx.cut(K - s * E::BK);
    }
  };

  typename Acc<KIND>::V acc[NI][NJ];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j) acc[i][j] = {0, 0, 0, 0};
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
  const int w0 = wave % WW * NI, x0 = wave / WW * NJ;        // first tiles of the wave

  if constexpr (KIND == I8 && MODE == DOWN) {
    // a K step is one group of h: its sums are whole numbers, scaled by the group's unit into 32-bit floats
    f4 sum[4][NJ];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < NJ; ++j) sum[i][j] = f4{0.f, 0.f, 0.f, 0.f};
    const int ng = g.ldf / QG;
    // the units, loaded before the operands of their step, since loads return in order; rows past the tile: the last's
    float next[NJ];
    auto units = [&](int s) {
#pragma unroll
      for (int j = 0; j < NJ; ++j) next[j] = g.hscale[(p0 + min(16 * (x0 + j) + r, rows - 1)) * ng + s];
    };
    units(0);
    fetch(0);
    for (int s = 0; s < steps; ++s) {
      trim(s);
      __syncthreads();
      tw.put(lw);
      tx.put(lx);
      __syncthreads();
      float u[NJ];
#pragma unroll
      for (int j = 0; j < NJ; ++j) u[j] = next[j];
      if (s + 1 < steps) {
        units(s + 1);
        fetch(s + 1);
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
    for (int i = 0; i < NI; ++i) {
      const int n = n0 + (w0 + i) * 16 + 4 * q;
      f4 sc;
#pragma unroll
      for (int v = 0; v < 4; ++v) sc[v] = g.out_scale[(int64_t)e * g.H + min(n + v, g.H - 1)];
#pragma unroll
      for (int j = 0; j < NJ; ++j) sum[i][j] *= sc;
    }
    __syncthreads();
    finish<KIND, MODE, NI, NJ, WW, BM>(g, RowTile{e, rows, p0, slots, rws}, n0, ci, wave % WW, w0, x0, sum,
                                       reinterpret_cast<float*>(lds));
  } else {
    fetch(0);
    for (int s = 0; s < steps; ++s) {
      trim(s);
      __syncthreads();
      tw.put(lw);
      tx.put(lx);
      __syncthreads();
      if (s + 1 < steps) fetch(s + 1);
      step<KIND, 4, NJ, TW, TX>(lw, lx, w0, x0, acc);
    }
    if constexpr (KIND == F32) {
      const int r = lane & 15, q = lane >> 4;
      int xe[NJ];
#pragma unroll
      for (int j = 0; j < NJ; ++j) xe[j] = row_exp(16 * (x0 + j) + r);
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const int we = weight_exp(16 * (w0 + i) + 4 * q + v);
#pragma unroll
          for (int j = 0; j < NJ; ++j) acc[i][j][v] = __builtin_amdgcn_ldexpf(acc[i][j][v], -(xe[j] + we));
        }
    }
    __syncthreads();                                         // the operands in LDS have been read
    finish<KIND, MODE, NI, NJ, WW, BM>(g, RowTile{e, rows, p0, slots, rws}, n0, ci, wave % WW, w0, x0, acc,
                                       reinterpret_cast<float*>(lds));
  }
}

// ---------------------------------------------------------------- weight gradients
// An expert's positions in shares of g.share, one after the other over the experts (one, empty, for an expert without
// rows): the expert, which of its shares, how many it has, the number of its first.
struct Share {
  int e, at, n;
  int64_t first;
};

// Runs f(e, shares of expert e, shares before the wave's 64 experts, inclusive sum over the lanes, all lanes) for 64
// experts at a time until it returns true.
template <typename F>
__device__ __forceinline__ void scan_shares(const Args& g, F&& f) {
  const int lane = threadIdx.x & 63;
  int before = 0;
  for (int e0 = 0; e0 < g.E; e0 += 64) {
    const int e = e0 + lane;
    const int rows = g.offsets[min(e + 1, g.E)] - g.offsets[min(e, g.E)];
    const int n = e >= g.E ? 0 : rows > 0 ? (rows - 1) / g.share + 1 : 1;
    int sum = n;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int u = __shfl_up(sum, off, 64);
      if (lane >= off) sum += u;
    }
    const int all = __shfl(sum, 63, 64);
    if (f(e0, n, before, sum, all)) return;
    before += all;
  }
}
// Every wave finds the same: the share of that number, false past the last.
__device__ __forceinline__ bool find_share(const Args& g, int unit, Share& s) {
  bool found = false;
  scan_shares(g, [&](int e0, int n, int before, int sum, int all) {
    if (unit >= before + all) return false;
    const int l = __ffsll((unsigned long long)__ballot(before + sum > unit)) - 1;
    const int ln = __shfl(n, l, 64), ls = __shfl(sum, l, 64);
    s = Share{__builtin_amdgcn_readfirstlane(e0 + l), __builtin_amdgcn_readfirstlane(unit - (before + ls - ln)),
              __builtin_amdgcn_readfirstlane(ln), __builtin_amdgcn_readfirstlane(before + ls - ln)};
    return found = true;
  });
  return found;
}
__device__ __forceinline__ int count_shares(const Args& g) {
  int total = 0;
  scan_shares(g, [&](int, int, int before, int, int all) {
    total = before + all;
    return false;
  });
  return __builtin_amdgcn_readfirstlane(total);
}

// dw_in[e][m][n] = sum over expert e's positions of da[.][m] x[.][n]; dw_out[e][m][n] = that of dy[.][m] hw[.][n].
// The matrix of the contiguous output index n is the MFMA's A operand; both are turned.  The reduction runs over the rows,
// whose numbers are loaded two steps ahead of their use, the rows themselves one step.  bf16 16,384 x 1,600, hidden 800:
// 296 us dw_in, 184 us dw_out (570 and 460 TFLOP/s); fp32 4,099 x 331, hidden 203, with shares: 46 + 9 and 26 + 7 us.
// FEW: h's arrays lie by slot and the block finds the expert's slots itself.
template <int KIND, typename S, int MODE, bool VEC, bool FEW>
__global__ __launch_bounds__(NT, 2) void weights_kernel(Args g) {
  using E = El<KIND>;
  using T = typename E::T;
  using RA = std::conditional_t<MODE == DWIN, S, T>;
  using RB = std::conditional_t<MODE == DWIN, T, S>;
  using TT = Tile<KIND, BN, true, RA, NT>;
  using TB = Tile<KIND, BN, true, RB, NT>;
  __shared__ __align__(16) char lds[TT::BYTES + TB::BYTES];
  char* la = lds;
  char* lb = lds + TT::BYTES;
  const int na = MODE == DWIN ? g.H : g.ldf, nb = MODE == DWIN ? 2 * g.ldf : g.H;   // columns of the operands
  const int ta = (na + BN - 1) / BN, tb = (nb + BN - 1) / BN;
  const int tiles = ta * tb, w = (int)(blockIdx.x >> 3), x = (int)(blockIdx.x & 7);
  Share sh;
  int c;
  if (FEW || one_share_each(g.M, g.share)) {
    const int per = (tiles + 7) / 8;
    sh = Share{w / per, 0, 1, 0};
    c = x * per + w % per;
    if (c >= tiles || sh.e >= g.E) return;
  } else if (runs_by_share(false, tiles)) {
    const int per = (tiles + 7) / 8;
    c = x * per + w % per;
    if (c >= tiles || !find_share(g, w / per, sh)) return;
  } else {
    const int64_t all = (int64_t)count_shares(g) * tiles, per = (all + 7) / 8, i = x * per + w;
    if (w >= per || i >= all) return;
    const int unit = (int)(i / tiles);
    c = (int)(i - (int64_t)unit * tiles);
    if (!find_share(g, unit, sh)) return;
  }
  const int e = sh.e;
  const int b0 = (c / ta) * BN, a0 = (c % ta) * BN;
  __shared__ int16_t list[FEW ? FEW_SLOTS : 1];
  int64_t p0 = 0, cnt;
  if constexpr (FEW) {
    cnt = few_slots(g, e, few_first(g), list);
    __syncthreads();
  } else {
    p0 = g.offsets[e] + (int64_t)sh.at * g.share;
    cnt = std::min<int64_t>(g.share, g.offsets[e + 1] - p0);
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
  // DWIN: A the gathered rows of x, B da's; DWOUT: A hw's rows, B the gathered rows of dy.  VEC as in rows_kernel,
  // the arrays between the kernels through a buffer over the step's rows.
  const int64_t gs = MODE == DWIN ? g.xs : g.ds, ps = MODE == DWIN ? 2 * (int64_t)g.ldf : g.ldf;
  const S* const gbase = MODE == DWIN ? (const S*)g.x : (const S*)g.dy;
  const T* const pbase = (MODE == DWIN ? (const T*)g.da : (const T*)g.hw) + p0 * ps;
  const __amdgpu_buffer_rsrc_t gr =
      buffer_rsrc_bytes(const_cast<S*>(gbase), (uint32_t)(((g.T - 1) * gs + whole_words<S>(g.H)) * sizeof(S)));
  auto fetch = [&](int64_t k0) {
    const int left = cnt - k0 < E::BK ? (int)(cnt - k0) : E::BK;
    const T* const prow = pbase + (FEW ? 0 : k0 * ps);
    const __amdgpu_buffer_rsrc_t pr =
        buffer_rsrc_bytes(const_cast<T*>(prow), (uint32_t)((FEW ? g.M : left) * ps) * sizeof(T));
#pragma unroll
    for (int i = 0; i < TT::PER; ++i) {
      const int cc = threadIdx.x + i * NT, kr = TT::row_of(cc), n = TT::chunk_of(cc) * 8;
      const int ng = (MODE == DWIN ? a0 : b0) + n, np = (MODE == DWIN ? b0 : a0) + n;   // columns of the two
      const int npc = MODE == DWIN ? nb : na;
      const int64_t gat = (int64_t)tok[i] * gs + ng, pat = (FEW ? (kr < left ? list[k0 + kr] : 0) : kr) * ps + np;
      const bool gin = kr < left && ng < g.H, pin = kr < left && np < npc;
      auto load = [&](auto& gt, auto& pt) {
        if constexpr (VEC) {
          gt.fetch(i, gr, gin ? (uint32_t)gat * (uint32_t)sizeof(S) : kDropOffset);
          pt.fetch(i, pr, pin ? (uint32_t)pat * (uint32_t)sizeof(T) : kDropOffset);
        } else {
          gt.fetch(i, gbase + gat, gin ? g.H - ng : 0);
          pt.fetch(i, prow + pat, pin ? npc - np : 0);
        }
      };
      if constexpr (MODE == DWIN) load(A, B);
      else load(B, A);
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
    // (out counts the experts before as well)
    float* part = g.dwsplit + (sh.first + sh.at - e) * ((int64_t)(MODE == DWIN ? 2 : 1) * g.F * g.H) + out;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int n = a0 + (w0 + i) * 16 + 4 * q;
      if (n >= len) continue;
      if (!FEW && sh.n > 1) store4(part + n, acc[i][j], len - n);
      else store4(dw + n, acc[i][j], len - n);
    }
  }
}

// The weight gradients (n entries an expert) of the experts with more than one share, in the shares' order; four entries
// and four shares at a time are on their way together.  Blocks (., y) take every gridDim.y-th of these experts.
template <typename S>
__global__ __launch_bounds__(NT) void sum_shares_kernel(Args g, int64_t n, S* __restrict__ dw) {
  const int64_t step = (int64_t)gridDim.x * NT;
  int turn = 0;
  scan_shares(g, [&](int e0, int shares, int before, int sum, int) {
    for (uint64_t some = __ballot(shares > 1); some; some &= some - 1) {
      if (turn++ % gridDim.y != blockIdx.y) continue;
      const int l = __ffsll((unsigned long long)some) - 1, k = __shfl(shares, l, 64);
      const float* part = g.dwsplit + (int64_t)(before + __shfl(sum, l, 64) - k) * n;
      S* out = dw + (e0 + l) * n;
      for (int64_t i0 = (int64_t)blockIdx.x * NT + threadIdx.x; i0 < n; i0 += 4 * step) {
        float t[4] = {0.f, 0.f, 0.f, 0.f};
        for (int s0 = 0; s0 < k; s0 += 4) {
          float v[4][4];
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) v[j][i] = part[min(s0 + j, k - 1) * n + min(i0 + i * step, n - 1)];
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (s0 + j < k)
#pragma unroll
              for (int i = 0; i < 4; ++i) t[i] += v[j][i];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (i0 + i * step < n) out[i0 + i * step] = from_f<S>(t[i]);
      }
    }
    return false;
  });
}

// ---------------------------------------------------------------- one pass over the rows of the caller's arrays
// A wave a row of up to four arrays: its largest magnitude (`most`, for the fp32 products' parts) and a copy padded with
// zeros to whole chunks (`copy`, where the array's rows cannot be read 16 bytes at a time); and zeros for what later
// kernels raise.
struct Pass {
  struct Array {
    const void* p;
    int64_t rows, ld;
    int n;
    uint32_t* most;
    void* copy;
    int cld;
  } a[4];
  int arrays;
  uint32_t* zero;
  int64_t zeros;
};

template <typename S>
__global__ __launch_bounds__(NT) void pass_kernel(Pass a) {
  const int lane = threadIdx.x & 63;
  const int64_t z = (int64_t)blockIdx.x * NT + threadIdx.x, zn = (int64_t)gridDim.x * NT;
  for (int64_t i = z; i < a.zeros; i += zn) a.zero[i] = 0;
  int64_t total = 0;
  for (int k = 0; k < a.arrays; ++k) total += a.a[k].rows;
  for (int64_t all = (int64_t)blockIdx.x * (NT / 64) + (threadIdx.x >> 6); all < total; all += (int64_t)gridDim.x * (NT / 64)) {
  int64_t row = all;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if (k >= a.arrays) break;
    const Pass::Array& v = a.a[k];
    if (row >= 0 && row < v.rows) {
      const S* p = (const S*)v.p + row * v.ld;
      constexpr int V = 16 / sizeof(S);
      uint32_t m = 0;
      if (v.copy) {
        S* c = (S*)v.copy + row * v.cld;
        for (int i = lane; i < v.cld; i += 64) {
          const S x = i < v.n ? p[i] : (S)0;
          c[i] = x;
          if constexpr (sizeof(S) > 1) m = max(m, abs_bits(to_f(x)));
        }
      } else if constexpr (sizeof(S) > 1) {
        if ((uintptr_t)p % 16 == 0 && v.n % V == 0) {
          for (int i = lane * V; i < v.n; i += 64 * V) {
            float x[V];
            load_vec<V>(p + i, x);
#pragma unroll
            for (int j = 0; j < V; ++j) m = max(m, abs_bits(x[j]));
          }
        } else {
          for (int i = lane; i < v.n; i += 64) m = max(m, abs_bits(to_f(p[i])));
        }
      }
      if constexpr (sizeof(S) > 1) {
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, off, 64));
        if (lane == 0 && v.most) v.most[row] = m;
      }
    }
    row -= v.rows;
  }
  }
}

// Columns of an expert's matrix (R x n): 64 columns and 64 rows a block, raised in `out` [E][n], zeros before.  One read of
// the weights: 26 MB 6 us.
template <typename S>
__global__ __launch_bounds__(NT) void col_most_kernel(const S* __restrict__ w, int R, int n, uint32_t* __restrict__ out) {
  const int c = blockIdx.x * 64 + (threadIdx.x & 63), r0 = blockIdx.y * 64 + (threadIdx.x >> 6);
  if (c >= n) return;
  const S* p = w + (int64_t)blockIdx.z * R * n + c;
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int r = r0 + 4 * i;
    m = max(m, abs_bits(to_f(p[(int64_t)(r < R ? r : r0 < R ? r0 : 0) * n])));
  }
  atomicMax(out + (int64_t)blockIdx.z * n + c, m);
}

// ---------------------------------------------------------------- rows from their experts, in slot order
// The row of a slot in the arrays between the kernels, -1 for a slot with no expert.
__device__ __forceinline__ int place_of(const int32_t* place, const int32_t* index, int E, int64_t s) {
  if (place) return place[s];
  const int e = index[s];
  return e >= 0 && e < E ? (int)s : -1;
}

// dweight by slot: the partial sums over the column tiles, in order; 0 for a slot with no expert.
struct Dweight {
  int64_t M;
  int parts;
  const float* part;
  float* out;
};
__device__ __forceinline__ void dweight_of(const Dweight& d, const int32_t* place, const int32_t* index, int E) {
  for (int64_t s = (int64_t)blockIdx.x * NT + threadIdx.x; s < d.M; s += (int64_t)gridDim.x * NT) {
    const int p = place_of(place, index, E, s);
    float t = 0.f;
#pragma unroll 8
    for (int i = 0; i < d.parts; ++i) t += d.part[(int64_t)i * d.M + max(p, 0)];
    d.out[s] = p >= 0 ? t : 0.f;
  }
}

// y_t = sum_j weight_tj o_tj in the order of j, the same every time; o in 32 bits.  Four slots' places, weights and products
// at a time are on their way together (a slot with none reads place 0).  Bound by memory: 16,384 x 1,600 bf16 from 210 MB of
// o 45 us (5.8 TB/s), 50,000 x 640 57 us (5.6 TB/s).
template <typename T>
__global__ __launch_bounds__(NT) void combine_kernel(int64_t rows, int H, int ldo, int k,
                                                     const int32_t* __restrict__ place,
                                                     const int32_t* __restrict__ index, int E,
                                                     const float* __restrict__ weight, const float* __restrict__ o,
                                                     T* __restrict__ y, Dweight d) {
  const int nv = (H + 3) / 4;
  const int64_t n = rows * nv;
  for (int64_t i = (int64_t)blockIdx.x * NT + threadIdx.x; i < n; i += (int64_t)gridDim.x * NT) {
    const int64_t t = i / nv;
    const int c = (int)(i - t * nv) * 4;
    f4 s = {0.f, 0.f, 0.f, 0.f};
    for (int j0 = 0; j0 < k; j0 += 4) {
      int p[4];
      float w[4];
      f4 v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t slot = t * k + min(j0 + j, k - 1);
        p[j] = place_of(place, index, E, slot);
        w[j] = weight ? weight[slot] : 1.f;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j0 + j < k) v[j] = ld4(o + (int64_t)max(p[j], 0) * ldo + c);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j0 + j < k && p[j] >= 0) s += w[j] * v[j];
    }
    store4(y + t * H + c, s, H - c);
  }
  if (d.out) dweight_of(d, place, index, E);
}

__global__ __launch_bounds__(NT) void dweight_kernel(Dweight d, const int32_t* __restrict__ place,
                                                     const int32_t* __restrict__ index, int E) {
  dweight_of(d, place, index, E);
}

// ---------------------------------------------------------------- host
inline int up8(int v) { return (v + 7) / 8 * 8; }

// Few rows: so few for each expert on average that reading the weights once, into registers, and no plan of the rows win
// over the tiles' matrix products; and few enough slots for a block to look through.  Rows' step (8 bits: forward), us,
// few against tiles, slots for each of eight experts: fp32 640 x 640 8: 72, 128; 30: 99, 129; 1,600 x 1,600 25: 292, 304; but
// for each of 32 experts 576 x 808 11: 145, 164; 21: 219, 188.
// bf16 640 8: 71, 75; 16: 81, 74; 1,600 12: 167, 143.  8 bits 640 16: 19, 23; 25: 24, 22; 1,600 8: 28, 36; 12: 37, 37.
inline bool few(const FscExpertDims& d) {
  const int64_t M = d.rows * d.k;
  const int most = d.dtype == FSC_BF16 ? 8 : d.dtype == FSC_F32 && M <= 256 ? 32 : 16;
  return M <= FEW_SLOTS && M <= most * (int64_t)d.n_experts;
}

// Forward by dot products (expert_one.hip): eight slots, or no more than experts, so that hardly any weight is read twice.
// Against the few-rows kernels, us, width and hidden 640, fp32 / bf16 / 8 bits: 2 slots 7.4 / 7.5 / 10.1 against 12.2 /
// 11.2 / 13.3; 16 of 32 experts 16 / 13 / 11 against 26 / 17 / 14; 64 of 64 39 / 37 / 22 against 70 / 45 / 26; but four for
// each of 16 experts 31 / 33 / 20 against 25 / 22 / 15, and two for each of 32 experts of 1,600 x 1,600 265 against 197.
inline bool one(int64_t M, int E) { return M <= 8 || (M <= FEW_SLOTS && M <= E); }

// Rows of a tile: 128 only where the products have enough tiles of 128 x 128 to fill the chip a few times (M rows by
// F + H columns, up and down alike), else more blocks with fewer rows.  Forward and all gradients, us with 128, 64, 32 rows:
// 1,024 tiles and more: 6,000 slots, 1,600 x 1,600, bf16 489, 576, 769; 625: 8,000 slots, 640 x 640, fp32 454, 455, 509, bf16
// 211, 208, 220; 113: 1,371 slots, 949 x 406, fp32 371, 346, 326; 16: 270 slots, 872 x 95, fp32 153, 128, 116.
inline int tile_rows(const FscExpertDims& d) {
  const int64_t M = d.rows * d.k, avg = M / d.n_experts, tiles = M * (d.width + d.hidden) / (128 * 128);
  return avg <= 32 || tiles < 224 ? 32 : avg <= 64 || tiles < 1024 ? 64 : 128;
}

// Whether rows at p can be read 16 bytes at a time through one buffer: whole 32-bit words, and all of them below
// kDropOffset bytes.
inline bool vec_ok(const void* p, int64_t rows, int64_t stride, int size, int n) {
  return !p || ((uintptr_t)p % 4 == 0 && stride * size % 4 == 0 && !odd_rows(n, size) &&
                ((rows - 1) * stride + n) * size < (int64_t)kDropOffset);
}
// The same for the few-rows kernels, which read 16 bytes through pointers as well and step through an expert's matrix with
// signed 32-bit offsets; 8-bit rows in whole 16 bytes.
inline bool few_vec_ok(const void* p, int64_t rows, int64_t stride, int size, int n) {
  return vec_ok(p, rows, stride, size, n) &&
         (!p || (n >= 8 && ((rows - 1) * stride + n) * size < (1ll << 31) &&
                 (size > 1 || ((uintptr_t)p % 16 == 0 && stride % 16 == 0 && n % 16 == 0))));
}

template <int KIND, typename S, int MODE>
void launch_rows(const Args& g, int tile, bool vec, hipStream_t st) {
  constexpr int WW = waves_w<KIND, MODE>(), NC = MODE == UP ? 32 * WW : 64 * WW;
  const int cols = KIND == I8 && MODE == UP ? g.ldf : MODE == UP || MODE == DH ? g.F : g.H;
  const unsigned grid = tile_grid(g.n_tiles, (cols + NC - 1) / NC);
  auto go = [&](auto NJ) {
    constexpr int nj = decltype(NJ)::value;
    if (vec) rows_kernel<KIND, S, MODE, nj, true><<<grid, 128 * WW, 0, st>>>(g);
    else rows_kernel<KIND, S, MODE, nj, false><<<grid, 128 * WW, 0, st>>>(g);
  };
  if constexpr (KIND == FINE) {               // 32 rows a tile (fine)
    go(std::integral_constant<int, 1>{});
  } else {
    if (tile == 128) go(std::integral_constant<int, 4>{});
    else if (tile == 64) go(std::integral_constant<int, 2>{});
    else go(std::integral_constant<int, 1>{});
  }
}

// bytes of a value of the arrays between the kernels
template <int KIND> constexpr int held_bytes() { return sizeof(typename El<KIND>::T); }

template <int KIND, typename S, int MODE, bool FEW = false>
void launch_weights(Args g, bool vec, hipStream_t st) {
  const int64_t na = MODE == DWIN ? g.H : g.ldf, nb = MODE == DWIN ? 2 * g.ldf : g.H;
  const int64_t tiles = weight_tiles(na, nb);
  g.share = FEW ? 0 : weight_share(g.M, g.E, held_bytes<KIND>(), tiles);
  const int64_t shares = FEW ? g.E : most_shares(g.M, g.E, g.share);
  const unsigned grid = (unsigned)weight_blocks(shares, tiles, runs_by_share(FEW || one_share_each(g.M, g.share), tiles));
  if (vec) weights_kernel<KIND, S, MODE, true, FEW><<<grid, NT, 0, st>>>(g);
  else weights_kernel<KIND, S, MODE, false, FEW><<<grid, NT, 0, st>>>(g);
  if (!FEW && shares > g.E) {
    const int64_t n = (int64_t)(MODE == DWIN ? 2 : 1) * g.F * g.H;
    sum_shares_kernel<S><<<dim3((unsigned)std::min<int64_t>((n + 4 * NT - 1) / (4 * NT), 512), std::min(g.E, 8)), NT, 0, st>>>(
        g, n, (S*)(MODE == DWIN ? g.dw_in : g.dw_out));
  }
}

template <typename S>
void launch_pass(const Pass& a, hipStream_t st) {
  int64_t rows = 0;
  for (int k = 0; k < a.arrays; ++k) rows += a.a[k].rows;
  if (rows == 0 && a.zeros == 0) return;
  pass_kernel<S><<<(unsigned)std::max<int64_t>(1, std::min<int64_t>((rows + 3) / 4, 1 << 20)), NT, 0, st>>>(a);
}

// Adds an array (E matrices of `rows` rows; E 0: the rows of x or dy) to a pass if it has to be looked at: its largest
// magnitudes are wanted or its rows cannot be read 16 bytes at a time and may be copied.  p and ld are then those of a
// padded copy in `room`.  Returns false where the products read single values: arrays too large for one buffer, fp32 rows
// too far apart for one, and weights whose rows are whole words from an address that is none.
template <typename S>
bool through(Pass& a, const void*& p, int64_t& ld, int64_t rows, int E, int n, uint32_t* most, Room& room) {
  const int cld = (int)copy_row(n, sizeof(S));
  const int64_t outer = std::max(1, E);
  const bool ok = vec_ok(p, rows, ld, sizeof(S), n);
  void* const copy = !ok && copies(E > 0, n, sizeof(S)) && rows * cld * (int64_t)sizeof(S) < (int64_t)kDropOffset
                         ? room.take(copy_bytes(rows * outer, n, sizeof(S)))
                         : nullptr;
  if (copy || most) {
    a.a[a.arrays++] = Pass::Array{p, rows * outer, ld, n, most, copy, cld};
    if (copy) {
      p = copy;
      ld = cld;
    }
  }
  return ok || copy;
}

template <typename T>
void launch_combine(const Args& g, const float* weight, T* y, const Dweight& d, hipStream_t st) {
  const int64_t n = g.T * ((g.H + 3) / 4);
  const unsigned grid = (unsigned)std::min<int64_t>((n + NT - 1) / NT, 1 << 20);
  combine_kernel<T><<<grid, NT, 0, st>>>(g.T, g.H, g.ldo, g.k, g.place, g.index, g.E, weight, g.o, y, d);
}

int check_dims(const FscExpertDims* d, bool q8) {
  FSC_CHECK_ARG(d != nullptr, "expert_mlp: null dims");
  FSC_CHECK_ARG(d->rows >= 0 && d->rows < (1ll << 31), "expert_mlp: rows must be below 2^31");
  FSC_CHECK_ARG(d->n_experts >= 1 && d->n_experts <= MAX_EXPERTS, "expert_mlp: 1 to 512 experts");
  FSC_CHECK_ARG(d->k >= 1 && d->k <= 64 && d->rows * d->k < (1ll << 31), "expert_mlp: 1 to 64 slots a row, fewer than 2^31 in all");
  FSC_CHECK_ARG(d->width >= 1 && d->width <= (1 << 17) && d->hidden >= 1 && d->hidden <= (1 << 17),
                "expert_mlp: width and hidden must be 1 to 2^17");
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
  return d.dtype == FSC_BF16 && (few(d) || M <= 32 * (int64_t)d.n_experts);
}
// bytes of a value of the arrays between the kernels
inline int64_t held_size(const FscExpertDims& d) {
  return d.dtype == FSC_I8 ? few(d) ? 4 : 1 : d.dtype == FSC_F32 || fine(d) ? 4 : 2;   // (few: h before its codes)
}

// Parts of a workspace, in bytes.
struct Space {
  int64_t h, o, da, hw, part, hs, most, split, pad, pad_end, total;
  Room room(char* ws) const { return Room{ws + pad, ws + pad_end}; }
};
// fp32 rows by tiles: two scaled parts an operand (three products, and one pass over the weights for their scales), or
// three parts (six products, no pass) where an expert has so few rows that the weights' bytes count for more.  Forward and
// all gradients of 640 x 640, us with two and three parts: 38 rows for each expert 193, 181; 62: 203, 191; 100: 241, 245; 250:
// 339, 364.
inline bool parts(const FscExpertDims& d) {
  return !few(d) && d.dtype == FSC_F32 && d.rows * d.k > 80 * (int64_t)d.n_experts;
}
inline int64_t pad_bytes(const FscExpertDims& d, int rows_arrays) {
  const int size = d.dtype == FSC_F32 ? 4 : d.dtype == FSC_BF16 ? 2 : 1;
  return copies_bytes(d.rows, d.width, d.hidden, d.n_experts, size, rows_arrays);
}
inline Space forward_space(const FscExpertDims& d) {
  const int64_t M = d.rows * d.k, ldf = ldf_of(d), size = held_size(d);
  Space s{};
  int64_t at = 0;
  s.h = at; at += align64(M * ldf * size);
  s.o = at; at += align64(M * ldo_of(d) * 4);
  if (parts(d)) {
    s.most = at; at += align64((d.rows + M + (int64_t)d.n_experts * (2 * d.hidden + d.width)) * 4);
  }
  if (d.dtype == FSC_I8) {
    s.hs = at; at += align64(M * (ldf / QG) * 4);
  }
  if (!few(d)) {
    s.pad = at; at += pad_bytes(d, 1); s.pad_end = at;
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
  if (parts(d)) {
    s.most = at; at += align64((d.rows + M + (int64_t)d.n_experts * (d.hidden + d.width)) * 4);
  }
  if (!few(d)) {
    s.pad = at; at += pad_bytes(d, 2); s.pad_end = at;
    // the two weight gradients use the same room, one after the other
    const int64_t si = most_shares(M, d.n_experts, weight_share(M, d.n_experts, (int)size, weight_tiles(d.width, 2 * ldf)));
    const int64_t so = most_shares(M, d.n_experts, weight_share(M, d.n_experts, (int)size, weight_tiles(ldf, d.width)));
    const int64_t n = (int64_t)d.hidden * d.width;
    s.split = at; at += align64(std::max(si > d.n_experts ? si * 2 * n : 0, so > d.n_experts ? so * n : 0) * 4);
  }
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
  g.li = d.width;
  g.lo = d.hidden;
  g.k_inv = ((1u << 20) + d.k - 1) / d.k;
  if (!few(d)) {
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
void forward(Args g, int tile, Room room, void* y, hipStream_t st) {
  if (!g.place) {
    if (one(g.M, g.E)) {
      if constexpr (KIND == I8) one_launch_q8(g, y, st);
      else one_launch<S>(g, y, st);
      return;
    }
    const bool vin = few_vec_ok(g.x, g.T, g.xs, sizeof(S), g.H) && few_vec_ok(g.w_in, 2 * g.F, g.H, sizeof(S), g.H);
    const bool vout = few_vec_ok(g.w_out, g.H, g.F, sizeof(S), g.F);
    if constexpr (KIND == I8) {
      few_launch_q8(g, vin, vout, st);
    } else {
      few_launch<S>(UP, g, vin, st);
      few_launch<S>(DOWN, g, vout, st);
    }
  } else {
    Pass a{};
    const bool vx = through<S>(a, g.x, g.xs, g.T, 0, g.H, g.xmost, room);
    const bool vin = through<S>(a, g.w_in, g.li, 2 * g.F, g.E, g.H, g.in_row, room) && vx;
    const bool vout = through<S>(a, g.w_out, g.lo, g.H, g.E, g.F, g.out_row, room);
    a.zero = g.hmost;
    a.zeros = g.hmost ? g.M : 0;
    launch_pass<S>(a, st);
    launch_rows<KIND, S, UP>(g, tile, vin, st);
    launch_rows<KIND, S, DOWN>(g, tile, vout, st);
  }
  using Y = std::conditional_t<KIND == I8, __bf16, S>;
  launch_combine<Y>(g, g.weight, (Y*)y, Dweight{}, st);
}

template <int KIND, typename S>
void backward(Args g, int tile, Room room, void* dx, float* dweight, hipStream_t st) {
  const bool by_slot = !g.place;
  bool vdy = vec_ok(g.dy, g.T, g.ds, sizeof(S), g.H), vx = vec_ok(g.x, g.T, g.xs, sizeof(S), g.H);
  bool vin = vec_ok(g.w_in, 2 * g.F, g.H, sizeof(S), g.H), vout = vec_ok(g.w_out, g.H, g.F, sizeof(S), g.F);
  if (by_slot) {
    const auto whole = [&](const void* p, int64_t rows, int64_t stride, int n) { return few_vec_ok(p, rows, stride, sizeof(S), n); };
    few_launch<S>(DH, g, whole(g.dy, g.T, g.ds, g.H) && whole(g.w_out, g.H, g.F, g.F), st);
    vin = whole(g.w_in, 2 * g.F, g.H, g.H);
  } else {
    Pass a{};
    if (g.out_col) {        // out_col, in_col and damost lie one after the other
      a.zero = g.out_col;
      a.zeros = (int64_t)g.E * (g.F + g.H) + g.M;
    }
    const void *w_in = g.w_in, *w_out = g.w_out;
    vdy = through<S>(a, g.dy, g.ds, g.T, 0, g.H, g.dymost, room);
    vout = through<S>(a, g.w_out, g.lo, g.H, g.E, g.F, nullptr, room);
    if (dx) vin = through<S>(a, g.w_in, g.li, 2 * g.F, g.E, g.H, nullptr, room);
    if (g.dw_in) vx = through<S>(a, g.x, g.xs, g.T, 0, g.H, nullptr, room);
    launch_pass<S>(a, st);
    if (g.out_col) {
      col_most_kernel<S><<<dim3((g.F + 63) / 64, (g.H + 63) / 64, g.E), NT, 0, st>>>((const S*)w_out, g.H, g.F, g.out_col);
      if (dx)
        col_most_kernel<S><<<dim3((g.H + 63) / 64, (2 * g.F + 63) / 64, g.E), NT, 0, st>>>((const S*)w_in, 2 * g.F, g.H, g.in_col);
    }
    launch_rows<KIND, S, DH>(g, tile, vdy && vout, st);
  }
  const Dweight d{g.M, by_slot ? few_parts(g.F, sizeof(S)) : (g.F + BN - 1) / BN, g.dwpart, dweight};
  if (dx) {
    if (by_slot) few_launch<S>(DX, g, vin, st);
    else launch_rows<KIND, S, DX>(g, tile, vin, st);
    launch_combine<S>(g, nullptr, (S*)dx, d, st);
  } else if (dweight) {
    dweight_kernel<<<(unsigned)((g.M + NT - 1) / NT), NT, 0, st>>>(d, g.place, g.index, g.E);
  }
  constexpr int WK = KIND == F32 ? X6 : KIND;
  if (by_slot) {
    if constexpr (KIND != BF16) {
      if (g.dw_in) launch_weights<WK, S, DWIN, true>(g, vx, st);
      if (g.dw_out) launch_weights<WK, S, DWOUT, true>(g, vdy, st);
    }
  } else {
    if (g.dw_in) launch_weights<WK, S, DWIN>(g, vx, st);
    if (g.dw_out) launch_weights<WK, S, DWOUT>(g, vdy, st);
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
  *plan_ints = few(*dims) ? 0 : fsc::experts::plan_ints(M, dims->n_experts, tile_rows(*dims));
  *saved_floats = dims->dtype == FSC_I8 ? 0 : M * 2 * ldf_of(*dims);
  *forward_bytes = forward_space(*dims).total;
  *backward_bytes = dims->dtype == FSC_I8 ? 0 : backward_space(*dims).total;
  return 0;
}

int fsc_expert_plan(const FscExpertDims* dims, const int32_t* index, int32_t* plan, hipStream_t stream) {
  using namespace fsc::experts;
  if (int rc = check_dims(dims, dims && dims->dtype == FSC_I8)) return rc;
  const int64_t M = dims->rows * dims->k;
  if (few(*dims)) return 0;       // the products find their rows themselves
  FSC_CHECK_ARG(plan && index, "expert_plan: null array");
  const int tile = tile_rows(*dims);
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
  FSC_CHECK_ARG(x && index && (plan || few(*dims)) && weight && w_in && w_out && workspace && y,
                "expert_mlp_forward: null array");
  FSC_CHECK_ARG(x_stride >= 0, "expert_mlp_forward: negative row stride");
  const int tile = tile_rows(*dims);
  const Plan p = plan_of(const_cast<int32_t*>(plan), M, dims->n_experts, tile);
  Args g = args_of(*dims, p);
  const Space s = forward_space(*dims);
  char* ws = (char*)workspace;
  g.index = index;
  g.x = x; g.xs = x_stride; g.weight = weight; g.w_in = w_in; g.w_out = w_out; g.a = saved;
  g.h = ws + s.h;
  g.o = (float*)(ws + s.o);
  if (parts(*dims)) {
    g.xmost = (uint32_t*)(ws + s.most);
    g.hmost = g.xmost + g.T;
    g.in_row = g.hmost + g.M;
    g.out_row = g.in_row + (int64_t)g.E * 2 * g.F;
  }
  if (parts(*dims)) forward<F32, float>(g, tile, s.room(ws), y, stream);
  else if (dims->dtype == FSC_F32) forward<X6, float>(g, tile, s.room(ws), y, stream);
  else if (fine(*dims)) forward<FINE, __bf16>(g, tile, s.room(ws), y, stream);
  else forward<BF16, __bf16>(g, tile, s.room(ws), y, stream);
  return fsc::check_launch("expert_mlp_forward") ? 2 : 0;
}

int fsc_expert_mlp_backward(const FscExpertDims* dims, int64_t x_stride, int64_t dy_stride, const void* dy,
                            const void* x, const int32_t* index, const int32_t* plan, const float* weight,
                            const void* w_in, const void* w_out, const float* saved, void* workspace, void* dx, float* dweight,
                            void* dw_in, void* dw_out, hipStream_t stream) {
  using namespace fsc::experts;
  if (int rc = check_dims(dims, false)) return rc;
  const int64_t M = dims->rows * dims->k;
  FSC_CHECK_ARG((plan || few(*dims)) && w_in && w_out, "expert_mlp_backward: null array");
  FSC_CHECK_ARG(M == 0 || (dy && x && index && weight && saved && workspace), "expert_mlp_backward: null array");
  FSC_CHECK_ARG(x_stride >= 0 && dy_stride >= 0, "expert_mlp_backward: negative row stride");
  const int tile = tile_rows(*dims);
  const Plan p = plan_of(const_cast<int32_t*>(plan), M, dims->n_experts, tile);
  Args g = args_of(*dims, p);
  const Space s = backward_space(*dims);
  char* ws = (char*)workspace;
  g.index = index;
  g.x = x; g.xs = x_stride; g.dy = dy; g.ds = dy_stride; g.weight = weight; g.w_in = w_in; g.w_out = w_out;
  g.a = const_cast<float*>(saved);
  g.o = (float*)(ws + s.o);
  g.da = ws + s.da;
  if (parts(*dims)) {
    g.dymost = (uint32_t*)(ws + s.most);
    g.out_col = g.dymost + g.T;
    g.in_col = g.out_col + (int64_t)g.E * g.F;
    g.damost = g.in_col + (int64_t)g.E * g.H;
  }
  g.hw = dw_out ? ws + s.hw : nullptr;
  g.dwpart = dweight ? (float*)(ws + s.part) : nullptr;
  g.dw_in = dw_in;
  g.dw_out = dw_out;
  g.dwsplit = (float*)(ws + s.split);
  if (M == 0) {              // no rows: zero weight gradients, written by the products' empty sums
    if (dims->dtype == FSC_F32) {
      if (dw_in) launch_weights<X6, float, DWIN, true>(g, false, stream);
      if (dw_out) launch_weights<X6, float, DWOUT, true>(g, false, stream);
    } else {
      if (dw_in) launch_weights<FINE, __bf16, DWIN, true>(g, false, stream);
      if (dw_out) launch_weights<FINE, __bf16, DWOUT, true>(g, false, stream);
    }
  } else if (parts(*dims)) {
    backward<F32, float>(g, tile, s.room(ws), dx, dweight, stream);
  } else if (dims->dtype == FSC_F32) {
    backward<X6, float>(g, tile, s.room(ws), dx, dweight, stream);
  } else if (fine(*dims)) {
    backward<FINE, __bf16>(g, tile, s.room(ws), dx, dweight, stream);
  } else {
    backward<BF16, __bf16>(g, tile, s.room(ws), dx, dweight, stream);
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
  FSC_CHECK_ARG(x && x_scale && index && (plan || few(*dims)) && weight && w_in && w_in_scale && w_out && w_out_scale && workspace && y,
                "expert_mlp_q8: null array");
  FSC_CHECK_ARG(x_stride >= 0, "expert_mlp_q8: negative row stride");
  const int tile = tile_rows(*dims);
  const Plan p = plan_of(const_cast<int32_t*>(plan), M, dims->n_experts, tile);
  Args g = args_of(*dims, p);
  const Space s = forward_space(*dims);
  char* ws = (char*)workspace;
  g.index = index;
  g.x = x; g.xs = x_stride; g.weight = weight; g.w_in = w_in; g.w_out = w_out;
  g.xscale = x_scale; g.in_scale = w_in_scale; g.out_scale = w_out_scale;
  g.h = ws + s.h;
  g.o = (float*)(ws + s.o);
  g.hscale = (float*)(ws + s.hs);
  forward<I8, int8_t>(g, tile, s.room(ws), y, stream);
  return fsc::check_launch("expert_mlp_q8") ? 2 : 0;
}

}  // extern "C"
