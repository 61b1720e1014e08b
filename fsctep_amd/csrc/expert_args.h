// Arguments shared by the kernels of the experts' products (expert_mlp.hip: by tiles, expert_few.hip: few rows).
#pragma once

#include <hip/hip_runtime.h>
#include <cstdint>

namespace fsc {
namespace experts {

enum Mode { UP = 0, DOWN = 1, DH = 2, DX = 3, DWIN = 4, DWOUT = 5 };

constexpr int QG = 128;          // hidden columns that share a unit in 8 bits
constexpr int FEW_SLOTS = 1024;  // slots that a block of the few-rows kernels looks through

struct Args {
  // sizes: rows T, slots M = T k, width H, hidden F (row length ldf in the arrays between), experts E
  int64_t T, M;
  int H, F, ldf, ldo, E, k, n_tiles;
  int64_t xs, ds;                   // row strides of x and dy, in elements
  int64_t li, lo;                   // row lengths of w_in and w_out (H and F, or padded to whole chunks)
  const int32_t *index;             // [M]
  uint32_t k_inv;                   // ceil(2^20 / k): slot / k = slot k_inv / 2^20 for the few-rows slots (below 1,024)
  const int32_t *offsets, *slot_of, *row_of, *tiles, *place;   // the rows by expert; null where there are few rows
  const void *x, *w_in, *w_out, *dy;
  const float* weight;              // [M]
  // arrays between the kernels, a row for each sorted position, or for each slot where there are few rows
  float* a;                         // [M][2 ldf] gate and up before the activation (null: not kept)
  void* h;                          // [M][ldf]
  float* o;                         // [M][ldo] products, before a row's experts are combined
  void* da;                         // [M][2 ldf]
  void* hw;                         // [M][ldf] weight h, for dw_out (null: not wanted)
  float* dwpart;                    // [column tiles of dh][M] partial dweight
  void *dw_in, *dw_out;
  float* dwsplit;                   // [shares] partial weight gradients of the experts with more than one share
  int share;                        // positions of a share (an expert's positions are dealt into shares of so many)
  // fp32 products: largest magnitudes (bits) of the rows of x and dy [T], of h and da [M], of the weights along each
  // output: rows of w_in [E][2 F] and w_out [E][H] (up, down), columns of w_out [E][F] and w_in [E][H] (dh, dx)
  uint32_t *xmost, *dymost, *hmost, *damost, *in_row, *out_row, *out_col, *in_col;
  // 8 bits: scales of x's rows, of the weights' rows and of h's groups [M][ldf / QG]
  const float *xscale, *in_scale, *out_scale;
  float* hscale;
};

// Few rows: S is float or __bf16 (the caller's arrays; h, da and hw are fp32), MODE UP, DOWN, DH or DX.
template <typename S>
void few_launch(int mode, const Args& g, bool vec, hipStream_t st);
// Columns of dh that share a partial dweight there.
int few_parts(int F, int size);
// Few rows in 8 bits: up (h in 32 bits) and down (from its codes).
void few_launch_q8(const Args& g, bool vin, bool vout, hipStream_t st);
// A handful of slots (expert_one.hip): up, down and the rows from their experts.
template <typename S>
void one_launch(const Args& g, void* y, hipStream_t st);
void one_launch_q8(const Args& g, void* y, hipStream_t st);

// 1 / (1 + 2^(-v log2 e)) by the hardware's exponential and reciprocal: within 1e-7 |v| of the value where it is
// small, within 1e-7 elsewhere; four instructions where expf and a division take about forty.
__device__ __forceinline__ float sigmoid(float v) {
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(v * -1.44269504f));
}

// n of four values to p, by one access where they are four and aligned
__device__ __forceinline__ void store4(float* p, const f4& v, int n) {
  if (n >= 4 && (uintptr_t)p % 16 == 0) st4(p, v);
  else
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < n) p[j] = v[j];
}
__device__ __forceinline__ void store4(__bf16* p, const f4& v, int n) {
  typedef __bf16 bf4 __attribute__((ext_vector_type(4)));
  if (n >= 4 && (uintptr_t)p % 8 == 0) *reinterpret_cast<bf4*>(p) = bf4{(__bf16)v.x, (__bf16)v.y, (__bf16)v.z, (__bf16)v.w};
  else
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < n) p[j] = (__bf16)v[j];
}

// The expert of a block of the few-rows kernels, or -1: experts in order, or, with fewer slots than experts, the
// expert of the b-th slot if no earlier slot has it.  Block-uniform; every thread calls it.
__device__ __forceinline__ int few_expert(const Args& g, int b) {
  if (g.M >= g.E) return b;
  const int e = g.index[b];
  if (e < 0 || e >= g.E) return -1;
  const int lane = threadIdx.x & 63;
  bool earlier = false;
  for (int s = lane; s < b; s += 64) earlier |= g.index[s] == e;
  return __ballot(earlier) ? -1 : e;
}
inline int few_blocks(const Args& g) { return (int)(g.M < g.E ? g.M : g.E); }
__device__ __forceinline__ int64_t few_row(const Args& g, int slot) { return (uint32_t)slot * g.k_inv >> 20; }

// The lane's expert among the first 64 slots (-1 past the last).  Loaded before the weights: loads return in order.
__device__ __forceinline__ int few_first(const Args& g) {
  const int lane = threadIdx.x & 63;
  return lane < g.M ? g.index[lane] : -1;
}

// The slots of expert e in order into list (FEW_SLOTS entries), `first` from few_first; returns their number.  Every
// wave of the block does the same work and writes the same values; the caller synchronises before it reads them.
__device__ __forceinline__ int few_slots(const Args& g, int e, int first, int16_t* list) {
  const int lane = threadIdx.x & 63;
  int n = 0;
  for (int s0 = 0; s0 < g.M; s0 += 64) {
    const int s = s0 + lane;
    if (s0) first = s < g.M ? g.index[s] : -1;
    const bool mine = first == e;
    const uint64_t m = __ballot(mine);
    if (mine) list[n + __popcll(m & ((1ull << lane) - 1))] = (int16_t)s;
    n += __popcll(m);
  }
  return n;
}

}  // namespace experts
}  // namespace fsc
