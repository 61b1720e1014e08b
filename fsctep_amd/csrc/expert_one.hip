// The experts' products of a handful of slots (a row or two as they arrive): no tile has two rows to share a weight, so
// every output is a dot product, and what counts is how many of them are on their way at once.
//
// up: a wave takes two hidden columns of one slot, their gate and up rows side by side: a lane reads 16 bytes of each
// row at every step, 1,024 bytes of a row a wave, and the four sums meet by shuffles.  down: a wave takes two columns of
// one row and goes through the row's k experts, whose weighted sum it writes: y needs no pass of its own.  Blocks of four
// waves; 640 x 640, k = 2: 160 blocks up, 80 down.  Sums in 32 bits.  One row of 640, two of eight experts, fp32: up 4.0, down
// 4.4 us (10 MB of weights; the tiles of 16 rows of the few-rows kernels and their pass over the rows 6.5 + 4.4 + 2.5 us).
//
// 8 bits: 16 lanes a weight row, 16 bytes a lane, v_dot4_i32_i8; up takes a whole group of 128 hidden columns a block of
// 16 waves, since the group's codes share a unit.  That is five blocks for a slot of 640 hidden columns, on ten CUs for one
// row: up 6.6, down 4.7 us, slower than fp32's 4.1 and 4.6 with four times the bytes.
#include <type_traits>

#include "common.h"
#include "expert_tiles.h"

namespace fsc {
namespace experts {

constexpr int OT = 256;             // four waves

__device__ __forceinline__ float wave_total(float v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}

// 16 bytes from p, of any alignment the hardware's loads take: a row of any width is read 16 bytes at a time.
template <int V, typename T>
__device__ __forceinline__ void load16(const T* p, float (&v)[V]) {
  if constexpr (V == 1) {
    v[0] = to_f(*p);
  } else {
    T t[V];
    __builtin_memcpy(t, p, sizeof(t));
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = to_f(t[i]);
  }
}

// Sums of NR weight rows (n values each) with x, lane by lane: 16 bytes of a weight row (V values) a step where a row
// has them (WIDE), single values elsewhere.  U steps' loads are on their way together.  The lane at the end of a row
// reads the row's last V values and adds those that no other lane has.
template <typename S, typename X, int NR, bool WIDE>
__device__ __forceinline__ void dots(const S* const (&w)[NR], const X* x, int n, float (&sum)[NR]) {
  constexpr int V = WIDE ? 16 / sizeof(S) : 1, U = WIDE ? 4 : 1;
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int i = 0; i < NR; ++i) sum[i] = 0.f;
  for (int k0 = 0; k0 < n; k0 += 64 * V * U) {
    float a[U][NR][V], b[U][V];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int at = min(k0 + (64 * u + lane) * V, n - V);
      if (k0 + 64 * u * V < n) {                         // the same for the whole wave
        load16<V>(x + at, b[u]);
#pragma unroll
        for (int i = 0; i < NR; ++i) load16<V>(w[i] + at, a[u][i]);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = k0 + (64 * u + lane) * V, skip = k - (n - V);
      if (skip <= 0) {
#pragma unroll
        for (int i = 0; i < NR; ++i)
#pragma unroll
          for (int j = 0; j < V; ++j) sum[i] += a[u][i][j] * b[u][j];
      } else if (skip < V) {
#pragma unroll
        for (int i = 0; i < NR; ++i)
#pragma unroll
          for (int j = 0; j < V; ++j)
            if (j >= skip) sum[i] += a[u][i][j] * b[u][j];
      }
    }
  }
}

// a = W_in[e] x of two hidden columns, h = silu(a_gate) a_up; columns up to the padded row length, zeros past the last.
template <typename S, bool WIDE>
__global__ __launch_bounds__(OT) void one_up_kernel(Args g) {
  const int slot = blockIdx.y, e = g.index[slot];
  if (e < 0 || e >= g.E) return;
  const int n0 = (blockIdx.x * (OT / 64) + (threadIdx.x >> 6)) * 2;
  if (n0 >= g.ldf) return;
  // columns past the last: the last one's rows, and zeros stored
  const int c0 = min(n0, g.F - 1), c1 = min(n0 + 1, g.F - 1);
  const S* m = (const S*)g.w_in + (int64_t)e * 2 * g.F * g.H;
  const S* const w[4] = {m + (int64_t)c0 * g.H, m + (int64_t)c1 * g.H, m + (int64_t)(g.F + c0) * g.H,
                         m + (int64_t)(g.F + c1) * g.H};
  float s[4];
  dots<S, S, 4, WIDE>(w, (const S*)g.x + few_row(g, slot) * g.xs, g.H, s);
#pragma unroll
  for (int i = 0; i < 4; ++i) s[i] = wave_total(s[i]);
  const int lane = threadIdx.x & 63;
  if (lane < 2) {
    const int n = n0 + lane;
    const bool in = n < g.F;
    const float ga = in ? s[lane] : 0.f, up = in ? s[2 + lane] : 0.f;
    if (g.a) {
      g.a[(int64_t)slot * 2 * g.ldf + n] = ga;
      g.a[(int64_t)slot * 2 * g.ldf + g.ldf + n] = up;
    }
    ((float*)g.h)[(int64_t)slot * g.ldf + n] = ga * sigmoid(ga) * up;
  }
}

// y_t = sum_j weight_tj (W_out[e_j] h_tj) of two columns, in the order of j.
template <typename S, bool WIDE>
__global__ __launch_bounds__(OT) void one_down_kernel(Args g, S* y) {
  const int64_t t = blockIdx.y;
  const int n0 = (blockIdx.x * (OT / 64) + (threadIdx.x >> 6)) * 2;
  if (n0 >= g.H) return;
  const int c1 = min(n0 + 1, g.H - 1);
  float y0 = 0.f, y1 = 0.f;
  for (int j = 0; j < g.k; ++j) {
    const int64_t slot = t * g.k + j;
    const int e = g.index[slot];
    if (e < 0 || e >= g.E) continue;
    const S* m = (const S*)g.w_out + (int64_t)e * g.H * g.F;
    const S* const w[2] = {m + (int64_t)n0 * g.F, m + (int64_t)c1 * g.F};
    float s[2];
    dots<S, float, 2, WIDE>(w, (const float*)g.h + slot * g.ldf, g.F, s);
    const float u = g.weight[slot];
    y0 += u * wave_total(s[0]);
    y1 += u * wave_total(s[1]);
  }
  const int lane = threadIdx.x & 63;
  if (lane < 2 && n0 + lane < g.H) y[t * g.H + n0 + lane] = from_f<S>(lane ? y1 : y0);
}

// ---------------------------------------------------------------- 8 bits
// 16 bytes of a row of n from k on, of any alignment.  At the row's end its last 16, with zeros for those before k where
// CUT; a row of fewer than 16 (not WIDE) byte by byte.
template <bool WIDE, bool CUT>
__device__ __forceinline__ i4v bytes16(const int8_t* p, int k, int n) {
  if constexpr (WIDE) {
    i4v v;
    __builtin_memcpy(&v, p + min(k, n - 16), 16);
    if (CUT && k + 16 > n) {
      const int skip = k + 16 - n;                       // 16 and more: nothing is left
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int z = min(max(skip - 4 * i, 0), 4);      // bytes of the word to clear
        v[i] = z >= 4 ? 0 : (int)((uint32_t)v[i] >> (8 * z) << (8 * z));
      }
    }
    return v;
  }
  uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 15; ++i) w[i / 4] |= (k + i < n ? (uint32_t)(uint8_t)p[min(k + i, n - 1)] : 0u) << (8 * (i % 4));
  return i4v{(int)w[0], (int)w[1], (int)w[2], (int)w[3]};
}
__device__ __forceinline__ int dot16(const i4v& a, const i4v& b, int c) {
#pragma unroll
  for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_sdot4(a[i], b[i], c, false);
  return c;
}

// A block a slot and a group; 16 waves of eight columns, a wave's four quarters the gate and up rows of two.
template <bool WIDE>
__global__ __launch_bounds__(1024) void one_up_q8_kernel(Args g) {
  __shared__ float hs[QG];
  const int slot = blockIdx.y, grp = blockIdx.x, e = g.index[slot];
  if (e < 0 || e >= g.E) return;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, r = lane & 15, part = lane >> 4;
  const int64_t row = few_row(g, slot);
  const int8_t* x = (const int8_t*)g.x + row * g.xs;
  const float xs = g.xscale[row];
  int sum[4] = {0, 0, 0, 0};
  int64_t wr[4];                                         // weight row of step i: column 8 wave + 2 i + part / 2
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int n = min(grp * QG + 8 * wave + 2 * i + (part >> 1), g.F - 1);
    wr[i] = (int64_t)e * 2 * g.F + (part & 1 ? g.F : 0) + n;
  }
  for (int k0 = 0; k0 < g.H; k0 += 1024) {
    i4v a[4][4], b[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int k = k0 + 256 * u + 16 * r;
      b[u] = bytes16<WIDE, true>(x, k, g.H);
#pragma unroll
      for (int i = 0; i < 4; ++i) a[u][i] = bytes16<WIDE, false>((const int8_t*)g.w_in + wr[i] * g.H, k, g.H);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) sum[i] = dot16(a[u][i], b[u], sum[i]);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int off = 8; off > 0; off >>= 1) sum[i] += __shfl_xor(sum[i], off, 64);
    const int c = 8 * wave + 2 * i + (part >> 1);
    const float v = grp * QG + c < g.F ? (float)sum[i] * (xs * g.in_scale[wr[i]]) : 0.f;
    const float up = __shfl_xor(v, 16, 64);
    if (r == 0 && !(part & 1)) hs[c] = v * sigmoid(v) * up;
  }
  __syncthreads();
  if (wave == 0) {
    const f4 h = ld4(hs + 4 * (lane & 31));
    uint32_t top = most4(h);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, off, 64));
    const float most = __uint_as_float(top), inv = most > 0.f ? 127.f / most : 0.f;
    if (lane < 32) *reinterpret_cast<uint32_t*>((int8_t*)g.h + (int64_t)slot * g.ldf + grp * QG + 4 * lane) = codes4(h, inv);
    if (lane == 0) g.hscale[(int64_t)slot * (g.ldf / QG) + grp] = most / 127.f;
  }
}

// A wave four columns of a row, 16 lanes each; eight lanes share a group of h.
template <bool WIDE>
__global__ __launch_bounds__(OT) void one_down_q8_kernel(Args g, __bf16* y) {
  const int64_t t = blockIdx.y;
  const int lane = threadIdx.x & 63, r = lane & 15;
  const int n = (blockIdx.x * (OT / 64) + (threadIdx.x >> 6)) * 4 + (lane >> 4), c = min(n, g.H - 1), ng = g.ldf / QG;
  float total = 0.f;
  for (int j = 0; j < g.k; ++j) {
    const int64_t slot = t * g.k + j;
    const int e = g.index[slot];
    if (e < 0 || e >= g.E) continue;
    const int8_t* h = (const int8_t*)g.h + slot * g.ldf;
    const int64_t wr = (int64_t)e * g.H + c;
    const int8_t* w = (const int8_t*)g.w_out + wr * g.F;
    float s = 0.f;
    for (int k0 = 0; k0 < g.F; k0 += 1024) {
      i4v a[4], b[4];
      float u[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int k = k0 + 256 * i + 16 * r;
        a[i] = bytes16<WIDE, true>(w, k, g.F);
        // h at the place of w's bytes (its row is whole groups, zeros past F)
        const int at = WIDE ? min(k, g.F - 16) : min(k, g.ldf - 16);
        __builtin_memcpy(&b[i], h + at, 16);
        u[i] = g.hscale[slot * ng + min(k, g.ldf - 1) / QG];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (k0 + 256 * i + 16 * r < g.F) s += (float)dot16(a[i], b[i], 0) * u[i];
    }
#pragma unroll
    for (int off = 8; off > 0; off >>= 1) s += __shfl_xor(s, off, 64);
    total += g.weight[slot] * (s * g.out_scale[wr]);
  }
  if (r == 0 && n < g.H) y[t * g.H + n] = (__bf16)total;
}

template <typename S>
void one_launch(const Args& g, void* y, hipStream_t st) {
  constexpr int V = 16 / sizeof(S);
  const dim3 up((g.ldf + 7) / 8, (unsigned)g.M), down((g.H + 7) / 8, (unsigned)g.T);
  if (g.H >= V) one_up_kernel<S, true><<<up, OT, 0, st>>>(g);
  else one_up_kernel<S, false><<<up, OT, 0, st>>>(g);
  if (g.F >= V) one_down_kernel<S, true><<<down, OT, 0, st>>>(g, (S*)y);
  else one_down_kernel<S, false><<<down, OT, 0, st>>>(g, (S*)y);
}
template void one_launch<float>(const Args&, void*, hipStream_t);
template void one_launch<__bf16>(const Args&, void*, hipStream_t);

void one_launch_q8(const Args& g, void* y, hipStream_t st) {
  const dim3 up(g.ldf / QG, (unsigned)g.M), down((g.H + 15) / 16, (unsigned)g.T);
  if (g.H >= 16) one_up_q8_kernel<true><<<up, 1024, 0, st>>>(g);
  else one_up_q8_kernel<false><<<up, 1024, 0, st>>>(g);
  if (g.F >= 16) one_down_q8_kernel<true><<<down, OT, 0, st>>>(g, (__bf16*)y);
  else one_down_q8_kernel<false><<<down, OT, 0, st>>>(g, (__bf16*)y);
}

}  // namespace experts
}  // namespace fsc
