// Rows by expert: a stable counting sort of the rows' slots (row t's j-th expert is slot t k + j), and the list of
// row tiles that the products run over.  Slots with an expert outside [0, E) stand in no tile.
//
//   offsets [E + 1]   first sorted position of each expert
//   slot_of [M]       slot at each sorted position          (M = T k)
//   row_of  [M]       its row, slot / k
//   place   [M]       sorted position of each slot, -1 for a slot with no expert
//   tiles   [2 n]     (expert, first sorted position) of each tile of `tile` rows, expert -1 past the last one
//                     (n = ceil(M / tile) + min(E, M) bounds their number)
#include <algorithm>

#include "common.h"
#include "expert_plan.h"
#include "fsctep.h"

namespace fsc {
namespace experts {

constexpr int PT = 1024;            // threads: 16 waves
constexpr int PW = PT / 64;

// The lanes of the wave with the same expert as this one (bits of lanes without an expert clear).
__device__ __forceinline__ uint64_t peers(int e, bool ok) {
  uint64_t m = __ballot(ok);
#pragma unroll
  for (int b = 0; b < 9; ++b) {
    const uint64_t v = __ballot(e >> b & 1);
    m &= (e >> b & 1) ? v : ~v;
  }
  return m;
}

// One block: wave w takes the w-th sixteenth of the slots, counts them by expert, and after a scan over (expert,
// wave) ranks them in order.
__global__ __launch_bounds__(PT) void plan_kernel(int64_t M, int E, int k, int tile, int n_tiles,
                                                  const int32_t* __restrict__ index, int32_t* __restrict__ offsets,
                                                  int32_t* __restrict__ slot_of, int32_t* __restrict__ row_of,
                                                  int32_t* __restrict__ place,
                                                  int32_t* __restrict__ tiles) {
  __shared__ int cnt[PW][MAX_EXPERTS];
  __shared__ int total[MAX_EXPERTS + 1], first[MAX_EXPERTS + 1];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  for (int i = threadIdx.x; i < PW * MAX_EXPERTS; i += PT) (&cnt[0][0])[i] = 0;
  __syncthreads();
  const int64_t per = ((M + PW - 1) / PW + 63) / 64 * 64, s0 = std::min<int64_t>(M, wave * per),
                s1 = std::min<int64_t>(M, s0 + per);
  for (int64_t s = s0 + lane; s < s1; s += 64) {
    const int e = index[s];
    if (e >= 0 && e < E) atomicAdd(&cnt[wave][e], 1);   // counts: the order of the additions does not matter
  }
  __syncthreads();
  for (int e = threadIdx.x; e < E; e += PT) {
    int t = 0;
    for (int w = 0; w < PW; ++w) {
      const int c = cnt[w][e];
      cnt[w][e] = t;
      t += c;
    }
    total[e] = t;
  }
  __syncthreads();
  if (wave == 0) {                                       // exclusive scans over the experts: rows and tiles
    int rows = 0, nt = 0;
    for (int e0 = 0; e0 < E; e0 += 64) {
      const int e = e0 + lane, c = e < E ? total[e] : 0;
      int a = c, b = (c + tile - 1) / tile;
      const int tb = b;
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) {
        const int ua = __shfl_up(a, off, 64), ub = __shfl_up(b, off, 64);
        if (lane >= off) { a += ua; b += ub; }
      }
      if (e < E) {
        offsets[e] = rows + a - c;
        total[e] = rows + a - c;
        first[e] = nt + b - tb;
      }
      rows += __shfl(a, 63, 64);
      nt += __shfl(b, 63, 64);
    }
    if (lane == 0) {
      offsets[E] = rows;
      total[E] = rows;
      first[E] = nt;
    }
  }
  __syncthreads();
  for (int e = wave; e < E; e += PW)
    for (int t = first[e] + lane; t < first[e + 1]; t += 64) {
      tiles[2 * t] = e;
      tiles[2 * t + 1] = total[e] + (t - first[e]) * tile;
    }
  for (int t = first[E] + threadIdx.x; t < n_tiles; t += PT) {
    tiles[2 * t] = -1;
    tiles[2 * t + 1] = 0;
  }
  for (int64_t b = s0; b < s1; b += 64) {
    const int64_t s = b + lane;
    const int e = s < s1 ? index[s] : -1;
    const bool ok = e >= 0 && e < E;
    const uint64_t m = peers(e, ok);
    int at = -1;
    if (ok) at = total[e] + cnt[wave][e] + __popcll(m & ((1ull << lane) - 1));
    // the last lane of each expert moves its counter on (one wave: the reads above come first)
    if (ok && (m >> lane) == 1ull) cnt[wave][e] += __popcll(m);
    if (s < s1) place[s] = at;
    if (ok) {
      slot_of[at] = (int32_t)s;
      row_of[at] = (int32_t)s / k;
    }
  }
}

Plan plan_of(int32_t* buf, int64_t M, int E, int tile) {
  Plan p;
  p.offsets = buf;
  p.slot_of = p.offsets + E + 1;
  p.row_of = p.slot_of + M;
  p.place = p.row_of + M;
  p.tiles = p.place + M;
  p.n_tiles = (int)((M + tile - 1) / tile + std::min<int64_t>(E, M));
  return p;
}

int64_t plan_ints(int64_t M, int E, int tile) {
  return (E + 1) + 3 * M + 2 * ((M + tile - 1) / tile + std::min<int64_t>(E, M));
}

void launch_plan(const Plan& p, int64_t M, int E, int k, int tile, const int32_t* index, hipStream_t st) {
  plan_kernel<<<1, PT, 0, st>>>(M, E, k, tile, p.n_tiles, index, p.offsets, p.slot_of, p.row_of, p.place, p.tiles);
}

}  // namespace experts
}  // namespace fsc
