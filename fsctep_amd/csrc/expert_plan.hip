// Rows by expert: a stable counting sort of the rows' slots (row t's j-th expert is slot t k + j), and the list of
// row tiles that the products run over.  Slots with an expert outside [0, E) stand in no tile.
//
//   offsets [E + 1]   first sorted position of each expert
//   slot_of [M]       slot at each sorted position          (M = T k)
//   row_of  [M]       its row, slot / k
//   place   [M]       sorted position of each slot, -1 for a slot with no expert
//   tiles   [2 n]     (expert, first sorted position) of each tile of `tile` rows, expert -1 past the last one
//                     (n = ceil(M / tile) + min(E, M) bounds their number)
//   counts  [blocks E] rows of each expert before each block of slots, with many slots
//
// Bound by latency (4 bytes in, 16 out for each slot): up to 4,096 slots one launch, 3 to 5 us; above that three, 17 us at
// 20,000 slots and 20 us at 100,000 (one block alone: 33 and 146 us).
#include <algorithm>

#include "common.h"
#include "expert_types.h"
#include "expert_plan.h"
#include "fsctep.h"

namespace fsc {
namespace experts {

constexpr int PT = 1024;            // threads: 16 waves
constexpr int PW = PT / 64;
// Slots of a block; up to so many, one block does all.
constexpr int BLOCK = 4096;

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

// Wave w of a block takes the w-th sixteenth of the block's slots: its counts by expert.
__device__ __forceinline__ void count_slots(const int32_t* __restrict__ index, int64_t b0, int64_t b1, int E,
                                            int (&cnt)[PW][MAX_EXPERTS], int64_t& s0, int64_t& s1) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  for (int i = threadIdx.x; i < PW * MAX_EXPERTS; i += PT) (&cnt[0][0])[i] = 0;
  __syncthreads();
  const int64_t per = ((b1 - b0 + PW - 1) / PW + 63) / 64 * 64;
  s0 = std::min<int64_t>(b1, b0 + wave * per);
  s1 = std::min<int64_t>(b1, s0 + per);
  for (int64_t s = s0 + lane; s < s1; s += 64) {
    const int e = index[s];
    if (e >= 0 && e < E) atomicAdd(&cnt[wave][e], 1);   // counts: the order of the additions does not matter
  }
  __syncthreads();
}

// The slots s0 .. s1 of a wave to their positions: expert e's begin at base[e] + cnt[e], in order.
__device__ __forceinline__ void place_slots(const int32_t* __restrict__ index, int64_t s0, int64_t s1, int E, int k,
                                            const int* base, int* cnt, const Plan& p) {
  const int lane = threadIdx.x & 63;
  for (int64_t b = s0; b < s1; b += 64) {
    const int64_t s = b + lane;
    const int e = s < s1 ? index[s] : -1;
    const bool ok = e >= 0 && e < E;
    const uint64_t m = peers(e, ok);
    int at = -1;
    if (ok) at = base[e] + cnt[e] + __popcll(m & ((1ull << lane) - 1));
    wave_sync();
    // the last lane of each expert moves its counter on
    if (ok && (m >> lane) == 1ull) cnt[e] += __popcll(m);
    wave_sync();
    if (s < s1) p.place[s] = at;
    if (ok) {
      p.slot_of[at] = (int32_t)s;
      p.row_of[at] = (int32_t)s / k;
    }
  }
}

// From total[e] (rows of expert e): offsets, also left in total, and the tiles.  One block.
__device__ __forceinline__ void lay_out(int E, int tile, const Plan& p, int* total, int* first) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
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
        p.offsets[e] = rows + a - c;
        total[e] = rows + a - c;
        first[e] = nt + b - tb;
      }
      rows += __shfl(a, 63, 64);
      nt += __shfl(b, 63, 64);
    }
    if (lane == 0) {
      p.offsets[E] = rows;
      total[E] = rows;
      first[E] = nt;
    }
  }
  __syncthreads();
  for (int e = wave; e < E; e += PW)
    for (int t = first[e] + lane; t < first[e + 1]; t += 64) {
      p.tiles[2 * t] = e;
      p.tiles[2 * t + 1] = total[e] + (t - first[e]) * tile;
    }
  for (int t = first[E] + threadIdx.x; t < p.n_tiles; t += PT) {
    p.tiles[2 * t] = -1;
    p.tiles[2 * t + 1] = 0;
  }
}

// All slots by one block.
__global__ __launch_bounds__(PT) void plan_kernel(int64_t M, int E, int k, int tile, const int32_t* __restrict__ index,
                                                  Plan p) {
  __shared__ int cnt[PW][MAX_EXPERTS];
  __shared__ int total[MAX_EXPERTS + 1], first[MAX_EXPERTS + 1];
  int64_t s0, s1;
  count_slots(index, 0, M, E, cnt, s0, s1);
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
  lay_out(E, tile, p, total, first);
  place_slots(index, s0, s1, E, k, total, cnt[threadIdx.x >> 6], p);
}

// Many slots: counts by blocks of BLOCK slots, the scan over blocks and experts, the places.
__global__ __launch_bounds__(PT) void count_kernel(int64_t M, int E, const int32_t* __restrict__ index, Plan p) {
  __shared__ int cnt[PW][MAX_EXPERTS];
  int64_t s0, s1;
  const int64_t b0 = (int64_t)blockIdx.x * BLOCK;
  count_slots(index, b0, std::min<int64_t>(M, b0 + BLOCK), E, cnt, s0, s1);
  for (int e = threadIdx.x; e < E; e += PT) {
    int t = 0;
    for (int w = 0; w < PW; ++w) t += cnt[w][e];
    p.counts[(int64_t)blockIdx.x * E + e] = t;
  }
}
__global__ __launch_bounds__(PT) void scan_kernel(int blocks, int E, int tile, Plan p) {
  __shared__ int total[MAX_EXPERTS + 1], first[MAX_EXPERTS + 1];
  for (int e = threadIdx.x; e < E; e += PT) {
    int t = 0;
#pragma unroll 8
    for (int b = 0; b < blocks; ++b) {
      const int c = p.counts[(int64_t)b * E + e];
      p.counts[(int64_t)b * E + e] = t;
      t += c;
    }
    total[e] = t;
  }
  __syncthreads();
  lay_out(E, tile, p, total, first);
}
__global__ __launch_bounds__(PT) void place_kernel(int64_t M, int E, int k, const int32_t* __restrict__ index, Plan p) {
  __shared__ int cnt[PW][MAX_EXPERTS];
  __shared__ int base[MAX_EXPERTS];
  int64_t s0, s1;
  const int64_t b0 = (int64_t)blockIdx.x * BLOCK;
  count_slots(index, b0, std::min<int64_t>(M, b0 + BLOCK), E, cnt, s0, s1);
  for (int e = threadIdx.x; e < E; e += PT) {
    int t = 0;
    for (int w = 0; w < PW; ++w) {
      const int c = cnt[w][e];
      cnt[w][e] = t;
      t += c;
    }
    base[e] = p.offsets[e] + p.counts[(int64_t)blockIdx.x * E + e];
  }
  __syncthreads();
  place_slots(index, s0, s1, E, k, base, cnt[threadIdx.x >> 6], p);
}

inline int64_t blocks_of(int64_t M) { return M > BLOCK ? (M + BLOCK - 1) / BLOCK : 0; }

Plan plan_of(int32_t* buf, int64_t M, int E, int tile) {
  Plan p;
  p.offsets = buf;
  p.slot_of = p.offsets + E + 1;
  p.row_of = p.slot_of + M;
  p.place = p.row_of + M;
  p.tiles = p.place + M;
  p.counts = p.tiles + 2 * ((M + tile - 1) / tile + std::min<int64_t>(E, M));
  p.n_tiles = (int)((M + tile - 1) / tile + std::min<int64_t>(E, M));
  return p;
}

int64_t plan_ints(int64_t M, int E, int tile) {
  return (E + 1) + 3 * M + 2 * ((M + tile - 1) / tile + std::min<int64_t>(E, M)) + blocks_of(M) * E;
}

void launch_plan(const Plan& p, int64_t M, int E, int k, int tile, const int32_t* index, hipStream_t st) {
  const int64_t blocks = blocks_of(M);
  if (blocks == 0) {
    plan_kernel<<<1, PT, 0, st>>>(M, E, k, tile, index, p);
    return;
  }
  count_kernel<<<(unsigned)blocks, PT, 0, st>>>(M, E, index, p);
  scan_kernel<<<1, PT, 0, st>>>((int)blocks, E, tile, p);
  place_kernel<<<(unsigned)blocks, PT, 0, st>>>(M, E, k, index, p);
}

}  // namespace experts
}  // namespace fsc
