// How the weight gradients of the experts' products deal out their work: arithmetic on sizes alone, from which the host
// takes launches and workspace and the kernels take their place.
#pragma once

#include <algorithm>
#include <cstdint>

namespace fsc {
namespace experts {

constexpr int WEIGHT_TILE = 128;   // rows and columns of a tile of a weight gradient
constexpr int MANY_TILES = 64;

// Tiles of a weight gradient, and the positions of a share: so many that about 1,024 (fp32) or 512 tiles of shares run
// whatever rows the experts have, of at least 128 (fp32: six products) or 256 positions, which outweigh writing and summing
// them, and of 1,024 or 2,048 where the experts' tiles fill the chip without it and only the fullest experts are worth
// dealing out.  Routing is uneven: 10,000 rows of 640, two of 16 experts, the fullest with three times the mean: forward
// and all gradients 979 us against 1,553 with an expert's positions in one block (bf16 409 against 534).
constexpr int64_t weight_tiles(int64_t na, int64_t nb) {
  return ((na + WEIGHT_TILE - 1) / WEIGHT_TILE) * ((nb + WEIGHT_TILE - 1) / WEIGHT_TILE);
}
constexpr int weight_share(int64_t M, int E, int size, int64_t tiles) {
  const int64_t least = (E * tiles >= 512 ? 1024 : 128) * (size == 4 ? 1 : 2);
  const int64_t share = std::max(least, M * tiles / (size == 4 ? 1024 : 512));
  return (int)std::min<int64_t>((share + 63) / 64 * 64, 1 << 30);
}
// Shares that M positions of E experts can make: an expert of c positions makes 1 + (c - 1) / share, one of none makes one.
// E exactly where no expert can have more than a share (M <= share).
constexpr int64_t most_shares(int64_t M, int E, int share) { return E + (M > 0 ? (M - 1) / share : 0); }
constexpr bool one_share_each(int64_t M, int share) { return M <= share; }

// Blocks of a weight gradient of `shares` shares.  Workgroup w runs on XCD w % 8.  Where every expert is one share, and
// with many tiles, every XCD takes a run of each share's tiles, whatever the shares' sizes; with few tiles a run of all
// tiles of all shares, which are then about equal.
constexpr bool runs_by_share(bool one_each, int64_t tiles) { return one_each || tiles >= MANY_TILES; }
constexpr int64_t weight_blocks(int64_t shares, int64_t tiles, bool by_share) {
  return 8 * (by_share ? shares * ((tiles + 7) / 8) : (shares * tiles + 7) / 8);
}

}  // namespace experts
}  // namespace fsc
