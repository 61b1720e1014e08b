// The weight gradients' shares and blocks on the host: for a sweep of sizes and of ways to spread the positions over the
// experts, the shares that the experts make fit those that are launched and that the workspace holds, and where every
// expert is one share the blocks are exactly the experts' tiles.
#include <cstdio>
#include <vector>

#include "expert_shares.h"

using namespace fsc::experts;

static long cases = 0, equal = 0, bad = 0;

static void check(bool ok, const char* what, int64_t M, int E, int size, int64_t tiles) {
  if (!ok && ++bad < 20) std::printf("%s: M %ld E %d size %d tiles %ld\n", what, (long)M, E, size, (long)tiles);
}

static int64_t shares_of(const std::vector<int64_t>& rows, int share) {
  int64_t n = 0;
  for (int64_t r : rows) n += r > 0 ? (r - 1) / share + 1 : 1;
  return n;
}

static void one(int64_t M, int E, int size, int64_t tiles) {
  const int share = weight_share(M, E, size, tiles);
  const int64_t most = most_shares(M, E, share);
  ++cases;
  equal += M == share;
  std::vector<int64_t> all(E, 0), even(E, M / E), halves(E, 0);
  all[E - 1] = M;
  even[0] += M % E;
  int64_t left = M;
  for (int e = 0; e < E && left > 0; ++e) {       // as many partial shares as possible
    halves[e] = left < share + 1 || e == E - 1 ? left : share + 1;
    left -= halves[e];
  }
  for (const auto& rows : {all, even, halves}) check(shares_of(rows, share) <= most, "more shares than launched", M, E, size, tiles);
  const bool each = one_share_each(M, share), by_share = runs_by_share(each, tiles);
  const int64_t blocks = weight_blocks(most, tiles, by_share), per = (tiles + 7) / 8;
  check(each == (most == E), "shares where every expert is one", M, E, size, tiles);
  check(blocks < (1ll << 24), "grid", M, E, size, tiles);
  if (each) {
    int64_t seen = 0;
    for (int64_t b = 0; b < blocks; ++b) {         // as the kernel takes its place
      const int64_t w = b >> 3, x = b & 7, e = w / per, c = x * per + w % per;
      check(e < E, "a block past the last expert", M, E, size, tiles);
      seen += c < tiles;
    }
    check(seen == E * tiles, "tiles", M, E, size, tiles);
  } else {
    check(by_share ? blocks / 8 / per == most : blocks >= most * tiles, "blocks of the shares", M, E, size, tiles);
  }
}

int main() {
  for (int size : {2, 4})
    for (int E : {1, 2, 3, 4, 5, 8, 16, 31, 64, 512})
      for (int H : {8, 40, 331, 640, 1600})
        for (int F : {8, 64, 203, 640, 1280})
          for (int side : {0, 1}) {
            const int ldf = (F + 7) / 8 * 8;
            const int64_t tiles = side ? weight_tiles(ldf, H) : weight_tiles(H, 2 * ldf);
            for (int64_t rows : {1, 7, 64, 128, 150, 512, 1024, 4099, 10000, 100000})
              for (int k : {1, 2, 3, 4, 8}) one(rows * k, E, size, tiles);
            // the slots of a share, one fewer and one more
            for (int64_t M : {128, 256, 1024, 2048})
              for (int d : {-1, 0, 1}) one(M + d, E, size, tiles);
          }
  std::printf("cases %ld, slots as many as a share %ld, wrong %ld\n", cases, equal, bad);
  return bad ? 1 : 0;
}
