// The copies of rows that the experts' products make, against the room that their sizes reserve: every type, width and
// hidden size on both sides of a word and a chunk, arrays that one buffer reads and arrays that it does not, forward (x,
// w_in, w_out) and backward (dy, w_out, w_in, x).
#include <cstdio>
#include <vector>

#include "expert_room.h"

using namespace fsc::experts;

int main() {
  long cases = 0, taken = 0, wrong = 0;
  char* const base = reinterpret_cast<char*>(1 << 20);   // an address to count from
  for (int size : {1, 2, 4})
    for (int width : {1, 16, 64, 331, 334, 640, 641})
      for (int hidden : {1, 40, 85, 86, 640})
        for (int64_t rows : {1, 300, 10007})
          for (int E : {1, 4, 31})
            for (int arrays : {1, 2})
              for (int far = 0; far < (arrays == 1 ? 2 : 4); ++far) {
                struct A { bool weights, reads; int64_t rows; int n; };
                std::vector<A> all;
                const A in{true, !odd_rows(width, size), (int64_t)E * 2 * hidden, width};
                const A out{true, !odd_rows(hidden, size), (int64_t)E * width, hidden};
                all.push_back({false, !(far & 1), rows, width});
                if (arrays == 1) all.insert(all.end(), {in, out});
                else all.insert(all.end(), {out, in, A{false, !(far & 2), rows, width}});
                const int64_t bytes = copies_bytes(rows, width, hidden, E, size, arrays);
                Room room{base, base + bytes};
                int64_t used = 0;
                ++cases;
                for (const A& a : all) {
                  if (a.reads || !copies(a.weights, a.n, size)) continue;
                  const int64_t need = copy_bytes(a.rows, a.n, size);
                  const char* p = (const char*)room.take(need);
                  used += need;
                  ++taken;
                  // there, inside, and as large as rows of whole chunks
                  if (!p || p - base + need > bytes || need < a.rows * copy_row(a.n, size) * size || need % 64) ++wrong;
                }
                if (used > bytes || room.at - base > bytes || room.take(bytes + 64)) ++wrong;
                if (size == 4 && bytes) ++wrong;      // fp32 rows are never copied
              }
  std::printf("cases %ld, copies %ld, wrong %ld\n", cases, taken, wrong);
  return wrong ? 1 : 0;
}
