// Room at the end of a workspace for padded copies of rows that cannot be read 16 bytes at a time: which arrays are copied,
// what is reserved for them, and how it is handed out.  Arithmetic on sizes alone, on the host.
#pragma once

#include <cstdint>

namespace fsc {
namespace experts {

constexpr int64_t align64(int64_t b) { return (b + 63) / 64 * 64; }
constexpr int64_t whole_chunks(int64_t n, int ce) { return (n + ce - 1) / ce * ce; }
// Rows of n values that end inside a 32-bit word.
constexpr bool odd_rows(int n, int size) { return n * (int64_t)size % 4 != 0; }

// A copy's row: whole 16-byte chunks of 8 values (16 in 8 bits).
constexpr int64_t copy_row(int n, int size) { return whole_chunks(n, size == 1 ? 16 : 8); }
constexpr int64_t copy_bytes(int64_t rows, int n, int size) { return align64(rows * copy_row(n, size) * size); }

// Whether an array that one buffer of 32-bit offsets does not read may be copied: rows of x or dy in 16 or 8 bits, and
// weights whose rows end inside a word.  fp32 rows are always whole words; where they lie too far apart for one buffer
// they are read value by value, as everything is that has no copy.
constexpr bool copies(bool weights, int n, int size) { return size < 4 && (!weights || odd_rows(n, size)); }

// Room for copies of `arrays` arrays of the caller's rows (whose strides and addresses the sizes do not tell) and of both
// weights.
constexpr int64_t copies_bytes(int64_t rows, int width, int hidden, int E, int size, int arrays) {
  return (copies(false, width, size) ? arrays * copy_bytes(rows, width, size) : 0) +
         (copies(true, width, size) ? copy_bytes((int64_t)E * 2 * hidden, width, size) : 0) +
         (copies(true, hidden, size) ? copy_bytes((int64_t)E * width, hidden, size) : 0);
}

struct Room {
  char *at, *end;
  // the next `bytes` (a multiple of 64), null where they are not there
  void* take(int64_t bytes) {
    if (end - at < bytes) return nullptr;
    char* const p = at;
    at += bytes;
    return p;
  }
};

}  // namespace experts
}  // namespace fsc
