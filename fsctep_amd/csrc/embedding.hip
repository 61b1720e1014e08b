// Lookup of table rows by token (atomic number, species pair, ..) with a scale, and its gradient: the sum of the rows'
// gradients by token.  Replaces the indexing of the training step's first convolution and of the expert readout's
// table of scores, whose gradient was an atomic addition into a handful of rows
// (models/pure_cartesian_sparse_layers.py:258-259 embeds the species of every atom).
//   out_i = scale table[index_i], zeros where index_i lies outside the table
//   dtable_v = scale sum over i with index_i = v, in ascending order of i in 32 bits
#include <algorithm>

#include "common.h"
#include "expert_types.h"
#include "fsctep.h"

namespace fsc {
namespace embed {

constexpr int NT = 256;

struct Args {
  int64_t rows, stride;        // row stride of the table (forward) or of dy (backward), in elements
  int64_t table_rows;
  int width;
  float scale;
  const void *in, *index;
  void* out;
};

template <typename T, typename I>
__global__ __launch_bounds__(NT) void lookup_kernel(Args a) {
  const int lane = threadIdx.x & 63;
  const int64_t waves = (int64_t)gridDim.x * (NT / 64);
  for (int64_t row = (int64_t)blockIdx.x * (NT / 64) + (threadIdx.x >> 6); row < a.rows; row += waves) {
    const int64_t v = ((const I*)a.index)[row];
    const bool there = v >= 0 && v < a.table_rows;
    const T* in = (const T*)a.in + (there ? v : 0) * a.stride;
    T* out = (T*)a.out + row * a.width;
    for (int c = lane; c < a.width; c += 64) out[c] = from_f<T>(there ? a.scale * to_f(in[c]) : 0.f);
  }
}

template <typename T, typename I>
__global__ __launch_bounds__(NT) void gather_kernel(Args a) {
  const int col = blockIdx.y * NT + threadIdx.x;
  for (int64_t v = blockIdx.x; v < a.table_rows; v += gridDim.x) {
    float s = 0.f;
    for (int64_t i = 0; i < a.rows; ++i)
      if (((const I*)a.index)[i] == v && col < a.width) s += to_f(((const T*)a.in)[i * a.stride + col]);
    if (col < a.width) ((T*)a.out)[v * a.width + col] = from_f<T>(a.scale * s);
  }
}

int check_sizes(int64_t rows, int32_t width, int64_t table_rows, int32_t dtype, int32_t index_bits) {
  FSC_CHECK_ARG(rows >= 0 && rows < (1ll << 31), "embedding: rows must be below 2^31");
  FSC_CHECK_ARG(width >= 1 && width <= (1 << 20), "embedding: width must be 1 to 2^20");
  FSC_CHECK_ARG(table_rows >= 0 && table_rows < (1ll << 31), "embedding: the table's rows must be below 2^31");
  FSC_CHECK_ARG(dtype == FSC_F32 || dtype == FSC_BF16, "embedding: the table is float32 or bfloat16");
  FSC_CHECK_ARG(index_bits == 32 || index_bits == 64, "embedding: the index is int32 or int64");
  return 0;
}

// runs the statement with (T, I)
#define FSC_EMBED_INDEX(...)                                     \
  if (index_bits == 32) { using I = int32_t; __VA_ARGS__; }      \
  else { using I = int64_t; __VA_ARGS__; }
#define FSC_EMBED_TYPES(...)                                     \
  if (dtype == FSC_F32) { using T = float; FSC_EMBED_INDEX(__VA_ARGS__) } \
  else { using T = __bf16; FSC_EMBED_INDEX(__VA_ARGS__) }

}  // namespace embed
}  // namespace fsc

extern "C" {

int fsc_embedding_forward(int64_t rows, int32_t width, int64_t table_rows, int32_t dtype, int32_t index_bits,
                          int64_t table_stride, const void* table, const void* index, float scale, void* out,
                          hipStream_t stream) {
  using namespace fsc;
  using namespace fsc::embed;
  if (int rc = check_sizes(rows, width, table_rows, dtype, index_bits)) return rc;
  if (rows == 0) return 0;
  FSC_CHECK_ARG(index && out && (table || table_rows == 0), "embedding: null array");
  FSC_CHECK_ARG(table_stride >= 0, "embedding: negative row stride");
  const Args a{rows, table_stride, table_rows, width, scale, table, index, out};
  const unsigned grid = (unsigned)std::min<int64_t>((rows + 3) / 4, 1 << 20);
  FSC_EMBED_TYPES((lookup_kernel<T, I><<<grid, NT, 0, stream>>>(a)));
  return check_launch("embedding") ? 2 : 0;
}

int fsc_embedding_workspace(int64_t rows, int32_t width, int64_t table_rows, int64_t* bytes) {
  FSC_CHECK_ARG(bytes != nullptr, "embedding: null output");
  if (int rc = fsc::embed::check_sizes(rows, width, table_rows, FSC_F32, 32)) return rc;
  *bytes = 0;
  return 0;
}

int fsc_embedding_backward(int64_t rows, int32_t width, int64_t table_rows, int32_t dtype, int32_t index_bits,
                           int64_t dy_stride, const void* dy, const void* index, float scale, void* dtable,
                           void* workspace, hipStream_t stream) {
  using namespace fsc;
  using namespace fsc::embed;
  if (int rc = check_sizes(rows, width, table_rows, dtype, index_bits)) return rc;
  if (table_rows == 0) return 0;
  FSC_CHECK_ARG(dtable && (rows == 0 || (dy && index)), "embedding_backward: null array");
  FSC_CHECK_ARG(dy_stride >= 0, "embedding_backward: negative row stride");
  const Args a{rows, dy_stride, table_rows, width, scale, dy, index, dtable};
  const dim3 grid((unsigned)std::min<int64_t>(table_rows, 1 << 16), (width + NT - 1) / NT);
  FSC_EMBED_TYPES((gather_kernel<T, I><<<grid, NT, 0, stream>>>(a)));
  return check_launch("embedding_backward") ? 2 : 0;
}

}  // extern "C"
