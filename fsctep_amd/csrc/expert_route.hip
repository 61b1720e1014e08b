// Router of the expert readout: for every row the k experts with the largest biased scores, and their weights.
//   s = softmax(l) or sigmoid(l);  c = s + bias;  an expert can be chosen where l > -inf and c > -inf
//   groups > 1: a group's rank is the sum of its `best` largest choosable c; the `kept` best groups stay
//   index = the k largest c, ties to the lowest expert;  weight = scale s / (sum of the chosen s, or 1)
// Slots with nothing to choose get index -1 and weight 0; a row with a NaN among its logits or choosable c gets
// the experts 0..k-1 with NaN weights, so that it shows in what the row becomes.
//
// Sixteen lanes own a row (four rows a wave), lane l the experts [l V, l V + V) in registers: maxima and sums
// across them are four DPP steps, "the lowest expert" is the lowest lane of a ballot, and the work of a round of
// the selection is spread over four rows.  Reads T E logits, writes 8 T k bytes.  The softmax's sum runs in 64
// bits and is rounded once, so that no choice hangs on the order of its terms.
//
// Measured: 100,000 x 256 fp32, sigmoid with a bias, 4 of 8 groups, k = 8: 72 us forward (109 MB: 25 us at a copy's
// rate; what bounds it is the issue of the selection's k rounds and the groups' ranks: 1,810 vector instructions for a
// wave's four rows, at which counters show every SIMD issuing all the time), 40 us backward (211 MB,
// 5.3 TB/s); 32 x 8: 2.7 us, a launch.
#include <cmath>

#include "common.h"
#include "expert_types.h"
#include "fsctep.h"

namespace fsc {
namespace route {

constexpr int NT = 256;          // 16 rows a block
constexpr int RL = 16;           // lanes of a row
constexpr int MAXE = 512;
constexpr float kNone = -INFINITY;

// The value of the lane s places further round in the same row of 16 lanes.
template <int S>
__device__ __forceinline__ float ror(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x120 + S, 0xf, 0xf, true));
}
__device__ __forceinline__ float row_max(float v) {
  v = fmaxf(v, ror<8>(v));
  v = fmaxf(v, ror<4>(v));
  v = fmaxf(v, ror<2>(v));
  return fmaxf(v, ror<1>(v));
}
__device__ __forceinline__ float row_sum(float v) {
  v += ror<8>(v);
  v += ror<4>(v);
  v += ror<2>(v);
  return v + ror<1>(v);
}
__device__ __forceinline__ double row_sum64(double v) {
#pragma unroll
  for (int off = 8; off > 0; off >>= 1) v += __shfl_xor(v, off, RL);
  return v;
}
// the 16 bits of the row's lanes
__device__ __forceinline__ unsigned row_ballot(bool p) {
  return (unsigned)(__ballot(p) >> (threadIdx.x & 48)) & 0xffffu;
}

struct Args {
  int64_t rows, ls;              // row stride of the logits, in elements
  int experts, k, groups, kept, best, renorm;
  float scale;
  const void* logits;
  const float* bias;
  int32_t* index;
  float* weight;
};

template <typename T, int V>
__device__ __forceinline__ void load_row(const T* l, int e0, int experts, bool vec, float (&v)[V]) {
  if (V >= 4 && vec) {           // experts is a multiple of 4: a chunk of 4 lies inside the row or outside
#pragma unroll
    for (int i = 0; i < V; i += 4) {
      if (e0 + i < experts) {
        if constexpr (sizeof(T) == 4) {
          const f4 t = ld4((const float*)l + e0 + i);
          v[i] = t.x; v[(i + 1) % V] = t.y; v[(i + 2) % V] = t.z; v[(i + 3) % V] = t.w;
        } else {
          const u2v t = *reinterpret_cast<const u2v*>(l + e0 + i);
          v[i] = __uint_as_float(t.x << 16);
          v[(i + 1) % V] = __uint_as_float(t.x & 0xffff0000u);
          v[(i + 2) % V] = __uint_as_float(t.y << 16);
          v[(i + 3) % V] = __uint_as_float(t.y & 0xffff0000u);
        }
      } else {
        v[i] = v[(i + 1) % V] = v[(i + 2) % V] = v[(i + 3) % V] = kNone;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = e0 + i < experts ? to_f(l[e0 + i]) : kNone;
  }
}

// 1 / y for y >= 1: the hardware's reciprocal and one Newton step in fused operations, the correctly rounded quotient
// unless y's fraction is all ones (a division takes three times the instructions).  Above 2^100 a division.
__device__ __forceinline__ float over(float y) {
  const float r = __builtin_amdgcn_rcpf(y);
  return fmaf(r, fmaf(-y, r, 1.f), r);
}

// Largest logit and sum of the row's softmax; ex becomes exp(l - m).
template <int V>
__device__ __forceinline__ void softmax_sum(float (&ex)[V], float& m, float& total) {
  m = ex[0];
#pragma unroll
  for (int i = 1; i < V; ++i) m = fmaxf(m, ex[i]);
  m = row_max(m);
  if (m == kNone) m = 0.f;
  double z = 0.0;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    ex[i] = expf(ex[i] - m);
    z += (double)ex[i];
  }
  total = (float)row_sum64(z);
  if (total == 0.f) total = 1.f;               // nothing to choose: scores of 0
}

// Scores of a lane's logits, 0 where the logit is -inf.  m, total: the softmax's, for the scores of single experts.
template <int V, bool SOFTMAX>
__device__ __forceinline__ void scores(float (&v)[V], float& m, float& total) {
  if constexpr (SOFTMAX) {
    softmax_sum<V>(v, m, total);
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = v[i] / total;
  } else {
    bool far = false;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      v[i] = 1.f + expf(-v[i]);
      far |= !(v[i] < 0x1p100f) && v[i] != INFINITY;
    }
    if (__ballot(far)) {
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = 1.f / v[i];
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = v[i] == INFINITY ? 0.f : over(v[i]);
    }
  }
}
template <bool SOFTMAX>
__device__ __forceinline__ float score_of(float l, float m, float total) {
  return SOFTMAX ? expf(l - m) / total : 1.f / (1.f + expf(-l));
}

// The value of the lane s places further round in the row (s the same for all): a step of a loop.
__device__ __forceinline__ float next_lane(float v) { return ror<1>(v); }

// A round: the largest of the row's remaining c (four DPP steps), the lowest lane that has it (a ballot), which writes
// the choice and drops it.  group_lanes: lanes of a group where groups lie in whole lanes that part the row's 16, so that ranks stay in registers;
// 0: through LDS.
template <typename T, int V, bool SOFTMAX>
__global__ __launch_bounds__(NT) void route_kernel(Args a, bool vec, int group_lanes) {
  // biased scores and group ranks, where a group does not lie in whole lanes; the choices in order
  extern __shared__ float extra[];
  __shared__ int pick[NT / RL][RL];
  const int lane = threadIdx.x & (RL - 1), slot = threadIdx.x / RL;
  const int64_t row = (int64_t)blockIdx.x * (NT / RL) + slot;
  const bool live = row < a.rows;              // the lanes of a row past the end take part with no expert
  const int e0 = lane * V;
  const T* const lrow = (const T*)a.logits + (live ? row : 0) * a.ls;
  float c[V];
  load_row<T, V>(lrow, e0, live ? a.experts : 0, vec, c);
  bool bad = false;
  unsigned open = 0;                           // bit i: the logit is above -inf
#pragma unroll
  for (int i = 0; i < V; ++i) {
    bad |= c[i] != c[i];
    open |= (c[i] > kNone ? 1u : 0u) << i;
  }
  float m = 0.f, total = 1.f;
  scores<V, SOFTMAX>(c, m, total);
  if (a.bias) {
    float b[V];
    load_row<float, V>(a.bias, e0, a.experts, V >= 4 && a.experts % 4 == 0 && (uintptr_t)a.bias % 16 == 0, b);
#pragma unroll
    for (int i = 0; i < V; ++i) c[i] += b[i];
  }
#pragma unroll
  for (int i = 0; i < V; ++i) {
    c[i] = open >> i & 1 ? c[i] : kNone;
    bad |= c[i] != c[i];
  }
  bad = row_ballot(bad) != 0;

  if (a.groups > 1 && group_lanes) {
    float t0 = kNone, t1 = kNone;              // the two largest of the lane, then of the group
#pragma unroll
    for (int i = 0; i < V; ++i) {
      t1 = fmaxf(t1, fminf(t0, c[i]));
      t0 = fmaxf(t0, c[i]);
    }
    for (int off = 1; off < group_lanes; off <<= 1) {
      const float o0 = __shfl_xor(t0, off, RL), o1 = __shfl_xor(t1, off, RL);
      t1 = fmaxf(fminf(t0, o0), fmaxf(t1, o1));
      t0 = fmaxf(t0, o0);
    }
    const float mine = a.best == 2 && t1 > kNone ? t0 + t1 : t0;
    // groups ahead: a larger rank, or the same and a lower place; every group is met group_lanes times
    int ahead = 0;
    float v = mine;
    const int g = lane / group_lanes;
#pragma unroll
    for (int s = 1; s < RL; ++s) {
      v = next_lane(v);                        // now of lane - s, round the row
      const int o = ((lane - s) & (RL - 1)) / group_lanes;
      ahead += v > mine || (v == mine && o < g);
    }
    if (ahead >= a.kept * group_lanes)
#pragma unroll
      for (int i = 0; i < V; ++i) c[i] = kNone;
  } else if (a.groups > 1) {
    float* const cs = extra + slot * (a.experts + a.groups);
    float* const gs = cs + a.experts;
    const int per = a.experts / a.groups;
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (e0 + i < a.experts) cs[e0 + i] = c[i];
    __syncthreads();
    for (int g = lane; g < a.groups; g += RL) {
      float t0 = kNone, t1 = kNone;            // the two largest
      for (int i = 0; i < per; ++i) {
        const float v = cs[g * per + i];
        t1 = fmaxf(t1, fminf(t0, v));
        t0 = fmaxf(t0, v);
      }
      gs[g] = a.best == 2 && t1 > kNone ? t0 + t1 : t0;
    }
    __syncthreads();
    const int g0 = e0 / per;                   // e0 < 2^13
    int g = g0, left = per - (e0 - g0 * per);
    bool keep = false;
    int last = -1;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if (e0 + i < a.experts && last != g) {   // groups ahead: a larger rank, or the same and a lower place
        int ahead = 0;
        const float mine = gs[g];
        for (int o = 0; o < a.groups; ++o) {
          const float v = gs[o];
          ahead += v > mine || (v == mine && o < g);
        }
        keep = ahead < a.kept;
        last = g;
      }
      if (!keep) c[i] = kNone;
      if (--left == 0) { ++g; left = per; }
    }
  }

  // k rounds: the row's largest, the lowest lane that has it, its lowest expert; that lane writes the choice down
  pick[slot][lane] = -1;
  wave_sync();
  for (int j = 0; j < a.k; ++j) {
    float most = c[0];
#pragma unroll
    for (int i = 1; i < V; ++i) most = fmaxf(most, c[i]);
    const float top = row_max(most);
    const unsigned who = row_ballot(most == top && top > kNone);
    if (__ballot(who != 0) == 0) break;        // none of the wave's rows has one left
    const bool win = who != 0 && lane == __ffs(who) - 1;
    int at = V;
#pragma unroll
    for (int i = V - 1; i >= 0; --i) at = c[i] == top ? i : at;
    if (!win) at = V;
#pragma unroll
    for (int i = 0; i < V; ++i) c[i] = i == at ? kNone : c[i];
    if (win) pick[slot][j] = e0 + at;
  }
  // lane j takes the j-th choice
  wave_sync();
  int my = lane < a.k ? pick[slot][lane] : -1;
  const float sc = my >= 0 ? score_of<SOFTMAX>(to_f(lrow[my]), m, total) : 0.f;
  const float sum = a.renorm ? row_sum(sc) : 1.f;
  float w = sum > 0.f || sum != sum ? a.scale * (sc / sum) : 0.f;
  if (bad) { my = lane; w = NAN; }
  if (live && lane < a.k) {
    a.index[row * a.k + lane] = my;
    a.weight[row * a.k + lane] = w;
  }
}

// Gradient of the weights with respect to the logits.  With u the weights' gradient and w = scale s / S:
//   renormalised: ds_j s_j = w_j (u_j - sum u (w / scale)); else ds_j s_j = scale s_j u_j = w_j u_j
// (a single choice has w / scale = 1 to the bit, and no gradient)
//   sigmoid: dl_j = (ds_j s_j)(1 - s_j);  softmax: dl_i = (ds_i s_i) - s_i sum_j ds_j s_j
// The last sum is zero for renormalised weights, so only sigmoid (the chosen logits) and softmax without
// renormalisation (all) read the logits again.  The chosen experts' gradients meet the rest of the row in LDS.
struct BackArgs {
  int64_t rows, ls;
  int experts, k, renorm;
  float scale;
  const void* logits;
  const int32_t* index;
  const float *weight, *dweight;
  void* dlogits;
};

template <typename T, int V, bool SOFTMAX>
__global__ __launch_bounds__(NT) void route_back_kernel(BackArgs a, bool vec) {
  constexpr int LD = RL * V + (V % 4 == 0 ? 4 : 0);
  __shared__ __align__(16) float buf[NT / RL][LD];
  const int lane = threadIdx.x & (RL - 1), slot = threadIdx.x / RL;
  const int64_t row = (int64_t)blockIdx.x * (NT / RL) + slot;
  const bool live = row < a.rows;
  const int e0 = lane * V;
  const T* l = (const T*)a.logits + (live ? row : 0) * a.ls;
  int idx = -1;
  float w = 0.f, u = 0.f;
  if (live && lane < a.k) {
    idx = a.index[row * a.k + lane];
    if (idx < 0 || idx >= a.experts) idx = -1;
    if (idx >= 0) {
      w = a.weight[row * a.k + lane];
      u = a.dweight[row * a.k + lane];
    }
  }
  if (a.renorm) u -= row_sum(u * (w / a.scale));
  float d = w * u;                             // ds_j s_j
  float o[V];
#pragma unroll
  for (int i = 0; i < V; ++i) o[i] = 0.f;
  if (SOFTMAX) {
    if (!a.renorm) {
      const float sum = row_sum(d);
      float m, total;
      load_row<T, V>(l, e0, live ? a.experts : 0, vec, o);
      scores<V, true>(o, m, total);
#pragma unroll
      for (int i = 0; i < V; ++i) o[i] *= -sum;
    }
  } else if (idx >= 0) {
    d *= 1.f - score_of<false>(to_f(l[idx]), 0.f, 1.f);
  }
  // one wave writes and reads its four rows
#pragma unroll
  for (int i = 0; i < V; ++i) buf[slot][e0 + i] = o[i];
  wave_sync();
  if (idx >= 0) atomicAdd(&buf[slot][idx], d);   // a row's experts differ: one addition to a place
  wave_sync();
#pragma unroll
  for (int i = 0; i < V; ++i) o[i] = buf[slot][e0 + i];
  if (!live) return;
  T* dl = (T*)a.dlogits + row * a.experts;
  if (V >= 4 && a.experts % 4 == 0) {
#pragma unroll
    for (int i = 0; i < V; i += 4)
      if (e0 + i < a.experts) {
        if constexpr (sizeof(T) == 4) {
          st4((float*)dl + e0 + i, f4{o[i], o[(i + 1) % V], o[(i + 2) % V], o[(i + 3) % V]});
        } else {
          typedef __bf16 bf4 __attribute__((ext_vector_type(4)));
          *reinterpret_cast<bf4*>(dl + e0 + i) =
              bf4{(__bf16)o[i], (__bf16)o[(i + 1) % V], (__bf16)o[(i + 2) % V], (__bf16)o[(i + 3) % V]};
        }
      }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (e0 + i < a.experts) dl[e0 + i] = from_f<T>(o[i]);
  }
}

// f with the number of experts a lane holds
template <typename F>
void by_experts(int experts, F&& f) {
  const int v = (experts + RL - 1) / RL;
  if (v <= 1) f(std::integral_constant<int, 1>{});
  else if (v <= 2) f(std::integral_constant<int, 2>{});
  else if (v <= 4) f(std::integral_constant<int, 4>{});
  else if (v <= 8) f(std::integral_constant<int, 8>{});
  else if (v <= 16) f(std::integral_constant<int, 16>{});
  else f(std::integral_constant<int, 32>{});
}

int check_sizes(int64_t rows, int32_t experts, int32_t dtype, int32_t k, int32_t score) {
  FSC_CHECK_ARG(rows >= 0 && rows < (1ll << 31), "route_experts: rows must be below 2^31");
  FSC_CHECK_ARG(experts >= 1 && experts <= MAXE, "route_experts: 1 to 512 experts");
  FSC_CHECK_ARG(k >= 1 && k <= RL && k <= experts, "route_experts: k must be 1 to 16 and at most the experts");
  FSC_CHECK_ARG(dtype == FSC_F32 || dtype == FSC_BF16, "route_experts: logits are float32 or bfloat16");
  FSC_CHECK_ARG(score == 0 || score == 1, "route_experts: score is 0 (softmax) or 1 (sigmoid)");
  return 0;
}

// rows of a launch (a grid has fewer than 2^32 threads, and a row takes 16)
constexpr int64_t MOST_ROWS = 1ll << 24;

}  // namespace route
}  // namespace fsc

extern "C" {

int fsc_route_experts(int64_t rows, int32_t n_experts, int32_t dtype, int64_t logits_stride, const void* logits,
                      const float* bias, int32_t k, int32_t score, int32_t groups, int32_t groups_kept,
                      int32_t group_best, int32_t renormalise, float scale, int32_t* index, float* weight,
                      hipStream_t stream) {
  using namespace fsc;
  using namespace fsc::route;
  if (int rc = check_sizes(rows, n_experts, dtype, k, score)) return rc;
  FSC_CHECK_ARG(groups >= 1 && groups <= MAXE / 4 && n_experts % groups == 0,
                "route_experts: groups must be 1 to 128 and divide the experts");
  FSC_CHECK_ARG(groups_kept >= 1 && groups_kept <= groups, "route_experts: groups_kept must be 1 to groups");
  FSC_CHECK_ARG(k <= groups_kept * (n_experts / groups), "route_experts: k is more than the kept groups' experts");
  FSC_CHECK_ARG(group_best == 1 || group_best == 2, "route_experts: group_best is 1 or 2");
  FSC_CHECK_ARG(logits_stride >= 0, "route_experts: negative row stride");
  FSC_CHECK_ARG(scale > 0.f && std::isfinite(scale), "route_experts: scale must be positive and finite");
  if (rows == 0) return 0;
  FSC_CHECK_ARG(logits && index && weight, "route_experts: null array");
  const int size = dtype == FSC_F32 ? 4 : 2;
  const bool vec = n_experts % 4 == 0 && logits_stride % 4 == 0 && (uintptr_t)logits % (4 * size) == 0;
  for (int64_t r0 = 0; r0 < rows; r0 += MOST_ROWS)
  by_experts(n_experts, [&](auto V) {
    constexpr int v = decltype(V)::value;
    const Args a{std::min(rows - r0, MOST_ROWS), logits_stride, n_experts, k, groups, groups_kept, group_best,
                 renormalise != 0, scale, (const char*)logits + r0 * logits_stride * size, bias, index + r0 * k,
                 weight + r0 * k};
    const unsigned grid = (unsigned)((a.rows + NT / RL - 1) / (NT / RL));
    // lanes of a group, 0 where groups do not lie in whole lanes, so many that they part the row's 16
    const int per = n_experts / groups, gl = per % v == 0 && RL % (per / v) == 0 ? per / v : 0;
    const size_t lds = groups > 1 && !gl ? NT / RL * (size_t)(n_experts + groups) * 4 : 0;
    if (dtype == FSC_F32) {
      if (score == 0) route_kernel<float, v, true><<<grid, NT, lds, stream>>>(a, vec, gl);
      else route_kernel<float, v, false><<<grid, NT, lds, stream>>>(a, vec, gl);
    } else {
      if (score == 0) route_kernel<__bf16, v, true><<<grid, NT, lds, stream>>>(a, vec, gl);
      else route_kernel<__bf16, v, false><<<grid, NT, lds, stream>>>(a, vec, gl);
    }
  });
  return check_launch("route_experts") ? 2 : 0;
}

int fsc_route_experts_backward(int64_t rows, int32_t n_experts, int32_t dtype, int64_t logits_stride,
                               const void* logits, const int32_t* index, const float* weight, const float* dweight,
                               int32_t k, int32_t score, int32_t renormalise, float scale, void* dlogits,
                               hipStream_t stream) {
  using namespace fsc;
  using namespace fsc::route;
  if (int rc = check_sizes(rows, n_experts, dtype, k, score)) return rc;
  FSC_CHECK_ARG(logits_stride >= 0, "route_experts_backward: negative row stride");
  FSC_CHECK_ARG(scale > 0.f && std::isfinite(scale), "route_experts_backward: scale must be positive and finite");
  if (rows == 0) return 0;
  FSC_CHECK_ARG(logits && index && weight && dweight && dlogits, "route_experts_backward: null array");
  const int size = dtype == FSC_F32 ? 4 : 2;
  const bool vec = n_experts % 4 == 0 && logits_stride % 4 == 0 && (uintptr_t)logits % (4 * size) == 0;
  for (int64_t r0 = 0; r0 < rows; r0 += MOST_ROWS)
  by_experts(n_experts, [&](auto V) {
    constexpr int v = decltype(V)::value;
    const BackArgs a{std::min(rows - r0, MOST_ROWS), logits_stride, n_experts, k, renormalise != 0, scale,
                     (const char*)logits + r0 * logits_stride * size, index + r0 * k, weight + r0 * k, dweight + r0 * k,
                     (char*)dlogits + r0 * n_experts * size};
    const unsigned grid = (unsigned)((a.rows + NT / RL - 1) / (NT / RL));
    if (dtype == FSC_F32) {
      if (score == 0) route_back_kernel<float, v, true><<<grid, NT, 0, stream>>>(a, vec);
      else route_back_kernel<float, v, false><<<grid, NT, 0, stream>>>(a, vec);
    } else {
      if (score == 0) route_back_kernel<__bf16, v, true><<<grid, NT, 0, stream>>>(a, vec);
      else route_back_kernel<__bf16, v, false><<<grid, NT, 0, stream>>>(a, vec);
    }
  });
  return check_launch("route_experts_backward") ? 2 : 0;
}

}  // extern "C"
