// The rows by expert (expert_plan.hip), as the products read them.
#pragma once

#include <hip/hip_runtime.h>
#include <cstdint>

namespace fsc {
namespace experts {

constexpr int MAX_EXPERTS = 512;

struct Plan {
  int32_t *offsets, *slot_of, *row_of, *place, *tiles, *counts;
  int n_tiles;
};

// int32 of a plan of M slots, E experts and row tiles of `tile` rows, and its parts in a buffer of that size.
int64_t plan_ints(int64_t M, int E, int tile);
Plan plan_of(int32_t* buf, int64_t M, int E, int tile);
void launch_plan(const Plan& p, int64_t M, int E, int k, int tile, const int32_t* index, hipStream_t st);

}  // namespace experts
}  // namespace fsc
