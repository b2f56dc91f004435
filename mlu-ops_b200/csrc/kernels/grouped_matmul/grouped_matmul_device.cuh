// Device side of the grouping: which rows a group has and which tile is whose, worked
// out by every block from the group ends (they are on the device only).
#ifndef MLUOP_B200_KERNELS_GROUPED_MATMUL_DEVICE_CUH_
#define MLUOP_B200_KERNELS_GROUPED_MATMUL_DEVICE_CUH_

#include <cuda_runtime.h>

#include <cstdint>

#include "kernels/grouped_matmul/grouped_matmul_kernels.h"

namespace mluop {
namespace grouped_matmul {

// In shared memory.  Group g has rows end[g] .. end[g+1]-1 and units first[g] .. first[g+1]-1; behind the last
// group lies one more "group" of the rows that belong to none.  slot[g]: chunks of split groups before g.
struct GroupMap {
  int end[kMaxGroups + 2];
  int first[kMaxGroups + 2];
  int slot[kMaxGroups + 2];
};

// Fills the map; called by the whole block, which is synchronised before and after.
// kRows: a group has ceil(rows / tile) * tiles_per_chunk units.  Weight gradient: max(1, ceil(rows / chunk_rows)) *
// tiles_per_chunk units, none for the rows of no group.
template <bool kWeightGrad>
__device__ __forceinline__ void buildGroupMap(GroupMap &map, const int32_t *ends, int groups, int64_t rows,
                                              int64_t chunk_rows, int tiles_per_chunk) {
  for (int g = threadIdx.x; g < groups; g += blockDim.x) map.end[g + 1] = ends[g];
  if (threadIdx.x == 0) {
    map.end[0] = 0;
    map.end[groups + 1] = (int)rows;
  }
  __syncthreads();
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    int highest = 0, units = 0, slots = 0;
    for (int base = 0; base <= groups; base += 32) {
      const int g = base + lane;  // this lane's group; `groups` itself: the rows of no group
      int e = g <= groups ? map.end[g + 1] : 0;
      e = e < 0 ? 0 : (e > rows ? (int)rows : e);
      // running maximum: an end below an earlier one counts as that one
      for (int o = 1; o < 32; o <<= 1) {
        const int other = __shfl_up_sync(0xffffffffu, e, o);
        if (lane >= o && other > e) e = other;
      }
      e = e > highest ? e : highest;
      int before = __shfl_up_sync(0xffffffffu, e, 1);
      if (lane == 0) before = highest;
      const int64_t count = g <= groups ? e - before : 0;
      int64_t chunks = (count + chunk_rows - 1) / chunk_rows;
      if (kWeightGrad) chunks = g >= groups ? 0 : (chunks < 1 ? 1 : chunks);
      int mine = (int)(chunks * tiles_per_chunk), split = kWeightGrad && chunks > 1 ? (int)chunks : 0;
      const int own_units = mine, own_slots = split;
      for (int o = 1; o < 32; o <<= 1) {
        const int other = __shfl_up_sync(0xffffffffu, mine, o), other_split = __shfl_up_sync(0xffffffffu, split, o);
        if (lane >= o) {
          mine += other;
          split += other_split;
        }
      }
      __syncwarp();
      if (g <= groups) {
        map.end[g + 1] = e;
        map.first[g] = units + mine - own_units;
        map.slot[g] = slots + split - own_slots;
        if (g == groups) {
          map.first[g + 1] = units + mine;
          map.slot[g + 1] = slots + split;
        }
      }
      highest = __shfl_sync(0xffffffffu, e, 31);
      units += __shfl_sync(0xffffffffu, mine, 31);
      slots += __shfl_sync(0xffffffffu, split, 31);
    }
  }
  __syncthreads();
}

// The group of unit `unit` (below first[groups + 1]).
__device__ __forceinline__ int groupOfUnit(const GroupMap &map, int groups, int unit) {
  int lo = 0, hi = groups + 1;  // first[lo] <= unit < first[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (map.first[mid] <= unit) lo = mid;
    else hi = mid;
  }
  return lo;
}

}  // namespace grouped_matmul
}  // namespace mluop

#endif  // MLUOP_B200_KERNELS_GROUPED_MATMUL_DEVICE_CUH_
