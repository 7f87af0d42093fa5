// Buckets of the distance between two positions, for a learned bias.
//
// One side of the query has `side` buckets.  Bucket k begins at the integer
// distance border[k] (border[0] = 0, non-decreasing), so the bucket of a
// distance d is the last k with border[k] <= d: comparisons of integers, the
// same on every machine, where floor(log(...)) would depend on the last bit of
// a logarithm next to a border.  With two sides the buckets of keys behind the
// query come after those of keys before it.
#pragma once

#include <cmath>

#include "as_device.h"
#include "as_internal.h"

namespace as {
namespace {

constexpr int kMaxBuckets = 256;

// Passed to a kernel by value (1 KB of kernel arguments).
struct PositionMap {
  int32_t border[kMaxBuckets];
  int32_t side;         // buckets of one side
  int32_t both_sides;   // != 0: keys behind the query have buckets of their own
  int32_t exact;        // distances below it are their own bucket
  float log_exact;      // an estimate of the others: exact + (log2 d - log_exact) * per_log
  float per_log;
};

inline int fill_position_map(PositionMap* map, const int32_t* borders, int64_t buckets, int both_sides) {
  if (buckets < 1 || buckets > kMaxBuckets)
    return fail(AS_ERR_INVALID_ARGUMENT, "the number of buckets must lie in [1, %d]", kMaxBuckets);
  if (both_sides && buckets % 2 != 0) return fail(AS_ERR_INVALID_ARGUMENT, "two sides need an even number of buckets");
  if (borders == nullptr) return fail(AS_ERR_INVALID_ARGUMENT, "null borders pointer");
  const int side = static_cast<int>(both_sides ? buckets / 2 : buckets);
  map->side = side;
  map->both_sides = both_sides ? 1 : 0;
  map->exact = 0;
  for (int k = 0; k < side; ++k) {
    if (borders[k] < (k == 0 ? 0 : borders[k - 1]) || (k == 0 && borders[0] != 0))
      return fail(AS_ERR_INVALID_ARGUMENT, "borders must start at 0 and not descend");
    map->border[k] = borders[k];
    // bucket k holds the distance k alone where k + 1 begins the next one
    if (map->exact == k && k + 1 < side && borders[k] == k && borders[k + 1] == k + 1) map->exact = k + 1;
  }
  for (int k = side; k < kMaxBuckets; ++k) map->border[k] = INT32_MAX;
  // the logarithm runs from the first border that is not exact to the last one
  const int first = map->exact < 1 ? 1 : map->exact;
  const float span = std::log2(static_cast<float>(borders[side - 1] > first ? borders[side - 1] : first + 1) /
                               static_cast<float>(first));
  map->log_exact = std::log2(static_cast<float>(first));
  map->per_log = static_cast<float>(side - 1 - map->exact > 0 ? side - 1 - map->exact : 0) / span;
  return AS_OK;
}

// The last k < side with border[k] <= d, for d >= 0; border (kMaxBuckets + 1
// entries of LDS, INT32_MAX behind the side's) decides.  The estimate, right or
// one off for borders that grow by a constant factor, only says where to look;
// a search by halves takes log2(side) reads that wait for one another.
__device__ __forceinline__ int bucket_of_distance(const int32_t* border, const PositionMap& map, int32_t d) {
  const float guess = (__builtin_amdgcn_logf(static_cast<float>(d)) - map.log_exact) * map.per_log;
  int k = map.exact + static_cast<int>(fmaxf(guess, 0.0f));
  k = d < map.exact ? d : (k < map.side ? k : map.side - 1);
  while (border[k] > d) --k;
  while (border[k + 1] <= d && k + 1 < map.side) ++k;
  return k;
}

// The bucket of key position - query position.
__device__ __forceinline__ int bucket_of_relative(const int32_t* border, const PositionMap& map, int64_t rel) {
  const bool behind = rel > 0;
  int64_t away = behind ? (map.both_sides ? rel : 0) : -rel;
  away = away > INT32_MAX ? INT32_MAX : away;
  const int k = bucket_of_distance(border, map, static_cast<int32_t>(away));
  return behind && map.both_sides ? k + map.side : k;
}

__device__ __forceinline__ void stage_borders(int32_t* border, const PositionMap& map) {
  for (int i = threadIdx.x; i <= kMaxBuckets; i += blockDim.x) border[i] = i < map.side ? map.border[i] : INT32_MAX;
}

}  // namespace
}  // namespace as
