// Buckets of the distance between two positions, for a learned bias.
//
// One side of the query has `side` buckets.  Bucket k begins at the integer
// distance border[k] (border[0] = 0, non-decreasing), so the bucket of a
// distance d is the last k with border[k] <= d: comparisons of integers, the
// same on every machine, where floor(log(...)) would depend on the last bit of
// a logarithm next to a border.  With two sides the buckets of keys behind the
// query come after those of keys before it.
#pragma once

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
};

inline int fill_position_map(PositionMap* map, const int32_t* borders, int64_t buckets, int both_sides) {
  if (buckets < 1 || buckets > kMaxBuckets)
    return fail(AS_ERR_INVALID_ARGUMENT, "the number of buckets must lie in [1, %d]", kMaxBuckets);
  if (both_sides && buckets % 2 != 0) return fail(AS_ERR_INVALID_ARGUMENT, "two sides need an even number of buckets");
  if (borders == nullptr) return fail(AS_ERR_INVALID_ARGUMENT, "null borders pointer");
  map->side = static_cast<int32_t>(both_sides ? buckets / 2 : buckets);
  map->both_sides = both_sides ? 1 : 0;
  for (int k = 0; k < map->side; ++k) {
    if (borders[k] < (k == 0 ? 0 : borders[k - 1]) || (k == 0 && borders[0] != 0))
      return fail(AS_ERR_INVALID_ARGUMENT, "borders must start at 0 and not descend");
    map->border[k] = borders[k];
  }
  for (int k = map->side; k < kMaxBuckets; ++k) map->border[k] = INT32_MAX;
  return AS_OK;
}

// The last k < side with border[k] <= d, for d >= 0.
__device__ __forceinline__ int bucket_of_distance(const int32_t* border, int side, int32_t d) {
  int lo = 0;
  int hi = side;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (border[mid] <= d) {
      lo = mid;
    } else {
      hi = mid;
    }
  }
  return lo;
}

// The bucket of key position - query position.
__device__ __forceinline__ int bucket_of_relative(const int32_t* border, int side, int both_sides, int64_t rel) {
  const bool behind = rel > 0;
  int64_t away = behind ? (both_sides ? rel : 0) : -rel;
  away = away > INT32_MAX ? INT32_MAX : away;
  const int k = bucket_of_distance(border, side, static_cast<int32_t>(away));
  return behind && both_sides ? k + side : k;
}

}  // namespace
}  // namespace as
