// Bytes of a row as 32-bit words, and loads that end with the row.  No device code of
// its own: constexpr functions belong to host and device alike, so that a host compiler
// takes this file too.
#pragma once

#include <cstdint>

namespace as {
namespace {

// BYTES consecutive bytes (2, 4, 8 or 16, naturally aligned) as 32-bit words;
// a 2-byte load fills the low half of w[0].
template <int BYTES>
struct RawVec {
  uint32_t w[BYTES >= 4 ? BYTES / 4 : 1];
};

// The first `left` of N elements, and zeros for the others (and for the half of a word that two bytes leave).  Exactly
// the elements are read: sizeof the result is more than those of two bytes.
template <typename E, int N>
constexpr RawVec<N * sizeof(E)> load_up_to(const E* from, int left) {
  RawVec<N * sizeof(E)> r{};
  if (left >= N) {
    __builtin_memcpy(&r, from, N * sizeof(E));
  } else {
    E part[N]{};
    for (int i = 0; i < N; ++i) part[i] = i < left ? from[i] : E{};
    __builtin_memcpy(&r, part, N * sizeof(E));
  }
  return r;
}

}  // namespace
}  // namespace as
