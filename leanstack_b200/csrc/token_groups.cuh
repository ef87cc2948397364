// Where the groups of 8 logits lie that token_rules.cu reads (plain C++ for any
// compiler, so that the index arithmetic is checked on the host).
#pragma once

#include <cstdint>

#ifdef __CUDACC__
#define LS_GROUPS_FN __host__ __device__ __forceinline__
#else
#define LS_GROUPS_FN inline
#endif

namespace lsb {

// Groups are aligned in the flattened [m, V] array: group g of a row holds the row's
// tokens 8 g - a .. 8 g - a + 7 with a = tr_offset(row, V), as far as there are such.
LS_GROUPS_FN int tr_offset(int64_t row, int64_t V) { return V % 8 ? (int)(row * V & 7) : 0; }
LS_GROUPS_FN int tr_groups(int a, int V) { return (V + a + 7) / 8; }
// Elements from the row's first group to the end of the array, as far as an int reaches:
// group g may be read up to its element tr_left - 8 g.  A short row's group reaches
// through several rows behind it, so the end matters to more rows than the last.
LS_GROUPS_FN int tr_left(int64_t row, int64_t V, int64_t m) {
  const int64_t left = (m - row) * V + tr_offset(row, V);
  return (int)(left < INT32_MAX ? left : INT32_MAX);
}

}  // namespace lsb
