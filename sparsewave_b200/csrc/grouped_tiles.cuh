// Groups of rows: what the kernels of products grouped by expert read of the caller's offsets.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace swb {

struct RowSpan {
  int begin, end;
  bool decreasing = false;  // the offsets are not in order
};

// Rows of group g.  The offsets are device data that no host check has seen: clipped to the operands' rows, so that wrong
// ones make no access outside the operands.  Without offsets one group has all rows.
__device__ __forceinline__ RowSpan group_rows(const int32_t *__restrict__ offsets, int g, int rows) {
  if (!offsets) return {0, rows};
  int begin = __ldg(offsets + g), end = __ldg(offsets + g + 1);
  const bool decreasing = end < begin;
  begin = begin < 0 ? 0 : begin > rows ? rows : begin;
  end = end < begin ? begin : end > rows ? rows : end;
  return {begin, end, decreasing};
}

}  // namespace swb
