// Index arithmetic shared by host code and kernels.  Every function states the
// reference construct whose values it reproduces bit for bit.
#pragma once
#include <stdint.h>

#if defined(__CUDACC__)
#define SWB_HD __host__ __device__ __forceinline__
#else
#define SWB_HD inline
#endif

namespace swb {

SWB_HD int64_t ceil_div(int64_t a, int64_t b) { return a / b + (a % b != 0); }
SWB_HD int64_t max1(int64_t v) { return v > 1 ? v : 1; }

// Largest x dimension of a CUDA grid.  `blocks` (at least one block is always launched) as a grid
// dimension, or false when it does not fit.
constexpr int64_t kMaxGridX = 2147483647LL;
inline bool grid_dim(int64_t blocks, unsigned *out) {
  const int64_t b = max1(blocks);
  if (b > kMaxGridX) return false;
  *out = (unsigned)b;
  return true;
}

// Rows of a slice of a long operand whose copy counts its slices along the y
// axis of a grid: at least 512, and as many as leave at most 16,384 slices.
// The slices of two operands, or of one and up to 1,024 matrices beside it, are
// then below the 65,535 that the axis holds.  (Not a reference construct.)
constexpr int64_t kMaxGridY = 65535, kMostSlices = 16384;
SWB_HD int64_t slice_rows(int64_t all) { return all > 512 * kMostSlices ? ceil_div(all, kMostSlices) : 512; }

// Bytes from row to row of a copy of `bytes`-byte rows that TMA can read, which
// wants multiples of 16: whole lines of 128 bytes from 512 bytes on (at most a
// quarter more than the rows), whole sectors of 32 below, 16 for the shortest.
// Measured, 16,384 rows in 8 groups, 512 columns, 16 bits, by 16, 32 and 128
// bytes: rows of 2 bytes 20.2, 19.6, 19.1 us; of 130 19.9, 19.7, 19.5; of 398
// 19.6, 18.9, 19.0; of 1,026 26.2, 24.2, 23.8; of 4,098 68.8, 64.4, 63.1.
// (Not a reference construct.)
SWB_HD int64_t copy_pitch(int64_t bytes) {
  const int64_t unit = bytes <= 16 ? 16 : bytes < 512 ? 32 : 128;
  return ceil_div(bytes, unit) * unit;
}

// Balanced contiguous partition of [lower, upper) over `count` workers:
// base = span / count, rem = span % count; worker w starts at
// lower + w*base + min(w, rem) and takes base + (w < rem) positions
// (sparsewave.position_space, SparsePositionToSCF.cpp:190-223).
SWB_HD void partition(int64_t lower, int64_t upper, int64_t worker,
                      int64_t count, int64_t &begin, int64_t &end) {
  int64_t span = upper - lower;
  int64_t base = span / count;
  int64_t rem = span % count;
  bool extra = worker < rem;
  begin = lower + worker * base + (extra ? worker : rem);
  end = begin + base + (extra ? 1 : 0);
}

// Chunk of `factor` consecutive positions owned by `worker`; workers at or
// beyond ceil(span / factor) get the empty range [lower, lower)
// (sparsewave.position_for, SparsePositionToSCF.cpp:38-98).
SWB_HD void chunk_bounds(int64_t lower, int64_t upper, int64_t worker,
                         int64_t factor, int64_t &begin, int64_t &end) {
  int64_t span = upper - lower;
  int64_t chunks = span / factor + (span % factor != 0);
  bool active = worker >= 0 && worker < chunks;
  int64_t safe = active ? worker : 0;
  begin = lower + safe * factor;
  int64_t remaining = upper - begin;
  int64_t size = active ? (remaining < factor ? remaining : factor) : 0;
  end = begin + size;
}

// Row owning `position`: the predecessor of the first row offset greater than
// the position, searched over [1, len) so that empty rows are skipped
// (sparsewave.csr_row_at_position, SparsePositionToSCF.cpp:225-271).
SWB_HD int64_t row_at_position(const int32_t *row_ptr, int64_t len,
                               int64_t position) {
  int64_t lo = 1, hi = len;
  while (lo < hi) {
    int64_t mid = lo + (hi - lo) / 2;
    if ((int64_t)row_ptr[mid] <= position)
      lo = mid + 1;
    else
      hi = mid;
  }
  return lo - 1;
}

// Wave-per-position schedule (SparsePositionScheduling.cpp:340-362): the
// launch has G = max(ceil(nnz / B), 1) blocks, hence W = G * (B / 32) waves,
// and wave w owns partition(0, nnz, w, W), at most 32 positions.
SWB_HD int64_t wave_position_wave_count(int64_t nnz, int64_t block_size) {
  return max1(ceil_div(nnz, block_size)) * (block_size / 32);
}

}  // namespace swb
