// 8-bit operands: scale = max(amax |x| / largest, 2^-126) over the elements that share it, q = fp8(x * (1 / scale)).
//
// The floor of 2^-126 (the smallest normal f32) keeps zeros and the tiniest values finite.  The reciprocal is rounded once per
// block; the product is within 2^-23 of the quotient, which is nothing against the rounding to 8 bits.  (With a division per element,
// some 40 instructions an element in all, 16,384 x 4096 bf16 rows took 81 us.)  An infinity makes its block's scale infinite, a NaN
// makes it NaN: every product with the block is then NaN.  Largest values are found on the bits without the sign, which order as the
// values do, with NaN above infinity.
//
// Rows: 16 lanes hold a row's 128 columns, 8 elements each, in registers between the maximum and the product: one read of X.
// Blocks of 128 x 128: a CTA holds the block in registers.
//
// What bounds it: HBM for f32 (16,384 x 4096: rows 49.9 us = 6.73 TB/s, blocks 50.4), issue slots and HBM together for 16 bits (rows
// 36 us = 5.7 TB/s, 69 % of issue slots, of 39 instructions per 8 elements some 18 convert; blocks 40.6).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "swb_chain.cuh"
#include "swb_index.h"
#include "swb_kernels.h"

namespace swb {
namespace {

constexpr float SMALLEST_SCALE = 1.17549435e-38f;  // 2^-126

__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

__device__ __forceinline__ float scale_of(float amax, float largest) {
  const float s = amax / largest;
  return s < SMALLEST_SCALE ? SMALLEST_SCALE : s;  // a NaN stays
}

template <bool E5M2>
__device__ __forceinline__ float largest() { return E5M2 ? 57344.0f : 448.0f; }

__device__ __forceinline__ float2 times(float2 v, float f) {  // both in one instruction
  uint64_t a, b, r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(a) : "f"(v.x), "f"(v.y));
  asm("mov.b64 %0, {%1, %1};" : "=l"(b) : "f"(f));
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  asm("mov.b64 {%0, %1}, %2;" : "=f"(v.x), "=f"(v.y) : "l"(r));
  return v;
}

// Eight elements of a row as they lie in memory.
template <typename T>
struct Eight {
  static constexpr int WORDS = 2 * sizeof(T);
  uint32_t w[WORDS];

  // The first `valid` elements; the others are zeros.  V = 1 for rows of any alignment, else whole vectors.
  template <int V>
  __device__ __forceinline__ void load(const T *p, int valid) {
    constexpr int PER_WORD = 4 / sizeof(T), BYTES = sizeof(T) * V;
#pragma unroll
    for (int i = 0; i < WORDS; ++i) w[i] = 0;
    if constexpr (BYTES >= 16) {
#pragma unroll
      for (int i = 0; i < WORDS; i += 4)
        if (i * PER_WORD < valid) {
          const uint4 v = __ldg(reinterpret_cast<const uint4 *>(p + i * PER_WORD));
          w[i] = v.x; w[i + 1] = v.y; w[i + 2] = v.z; w[i + 3] = v.w;
        }
    } else if constexpr (BYTES == 8) {
#pragma unroll
      for (int i = 0; i < WORDS; i += 2)
        if (i * PER_WORD < valid) {
          const uint2 v = __ldg(reinterpret_cast<const uint2 *>(p + i * PER_WORD));
          w[i] = v.x; w[i + 1] = v.y;
        }
    } else if constexpr (BYTES == 4 && sizeof(T) == 2) {
#pragma unroll
      for (int i = 0; i < WORDS; ++i)
        if (2 * i < valid) w[i] = __ldg(reinterpret_cast<const uint32_t *>(p) + i);
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < valid) w[i] = __ldg(reinterpret_cast<const uint32_t *>(p) + i);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < valid) w[i / 2] |= (uint32_t)__ldg(reinterpret_cast<const uint16_t *>(p) + i) << (i % 2 * 16);
    }
  }

  // The bits of the largest |x| as an f32.
  __device__ __forceinline__ uint32_t amax() const {
    if constexpr (sizeof(T) == 4) {
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < WORDS; ++i) m = max(m, w[i] & 0x7fffffffu);
      return m;
    } else {
      uint32_t two = 0;  // two at a time
#pragma unroll
      for (int i = 0; i < WORDS; ++i) asm("max.u16x2 %0, %0, %1;" : "+r"(two) : "r"(w[i] & 0x7fff7fffu));
      const uint16_t bits = (uint16_t)max(two & 0xffffu, two >> 16);
      T v;
      memcpy(&v, &bits, 2);
      return __float_as_uint(to_f32(v));
    }
  }

  template <bool E5M2, int V>
  __device__ __forceinline__ void store(uint8_t *q, float inverse, int valid) const {
    constexpr __nv_fp8_interpretation_t KIND = E5M2 ? __NV_E5M2 : __NV_E4M3;
    uint16_t out[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float2 v;
      if constexpr (sizeof(T) == 4) {
        v = make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
      } else {
        T two[2];
        memcpy(two, &w[i], 4);
        v = make_float2(to_f32(two[0]), to_f32(two[1]));
      }
      out[i] = __nv_cvt_float2_to_fp8x2(times(v, inverse), __NV_SATFINITE, KIND);
    }
    if constexpr (V == 8) {
      if (valid > 0) *reinterpret_cast<uint2 *>(q) = make_uint2(out[0] | (uint32_t)out[1] << 16, out[2] | (uint32_t)out[3] << 16);
    } else if constexpr (V == 4) {
#pragma unroll
      for (int i = 0; i < 4; i += 2)
        if (2 * i < valid) *reinterpret_cast<uint32_t *>(q + 2 * i) = out[i] | (uint32_t)out[i + 1] << 16;
    } else if constexpr (V == 2) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (2 * i < valid) *reinterpret_cast<uint16_t *>(q + 2 * i) = out[i];
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < valid) q[i] = (uint8_t)(out[i / 2] >> (i % 2 * 8));
    }
  }
};

constexpr int ROWS_THREADS = 256, ROWS_PER_GROUP = 4;  // rows in flight per 16 lanes

template <typename T, int V, bool E5M2>
__global__ void __launch_bounds__(ROWS_THREADS) quantize_rows_kernel(int64_t rows, int64_t cols, int64_t blocks,
                                                                     const T *__restrict__ X, uint8_t *__restrict__ Q,
                                                                     float *__restrict__ scales) {
  after_previous_kernel();
  const int group = threadIdx.x / 16, lane = threadIdx.x % 16;
  constexpr int GROUPS = ROWS_THREADS / 16;
  // neighbouring groups of lanes take neighbouring column blocks of the same rows
  const int64_t first = (int64_t)blockIdx.x * GROUPS, first_row = first / blocks;
  const uint32_t at = (uint32_t)(first - first_row * blocks) + group, past = at / (uint32_t)blocks;  // blocks is below 2^24
  const int64_t block = at - past * (uint32_t)blocks, row0 = (first_row + past) * ROWS_PER_GROUP, col = block * kScaleBlock + lane * 8;
  if (row0 >= rows) return;
  const int valid = cols - col < 8 ? (int)(cols - col) : 8;
  Eight<T> v[ROWS_PER_GROUP];
#pragma unroll
  for (int r = 0; r < ROWS_PER_GROUP; ++r) v[r].template load<V>(X + (row0 + r) * cols + col, row0 + r < rows ? valid : 0);
  // The maxima of four rows at a time: two steps in which a lane gives away half of its rows for the other lane's share of the
  // half that it keeps, two for the one row that is left.  Lanes 4 r ... 4 r + 3 end with row r, divide for it and store its scale.
  static_assert(ROWS_PER_GROUP == 4, "");
  const unsigned lanes = 0xffffu << (threadIdx.x & 16);
  const bool back = lane & 8, odd = lane & 4;
  uint32_t m[ROWS_PER_GROUP];
#pragma unroll
  for (int r = 0; r < ROWS_PER_GROUP; ++r) m[r] = v[r].amax();
  const uint32_t a0 = max(back ? m[2] : m[0], __shfl_xor_sync(lanes, back ? m[0] : m[2], 8));
  const uint32_t a1 = max(back ? m[3] : m[1], __shfl_xor_sync(lanes, back ? m[1] : m[3], 8));
  uint32_t mine = max(odd ? a1 : a0, __shfl_xor_sync(lanes, odd ? a0 : a1, 4));
  mine = max(mine, __shfl_xor_sync(lanes, mine, 2));
  mine = max(mine, __shfl_xor_sync(lanes, mine, 1));
  const float scale = scale_of(__uint_as_float(mine), largest<E5M2>()), inverse = 1.0f / scale;
  if (lane % 4 == 0 && row0 + lane / 4 < rows) scales[block * rows + row0 + lane / 4] = scale;
#pragma unroll
  for (int r = 0; r < ROWS_PER_GROUP; ++r) {
    const float f = __shfl_sync(lanes, inverse, 4 * r, 16);
    if (row0 + r < rows) v[r].template store<E5M2, V>(Q + (row0 + r) * cols + col, f, valid);
  }
}

constexpr int BLOCK_THREADS = 256, BLOCK_STEPS = 128 * 128 / (BLOCK_THREADS * 8);

template <typename T, int V, bool E5M2>
__global__ void __launch_bounds__(BLOCK_THREADS) quantize_blocks_kernel(int64_t rows, int64_t cols, int64_t row_blocks,
                                                                        int64_t col_blocks, const T *__restrict__ X,
                                                                        uint8_t *__restrict__ Q, float *__restrict__ scales) {
  __shared__ uint32_t warp_max[BLOCK_THREADS / 32];
  after_previous_kernel();
  const int64_t cb = blockIdx.x % col_blocks, rb = blockIdx.x / col_blocks % row_blocks, g = blockIdx.x / col_blocks / row_blocks;
  const int64_t col = cb * kScaleBlock + threadIdx.x % 16 * 8;
  const int valid = cols - col < 8 ? (int)(cols - col) : 8;
  Eight<T> v[BLOCK_STEPS];
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < BLOCK_STEPS; ++i) {
    const int64_t row = rb * kScaleBlock + i * (BLOCK_THREADS / 16) + threadIdx.x / 16;
    v[i].template load<V>(X + (g * rows + row) * cols + col, row < rows ? valid : 0);
  }
#pragma unroll
  for (int i = 0; i < BLOCK_STEPS; ++i) m = max(m, v[i].amax());
#pragma unroll
  for (int d = 16; d > 0; d /= 2) m = max(m, __shfl_xor_sync(0xffffffffu, m, d));
  if (threadIdx.x % 32 == 0) warp_max[threadIdx.x / 32] = m;
  __syncthreads();
  m = warp_max[0];
#pragma unroll
  for (int w = 1; w < BLOCK_THREADS / 32; ++w) m = max(m, warp_max[w]);
  const float scale = scale_of(__uint_as_float(m), largest<E5M2>()), inverse = 1.0f / scale;
  if (threadIdx.x == 0) scales[blockIdx.x] = scale;
#pragma unroll
  for (int i = 0; i < BLOCK_STEPS; ++i) {
    const int64_t row = rb * kScaleBlock + i * (BLOCK_THREADS / 16) + threadIdx.x / 16;
    if (row < rows) v[i].template store<E5M2, V>(Q + (g * rows + row) * cols + col, inverse, valid);
  }
}

// Elements per load and store: 8, 4 or 2 where rows of X and Q start on such a boundary, else 1.
template <typename T>
int vector_width(const QuantizeArgs &a) {
  for (int v : {8, 4, 2}) {
    const size_t bytes = sizeof(T) * v < 16 ? sizeof(T) * v : 16;
    if (a.cols % v == 0 && reinterpret_cast<uintptr_t>(a.X) % bytes == 0 && reinterpret_cast<uintptr_t>(a.Q) % v == 0) return v;
  }
  return 1;
}

template <typename T, int V, bool E5M2>
cudaError_t launch(const QuantizeArgs &a, bool by_rows, cudaStream_t s) {
  const int64_t col_blocks = ceil_div(a.cols, kScaleBlock), row_blocks = ceil_div(a.rows, kScaleBlock);
  const int64_t grid = by_rows ? ceil_div(ceil_div(a.rows, ROWS_PER_GROUP) * col_blocks, ROWS_THREADS / 16)
                               : a.groups * row_blocks * col_blocks;
  if (grid > 2147483647LL) return cudaErrorInvalidConfiguration;
  const T *X = static_cast<const T *>(a.X);
  uint8_t *Q = static_cast<uint8_t *>(a.Q);
  return by_rows ? launch_chained(quantize_rows_kernel<T, V, E5M2>, (unsigned)grid, ROWS_THREADS, 0, s, a.rows, a.cols, col_blocks, X, Q,
                                  a.scales)
                 : launch_chained(quantize_blocks_kernel<T, V, E5M2>, (unsigned)grid, BLOCK_THREADS, 0, s, a.rows, a.cols, row_blocks,
                                  col_blocks, X, Q, a.scales);
}

template <typename T, int V>
cudaError_t launch_type(const QuantizeArgs &a, bool by_rows, cudaStream_t s) {
  return a.fp8_type == kE5M2 ? launch<T, V, true>(a, by_rows, s) : launch<T, V, false>(a, by_rows, s);
}

template <typename T>
cudaError_t launch_width(const QuantizeArgs &a, bool by_rows, cudaStream_t s) {
  switch (vector_width<T>(a)) {
    case 8: return launch_type<T, 8>(a, by_rows, s);
    case 4: return launch_type<T, 4>(a, by_rows, s);
    case 2: return launch_type<T, 2>(a, by_rows, s);
  }
  return launch_type<T, 1>(a, by_rows, s);
}

cudaError_t launch_quantize(const QuantizeArgs &a, bool by_rows, cudaStream_t s, int64_t *launches) {
  if (a.groups == 0 || a.rows == 0 || a.cols == 0) return cudaSuccess;
  ++*launches;
  switch (a.type) {
    case kBF16: return launch_width<__nv_bfloat16>(a, by_rows, s);
    case kF16: return launch_width<__half>(a, by_rows, s);
  }
  return launch_width<float>(a, by_rows, s);
}

}  // namespace

cudaError_t launch_quantize_rows(const QuantizeArgs &a, cudaStream_t s, int64_t *launches) {
  return launch_quantize(a, true, s, launches);
}
cudaError_t launch_quantize_blocks(const QuantizeArgs &a, cudaStream_t s, int64_t *launches) {
  return launch_quantize(a, false, s, launches);
}

}  // namespace swb
