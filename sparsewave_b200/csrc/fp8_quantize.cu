// 8-bit operands: q = fp8(x / scale), scale = max(amax |x| / largest, 2^-126) over the elements that share it.
//
// The floor of 2^-126 (the smallest normal f32) keeps zeros and the tiniest values finite.  x / scale is the rounded f32
// quotient and not a product with a reciprocal, so that values at the middle of two 8-bit ones go where the definition sends
// them (bf16 inputs meet such middles often).  An infinity makes its block's scale infinite, a NaN makes it NaN: every product
// with the block is then NaN.
//
// Rows: 16 lanes hold a row's 128 columns, 8 elements each, in registers between the maximum and the division: one read of X.
// Blocks of 128 x 128: a CTA holds the block in registers.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "swb_chain.cuh"
#include "swb_index.h"
#include "swb_kernels.h"

namespace swb {
namespace {

constexpr float SMALLEST_SCALE = 1.17549435e-38f;  // 2^-126

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

// max that keeps a NaN
__device__ __forceinline__ float max_nan(float a, float b) { return a != a ? a : b != b ? b : fmaxf(a, b); }

__device__ __forceinline__ float scale_of(float amax, float largest) {
  const float s = amax / largest;
  return s < SMALLEST_SCALE ? SMALLEST_SCALE : s;  // a NaN stays
}

template <bool E5M2>
__device__ __forceinline__ float largest() { return E5M2 ? 57344.0f : 448.0f; }

// V elements of a row of which the first `valid` exist; the others are zeros.  V = 1 for rows of any alignment, else whole vectors.
template <typename T, int V>
__device__ __forceinline__ void load(float (&v)[8], const T *p, int valid) {
  struct __align__(sizeof(T) * V < 16 ? sizeof(T) * V : 16) Vector { T e[V]; };
#pragma unroll
  for (int i = 0; i < 8; i += V) {
    Vector t;
    if (i < valid) t = *reinterpret_cast<const Vector *>(p + i);
#pragma unroll
    for (int j = 0; j < V; ++j) v[i + j] = i < valid ? to_f32(t.e[j]) : 0.0f;
  }
}
template <bool E5M2, int V>
__device__ __forceinline__ void store(uint8_t *q, const float (&v)[8], float scale, int valid) {
  struct __align__(V) Vector { uint8_t e[V]; };
#pragma unroll
  for (int i = 0; i < 8; i += V) {
    Vector t;
    if constexpr (V == 1) {
      t.e[0] = __nv_cvt_float_to_fp8(v[i] / scale, __NV_SATFINITE, E5M2 ? __NV_E5M2 : __NV_E4M3);
    } else {
#pragma unroll
      for (int j = 0; j < V; j += 2) {
        const __nv_fp8x2_storage_t two = __nv_cvt_float2_to_fp8x2(make_float2(v[i + j] / scale, v[i + j + 1] / scale),
                                                                  __NV_SATFINITE, E5M2 ? __NV_E5M2 : __NV_E4M3);
        t.e[j] = (uint8_t)two;
        t.e[j + 1] = (uint8_t)(two >> 8);
      }
    }
    if (i < valid) *reinterpret_cast<Vector *>(q + i) = t;
  }
}
__device__ __forceinline__ float amax_of(const float (&v)[8]) {
  float m = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max_nan(m, fabsf(v[i]));
  return m;
}

constexpr int ROWS_THREADS = 256, ROWS_PER_GROUP = 4;  // rows in flight per 16 lanes

template <typename T, int V, bool E5M2>
__global__ void __launch_bounds__(ROWS_THREADS) quantize_rows_kernel(int64_t rows, int64_t cols, int64_t blocks,
                                                                     const T *__restrict__ X, uint8_t *__restrict__ Q,
                                                                     float *__restrict__ scales) {
  after_previous_kernel();
  const int group = threadIdx.x / 16, lane = threadIdx.x % 16;
  constexpr int GROUPS = ROWS_THREADS / 16;
  const int64_t row_blocks = (rows + ROWS_PER_GROUP - 1) / ROWS_PER_GROUP;
  // neighbouring groups of lanes take neighbouring column blocks of the same rows
  const int64_t unit = (int64_t)blockIdx.x * GROUPS + group;
  if (unit >= row_blocks * blocks) return;
  const int64_t block = unit % blocks, row0 = unit / blocks * ROWS_PER_GROUP, col = block * kScaleBlock + lane * 8;
  const int valid = cols - col < 8 ? (int)(cols - col) : 8;
  float v[ROWS_PER_GROUP][8];
#pragma unroll
  for (int r = 0; r < ROWS_PER_GROUP; ++r) load<T, V>(v[r], X + (row0 + r) * cols + col, row0 + r < rows ? valid : 0);
#pragma unroll
  for (int r = 0; r < ROWS_PER_GROUP; ++r) {
    float m = amax_of(v[r]);
#pragma unroll
    for (int d = 8; d > 0; d /= 2) m = max_nan(m, __shfl_xor_sync(0xffffu << (threadIdx.x & 16), m, d));
    const float scale = scale_of(m, largest<E5M2>());
    if (row0 + r < rows) {
      if (lane == 0) scales[block * rows + row0 + r] = scale;
      store<E5M2, V>(Q + (row0 + r) * cols + col, v[r], scale, valid);
    }
  }
}

constexpr int BLOCK_THREADS = 512, BLOCK_STEPS = 128 * 128 / (BLOCK_THREADS * 8);

template <typename T, int V, bool E5M2>
__global__ void __launch_bounds__(BLOCK_THREADS) quantize_blocks_kernel(int64_t rows, int64_t cols, int64_t row_blocks,
                                                                        int64_t col_blocks, const T *__restrict__ X,
                                                                        uint8_t *__restrict__ Q, float *__restrict__ scales) {
  __shared__ float warp_max[BLOCK_THREADS / 32];
  after_previous_kernel();
  const int64_t cb = blockIdx.x % col_blocks, rb = blockIdx.x / col_blocks % row_blocks, g = blockIdx.x / col_blocks / row_blocks;
  const int64_t col = cb * kScaleBlock + threadIdx.x % 16 * 8;
  const int valid = cols - col < 8 ? (int)(cols - col) : 8;
  float v[BLOCK_STEPS][8], m = 0.0f;
#pragma unroll
  for (int i = 0; i < BLOCK_STEPS; ++i) {
    const int64_t row = rb * kScaleBlock + i * (BLOCK_THREADS / 16) + threadIdx.x / 16;
    load<T, V>(v[i], X + (g * rows + row) * cols + col, row < rows ? valid : 0);
  }
#pragma unroll
  for (int i = 0; i < BLOCK_STEPS; ++i) m = max_nan(m, amax_of(v[i]));
#pragma unroll
  for (int d = 16; d > 0; d /= 2) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, d));
  if (threadIdx.x % 32 == 0) warp_max[threadIdx.x / 32] = m;
  __syncthreads();
  m = warp_max[0];
#pragma unroll
  for (int w = 1; w < BLOCK_THREADS / 32; ++w) m = max_nan(m, warp_max[w]);
  const float scale = scale_of(m, largest<E5M2>());
  if (threadIdx.x == 0) scales[blockIdx.x] = scale;
#pragma unroll
  for (int i = 0; i < BLOCK_STEPS; ++i) {
    const int64_t row = rb * kScaleBlock + i * (BLOCK_THREADS / 16) + threadIdx.x / 16;
    if (row < rows) store<E5M2, V>(Q + (g * rows + row) * cols + col, v[i], scale, valid);
  }
}

// Elements per load and store: 8 or 4 where rows of X and Q start on such a boundary, else 1.
template <typename T>
int vector_width(const QuantizeArgs &a) {
  for (int v : {8, 4}) {
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
  cudaError_t e = by_rows ? launch_chained(quantize_rows_kernel<T, V, E5M2>, (unsigned)grid, ROWS_THREADS, 0, s, a.rows, a.cols,
                                           col_blocks, X, Q, a.scales)
                          : launch_chained(quantize_blocks_kernel<T, V, E5M2>, (unsigned)grid, BLOCK_THREADS, 0, s, a.rows, a.cols,
                                           row_blocks, col_blocks, X, Q, a.scales);
  return e != cudaSuccess ? e : cudaGetLastError();
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
