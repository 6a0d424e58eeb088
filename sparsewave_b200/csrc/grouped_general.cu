// Products grouped by expert on operands of any size and alignment, with warp-level MMAs:
//   rows:  C[r, j] = sum_k A[r, k] B[g][k, j]            r in group g
//   inner: D[g][i, j] = sum over r in group g of A[r, i] B[r, j]   (the gradient of the weights)
// bf16 and fp16, or 8-bit values with a scale per row (block of 128 x 128) and 128 inner elements.
//
// Each block of four warps makes a tile of 64 x 64, 32 inner elements at a time: elements are loaded one by one (rows of no
// known alignment), along whichever axis is contiguous, a step ahead of the MMAs, and laid down as [row][inner] in shared memory.
// 8-bit values become fp16, which holds all of them.  The 32 (8-bit: 128) products of a step are a sum of the tensor core, which
// is added to the f32 sum, rounded to nearest.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "grouped_tiles.cuh"
#include "swb_chain.cuh"
#include "swb_index.h"
#include "swb_kernels.h"

namespace swb {
namespace {

constexpr int TILE = 64, STEP = 32, THREADS = 128;
constexpr int PITCH = STEP + 8;  // 80 bytes: eight rows of a fragment lie in different banks
constexpr int PER_THREAD = TILE * STEP / THREADS;

// An operand: element (i, k) at i * i_stride + k * k_stride (in elements), one of the strides 1.
struct Operand {
  const void *data;
  int64_t i_stride, k_stride, group_stride;
};
struct GeneralProduct {
  Operand a, b;
  void *c;
  int64_t c_pitch, c_group;
  int i_size, j_size, k_size;  // of one group, but for the ragged axis
  int rows, groups;
  const int32_t *offsets;
  int a_type, b_type;  // SWB_E4M3 ... of 8-bit operands
  const float *a_scales, *b_scales;
  int64_t b_scale_k, b_scale_j, b_scale_group;  // strides of b_scales
};

template <bool FP8>
__device__ __forceinline__ uint16_t load_element(const void *data, int64_t at, int type) {
  if constexpr (FP8) {
    const uint8_t v = __ldg(static_cast<const uint8_t *>(data) + at);
    return __half_raw(__nv_cvt_fp8_to_halfraw(v, type == kE5M2 ? __NV_E5M2 : __NV_E4M3)).x;
  } else {
    return __ldg(static_cast<const uint16_t *>(data) + at);
  }
}

// Elements (i0 + i, k0 + k), i < 64, k < 32, of which those below i_end and k_end exist; the others are zeros.
template <bool FP8>
__device__ __forceinline__ void load_tile(uint16_t (&v)[PER_THREAD], const Operand &o, const void *data, int64_t i0, int64_t i_end,
                                          int64_t k0, int64_t k_end, int type) {
  const int t = threadIdx.x;
#pragma unroll
  for (int u = 0; u < PER_THREAD; ++u) {
    const int64_t i = i0 + (o.k_stride == 1 ? t / STEP + u * (THREADS / STEP) : t % TILE);
    const int64_t k = k0 + (o.k_stride == 1 ? t % STEP : t / TILE + u * (THREADS / TILE));
    v[u] = i < i_end && k < k_end ? load_element<FP8>(data, i * o.i_stride + k * o.k_stride, type) : (uint16_t)0;
  }
}
__device__ __forceinline__ void lay_down(uint16_t (*tile)[PITCH], const uint16_t (&v)[PER_THREAD], bool k_contiguous) {
  const int t = threadIdx.x;
#pragma unroll
  for (int u = 0; u < PER_THREAD; ++u) {
    if (k_contiguous) tile[t / STEP + u * (THREADS / STEP)][t % STEP] = v[u];
    else tile[t % TILE][t / TILE + u * (THREADS / TILE)] = v[u];
  }
}

template <bool HALF>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (HALF)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The `t`-th tile of 64 rows over all groups: its group and first row; group = groups when there is none.
__device__ __forceinline__ void find_row_tile(const GeneralProduct &p, int64_t t, int *group, int64_t *first) {
  const int lane = threadIdx.x & 31;
  for (int g0 = 0; g0 < p.groups; g0 += 32) {
    const RowSpan span = g0 + lane < p.groups ? group_rows(p.offsets, g0 + lane, p.rows) : RowSpan{0, 0};
    const int64_t tiles = (span.end - (int64_t)span.begin + TILE - 1) / TILE;
    int64_t through = tiles;
    for (int d = 1; d < 32; d *= 2) {
      const int64_t before = __shfl_up_sync(0xffffffffu, through, d);
      if (lane >= d) through += before;
    }
    const unsigned behind = __ballot_sync(0xffffffffu, t < through);
    if (behind) {
      const int at = __ffs(behind) - 1;
      *group = g0 + at;
      *first = __shfl_sync(0xffffffffu, (int64_t)span.begin + (t - (through - tiles)) * TILE, at);
      return;
    }
    t -= __shfl_sync(0xffffffffu, through, 31);
  }
  *group = p.groups;
}

// RAGGED_ROWS: the groups divide i, else k.
template <bool RAGGED_ROWS, bool HALF, bool FP8>
__global__ void __launch_bounds__(THREADS) grouped_general_kernel(const GeneralProduct p) {
  __shared__ __align__(16) uint16_t tile_a[TILE][PITCH], tile_b[TILE][PITCH];
  after_previous_kernel();
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int64_t j0 = (int64_t)blockIdx.x * TILE;
  for (int64_t t = blockIdx.y;; t += gridDim.y) {
    int g = blockIdx.z;
    int64_t i0 = t * TILE, i_end = p.i_size, k0 = 0, k_end = p.k_size;
    if constexpr (RAGGED_ROWS) {
      find_row_tile(p, t, &g, &i0);
      if (g >= p.groups) return;
      i_end = group_rows(p.offsets, g, p.rows).end;
    } else {
      if (i0 >= i_end) return;
      const RowSpan span = group_rows(p.offsets, g, p.rows);
      k0 = span.begin;
      k_end = span.end;
    }
    constexpr int SIZE = FP8 ? 1 : 2;
    const void *a = p.a.data;
    const void *b = static_cast<const uint8_t *>(p.b.data) + (RAGGED_ROWS ? (int64_t)g * p.b.group_stride * SIZE : 0);
    float sum[2][4][4] = {}, part[2][4][4] = {};
    uint16_t va[PER_THREAD], vb[PER_THREAD];
    load_tile<FP8>(va, p.a, a, i0, i_end, k0, k_end, p.a_type);
    load_tile<FP8>(vb, p.b, b, j0, p.j_size, k0, k_end, p.b_type);
    for (int64_t k = k0; k < k_end; k += STEP) {
      __syncthreads();
      lay_down(tile_a, va, p.a.k_stride == 1);
      lay_down(tile_b, vb, p.b.k_stride == 1);
      __syncthreads();
      if (k + STEP < k_end) {
        load_tile<FP8>(va, p.a, a, i0, i_end, k + STEP, k_end, p.a_type);
        load_tile<FP8>(vb, p.b, b, j0, p.j_size, k + STEP, k_end, p.b_type);
      }
      const int wi = warp / 2 * 32, wj = warp % 2 * 32, r = lane / 4, c = lane % 4 * 2;
#pragma unroll
      for (int kk = 0; kk < STEP; kk += 16) {
        uint32_t fa[2][4], fb[4][2];
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int h = 0; h < 4; ++h)
            fa[x][h] = *reinterpret_cast<const uint32_t *>(&tile_a[wi + x * 16 + r + (h & 1) * 8][kk + c + (h >> 1) * 8]);
#pragma unroll
        for (int y = 0; y < 4; ++y)
#pragma unroll
          for (int h = 0; h < 2; ++h) fb[y][h] = *reinterpret_cast<const uint32_t *>(&tile_b[wj + y * 8 + r][kk + c + h * 8]);
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int y = 0; y < 4; ++y) mma<HALF>(part[x][y], fa[x], fb[y][0], fb[y][1]);
      }
      if (!FP8 || (k + STEP) % 128 == 0 || k + STEP >= k_end) {
        float sb = 1.0f;  // a tile of 64 columns lies in one block of 128
        if constexpr (FP8) sb = __ldg(p.b_scales + g * p.b_scale_group + k / 128 * p.b_scale_k + j0 / 128 * p.b_scale_j);
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float scale = 1.0f;
            if constexpr (FP8) {
              const int64_t i = i0 + wi + x * 16 + r + h * 8;
              scale = i < i_end ? sb * __ldg(p.a_scales + k / 128 * p.rows + i) : 0.0f;
            }
#pragma unroll
            for (int y = 0; y < 4; ++y)
#pragma unroll
              for (int e = 2 * h; e < 2 * h + 2; ++e) {
                sum[x][y][e] = FP8 ? fmaf(part[x][y][e], scale, sum[x][y][e]) : sum[x][y][e] + part[x][y][e];
                part[x][y][e] = 0.0f;
              }
          }
      }
    }
    __syncthreads();
    uint16_t *c = static_cast<uint16_t *>(p.c) + (RAGGED_ROWS ? 0 : (int64_t)g * p.c_group);
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int y = 0; y < 4; ++y)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int64_t i = i0 + warp / 2 * 32 + x * 16 + lane / 4 + e / 2 * 8;
          const int64_t j = j0 + warp % 2 * 32 + y * 8 + lane % 4 * 2 + e % 2;
          if (i < i_end && j < p.j_size) {
            const float v = sum[x][y][e];
            // one rounding to 16 bits, to nearest; the 8-bit product is bf16
            c[i * p.c_pitch + j] = HALF && !FP8 ? __half_as_ushort(__float2half_rn(v))
                                                : __bfloat16_as_ushort(__float2bfloat16_rn(v));
          }
        }
  }
}

template <bool RAGGED_ROWS, bool HALF, bool FP8>
cudaError_t launch(const GeneralProduct &p, cudaStream_t s) {
  const int64_t tiles = RAGGED_ROWS ? ceil_div(p.rows, TILE) + p.groups : ceil_div(p.i_size, TILE);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ceil_div(p.j_size, TILE), (unsigned)(tiles < 65535 ? tiles : 65535), RAGGED_ROWS ? 1u : (unsigned)p.groups);
  cfg.blockDim = dim3(THREADS);
  cfg.stream = s;
  cudaError_t e = cudaLaunchKernelEx(&cfg, grouped_general_kernel<RAGGED_ROWS, HALF, FP8>, p);
  return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace

cudaError_t launch_grouped_rows_general(const GroupedArgs &a, cudaStream_t s, int64_t *launches) {
  if (a.rows == 0) return cudaSuccess;
  ++*launches;
  GeneralProduct p = {};
  p.a = {a.A, a.inner, 1, 0};
  p.b = a.transpose_b ? Operand{a.B, a.inner, 1, a.inner * a.n} : Operand{a.B, 1, a.n, a.inner * a.n};
  p.c = a.C;
  p.c_pitch = a.n;
  p.i_size = (int)a.rows;
  p.j_size = (int)a.n;
  p.k_size = (int)a.inner;
  p.rows = (int)a.rows;
  p.groups = (int)a.groups;
  p.offsets = a.offsets;
  if (!a.a_scales) return a.type == kF16 ? launch<true, true, false>(p, s) : launch<true, false, false>(p, s);
  p.a_type = a.type;
  p.b_type = a.b_type;
  p.a_scales = a.a_scales;
  p.b_scales = a.b_scales;
  const int64_t kb = ceil_div(a.inner, 128), nb = ceil_div(a.n, 128);
  p.b_scale_k = a.transpose_b ? 1 : nb;
  p.b_scale_j = a.transpose_b ? kb : 1;
  p.b_scale_group = kb * nb;
  return launch<true, true, true>(p, s);
}

cudaError_t launch_grouped_inner_general(const GroupedInnerArgs &a, cudaStream_t s, int64_t *launches) {
  ++*launches;
  GeneralProduct p = {};
  p.a = {a.left, 1, a.i_size, 0};
  p.b = {a.right, 1, a.j_size, 0};
  p.c = a.out;
  p.c_pitch = a.j_size;
  p.c_group = a.i_size * a.j_size;
  p.i_size = (int)a.i_size;
  p.j_size = (int)a.j_size;
  p.rows = (int)a.rows;
  p.groups = (int)a.groups;
  p.offsets = a.offsets;
  return a.type == kF16 ? launch<false, true, false>(p, s) : launch<false, false, false>(p, s);
}

}  // namespace swb
