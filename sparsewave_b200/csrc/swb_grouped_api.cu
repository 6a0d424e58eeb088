// C ABI of the products grouped by expert and of the 8-bit operands: operand checks and dispatch to the kernels.
#include <cstdarg>
#include <cstdio>

#include "../../include/sparsewave_b200.h"
#include "swb_index.h"
#include "swb_kernels.h"

static_assert(int(SWB_BF16) == swb::kBF16 && int(SWB_F16) == swb::kF16 && int(SWB_F32) == swb::kF32 && int(SWB_E4M3) == swb::kE4M3 &&
              int(SWB_E5M2) == swb::kE5M2, "");

namespace {

constexpr int64_t kI32Max = 2147483647LL;

int fail(swb_context *ctx, int status, const char *fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  swb::set_context_error(ctx, buf);
  return status;
}

int cuda_status(swb_context *ctx, cudaError_t e, const char *op) {
  if (e == cudaSuccess) return SWB_OK;
  (void)cudaGetLastError();  // reported here, and not to the next launch
  return fail(ctx, SWB_ERR_CUDA, "CUDA error in %s launch: %s", op, cudaGetErrorString(e));
}

int check_context(swb_context *ctx) {
  if (!ctx) return fail(nullptr, SWB_ERR_INVALID_ARGUMENT, "context is NULL");
  const cudaError_t e = cudaSetDevice(swb::context_device(ctx));
  if (e == cudaSuccess) return SWB_OK;
  (void)cudaGetLastError();
  return fail(ctx, SWB_ERR_CUDA, "CUDA error in cudaSetDevice: %s", cudaGetErrorString(e));
}

// Sizes of a product grouped by expert; 2^31 - 513 keeps the kernels' 32-bit steps past the end of an axis in range.
int check_grouped(swb_context *ctx, const char *op, int64_t rows, int64_t inner, int64_t n, int64_t groups) {
  if (rows < 0 || inner < 0) return fail(ctx, SWB_ERR_INVALID_ARGUMENT, "%s: rows and inner size must be non-negative", op);
  if (n < 1) return fail(ctx, SWB_ERR_INVALID_SHAPE, "%s: the output must have at least one column, but got %lld", op, (long long)n);
  if (groups < 1) return fail(ctx, SWB_ERR_INVALID_SHAPE, "%s: there must be at least one group, but got %lld", op, (long long)groups);
  if (groups > swb::kMaxGroups)
    return fail(ctx, SWB_ERR_CAPACITY, "%s: at most %lld groups, but got %lld", op, (long long)swb::kMaxGroups, (long long)groups);
  if (rows > kI32Max - 512 || inner > kI32Max - 512 || n > kI32Max - 512)
    return fail(ctx, SWB_ERR_INVALID_SHAPE, "%s: rows, inner size and columns must be below 2^31 - 512", op);
  return SWB_OK;
}

cudaError_t rows_product(swb_context *ctx, const swb::GroupedArgs &a, swb_stream stream) {
  return swb::launch_grouped_rows_tcgen05(a, swb::context_status_flag(ctx), swb::context_device_info(ctx), swb::context_pool(ctx),
                                          static_cast<cudaStream_t>(stream), swb::context_launches(ctx));
}
cudaError_t inner_product(swb_context *ctx, const swb::GroupedInnerArgs &a, swb_stream stream) {
  return swb::launch_grouped_inner_tcgen05(a, swb::context_status_flag(ctx), swb::context_device_info(ctx), swb::context_pool(ctx),
                                           static_cast<cudaStream_t>(stream), swb::context_launches(ctx));
}

bool is_fp8(int32_t type) { return type == SWB_E4M3 || type == SWB_E5M2; }

int fp8_product(swb_context *ctx, const char *op, int32_t a_type, int32_t b_type, int64_t rows, int64_t inner, int64_t n,
                int64_t groups, const int32_t *offsets, const void *A, const float *a_scales, const void *B,
                const float *b_scales, int32_t transpose_b, uint16_t *C, swb_stream stream) {
  if (!is_fp8(a_type) || !is_fp8(b_type))
    return fail(ctx, SWB_ERR_INVALID_ARGUMENT, "%s: operands must be e4m3 or e5m2, but got types %d and %d", op, a_type, b_type);
  const bool a_needed = rows > 0 && inner > 0, b_needed = inner > 0;
  if ((a_needed && (!A || !a_scales)) || (b_needed && (!B || !b_scales)) || (rows > 0 && !C))
    return fail(ctx, SWB_ERR_INVALID_ARGUMENT, "%s: NULL operand pointer", op);
  swb::GroupedArgs a{rows, inner, n, groups, offsets, A, B, transpose_b != 0, C, a_type};
  a.b_type = b_type;
  a.a_scales = a_scales;
  a.b_scales = b_scales;
  return cuda_status(ctx, rows_product(ctx, a, stream), op);
}

int quantize(swb_context *ctx, const char *op, bool by_rows, int32_t type, int32_t fp8_type, int64_t groups, int64_t rows,
             int64_t cols, const void *X, void *Q, float *scales, swb_stream stream) {
  int st = check_context(ctx);
  if (st != SWB_OK) return st;
  if (type != SWB_BF16 && type != SWB_F16 && type != SWB_F32)
    return fail(ctx, SWB_ERR_INVALID_ARGUMENT, "%s: X must be bf16, f16 or f32, but got type %d", op, type);
  if (!is_fp8(fp8_type))
    return fail(ctx, SWB_ERR_INVALID_ARGUMENT, "%s: the output must be e4m3 or e5m2, but got type %d", op, fp8_type);
  if (groups < 0 || rows < 0 || cols < 0)
    return fail(ctx, SWB_ERR_INVALID_ARGUMENT, "%s: groups, rows and columns must be non-negative", op);
  if (groups > kI32Max || rows > kI32Max - 512 || cols > kI32Max - 512)
    return fail(ctx, SWB_ERR_INVALID_SHAPE, "%s: rows and columns must be below 2^31 - 512", op);
  // blocks of a launch, none of whose products can pass 64 bits
  const __int128 blocks = by_rows ? (__int128)swb::ceil_div(rows, 4) * swb::ceil_div(cols, 128) / 16 + 1
                                  : (__int128)groups * swb::ceil_div(rows, 128) * swb::ceil_div(cols, 128);
  if (blocks > kI32Max) return fail(ctx, SWB_ERR_UNSUPPORTED, "%s: the launch needs more blocks than a CUDA grid holds", op);
  if (groups > 0 && rows > 0 && cols > 0 && (!X || !Q || !scales))
    return fail(ctx, SWB_ERR_INVALID_ARGUMENT, "%s: NULL operand pointer", op);
  const swb::QuantizeArgs a{groups, rows, cols, X, Q, scales, type, fp8_type};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  int64_t *launches = swb::context_launches(ctx);
  return cuda_status(ctx, by_rows ? swb::launch_quantize_rows(a, s, launches) : swb::launch_quantize_blocks(a, s, launches), op);
}

}  // namespace

extern "C" {

int swb_grouped_mm(swb_context *ctx, int32_t dtype, int64_t rows, int64_t inner, int64_t n, int64_t groups,
                   const int32_t *offsets, const void *A, const void *B, int32_t transpose_b, void *C, swb_stream stream) {
  int st = check_context(ctx);
  if (st != SWB_OK) return st;
  st = check_grouped(ctx, "grouped_mm", rows, inner, n, groups);
  if (st != SWB_OK) return st;
  if (dtype != SWB_BF16 && dtype != SWB_F16)
    return fail(ctx, SWB_ERR_INVALID_ARGUMENT, "grouped_mm: operands must be bf16 or f16, but got type %d", dtype);
  if (!offsets || (rows > 0 && inner > 0 && !A) || (inner > 0 && !B) || (rows > 0 && !C))
    return fail(ctx, SWB_ERR_INVALID_ARGUMENT, "grouped_mm: NULL operand pointer");
  const swb::GroupedArgs a{rows, inner, n, groups, offsets, A, B, transpose_b != 0, C, dtype};
  return cuda_status(ctx, rows_product(ctx, a, stream), "grouped_mm");
}

int swb_grouped_mm_grad(swb_context *ctx, int32_t dtype, int64_t rows, int64_t inner, int64_t n, int64_t groups,
                        const int32_t *offsets, const void *A, const void *B, const void *dC, int32_t transpose_b, void *dA,
                        void *dB, swb_stream stream) {
  int st = check_context(ctx);
  if (st != SWB_OK) return st;
  st = check_grouped(ctx, "grouped_mm_grad", rows, inner, n, groups);
  if (st != SWB_OK) return st;
  if (inner < 1) return fail(ctx, SWB_ERR_INVALID_SHAPE, "grouped_mm_grad: the inner size must be at least 1, but got %lld", (long long)inner);
  if (dtype != SWB_BF16 && dtype != SWB_F16)
    return fail(ctx, SWB_ERR_INVALID_ARGUMENT, "grouped_mm_grad: operands must be bf16 or f16, but got type %d", dtype);
  if (!offsets || (rows > 0 && (!dC || (dB && !A))) || (rows > 0 && dA && !B))
    return fail(ctx, SWB_ERR_INVALID_ARGUMENT, "grouped_mm_grad: NULL operand pointer");
  if (dA) {  // dA = dC B^T: the same product with the weights read the other way round
    const swb::GroupedArgs a{rows, n, inner, groups, offsets, dC, B, transpose_b == 0, dA, dtype};
    st = cuda_status(ctx, rows_product(ctx, a, stream), "grouped_mm_grad");
    if (st != SWB_OK) return st;
  }
  if (dB) {
    const swb::GroupedInnerArgs a = transpose_b ? swb::GroupedInnerArgs{rows, n, inner, groups, offsets, dC, A, dB, dtype}
                                                : swb::GroupedInnerArgs{rows, inner, n, groups, offsets, A, dC, dB, dtype};
    st = cuda_status(ctx, inner_product(ctx, a, stream), "grouped_mm_grad");
  }
  return st;
}

int swb_fp8_grouped_mm(swb_context *ctx, int32_t a_dtype, int32_t b_dtype, int64_t rows, int64_t inner, int64_t n,
                       int64_t groups, const int32_t *offsets, const void *A, const float *a_scales, const void *B,
                       const float *b_scales, int32_t transpose_b, uint16_t *C, swb_stream stream) {
  int st = check_context(ctx);
  if (st != SWB_OK) return st;
  st = check_grouped(ctx, "fp8_grouped_mm", rows, inner, n, groups);
  if (st != SWB_OK) return st;
  if (!offsets) return fail(ctx, SWB_ERR_INVALID_ARGUMENT, "fp8_grouped_mm: NULL operand pointer");
  return fp8_product(ctx, "fp8_grouped_mm", a_dtype, b_dtype, rows, inner, n, groups, offsets, A, a_scales, B, b_scales,
                     transpose_b, C, stream);
}

int swb_fp8_mm(swb_context *ctx, int32_t a_dtype, int32_t b_dtype, int64_t rows, int64_t inner, int64_t n, const void *A,
               const float *a_scales, const void *B, const float *b_scales, int32_t transpose_b, uint16_t *C,
               swb_stream stream) {
  int st = check_context(ctx);
  if (st != SWB_OK) return st;
  st = check_grouped(ctx, "fp8_mm", rows, inner, n, 1);
  if (st != SWB_OK) return st;
  return fp8_product(ctx, "fp8_mm", a_dtype, b_dtype, rows, inner, n, 1, nullptr, A, a_scales, B, b_scales, transpose_b, C,
                     stream);
}

int swb_fp8_quantize_rows(swb_context *ctx, int32_t dtype, int32_t fp8_dtype, int64_t rows, int64_t cols, const void *X,
                          void *Q, float *scales, swb_stream stream) {
  return quantize(ctx, "fp8_quantize_rows", true, dtype, fp8_dtype, 1, rows, cols, X, Q, scales, stream);
}

int swb_fp8_quantize_blocks(swb_context *ctx, int32_t dtype, int32_t fp8_dtype, int64_t groups, int64_t rows, int64_t cols,
                            const void *X, void *Q, float *scales, swb_stream stream) {
  return quantize(ctx, "fp8_quantize_blocks", false, dtype, fp8_dtype, groups, rows, cols, X, Q, scales, stream);
}

}  // extern "C"
