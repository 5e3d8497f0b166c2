#pragma once
// Matrices in 8-bit floating point with a float32 scale for each block of 128 (or 128 x 128): the quantiser
// (fp8_quantize.cu), the product (fp8_gemm.cu) and their host side (fp8.cpp).
#include <metal_linalg/c_api.h>

#include <cuda_runtime.h>

#include <cstdint>

namespace mlb {
namespace fp8 {

struct QuantizeArgs {
    const void* x;
    uint32_t    rows, cols, batch;
    long long   batch_stride, row_stride, col_stride;
    uint32_t    block_rows;          // 1 or 128
    int         vec;                 // x can be read in 16-byte pieces along its contiguous dimension
    uint8_t*    values;
    uint64_t    values_stride, values_batch;
    float*      scales;
};
// dtype: of x; e5m2: the values' type. Straight where col_stride is 1, else along row_stride 1.
void launch_quantize(const QuantizeArgs& a, uint32_t dtype, bool e5m2, cudaStream_t stream);

struct GemmOperand {
    const void*  values;
    const float* scales;
    uint64_t     stride, batch_stride;
    bool         e5m2;
    uint32_t     block_rows;
    uint32_t     rows;
};
// c[z][row of a][row of b] = sum over k; enqueued on the current GPU.
void launch_gemm(cudaStream_t stream, int device, const GemmOperand& a, const GemmOperand& b, uint32_t batch, uint32_t k, void* c,
                 uint32_t c_dtype, unsigned* status);

} // namespace fp8
} // namespace mlb

namespace metal_linalg {
namespace core {

// What the C entry points of the same names do (fp8.cpp); std::invalid_argument for what they refuse.
void quantize_fp8(const void* x, uint32_t dtype, uint32_t batch, uint32_t rows, uint32_t cols, int64_t batch_stride,
                  int64_t row_stride, int64_t col_stride, uint32_t block_rows, uint32_t kind, void* values, uint64_t values_stride,
                  float* scales, int device);
void matmul_fp8(const metal_linalg_fp8_operand& a, const metal_linalg_fp8_operand& b, uint32_t batch, uint32_t m, uint32_t n,
                uint32_t k, void* c, uint32_t c_dtype, int device);

} // namespace core
} // namespace metal_linalg
