// Host side of the 8-bit products: what a call may be, and where it runs.
#include "fp8.h"
#include "runtime.h"

#include <metal_linalg/core.h>

#include <stdexcept>
#include <string>

namespace metal_linalg {
namespace core {

namespace {

[[noreturn]] void refuse(const char* who, const std::string& what) { throw std::invalid_argument(std::string(who) + " " + what); }

constexpr uint64_t kMostMatrices = 65535;       // of a quantiser's launch: its grid's second dimension

bool is_fp8(uint32_t kind) { return kind == METAL_LINALG_FLOAT8_E4M3 || kind == METAL_LINALG_FLOAT8_E5M2; }
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Where a call's pointers live: the device its caller vouches for, or what each of them is found to be on.
struct Place {
    const char* who;
    int  device;
    bool known;
    Place(const char* w, int d) : who(w), device(d), known(d >= 0) {
        if (d < -1) refuse(w, "device must be a GPU or -1");
    }
    void need(const void* p, const char* name) {
        if (!p) refuse(who, std::string(name) + " is NULL");
        if (known) return;
        const int d = mlb::pointer_device(p);
        if (d < 0) refuse(who, std::string(name) + " is not a device pointer");
        if (device >= 0 && d != device) refuse(who, std::string(name) + " lives on another GPU than the rest");
        device = d;
    }
};

mlb::fp8::GemmOperand operand(Place& where, char name, const metal_linalg_fp8_operand& o, uint32_t rows, uint32_t k, uint32_t batch) {
    const char* who = where.who;
    const std::string n(1, name);
    if (!is_fp8(o.kind)) refuse(who, n + ".kind must be METAL_LINALG_FLOAT8_E4M3 or _E5M2");
    if (o.block_rows != 1 && o.block_rows != 128) refuse(who, n + ".block_rows must be 1 or 128");
    where.need(o.values, name == 'a' ? "a.values" : "b.values");
    where.need(o.scales, name == 'a' ? "a.scales" : "b.scales");
    if (!aligned16(o.values) || o.stride % 16 || o.batch_stride % 16)
        refuse(who, n + ".values and its strides must be multiples of 16 bytes");
    if (o.stride < k) refuse(who, n + ".stride is smaller than a row");
    if (o.stride >= 1ull << 40 || o.batch_stride >= 1ull << 40) refuse(who, n + ".stride is too large");
    if (batch > 1 && o.batch_stride && (o.batch_stride % o.stride || o.batch_stride / o.stride < rows))
        refuse(who, n + ".batch_stride must be a multiple of its stride, and no smaller than a matrix");
    return {o.values, o.scales, o.stride, o.batch_stride, o.kind == METAL_LINALG_FLOAT8_E5M2, o.block_rows, rows};
}

} // namespace

void quantize_fp8(const void* x, uint32_t dtype, uint32_t batch, uint32_t rows, uint32_t cols, int64_t batch_stride,
                  int64_t row_stride, int64_t col_stride, uint32_t block_rows, uint32_t kind, void* values, uint64_t values_stride,
                  float* scales, int device) {
    const char* who = "[quantize_fp8]";
    if (dtype > METAL_LINALG_FLOAT16) refuse(who, "dtype must be float32, bfloat16 or float16");
    if (!is_fp8(kind)) refuse(who, "kind must be METAL_LINALG_FLOAT8_E4M3 or _E5M2");
    if (block_rows != 1 && block_rows != 128) refuse(who, "block_rows must be 1 or 128");
    if (cpu_only()) throw std::runtime_error(std::string(who) + " this thread is set CPU-only, and this build has no CPU path");
    if (batch == 0 || rows == 0 || cols == 0) return;
    if (col_stride != 1 && row_stride != 1) refuse(who, "one of row_stride and col_stride must be 1");
    if (rows >= 1u << 30 || cols >= 1u << 30 || (uint64_t)rows * ((cols + 127) / 128) >= 1ull << 31)
        refuse(who, "rows and cols must be below 2^30, and the matrix below 2^38 elements");
    if (!aligned16(values) || values_stride % 16 || values_stride < cols)
        refuse(who, "values must be on a 16-byte boundary, its rows a multiple of 16 bytes apart and no shorter than cols");
    Place where(who, device);
    where.need(x, "x");
    where.need(values, "values");
    where.need(scales, "scales");
    const int64_t size = dtype == METAL_LINALG_FLOAT32 ? 4 : 2;
    const int64_t across = col_stride == 1 ? row_stride : col_stride;
    mlb::fp8::QuantizeArgs a{};
    a.rows = rows; a.cols = cols;
    a.batch_stride = batch_stride; a.row_stride = row_stride; a.col_stride = col_stride;
    a.block_rows = block_rows;
    a.vec = aligned16(x) && across * size % 16 == 0 && (batch == 1 || batch_stride * size % 16 == 0);
    a.values_stride = values_stride;
    a.values_batch = values_stride * rows;
    mlb::DeviceGuard guard(where.device);
    const uint64_t scales_batch = (uint64_t)((rows + block_rows - 1) / block_rows) * ((cols + 127) / 128);
    for (uint64_t first = 0; first < batch; first += kMostMatrices) {       // a launch's
        a.batch = (uint32_t)(batch - first < kMostMatrices ? batch - first : kMostMatrices);
        a.x = static_cast<const char*>(x) + (int64_t)first * batch_stride * size;
        a.values = static_cast<uint8_t*>(values) + first * a.values_batch;
        a.scales = scales + first * scales_batch;
        mlb::fp8::launch_quantize(a, dtype, kind == METAL_LINALG_FLOAT8_E5M2, mlb::thread_stream());
    }
}

void matmul_fp8(const metal_linalg_fp8_operand& a, const metal_linalg_fp8_operand& b, uint32_t batch, uint32_t m, uint32_t n,
                uint32_t k, void* c, uint32_t c_dtype, int device) {
    const char* who = "[matmul_fp8]";
    if (c_dtype > METAL_LINALG_FLOAT16) refuse(who, "c must be float32, bfloat16 or float16");
    if (cpu_only()) throw std::runtime_error(std::string(who) + " this thread is set CPU-only, and this build has no CPU path");
    if (batch == 0 || m == 0 || n == 0) return;
    if (m >= 1u << 30 || n >= 1u << 30 || k >= 1u << 30) refuse(who, "m, n and k must be below 2^30");
    Place where(who, device);
    where.need(c, "c");
    if (k == 0) {
        mlb::DeviceGuard guard(where.device);
        mlb::cuda_check(cudaMemsetAsync(c, 0, (size_t)batch * m * n * (c_dtype == METAL_LINALG_FLOAT32 ? 4 : 2), mlb::thread_stream()),
                        "cudaMemsetAsync");
        return;
    }
    const auto oa = operand(where, 'a', a, m, k, batch), ob = operand(where, 'b', b, n, k, batch);
    mlb::DeviceGuard guard(where.device);
    mlb::fp8::launch_gemm(mlb::thread_stream(), where.device, oa, ob, batch, k, c, c_dtype, mlb::status_word(where.device));
}

} // namespace core
} // namespace metal_linalg
