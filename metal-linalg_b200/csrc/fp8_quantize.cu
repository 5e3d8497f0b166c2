// Blocks of 1 x 128 or 128 x 128 to 8-bit floating point with a float32 scale each:
//
//     scale = max(max|x| / M, 2^-126),   value = x / scale, a float32, rounded to the nearest (ties to even)
//
// The quotient is correctly rounded, so that the values are the definition's bit for bit. Every kernel reads x once: what
// bounds them is memory.
//   rows     x contiguous along columns, 1 x 128: 16 lanes a block, eight values a lane
//   tiles    the same in 128 x 128: 256 threads hold the tile in registers
//   turned   x contiguous along rows (a transposed matrix): a 128 x 128 tile through shared memory as it lies, read back a
//            row of the result a thread pair, either block shape
#include "fp8.h"
#include "runtime.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace mlb {
namespace fp8 {

namespace {

constexpr int kThreads = 256;
constexpr int kB = 128;

__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float as_float(__half v) { return __half2float(v); }

// The larger of two magnitudes; NaN wins.
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
template <bool kE5m2>
__device__ __forceinline__ float scale_of(float top) {
    const float s = __fdiv_rn(top, kE5m2 ? 57344.0f : 448.0f);
    return s < 1.17549435e-38f ? 1.17549435e-38f : s;          // NaN stays
}
template <bool kE5m2>
__device__ __forceinline__ uint32_t pair_of(float low, float high) {
    uint16_t r;
    if constexpr (kE5m2) asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;" : "=h"(r) : "f"(high), "f"(low));
    else                 asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(high), "f"(low));
    return r;
}
// x / scale, correctly rounded, for one scale and many x. With r the correctly rounded reciprocal and q = x r,
// q + (x - q scale) r in fused operations is the correctly rounded quotient (Markstein, IBM J. Res. Dev. 34, 1990) as long
// as the remainder is exact: three operations a value instead of a division's ten or so. Outside 2^-100 .. 2^120 the
// remainder can underflow (or the scale is infinite or NaN): there it is the division itself.
struct Quotient {
    float scale, r;
    bool  plain;
    __device__ __forceinline__ explicit Quotient(float s) : scale(s), r(1.0f / s), plain(!(s >= 0x1p-100f && s <= 0x1p120f)) {}
    __device__ __forceinline__ float operator()(float x) const {
        const float q = x * r;
        return fmaf(fmaf(-q, scale, x), r, q);
    }
};
template <bool kE5m2>
__device__ __forceinline__ uint32_t four_of(const float* v, const Quotient& by) {
    if (by.plain)
        return pair_of<kE5m2>(__fdiv_rn(v[0], by.scale), __fdiv_rn(v[1], by.scale)) |
               (pair_of<kE5m2>(__fdiv_rn(v[2], by.scale), __fdiv_rn(v[3], by.scale)) << 16);
    return pair_of<kE5m2>(by(v[0]), by(v[1])) | (pair_of<kE5m2>(by(v[2]), by(v[3])) << 16);
}

// Eight neighbouring values from column c on as they lie in memory; zero behind the last.
template <typename T> struct Eight {
    static constexpr int kWords = sizeof(T) / 2;           // 16-byte words
    uint4 w[kWords];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < kWords; ++i) w[i] = make_uint4(0, 0, 0, 0);
    }
    __device__ __forceinline__ void load(const T* row, uint32_t c, uint32_t cols, bool vec) {
        if (vec && c + 8 <= cols) {
#pragma unroll
            for (int i = 0; i < kWords; ++i) w[i] = __ldg(reinterpret_cast<const uint4*>(row + c) + i);
        } else {
            clear();
            T* e = reinterpret_cast<T*>(w);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (c + i < cols) e[i] = row[c + i];
        }
    }
    __device__ __forceinline__ void get(float (&v)[8]) const {
        const T* e = reinterpret_cast<const T*>(w);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = as_float(e[i]);
    }
};

template <typename T, bool kE5m2>
__global__ void __launch_bounds__(kThreads) quantize_rows_kernel(const QuantizeArgs a) {
    const uint32_t blocks = (a.cols + kB - 1) / kB, z = blockIdx.y;
    const uint64_t unit = ((uint64_t)blockIdx.x * kThreads + threadIdx.x) >> 4;
    const uint64_t units = (uint64_t)a.rows * blocks;
    const bool there = unit < units;                    // whole warps take part in the exchange
    const uint32_t row = there ? (uint32_t)(unit / blocks) : 0, block = there ? (uint32_t)(unit - (uint64_t)row * blocks) : 0;
    const uint32_t c = block * kB + (threadIdx.x & 15) * 8;
    Eight<T> x;
    x.clear();
    if (there) x.load(static_cast<const T*>(a.x) + z * a.batch_stride + (long long)row * a.row_stride, c, a.cols, a.vec);
    float v[8], top = 0.0f;
    x.get(v);
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max_nan(top, fabsf(v[i]));
#pragma unroll
    for (int o = 1; o < 16; o *= 2) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float scale = scale_of<kE5m2>(top);
    if (!there) return;
    const Quotient by(scale);
    if (c < a.cols)
        *reinterpret_cast<uint2*>(a.values + z * a.values_batch + row * a.values_stride + c) =
            make_uint2(four_of<kE5m2>(v, by), four_of<kE5m2>(v + 4, by));
    if ((threadIdx.x & 15) == 0) a.scales[((uint64_t)z * a.rows + row) * blocks + block] = scale;
}

__device__ __forceinline__ float block_max(float top, float* shared) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
    if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = top;
    __syncthreads();
    top = shared[0];
#pragma unroll
    for (int i = 1; i < kThreads / 32; ++i) top = max_nan(top, shared[i]);
    return top;
}

template <typename T, bool kE5m2>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 2 ? 3 : 2) quantize_tiles_kernel(const QuantizeArgs a) {
    __shared__ float tops[kThreads / 32];
    const uint32_t blocks = (a.cols + kB - 1) / kB, z = blockIdx.y;
    const uint32_t br = blockIdx.x / blocks, bc = blockIdx.x - br * blocks;
    const uint32_t c = bc * kB + (threadIdx.x & 15) * 8, r0 = br * kB + (threadIdx.x >> 4);
    const T* x = static_cast<const T*>(a.x) + z * a.batch_stride;
    Eight<T> held[8];
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t r = r0 + 16 * i;
        if (r < a.rows) held[i].load(x + (long long)r * a.row_stride, c, a.cols, a.vec);
        else            held[i].clear();
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        float v[8];
        held[i].get(v);
#pragma unroll
        for (int j = 0; j < 8; ++j) top = max_nan(top, fabsf(v[j]));
    }
    const float scale = scale_of<kE5m2>(block_max(top, tops));
    const Quotient by(scale);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t r = r0 + 16 * i;
        float v[8];
        held[i].get(v);
        if (r < a.rows && c < a.cols)
            *reinterpret_cast<uint2*>(a.values + z * a.values_batch + r * a.values_stride + c) =
                make_uint2(four_of<kE5m2>(v, by), four_of<kE5m2>(v + 4, by));
    }
    if (threadIdx.x == 0) a.scales[((uint64_t)z * ((a.rows + kB - 1) / kB) + br) * blocks + bc] = scale;
}

// x(r, c) at c * col_stride + r. The tile lies in shared memory as [column][row]; thread (r, half) then takes 64 columns of
// row r, neighbouring lanes neighbouring rows.
template <typename T, bool kE5m2>
__global__ void __launch_bounds__(kThreads) quantize_turned_kernel(const QuantizeArgs a) {
    extern __shared__ __align__(16) char raw[];
    T* tile = reinterpret_cast<T*>(raw);
    __shared__ float tops[2 * kB];
    const uint32_t blocks = (a.cols + kB - 1) / kB, z = blockIdx.y;
    const uint32_t br = blockIdx.x / blocks, bc = blockIdx.x - br * blocks;
    const uint32_t r0 = br * kB, c0 = bc * kB;
    const T* x = static_cast<const T*>(a.x) + z * a.batch_stride + r0;
    if (a.vec && r0 + kB <= a.rows) {
        constexpr int kPer = 16 / sizeof(T), kPieces = kB / kPer;
#pragma unroll
        for (int i = threadIdx.x; i < kB * kPieces; i += kThreads) {
            const uint32_t c = i / kPieces, r = (i - c * kPieces) * kPer;
            const bool there = c0 + c < a.cols;
            const T* src = there ? x + (long long)(c0 + c) * a.col_stride + r : x;
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;"
                         :: "r"((uint32_t)__cvta_generic_to_shared(tile + c * kB + r)), "l"(src), "r"(there ? 16 : 0) : "memory");
        }
        asm volatile("cp.async.commit_group;\n cp.async.wait_group 0;" ::: "memory");
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll 16
        for (int i = threadIdx.x; i < kB * kB; i += kThreads) {
            const uint32_t c = i / kB, r = i - c * kB;
            const bool there = c0 + c < a.cols && r0 + r < a.rows;
            const T* src = there ? x + (long long)(c0 + c) * a.col_stride + r : static_cast<const T*>(a.x);
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;"
                         :: "r"((uint32_t)__cvta_generic_to_shared(tile + c * kB + r)), "l"(src), "r"(there ? 4 : 0) : "memory");
        }
        asm volatile("cp.async.commit_group;\n cp.async.wait_group 0;" ::: "memory");
    } else {
#pragma unroll 16
        for (int i = threadIdx.x; i < kB * kB; i += kThreads) {
            const uint32_t c = i / kB, r = i - c * kB;
            tile[c * kB + r] = c0 + c < a.cols && r0 + r < a.rows ? x[(long long)(c0 + c) * a.col_stride + r] : T(0.0f);
        }
    }
    __syncthreads();
    const uint32_t r = threadIdx.x & (kB - 1), half = threadIdx.x / kB;
    float v[kB / 2];
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < kB / 2; ++i) {
        v[i] = as_float(tile[(half * (kB / 2) + i) * kB + r]);
        top = max_nan(top, fabsf(v[i]));
    }
    if (a.block_rows == 1) {
        tops[threadIdx.x] = top;
        __syncthreads();
        top = max_nan(tops[r], tops[kB + r]);
    } else {
        top = block_max(top, tops);
    }
    const float scale = scale_of<kE5m2>(top);
    const Quotient by(scale);
    if (r0 + r < a.rows) {
        uint8_t* out = a.values + z * a.values_batch + (r0 + r) * a.values_stride + c0 + half * (kB / 2);
#pragma unroll
        for (int i = 0; i < kB / 2; i += 16)
            if (c0 + half * (kB / 2) + i < a.cols)
                *reinterpret_cast<uint4*>(out + i) = make_uint4(four_of<kE5m2>(v + i, by), four_of<kE5m2>(v + i + 4, by),
                                                               four_of<kE5m2>(v + i + 8, by), four_of<kE5m2>(v + i + 12, by));
        if (a.block_rows == 1 && half == 0) a.scales[((uint64_t)z * a.rows + r0 + r) * blocks + bc] = scale;
    }
    if (a.block_rows != 1 && threadIdx.x == 0) a.scales[((uint64_t)z * ((a.rows + kB - 1) / kB) + br) * blocks + bc] = scale;
}

template <typename T, bool kE5m2>
void quantize_as(const QuantizeArgs& a, cudaStream_t stream) {
    const uint64_t blocks = (a.cols + kB - 1) / kB, tiles = (a.rows + kB - 1) / kB * blocks;
    if (a.col_stride != 1) {
        const size_t bytes = sizeof(T) * kB * kB;
        cuda_check(cudaFuncSetAttribute(quantize_turned_kernel<T, kE5m2>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes),
                   "quantize shared memory");
        quantize_turned_kernel<T, kE5m2><<<dim3((unsigned)tiles, a.batch), kThreads, bytes, stream>>>(a);
    } else if (a.block_rows == 1) {
        const uint64_t grid = (a.rows * blocks + kThreads / 16 - 1) / (kThreads / 16);
        quantize_rows_kernel<T, kE5m2><<<dim3((unsigned)grid, a.batch), kThreads, 0, stream>>>(a);
    } else {
        quantize_tiles_kernel<T, kE5m2><<<dim3((unsigned)tiles, a.batch), kThreads, 0, stream>>>(a);
    }
    cuda_check(cudaGetLastError(), "quantize launch");
}

} // namespace

void launch_quantize(const QuantizeArgs& a, uint32_t dtype, bool e5m2, cudaStream_t stream) {
    switch (dtype) {
        case METAL_LINALG_BFLOAT16:
            e5m2 ? quantize_as<__nv_bfloat16, true>(a, stream) : quantize_as<__nv_bfloat16, false>(a, stream); break;
        case METAL_LINALG_FLOAT16: e5m2 ? quantize_as<__half, true>(a, stream) : quantize_as<__half, false>(a, stream); break;
        default: e5m2 ? quantize_as<float, true>(a, stream) : quantize_as<float, false>(a, stream); break;
    }
}

} // namespace fp8
} // namespace mlb
