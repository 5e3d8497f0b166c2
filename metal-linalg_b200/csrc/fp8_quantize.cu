// Blocks of 1 x 128 or 128 x 128 to 8-bit floating point with a float32 scale each:
//
//     scale = max(max|x| / M, 2^-126),   value = x / scale, a float32, rounded to the nearest (ties to even)
//
// The quotient is correctly rounded, so that the values are the definition's byte for byte. Every kernel reads x once: what
// bounds them is memory, and for 16-bit inputs about as much the issue of 13 to 18 instructions a value, since a block loads,
// waits, computes and stores one after the other.
//   rows     x contiguous along columns, 1 x 128: 16 lanes a block, eight values a lane. 4096 x 4096 in bfloat16 13 us,
//            8192 x 8192 in float32 55 us (6.1 TB/s)
//   tiles    the same in 128 x 128: 256 threads hold the tile as it lies in memory. 4096 x 8192 in bfloat16 23.4 us (4.3 TB/s;
//            22.9 with every zero positive)
//   turned   x contiguous along rows (a transposed matrix): a 128 x 128 tile through shared memory as it lies, read back a
//            quarter of a row of the result a thread, either block shape. 2048 x 4096 in bfloat16 11 us
#include "common.cuh"
#include "fp8.h"
#include "runtime.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace mlb {
namespace fp8 {

namespace {

constexpr int kRowThreads = 256;       // quantize_rows_kernel's
constexpr int kTileThreads = 256;      // quantize_tiles_kernel's
constexpr int kThreads = 512;          // quantize_turned_kernel's
constexpr int kB = 128;

__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float as_float(__half v) { return __half2float(v); }

// The largest of two (three) magnitudes; NaN wins.
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// Pairs of float32 in one instruction.
using Pair = unsigned long long;
__device__ __forceinline__ Pair pair_of(float x, float y) {
    Pair r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
    Pair r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
    Pair r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// x / y, correctly rounded, with r the correctly rounded reciprocal of y: q + (x - q y) r in fused operations for q = x r
// (Markstein, IBM J. Res. Dev. 34, 1990), as long as the remainder is exact. Outside 2^-100 .. 2^120 the remainder can underflow
// (or y is infinite or NaN): there it is the division itself.
__device__ __forceinline__ bool markstein_holds(float y) { return y >= 0x1p-100f && y <= 0x1p120f; }

template <bool kE5m2>
__device__ __forceinline__ float scale_of(float top) {
    constexpr float kMost = kE5m2 ? 57344.0f : 448.0f, kInverse = 1.0f / kMost;
    if (markstein_holds(top)) {                     // the remainder of top / M is as far from underflow as top is
        const float q = top * kInverse;
        return fmaf(fmaf(-q, kMost, top), kInverse, q);
    }
    const float s = __fdiv_rn(top, kMost);
    return s < 1.17549435e-38f ? 1.17549435e-38f : s;          // NaN stays
}
template <bool kE5m2>
__device__ __forceinline__ uint32_t bytes_of(float low, float high) {
    uint16_t r;
    if constexpr (kE5m2) asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;" : "=h"(r) : "f"(high), "f"(low));
    else                 asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(high), "f"(low));
    return r;
}
// N values (a multiple of four) divided by their scale, packed.
template <bool kE5m2, int N>
__device__ __forceinline__ void divided(const float (&v)[N], float scale, uint32_t (&out)[N / 4]) {
    if (!markstein_holds(scale)) {
#pragma unroll
        for (int i = 0; i < N; i += 4)
            out[i / 4] = bytes_of<kE5m2>(__fdiv_rn(v[i], scale), __fdiv_rn(v[i + 1], scale)) |
                         (bytes_of<kE5m2>(__fdiv_rn(v[i + 2], scale), __fdiv_rn(v[i + 3], scale)) << 16);
        return;
    }
    // the quotients' negatives, whose sign of zero is right: with x = -0 the remainder is +0, and added to q = -0 it would leave +0,
    // while (+0)(-r) + (+0) is the +0 that stands for -(-0). (0.25 instructions a value for the signs, back in the packed bytes;
    // no NaN comes here.)
    const float r = -1.0f / scale;
    const Pair r2 = pair_of(r, r), plus = pair_of(scale, scale);
#pragma unroll
    for (int i = 0; i < N; i += 4) {
        uint32_t half[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const Pair x = pair_of(v[i + 2 * j], v[i + 2 * j + 1]), q = mul2(x, r2), y = fma2(fma2(q, plus, x), r2, q);
            float low, high;
            asm("mov.b64 {%0, %1}, %2;" : "=f"(low), "=f"(high) : "l"(y));
            half[j] = bytes_of<kE5m2>(low, high);
        }
        out[i / 4] = (half[0] | (half[1] << 16)) ^ 0x80808080u;
    }
}

// 16 bytes, opaque to the compiler (4096 x 4096 in bfloat16 in rows: 13.0 us, 18.4 where it takes them apart by values) and in
// their place behind the wait for the kernel before this one, which may still write them when this one starts: no __ldg.
__device__ __forceinline__ uint4 load16(const void* at) {
    uint4 r;
    asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(at) : "memory");
    return r;
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
            for (int i = 0; i < kWords; ++i) w[i] = load16(reinterpret_cast<const uint4*>(row + c) + i);
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
    __device__ __forceinline__ float top() const {
        float v[8], t = 0.0f;
        get(v);
#pragma unroll
        for (int i = 0; i < 8; i += 2) t = max_nan(t, fabsf(v[i]), fabsf(v[i + 1]));
        return t;
    }
    template <bool kE5m2> __device__ __forceinline__ uint2 divided_by(float scale) const {
        float v[8];
        uint32_t out[2];
        get(v);
        divided<kE5m2, 8>(v, scale, out);
        return make_uint2(out[0], out[1]);
    }
};

// kUnits blocks of 128 for every 16 lanes, all fetched before the first is used.
template <typename T, bool kE5m2, int kUnits>
__global__ void __launch_bounds__(kRowThreads) quantize_rows_kernel(const QuantizeArgs a) {
    dependency_wait_only();
    const uint32_t blocks = (a.cols + kB - 1) / kB, z = blockIdx.y;
    const uint32_t first = blockIdx.x * (kRowThreads / 16 * kUnits) + (threadIdx.x >> 4);
    const uint32_t in = (threadIdx.x & 15) * 8;
    // one division; the next units are 16 further along the row, or in rows behind it
    uint32_t row[kUnits], block[kUnits];
    row[0] = first / blocks;
    block[0] = first - row[0] * blocks;
#pragma unroll
    for (int i = 1; i < kUnits; ++i) {
        row[i] = row[i - 1];
        block[i] = block[i - 1] + kRowThreads / 16;
        while (block[i] >= blocks) {
            block[i] -= blocks;
            ++row[i];
        }
    }
    Eight<T> x[kUnits];
    const T* src = static_cast<const T*>(a.x) + z * a.batch_stride;
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
        if (row[i] < a.rows) x[i].load(src + (long long)row[i] * a.row_stride, block[i] * kB + in, a.cols, a.vec);
        else                 x[i].clear();          // a unit past the last takes part in the exchange all the same
    }
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
        float top = x[i].top();
#pragma unroll
        for (int o = 1; o < 16; o *= 2) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
        if (row[i] >= a.rows) continue;
        const uint32_t c = block[i] * kB + in;
        const float scale = scale_of<kE5m2>(top);
        if (c < a.cols)
            *reinterpret_cast<uint2*>(a.values + z * a.values_batch + row[i] * a.values_stride + c) = x[i].template divided_by<kE5m2>(scale);
        if ((threadIdx.x & 15) == 0) a.scales[((uint64_t)z * a.rows + row[i]) * blocks + block[i]] = scale;
    }
}

template <int kCount>
__device__ __forceinline__ float block_max(float top, float* shared) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
    if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = top;
    __syncthreads();
    top = shared[0];
#pragma unroll
    for (int i = 1; i < kCount / 32; ++i) top = max_nan(top, shared[i]);
    return top;
}

template <typename T, bool kE5m2>
__global__ void __launch_bounds__(kTileThreads, sizeof(T) == 2 ? 4 : 2) quantize_tiles_kernel(const QuantizeArgs a) {
    dependency_wait_only();
    constexpr int kRows = kTileThreads / 16, kHeld = kB / kRows;
    __shared__ float tops[kTileThreads / 32];
    const uint32_t blocks = (a.cols + kB - 1) / kB, z = blockIdx.y;
    const uint32_t br = blockIdx.x / blocks, bc = blockIdx.x - br * blocks;
    const uint32_t c = bc * kB + (threadIdx.x & 15) * 8, r0 = br * kB + (threadIdx.x >> 4);
    const T* x = static_cast<const T*>(a.x) + z * a.batch_stride;
    Eight<T> held[kHeld];
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
        const uint32_t r = r0 + kRows * i;
        if (r < a.rows) held[i].load(x + (long long)r * a.row_stride, c, a.cols, a.vec);
        else            held[i].clear();
    }
#pragma unroll
    for (int i = 0; i < kHeld; ++i) top = max_nan(top, held[i].top());
    const float scale = scale_of<kE5m2>(block_max<kTileThreads>(top, tops));
    // as they lie in memory until here: unpacked twice, they take half the registers
#pragma unroll
    for (int i = 0; i < kHeld; ++i)
#pragma unroll
        for (int j = 0; j < Eight<T>::kWords; ++j) asm volatile("" : "+r"(held[i].w[j].x), "+r"(held[i].w[j].y), "+r"(held[i].w[j].z), "+r"(held[i].w[j].w));
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
        const uint32_t r = r0 + kRows * i;
        if (r < a.rows && c < a.cols)
            *reinterpret_cast<uint2*>(a.values + z * a.values_batch + r * a.values_stride + c) = held[i].template divided_by<kE5m2>(scale);
    }
    if (threadIdx.x == 0) a.scales[((uint64_t)z * ((a.rows + kB - 1) / kB) + br) * blocks + bc] = scale;
}

// x(r, c) at c * col_stride + r. The tile lies in shared memory as [column][row]; thread (r, part) then takes 32 columns of
// row r, neighbouring lanes neighbouring rows.
template <typename T, bool kE5m2>
__global__ void __launch_bounds__(kThreads, 2) quantize_turned_kernel(const QuantizeArgs a) {
    dependency_wait_only();
    extern __shared__ __align__(16) char raw[];
    T* tile = reinterpret_cast<T*>(raw);
    __shared__ float tops[kThreads];
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
    constexpr int kMine = kB * kB / kThreads;
    const uint32_t r = threadIdx.x & (kB - 1), part = threadIdx.x / kB;
    float v[kMine];
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
        v[i] = as_float(tile[(part * kMine + i) * kB + r]);
        if (i & 1) top = max_nan(top, fabsf(v[i - 1]), fabsf(v[i]));
    }
    if (a.block_rows == 1) {
        tops[threadIdx.x] = top;
        __syncthreads();
        top = max_nan(max_nan(tops[r], tops[kB + r]), max_nan(tops[2 * kB + r], tops[3 * kB + r]));
    } else {
        top = block_max<kThreads>(top, tops);
    }
    const float scale = scale_of<kE5m2>(top);
    if (r0 + r < a.rows) {
        uint8_t* out = a.values + z * a.values_batch + (r0 + r) * a.values_stride + c0 + part * kMine;
#pragma unroll
        for (int i = 0; i < kMine; i += 16)
            if (c0 + part * kMine + i < a.cols) {
                uint32_t bytes[4];
                divided<kE5m2, 16>(*reinterpret_cast<const float (*)[16]>(v + i), scale, bytes);
                *reinterpret_cast<uint4*>(out + i) = make_uint4(bytes[0], bytes[1], bytes[2], bytes[3]);
            }
        if (a.block_rows == 1 && part == 0) a.scales[((uint64_t)z * a.rows + r0 + r) * blocks + bc] = scale;
    }
    if (a.block_rows != 1 && threadIdx.x == 0) a.scales[((uint64_t)z * ((a.rows + kB - 1) / kB) + br) * blocks + bc] = scale;
}

template <typename T, bool kE5m2>
void quantize_as(const QuantizeArgs& a, cudaStream_t stream) {
    const uint64_t blocks = (a.cols + kB - 1) / kB, tiles = (a.rows + kB - 1) / kB * blocks;
    if (a.col_stride != 1) {
        const size_t bytes = sizeof(T) * kB * kB;
        static PerDeviceOnce once;          // the opt-in is recorded per GPU
        if (const int device = current_device(); once.first(device)) {
            cuda_check(cudaFuncSetAttribute(quantize_turned_kernel<T, kE5m2>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes),
                       "quantize shared memory");
            once.mark(device);
        }
        launch_dependent(quantize_turned_kernel<T, kE5m2>, dim3((unsigned)tiles, a.batch), kThreads, bytes, stream, a);
    } else if (a.block_rows == 1) {
        // four blocks of 128 a thread where that still leaves every multiprocessor two thread blocks
        const uint64_t units = a.rows * blocks, each = kRowThreads / 16;
        if (units * a.batch >= 4 * each * 2 * (uint64_t)sm_count(current_device()))
            launch_dependent(quantize_rows_kernel<T, kE5m2, 4>, dim3((unsigned)((units + 4 * each - 1) / (4 * each)), a.batch), kRowThreads, 0, stream, a);
        else
            launch_dependent(quantize_rows_kernel<T, kE5m2, 1>, dim3((unsigned)((units + each - 1) / each), a.batch), kRowThreads, 0, stream, a);
    } else {
        launch_dependent(quantize_tiles_kernel<T, kE5m2>, dim3((unsigned)tiles, a.batch), kTileThreads, 0, stream, a);
    }
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
