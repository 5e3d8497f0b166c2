#pragma once
// Warp-level tensor-core products of the gated delta rule in float32 accuracy, and the loads that feed them.
//
// mma.sync and not tcgen05: the sequential pass is a chain of products of 16 x 64 x 128, each of which needs the one
// before it, and the accumulators of one (a lane holds columns 2t and 2t + 1 of rows g and g + 8) are, with k's order
// permuted in pairs, the A fragment of the next. The chain so stays in a warp's registers: no shared or tensor memory
// and no barrier between its products.
//
// Float32 operands go in parts, smallest products first:
//   bfloat16 inputs   the other operand x = hi + mid + lo in bfloat16 (24 bits): 3 m16n8k16 for a k of 16
//   float16 inputs    x = hi + lo in tf32 (22 bits), the input exact in tf32: 2 x 2 m16n8k8
//   float32 inputs    both in two tf32 parts, lo lo dropped (2^-22): 3 x 2 m16n8k8
// m16n8k16 in 16 bits and m16n8k8 in tf32 both take 8.2 clocks of a multiprocessor's quarter here (measured, eight
// independent accumulators; 21 clocks one after another), so the first form costs three quarters of the second.
#include "delta.h"
#include "runtime.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace mlb {
namespace delta {

using bf16 = __nv_bfloat16;

template <typename T> struct Is16 { static constexpr bool value = sizeof(T) == 2; };

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(bf16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ bf16 from_f<bf16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

// c = a b (kFirst) or c += a b. Not volatile: products of different accumulators may pass one another.
template <bool kFirst>
__device__ __forceinline__ void mma_tf32(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    if constexpr (kFirst)
        asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3},{%4,%5,%6,%7},{%8,%9},{%10,%10,%10,%10};"
            : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
    else
        asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3},{%4,%5,%6,%7},{%8,%9},{%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <bool kFirst>
__device__ __forceinline__ void mma_16(bf16, float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (kFirst)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3},{%4,%5,%6,%7},{%8,%9},{%10,%10,%10,%10};"
            : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3},{%4,%5,%6,%7},{%8,%9},{%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <bool kFirst>
__device__ __forceinline__ void mma_16(__half, float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    static_assert(kFirst, "two float16 operands are multiplied a k of 16 at a time");
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3},{%4,%5,%6,%7},{%8,%9},{%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}

// x to the nearest tf32 (halves away from zero) and what is left, exact in float32; the tensor core cuts the rest's
// last bits, 2^-22 of x. Infinities and NaN keep the result not finite through the rest.
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo) {
    hi = (__float_as_uint(x) + 0x1000u) & 0xFFFFE000u;
    lo = __float_as_uint(x - __uint_as_float(hi));
}
__device__ __forceinline__ uint32_t pack_bf16(float low, float high) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(high), "f"(low));
    return r;
}
__device__ __forceinline__ float low_f(uint32_t packed) { return __uint_as_float(packed << 16); }
__device__ __forceinline__ float high_f(uint32_t packed) { return __uint_as_float(packed & 0xFFFF0000u); }
// two floats as three pairs of bfloat16
__device__ __forceinline__ void split_bf16(float x, float y, uint32_t& hi, uint32_t& mid, uint32_t& lo) {
    hi = pack_bf16(x, y);
    const float x1 = x - low_f(hi), y1 = y - high_f(hi);
    mid = pack_bf16(x1, y1);
    lo = pack_bf16(x1 - low_f(mid), y1 - high_f(mid));
}

// Pairs of float32 in one instruction.
__device__ __forceinline__ void add_to(float (&acc)[4], const float (&c)[4]) {
#pragma unroll
    for (int i = 0; i < 4; i += 2)
        asm("{\n .reg .b64 a, b;\n mov.b64 a, {%0, %1};\n mov.b64 b, {%2, %3};\n add.rn.f32x2 a, a, b;\n mov.b64 {%0, %1}, a;\n}"
            : "+f"(acc[i]), "+f"(acc[i + 1]) : "f"(c[i]), "f"(c[i + 1]));
}
__device__ __forceinline__ void scale_by(float (&acc)[4], float f) {
#pragma unroll
    for (int i = 0; i < 4; i += 2)
        asm("{\n .reg .b64 a, b;\n mov.b64 a, {%0, %1};\n mov.b64 b, {%2, %2};\n mul.rn.f32x2 a, a, b;\n mov.b64 {%0, %1}, a;\n}"
            : "+f"(acc[i]), "+f"(acc[i + 1]) : "f"(f));
}

// ---------------------------------------------------------------------------
// Operands of a k of 16. A pair of accumulator tiles (x: k 0-7, y: k 8-15; element 0 and 1: row g, k 2t and 2t + 1;
// 2 and 3: row g + 8) is an A operand as it stands.
// ---------------------------------------------------------------------------

// One accumulator tile (a k of 8) of a float32 operand, in its parts: what warps that share a chain hand one another.
struct TileTf32 {
    uint4 hi, lo;                   // fragment registers 0-3 of m16n8k8
    __device__ __forceinline__ void set(const float (&x)[4]) {
        split_tf32(x[0], hi.x, lo.x);
        split_tf32(x[2], hi.y, lo.y);
        split_tf32(x[1], hi.z, lo.z);
        split_tf32(x[3], hi.w, lo.w);
    }
    __device__ __forceinline__ void put(uint4* at, int tile, int lane) const {
        at[(2 * tile) * 32 + lane] = hi;
        at[(2 * tile + 1) * 32 + lane] = lo;
    }
    __device__ __forceinline__ void get(const uint4* at, int tile, int lane) {
        hi = at[(2 * tile) * 32 + lane];
        lo = at[(2 * tile + 1) * 32 + lane];
    }
};
struct TileBf16 {
    uint2 part[3];                  // hi, mid, lo; x: row g, y: row g + 8
    __device__ __forceinline__ void set(const float (&x)[4]) {
        split_bf16(x[0], x[1], part[0].x, part[1].x, part[2].x);
        split_bf16(x[2], x[3], part[0].y, part[1].y, part[2].y);
    }
    __device__ __forceinline__ void put(uint4* at, int tile, int lane) const {
        uint2* to = reinterpret_cast<uint2*>(at) + tile * 96 + lane;
#pragma unroll
        for (int i = 0; i < 3; ++i) to[32 * i] = part[i];
    }
    __device__ __forceinline__ void get(const uint4* at, int tile, int lane) {
        const uint2* from = reinterpret_cast<const uint2*>(at) + tile * 96 + lane;
#pragma unroll
        for (int i = 0; i < 3; ++i) part[i] = from[32 * i];
    }
};
constexpr int kTileWords = 2 * 32;      // uint4 of shared memory a tile takes (the larger of the two)

// A float32 operand of a k of 16 in tf32 parts.
struct SplitTf32 {
    uint32_t hi[8], lo[8];
    __device__ __forceinline__ void set(const TileTf32& x, const TileTf32& y) {
        hi[0] = x.hi.x; hi[1] = x.hi.y; hi[2] = x.hi.z; hi[3] = x.hi.w;
        hi[4] = y.hi.x; hi[5] = y.hi.y; hi[6] = y.hi.z; hi[7] = y.hi.w;
        lo[0] = x.lo.x; lo[1] = x.lo.y; lo[2] = x.lo.z; lo[3] = x.lo.w;
        lo[4] = y.lo.x; lo[5] = y.lo.y; lo[6] = y.lo.z; lo[7] = y.lo.w;
    }
    __device__ __forceinline__ void set(const float (&x)[4], const float (&y)[4]) {
        TileTf32 a, b;
        a.set(x);
        b.set(y);
        set(a, b);
    }
};
// The same in bfloat16 parts.
struct SplitBf16 {
    uint32_t part[3][4];     // hi, mid, lo
    __device__ __forceinline__ void set(const TileBf16& x, const TileBf16& y) {
#pragma unroll
        for (int i = 0; i < 3; ++i) {
            part[i][0] = x.part[i].x;
            part[i][1] = x.part[i].y;
            part[i][2] = y.part[i].x;
            part[i][3] = y.part[i].y;
        }
    }
    __device__ __forceinline__ void set(const float (&x)[4], const float (&y)[4]) {
        TileBf16 a, b;
        a.set(x);
        b.set(y);
        set(a, b);
    }
};

// A B operand of a k of 16 and 8 columns read from a tile of T.
template <typename T> struct FragB;
template <> struct FragB<bf16> { uint32_t r[2]; };
template <> struct FragB<__half> { uint32_t r[2]; };
template <> struct FragB<float> { uint32_t hi[4], lo[4]; };   // k 2t, 2t + 1, 2t + 8, 2t + 9

template <typename T> struct Split;                 // the split of the other operand that goes with inputs of type T
template <> struct Split<bf16>   { using type = SplitBf16; using tile = TileBf16; static constexpr int kTerms = 3; };
template <> struct Split<__half> { using type = SplitTf32; using tile = TileTf32; static constexpr int kTerms = 2; };
template <> struct Split<float>  { using type = SplitTf32; using tile = TileTf32; static constexpr int kTerms = 3; };

// One part of the product of a float32 operand with a tile's; term 0 is the smallest, and c's first.
template <int kTerm>
__device__ __forceinline__ void mma_term(float (&c)[4], const SplitBf16& a, const FragB<bf16>& b) {
    mma_16<kTerm == 0>(bf16(), c, a.part[2 - kTerm], b.r[0], b.r[1]);
}
template <int kTerm>
__device__ __forceinline__ void mma_term(float (&c)[4], const SplitTf32& a, const FragB<__half>& b) {
    const uint32_t (&p)[8] = kTerm == 0 ? a.lo : a.hi;
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&b.r[0])), g = __half22float2(*reinterpret_cast<const __half2*>(&b.r[1]));
    mma_tf32<kTerm == 0>(c, p[0], p[1], p[2], p[3], __float_as_uint(f.x), __float_as_uint(f.y));
    mma_tf32<false>(c, p[4], p[5], p[6], p[7], __float_as_uint(g.x), __float_as_uint(g.y));
}
// kExact: the A operand is exact in its first part, so that term 1 is c's first.
template <int kTerm, bool kExact = false>
__device__ __forceinline__ void mma_term(float (&c)[4], const SplitTf32& a, const FragB<float>& b) {
    if constexpr (kExact && kTerm == 0) return;
    const uint32_t (&p)[8] = kTerm == 0 ? a.lo : a.hi;
    const uint32_t (&q)[4] = kTerm == 1 ? b.lo : b.hi;
    mma_tf32<kTerm == (kExact ? 1 : 0)>(c, p[0], p[1], p[2], p[3], q[0], q[1]);
    mma_tf32<false>(c, p[4], p[5], p[6], p[7], q[2], q[3]);
}

__device__ __forceinline__ uint32_t smem_at(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4t(uint32_t addr, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3) : "r"(addr) : "memory");
}

// Two B operands (columns n0 .. n0 + 15, k0 .. k0 + 15) of a tile in shared memory, row length `ld` elements.
// rows: B[k][n] = tile[n][k]; cols: B[k][n] = tile[k][n].
template <typename T>
__device__ __forceinline__ void load_b_rows(FragB<T> (&b)[2], const T* tile, int ld, int n0, int k0) {
    const int lane = threadIdx.x & 31;
    if constexpr (Is16<T>::value) {
        const int r = lane & 7, m = lane >> 3;
        ldmatrix4(smem_at(tile + (n0 + (m >> 1) * 8 + r) * ld + k0 + (m & 1) * 8), b[0].r[0], b[0].r[1], b[1].r[0], b[1].r[1]);
    } else {
        const int g = lane >> 2, t = lane & 3;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const float2 x = *reinterpret_cast<const float2*>(tile + (n0 + 8 * j + g) * ld + k0 + 2 * t);
            const float2 y = *reinterpret_cast<const float2*>(tile + (n0 + 8 * j + g) * ld + k0 + 8 + 2 * t);
            split_tf32(x.x, b[j].hi[0], b[j].lo[0]);
            split_tf32(x.y, b[j].hi[1], b[j].lo[1]);
            split_tf32(y.x, b[j].hi[2], b[j].lo[2]);
            split_tf32(y.y, b[j].hi[3], b[j].lo[3]);
        }
    }
}
template <typename T>
__device__ __forceinline__ void load_b_cols(FragB<T> (&b)[2], const T* tile, int ld, int n0, int k0) {
    const int lane = threadIdx.x & 31;
    if constexpr (Is16<T>::value) {
        const int r = lane & 7, m = lane >> 3;
        ldmatrix4t(smem_at(tile + (k0 + (m & 1) * 8 + r) * ld + n0 + (m >> 1) * 8), b[0].r[0], b[0].r[1], b[1].r[0], b[1].r[1]);
    } else {
        const int g = lane >> 2, t = lane & 3;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const T* at = tile + (k0 + 2 * t) * ld + n0 + 8 * j + g;
            split_tf32(at[0], b[j].hi[0], b[j].lo[0]);
            split_tf32(at[ld], b[j].hi[1], b[j].lo[1]);
            split_tf32(at[8 * ld], b[j].hi[2], b[j].lo[2]);
            split_tf32(at[9 * ld], b[j].hi[3], b[j].lo[3]);
        }
    }
}

// The B operands of columns n0 .. n0 + 8 NT - 1, k0 .. k0 + 15 of a tile.
template <typename T, int NT, bool kCols>
struct Columns {
    FragB<T> b[NT / 2][2];
    __device__ __forceinline__ void load(const T* tile, int ld, int n0, int k0) {
        static_assert(NT % 2 == 0, "columns come in pairs of eight");
#pragma unroll
        for (int j = 0; j < NT / 2; ++j) {
            if constexpr (kCols) load_b_cols<T>(b[j], tile, ld, n0 + 16 * j, k0);
            else                 load_b_rows<T>(b[j], tile, ld, n0 + 16 * j, k0);
        }
    }
};
// acc[n] += the float32 operand `a` times NT columns of eight. The tensor core cuts its sums instead of rounding them, always
// towards zero, so every k of 16 is summed from nothing, smallest parts first, and added in float32: with one accumulator
// all along the gradients were 2e-6 off, an error that grows with the number of additions. The columns' parts are
// issued in turn, so that one's lie NT apart (21 clocks of latency against NT x 8.2).
template <typename T, int NT, bool kCols>
__device__ __forceinline__ void mma_columns(float (*acc)[4], const typename Split<T>::type& a, const Columns<T, NT, kCols>& f) {
    float c[NT][4];
#pragma unroll
    for (int j = 0; j < NT; ++j) mma_term<0>(c[j], a, f.b[j / 2][j & 1]);
#pragma unroll
    for (int j = 0; j < NT; ++j) mma_term<1>(c[j], a, f.b[j / 2][j & 1]);
    if constexpr (Split<T>::kTerms == 3)
#pragma unroll
        for (int j = 0; j < NT; ++j) mma_term<2>(c[j], a, f.b[j / 2][j & 1]);
#pragma unroll
    for (int j = 0; j < NT; ++j) add_to(acc[j], c[j]);
}
// acc[NT] += `a` times the tile's columns n0 .. n0 + 8 NT - 1, k0 .. k0 + 15, four columns of eight at a time.
template <typename T, int NT, bool kCols>
__device__ __forceinline__ void mma_tile(float (&acc)[NT][4], const typename Split<T>::type& a, const T* tile, int ld, int n0,
                                         int k0) {
    constexpr int kGroup = NT % 4 == 0 ? 4 : 2;
#pragma unroll
    for (int n = 0; n < NT; n += kGroup) {
        Columns<T, kGroup, kCols> f;
        f.load(tile, ld, n0 + 8 * n, k0);
        mma_columns<T, kGroup, kCols>(&acc[n], a, f);
    }
}

// The exact product of rows m0 .. m0 + 15 of one tile with rows n0 .. n0 + 8 NT - 1 of another over k0 .. k0 + 15 (16-bit
// inputs: their products are exact in float32, one term; float32 inputs: three).
template <typename T, int NT>
__device__ __forceinline__ void mma_rows_rows(float (&acc)[NT][4], const T* a_tile, int lda, int m0, const T* b_tile, int ldb,
                                              int n0, int k0) {
    const int lane = threadIdx.x & 31;
    if constexpr (Is16<T>::value) {
        const int r = lane & 7, m = lane >> 3;
        uint32_t a[4];
        ldmatrix4(smem_at(a_tile + (m0 + (m & 1) * 8 + r) * lda + k0 + (m >> 1) * 8), a[0], a[1], a[2], a[3]);
#pragma unroll
        for (int n = 0; n < NT; n += 2) {
            FragB<T> b[2];
            load_b_rows<T>(b, b_tile, ldb, n0 + 8 * n, k0);
            float c[2][4];
            mma_16<true>(T(), c[0], a, b[0].r[0], b[0].r[1]);
            mma_16<true>(T(), c[1], a, b[1].r[0], b[1].r[1]);
            add_to(acc[n], c[0]);
            add_to(acc[n + 1], c[1]);
        }
    } else {
        const int g = lane >> 2, t = lane & 3;
        float x[4], y[4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const float2 f = *reinterpret_cast<const float2*>(a_tile + (m0 + 8 * h + g) * lda + k0 + 2 * t);
            const float2 e = *reinterpret_cast<const float2*>(a_tile + (m0 + 8 * h + g) * lda + k0 + 8 + 2 * t);
            x[2 * h] = f.x; x[2 * h + 1] = f.y;
            y[2 * h] = e.x; y[2 * h + 1] = e.y;
        }
        SplitTf32 a;
        a.set(x, y);
        mma_tile<T, NT, false>(acc, a, b_tile, ldb, n0, k0);
    }
}

// The tiles of a lower triangle, (row tile i, column tile j <= i), one after another.
__device__ __forceinline__ constexpr int tri_tile(int i, int j) { return i * (i + 1) / 2 + j; }

// One part of a k of 8 of a float32 operand times a fragment in tf32 parts (hi of k 2t, hi of k 2t + 1, lo, lo); term 0 is c's
// first.
template <int kTerm>
__device__ __forceinline__ void mma_term8(float (&c)[4], const TileTf32& a, const uint4& b) {
    const uint4& p = kTerm == 0 ? a.lo : a.hi;
    mma_tf32<kTerm == 0>(c, p.x, p.y, p.z, p.w, kTerm == 1 ? b.z : b.x, kTerm == 1 ? b.w : b.y);
}
__device__ __forceinline__ uint4 split_pair(float x, float y) {
    uint4 r;
    split_tf32(x, r.x, r.z);
    split_tf32(y, r.y, r.w);
    return r;
}
// acc[i] += a k of 8 of a float32 operand times fragment(i), a lane's k 2t and k 2t + 1, for every i that wanted(i) names, as
// mma_tile.
template <int N, typename Wanted, typename Fragment>
__device__ __forceinline__ void mma_triangle(float (&acc)[N][4], const TileTf32& a, Wanted wanted, Fragment fragment) {
    constexpr int kGroup = N < 4 ? N : 4;
#pragma unroll
    for (int n0 = 0; n0 < N; n0 += kGroup) {
        float c[kGroup][4];
        uint4 b[kGroup];
#pragma unroll
        for (int n = 0; n < kGroup; ++n)
            if (wanted(n0 + n)) {
                const float2 f = fragment(n0 + n);
                b[n] = split_pair(f.x, f.y);
            }
#pragma unroll
        for (int n = 0; n < kGroup; ++n)
            if (wanted(n0 + n)) mma_term8<0>(c[n], a, b[n]);
#pragma unroll
        for (int n = 0; n < kGroup; ++n)
            if (wanted(n0 + n)) mma_term8<1>(c[n], a, b[n]);
#pragma unroll
        for (int n = 0; n < kGroup; ++n)
            if (wanted(n0 + n)) mma_term8<2>(c[n], a, b[n]);
#pragma unroll
        for (int n = 0; n < kGroup; ++n)
            if (wanted(n0 + n)) add_to(acc[n0 + n], c[n]);
    }
}

// ---------------------------------------------------------------------------
// Chunks and tiles
// ---------------------------------------------------------------------------

struct Chunk {
    int batch, token, rows;          // rows 0: no such chunk
};
__device__ __forceinline__ Chunk chunk_at(const Args& a, uint32_t c) {
    Chunk r;
    if (a.sequences) {
        if (c >= (uint32_t)a.first[a.sequences]) return {0, 0, 0};
        const int2 e = reinterpret_cast<const int2*>(a.table)[c];
        r = {0, e.x, e.y};
    } else {
        const uint32_t b = c / a.row_chunks, i = c - b * a.row_chunks;
        r = {(int)b, (int)(i * kChunk), (int)min((uint32_t)kChunk, a.tokens - i * kChunk)};
    }
    return r;
}

// A ragged batch's tokens of no sequence, token(i) of i < count: those before the first sequence, then those behind the last one.
struct Unused {
    long long front, end, count;
    __device__ __forceinline__ explicit Unused(const Args& a)
        : front(a.first[a.sequences + 2]), end(a.first[a.sequences + 1]), count(front + (long long)a.tokens - end) {}
    __device__ __forceinline__ long long token(long long i) const { return i < front ? i : i - front + end; }
};

__device__ __forceinline__ void cp_async16(void* dst, const void* src, bool valid) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" :: "r"(smem_at(dst)), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" :: "n"(N) : "memory"); }

// A tile of kChunk token rows, kWidth columns (a multiple of 8) of which `valid` exist, into shared memory by the kThreads
// threads whose number `tid` is; rows from `rows` on and columns from `valid` on become zero. vec: asynchronously, in
// 16-byte pieces (`valid` columns and all addresses are multiples of 16 bytes then); else value by value, done at the next
// barrier.
template <typename T, int kThreads, int kWidth>
__device__ __forceinline__ void load_rows(T* tile, int ld, const void* base, long long offset, long long stride, int rows, int valid,
                                          bool vec, int tid) {
    const T* src = static_cast<const T*>(base) + offset;
    if (vec) {
        constexpr int kPer = 16 / sizeof(T), kPieces = kWidth / kPer;
        constexpr int kStep = kThreads / kPieces > 0 ? kThreads / kPieces : 1;      // rows at a time
        constexpr int kAcross = kPieces > kThreads ? kPieces / kThreads : 1;
        static_assert(kThreads % kPieces == 0 || kPieces % kThreads == 0, "pieces of a row and threads go into one another");
        const int r0 = kPieces > kThreads ? 0 : tid / kPieces, c0 = kPieces > kThreads ? tid * kPer : (tid % kPieces) * kPer;
#pragma unroll
        for (int a = 0; a < kAcross; ++a) {
            const int c = c0 + a * kThreads * kPer;
            const T* from = src + r0 * stride + c;
            T* to = tile + r0 * ld + c;
            const int limit = c < valid ? rows : 0;
#pragma unroll
            for (int r = 0; r < kChunk; r += kStep) {
                const bool there = r + r0 < limit;
                if (kChunk % kStep == 0 || r + r0 < kChunk) cp_async16(to, there ? from : src, there);
                from += kStep * stride;
                to += kStep * ld;
            }
        }
    } else {
        for (int i = tid; i < kChunk * kWidth; i += kThreads) {
            const int r = i / kWidth, c = i - r * kWidth;
            tile[r * ld + c] = r < rows && c < valid ? src[r * stride + c] : from_f<T>(0.0f);
        }
    }
}
// kCount floats (a multiple of 4, 16-byte aligned on both sides), asynchronously.
template <int kThreads, int kCount>
__device__ __forceinline__ void load_floats(float* dst, const float* src, int tid) {
#pragma unroll
    for (int i = 0; i < kCount / 4; i += kThreads)
        if ((kCount / 4) % kThreads == 0 || i + tid < kCount / 4) cp_async16(dst + 4 * (i + tid), src + 4 * (i + tid), true);
}

__device__ __forceinline__ long long at3(const long long (&stride)[3], long long b, long long t, long long h) {
    return b * stride[0] + t * stride[1] + h * stride[2];
}

// exp of x = h + l, l the small rest: the float exp of h times 1 + l.
__device__ __forceinline__ float exp_of(float h, float l) {
    if (!(h > -104.0f)) return h != h ? h : 0.0f;      // below the smallest float32
    if (h > 88.8f) return __int_as_float(0x7F800000);
    const float e = expf(h);
    return fmaf(e, l, e);
}
__device__ __forceinline__ float exp_of(double x) { return exp_of((float)x, (float)(x - (double)(float)x)); }
// e^{G_i - G_j}. The difference of the leading parts is rounded once, 2^-24 of it: e^-x x 2^-24 is at most 2^-25 of e^0.
__device__ __forceinline__ float decay_of(const Gates& g, int i, int j) { return exp_of(g.sum[i] - g.sum[j], g.rest[i] - g.rest[j]); }

// A chain's 16 value columns as rows of its A operands: fragment rows g and g + 8 are columns 2g and 2g + 1, so that a lane
// reads and writes pairs.
template <typename T> __device__ __forceinline__ float2 pair_at(const T* p) {
    if constexpr (sizeof(T) == 4) return *reinterpret_cast<const float2*>(p);
    else {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(p);
        if constexpr (__is_same(T, __half)) return __half22float2(*reinterpret_cast<const __half2*>(&w));
        else                                return make_float2(low_f(w), high_f(w));
    }
}
template <typename T> __device__ __forceinline__ void put_pair(T* p, float x, float y) {
    if constexpr (sizeof(T) == 4) *reinterpret_cast<float2*>(p) = make_float2(x, y);
    else if constexpr (__is_same(T, __half)) *reinterpret_cast<__half2*>(p) = __floats2half2_rn(x, y);
    else *reinterpret_cast<uint32_t*>(p) = pack_bf16(x, y);
}
// A tile's two token (or key) rows 2t and 2t + 1, `ld` apart.
__device__ __forceinline__ void put_tile(float* p, size_t ld, const float (&x)[4]) {
    *reinterpret_cast<float2*>(p) = make_float2(x[0], x[2]);
    *reinterpret_cast<float2*>(p + ld) = make_float2(x[1], x[3]);
}

// Of a chain's 8 token tiles, the i-th that warp `part` of its KS computes: 0 and 7 together, 1 and 6 ..., so that the
// triangle's work is even.
template <int KS>
__device__ __forceinline__ int own_tile(int part, int i) {
    constexpr int kOwn = 8 / KS;
    return i < kOwn / 2 ? part + KS * i : 7 - (part + KS * (kOwn - 1 - i));
}

// ---------------------------------------------------------------------------
// Launches
// ---------------------------------------------------------------------------

// More than 48 KB of shared memory, recorded per GPU and kernel.
template <auto kKernel>
void opt_in(size_t bytes) {
    static PerDeviceOnce once;
    if (const int device = current_device(); once.first(device)) {
        cuda_check(cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes), "delta rule shared memory");
        once.mark(device);
    }
}

// F<T, DKP> for the problem's type and width.
#define DELTA_DISPATCH(F, a, ...)                                                                        \
    do {                                                                                                 \
        const bool wide = (a).dkp == 128;                                                                \
        switch ((a).dtype) {                                                                             \
            case METAL_LINALG_BFLOAT16: wide ? F<bf16, 128>(a, __VA_ARGS__) : F<bf16, 64>(a, __VA_ARGS__); break; \
            case METAL_LINALG_FLOAT16: wide ? F<__half, 128>(a, __VA_ARGS__) : F<__half, 64>(a, __VA_ARGS__); break; \
            default: wide ? F<float, 128>(a, __VA_ARGS__) : F<float, 64>(a, __VA_ARGS__); break;         \
        }                                                                                                \
    } while (0)

} // namespace delta
} // namespace mlb
