// The gated delta rule a token at a time, for decoding: states of a pool updated in place.
//
//     s_k = S^T k, s_q = S^T q (before the decay)      d = beta (v - e^g s_k)
//     o = scale (e^g s_q + (k . q) d)                  S <- e^g S + k d^T
//
// Both products with S are taken in one sweep, so that a token needs one exchange between the block's threads. What bounds
// it is the state: 2 x 4 x dk x dv bytes a head, read and written once whatever the number of tokens. A block holds dk rows
// of 32 columns in registers (128 threads: 8 column quads x 16 groups of rows, every load issued before the first is used),
// four blocks a head of 128 columns, so that one request alone still spreads over the multiprocessors. Slots, inputs and
// states are asked for together, ahead of the search for rows of the same slot: 128 rows of 32 heads of 128 x 128 take 100 us
// (5.4 TB/s), 143 with the search first; one row of 8 heads 3.4 us.
#include "common.cuh"
#include "delta.h"
#include "delta_tiles.cuh"
#include "runtime.h"

namespace mlb {
namespace delta {

namespace {

constexpr int kStepThreads = 128;
constexpr int kStepCols = 32;
constexpr int kRowGroups = 16;      // threads that share a column quad
constexpr int kMaxRows = 8;         // rows a thread: dk <= 128

__device__ __forceinline__ long long slot_of(const StepArgs& a, uint32_t row) {
    if (!a.slots) return (long long)row;
    return a.slots64 ? static_cast<const long long*>(a.slots)[row] : (long long)static_cast<const int*>(a.slots)[row];
}

// kVec: a state's rows can be read in pieces of 16 bytes; a thread's four columns are neighbours. Else they lie eight apart, so
// that neighbouring lanes read neighbouring values (128 rows of 32 heads of 128 x 127 112 us, 134 with neighbours).
template <typename T, bool kVec>
__global__ void __launch_bounds__(kStepThreads, 7) delta_step_kernel(const StepArgs a) {
    dependency_wait_only();
    __shared__ float qs[128], ks[128];
    __shared__ float sums[4][2][kStepCols + 4];     // a warp's sums of s_k and s_q, and of k . q behind them
    __shared__ int same[4];                         // a warp's rows of the same slot: 1 there are earlier ones, 2 later ones
    const uint32_t hv = blockIdx.y, row = blockIdx.z, h = hv / (a.value_heads / a.heads);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int quad = threadIdx.x & 7, group = threadIdx.x >> 3;
    constexpr int apart = kVec ? 1 : 8;
    const int col = blockIdx.x * kStepCols + (kVec ? 4 * quad : quad);
    T* o = static_cast<T*>(a.o);
    const long long slot = slot_of(a, row);
    // a token's inputs need no slot: the first one's are on their way with it
    float q_in, k_in, gate, beta, v[4];
    const auto fetch = [&](uint32_t r, uint32_t t) {
        const int at = threadIdx.x;
        const bool there = at < (int)a.dk;
        q_in = there ? to_f(static_cast<const T*>(a.q)[at3(a.q_stride, r, t, h) + at]) : 0.0f;
        k_in = there ? to_f(static_cast<const T*>(a.k)[at3(a.k_stride, r, t, h) + at]) : 0.0f;
        gate = a.g[at3(a.g_stride, r, t, hv)];
        beta = a.beta[at3(a.beta_stride, r, t, hv)];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            v[i] = col + apart * i < (int)a.dv ? to_f(static_cast<const T*>(a.v)[at3(a.v_stride, r, t, hv) + col + apart * i]) : 0.0f;
    };
    fetch(row, 0);
    int found = 0;
    if (a.slots) {
        for (uint32_t r = threadIdx.x; r < a.batch; r += kStepThreads)
            if (r != row && slot_of(a, r) == slot) found |= r < row ? 1 : 2;
    }
    if (slot < 0 || slot >= (long long)a.pool_size) {          // padding
        for (uint32_t t = 0; t < a.tokens; ++t)
            if (group == 0)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (col + apart * i < (int)a.dv)
                        o[(((size_t)row * a.tokens + t) * a.value_heads + hv) * a.dv + col + apart * i] = from_f<T>(0.0f);
        return;
    }
    // the state: every load issued before the first value is needed
    float* pool = a.pool + slot * a.pool_stride + (size_t)hv * a.dk * a.dv;
    float s[kMaxRows][4];
#pragma unroll
    for (int j = 0; j < kMaxRows; ++j) {
        const int r = group + kRowGroups * j;
        const float* src = pool + (size_t)r * a.dv + col;
        if (kVec && r < (int)a.dk && col < (int)a.dv) {
            const float4 f = *reinterpret_cast<const float4*>(src);
            s[j][0] = f.x; s[j][1] = f.y; s[j][2] = f.z; s[j][3] = f.w;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) s[j][i] = r < (int)a.dk && col + apart * i < (int)a.dv ? src[apart * i] : 0.0f;
        }
    }
    // rows of one slot: the first of them runs them all, in order
    {
        const int earlier = __any_sync(0xffffffffu, found & 1), later = __any_sync(0xffffffffu, found & 2);
        if (lane == 0) same[warp] = (earlier ? 1 : 0) | (later ? 2 : 0);
    }
    bool first = true, later = false;
    for (uint32_t r = row; r < a.batch && (first || later); ++r) {
        if (r != row && slot_of(a, r) != slot) continue;
        for (uint32_t t = 0; t < a.tokens; ++t) {
            if (!first) {
                fetch(r, t);
                __syncthreads();                    // the last token's q, k and sums are done with
            }
            qs[threadIdx.x] = q_in;
            ks[threadIdx.x] = k_in;
            __syncthreads();
            if (first) {
                const int all = same[0] | same[1] | same[2] | same[3];
                if (all & 1) return;                // an earlier row of this slot runs this one too
                later = (all & 2) != 0;
                first = false;
            }
            const float decay = expf(gate);
            float sk[4] = {}, sq[4] = {}, kq = 0.0f;
#pragma unroll
            for (int j = 0; j < kMaxRows; ++j) {
                const float q = qs[group + kRowGroups * j], k = ks[group + kRowGroups * j];
                kq = fmaf(k, q, kq);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    sk[i] = fmaf(k, s[j][i], sk[i]);
                    sq[i] = fmaf(q, s[j][i], sq[i]);
                }
            }
#pragma unroll
            for (int m = 8; m < 32; m *= 2) {       // the four row groups of a warp
                kq += __shfl_xor_sync(0xffffffffu, kq, m);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    sk[i] += __shfl_xor_sync(0xffffffffu, sk[i], m);
                    sq[i] += __shfl_xor_sync(0xffffffffu, sq[i], m);
                }
            }
            if (lane < 8) {
                *reinterpret_cast<float4*>(&sums[warp][0][4 * quad]) = make_float4(sk[0], sk[1], sk[2], sk[3]);
                *reinterpret_cast<float4*>(&sums[warp][1][4 * quad]) = make_float4(sq[0], sq[1], sq[2], sq[3]);
                if (lane == 0) sums[warp][0][kStepCols] = kq;
            }
            __syncthreads();
            kq = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i) sk[i] = sq[i] = 0.0f;
#pragma unroll
            for (int w = 0; w < 4; ++w) {           // always in the same order
                kq += sums[w][0][kStepCols];
                const float4 f = *reinterpret_cast<const float4*>(&sums[w][0][4 * quad]);
                const float4 e = *reinterpret_cast<const float4*>(&sums[w][1][4 * quad]);
                sk[0] += f.x; sk[1] += f.y; sk[2] += f.z; sk[3] += f.w;
                sq[0] += e.x; sq[1] += e.y; sq[2] += e.z; sq[3] += e.w;
            }
            float d[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                d[i] = beta * fmaf(-decay, sk[i], v[i]);
                if (group == 0 && col + apart * i < (int)a.dv)
                    o[(((size_t)r * a.tokens + t) * a.value_heads + hv) * a.dv + col + apart * i] =
                        from_f<T>(a.scale * fmaf(decay, sq[i], kq * d[i]));
            }
#pragma unroll
            for (int j = 0; j < kMaxRows; ++j) {
                const float k = ks[group + kRowGroups * j];
#pragma unroll
                for (int i = 0; i < 4; ++i) s[j][i] = fmaf(k, d[i], decay * s[j][i]);
            }
        }
    }
#pragma unroll
    for (int j = 0; j < kMaxRows; ++j) {
        const int r = group + kRowGroups * j;
        float* dst = pool + (size_t)r * a.dv + col;
        if (kVec && r < (int)a.dk && col < (int)a.dv) {
            *reinterpret_cast<float4*>(dst) = make_float4(s[j][0], s[j][1], s[j][2], s[j][3]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (r < (int)a.dk && col + apart * i < (int)a.dv) dst[apart * i] = s[j][i];
        }
    }
}

} // namespace

void launch_step(const StepArgs& a, cudaStream_t stream) {
    const dim3 grid((a.dv + kStepCols - 1) / kStepCols, a.value_heads, a.batch);
    const auto launch = [&](auto plain, auto vec) { launch_dependent(a.vec ? vec : plain, grid, kStepThreads, 0, stream, a); };
    switch (a.dtype) {
        case METAL_LINALG_BFLOAT16: launch(delta_step_kernel<bf16, false>, delta_step_kernel<bf16, true>); break;
        case METAL_LINALG_FLOAT16: launch(delta_step_kernel<__half, false>, delta_step_kernel<__half, true>); break;
        default: launch(delta_step_kernel<float, false>, delta_step_kernel<float, true>); break;
    }
}

} // namespace delta
} // namespace mlb
