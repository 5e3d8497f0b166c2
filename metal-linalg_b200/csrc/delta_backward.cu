// The gated delta rule's backward kernels (the formulas of the forward stand in delta.h). With dO the outputs' gradient and
// dS' the gradient of the state behind a chunk:
//
//     dD = scale P^T dO + (e^{G_63 - G} K) dS'        dR = T^T dD        dV = beta dR
//     dS = e^{G_63} dS' + scale (e^G Q)^T dO - (beta e^G K)^T dR
//     M_ij = scale e^{G_i - G_j} dO_i . D_j  (j <= i)      N_ij = -beta_i e^{G_i - G_j} dR_i . D_j  (j < i)
//     dQ = scale e^G (dO S^T) + M K
//     dK = M^T Q + (N + N^T) K - beta e^G (dR S^T) + e^{G_63 - G} (D dS'^T)
//     dbeta_i = dR_i . V_i - e^{G_i} k_i . (dR S^T)_i + sum_j N_ij (k_i . k_j) / beta_i
//     dG_i = sum_j W_ij - sum_j W_ji + scale e^{G_i} q_i . (dO S^T)_i - beta_i e^{G_i} k_i . (dR S^T)_i - w_i
//       with W = M . (Q K^T) + N . (K K^T), w_j = e^{G_63 - G_j} k_j . (D dS'^T)_j;  dG_63 += sum_j w_j + e^{G_63} <S, dS'>
//     dg = the sums of dG from the chunk's end
//
// S and D come from the forward's preparation and sequential pass, run again: keeping them from the forward would hold
// 109 kB a chunk and head for the time between (the inputs are 49 kB in bfloat16).
#include "common.cuh"
#include "delta.h"
#include "delta_tiles.cuh"
#include "runtime.h"

namespace mlb {
namespace delta {

namespace {

// ---------------------------------------------------------------------------
// scale P^T dO, ahead of the sequential pass
// ---------------------------------------------------------------------------
//
// A block takes a chunk and a value head, a warp 16 tokens' rows of P^T, whose accumulators stay as the A operand of the second
// product; dO in slices of 64 value columns, two of them asked for with Q and K. Bound by memory's latency, four blocks a
// multiprocessor hide some of it: 64 chunks of 16 heads of 128 x 128 26 us (36 with a slice fetched when its turn came),
// 128 of them 44.

constexpr int kDoThreads = 128;

template <typename T, int DKP>
struct DoShared {
    alignas(16) T     q[kChunk * (DKP + 8)];
    alignas(16) T     k[kChunk * (DKP + 8)];
    alignas(16) T     d_o[2][kChunk * (64 + 8)];
    alignas(16) Gates gates;
};

template <typename T, int DKP>
__global__ void __launch_bounds__(kDoThreads, sizeof(T) == 2 ? 4 : 2) delta_do_kernel(const Args p) {
    dependency_wait_only();
    extern __shared__ __align__(16) char raw[];
    using Sp = typename Split<T>::type;
    DoShared<T, DKP>& sh = *reinterpret_cast<DoShared<T, DKP>*>(raw);
    constexpr int LD = DKP + 8, LDO = 64 + 8;
    const uint32_t c = blockIdx.x, hv = blockIdx.y, h = hv / (p.value_heads / p.heads);
    const Chunk ch = chunk_at(p, c);
    if (ch.rows == 0) return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const size_t at = (size_t)c * p.value_heads + hv;
    load_rows<T, kDoThreads, DKP>(sh.q, LD, p.q, at3(p.q_stride, ch.batch, ch.token, h), p.q_stride[1], ch.rows, (int)p.dk, p.vec, threadIdx.x);
    load_rows<T, kDoThreads, DKP>(sh.k, LD, p.k, at3(p.k_stride, ch.batch, ch.token, h), p.k_stride[1], ch.rows, (int)p.dk, p.vec, threadIdx.x);
    load_floats<kDoThreads, sizeof(Gates) / 4>(reinterpret_cast<float*>(&sh.gates), reinterpret_cast<const float*>(p.gates + at), threadIdx.x);
    cp_commit();
    const auto fetch = [&](int dv0, int which) {            // a slice of dO, if there is one; a group in any case
        if (dv0 < (int)p.dvp)
            load_rows<T, kDoThreads, 64>(sh.d_o[which], LDO, p.d_o, at3(p.do_stride, ch.batch, ch.token, hv) + dv0, p.do_stride[1], ch.rows,
                                         (int)p.dv - dv0, p.vec, threadIdx.x);
        cp_commit();
    };
    fetch(0, 0);
    fetch(64, 1);
    cp_wait<2>();
    __syncthreads();
    // P^T: warp w the rows (tokens j) 16 w .. 16 w + 15; its accumulators are the next product's A operand
    float pt[8][4] = {};
#pragma unroll
    for (int k0 = 0; k0 < DKP; k0 += 16) mma_rows_rows<T, 8>(pt, sh.k, LD, 16 * warp, sh.q, LD, 0, k0);
#pragma unroll
    for (int n = 0; n < 8; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int j = 16 * warp + g + 8 * (i >> 1), r = 8 * n + 2 * t + (i & 1);
            pt[n][i] = r >= j ? p.scale * pt[n][i] * decay_of(sh.gates, r, j) : 0.0f;
        }
    for (int dv0 = 0; dv0 < (int)p.dvp; dv0 += 64) {
        const int which = (dv0 >> 6) & 1;
        cp_wait<1>();
        __syncthreads();
        float acc[8][4] = {};
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
            if (kk < warp) continue;                        // tokens before these: zero
            Sp a;
            a.set(pt[2 * kk], pt[2 * kk + 1]);
            mma_tile<T, 8, true>(acc, a, sh.d_o[which], LDO, 0, 16 * kk);
        }
        float* out = p.dr + at * kChunk * p.dvp;
#pragma unroll
        for (int n = 0; n < 8; ++n) {
            const int column = dv0 + 8 * n + 2 * t;
            if (column < (int)p.dvp) {
                *reinterpret_cast<float2*>(out + (size_t)(16 * warp + g) * p.dvp + column) = make_float2(acc[n][0], acc[n][1]);
                *reinterpret_cast<float2*>(out + (size_t)(16 * warp + 8 + g) * p.dvp + column) = make_float2(acc[n][2], acc[n][3]);
            }
        }
        if (dv0 + 128 < (int)p.dvp) __syncthreads();        // the buffer is free
        fetch(dv0 + 128, which);
    }
}

// ---------------------------------------------------------------------------
// The sequential pass backward: dS and dR
// ---------------------------------------------------------------------------
//
// The forward's chain with dS'^T in the accumulators: Y^T = dS'^T K^T, dD^T = e^{G_63 - G} Y^T + (scale P^T dO)^T,
// dR^T = dD^T T, dS^T = e^{G_63} dS'^T + (scale e^G dO)^T Q - (beta e^G dR)^T K. Bound by the chain, as the forward's: 2.5 us a
// chunk with four warps a chain (3.7 with one stage, where the fetch was waited for), 3.9 us for twice the chains with two.
// 64 chunks of 16 heads of 128 x 128 164 us.
constexpr int kReverseThreads = 192;      // two fetching warps, as the forward's

template <typename T, int DKP, int KS>
struct ReverseShared {
    static constexpr int kGroups = 4 / KS;
    static constexpr int kLdV = 16 * kGroups + 8;
    static constexpr int kStages = sizeof(T) == 4 && KS < 4 ? 1 : 2;       // two of float32 are more than a multiprocessor holds
    struct Stage {
        alignas(16) T     k[kChunk * (DKP + 8)];
        alignas(16) T     q[kChunk * (DKP + 8)];
        alignas(16) T     d_o[kChunk * kLdV];
        alignas(16) float dd[kChunk * kLdV];
        alignas(16) float tri[kTriFloats];
        alignas(16) float gates[3 * kChunk];
    } stage[kStages];
    uint4 part[KS > 1 ? 4 * 8 * 32 : 1];                    // partial Y; then -beta e^G dR in parts
    uint4 dd[KS > 1 ? kGroups * 8 * kTileWords : 1];        // dD in parts
    uint4 d_o[KS > 1 ? kGroups * 8 * kTileWords : 1];       // scale e^G dO in parts
};

template <typename T, int DKP, int KS>
__global__ void __launch_bounds__(kReverseThreads) delta_reverse_kernel(const Args p) {
    dependency_wait_only();
    using Sh = ReverseShared<T, DKP, KS>;
    using Sp = typename Split<T>::type;
    using Tile = typename Split<T>::tile;
    extern __shared__ __align__(16) char raw[];
    Sh& sh = *reinterpret_cast<Sh*>(raw);
    constexpr int LD = DKP + 8, NT = DKP / 8 / KS, LDV = Sh::kLdV, kOwn = 8 / KS;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint32_t hv = blockIdx.y, seq = p.sequences ? p.order[blockIdx.z] : blockIdx.z, h = hv / (p.value_heads / p.heads);
    const int dv_block = blockIdx.x * 16 * Sh::kGroups;
    uint32_t c0, c1;
    if (p.sequences) {
        c0 = p.first[seq];
        c1 = p.first[seq + 1];
    } else {
        c0 = seq * p.row_chunks;
        c1 = c0 + p.row_chunks;
    }
    if (warp >= 4) {
        const int tid = threadIdx.x - 128;
        const auto fetch = [&](uint32_t c, int which) {
            typename Sh::Stage& st = sh.stage[which];
            const Chunk ch = chunk_at(p, c);
            const size_t at = (size_t)c * p.value_heads + hv;
            load_rows<T, 64, DKP>(st.k, LD, p.k, at3(p.k_stride, ch.batch, ch.token, h), p.k_stride[1], ch.rows, (int)p.dk, p.vec, tid);
            load_rows<T, 64, DKP>(st.q, LD, p.q, at3(p.q_stride, ch.batch, ch.token, h), p.q_stride[1], ch.rows, (int)p.dk, p.vec, tid);
            load_rows<T, 64, 16 * Sh::kGroups>(st.d_o, LDV, p.d_o, at3(p.do_stride, ch.batch, ch.token, hv) + dv_block, p.do_stride[1],
                                               ch.rows, (int)p.dv - dv_block, p.vec, tid);
            load_rows<float, 64, 16 * Sh::kGroups>(st.dd, LDV, p.dr, (long long)(at * kChunk * p.dvp) + dv_block, p.dvp, kChunk,
                                                   (int)p.dvp - dv_block, true, tid);
            load_floats<64, kTriFloats>(st.tri, p.tri_b + at * kTriFloats, tid);
            load_floats<64, 3 * kChunk>(st.gates, p.gates[at].e, tid);
            cp_commit();
        };
        if (Sh::kStages == 2 && c0 < c1) fetch(c1 - 1, 0);
        for (uint32_t i0 = 0; i0 < c1 - c0; ++i0) {
            const uint32_t c = c1 - 1 - i0;
            if constexpr (Sh::kStages == 1) {
                __syncthreads();                        // the stage is free
                fetch(c, 0);
            }
            cp_wait<0>();
            __syncthreads();
            if (Sh::kStages == 2 && c > c0) fetch(c - 1, (i0 + 1) & 1);
        }
        return;
    }
    const int chain = warp / KS, part = warp % KS;
    const int dv0 = dv_block + 16 * chain, k_base = part * NT * 8;
    const bool live = dv0 < (int)p.dvp;
    float s[NT][4];                     // dS'^T
    const size_t state0 = ((size_t)seq * p.value_heads + hv) * p.dk * p.dv;
    const auto col = [&](int i) { return dv0 + 2 * g + (i >> 1); };
    const auto row = [&](int n, int i) { return k_base + 8 * n + 2 * t + (i & 1); };
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            s[n][i] = p.d_final && row(n, i) < (int)p.dk && col(i) < (int)p.dv
                          ? p.d_final[state0 + (size_t)row(n, i) * p.dv + col(i)] : 0.0f;

    uint4* dd_parts = sh.dd + (KS > 1 ? chain * 8 * kTileWords : 0);
    uint4* dr_parts = sh.part + (KS > 1 ? chain * 8 * kTileWords : 0);
    uint4* do_parts = sh.d_o + (KS > 1 ? chain * 8 * kTileWords : 0);
    for (uint32_t i0 = 0; i0 < c1 - c0; ++i0) {
        const uint32_t c = c1 - 1 - i0;
        const typename Sh::Stage& st = sh.stage[i0 % Sh::kStages];
        if constexpr (Sh::kStages == 1) __syncthreads();
        __syncthreads();
        const size_t at = (size_t)c * p.value_heads + hv;
        const float *e = st.gates, *left = e + kChunk, *beta = left + kChunk;
        if (live) {
            float* out = p.d_states + at * p.dkp * p.dvp + (size_t)(k_base + 2 * t) * p.dvp + dv0 + 2 * g;
#pragma unroll
            for (int n = 0; n < NT; ++n, out += 8 * p.dvp) put_tile(out, p.dvp, s[n]);
        }
        float x[8][4] = {};
#pragma unroll
        for (int kk = 0; kk < NT / 2; ++kk) {
            Sp a;
            a.set(s[2 * kk], s[2 * kk + 1]);
            mma_tile<T, 8, false>(x, a, st.k, LD, 0, k_base + 16 * kk);
        }
        if constexpr (KS > 1) {
#pragma unroll
            for (int n = 0; n < 8; ++n)
                *reinterpret_cast<float4*>(sh.part + (warp * 8 + n) * 32 + lane) = make_float4(x[n][0], x[n][1], x[n][2], x[n][3]);
            asm volatile("bar.sync %0, %1;" :: "r"(1 + chain), "n"(32 * KS) : "memory");
        }
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
            const int n = KS > 1 ? own_tile<KS>(part, i) : i;
            float f[4] = {};
            if constexpr (KS > 1) {
#pragma unroll
                for (int w = 0; w < KS; ++w) {
                    const float4 q = *reinterpret_cast<const float4*>(sh.part + ((chain * KS + w) * 8 + n) * 32 + lane);
                    const float u[4] = {q.x, q.y, q.z, q.w};
                    add_to(f, u);
                }
            } else {
                add_to(f, x[i]);
            }
            const float2 le = *reinterpret_cast<const float2*>(left + 8 * n + 2 * t);
            const float* dd = st.dd + (8 * n + 2 * t) * LDV + 16 * chain + 2 * g;
            const float2 d0 = pair_at(dd), d1 = pair_at(dd + LDV);
            f[0] = fmaf(le.x, f[0], d0.x);
            f[1] = fmaf(le.y, f[1], d1.x);
            f[2] = fmaf(le.x, f[2], d0.y);
            f[3] = fmaf(le.y, f[3], d1.y);
            if constexpr (KS > 1) {
                TileTf32 a;
                a.set(f);
                a.put(dd_parts, n, lane);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) x[i][j] = f[j];
            }
        }
        const auto out_tile = [&](int n, float (&u)[4]) {          // scale e^G dO of token tile n
            const float2 ee = *reinterpret_cast<const float2*>(e + 8 * n + 2 * t);
            const T* d_o = st.d_o + (8 * n + 2 * t) * LDV + 16 * chain + 2 * g;
            const float2 o0 = pair_at(d_o), o1 = pair_at(d_o + LDV);
            u[0] = p.scale * ee.x * o0.x;
            u[1] = p.scale * ee.y * o1.x;
            u[2] = p.scale * ee.x * o0.y;
            u[3] = p.scale * ee.y * o1.y;
        };
        if constexpr (KS > 1) {
#pragma unroll
            for (int i = 0; i < kOwn; ++i) {
                const int n = own_tile<KS>(part, i);
                float u[4];
                out_tile(n, u);
                Tile a;
                a.set(u);
                a.put(do_parts, n, lane);
            }
            asm volatile("bar.sync %0, %1;" :: "r"(1 + chain), "n"(32 * KS) : "memory");
        }
        // dR^T = dD^T T: tokens from the column's own on
        float d[kOwn][4] = {};
        const float2* tri = reinterpret_cast<const float2*>(st.tri) + lane;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            TileTf32 a;
            if constexpr (KS > 1) a.get(dd_parts, j, lane);
            else                  a.set(x[j]);
            mma_triangle(d, a, [&](int i) { return KS == 1 ? i <= j : i < kOwn / 2 ? j >= 3 || own_tile<KS>(part, i) <= j
                                                                                   : j >= 4 && own_tile<KS>(part, i) <= j; },
                         [&](int i) { return tri[tri_tile(j, KS > 1 ? own_tile<KS>(part, i) : i) * 32]; });
        }
        float* d_out = p.dr + at * kChunk * p.dvp + (size_t)(2 * t) * p.dvp + dv0 + 2 * g;
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
            const int n = KS > 1 ? own_tile<KS>(part, i) : i;
            if (live) put_tile(d_out + (size_t)(8 * n) * p.dvp, p.dvp, d[i]);
            const float2 be = *reinterpret_cast<const float2*>(beta + 8 * n + 2 * t), ee = *reinterpret_cast<const float2*>(e + 8 * n + 2 * t);
            d[i][0] *= -be.x * ee.x; d[i][1] *= -be.y * ee.y; d[i][2] *= -be.x * ee.x; d[i][3] *= -be.y * ee.y;
            if constexpr (KS > 1) {
                Tile a;
                a.set(d[i]);
                a.put(dr_parts, n, lane);
            }
        }
        // dS = e^{G_63} dS' + scale (e^G Q)^T dO - (beta e^G K)^T dR; the part that needs no dR before the barrier
        const float whole = e[kChunk - 1];
#pragma unroll
        for (int n = 0; n < NT; ++n) scale_by(s[n], whole);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            Sp a;
            if constexpr (KS > 1) {
                Tile u, v;
                u.get(do_parts, 2 * j, lane);
                v.get(do_parts, 2 * j + 1, lane);
                a.set(u, v);
            } else {
                float u[4], v[4];
                out_tile(2 * j, u);
                out_tile(2 * j + 1, v);
                a.set(u, v);
            }
            mma_tile<T, NT, true>(s, a, st.q, LD, k_base, 16 * j);
        }
        if constexpr (KS > 1) asm volatile("bar.sync %0, %1;" :: "r"(1 + chain), "n"(32 * KS) : "memory");
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            Sp a;
            if constexpr (KS > 1) {
                Tile u, v;
                u.get(dr_parts, 2 * j, lane);
                v.get(dr_parts, 2 * j + 1, lane);
                a.set(u, v);
            } else {
                a.set(d[2 * j], d[2 * j + 1]);
            }
            mma_tile<T, NT, true>(s, a, st.k, LD, k_base, 16 * j);
        }
    }
    if (p.d_initial)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (row(n, i) < (int)p.dk && col(i) < (int)p.dv) p.d_initial[state0 + (size_t)row(n, i) * p.dv + col(i)] = s[n][i];
}

// ---------------------------------------------------------------------------
// dQ, dK, dV, dbeta, dg of a chunk
// ---------------------------------------------------------------------------
//
// Sixteen warps: 16 tokens (warp % 4) x a quarter of the key columns (warp / 4) of dO S^T, dR S^T and D dS'^T, and as much
// of dO D^T and dR D^T, summed over slices of 16 value columns that are fetched one ahead; then M, N and K K^T, Q K^T. One
// block fills a multiprocessor. What bounds it is the instructions around the products: the tensor core is busy 39 % of the
// time, a slice takes 5200 clocks for 2700 of products, the rest is splitting operands, and sums in float32. (Eight warps of
// twice the columns split fewer operands and take the same time.) 64 chunks of 16 heads of 128 x 128 239 us, 128 of
// them 467.
constexpr int kGradThreads = 512;
constexpr int kLdS = 24;            // row length of a slice: 64-bit fragment reads meet no bank twice
constexpr int kLdM = 72;

template <typename T, int DKP>
struct GradShared {
    alignas(16) T     q[kChunk * (DKP + 8)];
    alignas(16) T     k[kChunk * (DKP + 8)];
    struct Slice {
        alignas(16) float s[DKP * kLdS];
        alignas(16) float ds[DKP * kLdS];
        alignas(16) float d[kChunk * kLdS];
        alignas(16) float dr[kChunk * kLdS];
        alignas(16) T     d_o[kChunk * kLdS];
        alignas(16) T     v[kChunk * kLdS];
    } slice[2];
    alignas(16) float m[kChunk * kLdM];
    alignas(16) float n[kChunk * kLdM];        // N + N^T
    alignas(16) Gates gates;
    float row_w[4][kChunk], row_u[4][kChunk], col_w[4][kChunk];
    float qx[4][kChunk], kx2[4][kChunk], kx3[4][kChunk];
    float drv[kChunk], pair[kGradThreads / 32];
};

// The A operand of a k of 16 from a slice's rows m0 .. m0 + 15: exact for 16-bit values (hi alone), in two parts for float32.
template <typename T>
__device__ __forceinline__ void slice_a(SplitTf32& a, const T* tile, int m0) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    if constexpr (Is16<T>::value) {
        const int r = lane & 7, m = lane >> 3;
        uint32_t f[4];
        ldmatrix4(smem_at(tile + (m0 + (m & 1) * 8 + r) * kLdS + (m >> 1) * 8), f[0], f[1], f[2], f[3]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float lo, hi;
            if constexpr (sizeof(T) == 2 && !__is_same(T, __half)) {
                lo = low_f(f[i]);
                hi = high_f(f[i]);
            } else {
                const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&f[i]));
                lo = x.x;
                hi = x.y;
            }
            // f 0, 1: rows g, g + 8 of k 0-7; f 2, 3: of k 8-15
            a.hi[4 * (i >> 1) + (i & 1)] = __float_as_uint(lo);
            a.hi[4 * (i >> 1) + 2 + (i & 1)] = __float_as_uint(hi);
        }
    } else {
        float x[4], y[4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const float2 f = *reinterpret_cast<const float2*>(tile + (m0 + 8 * h + g) * kLdS + 2 * t);
            const float2 e = *reinterpret_cast<const float2*>(tile + (m0 + 8 * h + g) * kLdS + 8 + 2 * t);
            x[2 * h] = f.x; x[2 * h + 1] = f.y;
            y[2 * h] = e.x; y[2 * h + 1] = e.y;
        }
        a.set(x, y);
    }
}
template <typename T, int DKP>
__global__ void __launch_bounds__(kGradThreads) delta_grad_kernel(const Args p) {
    dependency_wait_only();
    extern __shared__ __align__(16) char raw[];
    using Sh = GradShared<T, DKP>;
    using Sp = typename Split<T>::type;
    Sh& sh = *reinterpret_cast<Sh*>(raw);
    constexpr int LD = DKP + 8, NT = DKP / 32;
    constexpr bool kExact = Is16<T>::value;
    const uint32_t c = blockIdx.x, hv = blockIdx.y, up = p.value_heads / p.heads, h = hv / up;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int m0 = 16 * (warp & 3), part = warp >> 2, n0 = part * (DKP / 4), j0 = 16 * part;
    T *dq = static_cast<T*>(p.dq), *dk = static_cast<T*>(p.dk_out), *dv = static_cast<T*>(p.dv_out);
    const bool pairs = p.dk % 2 == 0 && ((reinterpret_cast<size_t>(dq) | reinterpret_cast<size_t>(dk)) & 7) == 0;
    const Chunk ch = chunk_at(p, c);
    const auto put_qk = [&](size_t token, int column, float q0, float q1, float k0, float k1) {     // columns `column`, + 1
        const size_t to = (token * p.value_heads + hv) * p.dk + column;     // heads and value heads are the same where up is 1
        const bool two = column + 1 < (int)p.dk;
        if (column >= (int)p.dk) return;
        if (pairs) {
            if (up == 1) {
                put_pair(dq + to, q0, q1);
                put_pair(dk + to, k0, k1);
            } else {
                put_pair(p.fold_q + to, q0, q1);
                put_pair(p.fold_k + to, k0, k1);
            }
            return;
        }
        if (up == 1) {
            dq[to] = from_f<T>(q0);
            dk[to] = from_f<T>(k0);
            if (two) {
                dq[to + 1] = from_f<T>(q1);
                dk[to + 1] = from_f<T>(k1);
            }
        } else {
            p.fold_q[to] = q0;
            p.fold_k[to] = k0;
            if (two) {
                p.fold_q[to + 1] = q1;
                p.fold_k[to + 1] = k1;
            }
        }
    };
    if (ch.rows == 0) {             // a ragged batch's blocks behind its chunks: tokens of no sequence get zeros
        const uint32_t used = p.first[p.sequences], spare = gridDim.x - used;
        const Unused none(p);
        for (long long r0 = (long long)(c - used) * kChunk; r0 < none.count; r0 += (long long)spare * kChunk)
            for (int r = warp; r < kChunk && r0 + r < none.count; r += kGradThreads / 32) {
                const size_t token = none.token(r0 + r);
                for (int i = 2 * lane; i < (int)p.dk; i += 64) put_qk(token, i, 0.0f, 0.0f, 0.0f, 0.0f);
                for (int i = lane; i < (int)p.dv; i += 32) dv[(token * p.value_heads + hv) * p.dv + i] = from_f<T>(0.0f);
                if (lane == 0) p.dg[token * p.value_heads + hv] = p.dbeta[token * p.value_heads + hv] = 0.0f;
            }
        return;
    }
    const size_t at = (size_t)c * p.value_heads + hv;
    const size_t token0 = (size_t)ch.batch * p.tokens + ch.token;
    const auto fetch = [&](int dv0, int which) {
        typename Sh::Slice& sl = sh.slice[which];
        const float* s = p.states + at * p.dkp * p.dvp + dv0;
        const float* ds = p.d_states + at * p.dkp * p.dvp + dv0;
        for (int i = threadIdx.x; i < DKP * 4; i += kGradThreads) {
            const int r = i >> 2, q = (i & 3) * 4;
            cp_async16(sl.s + r * kLdS + q, s + (size_t)r * p.dvp + q, true);
            cp_async16(sl.ds + r * kLdS + q, ds + (size_t)r * p.dvp + q, true);
        }
        const float* d = p.d + at * kChunk * p.dvp + dv0;
        const float* dr = p.dr + at * kChunk * p.dvp + dv0;
        {
            const int r = (threadIdx.x & 255) >> 2, q = (threadIdx.x & 3) * 4;
            if (threadIdx.x < 256) cp_async16(sl.d + r * kLdS + q, d + (size_t)r * p.dvp + q, true);
            else                   cp_async16(sl.dr + r * kLdS + q, dr + (size_t)r * p.dvp + q, true);
        }
        load_rows<T, kGradThreads, 16>(sl.d_o, kLdS, p.d_o, at3(p.do_stride, ch.batch, ch.token, hv) + dv0, p.do_stride[1], ch.rows,
                                       (int)p.dv - dv0, p.vec, threadIdx.x);
        load_rows<T, kGradThreads, 16>(sl.v, kLdS, p.v, at3(p.v_stride, ch.batch, ch.token, hv) + dv0, p.v_stride[1], ch.rows,
                                       (int)p.dv - dv0, p.vec, threadIdx.x);
        cp_commit();
    };
    load_rows<T, kGradThreads, DKP>(sh.q, LD, p.q, at3(p.q_stride, ch.batch, ch.token, h), p.q_stride[1], ch.rows, (int)p.dk, p.vec, threadIdx.x);
    load_rows<T, kGradThreads, DKP>(sh.k, LD, p.k, at3(p.k_stride, ch.batch, ch.token, h), p.k_stride[1], ch.rows, (int)p.dk, p.vec, threadIdx.x);
    load_floats<kGradThreads, sizeof(Gates) / 4>(reinterpret_cast<float*>(&sh.gates), reinterpret_cast<const float*>(p.gates + at), threadIdx.x);
    fetch(0, 0);

    float x1[NT][4] = {}, x2[NT][4] = {}, x3[NT][4] = {}, mo[2][4] = {}, mr[2][4] = {};
    float drv = 0.0f, pair = 0.0f;
    for (int dv0 = 0; dv0 < (int)p.dvp; dv0 += 16) {
        const typename Sh::Slice& sl = sh.slice[(dv0 >> 4) & 1];
        cp_wait<0>();
        __syncthreads();
        if (dv0 + 16 < (int)p.dvp) fetch(dv0 + 16, ((dv0 >> 4) + 1) & 1);
        {
            SplitTf32 a_do, a_dr;
            slice_a<T>(a_do, sl.d_o, m0);
            slice_a<float>(a_dr, sl.dr, m0);
            // two tiles of dO and dR against rows of `tile`; every slice from nothing, then added in float32 (see mma_tile)
            const auto both = [&](const float* tile, int row, float (&u)[4], float (&v)[4], float (&w)[4], float (&x)[4]) {
                FragB<float> b[2];
                load_b_rows<float>(b, tile, kLdS, row, 0);
                float c[4][4];
#pragma unroll
                for (int j = 0; j < 2; ++j) { mma_term<0, kExact>(c[j], a_do, b[j]); mma_term<0>(c[2 + j], a_dr, b[j]); }
#pragma unroll
                for (int j = 0; j < 2; ++j) { mma_term<1, kExact>(c[j], a_do, b[j]); mma_term<1>(c[2 + j], a_dr, b[j]); }
#pragma unroll
                for (int j = 0; j < 2; ++j) { mma_term<2, kExact>(c[j], a_do, b[j]); mma_term<2>(c[2 + j], a_dr, b[j]); }
                add_to(u, c[0]);
                add_to(v, c[1]);
                add_to(w, c[2]);
                add_to(x, c[3]);
            };
#pragma unroll
            for (int n = 0; n < NT; n += 2) both(sl.s, n0 + 8 * n, x1[n], x1[n + 1], x2[n], x2[n + 1]);
            if (j0 <= m0) both(sl.d, j0, mo[0], mo[1], mr[0], mr[1]);      // above the diagonal: nothing
        }
        {
            SplitTf32 a_d;
            slice_a<float>(a_d, sl.d, m0);
#pragma unroll
            for (int n = 0; n < NT; n += 2) {
                FragB<float> b[2];
                load_b_rows<float>(b, sl.ds, kLdS, n0 + 8 * n, 0);
                float e[2][4];
#pragma unroll
                for (int j = 0; j < 2; ++j) mma_term<0>(e[j], a_d, b[j]);
#pragma unroll
                for (int j = 0; j < 2; ++j) mma_term<1>(e[j], a_d, b[j]);
#pragma unroll
                for (int j = 0; j < 2; ++j) mma_term<2>(e[j], a_d, b[j]);
#pragma unroll
                for (int j = 0; j < 2; ++j) add_to(x3[n + j], e[j]);
            }
        }
        {           // dV = beta dR, dR . V: a token's two columns a thread
            const int r = threadIdx.x >> 3, q = (threadIdx.x & 7) * 2;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float x = sl.dr[r * kLdS + q + i];
                drv = fmaf(x, to_f(sl.v[r * kLdS + q + i]), drv);
                if (r < ch.rows && dv0 + q + i < (int)p.dv)
                    dv[((token0 + r) * p.value_heads + hv) * p.dv + dv0 + q + i] = from_f<T>(sh.gates.beta[r] * x);
            }
        }
        for (int i = threadIdx.x; i < DKP * 16; i += kGradThreads)
            pair = fmaf(sl.s[(i >> 4) * kLdS + (i & 15)], sl.ds[(i >> 4) * kLdS + (i & 15)], pair);
    }
    drv += __shfl_xor_sync(0xffffffffu, drv, 1);
    drv += __shfl_xor_sync(0xffffffffu, drv, 2);
    drv += __shfl_xor_sync(0xffffffffu, drv, 4);
    if ((threadIdx.x & 7) == 0) sh.drv[threadIdx.x >> 3] = drv;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) pair += __shfl_xor_sync(0xffffffffu, pair, o);
    if (lane == 0) sh.pair[warp] = pair;

    // M, N, and what their products with Q K^T and K K^T give the gates
    {
        float qk[2][4] = {}, kk[2][4] = {};
        if (j0 <= m0)
#pragma unroll
            for (int k0 = 0; k0 < DKP; k0 += 16) {
                mma_rows_rows<T, 2>(qk, sh.q, LD, m0, sh.k, LD, j0, k0);
                mma_rows_rows<T, 2>(kk, sh.k, LD, m0, sh.k, LD, j0, k0);
            }
        float row_w[2] = {0.0f, 0.0f}, row_u[2] = {0.0f, 0.0f};
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            float col[2] = {0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = m0 + g + 8 * (i >> 1), j = j0 + 8 * n + 2 * t + (i & 1);
                float m = 0.0f, w = 0.0f;
                if (j <= r) {
                    const float dec = decay_of(sh.gates, r, j);
                    m = p.scale * dec * mo[n][i];
                    w = m * qk[n][i];
                    if (j < r) {
                        const float u = -dec * mr[n][i], nn = sh.gates.beta[r] * u;
                        row_u[i >> 1] = fmaf(u, kk[n][i], row_u[i >> 1]);
                        w = fmaf(nn, kk[n][i], w);
                        sh.n[r * kLdM + j] = nn;
                        sh.n[j * kLdM + r] = nn;
                    } else {
                        sh.n[r * kLdM + j] = 0.0f;
                    }
                }
                sh.m[r * kLdM + j] = m;
                row_w[i >> 1] += w;
                col[i & 1] += w;
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
#pragma unroll
                for (int o = 4; o < 32; o *= 2) col[i] += __shfl_xor_sync(0xffffffffu, col[i], o);
                if (g == 0) sh.col_w[warp & 3][j0 + 8 * n + 2 * t + i] = col[i];
            }
        }
        float dots[3][2] = {};          // q . X1, k . X2, k . X3 of rows g and g + 8
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = m0 + g + 8 * (i >> 1), column = n0 + 8 * n + 2 * t + (i & 1);
                const float q = to_f(sh.q[r * LD + column]), k = to_f(sh.k[r * LD + column]);
                dots[0][i >> 1] = fmaf(q, x1[n][i], dots[0][i >> 1]);
                dots[1][i >> 1] = fmaf(k, x2[n][i], dots[1][i >> 1]);
                dots[2][i >> 1] = fmaf(k, x3[n][i], dots[2][i >> 1]);
            }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
            for (int o = 1; o < 4; o *= 2) {
                row_w[i] += __shfl_xor_sync(0xffffffffu, row_w[i], o);
                row_u[i] += __shfl_xor_sync(0xffffffffu, row_u[i], o);
#pragma unroll
                for (int j = 0; j < 3; ++j) dots[j][i] += __shfl_xor_sync(0xffffffffu, dots[j][i], o);
            }
            if (t == 0) {
                const int r = m0 + g + 8 * i;
                sh.row_w[part][r] = row_w[i];
                sh.row_u[part][r] = row_u[i];
                sh.qx[part][r] = dots[0][i];
                sh.kx2[part][r] = dots[1][i];
                sh.kx3[part][r] = dots[2][i];
            }
        }
    }
    __syncthreads();

    // dQ and dK
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = m0 + g + 8 * (i >> 1);
            x1[n][i] *= p.scale * sh.gates.e[r];
            x2[n][i] = sh.gates.left[r] * x3[n][i] - sh.gates.beta[r] * sh.gates.e[r] * x2[n][i];
        }
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
        float x[4], y[4];
        Sp a;
        if (16 * kk <= m0) {            // M K
#pragma unroll
            for (int hh = 0; hh < 2; ++hh) {
                const float2 f = *reinterpret_cast<const float2*>(sh.m + (m0 + 8 * hh + g) * kLdM + 16 * kk + 2 * t);
                const float2 e = *reinterpret_cast<const float2*>(sh.m + (m0 + 8 * hh + g) * kLdM + 16 * kk + 8 + 2 * t);
                x[2 * hh] = f.x; x[2 * hh + 1] = f.y;
                y[2 * hh] = e.x; y[2 * hh + 1] = e.y;
            }
            a.set(x, y);
            mma_tile<T, NT, true>(x1, a, sh.k, LD, n0, 16 * kk);
        }
        if (16 * kk >= m0) {            // M^T Q
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[i] = sh.m[(16 * kk + 2 * t + (i & 1)) * kLdM + m0 + g + 8 * (i >> 1)];
                y[i] = sh.m[(16 * kk + 8 + 2 * t + (i & 1)) * kLdM + m0 + g + 8 * (i >> 1)];
            }
            a.set(x, y);
            mma_tile<T, NT, true>(x2, a, sh.q, LD, n0, 16 * kk);
        }
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {        // (N + N^T) K
            const float2 f = *reinterpret_cast<const float2*>(sh.n + (m0 + 8 * hh + g) * kLdM + 16 * kk + 2 * t);
            const float2 e = *reinterpret_cast<const float2*>(sh.n + (m0 + 8 * hh + g) * kLdM + 16 * kk + 8 + 2 * t);
            x[2 * hh] = f.x; x[2 * hh + 1] = f.y;
            y[2 * hh] = e.x; y[2 * hh + 1] = e.y;
        }
        a.set(x, y);
        mma_tile<T, NT, true>(x2, a, sh.k, LD, n0, 16 * kk);
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
            const int r = m0 + g + 4 * i;
            if (r < ch.rows)
                put_qk(token0 + r, n0 + 8 * n + 2 * t, x1[n][i], x1[n][i + 1], x2[n][i], x2[n][i + 1]);
        }

    // the gates' and betas' gradients, two tokens a lane
    if (warp == 0) {
        float dg[2], w[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int r = 2 * lane + j;
            const float e = sh.gates.e[r], beta = sh.gates.beta[r];
            const auto sum = [&](const float (&x)[4][kChunk]) { return (x[0][r] + x[1][r]) + (x[2][r] + x[3][r]); };
            const float kx2 = e * sum(sh.kx2);
            w[j] = sh.gates.left[r] * sum(sh.kx3);
            dg[j] = sum(sh.row_w) - sum(sh.col_w) + p.scale * e * sum(sh.qx) - beta * kx2 - w[j];
            if (r < ch.rows) p.dbeta[(token0 + r) * p.value_heads + hv] = sh.drv[r] - kx2 + sum(sh.row_u);
        }
        float all = w[0] + w[1];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
        float inner = 0.0f;
#pragma unroll
        for (int i = 0; i < kGradThreads / 32; ++i) inner += sh.pair[i];
        if (lane == 31) dg[1] += all + sh.gates.e[kChunk - 1] * inner;
        float sum = dg[0] + dg[1];                      // from this lane's tokens to the chunk's end
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const float v = __shfl_down_sync(0xffffffffu, sum, o);
            if (lane + o < 32) sum += v;
        }
        if (2 * lane < ch.rows) p.dg[(token0 + 2 * lane) * p.value_heads + hv] = sum;
        if (2 * lane + 1 < ch.rows) p.dg[(token0 + 2 * lane + 1) * p.value_heads + hv] = sum - dg[0];
    }
}

// The gradients of shared heads: the sums over the value heads that read them, in their order. A warp takes a token and head.
// Bound by memory: 8192 tokens of 8 heads of
// 128, two value heads each, 25 us (6.7 TB/s of reads and writes, some of them the L2's).
template <typename T, int DKP>
__global__ void __launch_bounds__(256) delta_fold_kernel(const Args p) {
    dependency_wait_only();
    const size_t rows = (size_t)p.batch * p.tokens * p.heads;
    const uint32_t up = p.value_heads / p.heads, lane = threadIdx.x & 31;
    const bool quads = p.dk % 4 == 0 && ((reinterpret_cast<size_t>(p.dq) | reinterpret_cast<size_t>(p.dk_out)) & 15) == 0;
    for (size_t row = (size_t)blockIdx.x * 8 + (threadIdx.x >> 5); row < rows; row += (size_t)gridDim.x * 8) {
        const size_t from = row * up * p.dk, to = row * p.dk;       // [token][head][its value heads][dk]
        if (quads) {
            const uint32_t column = 4 * lane;
            if (column >= p.dk) continue;
            float q[4] = {}, k[4] = {};
            for (uint32_t j = 0; j < up; ++j) {
                const float4 x = *reinterpret_cast<const float4*>(p.fold_q + from + (size_t)j * p.dk + column);
                const float4 y = *reinterpret_cast<const float4*>(p.fold_k + from + (size_t)j * p.dk + column);
                q[0] += x.x; q[1] += x.y; q[2] += x.z; q[3] += x.w;
                k[0] += y.x; k[1] += y.y; k[2] += y.z; k[3] += y.w;
            }
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
                put_pair(static_cast<T*>(p.dq) + to + column + i, q[i], q[i + 1]);
                put_pair(static_cast<T*>(p.dk_out) + to + column + i, k[i], k[i + 1]);
            }
        } else {
            for (uint32_t column = lane; column < p.dk; column += 32) {
                float q = 0.0f, k = 0.0f;
                for (uint32_t j = 0; j < up; ++j) {
                    q += p.fold_q[from + (size_t)j * p.dk + column];
                    k += p.fold_k[from + (size_t)j * p.dk + column];
                }
                static_cast<T*>(p.dq)[to + column] = from_f<T>(q);
                static_cast<T*>(p.dk_out)[to + column] = from_f<T>(k);
            }
        }
    }
}

template <typename T, int DKP, int KS>
void reverse_as(const Args& a, cudaStream_t stream) {
    using Sh = ReverseShared<T, DKP, KS>;
    opt_in<delta_reverse_kernel<T, DKP, KS>>(sizeof(Sh));
    const dim3 grid((a.dvp / 16 + Sh::kGroups - 1) / Sh::kGroups, a.value_heads, a.seqs);
    launch_dependent(delta_reverse_kernel<T, DKP, KS>, grid, kReverseThreads, sizeof(Sh), stream, a);
}

template <typename T, int DKP>
void backward_as(const Args& a, cudaStream_t stream, int sm_count) {
    if (a.chunks) {
        opt_in<delta_do_kernel<T, DKP>>(sizeof(DoShared<T, DKP>));
        launch_dependent(delta_do_kernel<T, DKP>, dim3(a.chunks, a.value_heads), kDoThreads, sizeof(DoShared<T, DKP>), stream, a);
    }
    // Four warps to a chain while there is at most one chain a multiprocessor (their two stages fill it), two up to two chains
    // (or where sequences of uneven lengths leave the longest ones running alone), one beyond, but for float16, whose
    // one-warp chain spills. 64 chunks of 128 x 128 in bfloat16: 128 chains 164 (four) 252 (two) 463 us (one); 256 chains 253 (two)
    // 463 (one); 512 chains 504, 467; 1408 chains of eleven ragged sequences 240, 297. 32 chunks in float32: 128 chains
    // 129, 273, 482; 512 chains 546 (two) 488 (one); in float16: 316, 341.
    const uint64_t chains = (uint64_t)(a.dvp / 16) * a.value_heads * a.seqs;
    if (chains <= (uint64_t)sm_count) reverse_as<T, DKP, 4>(a, stream);
    else if (chains <= 2 * (uint64_t)sm_count || a.sequences || __is_same(T, __half)) reverse_as<T, DKP, 2>(a, stream);
    else if constexpr (!__is_same(T, __half)) reverse_as<T, DKP, 1>(a, stream);
    if (a.chunks) {
        opt_in<delta_grad_kernel<T, DKP>>(sizeof(GradShared<T, DKP>));
        launch_dependent(delta_grad_kernel<T, DKP>, dim3(a.chunks + (a.sequences ? 1 : 0), a.value_heads), kGradThreads, sizeof(GradShared<T, DKP>),
                         stream, a);
        if (a.value_heads != a.heads) {
            const size_t blocks = (size_t)a.batch * a.tokens * a.heads / 8 + 1, most = (size_t)sm_count * 32;
            launch_dependent(delta_fold_kernel<T, DKP>, (unsigned)(blocks < most ? blocks : most), 256, 0, stream, a);
        }
    }
}

} // namespace

void launch_backward(const Args& a, cudaStream_t stream, int sm_count) {
    launch_prepare(a, stream, true);
    launch_states(a, stream, sm_count);
    DELTA_DISPATCH(backward_as, a, stream, sm_count);
}

} // namespace delta
} // namespace mlb
