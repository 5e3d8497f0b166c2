// The gated delta rule's forward kernels: the table of chunks, T and the decays (a chunk a block), the sequential pass
// over chunks (16 value columns a chain of products), the outputs (a chunk a block). The formulas stand in delta.h.
#include "common.cuh"
#include "delta.h"
#include "delta_tiles.cuh"
#include "runtime.h"

namespace mlb {
namespace delta {

namespace {

// ---------------------------------------------------------------------------
// Ragged batches: chunk c's first token, length and sequence; every sequence's first chunk
// ---------------------------------------------------------------------------
//
// One block: sums of the sequences' chunks, 256 sequences at a time, then a thread a sequence writes its chunks. The
// sequences are also put in an order for the sequential passes, whose blocks start in it: the long ones first, by classes a
// quarter of an octave wide (any order gives the same results). 4 us for eleven sequences: a launch and a few memory
// round trips.

constexpr int kIndexThreads = 256;

__device__ __forceinline__ long long cu_at(const Args& a, uint32_t i) {
    return a.cu64 ? static_cast<const long long*>(a.cu)[i] : (long long)static_cast<const int*>(a.cu)[i];
}
// The bounds of sequence i, whatever cu_seqlens holds: inside the tokens, and not before their start.
__device__ __forceinline__ void bounds_at(const Args& a, uint32_t i, int& begin, int& end) {
    const long long total = a.tokens;
    const long long b = min(max(cu_at(a, i), 0ll), total), e = min(max(cu_at(a, i + 1), b), total);
    begin = (int)b;
    end = (int)e;
}

constexpr int kClasses = 4 * 31 + 1;
__device__ __forceinline__ int class_of(int chunks) {
    if (chunks <= 0) return 0;
    const int octave = 31 - __clz(chunks);
    return 1 + 4 * octave + (int)((((uint64_t)chunks << 2) >> octave) & 3);
}

__global__ void __launch_bounds__(kIndexThreads) delta_index_kernel(const Args a) {
    dependency_wait();
    __shared__ int sums[kIndexThreads], classes[kClasses];
    __shared__ int carry;
    // Sequences that overlap (a falling cu_seqlens) can name more chunks than there is room for, or than an int counts: every
    // sum stops at the room, and what lies behind it has no chunks. Bounds that do not fall never name more.
    const int room = (int)a.chunks;
    if (threadIdx.x == 0) carry = 0;
    if (threadIdx.x < kClasses) classes[threadIdx.x] = 0;
    __syncthreads();
    for (uint32_t s0 = 0; s0 < a.sequences; s0 += kIndexThreads) {
        const uint32_t s = s0 + threadIdx.x;
        int begin = 0, end = 0;
        if (s < a.sequences) bounds_at(a, s, begin, end);
        const int mine = (end - begin + kChunk - 1) / kChunk;
        sums[threadIdx.x] = min(mine, room);
        __syncthreads();
        for (int o = 1; o < kIndexThreads; o *= 2) {
            const int v = threadIdx.x >= o ? sums[threadIdx.x - o] : 0;
            __syncthreads();
            sums[threadIdx.x] = min(sums[threadIdx.x] + v, room);
            __syncthreads();
        }
        const int first = min(carry + (threadIdx.x ? sums[threadIdx.x - 1] : 0), room);
        const int last = min(carry + sums[threadIdx.x], room);
        if (s < a.sequences) {
            a.first[s] = first;
            atomicAdd(&classes[class_of(mine)], 1);
            for (int c = first; c < last; ++c) {
                const int t = begin + (c - first) * kChunk;
                reinterpret_cast<int2*>(a.table)[c] = make_int2(t, min(kChunk, end - t));
            }
        }
        __syncthreads();
        if (threadIdx.x == 0) carry = min(carry + sums[kIndexThreads - 1], room);
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        int begin, end;
        bounds_at(a, a.sequences - 1, begin, end);
        a.first[a.sequences] = carry;
        a.first[a.sequences + 1] = end;             // tokens from here on belong to no sequence
        bounds_at(a, 0, begin, end);
        a.first[a.sequences + 2] = begin;           // nor do those before
        int before = 0;                             // the sequences of higher classes
        for (int i = kClasses - 1; i >= 0; --i) {
            const int count = classes[i];
            classes[i] = before;
            before += count;
        }
    }
    __syncthreads();
    for (uint32_t s = threadIdx.x; s < a.sequences; s += kIndexThreads) {
        int begin, end;
        bounds_at(a, s, begin, end);
        a.order[atomicAdd(&classes[class_of((end - begin + kChunk - 1) / kChunk)], 1)] = (int)s;
    }
}

// ---------------------------------------------------------------------------
// T = (I + A)^-1 and the decays
// ---------------------------------------------------------------------------
//
// A block takes a chunk and a value head: K K^T (again for every value head that reads the same keys: a tenth of the
// block's time, against twice the blocks), A from it in place, its inverse by blocks of 16 (diagonal blocks by
// substitution, a column a lane; T_ij = -T_ii sum_m A_im T_mj outward from the diagonal on the tensor cores, whose
// transposed inner product is the outer one's operand as it stands) and T as fragments for the products that follow.
// What bounds it is latency, so T takes the place of K in shared memory and five blocks or more fit a multiprocessor (four of
// float32 at 128 key columns).
// 64 chunks of 16 heads of 128 (bfloat16): 27 us; 128 of them 44.
constexpr int kPrepThreads = 128;
constexpr int kLdA = 72;            // row length of A and T in shared memory: 64-bit reads of a fragment meet no bank twice

template <typename T, int DKP>
struct PrepShared {
    union {
        T      k[kChunk * (DKP + 8)];
        float  t[kChunk * kLdA];
    };
    float  a[kChunk * kLdA];
    Gates  gates;
};

template <typename T, int DKP>
__global__ void __launch_bounds__(kPrepThreads) delta_prep_kernel(const Args p, bool backward) {
    dependency_wait_only();
    extern __shared__ __align__(16) char raw[];
    PrepShared<T, DKP>& sh = *reinterpret_cast<PrepShared<T, DKP>*>(raw);
    constexpr int LD = DKP + 8;
    const uint32_t c = blockIdx.x, hv = blockIdx.y, h = hv / (p.value_heads / p.heads);
    const size_t at = (size_t)c * p.value_heads + hv;
    const Chunk ch = chunk_at(p, c);
    if (ch.rows == 0) return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    load_rows<T, kPrepThreads, DKP>(sh.k, LD, p.k, at3(p.k_stride, ch.batch, ch.token, h), p.k_stride[1], ch.rows, (int)p.dk, p.vec, threadIdx.x);
    cp_commit();
    if (warp == 0) {            // the gates' sums, two tokens a lane
        double x[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int r = 2 * lane + j;
            const float gate = r < ch.rows ? p.g[at3(p.g_stride, ch.batch, ch.token + r, hv)] : 0.0f;
            // e^-256 is zero in float32 with room to spare: a gate that closes for good, or -inf, adds no more than that,
            // so that the sums behind it keep their last bits
            x[j] = gate < -256.0f ? -256.0 : (double)gate;
            sh.gates.beta[r] = r < ch.rows ? p.beta[at3(p.beta_stride, ch.batch, ch.token + r, hv)] : 0.0f;
        }
        double sum = x[0] + x[1];
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const double v = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += v;
        }
        const double end = __shfl_sync(0xffffffffu, sum, 31);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const double s = j ? sum : sum - x[1];
            sh.gates.sum[2 * lane + j] = (float)s;
            sh.gates.rest[2 * lane + j] = (float)(s - (double)(float)s);
            sh.gates.e[2 * lane + j] = exp_of(s);
            sh.gates.left[2 * lane + j] = exp_of(end - s);
        }
    }
    cp_wait<0>();
    __syncthreads();
    {       // K K^T: warp w the rows 16 w .. 16 w + 15, columns up to the diagonal's
        float acc[8][4] = {};
#pragma unroll
        for (int k0 = 0; k0 < DKP; k0 += 16) {
            if (warp >= 2) mma_rows_rows<T, 8>(acc, sh.k, LD, 16 * warp, sh.k, LD, 0, k0);
            else           mma_rows_rows<T, 4>(reinterpret_cast<float (&)[4][4]>(acc), sh.k, LD, 16 * warp, sh.k, LD, 0, k0);
        }
#pragma unroll
        for (int n = 0; n < 8; ++n) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int r = 16 * warp + 8 * half + g, q = 8 * n + 2 * t;
                const float beta = sh.gates.beta[r];
                *reinterpret_cast<float2*>(&sh.a[r * kLdA + q]) =
                    make_float2(q < r ? beta * decay_of(sh.gates, r, q) * acc[n][2 * half] : 0.0f,
                                q + 1 < r ? beta * decay_of(sh.gates, r, q + 1) * acc[n][2 * half + 1] : 0.0f);
            }
        }
    }
    __syncthreads();
    {
        const float* src = reinterpret_cast<const float*>(&sh.gates);
        float* dst = reinterpret_cast<float*>(p.gates + at);
        for (int j = threadIdx.x; j < (int)(sizeof(Gates) / 4); j += kPrepThreads) dst[j] = src[j];
    }
    for (int j = threadIdx.x; j < kChunk * kChunk; j += kPrepThreads) sh.t[(j >> 6) * kLdA + (j & 63)] = 0.0f;
    __syncthreads();
    if (lane < 16) {            // diagonal blocks: column `lane` of block `warp`
        const float* a = sh.a + (16 * warp) * kLdA + 16 * warp;
        float x[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            float v = r == lane ? 1.0f : 0.0f;
#pragma unroll
            for (int m = 0; m < r; ++m) v = fmaf(-a[r * kLdA + m], x[m], v);
            x[r] = v;
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) sh.t[(16 * warp + r) * kLdA + 16 * warp + lane] = x[r];
    }
    __syncthreads();
    for (int dist = 1; dist < 4; ++dist) {
        if (warp < 4 - dist) {
            const int bj = warp, bi = warp + dist;
            float w[2][4] = {};                                     // W^T, W = sum_m A_im T_mj: rows are T's columns
            for (int m = bj; m < bi; ++m) {
                const float* tm = sh.t + (16 * m) * kLdA + 16 * bj;     // T_mj
                const float* am = sh.a + (16 * bi) * kLdA + 16 * m;     // A_im
                const float x[4] = {tm[2 * t * kLdA + g], tm[(2 * t + 1) * kLdA + g], tm[2 * t * kLdA + g + 8], tm[(2 * t + 1) * kLdA + g + 8]};
                const float y[4] = {tm[(2 * t + 8) * kLdA + g], tm[(2 * t + 9) * kLdA + g], tm[(2 * t + 8) * kLdA + g + 8],
                                    tm[(2 * t + 9) * kLdA + g + 8]};
                SplitTf32 s;
                s.set(x, y);
                mma_tile<float, 2, false>(w, s, am, kLdA, 0, 0);
            }
            float out[2][4] = {};
            const float* ti = sh.t + (16 * bi) * kLdA + 16 * bi;        // T_ii
#pragma unroll
            for (int k8 = 0; k8 < 2; ++k8) {
                const float2 u = *reinterpret_cast<const float2*>(ti + g * kLdA + 8 * k8 + 2 * t);
                const float2 v = *reinterpret_cast<const float2*>(ti + (g + 8) * kLdA + 8 * k8 + 2 * t);
                const float x[4] = {-u.x, -u.y, -v.x, -v.y};
                TileTf32 s;
                s.set(x);
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    const uint4 b = split_pair(w[k8][2 * n], w[k8][2 * n + 1]);
                    float c[4];
                    mma_term8<0>(c, s, b);
                    mma_term8<1>(c, s, b);
                    mma_term8<2>(c, s, b);
                    add_to(out[n], c);
                }
            }
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                float* o = sh.t + (16 * bi + g) * kLdA + 16 * bj + 8 * n + 2 * t;
                *reinterpret_cast<float2*>(o) = make_float2(out[n][0], out[n][1]);
                *reinterpret_cast<float2*>(o + 8 * kLdA) = make_float2(out[n][2], out[n][3]);
            }
        }
        __syncthreads();
    }
    for (int tile = warp; tile < kTriTiles; tile += kPrepThreads / 32) {
        int ti = 0;
        while (tri_tile(ti + 1, 0) <= tile) ++ti;
        const int tj = tile - tri_tile(ti, 0);
        const float2 f = *reinterpret_cast<const float2*>(sh.t + (8 * ti + g) * kLdA + 8 * tj + 2 * t);
        reinterpret_cast<float2*>(p.tri + at * kTriFloats)[tile * 32 + lane] = f;
        if (backward)
            reinterpret_cast<float2*>(p.tri_b + at * kTriFloats)[tile * 32 + lane] =
                make_float2(sh.t[(8 * ti + 2 * t) * kLdA + 8 * tj + g], sh.t[(8 * ti + 2 * t + 1) * kLdA + 8 * tj + g]);
    }
}

// ---------------------------------------------------------------------------
// The sequential pass
// ---------------------------------------------------------------------------
//
// A chain is 16 value columns: S^T [16 x dk] lives in accumulators. X^T = S^T K^T; R^T = beta (V^T - e^G X^T);
// D^T = R^T T^T; S^T = e^{G_63} S^T + (D^T e^{G_63 - G}) K: every product's accumulators are the next one's A operand, and
// K comes from shared memory as B operands both ways round. KS warps share a chain, each with dk / KS of S's rows, since
// a chain is a sequence of dependent products and there are few chains; partial X crosses through shared memory as whole
// fragments (a lane's 16 bytes, no bank met twice), R and D already in their parts. Two more warps fetch the next chunk
// meanwhile (one took longer to issue its copies than the chain to use them). A chain is alone on its quarter of the
// multiprocessor, so what a product needs besides the one before it is read ahead of the barrier that opens it.
//
// What bounds it is the chain: a chunk takes 1.7 us (X 970 clocks, T R 470, S 590, the rest R, exchanges and
// barriers), whatever the number of chains up to one a multiprocessor; 64 chunks of 16 heads of 128 x 128 108 us. Beside the
// outputs of chunks already done, on a second stream, it slowed to 2.7 us a chunk and the whole gained nothing.
constexpr int kStateThreads = 192;

template <typename T, int DKP, int KS>
struct StateShared {
    static constexpr int kGroups = 4 / KS;          // chains of a block
    static constexpr int kLdV = 16 * kGroups + 8;
    struct Stage {
        alignas(16) T     k[kChunk * (DKP + 8)];
        alignas(16) T     v[kChunk * kLdV];
        alignas(16) float tri[kTriFloats];
        alignas(16) float gates[3 * kChunk];        // e, left, beta
    } stage[2];
    // [warp][tile][lane]: partial X; then, when every R is there, [chain][tile]: e^{G_63 - G} D in parts
    uint4 part[4 * 8 * 32];
    uint4 r[kGroups * 8 * kTileWords];              // [chain][tile]: R in parts
};

template <typename T, int DKP, int KS>
__global__ void __launch_bounds__(kStateThreads, sizeof(T) == 2 ? 2 : 1) delta_state_kernel(const Args p) {
    dependency_wait_only();
    using Sh = StateShared<T, DKP, KS>;
    using Sp = typename Split<T>::type;
    using Tile = typename Split<T>::tile;
    extern __shared__ __align__(16) char raw[];
    Sh& sh = *reinterpret_cast<Sh*>(raw);
    constexpr int LD = DKP + 8, NT = DKP / 8 / KS, kOwn = 8 / KS;
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
    if (warp >= 4) {            // the fetching warps: a chunk ahead, complete at the barrier that opens it
        const int tid = threadIdx.x - 128;
        const auto fetch = [&](uint32_t c, int which) {
            typename Sh::Stage& st = sh.stage[which];
            const Chunk ch = chunk_at(p, c);
            const size_t at = (size_t)c * p.value_heads + hv;
            load_rows<T, 64, DKP>(st.k, LD, p.k, at3(p.k_stride, ch.batch, ch.token, h), p.k_stride[1], ch.rows, (int)p.dk, p.vec, tid);
            load_rows<T, 64, 16 * Sh::kGroups>(st.v, Sh::kLdV, p.v, at3(p.v_stride, ch.batch, ch.token, hv) + dv_block, p.v_stride[1],
                                               ch.rows, (int)p.dv - dv_block, p.vec, tid);
            load_floats<64, kTriFloats>(st.tri, p.tri + at * kTriFloats, tid);
            load_floats<64, 3 * kChunk>(st.gates, p.gates[at].e, tid);
            cp_commit();
        };
        if (c0 < c1) fetch(c0, 0);
        for (uint32_t c = c0; c < c1; ++c) {
            cp_wait<0>();
            __syncthreads();
            if (c + 1 < c1) fetch(c + 1, (c - c0 + 1) & 1);
        }
        return;
    }
    const int chain = warp / KS, part = warp % KS;
    const int dv0 = dv_block + 16 * chain, k_base = part * NT * 8;
    const bool live = dv0 < (int)p.dvp;                 // a chain past the last columns computes on zeros and writes nothing

    float s[NT][4];
    const size_t state0 = ((size_t)seq * p.value_heads + hv) * p.dk * p.dv;
    const auto col = [&](int i) { return dv0 + 2 * g + (i >> 1); };
    const auto row = [&](int n, int i) { return k_base + 8 * n + 2 * t + (i & 1); };
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            s[n][i] = p.initial_state && row(n, i) < (int)p.dk && col(i) < (int)p.dv
                          ? p.initial_state[state0 + (size_t)row(n, i) * p.dv + col(i)] : 0.0f;

    uint4* r_parts = sh.r + chain * 8 * kTileWords;
    uint4* d_parts = sh.part + chain * 8 * kTileWords;
    for (uint32_t c = c0; c < c1; ++c) {
        const typename Sh::Stage& st = sh.stage[(c - c0) & 1];
        __syncthreads();                                // this chunk is here, and every warp is done with the one before
        const size_t at = (size_t)c * p.value_heads + hv;
        const float *e = st.gates, *left = e + kChunk, *beta = left + kChunk;

        // the state at the chunk's start
        if (live) {
            float* out = p.states + at * p.dkp * p.dvp + (size_t)(k_base + 2 * t) * p.dvp + dv0 + 2 * g;
#pragma unroll
            for (int n = 0; n < NT; ++n, out += 8 * p.dvp) put_tile(out, p.dvp, s[n]);
        }

        // X^T, the next k's operands on their way while one is multiplied
        float x[8][4] = {};
        {
            Columns<T, 8, false> f[2];
            f[0].load(st.k, LD, 0, k_base);
#pragma unroll
            for (int kk = 0; kk < NT / 2; ++kk) {
                if (kk + 1 < NT / 2) f[(kk + 1) & 1].load(st.k, LD, 0, k_base + 16 * (kk + 1));
                Sp a;
                a.set(s[2 * kk], s[2 * kk + 1]);
                mma_columns<T, 8, false>(x, a, f[kk & 1]);
            }
        }
#pragma unroll
        for (int n = 0; n < 8; ++n)
            *reinterpret_cast<float4*>(sh.part + (warp * 8 + n) * 32 + lane) = make_float4(x[n][0], x[n][1], x[n][2], x[n][3]);
        // what R and D of this warp's token tiles need besides
        float value[kOwn][4];
        float2 beta2[kOwn], e2[kOwn], left2[kOwn], t_lo[kOwn / 2][4], t_hi[kOwn / 2][8];
        const float2* tri = reinterpret_cast<const float2*>(st.tri) + lane;
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
            const int n = own_tile<KS>(part, i);
            const T* v = st.v + (8 * n + 2 * t) * Sh::kLdV + 16 * chain + 2 * g;
            const float2 v0 = pair_at(v), v1 = pair_at(v + Sh::kLdV);
            value[i][0] = v0.x;
            value[i][1] = v1.x;
            value[i][2] = v0.y;
            value[i][3] = v1.y;
            beta2[i] = *reinterpret_cast<const float2*>(beta + 8 * n + 2 * t);
            e2[i] = *reinterpret_cast<const float2*>(e + 8 * n + 2 * t);
            left2[i] = *reinterpret_cast<const float2*>(left + 8 * n + 2 * t);
        }
        // T's tiles: own_tile's first half lies in rows 0-3, the second in rows 4-7; those past the diagonal are not used
#pragma unroll
        for (int i = 0; i < kOwn / 2; ++i) {
#pragma unroll
            for (int j = 0; j < 4; ++j) t_lo[i][j] = tri[tri_tile(own_tile<KS>(part, i), min(j, own_tile<KS>(part, i))) * 32];
#pragma unroll
            for (int j = 0; j < 8; ++j)
                t_hi[i][j] = tri[tri_tile(own_tile<KS>(part, kOwn / 2 + i), min(j, own_tile<KS>(part, kOwn / 2 + i))) * 32];
        }
        asm volatile("bar.sync %0, %1;" :: "r"(1 + chain), "n"(32 * KS) : "memory");
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
            const int n = own_tile<KS>(part, i);
            float f[4] = {};
#pragma unroll
            for (int w = 0; w < KS; ++w) {          // always in the same order
                const float4 q = *reinterpret_cast<const float4*>(sh.part + ((chain * KS + w) * 8 + n) * 32 + lane);
                const float u[4] = {q.x, q.y, q.z, q.w};
                add_to(f, u);
            }
            f[0] = beta2[i].x * fmaf(-e2[i].x, f[0], value[i][0]);
            f[1] = beta2[i].y * fmaf(-e2[i].y, f[1], value[i][1]);
            f[2] = beta2[i].x * fmaf(-e2[i].x, f[2], value[i][2]);
            f[3] = beta2[i].y * fmaf(-e2[i].y, f[3], value[i][3]);
            TileTf32 a;
            a.set(f);
            a.put(r_parts, n, lane);
        }
        asm volatile("bar.sync %0, %1;" :: "r"(1 + chain), "n"(32 * KS) : "memory");
        // D^T = R^T T^T, two k's of 8 at a time against the rows of T that reach them
        float d[kOwn][4] = {};
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            TileTf32 a[2];
            a[0].get(r_parts, j, lane);
            a[1].get(r_parts, j + 1, lane);
            float c[2][kOwn][4];
            uint4 b[2][kOwn];
            const auto wanted = [&](int i, int u) {     // mostly known beforehand
                return i < kOwn / 2 ? u < 4 && own_tile<KS>(part, i) >= u : u <= 4 || own_tile<KS>(part, i) >= u;
            };
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int i = 0; i < kOwn; ++i)
                    if (wanted(i, j + u)) {
                        const float2 f = i < kOwn / 2 ? t_lo[i][(j + u) & 3] : t_hi[i - kOwn / 2][j + u];
                        b[u][i] = split_pair(f.x, f.y);
                        mma_term8<0>(c[u][i], a[u], b[u][i]);
                    }
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int i = 0; i < kOwn; ++i)
                    if (wanted(i, j + u)) mma_term8<1>(c[u][i], a[u], b[u][i]);
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int i = 0; i < kOwn; ++i)
                    if (wanted(i, j + u)) mma_term8<2>(c[u][i], a[u], b[u][i]);
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int i = 0; i < kOwn; ++i)
                    if (wanted(i, j + u)) add_to(d[i], c[u][i]);
        }
        // e^{G_63 - G} D to the chain's other warps, D itself to memory
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
            const float f[4] = {d[i][0] * left2[i].x, d[i][1] * left2[i].y, d[i][2] * left2[i].x, d[i][3] * left2[i].y};
            Tile a;
            a.set(f);
            a.put(d_parts, own_tile<KS>(part, i), lane);
        }
        Columns<T, NT, true> f[2];
        f[0].load(st.k, LD, k_base, 0);
        asm volatile("bar.sync %0, %1;" :: "r"(1 + chain), "n"(32 * KS) : "memory");
        // S' = e^{G_63} S + (e^{G_63 - G} K)^T D
        const float whole = e[kChunk - 1];
#pragma unroll
        for (int n = 0; n < NT; ++n) scale_by(s[n], whole);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (j < 3) f[(j + 1) & 1].load(st.k, LD, k_base, 16 * (j + 1));
            Sp a;
            Tile u, v;
            u.get(d_parts, 2 * j, lane);
            v.get(d_parts, 2 * j + 1, lane);
            a.set(u, v);
            mma_columns<T, NT, true>(s, a, f[j & 1]);
        }
        if (live) {
            float* d_out = p.d + at * kChunk * p.dvp + (size_t)(2 * t) * p.dvp + dv0 + 2 * g;
#pragma unroll
            for (int i = 0; i < kOwn; ++i) put_tile(d_out + (size_t)(8 * own_tile<KS>(part, i)) * p.dvp, p.dvp, d[i]);
        }
    }
    if (p.final_state)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (row(n, i) < (int)p.dk && col(i) < (int)p.dv) p.final_state[state0 + (size_t)row(n, i) * p.dv + col(i)] = s[n][i];
}

// ---------------------------------------------------------------------------
// The outputs
// ---------------------------------------------------------------------------
//
// A block takes a chunk and a value head; a warp 16 value columns of all 64 tokens: O^T = S^T (e^G Q)^T + D^T P^T, with S
// and D read from memory as A operands (each value once, split once), Q from shared memory, and P (20 tiles of 16 x 8 over
// the warps) kept there as the B fragments that its accumulators are. What bounds it is memory's latency and then the tensor
// core: with 16-bit inputs all of S is on its way to shared memory and all of D to registers while P is made, two blocks a
// multiprocessor (float32: half of S in registers, each further part fetched while the one before it is multiplied). 64
// chunks of 16 heads of 128 x 128: 59 us (S, D, Q, K and O at 2.3 TB/s; 70 with S by registers); 128 chunks 109.
constexpr int kOutThreads = 256;
constexpr int kOutCols = 16 * (kOutThreads / 32);       // value columns at a time

template <typename T, int DKP>
struct OutShared {
    alignas(16) T q[kChunk * (DKP + 8)];
    union {
        alignas(16) T k[kChunk * (DKP + 8)];
        T o[kChunk * (kOutCols + 8)];                   // the outputs on their way to memory, whole rows at a time
    };
    alignas(16) float2 p[kTriTiles * 32];
    alignas(16) Gates  gates;
    // S, where two blocks a multiprocessor still have room for it; 64-bit reads of a fragment meet no bank twice
    static constexpr bool kStaged = sizeof(T) == 2;
    static constexpr int  kLdS = kOutCols + 4;
    alignas(16) float  s[kStaged ? DKP * kLdS : 4];
};

template <typename T, int DKP>
__global__ void __launch_bounds__(kOutThreads, 2) delta_output_kernel(const Args p) {
    dependency_wait_only();
    extern __shared__ __align__(16) char raw[];
    using Sh = OutShared<T, DKP>;
    using Sp = typename Split<T>::type;
    Sh& sh = *reinterpret_cast<Sh*>(raw);
    constexpr int LD = DKP + 8, kHeld = Sh::kStaged ? 4 : DKP / 32, LDO = kOutCols + 8;
    const uint32_t c = blockIdx.x, hv = blockIdx.y, h = hv / (p.value_heads / p.heads);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    T* o = static_cast<T*>(p.o);
    const Chunk ch = chunk_at(p, c);
    if (ch.rows == 0) {             // a ragged batch's blocks behind its chunks: tokens of no sequence become zero
        const uint32_t used = p.first[p.sequences], spare = gridDim.x - used;
        const Unused none(p);
        for (long long r0 = (long long)(c - used) * kChunk; r0 < none.count; r0 += (long long)spare * kChunk)
            for (int i = threadIdx.x; i < kChunk * (int)p.dv; i += kOutThreads) {
                const long long r = r0 + i / (int)p.dv;
                if (r < none.count) o[(none.token(r) * p.value_heads + hv) * p.dv + i % (int)p.dv] = from_f<T>(0.0f);
            }
        return;
    }
    const size_t at = (size_t)c * p.value_heads + hv;
    load_rows<T, kOutThreads, DKP>(sh.q, LD, p.q, at3(p.q_stride, ch.batch, ch.token, h), p.q_stride[1], ch.rows, (int)p.dk, p.vec, threadIdx.x);
    load_rows<T, kOutThreads, DKP>(sh.k, LD, p.k, at3(p.k_stride, ch.batch, ch.token, h), p.k_stride[1], ch.rows, (int)p.dk, p.vec, threadIdx.x);
    load_floats<kOutThreads, sizeof(Gates) / 4>(reinterpret_cast<float*>(&sh.gates), reinterpret_cast<const float*>(p.gates + at), threadIdx.x);
    cp_commit();
    // a k of 16 of S^T or D^T as two accumulator tiles: rows 2t, 2t + 1, 2t + 8, 2t + 9 of columns 2g, 2g + 1
    float2 held[kHeld][4];
    const auto fetch = [&](const float* base, int row, float2 (&to)[4]) {
        const float* src = base + (size_t)(row + 2 * t) * p.dvp + 2 * g;
        to[0] = *reinterpret_cast<const float2*>(src);
        to[1] = *reinterpret_cast<const float2*>(src + p.dvp);
        src += 8 * p.dvp;
        to[2] = *reinterpret_cast<const float2*>(src);
        to[3] = *reinterpret_cast<const float2*>(src + p.dvp);
    };
    const auto tiles = [](const float2 (&from)[4], float (&x)[4], float (&y)[4]) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            x[i] = from[i].x;
            x[2 + i] = from[i].y;
            y[i] = from[2 + i].x;
            y[2 + i] = from[2 + i].y;
        }
    };
    const float *s = p.states + at * p.dkp * p.dvp, *d = p.d + at * kChunk * p.dvp;
    // staged: all of the warp's own columns of S to shared memory and of D to registers, else half of S's to registers
    float* mine = sh.s + 16 * warp;
    const auto ahead = [&](int dv0) {
        if constexpr (Sh::kStaged) {
            const int r = lane >> 2, q = (lane & 3) * 4;
#pragma unroll
            for (int i = 0; i < DKP; i += 8) cp_async16(mine + (i + r) * Sh::kLdS + q, s + (size_t)(i + r) * p.dvp + dv0 + q, true);
        }
#pragma unroll
        for (int i = 0; i < kHeld; ++i) fetch((Sh::kStaged ? d : s) + dv0, 16 * i, held[i]);
    };
    if (16 * warp < (int)p.dvp) ahead(16 * warp);
    cp_commit();
    cp_wait<1>();
    __syncthreads();
    // P's tiles of 16 x 8 on and below the diagonal, two neighbours at a time: (0, 0), (1, 0), (1, 1), (2, 0) ...
    for (int pair = warp; pair < 10; pair += kOutThreads / 32) {
        int a = 0;
        while ((a + 1) * (a + 2) / 2 <= pair) ++a;
        const int j16 = pair - a * (a + 1) / 2;
        float acc[2][4] = {};
#pragma unroll
        for (int k0 = 0; k0 < DKP; k0 += 16) mma_rows_rows<T, 2>(acc, sh.q, LD, 16 * a, sh.k, LD, 16 * j16, k0);
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            float f[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = 16 * a + g + 8 * (i >> 1), q = 16 * j16 + 8 * n + 2 * t + (i & 1);
                f[i] = q <= r ? acc[n][i] * decay_of(sh.gates, r, q) : 0.0f;
            }
            const int j8 = 2 * j16 + n;
            if (j8 <= 2 * a) sh.p[tri_tile(2 * a, j8) * 32 + lane] = make_float2(f[0], f[1]);
            sh.p[tri_tile(2 * a + 1, j8) * 32 + lane] = make_float2(f[2], f[3]);
        }
    }
    __syncthreads();
    for (int pass = 0; pass < (int)p.dvp; pass += kOutCols) {
        const int dv0 = pass + 16 * warp;
        if (dv0 < (int)p.dvp) {
            [[maybe_unused]] const float *sv = s + dv0, *dv = d + dv0;
            if (pass) {
                ahead(dv0);             // (every lane is past the barrier behind its last reads)
                cp_commit();
            }
            float acc[8][4] = {};
            if constexpr (Sh::kStaged) {
                cp_wait<0>();
                __syncwarp();
#pragma unroll
                for (int kk = 0; kk < DKP / 16; ++kk) {
                    const float* at = mine + (16 * kk + 2 * t) * Sh::kLdS + 2 * g;
                    const float2 f[4] = {pair_at(at), pair_at(at + Sh::kLdS), pair_at(at + 8 * Sh::kLdS), pair_at(at + 9 * Sh::kLdS)};
                    float x[4], y[4];
                    tiles(f, x, y);
                    Sp a;
                    a.set(x, y);
                    mma_tile<T, 8, false>(acc, a, sh.q, LD, 0, 16 * kk);
                }
            } else {
#pragma unroll
                for (int kk = 0; kk < 2 * kHeld; ++kk) {
                    float x[4], y[4];
                    tiles(held[kk % kHeld], x, y);
                    if (kk < kHeld) fetch(sv, 16 * (kHeld + kk), held[kk]);
                    else            fetch(dv, 16 * (kk - kHeld), held[kk - kHeld]);
                    Sp a;
                    a.set(x, y);
                    mma_tile<T, 8, false>(acc, a, sh.q, LD, 0, 16 * kk);
                }
            }
#pragma unroll
            for (int n = 0; n < 8; ++n) {
                const float2 e = *reinterpret_cast<const float2*>(sh.gates.e + 8 * n + 2 * t);
                acc[n][0] *= e.x; acc[n][1] *= e.y; acc[n][2] *= e.x; acc[n][3] *= e.y;
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float x[2][4];
                tiles(held[j % kHeld], x[0], x[1]);
                if (j + kHeld < 4) fetch(dv, 16 * (j + kHeld), held[j % kHeld]);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    TileTf32 a;
                    a.set(x[i]);
                    mma_triangle(acc, a, [&](int n) { return n >= 2 * j + i; }, [&](int n) { return sh.p[tri_tile(n, 2 * j + i) * 32 + lane]; });
                }
            }
#pragma unroll
            for (int n = 0; n < 8; ++n)
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    put_pair(sh.o + (8 * n + 2 * t + i) * LDO + 16 * warp + 2 * g, p.scale * acc[n][i], p.scale * acc[n][2 + i]);
        }
        __syncthreads();
        const int width = min(kOutCols, (int)p.dv - pass);
        T* to = o + (((size_t)ch.batch * p.tokens + ch.token) * p.value_heads + hv) * p.dv + pass;
        const size_t step = (size_t)p.value_heads * p.dv;
        constexpr int kPer = 16 / sizeof(T), kPieces = kOutCols / kPer;
        if (p.dv % kPer == 0 && (reinterpret_cast<size_t>(o) & 15) == 0) {
            for (int i = threadIdx.x; i < ch.rows * kPieces; i += kOutThreads) {
                const int r = i / kPieces, q = (i % kPieces) * kPer;
                if (q < width) *reinterpret_cast<uint4*>(to + r * step + q) = *reinterpret_cast<const uint4*>(sh.o + r * LDO + q);
            }
        } else {
            for (int i = threadIdx.x; i < ch.rows * kOutCols; i += kOutThreads) {
                const int r = i / kOutCols, q = i % kOutCols;
                if (q < width) to[r * step + q] = sh.o[r * LDO + q];
            }
        }
        if (pass + kOutCols < (int)p.dvp) __syncthreads();
    }
}

// ---------------------------------------------------------------------------
// Launches
// ---------------------------------------------------------------------------

template <typename T, int DKP>
void prepare_as(const Args& a, cudaStream_t stream, bool backward) {
    const size_t bytes = sizeof(PrepShared<T, DKP>);
    opt_in<delta_prep_kernel<T, DKP>>(bytes);
    launch_dependent(delta_prep_kernel<T, DKP>, dim3(a.chunks, a.value_heads), kPrepThreads, bytes, stream, a, backward);
}

template <typename T, int DKP, int KS>
void states_as(const Args& a, cudaStream_t stream) {
    using Sh = StateShared<T, DKP, KS>;
    opt_in<delta_state_kernel<T, DKP, KS>>(sizeof(Sh));
    const dim3 grid((a.dvp / 16 + Sh::kGroups - 1) / Sh::kGroups, a.value_heads, a.seqs);
    launch_dependent(delta_state_kernel<T, DKP, KS>, grid, kStateThreads, sizeof(Sh), stream, a);
}

template <typename T, int DKP>
void states_of(const Args& a, cudaStream_t stream, int sm_count) {
    // Four warps to a chain while their blocks are all resident (two a multiprocessor, one in float32), two beyond. 64 chunks of 128 x 128 in bfloat16: 128
    // chains 108 (four) 186 us (two); 256 chains 174, 188; 512 chains 344, 304. 32 chunks in float32: 128 chains 83, 138;
    // 256 chains 163, 144; 512 chains 323, 271. (One warp a chain: 367 us in bfloat16 whatever their number up to 512.)
    const uint64_t chains = (uint64_t)(a.dvp / 16) * a.value_heads * a.seqs;
    if (chains <= (sizeof(T) == 2 ? 2 : 1) * (uint64_t)sm_count) states_as<T, DKP, 4>(a, stream);
    else states_as<T, DKP, 2>(a, stream);
}

template <typename T, int DKP>
void output_as(const Args& a, cudaStream_t stream) {
    const size_t bytes = sizeof(OutShared<T, DKP>);
    opt_in<delta_output_kernel<T, DKP>>(bytes);
    // one block more than there can be chunks: a ragged batch's tokens of no sequence have a block to clear them
    launch_dependent(delta_output_kernel<T, DKP>, dim3(a.chunks + (a.sequences ? 1 : 0), a.value_heads), kOutThreads, bytes, stream, a);
}

} // namespace

void launch_prepare(const Args& a, cudaStream_t stream, bool backward) {
    if (a.sequences) launch_dependent(delta_index_kernel, 1, kIndexThreads, 0, stream, a);
    if (a.chunks) DELTA_DISPATCH(prepare_as, a, stream, backward);
}

void launch_states(const Args& a, cudaStream_t stream, int sm_count) { DELTA_DISPATCH(states_of, a, stream, sm_count); }

void launch_forward(const Args& a, cudaStream_t stream, int sm_count) {
    launch_prepare(a, stream, false);
    launch_states(a, stream, sm_count);
    if (a.chunks) DELTA_DISPATCH(output_as, a, stream);
}

} // namespace delta
} // namespace mlb
