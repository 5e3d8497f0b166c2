// The product of two matrices in 8-bit floating point with float32 scales for blocks of 128 along k:
//
//     C[i][j] = sum over blocks kb of  sa[i][kb] sb[j][kb]  sum over k in kb of  a[i][k] b[j][k]
//
// A block of k is 128 bytes of a row: one swizzled row of a TMA tile and four tcgen05.mma (kind::f8f6f4, k of 32). Its
// product goes to tensor memory on its own (the scales change from block to block), is read back by the epilogue warps and
// added, times the scales, to float32 sums in registers, while the tensor core fills the next accumulator: so the sums of
// many blocks never pass through the tensor core's adder.
//
// A thread block: eight (or four) epilogue warps, a warp whose first lane issues the TMA loads of the stages' ring, a warp
// whose first lane issues the products. Tiles are 128 rows (lanes of tensor memory) x BN columns. The operand with more rows
// lies along the lanes where the other has at most 64 (decoding: 128 rows of the weight against 16 to 64 tokens); C is then
// written along its contiguous dimension by neighbouring lanes. Where there are fewer tiles than multiprocessors, up to
// eight blocks of a cluster share a tile's k and add their sums through distributed shared memory, each a part of the columns, always in
// the same order: no atomics, no workspace.
//
// What bounds a large product is the hand-over of accumulators: a block of 128 x 256 x 128 takes the tensor core 512 clocks, and
// the eight epilogue warps 1250 to 1400 to wait for it, read it, scale it, add it and hand it back, two accumulators
// taking turns: 8192 x 8192 x 4096 in 304 us, 1.81 PFLOP/s (347 us when it runs for seconds and the clocks fall). With a scale
// for every row of both operands a second multiplication and a load of scales for four sums make that 2200 clocks: 522 us
// (tiles of 128 columns 10 % more). 4096 x 4096 x 2048 55 us; 1024 x 1024 x 4096 14; 16 rows x 4096 x 8192 11.4 us (the
// weight's 33.6 MB at 3.0 TB/s: the ring's start and the cluster's exchange are half of it).
//
// Every wait on an mbarrier is bounded. One that runs out makes the block's outputs NaN, sets the status word, waits
// (bounded) for the block's own loads and products and ends.
#include "common.cuh"
#include "fp8.h"
#include "runtime.h"

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

namespace mlb {
namespace fp8 {

namespace {

constexpr int kRowsTile = 128;
constexpr int kBlockK = 128;
constexpr uint32_t kWaitLimit = 1u << 21;
constexpr int kMaxSplit = 8;

struct GemmArgs {
    const float *sp, *sq;              // scales of the rows' and the columns' operand
    uint64_t sp_batch, sq_batch;       // floats between matrices (0: one for all)
    uint32_t p, q, kb;                 // rows, columns, blocks of k
    uint32_t p_shift, q_shift;         // log2 of the scale blocks' rows: 0 or 7
    uint32_t p_tiles, q_tiles, tiles;  // tiles = p_tiles * q_tiles * batch
    uint32_t batched_p, batched_q;     // 0: the operand is one matrix for the whole batch
    uint32_t split, split_log;         // blocks that share a tile, a power of two
    uint32_t idesc;
    void*    c;
    uint64_t c_batch;
    uint64_t ldp, ldq;                 // C's strides along rows and columns of the tile: one of them is 1
    uint32_t c_dtype;
    uint32_t wide;                     // C's rows (ldq == 1) can be written in 16-byte pieces
    unsigned* status;
    uint32_t give_up;                  // as if every wait had run out at once: no load or product is issued (inject_wait_failures)

    // Tile t's matrix, first row and first column: tiles of a column of C behind one another.
    template <int BN> __device__ __forceinline__ void place(uint32_t t, uint32_t& z, uint32_t& p0, uint32_t& q0) const {
        z = t / (p_tiles * q_tiles);
        t -= z * p_tiles * q_tiles;
        q0 = t / p_tiles;
        p0 = (t - q0 * p_tiles) * kRowsTile;
        q0 *= BN;
    }
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

// K-major tile of 128-byte rows, 128-byte swizzle: eight rows (1024 bytes) apart.
__device__ __forceinline__ uint64_t tile_desc(uint32_t addr) {
    const uint32_t lo = ((addr >> 4) & 0x3FFFu) | (1u << 16);
    const uint32_t hi = (1024u >> 4) | (1u << 14) | (2u << 29);     // version 1, SWIZZLE_128B
    return ((uint64_t)hi << 32) | lo;
}

__device__ __forceinline__ bool try_wait(uint32_t bar, uint32_t parity) {
    uint32_t done;
    asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
                 : "=r"(done) : "r"(bar), "r"(parity) : "memory");
    return done != 0;
}
// The one lane of a converged warp that issues its copies or products. The compiler knows that elect.sync leaves one lane, and
// so gives tcgen05 and TMA instructions their uniform operands directly; behind `lane == 0` it asks lane by lane (four
// products and two commits: 365 clocks, 100 this way).
__device__ __forceinline__ bool elect_one() {
    uint32_t one;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(one) :: "memory");
    return one != 0;
}
// False if the wait ran out, here or (sooner) anywhere else in the block.
__device__ __forceinline__ bool wait_on(uint32_t bar, uint32_t parity, volatile int* failed) {
    for (uint32_t i = 0; i < kWaitLimit; ++i) {
        if (try_wait(bar, parity)) return true;
        if ((i & 15) == 15 && *failed) return false;
    }
    *failed = 1;
    return false;
}
__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity, volatile int* failed) {
    return try_wait(bar, parity) || wait_on(bar, parity, failed);
}

template <int N> struct TmemLoad;
template <> struct TmemLoad<16> {
    static __device__ __forceinline__ void load(uint32_t (&v)[16], uint32_t at) {
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                     : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
                       "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
                     : "r"(at) : "memory");
    }
};
template <> struct TmemLoad<32> {
    static __device__ __forceinline__ void load(uint32_t (&v)[32], uint32_t at) {
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
                     "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                     : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
                       "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]),
                       "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]),
                       "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
                     : "r"(at) : "memory");
    }
};

__device__ __forceinline__ void store_one(void* c, uint64_t at, uint32_t dtype, float v) {
    if (dtype == METAL_LINALG_BFLOAT16) static_cast<__nv_bfloat16*>(c)[at] = __float2bfloat16_rn(v);
    else if (dtype == METAL_LINALG_FLOAT16) static_cast<__half*>(c)[at] = __float2half_rn(v);
    else static_cast<float*>(c)[at] = v;
}
__device__ __forceinline__ uint32_t pack_two(uint32_t dtype, float2 v) {
    if (dtype == METAL_LINALG_BFLOAT16) {
        const __nv_bfloat162 r = __floats2bfloat162_rn(v.x, v.y);
        return *reinterpret_cast<const uint32_t*>(&r);
    }
    const __half2 r = __floats2half2_rn(v.x, v.y);
    return *reinterpret_cast<const uint32_t*>(&r);
}

// Two neighbouring sums in one 64-bit register: sum += (x, y) * by.
using Pair = unsigned long long;
__device__ __forceinline__ Pair pair_of(float x, float y) {
    Pair r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ float2 both_of(Pair p) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(p));
    return r;
}
__device__ __forceinline__ void add_scaled(Pair& sum, uint32_t x, uint32_t y, Pair by) {
    asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(sum) : "l"(pair_of(__uint_as_float(x), __uint_as_float(y))), "l"(by));
}
__device__ __forceinline__ Pair times(Pair a, Pair b) {
    Pair r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

template <int N> constexpr uint32_t kLog = 1 + kLog<N / 2>;
template <> constexpr uint32_t kLog<1> = 0;

template <int BN>
struct Shape {
    static constexpr int kEpilogueWarps = BN >= 128 ? 8 : 4;
    // 256 columns: 128 sums and two loads of 32 a thread are more registers than twelve warps' even share (168), so the four
    // warps behind the epilogue's (two of them idle: registers change hands by fours) give theirs up: 256 x 224 + 128 x 56
    // of the launch's 384 x 168
    static constexpr bool kUneven = BN == 256;
    static constexpr int kThreads = 32 * (kEpilogueWarps + (kUneven ? 4 : 2));
    static constexpr int kCols = BN / (kEpilogueWarps / 4);        // columns an epilogue thread sums
    static constexpr int kAcc = BN == 256 ? 2 : 4;                 // accumulators in tensor memory
    static constexpr int kTmem = kAcc * BN < 32 ? 32 : kAcc * BN;
    static constexpr int kStageBytes = (kRowsTile + BN) * kBlockK;
    static constexpr int kStages = BN == 256 ? 4 : BN == 128 ? 4 : BN == 64 ? 7 : 8;
    static constexpr int kReduceBytes = BN <= 128 ? BN * kRowsTile * 4 : 0;     // partial sums from the cluster's other blocks
    static constexpr int kScaleBytes = kEpilogueWarps / 4 * 2 * kCols * 4;
    static constexpr size_t kShared = (size_t)kStages * kStageBytes + kReduceBytes + kScaleBytes + 1024;
    static_assert(kShared + 512 <= 232448, "with the barriers, more than a block's shared memory");
};

// kByColumn: the columns' operand has a scale a row (else one for 128 rows, the same for all of a thread's columns).
template <int BN, bool kByColumn>
__global__ void __launch_bounds__(Shape<BN>::kThreads, 1)
fp8_gemm_kernel(const __grid_constant__ CUtensorMap map_p, const __grid_constant__ CUtensorMap map_q, const GemmArgs a) {
    using S = Shape<BN>;
    extern __shared__ char raw[];
    char* base = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
    float* reduce = reinterpret_cast<float*>(base + S::kStages * S::kStageBytes);
    float* scales = reinterpret_cast<float*>(base + S::kStages * S::kStageBytes + S::kReduceBytes);
    __shared__ __align__(8) unsigned long long full[S::kStages], empty[S::kStages], acc_full[S::kAcc], acc_empty[S::kAcc], drain;
    __shared__ uint32_t tmem_slot;
    __shared__ int failed_word;
    volatile int* failed = &failed_word;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = a.split > 1 ? blockIdx.x % a.split : 0;
    const uint32_t first = blockIdx.x / a.split, step = gridDim.x / a.split;
    // this block's blocks of k
    const uint32_t kb0 = (uint32_t)((uint64_t)a.kb * rank / a.split), kb1 = (uint32_t)((uint64_t)a.kb * (rank + 1) / a.split);

    if (threadIdx.x == 0) {
        failed_word = (int)a.give_up;
        for (int i = 0; i < S::kStages; ++i) {
            asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" :: "r"(smem_u32(&full[i])));
            asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" :: "r"(smem_u32(&empty[i])));
        }
        for (int i = 0; i < S::kAcc; ++i) {
            asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" :: "r"(smem_u32(&acc_full[i])));
            asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" :: "r"(smem_u32(&acc_empty[i])), "n"(S::kEpilogueWarps));
        }
        asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" :: "r"(smem_u32(&drain)));
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == S::kEpilogueWarps) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(smem_u32(&tmem_slot)), "n"(S::kTmem) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = tmem_slot;
    dependency_wait_only();         // nothing above reads or writes memory that another kernel may hold
    if (a.split > 1) {          // the other blocks are there before anything is sent to them (arrival now, the wait before the first use)
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    }

    if (warp < S::kEpilogueWarps) {             // sums
        if constexpr (S::kUneven) asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
        const int quarter = warp & 3, part = warp >> 2;
        const uint32_t row = 32 * quarter + lane;
        float* part_scales = scales + part * 2 * S::kCols;      // of this part's columns, two blocks of k
        uint32_t i = 0;
        bool ok = !a.give_up;
        for (uint32_t tile = first; tile < a.tiles; tile += step) {
            const float *sp, *sq;               // this block's first scales of the thread's row, of its columns
            bool q_there = false;               // by column: the four warps of a part fetch a quarter of its columns each
            {
                uint32_t z, p, q0;
                a.place<BN>(tile, z, p, q0);
                p = min(p + row, a.p - 1);
                q0 += part * S::kCols;
                sp = a.sp + (a.batched_p ? z * a.sp_batch : 0) + (uint64_t)(p >> a.p_shift) * a.kb + kb0;
                sq = a.sq + (a.batched_q ? z * a.sq_batch : 0) + kb0;
                if constexpr (kByColumn) {
                    const uint32_t column = q0 + quarter * (S::kCols / 4) + lane;
                    sq += (uint64_t)column * a.kb;
                    q_there = lane < S::kCols / 4 && column < a.q;
                } else {
                    sq += (uint64_t)(min(q0, a.q - 1) >> 7) * a.kb;
                }
            }
            Pair sum[S::kCols / 2];
#pragma unroll
            for (int j = 0; j < S::kCols / 2; ++j) sum[j] = 0;
            // the next block's scales are fetched while this one's product is awaited (by plain loads: the kernel before this one may
            // still write them when this one starts, so they are not constant for its whole run)
            float row_scale = 0.0f, col_scale = 0.0f;
            const auto fetch = [&]() {
                row_scale = *sp++;
                if (!kByColumn || q_there) col_scale = *sq;
                ++sq;
            };
            if (kb0 < kb1) fetch();
#pragma unroll 1
            for (uint32_t kb = kb0; kb < kb1; ++kb, ++i) {
                const uint32_t acc = i % S::kAcc;
                float scale = row_scale;
                float* by_column = part_scales + (i & 1) * S::kCols;
                if constexpr (kByColumn) {
                    if (lane < S::kCols / 4) by_column[quarter * (S::kCols / 4) + lane] = col_scale;
                    // every one of the four warps comes here for every block of k, a failed wait behind it or not
                    asm volatile("bar.sync %0, 128;" :: "r"(1 + part) : "memory");
                } else {
                    scale *= col_scale;
                }
                const Pair scale2 = pair_of(scale, scale);
                if (kb + 1 < kb1) fetch();
                ok = ok && wait(smem_u32(&acc_full[acc]), (i / S::kAcc) & 1, failed);
                ok = __all_sync(0xffffffffu, ok);       // (one lane asking for its warp was 8 % slower)
                if (!ok) continue;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint32_t at = tmem + acc * BN + part * S::kCols + ((32u * quarter) << 16);
                // two loads in flight; the next two go out as their registers are used up
                // (by column in pieces of 16: the scales of two of them take the registers)
                constexpr int kPiece = S::kCols >= 32 && !kByColumn ? 32 : 16, kFlight = S::kCols > kPiece ? 2 : 1;
                uint32_t v[kFlight][kPiece];
#pragma unroll
                for (int f = 0; f < kFlight; ++f) TmemLoad<kPiece>::load(v[f], at + f * kPiece);
#pragma unroll
                for (int j = 0; j < S::kCols; j += kFlight * kPiece) {
                    ulonglong2 c[kByColumn ? kFlight * kPiece / 4 : 1];     // on their way while the accumulator is
                    if constexpr (kByColumn)
#pragma unroll
                        for (int e = 0; e < kFlight * kPiece / 4; ++e) c[e] = *reinterpret_cast<const ulonglong2*>(by_column + j + 4 * e);
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                    if (j + kFlight * kPiece >= S::kCols) {     // everything is read: the accumulator is free
                        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                        if (lane == 0)
                            asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" :: "r"(smem_u32(&acc_empty[acc])) : "memory");
                    }
#pragma unroll
                    for (int f = 0; f < kFlight; ++f) {
#pragma unroll
                        for (int e = 0; e < kPiece; e += 4) {
                            const int to = j + f * kPiece + e;
                            Pair by[2] = {scale2, scale2};
                            if constexpr (kByColumn) {
                                by[0] = times(scale2, c[(f * kPiece + e) / 4].x);
                                by[1] = times(scale2, c[(f * kPiece + e) / 4].y);
                            }
                            add_scaled(sum[to / 2], v[f][e], v[f][e + 1], by[0]);
                            add_scaled(sum[to / 2 + 1], v[f][e + 2], v[f][e + 3], by[1]);
                        }
                        if (j + (kFlight + f) * kPiece < S::kCols) TmemLoad<kPiece>::load(v[f], at + j + (kFlight + f) * kPiece);
                    }
                }
            }
            if (!ok)
#pragma unroll
                for (int j = 0; j < S::kCols / 2; ++j) sum[j] = pair_of(qnan(), qnan());

            if constexpr (S::kReduceBytes > 0) {
                if (a.split > 1) {
                    // block r of the cluster adds columns r * BN / split ..: part `rank` of everyone's, in the ranks' order
                    const uint32_t log = kLog<BN> - a.split_log;        // of a share's columns
                    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");       // everyone has started
                    // [rank][row][column], four columns at a time; rows' quads are permuted so that neighbouring lanes
                    // meet different banks
#pragma unroll
                    for (int j = 0; j < S::kCols; j += 4) {
                        const float2 f = both_of(sum[j / 2]), g = both_of(sum[j / 2 + 1]);
                        const uint32_t q = part * S::kCols + j, to = q >> log, quad = (q & ((1u << log) - 1)) >> 2;
                        const uint32_t local = smem_u32(reduce) + (((rank * kRowsTile + row) << log) << 2) +
                                               ((quad ^ (row & ((1u << log) / 4 - 1) & 7)) << 4);
                        uint32_t remote;
                        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local), "r"(to));
                        asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" :: "r"(remote), "f"(f.x), "f"(f.y), "f"(g.x), "f"(g.y) : "memory");
                    }
                }
            }
            uint32_t again = tile, z, p, q0;            // worked out anew: the sums leave no registers to keep it in
            asm volatile("" : "+r"(again));
            a.place<BN>(again, z, p, q0);
            p += row;
            q0 += part * S::kCols;
            if (a.split == 1 && p < a.p) {
                uint64_t ldq = a.ldq;           // (nor to keep its multiples in)
                asm volatile("" : "+l"(ldq));
                uint64_t at = z * a.c_batch + (uint64_t)p * a.ldp + (uint64_t)q0 * ldq;
                if (a.wide && q0 + S::kCols <= a.q) {
                    if (a.c_dtype == METAL_LINALG_FLOAT32) {
#pragma unroll
                        for (int j = 0; j < S::kCols; j += 4) {
                            const float2 x = both_of(sum[j / 2]), y = both_of(sum[j / 2 + 1]);
                            *reinterpret_cast<float4*>(static_cast<float*>(a.c) + at + j) = make_float4(x.x, x.y, y.x, y.y);
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < S::kCols; j += 8)
                            *reinterpret_cast<uint4*>(static_cast<__half*>(a.c) + at + j) =
                                make_uint4(pack_two(a.c_dtype, both_of(sum[j / 2])), pack_two(a.c_dtype, both_of(sum[j / 2 + 1])),
                                           pack_two(a.c_dtype, both_of(sum[j / 2 + 2])), pack_two(a.c_dtype, both_of(sum[j / 2 + 3])));
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < S::kCols; ++j, at += ldq)
                        if (q0 + j < a.q) store_one(a.c, at, a.c_dtype, j & 1 ? both_of(sum[j / 2]).y : both_of(sum[j / 2]).x);
                }
            }
        }
    } else {
    if constexpr (S::kUneven) asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp == S::kEpilogueWarps) {            // loads
        if (elect_one()) {
            uint32_t i = 0;                     // blocks of k so far
            bool ok = !a.give_up;
            const uint32_t full0 = smem_u32(&full[0]), empty0 = smem_u32(&empty[0]), ring = smem_u32(base);
            uint32_t tile = first, kb = kb0, z, p0, q0;
            if (tile < a.tiles) a.place<BN>(tile, z, p0, q0);
            for (uint32_t round = 0; ok && tile < a.tiles; ++round) {
#pragma unroll 1
                for (int s = 0; s < S::kStages; ++s) {
                    if (tile >= a.tiles) break;
                    if (round && !wait(empty0 + 8 * s, (round - 1) & 1, failed)) { ok = false; break; }
                    const uint32_t bar = full0 + 8 * s, dst = ring + s * S::kStageBytes;
                    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" :: "r"(bar), "n"(S::kStageBytes) : "memory");
                    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                                 :: "r"(dst), "l"(&map_p), "r"((int)(kb * kBlockK)), "r"(p0), "r"(a.batched_p ? z : 0), "r"(bar) : "memory");
                    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                                 :: "r"(dst + kRowsTile * kBlockK), "l"(&map_q), "r"((int)(kb * kBlockK)), "r"(q0), "r"(a.batched_q ? z : 0), "r"(bar) : "memory");
                    ++i;
                    if (++kb == kb1) {
                        kb = kb0;
                        tile += step;
                        if (tile < a.tiles) a.place<BN>(tile, z, p0, q0);
                    }
                }
            }
            if (!ok) {                          // nothing of this block's is on its way when it ends
                for (uint32_t j = i > (uint32_t)S::kStages ? i - S::kStages : 0; j < i; ++j)
                    for (uint32_t n = 0; n < kWaitLimit && !try_wait(smem_u32(&full[j % S::kStages]), (j / S::kStages) & 1); ++n) {}
            }
        }
        __syncwarp();
    } else if (warp == S::kEpilogueWarps + 1) { // products
        if (elect_one()) {
            bool ok = !a.give_up;
            const uint32_t full0 = smem_u32(&full[0]), empty0 = smem_u32(&empty[0]), acc_full0 = smem_u32(&acc_full[0]),
                           acc_empty0 = smem_u32(&acc_empty[0]);
            const uint64_t ring = tile_desc(smem_u32(base));
            uint32_t left = first < a.tiles ? ((a.tiles - 1 - first) / step + 1) * (kb1 - kb0) : 0;     // blocks of k to come
            uint32_t acc = 0, acc_round = 0;
            for (uint32_t round = 0; ok && left; ++round) {
#pragma unroll 1
                for (int s = 0; s < S::kStages; ++s) {
                    if (!left) break;
                    --left;
                    // the operands first: they are there early, and the accumulator is what a product waits for
                    if (!wait(full0 + 8 * s, round & 1, failed)) { ok = false; break; }
                    if (acc_round && !wait(acc_empty0 + 8 * acc, (acc_round - 1) & 1, failed)) { ok = false; break; }
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint64_t dp = ring + (s * S::kStageBytes >> 4), dq = dp + (kRowsTile * kBlockK >> 4);
#pragma unroll
                    for (int j = 0; j < kBlockK / 32; ++j)
                        asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
                                     " tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n}"
                                     :: "r"(tmem + acc * BN), "l"(dp + 2 * j), "l"(dq + 2 * j), "r"(a.idesc), "r"(j) : "memory");
                    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" :: "r"(empty0 + 8 * s) : "memory");
                    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" :: "r"(acc_full0 + 8 * acc) : "memory");
                    if (++acc == S::kAcc) {
                        acc = 0;
                        ++acc_round;
                    }
                }
            }
            if (!ok) {
                asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" :: "r"(smem_u32(&drain)) : "memory");
                for (uint32_t n = 0; n < kWaitLimit && !try_wait(smem_u32(&drain), 0); ++n) {}
            }
        }
        __syncwarp();
    }
    }
    if (a.split > 1) {
        // loads' and products' warps took no part in the first wait yet
        if (warp >= S::kEpilogueWarps) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");                   // every partial sum has come
        if constexpr (S::kReduceBytes > 0) {
            const uint32_t log = kLog<BN> - a.split_log, mine = 1u << log;
            uint32_t z, p0, q0;
            a.place<BN>(first, z, p0, q0);
            q0 += rank << log;
            for (uint32_t e = threadIdx.x; e < mine / 4 * kRowsTile; e += S::kThreads) {
                // along whichever dimension C is contiguous
                const uint32_t r = a.ldp == 1 ? e % kRowsTile : e >> (log - 2), quad = a.ldp == 1 ? e / kRowsTile : e & (mine / 4 - 1);
                if (p0 + r >= a.p || q0 + 4 * quad >= a.q) continue;
                float sum[4] = {};
#pragma unroll
                for (uint32_t w = 0; w < kMaxSplit; ++w)
                    if (w < a.split) {
                        const float4 f = *reinterpret_cast<const float4*>(
                            reduce + ((w * kRowsTile + r) << log) + ((quad ^ (r & (mine / 4 - 1) & 7)) << 2));
                        sum[0] += f.x; sum[1] += f.y; sum[2] += f.z; sum[3] += f.w;
                    }
                const uint64_t at = z * a.c_batch + (uint64_t)(p0 + r) * a.ldp + (uint64_t)(q0 + 4 * quad) * a.ldq;
                if (a.wide && q0 + 4 * quad + 4 <= a.q) {
                    if (a.c_dtype == METAL_LINALG_FLOAT32)
                        *reinterpret_cast<float4*>(static_cast<float*>(a.c) + at) = make_float4(sum[0], sum[1], sum[2], sum[3]);
                    else
                        *reinterpret_cast<uint2*>(static_cast<__half*>(a.c) + at) =
                            make_uint2(pack_two(a.c_dtype, make_float2(sum[0], sum[1])), pack_two(a.c_dtype, make_float2(sum[2], sum[3])));
                } else {
#pragma unroll
                    for (uint32_t j = 0; j < 4; ++j)
                        if (q0 + 4 * quad + j < a.q) store_one(a.c, at + j * a.ldq, a.c_dtype, sum[j]);
                }
            }
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0 && *failed) atomicOr(a.status, (unsigned)kStatusProductWait);
    if (warp == S::kEpilogueWarps) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(tmem), "n"(S::kTmem) : "memory");
}

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                 const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encoder() {
    static const EncodeTiled fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult found{};
        cuda_check(cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found), "cuTensorMapEncodeTiled");
        if (!p) throw std::runtime_error("the driver has no cuTensorMapEncodeTiled");
        return reinterpret_cast<EncodeTiled>(p);
    }();
    return fn;
}

// Tiles of `rows` rows x 128 bytes of [batch][rows][k]; what lies outside reads as zero.
CUtensorMap tile_map(const GemmOperand& o, uint32_t batch, uint32_t k, uint32_t rows) {
    CUtensorMap map;
    const bool batched = o.batch_stride != 0 && batch > 1;
    const cuuint64_t dims[3] = {k, o.rows, batched ? batch : 1};
    const cuuint64_t strides[2] = {o.stride, batched ? o.batch_stride : o.stride * o.rows};
    const cuuint32_t box[3] = {kBlockK, rows, 1}, unit[3] = {1, 1, 1};
    const CUresult r = encoder()(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(o.values), dims, strides, box, unit,
                                 CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                 CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) throw std::runtime_error("cuTensorMapEncodeTiled failed with " + std::to_string((int)r));
    return map;
}

template <int BN, bool kByColumn>
void gemm_as(cudaStream_t stream, const CUtensorMap& mp, const CUtensorMap& mq, const GemmArgs& a, int sm_count) {
    using S = Shape<BN>;
    static PerDeviceOnce once;          // the opt-in is recorded per GPU
    if (const int device = current_device(); once.first(device)) {
        cuda_check(cudaFuncSetAttribute(fp8_gemm_kernel<BN, kByColumn>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::kShared),
                   "fp8 product shared memory");
        once.mark(device);
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(a.split > 1 ? a.tiles * a.split : std::min<uint32_t>(a.tiles, (uint32_t)sm_count));
    cfg.blockDim = dim3(S::kThreads);
    cfg.dynamicSmemBytes = S::kShared;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    unsigned count = 0;
    if (a.split > 1) {
        attr[count].id = cudaLaunchAttributeClusterDimension;
        attr[count].val.clusterDim.x = a.split;
        attr[count].val.clusterDim.y = attr[count].val.clusterDim.z = 1;
        ++count;
    }
    if (dependent_launches_enabled()) {         // as launch_dependent: the kernel's set-up beside the end of the one before it
        attr[count].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[count].val.programmaticStreamSerializationAllowed = 1;
        ++count;
    }
    cfg.attrs = attr;
    cfg.numAttrs = count;
    cuda_check(cudaLaunchKernelEx(&cfg, fp8_gemm_kernel<BN, kByColumn>, mp, mq, a), "fp8 product launch");
}

} // namespace

void launch_gemm(cudaStream_t stream, int device, const GemmOperand& oa, const GemmOperand& ob, uint32_t batch, uint32_t k, void* c,
                 uint32_t c_dtype, unsigned* status) {
    const uint32_t m = oa.rows, n = ob.rows;
    const int sms = sm_count(device);
    // the longer operand along the lanes where the other has at most 64 rows; else C's rows, so that a thread writes along them
    const bool turned = m <= 64 && n > m;
    const GemmOperand &p = turned ? ob : oa, &q = turned ? oa : ob;
    GemmArgs a{};
    a.p = p.rows; a.q = q.rows; a.kb = (k + kBlockK - 1) / kBlockK;
    a.p_tiles = (a.p + kRowsTile - 1) / kRowsTile;
    // 256 columns a tile where that still gives every multiprocessor one
    const uint32_t bn = a.q <= 16 ? 16 : a.q <= 32 ? 32 : a.q <= 64 ? 64
                      : (uint64_t)a.p_tiles * ((a.q + 255) / 256) * batch >= (uint64_t)sms ? 256 : 128;
    a.q_tiles = (a.q + bn - 1) / bn;
    const uint64_t tiles = (uint64_t)a.p_tiles * a.q_tiles * batch;
    if (tiles >= 1ull << 28) throw std::invalid_argument("[matmul_fp8] the product is too large");
    a.tiles = (uint32_t)tiles;
    a.split = 1;
    a.split_log = 0;                // shares of k: powers of two, four columns a share, none without a block of k, no more blocks than multiprocessors
    if (bn <= 128)
        while (a.split < kMaxSplit && a.split * 8 <= bn && a.tiles * a.split * 2 <= (uint32_t)sms && a.split * 2 <= a.kb) {
            a.split *= 2;
            ++a.split_log;
        }
    a.sp = p.scales; a.sq = q.scales;
    a.p_shift = p.block_rows == 128 ? 7 : 0;
    a.q_shift = q.block_rows == 128 ? 7 : 0;
    a.batched_p = p.batch_stride != 0; a.batched_q = q.batch_stride != 0;
    a.sp_batch = (uint64_t)((p.rows + p.block_rows - 1) / p.block_rows) * a.kb;
    a.sq_batch = (uint64_t)((q.rows + q.block_rows - 1) / q.block_rows) * a.kb;
    // kind::f8f6f4, float32 accumulator, both operands K-major
    a.idesc = (1u << 4) | ((p.e5m2 ? 1u : 0u) << 7) | ((q.e5m2 ? 1u : 0u) << 10) | ((bn >> 3) << 17) | ((128u >> 4) << 24);
    a.c = c;
    a.c_batch = (uint64_t)m * n;
    a.ldp = turned ? 1 : n;
    a.ldq = turned ? n : 1;
    a.c_dtype = c_dtype;
    const uint32_t size = c_dtype == METAL_LINALG_FLOAT32 ? 4 : 2;
    a.wide = !turned && (uint64_t)n * size % 16 == 0 && (reinterpret_cast<uintptr_t>(c) & 15) == 0;
    a.status = status;
    a.give_up = take_injected_wait_failure();
    const CUtensorMap mp = tile_map(p, batch, k, kRowsTile), mq = tile_map(q, batch, k, bn);
    const bool by_column = a.q_shift == 0;
    switch (bn) {
        case 16: by_column ? gemm_as<16, true>(stream, mp, mq, a, sms) : gemm_as<16, false>(stream, mp, mq, a, sms); break;
        case 32: by_column ? gemm_as<32, true>(stream, mp, mq, a, sms) : gemm_as<32, false>(stream, mp, mq, a, sms); break;
        case 64: by_column ? gemm_as<64, true>(stream, mp, mq, a, sms) : gemm_as<64, false>(stream, mp, mq, a, sms); break;
        case 128: by_column ? gemm_as<128, true>(stream, mp, mq, a, sms) : gemm_as<128, false>(stream, mp, mq, a, sms); break;
        default: by_column ? gemm_as<256, true>(stream, mp, mq, a, sms) : gemm_as<256, false>(stream, mp, mq, a, sms); break;
    }
}

} // namespace fp8
} // namespace mlb
