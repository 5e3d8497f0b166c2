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
    uint32_t split;                    // blocks that share a tile
    uint32_t idesc;
    void*    c;
    uint64_t c_batch;
    uint64_t ldp, ldq;                 // C's strides along rows and columns of the tile: one of them is 1
    uint32_t c_dtype;
    uint32_t wide;                     // C's rows (ldq == 1) can be written in 16-byte pieces
    unsigned* status;
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
// False if the wait ran out, here or (sooner) anywhere else in the block.
__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity, volatile int* failed) {
    for (uint32_t i = 0; i < kWaitLimit; ++i) {
        if (try_wait(bar, parity)) return true;
        if ((i & 15) == 15 && *failed) return false;
    }
    *failed = 1;
    return false;
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
__device__ __forceinline__ uint32_t pack_two(uint32_t dtype, float a, float b) {
    if (dtype == METAL_LINALG_BFLOAT16) {
        const __nv_bfloat162 r = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&r);
    }
    const __half2 r = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&r);
}

template <int BN>
struct Shape {
    static constexpr int kEpilogueWarps = BN >= 128 ? 8 : 4;
    static constexpr int kThreads = 32 * (kEpilogueWarps + 2);
    static constexpr int kCols = BN / (kEpilogueWarps / 4);        // columns an epilogue thread sums
    static constexpr int kAcc = BN == 256 ? 2 : 4;                 // accumulators in tensor memory
    static constexpr int kTmem = kAcc * BN < 32 ? 32 : kAcc * BN;
    static constexpr int kStageBytes = (kRowsTile + BN) * kBlockK;
    static constexpr int kStages = BN == 256 ? 4 : BN == 128 ? 4 : BN == 64 ? 7 : 8;
    static constexpr int kReduceBytes = BN <= 128 ? BN * kRowsTile * 4 : 0;     // partial sums from the cluster's other blocks
    static constexpr int kScaleBytes = kEpilogueWarps * 2 * kCols * 4;
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
        failed_word = 0;
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
    if (a.split > 1) {          // the other blocks are there before anything is sent to them (arrival now, the wait before the first use)
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    }

    if (warp == S::kEpilogueWarps) {            // loads
        if (lane == 0) {
            uint32_t i = 0;                     // blocks of k so far
            bool ok = true;
            for (uint32_t tile = first; ok && tile < a.tiles; tile += step) {
                const uint32_t z = tile / (a.p_tiles * a.q_tiles), t = tile - z * a.p_tiles * a.q_tiles;
                const int p0 = (int)(t % a.p_tiles) * kRowsTile, q0 = (int)(t / a.p_tiles) * BN;
                const int zp = a.batched_p ? (int)z : 0, zq = a.batched_q ? (int)z : 0;
                for (uint32_t kb = kb0; kb < kb1; ++kb, ++i) {
                    const uint32_t s = i % S::kStages, round = i / S::kStages;
                    if (round && !wait(smem_u32(&empty[s]), (round - 1) & 1, failed)) { ok = false; break; }
                    const uint32_t bar = smem_u32(&full[s]), dst = smem_u32(base + s * S::kStageBytes);
                    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" :: "r"(bar), "n"(S::kStageBytes) : "memory");
                    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                                 :: "r"(dst), "l"(&map_p), "r"((int)(kb * kBlockK)), "r"(p0), "r"(zp), "r"(bar) : "memory");
                    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                                 :: "r"(dst + kRowsTile * kBlockK), "l"(&map_q), "r"((int)(kb * kBlockK)), "r"(q0), "r"(zq), "r"(bar) : "memory");
                }
            }
            if (!ok) {                          // nothing of this block's is on its way when it ends
                for (uint32_t j = i > (uint32_t)S::kStages ? i - S::kStages : 0; j < i; ++j)
                    for (uint32_t n = 0; n < kWaitLimit && !try_wait(smem_u32(&full[j % S::kStages]), (j / S::kStages) & 1); ++n) {}
            }
        }
        __syncwarp();
    } else if (warp == S::kEpilogueWarps + 1) { // products
        if (lane == 0) {
            uint32_t i = 0;
            bool ok = true;
            for (uint32_t tile = first; ok && tile < a.tiles; tile += step)
                for (uint32_t kb = kb0; kb < kb1; ++kb, ++i) {
                    const uint32_t s = i % S::kStages, acc = i % S::kAcc;
                    if (i >= (uint32_t)S::kAcc && !wait(smem_u32(&acc_empty[acc]), (i / S::kAcc - 1) & 1, failed)) { ok = false; break; }
                    if (!wait(smem_u32(&full[s]), (i / S::kStages) & 1, failed)) { ok = false; break; }
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint32_t at = smem_u32(base + s * S::kStageBytes);
                    const uint64_t dp = tile_desc(at), dq = tile_desc(at + kRowsTile * kBlockK);
#pragma unroll
                    for (int j = 0; j < kBlockK / 32; ++j)
                        asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
                                     " tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n}"
                                     :: "r"(tmem + acc * BN), "l"(dp + 2 * j), "l"(dq + 2 * j), "r"(a.idesc), "r"(j) : "memory");
                    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" :: "r"(smem_u32(&empty[s])) : "memory");
                    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" :: "r"(smem_u32(&acc_full[acc])) : "memory");
                }
            if (!ok) {
                asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" :: "r"(smem_u32(&drain)) : "memory");
                for (uint32_t n = 0; n < kWaitLimit && !try_wait(smem_u32(&drain), 0); ++n) {}
            }
        }
        __syncwarp();
    } else {                                    // sums
        const int quarter = warp & 3, part = warp >> 2;
        const uint32_t row = 32 * quarter + lane;
        float* my_scales = scales + warp * 2 * S::kCols;
        uint32_t i = 0;
        bool ok = true;
        for (uint32_t tile = first; tile < a.tiles; tile += step) {
            const uint32_t z = tile / (a.p_tiles * a.q_tiles), t = tile - z * a.p_tiles * a.q_tiles;
            const uint32_t p = (t % a.p_tiles) * kRowsTile + row, q0 = (t / a.p_tiles) * BN + part * S::kCols;
            const float* sp = a.sp + (a.batched_p ? z * a.sp_batch : 0) + (uint64_t)(min(p, a.p - 1) >> a.p_shift) * a.kb;
            const float* sq = a.sq + (a.batched_q ? z * a.sq_batch : 0);
            float sum[S::kCols];
#pragma unroll
            for (int j = 0; j < S::kCols; ++j) sum[j] = 0.0f;
            // the next block's scales are fetched while this one's product is awaited
            float row_scale = 0.0f, col_scale[kByColumn ? (S::kCols + 31) / 32 : 1];
            const auto fetch = [&](uint32_t kb) {
                row_scale = __ldg(sp + kb);
                if constexpr (kByColumn) {
#pragma unroll
                    for (int j = 0; j < (S::kCols + 31) / 32; ++j) {
                        const uint32_t q = q0 + 32 * j + lane;
                        col_scale[j] = q < a.q && 32 * j + lane < (uint32_t)S::kCols ? __ldg(sq + (uint64_t)q * a.kb + kb) : 0.0f;
                    }
                } else {
                    col_scale[0] = q0 < a.q ? __ldg(sq + (uint64_t)(q0 >> 7) * a.kb + kb) : 0.0f;
                }
            };
            if (kb0 < kb1) fetch(kb0);
            for (uint32_t kb = kb0; ok && kb < kb1; ++kb, ++i) {
                const uint32_t acc = i % S::kAcc;
                float scale = row_scale;
                float* by_column = my_scales + (kb & 1) * S::kCols;
                if constexpr (kByColumn) {
#pragma unroll
                    for (int j = 0; j < (S::kCols + 31) / 32; ++j)
                        if (32 * j + lane < S::kCols) by_column[32 * j + lane] = col_scale[j];
                    __syncwarp();
                } else {
                    scale *= col_scale[0];
                }
                if (kb + 1 < kb1) fetch(kb + 1);
                ok = wait(smem_u32(&acc_full[acc]), (i / S::kAcc) & 1, failed);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint32_t at = tmem + acc * BN + part * S::kCols + ((32u * quarter) << 16);
                constexpr int kPiece = S::kCols >= 32 ? 32 : 16;
                uint32_t v[2][kPiece];
                TmemLoad<kPiece>::load(v[0], at);
#pragma unroll
                for (int j = 0; j < S::kCols; j += kPiece) {
                    const int w = (j / kPiece) & 1;
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                    if (j + kPiece < S::kCols) TmemLoad<kPiece>::load(v[w ^ 1], at + j + kPiece);
                    else {                      // everything is read: the accumulator is free
                        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                        if (lane == 0)
                            asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" :: "r"(smem_u32(&acc_empty[acc])) : "memory");
                    }
#pragma unroll
                    for (int e = 0; e < kPiece; ++e) {
                        if constexpr (kByColumn) sum[j + e] = fmaf(__uint_as_float(v[w][e]), scale * by_column[j + e], sum[j + e]);
                        else                     sum[j + e] = fmaf(__uint_as_float(v[w][e]), scale, sum[j + e]);
                    }
                }
            }
            if (!ok)
#pragma unroll
                for (int j = 0; j < S::kCols; ++j) sum[j] = qnan();

            if constexpr (S::kReduceBytes > 0) {
                if (a.split > 1) {
                    // block r of the cluster adds columns r * BN / split ..: part `rank` of everyone's, in the ranks' order
                    const uint32_t mine = BN / a.split;
                    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");       // everyone has started
#pragma unroll
                    for (int j = 0; j < S::kCols; ++j) {
                        const uint32_t q = part * S::kCols + j, to = q / mine, slot = q - to * mine;
                        const uint32_t local = smem_u32(reduce + (rank * mine + slot) * kRowsTile + row);
                        uint32_t remote;
                        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local), "r"(to));
                        asm volatile("st.shared::cluster.f32 [%0], %1;" :: "r"(remote), "f"(sum[j]) : "memory");
                    }
                }
            }
            if (a.split == 1 && p < a.p) {
                const uint64_t at = z * a.c_batch + (uint64_t)p * a.ldp + (uint64_t)q0 * a.ldq;
                if (a.wide && q0 + S::kCols <= a.q) {
                    if (a.c_dtype == METAL_LINALG_FLOAT32) {
#pragma unroll
                        for (int j = 0; j < S::kCols; j += 4)
                            *reinterpret_cast<float4*>(static_cast<float*>(a.c) + at + j) = make_float4(sum[j], sum[j + 1], sum[j + 2], sum[j + 3]);
                    } else {
#pragma unroll
                        for (int j = 0; j < S::kCols; j += 8)
                            *reinterpret_cast<uint4*>(static_cast<__half*>(a.c) + at + j) =
                                make_uint4(pack_two(a.c_dtype, sum[j], sum[j + 1]), pack_two(a.c_dtype, sum[j + 2], sum[j + 3]),
                                           pack_two(a.c_dtype, sum[j + 4], sum[j + 5]), pack_two(a.c_dtype, sum[j + 6], sum[j + 7]));
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < S::kCols; ++j)
                        if (q0 + j < a.q) store_one(a.c, at + (uint64_t)j * a.ldq, a.c_dtype, sum[j]);
                }
            }
        }
    }
    if (a.split > 1) {
        // loads' and products' warps took no part in the first wait yet
        if (warp >= S::kEpilogueWarps) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");                   // every partial sum has come
        if constexpr (S::kReduceBytes > 0) {
            const uint32_t mine = BN / a.split, tile = first;
            const uint32_t z = tile / (a.p_tiles * a.q_tiles), t = tile - z * a.p_tiles * a.q_tiles;
            const uint32_t p0 = (t % a.p_tiles) * kRowsTile, q0 = (t / a.p_tiles) * BN + rank * mine;
            for (uint32_t e = threadIdx.x; e < mine * kRowsTile; e += S::kThreads) {
                // along whichever dimension C is contiguous
                const uint32_t r = a.ldp == 1 ? e % kRowsTile : e / mine, j = a.ldp == 1 ? e / kRowsTile : e % mine;
                if (p0 + r >= a.p || q0 + j >= a.q) continue;
                float sum = 0.0f;
                for (uint32_t w = 0; w < a.split; ++w) sum += reduce[(w * mine + j) * kRowsTile + r];
                store_one(a.c, z * a.c_batch + (uint64_t)(p0 + r) * a.ldp + (uint64_t)(q0 + j) * a.ldq, a.c_dtype, sum);
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
    cuda_check(cudaFuncSetAttribute(fp8_gemm_kernel<BN, kByColumn>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::kShared),
               "fp8 product shared memory");
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(a.split > 1 ? a.tiles * a.split : std::min<uint32_t>(a.tiles, (uint32_t)sm_count));
    cfg.blockDim = dim3(S::kThreads);
    cfg.dynamicSmemBytes = S::kShared;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = a.split;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = a.split > 1 ? 1 : 0;
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
    a.split = 1;                    // shares of k: powers of two, no share without a block, no more blocks than multiprocessors
    if (bn <= 128)
        while (a.split < kMaxSplit && a.tiles * a.split * 2 <= (uint32_t)sms && a.split * 2 <= a.kb) a.split *= 2;
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
