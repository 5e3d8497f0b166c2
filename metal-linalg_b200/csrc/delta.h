#pragma once
// The gated delta rule behind metal_linalg_gated_delta_rule, its backward pass and
// metal_linalg_gated_delta_step: what the host and the kernels share.
//
// A chunk of kChunk = 64 tokens of a value head, with G the inclusive sums of g inside it and S the state at its start:
//
//     A_ij = beta_i e^{G_i - G_j} k_i . k_j  (j < i)       T = (I + A)^-1, unit lower triangular
//     R = beta (V - e^G K S)                               D = T R
//     O = scale (e^G Q S + P D), P_ij = e^{G_i - G_j} q_i . k_j  (j <= i)
//     S' = e^{G_63} S + (e^{G_63 - G} K)^T D
//
// K and T are the compact-WY form of the chunk's product of reflections. Everything is held in float32: the products
// run on the tensor cores with their float32 operands in several parts (delta_tiles.cuh), because states, gates'
// gradients and betas' gradients are float32 results. Sums of g are kept in 64 bits, so that the exponents' differences
// stay exact behind a gate that closes.
//
// Kernels: delta_index_kernel (ragged batches: the table of chunks), delta_prep_kernel (T and the decays, a chunk a
// block), delta_state_kernel (the only sequential pass: S and D chunk after chunk, 16 value columns a chain),
// delta_output_kernel (O, a chunk a block); backward: delta_do_kernel (P^T dO), delta_reverse_kernel (dS and dR, chunks
// backward), delta_grad_kernel (everything else, a chunk a block), delta_fold_kernel (heads that share q and k).
#include <metal_linalg/c_api.h>

#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

namespace mlb {
namespace delta {

constexpr int kChunk = 64;
constexpr int kTriTiles = 36;                            // 8 x 8 tiles of a lower triangle of 64
constexpr int kTriFloats = kTriTiles * 32 * 2;           // a tile: 32 lanes x 2 values of a fragment

// exp of a gate's running sums, a chunk and head.
struct Gates {
    float  sum[kChunk], rest[kChunk];   // G, in two parts: a float32 and what it leaves of the 64-bit sum
    float  e[kChunk];            // e^G
    float  left[kChunk];         // e^{G_63 - G}
    float  beta[kChunk];
};

struct Args {
    uint32_t batch, tokens, heads, value_heads, dk, dv, sequences, dtype;
    float    scale;
    const void *q, *k, *v, *d_o;
    const float *g, *beta, *initial_state;
    long long q_stride[3], k_stride[3], v_stride[3], g_stride[3], beta_stride[3], do_stride[3];
    const void* cu;
    int       cu64;
    int       vec;               // q, k, v (and d_o) can be read in 16-byte pieces
    uint32_t  dkp, dvp;          // dk up to 64 or 128, dv up to a multiple of 16
    uint32_t  seqs;              // batch, or sequences
    uint32_t  row_chunks;        // chunks of a batch row (sequences == 0)
    uint32_t  chunks;            // all of them; an upper bound for a ragged batch
    // workspace
    int*      table;             // ragged: {first token, tokens} a chunk
    int*      first;             // ragged: [sequences + 3] first chunk of a sequence; then the number of chunks, the tokens
                                 // behind the last sequence's end and those before the first one's start
    int*      order;             // ragged: [sequences] the sequences, long ones first
    Gates*    gates;             // [chunk][value head]
    float*    tri;               // [chunk][value head][kTriFloats]: T as B fragments, k along columns
    float*    tri_b;             // the same with k along rows (backward)
    float*    states;            // [chunk][value head][dkp][dvp]: S at the chunk's start
    float*    d;                 // [chunk][value head][64][dvp]: D
    float*    d_states;          // the gradient of the state behind the chunk
    float*    dr;                // [chunk][value head][64][dvp]: scale P^T dO, then dR
    float *   fold_q, *fold_k;   // [batch * tokens][value head][dk]: gradients of shared heads before their sum
    // outputs
    void *    o, *dq, *dk_out, *dv_out;
    float *   final_state, *dg, *dbeta, *d_initial;
    const float* d_final;
};

// The step kernel's own few arguments.
struct StepArgs {
    uint32_t batch, tokens, heads, value_heads, dk, dv, dtype, pool_size;
    float    scale;
    const void *q, *k, *v;
    const float *g, *beta;
    long long q_stride[3], k_stride[3], v_stride[3], g_stride[3], beta_stride[3], pool_stride;
    float*   pool;
    const void* slots;
    int      slots64, vec;
    void*    o;
};

void launch_forward(const Args& a, cudaStream_t stream, int sm_count);      // delta_forward.cu
void launch_prepare(const Args& a, cudaStream_t stream, bool backward);     // index, prep
void launch_states(const Args& a, cudaStream_t stream, int sm_count);
void launch_backward(const Args& a, cudaStream_t stream, int sm_count);     // delta_backward.cu
void launch_step(const StepArgs& a, cudaStream_t stream);                   // delta_step.cu

} // namespace delta
} // namespace mlb

namespace metal_linalg {
namespace core {

// What the C entry points of the same names do (delta.cpp); std::invalid_argument for what they refuse.
uint64_t gated_delta_rule_workspace_bytes(const metal_linalg_delta& p, bool backward);
void gated_delta_rule(const metal_linalg_delta& p, void* o, float* final_state, void* workspace, uint64_t bytes);
void gated_delta_rule_backward(const metal_linalg_delta& p, const void* d_o, const int64_t* d_o_stride,
                               const float* d_final_state, void* dq, void* dk, void* dv, float* dg, float* dbeta,
                               float* d_initial_state, void* workspace, uint64_t bytes);
void gated_delta_step(const metal_linalg_delta& p, void* o, float* pool, int64_t pool_stride, uint32_t pool_size,
                      const void* slots);

} // namespace core
} // namespace metal_linalg
