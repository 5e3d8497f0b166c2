// The gated delta rule's host side: what a call may be, where its workspace's parts lie, the launches. Nothing is
// allocated and nothing waits.
#include "delta.h"
#include "runtime.h"

#include <metal_linalg/core.h>

#include <stdexcept>
#include <string>

namespace metal_linalg {
namespace core {

namespace {

using mlb::delta::Args;
using mlb::delta::Gates;
using mlb::delta::kChunk;
using mlb::delta::kTriFloats;

[[noreturn]] void refuse(const char* who, const std::string& what) { throw std::invalid_argument(std::string(who) + " " + what); }

size_t element_bytes(uint32_t dtype) { return dtype == METAL_LINALG_FLOAT32 ? 4 : 2; }

// The shape alone: what workspace_bytes can say of it.
void check_shape(const char* who, const metal_linalg_delta& p) {
    if (p.dtype > METAL_LINALG_FLOAT16) refuse(who, "dtype must be float32, bfloat16 or float16");
    if (p.heads == 0 || p.value_heads == 0 || p.value_heads % p.heads) refuse(who, "value_heads must be a multiple of heads");
    if (p.value_heads > 65535) refuse(who, "value_heads must be at most 65535");
    if (p.key_dim == 0 || p.key_dim > 128) refuse(who, "key_dim must be 1 to 128");
    if (p.value_dim == 0 || p.value_dim > 256) refuse(who, "value_dim must be 1 to 256");
    if (p.tokens >= 1u << 30) refuse(who, "tokens must be below 2^30");
}
void check_sequences(const char* who, const metal_linalg_delta& p) {
    if (p.sequences && p.batch != 1) refuse(who, "batch must be 1 where cu_seqlens names the sequences");
    if ((p.sequences ? p.sequences : p.batch) > 65535) refuse(who, "at most 65535 sequences");
    const uint64_t chunks = (uint64_t)p.batch * ((uint64_t)p.tokens + kChunk) / kChunk + p.sequences;
    // (2^32 chunks and heads: a workspace of 400 TB and more, whose size so never passes 64 bits)
    if (chunks >= 1ull << 30 || chunks * p.value_heads >= 1ull << 32) refuse(who, "too many tokens");
}

// Every pointer is on one GPU, which is returned.
struct Placement {
    const char* who;
    int  device;
    bool known;                 // the caller vouches for it
    bool any = false;           // there is a pointer at all
    Placement(const char* w, int d) : who(w), device(d), known(d >= 0) {
        if (d < -1) refuse(w, "device must be a GPU or -1");
    }
    void need(const void* ptr, const char* name) {
        if (!ptr) refuse(who, std::string(name) + " is NULL");
        optional(ptr, name);
    }
    void optional(const void* ptr, const char* name) {
        if (!ptr) return;
        any = true;
        if (known) return;
        const int d = mlb::pointer_device(ptr);
        if (d < 0) refuse(who, std::string(name) + " is not a device pointer");
        if (device < 0) device = d;
        else if (d != device) refuse(who, std::string(name) + " lives on another GPU than the rest");
    }
};

bool on16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
// Whether every row of a [batch, tokens, heads, dim] tensor starts on 16 bytes and holds whole pieces of 16.
bool in_pieces(const void* p, const int64_t (&stride)[3], uint32_t dim, size_t size) {
    return on16(p) && dim * size % 16 == 0 && stride[0] * (int64_t)size % 16 == 0 && stride[1] * (int64_t)size % 16 == 0 &&
           stride[2] * (int64_t)size % 16 == 0;
}

// Hands out parts of the workspace (or, with no workspace, counts their bytes).
struct Carver {
    char* base;
    uint64_t at = 0;
    template <typename T> T* take(uint64_t count) {
        T* r = base ? reinterpret_cast<T*>(base + at) : nullptr;
        at += (count * sizeof(T) + 255) / 256 * 256;
        return r;
    }
};

Args args_of(const metal_linalg_delta& p) {
    Args a{};
    a.batch = p.batch; a.tokens = p.tokens; a.heads = p.heads; a.value_heads = p.value_heads;
    a.dk = p.key_dim; a.dv = p.value_dim; a.sequences = p.sequences; a.dtype = p.dtype; a.scale = p.scale;
    a.q = p.q; a.k = p.k; a.v = p.v; a.g = p.g; a.beta = p.beta; a.initial_state = p.initial_state;
    for (int i = 0; i < 3; ++i) {
        a.q_stride[i] = p.q_stride[i]; a.k_stride[i] = p.k_stride[i]; a.v_stride[i] = p.v_stride[i];
        a.g_stride[i] = p.g_stride[i]; a.beta_stride[i] = p.beta_stride[i];
    }
    a.cu = p.cu_seqlens;
    a.cu64 = p.index_bytes == 8;
    const size_t size = element_bytes(p.dtype);
    a.vec = in_pieces(p.q, p.q_stride, p.key_dim, size) && in_pieces(p.k, p.k_stride, p.key_dim, size) &&
            in_pieces(p.v, p.v_stride, p.value_dim, size);
    a.dkp = p.key_dim <= 64 ? 64 : 128;
    a.dvp = (p.value_dim + 15) / 16 * 16;
    a.seqs = p.sequences ? p.sequences : p.batch;
    a.row_chunks = (p.tokens + kChunk - 1) / kChunk;
    // ragged: sum ceil(len / 64) <= total / 64 + sequences
    a.chunks = p.sequences ? p.tokens / kChunk + p.sequences : p.batch * a.row_chunks;
    return a;
}

uint64_t carve(Args& a, char* base, bool backward) {
    Carver w{base};
    const uint64_t heads = (uint64_t)a.chunks * a.value_heads;
    if (a.sequences) {
        a.table = w.take<int>(2ull * a.chunks);
        a.first = w.take<int>((uint64_t)a.sequences + 3);
        a.order = w.take<int>(a.sequences);
    }
    a.gates = w.take<Gates>(heads);
    a.tri = w.take<float>(heads * kTriFloats);
    a.states = w.take<float>(heads * a.dkp * a.dvp);
    a.d = w.take<float>(heads * kChunk * a.dvp);
    if (backward) {
        a.tri_b = w.take<float>(heads * kTriFloats);
        a.d_states = w.take<float>(heads * a.dkp * a.dvp);
        a.dr = w.take<float>(heads * kChunk * a.dvp);
        if (a.value_heads != a.heads) {
            const uint64_t rows = (uint64_t)a.batch * a.tokens * a.value_heads * a.dk;
            a.fold_q = w.take<float>(rows);
            a.fold_k = w.take<float>(rows);
        }
    }
    return w.at;
}

// The inputs of either direction, checked.
void check_inputs(const char* who, const metal_linalg_delta& p, Placement& where) {
    check_shape(who, p);
    check_sequences(who, p);
    if (cpu_only()) throw std::runtime_error(std::string(who) + " this thread is set CPU-only, and this build has no CPU path");
    if (p.sequences) {
        if (p.index_bytes != 4 && p.index_bytes != 8) refuse(who, "index_bytes must be 4 or 8");
        where.need(p.cu_seqlens, "cu_seqlens");
    }
    if ((uint64_t)p.batch * p.tokens) {
        where.need(p.q, "q");
        where.need(p.k, "k");
        where.need(p.v, "v");
        where.need(p.g, "g");
        where.need(p.beta, "beta");
    }
    where.optional(p.initial_state, "initial_state");
}

void check_workspace(const char* who, uint64_t need, void* workspace, uint64_t bytes, Placement& where) {
    if (need == 0) return;
    where.need(workspace, "workspace");
    if (reinterpret_cast<uintptr_t>(workspace) & 255) refuse(who, "workspace is not on a 256-byte boundary");
    if (bytes < need) refuse(who, "workspace has " + std::to_string(bytes) + " bytes of the " + std::to_string(need) + " needed");
}

} // namespace

uint64_t gated_delta_rule_workspace_bytes(const metal_linalg_delta& p, bool backward) {
    check_shape("[gated_delta_rule]", p);
    check_sequences("[gated_delta_rule]", p);
    Args a = args_of(p);
    return carve(a, nullptr, backward);
}

void gated_delta_rule(const metal_linalg_delta& p, void* o, float* final_state, void* workspace, uint64_t bytes) {
    const char* who = "[gated_delta_rule]";
    Placement where(who, p.device);
    check_inputs(who, p, where);
    if ((uint64_t)p.batch * p.tokens) where.need(o, "o");
    where.optional(final_state, "final_state");
    Args a = args_of(p);
    check_workspace(who, carve(a, nullptr, false), workspace, bytes, where);
    if (!where.any || a.seqs == 0) return;
    carve(a, static_cast<char*>(workspace), false);
    a.o = o;
    a.final_state = final_state;
    mlb::DeviceGuard guard(where.device);
    mlb::delta::launch_forward(a, mlb::thread_stream(), mlb::sm_count(where.device));
}

void gated_delta_rule_backward(const metal_linalg_delta& p, const void* d_o, const int64_t* d_o_stride,
                               const float* d_final_state, void* dq, void* dk, void* dv, float* dg, float* dbeta,
                               float* d_initial_state, void* workspace, uint64_t bytes) {
    const char* who = "[gated_delta_rule_backward]";
    Placement where(who, p.device);
    check_inputs(who, p, where);
    Args a = args_of(p);
    if ((uint64_t)p.batch * p.tokens) {
        where.need(d_o, "d_o");
        if (!d_o_stride) refuse(who, "d_o_stride is NULL");
        where.need(dq, "dq");
        where.need(dk, "dk");
        where.need(dv, "dv");
        where.need(dg, "dg");
        where.need(dbeta, "dbeta");
        const int64_t stride[3] = {d_o_stride[0], d_o_stride[1], d_o_stride[2]};
        for (int i = 0; i < 3; ++i) a.do_stride[i] = stride[i];
        a.vec = a.vec && in_pieces(d_o, stride, p.value_dim, element_bytes(p.dtype));
    }
    where.optional(d_final_state, "d_final_state");
    where.optional(d_initial_state, "d_initial_state");
    check_workspace(who, carve(a, nullptr, true), workspace, bytes, where);
    if (!where.any || a.seqs == 0) return;
    carve(a, static_cast<char*>(workspace), true);
    a.d_o = d_o;
    a.d_final = d_final_state;
    a.dq = dq; a.dk_out = dk; a.dv_out = dv; a.dg = dg; a.dbeta = dbeta; a.d_initial = d_initial_state;
    mlb::DeviceGuard guard(where.device);
    mlb::delta::launch_backward(a, mlb::thread_stream(), mlb::sm_count(where.device));
}

void gated_delta_step(const metal_linalg_delta& p, void* o, float* pool, int64_t pool_stride, uint32_t pool_size,
                      const void* slots) {
    const char* who = "[gated_delta_step]";
    check_shape(who, p);
    if (p.batch > 65535) refuse(who, "batch must be at most 65535");
    if (cpu_only()) throw std::runtime_error(std::string(who) + " this thread is set CPU-only, and this build has no CPU path");
    if (slots && p.index_bytes != 4 && p.index_bytes != 8) refuse(who, "index_bytes must be 4 or 8");
    if ((uint64_t)p.batch * p.tokens == 0) return;
    const int64_t state = (int64_t)p.value_heads * p.key_dim * p.value_dim;
    if (pool_size > 1 && pool_stride < state) refuse(who, "pool_stride is smaller than a state");
    Placement where(who, p.device);
    where.need(p.q, "q");
    where.need(p.k, "k");
    where.need(p.v, "v");
    where.need(p.g, "g");
    where.need(p.beta, "beta");
    where.need(o, "o");
    if (pool_size) where.need(pool, "pool");
    where.optional(slots, "slots");
    mlb::delta::StepArgs a{};
    a.batch = p.batch; a.tokens = p.tokens; a.heads = p.heads; a.value_heads = p.value_heads;
    a.dk = p.key_dim; a.dv = p.value_dim; a.dtype = p.dtype; a.pool_size = pool_size; a.scale = p.scale;
    a.q = p.q; a.k = p.k; a.v = p.v; a.g = p.g; a.beta = p.beta;
    for (int i = 0; i < 3; ++i) {
        a.q_stride[i] = p.q_stride[i]; a.k_stride[i] = p.k_stride[i]; a.v_stride[i] = p.v_stride[i];
        a.g_stride[i] = p.g_stride[i]; a.beta_stride[i] = p.beta_stride[i];
    }
    a.pool_stride = pool_stride;
    a.pool = pool;
    a.slots = slots;
    a.slots64 = p.index_bytes == 8;
    a.vec = on16(pool) && p.value_dim % 4 == 0 && pool_stride % 4 == 0;
    a.o = o;
    mlb::DeviceGuard guard(where.device);
    mlb::delta::launch_step(a, mlb::thread_stream());
}

} // namespace core
} // namespace metal_linalg
