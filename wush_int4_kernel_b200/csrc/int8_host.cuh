// Host-side declarations shared by the 8-bit operators: quant_int8.cu, expert_order.cu, gemm_w8a8.cu, expert_ffn.cu.
#pragma once
#include <type_traits>

#include "common.cuh"

namespace wush {

static inline bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }
static inline bool aligned8(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 7u) == 0; }

// Limits of the entries (token, expert) that the expert operators take: positions are 32-bit.
static inline int check_entries(const char* op, int64_t tokens, int64_t k, int64_t n_experts)
{
    if (tokens < 0 || k < 1 || k > WUSH_EXPERT_MAX_K || n_experts < 1 || n_experts > WUSH_EXPERT_MAX)
        return fail(WUSH_ERR_INVALID_ARGUMENT, "%s: takes 1..%d experts per token and 1..%d experts (got %lld of %lld)", op,
                    WUSH_EXPERT_MAX_K, WUSH_EXPERT_MAX, (long long)k, (long long)n_experts);
    if (tokens * k > 0x7fffffffll)
        return fail(WUSH_ERR_UNSUPPORTED, "%s: more than 2^31 - 1 entries (%lld tokens of %lld)", op, (long long)tokens, (long long)k);
    return WUSH_OK;
}

// Launchers used by the entry points of one operator and by the expert block, which chains them.  `dependent`: launched
// with programmatic serialisation, so the kernel may start under the one before it; it waits for that one before it reads
// anything that the one before it wrote.
struct QuantRows {
    const void* x;
    int dtype;
    int64_t rows, K;
    int8_t* q;
    float* s;
    const int32_t* pos;      // (rows, k) destinations, or null: row r to row r
    int k;
    const int32_t* n_used;   // with pos: rows of the result from *n_used on become zero
    int32_t* counters;       // W8A8_COUNTER_BYTES to zero for the product that follows, or null
};
int quant_int8_launch(const QuantRows& a, bool dependent, cudaStream_t st);
int expert_sort_launch(const void* ids, int id_bytes, int64_t n, int n_experts, int32_t* pos, int32_t* offsets, cudaStream_t st);
int expert_combine_launch(const void* rows, int dtype, int out_dtype, int64_t tokens, int64_t H, const int32_t* pos, int k, const float* weights,
                          void* y, bool dependent, cudaStream_t st);

struct W8A8Problem {
    const int8_t* xq;        // (rows, K)
    const float* xs;         // (rows)
    const int8_t* wq;        // (experts, N, K); gated: (experts, 2 * N, K), the N gate channels first
    const float* ws;         // (experts, N) or (experts, 2 * N)
    const float* bias;       // (N) or null; one expert only
    const int32_t* offsets;  // (experts + 1) first row of each expert, or null: one expert with all rows
    int64_t rows, N, K, experts;
    bool gated;
    int out_dtype;           // gated: always fp32
    void* y;                 // (rows, N)
};
// The product's workspace: counters, which are zero when its kernel starts, then slots.
constexpr size_t W8A8_COUNTER_BYTES = 1024;
size_t w8a8_workspace_bytes(int64_t rows, int64_t experts);
// Dependent: weights and offsets are older than the kernel in front, so they are read before the wait for it.
int w8a8_launch(const W8A8Problem& p, void* workspace, bool dependent, cudaStream_t st);

}  // namespace wush
