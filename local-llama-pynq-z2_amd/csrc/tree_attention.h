// Attention of drafted tokens over a cache: kernel arguments (internal header).  tree_attention.hip holds the entry point,
// tree_kernel.hip the kernel, compiled once for each head size.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/llm_hip.h"

struct TreeArgs {
    const uint8_t *k, *v;
    const float *ks, *vs;
    int64_t seq, head, pos;        // cache strides in bytes
    int64_t s_seq, s_head, s_pos;  // of the scales, in floats
    const uint8_t *q;
    uint8_t *o;
    int64_t q_seq, q_tok, q_head;  // bytes
    int64_t o_seq, o_tok, o_head;
    const int *lens, *n;
    const uint64_t *mask;
    int n_seq, n_kv, hs, ctx, group, max_n, zero_rest;
    int splits;                    // slices of a sequence's positions, at most
    float c;                       // softmax scale * log2(e)
    float *ml, *acc;               // slices: [seq][kv head][slice][row] (max, sum), the same with hs sums of values
};

// A wave's step over the positions, a block's four waves side by side.
__host__ __device__ constexpr int tree_positions(int hsp, int type) {
    return hsp * (type == LLM_F32 ? 4 : type == LLM_BF16 ? 2 : 1) <= 128 ? 64 : 32;
}
// Slices of `end` positions: a block's four waves have a step each at least; none is empty.
__host__ __device__ inline int tree_slices(int end, int tp, int splits, int *steps) {
    const int all = (end + tp - 1) / tp;
    int s = (all + 3) / 4;
    if (s > splits) s = splits;
    if (s < 1) s = 1;
    *steps = (all + s - 1) / s;
    if (*steps < 1) *steps = 1;
    s = (all + *steps - 1) / *steps;
    return s < 1 ? 1 : s;
}

typedef void (*TreeKernel)(TreeArgs);
// The kernel for caches of `type` and queries of `q_type`, `tiles` tiles of 16 rows a wave, and its LDS bytes.
TreeKernel tree_kernel_64(int type, int q_type, int tiles, size_t *lds);
TreeKernel tree_kernel_128(int type, int q_type, int tiles, size_t *lds);
TreeKernel tree_kernel_192(int type, int q_type, int tiles, size_t *lds);
TreeKernel tree_kernel_256(int type, int q_type, int tiles, size_t *lds);
