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
    int row_blocks, block_rows;    // blocks that share a kv head's rows, rows of each
    int splits, quantum;           // slices of a sequence's positions: at most, and their steps
    float c;                       // |softmax scale| * log2(e), positive
    int negate;                    // the scale is negative: the queries change their sign
    float *ml, *acc;               // slices: [seq][kv head][slice][row] (max, sum), the same with hs sums of values
};

// Positions of a step.  Few rows: a wave's step, its rows held in registers; many rows: the block's, in LDS.
__host__ __device__ constexpr int tree_positions(int hsp, int type, int many) {
    return many || hsp * (type == LLM_F32 ? 4 : type == LLM_BF16 ? 2 : 1) <= 128 ? 64 : 32;
}
// Slices of `end` positions in steps of tp: of `quantum` steps, more where that gives more than `splits`; none is empty.
__host__ __device__ inline int tree_slices(int end, int tp, int splits, int quantum, int *steps) {
    const int all = max((end + tp - 1) / tp, 1);
    *steps = max(quantum, (all + splits - 1) / splits);
    return (all + *steps - 1) / *steps;
}

typedef void (*TreeKernel)(TreeArgs);
// The kernel for caches of `type` and queries of `q_type`, `tiles` tiles of 16 rows a wave, its waves taking positions
// (many 0) or rows (many: 4 or 8 waves), and its LDS bytes.
TreeKernel tree_kernel_64(int type, int q_type, int tiles, int many, size_t *lds);
TreeKernel tree_kernel_128(int type, int q_type, int tiles, int many, size_t *lds);
TreeKernel tree_kernel_192(int type, int q_type, int tiles, int many, size_t *lds);
TreeKernel tree_kernel_256(int type, int q_type, int tiles, int many, size_t *lds);
