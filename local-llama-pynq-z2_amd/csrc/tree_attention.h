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
    int cap, each, least, tp;      // slices of positions: at most in all (0: none) and of a head, their steps at least, a
                                   // step's positions
    float c;                       // |softmax scale| * log2(e), positive
    float sign;                    // the queries' factor: the scale's sign, 0 where the scale is
    float *ml, *acc;               // slices: [slice][row] (max, sum), the same with hs sums of values
    int2 *plan;                    // [seq][kv head]: first slice, slices
};

// Positions of a step.  Few rows: a wave's step, its rows held in registers; many rows: the block's, in LDS.
__host__ __device__ constexpr int tree_positions(int hsp, int type, int many, int tiles) {
    return many || hsp * tiles * (type == LLM_F32 ? 4 : type == LLM_BF16 ? 2 : 1) <= 128 ? 64 : 32;
}
constexpr int TREE_MAX_SLICES = 128; // of a sequence's kv head
constexpr int TREE_MAX_SEQS = 512;   // of a call whose positions are cut
// A sequence of so many times the least steps stays whole: cutting it costs the join (7 rows over 300 int8 positions: 11.0 us
// whole, 12.4 in two slices; over 800, four times the least: 14.8 and 12.4).
constexpr int TREE_WHOLE = 3;

// Steps of a sequence: of its positions in the cache and its new tokens (at least one: its block writes the empty rows).
__device__ __forceinline__ int tree_steps(const TreeArgs &a, int seq) {
    const int len = min(max(a.lens[seq], 0), a.ctx), nn = a.n ? min(max(a.n[seq], 0), a.max_n) : a.max_n;
    return max(((int)min((int64_t)len + nn, (int64_t)a.ctx) + a.tp - 1) / a.tp, 1);
}
// Slices of the only sequence of a call, of `all` steps: head h has numbers h * each and on.
__device__ __forceinline__ int tree_one(const TreeArgs &a, int all, int &steps) {
    steps = all <= TREE_WHOLE * a.least ? all : max(a.least, (all + a.each - 1) / a.each);
    return (all + steps - 1) / steps;
}

typedef void (*TreeKernel)(TreeArgs);
// The kernel for caches of `type` and queries of `q_type`, `tiles` tiles of 16 rows a wave, its waves taking positions
// (many 0) or rows (many: 4 or 8 waves), and its LDS bytes.
TreeKernel tree_kernel_64(int type, int q_type, int tiles, int many, size_t *lds);
TreeKernel tree_kernel_128(int type, int q_type, int tiles, int many, size_t *lds);
TreeKernel tree_kernel_192(int type, int q_type, int tiles, int many, size_t *lds);
TreeKernel tree_kernel_256(int type, int q_type, int tiles, int many, size_t *lds);
