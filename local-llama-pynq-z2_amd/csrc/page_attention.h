// Attention over a cache in pages: kernel arguments (internal header).  page_attention.hip holds the entry point,
// page_kernel.hip the kernel, compiled once for each head size.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/llm_hip.h"
#include "operators.h"
#include "slices.h"

struct PageArgs {
    const uint8_t *k, *v;
    const float *ks, *vs;
    int64_t id, head, s_id, s_head; // pool strides: codes, floats
    const uint8_t *q, *kr, *vr;     // queries, the new tokens' rows (NULL: none)
    uint8_t *o;
    int64_t q_seq, q_tok, q_head;   // bytes
    int64_t k_seq, k_tok, k_head;
    int64_t v_seq, v_tok, v_head;
    int64_t o_seq, o_tok, o_head;
    const int *table, *lens, *n;
    const uint64_t *mask;
    int per, n_pages, page, n_seq, n_kv, hs, group, max_n, zero_rest;
    int row_blocks;                 // workgroups that share a kv head's rows
    int new_tokens;                 // new tokens that count as a step
    int cap, each, least;           // slices of positions: at most in all (0: none) and of a head, their steps at least
    float c;                        // |softmax scale| * log2(e)
    float sign;                     // the queries' factor: the scale's sign, 0 where the scale is
    float *ml, *acc;                // slices: [slice][row] (exponent, sum), the same with hs sums of values
    int2 *plan;                     // [seq][kv head]: first slice, slices
};

__device__ __forceinline__ int page_len(const PageArgs &a, int seq) {
    return (int)min((int64_t)max(a.lens[seq], 0), (int64_t)a.per * a.page);
}
// Steps that a sequence's new tokens' own rows count as, and all of them: these and the blocks of its positions.
__device__ __forceinline__ int new_steps(const PageArgs &a, int nn) { return a.kr ? (nn + a.new_tokens - 1) / a.new_tokens : 0; }
__device__ __forceinline__ int steps_of(const PageArgs &a, int seq) {
    const int nn = a.n ? min(max(a.n[seq], 0), a.max_n) : a.max_n;
    return max((page_len(a, seq) + PAGE_BLOCK - 1) / PAGE_BLOCK + new_steps(a, nn), 1);
}

typedef void (*PageKernel)(PageArgs);
// The kernel for pages of `type` and queries of `q_type`, `tiles` tiles of 16 rows a wave, its waves taking positions or
// rows, and its LDS bytes.
PageKernel page_kernel_64(int type, int q_type, int tiles, int rows, size_t *lds);
PageKernel page_kernel_128(int type, int q_type, int tiles, int rows, size_t *lds);
PageKernel page_kernel_192(int type, int q_type, int tiles, int rows, size_t *lds);
PageKernel page_kernel_256(int type, int q_type, int tiles, int rows, size_t *lds);
