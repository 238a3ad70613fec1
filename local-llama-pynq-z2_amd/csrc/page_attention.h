// Attention over a cache in pages: kernel arguments (internal header).  page_attention.hip holds the entry point,
// page_kernel.hip the kernel, compiled once for each head size.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/llm_hip.h"
#include "operators.h"

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
    float c;                        // |softmax scale| * log2(e)
    float sign;                     // the queries' factor: the scale's sign, 0 where the scale is
};

typedef void (*PageKernel)(PageArgs);
// The kernel for pages of `type` and queries of `q_type`, and its LDS bytes.
PageKernel page_kernel_64(int type, int q_type, size_t *lds);
PageKernel page_kernel_128(int type, int q_type, size_t *lds);
PageKernel page_kernel_192(int type, int q_type, size_t *lds);
PageKernel page_kernel_256(int type, int q_type, size_t *lds);
