// llm_page_attention: how a call is cut, and the entry point (the kernel is in page_kernel.hip).
#include <string.h>

#include <algorithm>
#include <cmath>

#include "device.h"
#include "operators.h"
#include "page_attention.h"

namespace {

constexpr float LOG2E = 1.44269504088896340736f;

struct PagePlan {
    int hsp, tiles, rows, row_blocks, block_rows, new_tokens, cap, each, least;
    size_t bytes;
};

// How a call is cut.  Times: one call, heads of 128, int8 pages.
// Rows.  The four waves of a workgroup share the positions, with one tile of 16 rows, or two where that is work enough: two read
// and convert the codes half as often, one gives twice the workgroups.  One sequence, one tile and two, bf16 rows and fp32: 37
// tokens of 7 heads over 9500 positions 32.0 and 33.2, 32.3 and 32.1 us, over 10500 34.0 and 33.8, 33.5 and 32.8, over 11500 35.1
// and 32.9, 35.4 and 34.5; 16 tokens over 26k 30.8 and 31.7, 31.5 and 33.3, over 30k 33.8 and 33.2, 34.5 and 34.5; 64 over 5000
// 30.1 and 29.7, 30.3 and 30.5, over 6000 33.3 and 31.7, 33.7 and 32.9: they cross between 1.1e6 and 1.6e6.  Several: 448 rows over
// 4 x 8000 70.6 and 62.0, 73.2 and 64.7.  Many rows over long contexts: the waves have two other tiles each of the same positions,
// which need no join of waves, and whose pages the L1 then holds for all four (448 rows over eight sequences of up to 16k: 200 us
// with waves over positions, 139 over rows; over eight of 3000 55 and 61, over two of 16k 72 and 72, fp32 58 and 62, 77 and 83).
// Positions.  One sequence: as many slices as give a workgroup a CU, or two a CU where whole row blocks would leave much of the
// chip idle.  Several: two workgroups a CU over all sequences, of equal steps (more of them cost more in find_slice and the join
// than they even out: 32 decode steps over 0 to 8190 e4m3 positions 32 us, with four a CU 35; with heads of 64 15.3 and 19.1, of
// int8 and fp32 rows 16.0 and 19.8, with six heads of 48 18.1 and 20.8).
PagePlan page_plan(const llm_pages *c, int n_seq, int n_heads, int max_n, int max_len) {
    PagePlan p;
    p.hsp = (c->hs + 63) / 64 * 64;
    const int group = n_heads / c->n_kv, rows = group * max_n, tiles = (rows + 15) / 16;
    const int64_t heads = (int64_t)n_seq * c->n_kv, blocks = ((int64_t)std::max(max_len, 0) + PAGE_BLOCK - 1) / PAGE_BLOCK;
    const double work = p.hsp <= 128 && tiles > 1 ? (double)tiles * heads * blocks * p.hsp : 0.0;
    p.tiles = work >= (n_seq > 1 ? 2e6 : 1.4e6) ? 2 : 1; // (of several sequences most are shorter than max_len)
    p.rows = work >= 6e6 && tiles > 8;
    p.block_rows = 16 * p.tiles * (p.rows ? 4 : 1);
    p.row_blocks = (rows + p.block_rows - 1) / p.block_rows;
    p.least = p.rows ? 2 : 4; // steps of a slice (one a wave)
    p.new_tokens = 16;        // (16 new tokens' rows take about as long as a block)
    const int64_t steps = blocks + (max_n + p.new_tokens - 1) / p.new_tokens;
    // per XCD; a single sequence: one workgroup a CU, two where whole row blocks would leave much of the chip idle
    const int64_t one = std::max(32 / p.row_blocks, 1) * 8, both = std::max(64 / p.row_blocks, 1) * 8;
    int64_t cap = both, each = MAX_SLICES;
    if (n_seq == 1) {
        cap = p.tiles > 1 || both / c->n_kv * 5 > one / c->n_kv * 11 ? both : one;
        each = std::max<int64_t>(std::min({cap / c->n_kv, (steps + p.least - 1) / p.least, each}), 1);
        cap = each * c->n_kv;
    }
    p.cap = cap <= heads || n_seq > MAX_CUT_SEQS || steps <= WHOLE_STEPS * p.least ? 0 : (int)cap;
    p.each = (int)each;
    p.bytes = p.cap ? (size_t)p.cap * rows * (c->hs + 2) * 4 + heads * sizeof(int2) : 0;
    return p;
}

int64_t page_blocks(const llm_pages *c, int n_seq, const PagePlan &p) { // (rounded up to a slice for each XCD)
    return ((p.cap ? p.cap : (int64_t)n_seq * c->n_kv) + 7) / 8 * 8 * p.row_blocks;
}

bool page_shape_ok(const llm_pages *c, int n_heads, int max_n) {
    return c && c->n_kv > 0 && max_n >= 0 && max_n <= 64 && n_heads > 0 && n_heads % c->n_kv == 0 &&
           n_heads / c->n_kv <= 64;
}

} // namespace

extern "C" size_t llm_page_attention_work(const llm_pages *c, int n_seq, int n_heads, int max_n, int max_len) {
    return page_shape_ok(c, n_heads, max_n) && max_n > 0 && n_seq > 0 && c->hs >= 16 && c->hs <= 256
               ? page_plan(c, n_seq, n_heads, max_n, max_len).bytes : 0;
}

extern "C" int llm_page_attention(const llm_pages *c, const llm_rows *q, const llm_rows *k, const llm_rows *v,
                                  const llm_rows *out, int n_heads, int n_seq, const int *table, int per, const int *lens,
                                  const int *n, const uint64_t *mask, int max_n, int max_len, float scale, int zero_rest,
                                  void *work, size_t work_bytes, void *stream) {
    const char *who = "llm_page_attention";
    if (c && !op_check_pages(c, nullptr, who)) return -1;
    if (!c || !q || !out || (k == nullptr) != (v == nullptr) || !page_shape_ok(c, n_heads, max_n)) {
        fprintf(stderr, "%s: bad arguments (at most 64 new tokens, query heads a multiple of the kv heads, at most 64 each, "
                "new rows of K and V or neither)\n", who);
        return -1;
    }
    if (!op_check_table(table, n_seq, per, nullptr, who)) return -1;
    if (!std::isfinite(scale * LOG2E)) {
        fprintf(stderr, "%s: scale %g\n", who, scale);
        return -1;
    }
    const int count[] = {n_seq, max_n, n_heads};
    const int64_t stride[] = {out->seq, out->tok, out->head};
    if (!op_check_apart(who, "out", 3, count, stride)) return -1;
    PagePlan p = {};
    if (max_n && n_seq) p = page_plan(c, n_seq, n_heads, max_n, max_len);
    if (n_seq > 65535 || c->n_kv > 65535 || (p.row_blocks && page_blocks(c, n_seq, p) >= 1 << 24)) { // (a grid has 2^32 threads)
        fprintf(stderr, "%s: %d sequences of %d kv heads\n", who, n_seq, c->n_kv);
        return -1;
    }
    OpDevice dev(who);
    if (!op_check_pages(c, &dev, who)) return -1;
    if (!max_n || !n_seq) return 0;
    if (!op_check_rows(q, "q", &dev, who) || !op_check_rows(out, "out", &dev, who) ||
        (k && (!op_check_rows(k, "k", &dev, who) || !op_check_rows(v, "v", &dev, who))) ||
        !op_check_table(table, n_seq, per, &dev, who) || !dev.holds(lens, "lens") || (n && !dev.holds(n, "n")) ||
        (mask && !dev.holds(mask, "mask")))
        return -1;
    if (q->type != out->type || (k && (k->type != q->type || v->type != q->type))) {
        fprintf(stderr, "%s: q, out and the new rows are of different types\n", who);
        return -1;
    }
    if (p.bytes && (work_bytes < p.bytes || ((uintptr_t)work & 15) || !dev.holds(work, "the work memory"))) {
        fprintf(stderr, "%s: %zu bytes of work memory are needed, 16-byte aligned\n", who, p.bytes);
        return -1;
    }
    if (!dev.select()) return -1;
    const int qs = op_type_bytes(q->type);
    PageArgs a;
    memset(&a, 0, sizeof a);
    a.k = (const uint8_t *)c->k, a.v = (const uint8_t *)c->v, a.ks = c->k_scale, a.vs = c->v_scale;
    a.id = c->id, a.head = c->head, a.s_id = c->s_id, a.s_head = c->s_head;
    a.q = (const uint8_t *)q->p, a.o = (uint8_t *)out->p;
    a.q_seq = q->seq * qs, a.q_tok = q->tok * qs, a.q_head = q->head * qs;
    a.o_seq = out->seq * qs, a.o_tok = out->tok * qs, a.o_head = out->head * qs;
    if (k) {
        a.kr = (const uint8_t *)k->p, a.vr = (const uint8_t *)v->p;
        a.k_seq = k->seq * qs, a.k_tok = k->tok * qs, a.k_head = k->head * qs;
        a.v_seq = v->seq * qs, a.v_tok = v->tok * qs, a.v_head = v->head * qs;
    }
    a.table = table, a.lens = lens, a.n = n, a.mask = mask;
    a.per = per, a.n_pages = c->n_pages, a.page = c->page, a.n_seq = n_seq, a.n_kv = c->n_kv, a.hs = c->hs;
    a.group = n_heads / c->n_kv, a.max_n = max_n, a.zero_rest = zero_rest;
    a.row_blocks = p.row_blocks, a.cap = p.cap, a.each = p.each, a.least = p.least;
    a.new_tokens = p.new_tokens;
    a.c = std::fabs(scale) * LOG2E;
    a.sign = scale > 0.0f ? 1.0f : scale < 0.0f ? -1.0f : 0.0f;
    a.acc = (float *)work; // (rows of hs values, hs a multiple of 16: 16-byte aligned)
    const size_t parts = (size_t)p.cap * a.group * max_n;
    a.ml = a.acc + parts * c->hs;
    a.plan = (int2 *)(a.ml + 2 * parts);
    auto *pick = p.hsp == 64 ? page_kernel_64 : p.hsp == 128 ? page_kernel_128 : p.hsp == 192 ? page_kernel_192 : page_kernel_256;
    size_t lds = 0;
    PageKernel kern = pick(c->type, q->type, p.tiles, p.rows, &lds);
    if (!kern) {
        fprintf(stderr, "%s: no kernel\n", who);
        return -1;
    }
    hipStream_t st = (hipStream_t)stream;
    hipLaunchKernelGGL(kern, dim3((unsigned)page_blocks(c, n_seq, p)), dim3(256), lds, st, a);
    HIP_OR_FAIL(who, hipGetLastError());
    if (!p.cap) return 0;
    // a wave a row up to 16 slices a head, the block's four above
    const bool wide = p.cap > 16 * n_seq * c->n_kv;
    const dim3 grid(wide ? max_n * a.group : (max_n * a.group + 3) / 4, c->n_kv, n_seq);
    auto *join = q->type == LLM_F32 ? wide ? k_join_slices<PageArgs, LLM_F32, 4> : k_join_slices<PageArgs, LLM_F32, 1>
                                    : wide ? k_join_slices<PageArgs, LLM_BF16, 4> : k_join_slices<PageArgs, LLM_BF16, 1>;
    hipLaunchKernelGGL(join, grid, dim3(256), 0, st, a);
    HIP_OR_FAIL(who, hipGetLastError());
    return 0;
}
