// llm_page_attention: the entry point (the kernel is in page_kernel.hip).
#include <string.h>

#include <algorithm>
#include <cmath>

#include "device.h"
#include "operators.h"
#include "page_attention.h"

namespace {

constexpr float LOG2E = 1.44269504088896340736f;

bool page_shape_ok(const llm_pages *c, int n_heads, int max_n) {
    return c && c->n_kv > 0 && max_n >= 0 && max_n <= 64 && n_heads > 0 && n_heads % c->n_kv == 0 &&
           n_heads / c->n_kv <= 64;
}

} // namespace

extern "C" size_t llm_page_attention_work(const llm_pages *, int, int, int, int) { return 0; }

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
    if (n_seq > 65535 || c->n_kv > 65535) {
        fprintf(stderr, "%s: %d sequences of %d kv heads\n", who, n_seq, c->n_kv);
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
    a.row_blocks = (a.group * max_n + 15) / 16;
    a.c = std::fabs(scale) * LOG2E;
    a.sign = scale > 0.0f ? 1.0f : scale < 0.0f ? -1.0f : 0.0f;
    const int hsp = (c->hs + 63) / 64 * 64;
    auto *pick = hsp == 64 ? page_kernel_64 : hsp == 128 ? page_kernel_128 : hsp == 192 ? page_kernel_192 : page_kernel_256;
    size_t lds = 0;
    PageKernel kern = pick(c->type, q->type, &lds);
    hipLaunchKernelGGL(kern, dim3(a.row_blocks, c->n_kv, n_seq), dim3(256), lds, (hipStream_t)stream, a);
    HIP_OR_FAIL(who, hipGetLastError());
    return 0;
}
