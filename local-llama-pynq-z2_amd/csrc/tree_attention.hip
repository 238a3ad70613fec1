// llm_tree_attention: the slices' join and the entry point (the kernel is in tree_kernel.hip).
#include <string.h>

#include <algorithm>

#include "device.h"
#include "operators.h"
#include "tree_attention.h"

namespace {

constexpr int TREE_MAX_SPLITS = 128;

// A row's slices joined: weights exp2(max_s - max), the four waves every fourth slice each.
template <int QT>
__global__ void __launch_bounds__(256) k_tree_join(TreeArgs a, int tp) {
    __shared__ float sm_f[TREE_MAX_SPLITS];
    __shared__ float sm_o[3][256];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int row = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
    const int len = min(max(a.lens[b], 0), a.ctx), nn = a.n ? min(max(a.n[b], 0), a.max_n) : a.max_n;
    int steps;
    const int slices = tree_slices((int)min((int64_t)len + nn, (int64_t)a.ctx), tp, a.splits, &steps);
    if (slices == 1 || row >= nn * a.group) return;
    const int64_t stride = (int64_t)a.max_n * a.group, base = ((int64_t)b * a.n_kv + h) * a.splits * stride + row;
    // every wave forms the weights; the loads of the values do not wait for them
    float m[TREE_MAX_SPLITS / 64], l[TREE_MAX_SPLITS / 64], mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < TREE_MAX_SPLITS / 64; i++) {
        const int s = lane + 64 * i;
        m[i] = s < slices ? a.ml[2 * (base + s * stride)] : -INFINITY;
        l[i] = s < slices ? a.ml[2 * (base + s * stride) + 1] : 0.0f;
        mx = fmaxf(mx, m[i]);
    }
    mx = wave_max(mx);
    const float mu = mx == -INFINITY ? 0.0f : mx;
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < TREE_MAX_SPLITS / 64; i++) {
        const float f = __builtin_amdgcn_exp2f(m[i] - mu);
        sum += l[i] * f;
        if (wave == 0) sm_f[lane + 64 * i] = f;
    }
    sum = wave_sum(sum);
    __syncthreads();
    float o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int s = wave; s < slices; s += 4) {
        const float f = sm_f[s];
        const float *acc = a.acc + (base + s * stride) * a.hs;
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (lane + 64 * i < a.hs) o[i] += acc[lane + 64 * i] * f;
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (wave) sm_o[wave - 1][lane + 64 * i] = o[i];
    __syncthreads();
    if (wave) return;
    const int t = row / a.group, g = row - t * a.group;
    uint8_t *op = a.o + b * a.o_seq + t * a.o_tok + (h * a.group + g) * a.o_head;
    const float il = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int d = lane + 64 * i;
        if (d >= a.hs) continue;
        const float v = (((o[i] + sm_o[0][d]) + sm_o[1][d]) + sm_o[2][d]) * il;
        if constexpr (QT == LLM_F32) ((float *)op)[d] = v;
        else ((__bf16 *)op)[d] = (__bf16)v;
    }
}

struct TreePlan {
    int hsp, tp, tiles, row_blocks, splits;
    size_t bytes;
};

// How a call is cut: rows of a kv head in tiles of 16, one tile a wave up to 16 rows and two from there where the registers
// allow it; positions in slices until the grid has two blocks a CU.
TreePlan tree_plan(const llm_kv *c, int n_heads, int max_n, int max_len) {
    TreePlan p;
    p.hsp = (c->hs + 63) / 64 * 64;
    p.tp = tree_positions(p.hsp, c->type);
    const int group = n_heads / c->n_kv, rows = group * max_n;
    p.tiles = rows > 16 && p.hsp <= 128 ? 2 : 1;
    p.row_blocks = (rows + 16 * p.tiles - 1) / (16 * p.tiles);
    const int64_t end = std::min<int64_t>((int64_t)std::max(max_len, 0) + max_n, c->ctx);
    const int64_t steps = (end + p.tp - 1) / p.tp, blocks = (int64_t)c->n_seq * c->n_kv * p.row_blocks;
    const int64_t want = std::max<int64_t>(1, 512 / std::max<int64_t>(blocks, 1));
    p.splits = (int)std::max<int64_t>(1, std::min({want, (steps + 3) / 4, (int64_t)TREE_MAX_SPLITS}));
    p.bytes = p.splits > 1 ? (size_t)c->n_seq * c->n_kv * p.splits * rows * (c->hs + 2) * 4 : 0;
    return p;
}

bool tree_shape_ok(const llm_kv *c, int n_heads, int max_n) {
    return c && op_type_bytes(c->type) && c->n_seq >= 0 && c->n_kv > 0 && c->hs >= 16 && c->hs <= 256 && c->hs % 16 == 0 &&
           c->ctx > 0 && max_n >= 0 && max_n <= 64 && n_heads > 0 && n_heads % c->n_kv == 0 && n_heads / c->n_kv <= 64;
}

} // namespace

extern "C" size_t llm_tree_attention_work(const llm_kv *c, int n_heads, int max_n, int max_len) {
    return tree_shape_ok(c, n_heads, max_n) ? tree_plan(c, n_heads, max_n, max_len).bytes : 0;
}

extern "C" int llm_tree_attention(const llm_kv *c, const llm_rows *q, const llm_rows *out, int n_heads, const int *lens,
                                  const int *n, const uint64_t *mask, int max_n, int max_len, float scale, int zero_rest,
                                  void *work, size_t work_bytes, void *stream) {
    const char *who = "llm_tree_attention";
    if (c && !op_check_cache(c, nullptr, who)) return -1;
    if (!c || !q || !out || !tree_shape_ok(c, n_heads, max_n)) {
        fprintf(stderr, "%s: bad arguments (at most 64 new tokens, query heads a multiple of the kv heads, at most 64 each)\n",
                who);
        return -1;
    }
    OpDevice dev(who);
    if (!op_check_cache(c, &dev, who)) return -1;
    if (!max_n || !c->n_seq) return 0;
    if (!op_check_rows(q, "q", &dev, who) || !op_check_rows(out, "out", &dev, who) || !dev.holds(lens, "lens") ||
        (n && !dev.holds(n, "n")) || (mask && !dev.holds(mask, "mask")))
        return -1;
    if (q->type != out->type) {
        fprintf(stderr, "%s: q and out of different types\n", who);
        return -1;
    }
    const TreePlan p = tree_plan(c, n_heads, max_n, max_len);
    if (p.bytes && (work_bytes < p.bytes || ((uintptr_t)work & 15) || !dev.holds(work, "the work memory"))) {
        fprintf(stderr, "%s: %zu bytes of work memory are needed, 16-byte aligned\n", who, p.bytes);
        return -1;
    }
    const int64_t blocks = (int64_t)c->n_seq * c->n_kv * p.splits;
    if (blocks > 0x7fffffff || c->n_seq > 65535 || c->n_kv > 65535) {
        fprintf(stderr, "%s: %d sequences of %d kv heads\n", who, c->n_seq, c->n_kv);
        return -1;
    }
    if (!dev.select()) return -1;
    const int cs = op_type_bytes(c->type), qs = op_type_bytes(q->type);
    TreeArgs a;
    memset(&a, 0, sizeof a);
    a.k = (const uint8_t *)c->k, a.v = (const uint8_t *)c->v;
    a.ks = c->k_scale, a.vs = c->v_scale;
    a.seq = c->seq * cs, a.head = c->head * cs, a.pos = c->pos * cs;
    a.s_seq = c->s_seq, a.s_head = c->s_head, a.s_pos = c->s_pos;
    a.q = (const uint8_t *)q->p, a.o = (uint8_t *)out->p;
    a.q_seq = q->seq * qs, a.q_tok = q->tok * qs, a.q_head = q->head * qs;
    a.o_seq = out->seq * qs, a.o_tok = out->tok * qs, a.o_head = out->head * qs;
    a.lens = lens, a.n = n, a.mask = mask;
    a.n_seq = c->n_seq, a.n_kv = c->n_kv, a.hs = c->hs, a.ctx = c->ctx;
    a.group = n_heads / c->n_kv, a.max_n = max_n, a.splits = p.splits, a.zero_rest = zero_rest;
    a.c = scale * 1.44269504088896340736f;
    a.acc = (float *)work; // (rows of hs values, hs a multiple of 16: 16-byte aligned)
    a.ml = (float *)work + (p.bytes / 4 / (c->hs + 2)) * c->hs;
    size_t lds = 0;
    auto *pick = p.hsp == 64 ? tree_kernel_64 : p.hsp == 128 ? tree_kernel_128 : p.hsp == 192 ? tree_kernel_192 : tree_kernel_256;
    TreeKernel kern = pick(c->type, q->type, p.tiles, &lds);
    if (!kern) {
        fprintf(stderr, "%s: internal error: no kernel\n", who);
        return -1;
    }
    hipLaunchKernelGGL(kern, dim3((unsigned)blocks, p.row_blocks), dim3(256), lds, (hipStream_t)stream, a);
    HIP_OR_FAIL(who, hipGetLastError());
    if (p.splits > 1) {
        const dim3 grid(max_n * a.group, c->n_kv, c->n_seq);
        if (q->type == LLM_F32) hipLaunchKernelGGL(k_tree_join<LLM_F32>, grid, dim3(256), 0, (hipStream_t)stream, a, p.tp);
        else hipLaunchKernelGGL(k_tree_join<LLM_BF16>, grid, dim3(256), 0, (hipStream_t)stream, a, p.tp);
        HIP_OR_FAIL(who, hipGetLastError());
    }
    return 0;
}
