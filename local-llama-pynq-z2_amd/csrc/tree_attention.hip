// llm_tree_attention: the slices' join and the entry point (the kernel is in tree_kernel.hip).
#include <string.h>

#include <algorithm>
#include <cmath>

#include "device.h"
#include "operators.h"
#include "tree_attention.h"

namespace {

constexpr int TREE_MAX_SPLITS = 128;

// A row's slices joined: weights exp2(max_s - max).  W waves a row (the block has four): a thread takes four values of
// every (64 W / (hs / 4))-th slice, eight slices' loads at once.
template <int QT, int W>
__global__ void __launch_bounds__(256) k_tree_join(TreeArgs a, int tp) {
    __shared__ float sm_f[4 / W][TREE_MAX_SPLITS + 64]; // (a group's last loads may be past the last slice: weight 0)
    __shared__ float4 sm_o[256];
    constexpr int T = 64 * W;
    const int lane = threadIdx.x & 63, part = threadIdx.x / T, tid = threadIdx.x % T;
    const int row = blockIdx.x * (4 / W) + part, h = blockIdx.y, b = blockIdx.z;
    const int len = min(max(a.lens[b], 0), a.ctx), nn = a.n ? min(max(a.n[b], 0), a.max_n) : a.max_n;
    int steps;
    const int slices = tree_slices((int)min((int64_t)len + nn, (int64_t)a.ctx), tp, a.splits, a.quantum, &steps);
    if (slices == 1) return; // (every row of the sequence was finished by its block)
    const bool there = row < nn * a.group;
    const int64_t stride = (int64_t)a.max_n * a.group, base = ((int64_t)b * a.n_kv + h) * a.splits * stride + row;
    const int per = a.hs / 4, groups = T / per, g = tid / per, d = 4 * (tid - g * per);
    constexpr int U = 8;
    float4 v[U];
    auto load = [&](int s0) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int s = s0 + u * groups;
            v[u] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (there && g < groups && s < slices) v[u] = *(const float4 *)(a.acc + (base + s * stride) * a.hs + d);
        }
    };
    load(g); // (the first values do not wait for the weights)
    float m[TREE_MAX_SPLITS / 64], l[TREE_MAX_SPLITS / 64], mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < TREE_MAX_SPLITS / 64; i++) {
        const int s = lane + 64 * i;
        const bool have = there && s < slices;
        m[i] = have ? a.ml[2 * (base + s * stride)] : -INFINITY;
        l[i] = have ? a.ml[2 * (base + s * stride) + 1] : 0.0f;
        mx = fmaxf(mx, m[i]);
    }
    mx = wave_max(mx);
    const float mu = mx == -INFINITY ? 0.0f : mx;
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < TREE_MAX_SPLITS / 64; i++) {
        const float f = __builtin_amdgcn_exp2f(m[i] - mu);
        sum += l[i] * f;
        if (tid < 64) sm_f[part][lane + 64 * i] = f;
    }
    sum = wave_sum(sum);
    if (tid < 64) sm_f[part][lane + TREE_MAX_SPLITS] = 0.0f;
    __syncthreads();
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int s0 = g; s0 < slices; s0 += U * groups) {
        if (s0 != g) load(s0);
#pragma unroll
        for (int u = 0; u < U; u++) {
            const float f = sm_f[part][min(s0 + u * groups, TREE_MAX_SPLITS)];
            o.x += v[u].x * f, o.y += v[u].y * f, o.z += v[u].z * f, o.w += v[u].w * f;
        }
    }
    sm_o[threadIdx.x] = o;
    __syncthreads();
    if (g || !there) return;
    for (int k = 1; k < groups; k++) {
        const float4 x = sm_o[part * T + k * per + tid];
        o.x += x.x, o.y += x.y, o.z += x.z, o.w += x.w;
    }
    const int t = row / a.group, gr = row - t * a.group;
    uint8_t *op = a.o + b * a.o_seq + t * a.o_tok + (h * a.group + gr) * a.o_head;
    const float il = sum == 0.0f ? 0.0f : 1.0f / sum;
    o = make_float4(o.x * il, o.y * il, o.z * il, o.w * il);
    if constexpr (QT == LLM_F32) *(float4 *)(op + (size_t)d * 4) = o;
    else {
        typedef float f2 __attribute__((ext_vector_type(2)));
        typedef __bf16 b2 __attribute__((ext_vector_type(2)));
        *(uint2 *)(op + (size_t)d * 2) = make_uint2(__builtin_bit_cast(uint32_t, __builtin_convertvector((f2){o.x, o.y}, b2)),
                                                    __builtin_bit_cast(uint32_t, __builtin_convertvector((f2){o.z, o.w}, b2)));
    }
}

struct TreePlan {
    int hsp, tp, many, tiles, row_blocks, block_rows, splits, quantum;
    size_t bytes;
};

// How a call is cut.  Up to 32 rows a kv head: the block's four waves share the positions, with one or two tiles of 16 rows
// each.  More rows: the waves share the rows, 16 each (four waves up to 64 rows, else eight), and the cache's rows go
// through LDS.  (Not for fp32 caches, whose rows need no conversion, nor head sizes above 128, whose rows do not fit twice.
// fp32 queries over bf16 caches, three pieces, take two tiles in each of four waves: eight would spill.)  The rows are
// spread evenly over their blocks.  Positions in slices, the same number of steps for every sequence, until the grid has a
// block a CU (few rows) or two; four for several sequences, whose lengths the host does not know.
TreePlan tree_plan(const llm_kv *c, int q_type, int n_heads, int max_n, int max_len) {
    TreePlan p;
    p.hsp = (c->hs + 63) / 64 * 64;
    const int group = n_heads / c->n_kv, rows = group * max_n, tiles = (rows + 15) / 16;
    const bool many = rows > 32 && p.hsp <= 128 && c->type != LLM_F32, pieces = c->type == LLM_BF16 && q_type == LLM_F32;
    p.many = !many ? 0 : tiles <= 4 || pieces ? 4 : 8;
    p.tiles = many ? (tiles > 4 && pieces ? 2 : 1) : tiles > 1 && p.hsp <= 128 ? 2 : 1;
    const int per_block = p.tiles * (many ? p.many : 1); // tiles
    p.row_blocks = (tiles + per_block - 1) / per_block;
    p.block_rows = 16 * (many ? (tiles + p.row_blocks - 1) / p.row_blocks : per_block);
    p.tp = tree_positions(p.hsp, c->type, p.many);
    const int64_t end = std::min<int64_t>((int64_t)std::max(max_len, 0) + max_n, c->ctx);
    const int64_t steps = std::max<int64_t>((end + p.tp - 1) / p.tp, 1), blocks = (int64_t)c->n_seq * c->n_kv * p.row_blocks;
    const int64_t least = many ? 2 : 4; // steps of a slice (few rows: one a wave)
    const int64_t grid = c->n_seq > 1 ? 1024 : many ? 512 : 256;
    const int64_t cap = std::min({std::max<int64_t>(1, grid / std::max<int64_t>(blocks, 1)), (steps + least - 1) / least,
                                  (int64_t)TREE_MAX_SPLITS});
    // one sequence: as many slices as its length, known to the kernel, gives of the least size, up to that number
    p.quantum = (int)(c->n_seq > 1 ? (steps + cap - 1) / cap : least);
    p.splits = (int)(c->n_seq > 1 ? (steps + p.quantum - 1) / p.quantum : cap);
    p.bytes = p.splits > 1 ? (size_t)c->n_seq * c->n_kv * p.splits * rows * (c->hs + 2) * 4 : 0;
    return p;
}

int64_t tree_blocks(const llm_kv &c, const TreePlan &p) { // (rounded up to a slice for each XCD)
    return ((int64_t)c.n_seq * c.n_kv * p.splits + 7) / 8 * 8 * p.row_blocks;
}

bool tree_shape_ok(const llm_kv *c, int n_heads, int max_n) {
    return c && op_type_bytes(c->type) && c->n_seq >= 0 && c->n_kv > 0 && c->hs >= 16 && c->hs <= 256 && c->hs % 16 == 0 &&
           c->ctx > 0 && max_n >= 0 && max_n <= 64 && n_heads > 0 && n_heads % c->n_kv == 0 && n_heads / c->n_kv <= 64;
}

} // namespace

extern "C" size_t llm_tree_attention_work(const llm_kv *c, int n_heads, int max_n, int max_len) {
    return tree_shape_ok(c, n_heads, max_n) ? std::max(tree_plan(c, LLM_F32, n_heads, max_n, max_len).bytes,
                                                       tree_plan(c, LLM_BF16, n_heads, max_n, max_len).bytes) : 0;
}

hipError_t launch_tree_attention(const llm_kv &c, const llm_rows &q, const llm_rows &out, const TreeCall &t, hipStream_t st) {
    const TreePlan p = tree_plan(&c, q.type, t.n_heads, t.max_n, t.max_len);
    const int64_t blocks = tree_blocks(c, p);
    const int cs = op_type_bytes(c.type), qs = op_type_bytes(q.type);
    TreeArgs a;
    memset(&a, 0, sizeof a);
    a.k = (const uint8_t *)c.k, a.v = (const uint8_t *)c.v;
    a.ks = c.k_scale, a.vs = c.v_scale;
    a.seq = c.seq * cs, a.head = c.head * cs, a.pos = c.pos * cs;
    a.s_seq = c.s_seq, a.s_head = c.s_head, a.s_pos = c.s_pos;
    a.q = (const uint8_t *)q.p, a.o = (uint8_t *)out.p;
    a.q_seq = q.seq * qs, a.q_tok = q.tok * qs, a.q_head = q.head * qs;
    a.o_seq = out.seq * qs, a.o_tok = out.tok * qs, a.o_head = out.head * qs;
    a.lens = t.lens, a.n = t.n, a.mask = t.mask;
    a.n_seq = c.n_seq, a.n_kv = c.n_kv, a.hs = c.hs, a.ctx = c.ctx;
    a.group = t.n_heads / c.n_kv, a.max_n = t.max_n, a.row_blocks = p.row_blocks, a.block_rows = p.block_rows;
    a.splits = p.splits, a.quantum = p.quantum, a.zero_rest = t.zero_rest;
    // (a scale of 0 as one so small that every weight is 1)
    a.c = std::max(std::fabs(t.scale) * 1.44269504088896340736f, 1e-30f);
    a.negate = t.scale < 0.0f;
    a.acc = (float *)t.work; // (rows of hs values, hs a multiple of 16: 16-byte aligned)
    a.ml = (float *)t.work + (p.bytes / 4 / (c.hs + 2)) * c.hs;
    size_t lds = 0;
    auto *pick = p.hsp == 64 ? tree_kernel_64 : p.hsp == 128 ? tree_kernel_128 : p.hsp == 192 ? tree_kernel_192 : tree_kernel_256;
    TreeKernel kern = pick(c.type, q.type, p.tiles, p.many, &lds);
    if (!kern) return hipErrorInvalidValue;
    hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3(p.many ? 64 * p.many : 256), lds, st, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.splits == 1) return e;
    // a wave a row up to 8 slices, the block's four above
    const bool wide = p.splits > 8;
    const dim3 grid(wide ? t.max_n * a.group : (t.max_n * a.group + 3) / 4, c.n_kv, c.n_seq);
    auto *join = q.type == LLM_F32 ? wide ? k_tree_join<LLM_F32, 4> : k_tree_join<LLM_F32, 1>
                                   : wide ? k_tree_join<LLM_BF16, 4> : k_tree_join<LLM_BF16, 1>;
    hipLaunchKernelGGL(join, grid, dim3(256), 0, st, a, p.tp);
    return hipGetLastError();
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
    if (!std::isfinite(scale)) {
        fprintf(stderr, "%s: scale %g\n", who, scale);
        return -1;
    }
    if (q->type != out->type) {
        fprintf(stderr, "%s: q and out of different types\n", who);
        return -1;
    }
    const TreePlan p = tree_plan(c, q->type, n_heads, max_n, max_len);
    if (p.bytes && (work_bytes < p.bytes || ((uintptr_t)work & 15) || !dev.holds(work, "the work memory"))) {
        fprintf(stderr, "%s: %zu bytes of work memory are needed, 16-byte aligned\n", who, p.bytes);
        return -1;
    }
    if (tree_blocks(*c, p) > 0x7fffffff || c->n_seq > 65535 || c->n_kv > 65535) {
        fprintf(stderr, "%s: %d sequences of %d kv heads\n", who, c->n_seq, c->n_kv);
        return -1;
    }
    if (!dev.select()) return -1;
    const TreeCall t = {n_heads, lens, n, mask, max_n, max_len, scale, zero_rest, work};
    HIP_OR_FAIL(who, launch_tree_attention(*c, *q, *out, t, (hipStream_t)stream));
    return 0;
}
