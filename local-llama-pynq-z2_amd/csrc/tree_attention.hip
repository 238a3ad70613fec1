// llm_tree_attention: the slices' join and the entry point (the kernel is in tree_kernel.hip).
#include <string.h>

#include <algorithm>
#include <cmath>

#include "device.h"
#include "operators.h"
#include "tree_attention.h"

namespace {

// A row's slices joined: weights exp2(max_s - max).  W waves a row (the block has four): a thread takes four values of
// every (64 W / (hs / 4))-th slice, eight slices' loads at once.
template <int QT, int W>
__global__ void __launch_bounds__(256) k_tree_join(TreeArgs a) {
    __shared__ float sm_f[4 / W][TREE_MAX_SLICES + 64]; // (a group's last loads may be past the last slice: weight 0)
    __shared__ float4 sm_o[256];
    constexpr int T = 64 * W;
    const int lane = threadIdx.x & 63, part = threadIdx.x / T, tid = threadIdx.x % T;
    const int row = blockIdx.x * (4 / W) + part, h = blockIdx.y, b = blockIdx.z;
    const int nn = a.n ? min(max(a.n[b], 0), a.max_n) : a.max_n;
    int slices, first;
    if (a.n_seq == 1) {
        int steps;
        slices = tree_one(a, tree_steps(a, 0), steps);
        first = h * a.each;
    } else {
        const int2 plan = a.plan[b * a.n_kv + h];
        first = plan.x;
        slices = plan.y;
    }
    if (slices == 1) return; // (every row of the sequence was finished by its block)
    const bool there = row < nn * a.group;
    const int64_t stride = (int64_t)a.max_n * a.group, base = first * stride + row;
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
    float m[TREE_MAX_SLICES / 64], l[TREE_MAX_SLICES / 64], mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < TREE_MAX_SLICES / 64; i++) {
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
    for (int i = 0; i < TREE_MAX_SLICES / 64; i++) {
        const float f = __builtin_amdgcn_exp2f(m[i] - mu);
        sum += l[i] * f;
        if (tid < 64) sm_f[part][lane + 64 * i] = f;
    }
    sum = wave_sum(sum);
    if (tid < 64) sm_f[part][lane + TREE_MAX_SLICES] = 0.0f;
    __syncthreads();
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int s0 = g; s0 < slices; s0 += U * groups) {
        if (s0 != g) load(s0);
#pragma unroll
        for (int u = 0; u < U; u++) {
            const float f = sm_f[part][min(s0 + u * groups, TREE_MAX_SLICES)];
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

constexpr float LOG2E = 1.44269504088896340736f;

struct TreePlan {
    int hsp, tp, many, tiles, row_blocks, block_rows, cap, each, least;
    size_t bytes;
};

// How a call is cut.  Times: one call, heads of 128.
// Rows.  The block's four waves share the positions, with one tile of 16 rows, or two where that is work enough: two read
// and convert half as often, one gives twice the blocks (112 rows over 32k bf16 positions, 4 kv heads: 44 us with one tile, 31
// with two; over 700: 10.8 and 13.7.  448 rows over 8 x 4000 int8 positions: 113 and 91; 63 rows over 32 x 2000: 39 and 41).
// Not for fp32 caches, nor fp32 queries over bf16 ones (three pieces), whose registers leave one wave a SIMD.  Many rows over
// a bf16 cache, whose L2 traffic then bounds: the waves share the rows, and the cache's rows go through LDS (eight
// sequences of up to 16k positions, 448 rows: 186 us with two tiles, 144 with LDS; one sequence of 700: 14 and 18).  fp32
// queries take two tiles in each of four waves there (eight waves of one would spill), bf16 ones one in each of eight.  The
// rows are spread evenly over these blocks.
// The thresholds were measured at heads of 128 and hold at 64 for one sequence (448 rows over 32k int8 positions: 50 us with one
// tile, 43 with two, which it takes; 259 over 12k: 17.9 with one, which it takes, 20.4; bf16: 49 and 32, 21 and 18, two); for
// batches there it can be a third off (448 rows over 8 x 4000 int8 positions: 28 us with one, 34 with two, which it takes; over
// 8 x 700 bf16 ones: 13.6 and 18.9, two).
// Positions.  One sequence: as many slices as give a block a CU, or two a CU where whole row blocks would leave much of the
// chip idle (192 rows over 32k int8 positions: 70 us with 192 blocks, 55 with 480; 7 rows: 16 with 256, 18 with 512).
// Several: two blocks a CU over all sequences, of equal steps (a decode step of 32 sequences, 0 to 8190 e4m3 positions: 31 us,
// 37 with four a CU; with the same number of slices for each sequence, 37).
TreePlan tree_plan(const llm_kv *c, int q_type, int n_heads, int max_n, int max_len) {
    TreePlan p;
    p.hsp = (c->hs + 63) / 64 * 64;
    const int group = n_heads / c->n_kv, rows = group * max_n, tiles = (rows + 15) / 16;
    const int64_t end = std::min<int64_t>((int64_t)std::max(max_len, 0) + max_n, c->ctx), heads = (int64_t)c->n_seq * c->n_kv;
    const bool bf16 = c->type == LLM_BF16, pieces = bf16 && q_type == LLM_F32, small = p.hsp <= 128;
    const double work = (double)tiles * heads * end;
    const bool many = bf16 && p.hsp == 128 && tiles > 8 && work >= (pieces ? 8e5 : 2e6);
    p.many = !many ? 0 : pieces ? 4 : 8;
    const bool two = small && c->type != LLM_F32 && !pieces &&
                     (bf16 ? tiles > 2 && work >= 2.5e5 : tiles > 5 && work * p.hsp >= 1e8);
    p.tiles = many ? (pieces ? 2 : 1) : two ? 2 : 1;
    const int per_block = p.tiles * (many ? p.many : 1); // tiles
    p.row_blocks = (tiles + per_block - 1) / per_block;
    const int waves = (tiles + p.row_blocks * p.tiles - 1) / (p.row_blocks * p.tiles); // that have rows
    p.block_rows = 16 * (many ? waves * p.tiles : per_block);
    p.tp = tree_positions(p.hsp, c->type, p.many, p.tiles);
    const int64_t steps = std::max<int64_t>((end + p.tp - 1) / p.tp, 1);
    p.least = many ? 2 : 4; // steps of a slice (few rows: one a wave)
    // per XCD; a single sequence: one block a CU, two where whole blocks would leave much of the chip idle
    const int64_t one = 32 / p.row_blocks * 8, both = 64 / p.row_blocks * 8;
    int64_t cap = both, each = TREE_MAX_SLICES;
    if (c->n_seq == 1) {
        cap = both / c->n_kv * 5 > one / c->n_kv * 11 ? both : one;
        each = std::min({cap / c->n_kv, (steps + p.least - 1) / p.least, each});
        cap = each * c->n_kv;
    }
    p.cap = cap <= heads || c->n_seq > TREE_MAX_SEQS || steps <= TREE_WHOLE * p.least ? 0 : (int)cap;
    p.each = (int)each;
    p.bytes = p.cap ? (size_t)p.cap * rows * (c->hs + 2) * 4 + heads * sizeof(int2) : 0;
    return p;
}

int64_t tree_blocks(const llm_kv &c, const TreePlan &p) { // (rounded up to a slice for each XCD)
    return ((p.cap ? p.cap : (int64_t)c.n_seq * c.n_kv) + 7) / 8 * 8 * p.row_blocks;
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
    a.cap = p.cap, a.each = p.each, a.least = p.least, a.tp = p.tp, a.zero_rest = t.zero_rest;
    a.c = t.scale == 0.0f ? 1.0f : std::max(std::fabs(t.scale) * LOG2E, 1e-37f);
    a.sign = t.scale > 0.0f ? 1.0f : t.scale < 0.0f ? -1.0f : 0.0f;
    a.acc = (float *)t.work; // (rows of hs values, hs a multiple of 16: 16-byte aligned)
    const size_t parts = (size_t)p.cap * a.group * t.max_n;
    a.ml = a.acc + parts * c.hs;
    a.plan = (int2 *)(a.ml + 2 * parts);
    size_t lds = 0;
    auto *pick = p.hsp == 64 ? tree_kernel_64 : p.hsp == 128 ? tree_kernel_128 : p.hsp == 192 ? tree_kernel_192 : tree_kernel_256;
    TreeKernel kern = pick(c.type, q.type, p.tiles, p.many, &lds);
    if (!kern) return hipErrorInvalidValue;
    hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3(p.many ? 64 * p.many : 256), lds, st, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || !p.cap) return e;
    // a wave a row up to 16 slices a head, the block's four above (7 rows of 64 slices over 32k positions: 18.9 us a call
    // with one, 16.7 with four; 448 rows of up to 4, eight sequences: 124 and 135)
    const bool wide = p.cap > 16 * c.n_seq * c.n_kv;
    const dim3 grid(wide ? t.max_n * a.group : (t.max_n * a.group + 3) / 4, c.n_kv, c.n_seq);
    auto *join = q.type == LLM_F32 ? wide ? k_tree_join<LLM_F32, 4> : k_tree_join<LLM_F32, 1>
                                   : wide ? k_tree_join<LLM_BF16, 4> : k_tree_join<LLM_BF16, 1>;
    hipLaunchKernelGGL(join, grid, dim3(256), 0, st, a);
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
    if (!std::isfinite(scale * LOG2E)) {
        fprintf(stderr, "%s: scale %g\n", who, scale);
        return -1;
    }
    const int count[] = {c->n_seq, max_n, n_heads};
    const int64_t stride[] = {out->seq, out->tok, out->head};
    if (!op_check_apart(who, "out", 3, count, stride)) return -1;
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
