// K and V rows written into a cache of 8 bits (or fp32 / bf16) and read back: llm_kv_write, llm_kv_read.
#include <string.h>

#include "device.h"
#include "operators.h"
#include "rows.h"

namespace {

// One side (K or V) of the cache and the rows that go with it; strides in bytes, of the scales in floats.
struct KvSide {
    uint8_t *c, *r;
    float *s;
};
struct KvArgs {
    KvSide side[2];
    int64_t seq, head, pos, s_seq, s_head, s_pos; // cache
    int64_t r_seq[2], r_tok[2], r_head[2];        // rows, of K and V
    const int *at, *n;
    int at0, by_pos; // at NULL: every sequence's position; the rows lie at their positions, not from 0
    int n_kv, hs, ctx, max_n, zero_rest;
    uint32_t rows; // n_seq * max_n * n_kv
};

// A row: scale = largest magnitude / 127 (448), codes = value / scale.  Bytes in, bytes out: a DPP row of 16 lanes takes one
// row of a head, lane l its values 4 l .. 4 l + 3 and every 64th from there; the largest magnitude is four DPP steps, the scale
// and the codes follow from registers, so the row is read once.  Few rows are bound by a launch's latency (one token 2.7 us), many
// by vector instructions, a wave's 402 with the exact quotients: 2048 fp32 tokens of 4 heads of 128 into int8 6.4 us (1.7 TB/s),
// and they are issued in 6.4k of the 10k cycles that a SIMD's waves live.
template <int CT, int RT>
__global__ void __launch_bounds__(256) k_kv_write(KvArgs a) {
    constexpr int RS = RT == LLM_F32 ? 4 : 2;
    const uint32_t item = blockIdx.x * 16u + threadIdx.x / 16;
    const int side = blockIdx.y, l = threadIdx.x & 15;
    if (item >= a.rows) return; // (whole DPP rows leave)
    const uint32_t h = item % a.n_kv, bt = item / a.n_kv, t = bt % a.max_n, b = bt / a.max_n;
    const int64_t p = (int64_t)(a.at ? a.at[b] : a.at0) + t;
    if ((a.n && (int)t >= a.n[b]) || p < 0 || p >= a.ctx) return;
    const uint8_t *src = a.side[side].r + b * a.r_seq[side] + (a.by_pos ? p : t) * a.r_tok[side] + h * a.r_head[side];
    uint8_t *dst = a.side[side].c + b * a.seq + h * a.head + p * a.pos;
    float4 x[4];
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int e = 4 * l + 64 * i;
        x[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (e < a.hs) x[i] = row4<RT>(src + (size_t)e * RS);
    }
    if constexpr (CT == LLM_F32 || CT == LLM_BF16) {
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (4 * l + 64 * i < a.hs) put4<CT>(dst + (size_t)(4 * l + 64 * i) * (CT == LLM_F32 ? 4 : 2), x[i]);
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
        for (float v : {x[i].x, x[i].y, x[i].z, x[i].w}) m = max(m, __float_as_uint(v) & 0x7fffffffu);
    m = umax16(m);
    const float amax = __uint_as_float(m), top = CT == LLM_I8 ? 127.0f : 448.0f;
    const bool bad = m >= 0x7f800000u;
    float s = amax / top;
    // rows of tiny values: scaled by 2^80 for the division, whose remainders would underflow
    const float up = amax < 0x1p-60f ? 0x1p80f : 1.0f, su = s * up;
    const bool zero = bad || s == 0.0f;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if (4 * l + 64 * i >= a.hs) continue;
        float q[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
        for (float &v : q) v = zero ? 0.0f : fminf(fmaxf(div_to_odd(v * up, su), -top), top);
        uint32_t w;
        if constexpr (CT == LLM_I8) {
            w = 0;
#pragma unroll
            for (int k = 0; k < 4; k++) w |= ((uint32_t)(int)rintf(q[k]) & 0xffu) << (8 * k);
        } else {
            int c = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
            w = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], c, true);
        }
        *(uint32_t *)(dst + 4 * l + 64 * i) = w;
    }
    if (l == 0) a.side[side].s[b * a.s_seq + h * a.s_head + p * a.s_pos] = bad ? __uint_as_float(0x7fc00000u) : s;
}

// The same the other way, code * scale: 7069 int8 tokens of 4 heads of 128 into fp32 8.7 us (4.2 TB/s), 24 sequences of up to
// 517 e4m3 tokens, the rows that are not read set to zero, 12.3.
template <int CT, int RT>
__global__ void __launch_bounds__(256) k_kv_read(KvArgs a) {
    constexpr int RS = RT == LLM_F32 ? 4 : 2, CS = CT == LLM_F32 ? 4 : CT == LLM_BF16 ? 2 : 1;
    const uint32_t item = blockIdx.x * 16u + threadIdx.x / 16;
    const int side = blockIdx.y, l = threadIdx.x & 15;
    if (item >= a.rows) return;
    const uint32_t h = item % a.n_kv, bt = item / a.n_kv, t = bt % a.max_n, b = bt / a.max_n;
    const int64_t p = (int64_t)(a.at ? a.at[b] : a.at0) + t;
    uint8_t *dst = a.side[side].r + b * a.r_seq[side] + t * a.r_tok[side] + h * a.r_head[side];
    if ((a.n && (int)t >= a.n[b]) || p < 0 || p >= a.ctx) {
        if (a.zero_rest)
            for (int e = 4 * l; e < a.hs; e += 64) put4<RT>(dst + (size_t)e * RS, make_float4(0.0f, 0.0f, 0.0f, 0.0f));
        return;
    }
    const uint8_t *src = a.side[side].c + b * a.seq + h * a.head + p * a.pos;
    float s = 1.0f;
    if constexpr (CS == 1) s = a.side[side].s[b * a.s_seq + h * a.s_head + p * a.s_pos];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int e = 4 * l + 64 * i;
        if (e >= a.hs) continue;
        float4 v;
        if constexpr (CS > 1) {
            if constexpr (CS == 4) {
                const f32x4u f = *(const f32x4u *)(src + (size_t)e * 4);
                v = make_float4(f[0], f[1], f[2], f[3]);
            } else {
                const u32x2u u = *(const u32x2u *)(src + (size_t)e * 2);
                v = make_float4(__uint_as_float(u[0] << 16), __uint_as_float(u[0] & 0xffff0000u), __uint_as_float(u[1] << 16),
                                __uint_as_float(u[1] & 0xffff0000u));
            }
        } else {
            const uint32_t w = *(const uint32_t *)(src + e);
            if constexpr (CT == LLM_I8) {
                v = make_float4((float)(int8_t)w, (float)(int8_t)(w >> 8), (float)(int8_t)(w >> 16), (float)(int8_t)(w >> 24));
            } else {
                const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
                v = make_float4(lo[0], lo[1], hi[0], hi[1]);
            }
            v = make_float4(v.x * s, v.y * s, v.z * s, v.w * s);
        }
        put4<RT>(dst + (size_t)e * RS, v);
    }
}

struct KeepArgs {
    uint8_t *side[2];
    float *scale[2];
    int64_t layer, head, pos, s_layer, s_head, s_pos; // strides: bytes, of the scales floats
    int words, pos0, n;                               // 4-byte words of a row
    uint8_t path[64];
};
// Rows pos0 + path[j] to pos0 + j, in the order of j (path rising: a row is read before it is written over): a thread has
// the same word of every row.
__global__ void __launch_bounds__(64) k_kv_keep(KeepArgs a) {
    const int head = blockIdx.x, layer = blockIdx.y, side = blockIdx.z;
    uint8_t *rows = a.side[side] + layer * a.layer + head * a.head + (int64_t)a.pos0 * a.pos;
    float *s = a.scale[side] ? a.scale[side] + layer * a.s_layer + head * a.s_head + (int64_t)a.pos0 * a.s_pos : nullptr;
    for (int j = 0; j < a.n; j++) {
        const int from = a.path[j];
        if (from == j) continue;
        for (int w = threadIdx.x; w < a.words; w += 64)
            ((uint32_t *)(rows + j * a.pos))[w] = ((const uint32_t *)(rows + from * a.pos))[w];
        if (s && threadIdx.x == 0) s[j * a.s_pos] = s[from * a.s_pos];
    }
}

int kv_rows(const char *who, bool write, const llm_kv *c, const llm_rows *k, const llm_rows *v, const int *pos,
            const int *n, int max_n, int zero_rest, void *stream) {
    if (!c || !k || !v || max_n < 0) {
        fprintf(stderr, "%s: bad arguments\n", who);
        return -1;
    }
    if (!op_check_cache(c, nullptr, who)) return -1;
    if (write) {
        const int count[] = {c->n_seq, c->n_kv, c->n_seq, c->n_kv};
        const int64_t stride[] = {c->seq, c->head, c->s_seq, c->s_head};
        if (!op_check_apart(who, "the cache", op_scaled(c->type) ? 4 : 2, count, stride)) return -1;
    } else {
        for (const llm_rows *r : {k, v}) {
            const int count[] = {c->n_seq, max_n, c->n_kv};
            const int64_t stride[] = {r->seq, r->tok, r->head};
            if (!op_check_apart(who, "the rows", 3, count, stride)) return -1;
        }
    }
    if ((__int128)c->n_seq * max_n * c->n_kv >= 1 << 28) { // (16 threads a row, and a grid has 2^32)
        fprintf(stderr, "%s: %d sequences of %d rows\n", who, c->n_seq, max_n);
        return -1;
    }
    OpDevice dev(who);
    if (!op_check_cache(c, &dev, who)) return -1;
    if (!max_n || !c->n_seq) return 0;
    if (!op_check_rows(k, "k", &dev, who) || !op_check_rows(v, "v", &dev, who) || !dev.holds(pos, "pos") ||
        (n && !dev.holds(n, "n")))
        return -1;
    if (write && c->k == c->v) {
        fprintf(stderr, "%s: k and v are the same memory\n", who);
        return -1;
    }
    if (k->type != v->type) {
        fprintf(stderr, "%s: k and v rows of different types\n", who);
        return -1;
    }
    if (!dev.select()) return -1;
    KvCall q;
    memset(&q, 0, sizeof q);
    q.pos = pos;
    q.n = n;
    q.max_n = max_n;
    q.zero_rest = zero_rest;
    HIP_OR_FAIL(who, launch_kv(write, *c, *k, *v, q, (hipStream_t)stream));
    return 0;
}

} // namespace

bool op_check_cache(const llm_kv *c, OpDevice *dev, const char *who) {
    const int cs = op_type_bytes(c->type);
    if (!cs || c->n_seq < 0 || c->n_kv < 1 || c->ctx < 1 || c->hs < 16 || c->hs > 256 || c->hs % 16) {
        fprintf(stderr, "%s: a cache of type %d, %d sequences, %d heads of %d values, %d positions is not taken\n", who,
                c->type, c->n_seq, c->n_kv, c->hs, c->ctx);
        return false;
    }
    if (!c->n_seq) return true; // (nothing to walk)
    auto odd = [&](int64_t stride) { return stride < 0 || stride * cs % 4; };
    if (odd(c->seq) || odd(c->head) || odd(c->pos) || (((uintptr_t)c->k | (uintptr_t)c->v) & 3) || c->pos < c->hs ||
        c->pos > ((int64_t)16 << 20) / cs) {
        fprintf(stderr, "%s: the cache's rows have to start at multiples of 4 bytes, a position at least a row's values and "
                "at most 16 MiB from the next\n", who);
        return false;
    }
    if (op_scaled(c->type)) {
        if (c->s_seq < 0 || c->s_head < 0 || c->s_pos < 1 || c->s_pos > ((int64_t)4 << 20)) {
            fprintf(stderr, "%s: strides of the scales (%lld, %lld, %lld)\n", who, (long long)c->s_seq,
                    (long long)c->s_head, (long long)c->s_pos);
            return false;
        }
        if (((uintptr_t)c->k_scale | (uintptr_t)c->v_scale) & 3) {
            fprintf(stderr, "%s: the scales are not aligned\n", who);
            return false;
        }
    }
    if (!dev) return true;
    if (!dev->holds(c->k, "the K cache") || !dev->holds(c->v, "the V cache")) return false;
    if (!op_scaled(c->type)) return true;
    return dev->holds(c->k_scale, "the K scales") && dev->holds(c->v_scale, "the V scales");
}

bool op_check_rows(const llm_rows *r, const char *what, OpDevice *dev, const char *who) {
    if (r->type != LLM_F32 && r->type != LLM_BF16) {
        fprintf(stderr, "%s: rows of type %d in %s (fp32 or bf16)\n", who, r->type, what);
        return false;
    }
    if (r->seq < 0 || r->tok < 0 || r->head < 0 || r->seq % 4 || r->tok % 4 || r->head % 4 ||
        ((uintptr_t)r->p & (4 * op_type_bytes(r->type) - 1))) {
        fprintf(stderr, "%s: the rows of %s have to start at multiples of 4 values\n", who, what);
        return false;
    }
    return dev->holds(r->p, what);
}

hipError_t launch_kv(bool write, const llm_kv &c, const llm_rows &k, const llm_rows &v, const KvCall &q, hipStream_t st) {
    const int cs = op_type_bytes(c.type), rs = op_type_bytes(k.type);
    KvArgs a;
    memset(&a, 0, sizeof a);
    a.side[0] = {(uint8_t *)c.k, (uint8_t *)k.p, c.k_scale};
    a.side[1] = {(uint8_t *)c.v, (uint8_t *)v.p, c.v_scale};
    a.seq = c.seq * cs, a.head = c.head * cs, a.pos = c.pos * cs;
    a.s_seq = c.s_seq, a.s_head = c.s_head, a.s_pos = c.s_pos;
    for (int i = 0; i < 2; i++) {
        const llm_rows &r = i ? v : k;
        a.r_seq[i] = r.seq * rs, a.r_tok[i] = r.tok * rs, a.r_head[i] = r.head * rs;
    }
    a.at = q.pos, a.at0 = q.pos0, a.by_pos = q.by_pos;
    a.n = q.n;
    a.n_kv = c.n_kv, a.hs = c.hs, a.ctx = c.ctx, a.max_n = q.max_n, a.zero_rest = q.zero_rest;
    a.rows = (uint32_t)c.n_seq * q.max_n * c.n_kv;
    void (*kern)(KvArgs) = nullptr;
#define KV_PICK(C, R)                                                                 \
    if (c.type == C && k.type == R) kern = write ? k_kv_write<C, R> : k_kv_read<C, R>;
    KV_PICK(LLM_F32, LLM_F32) KV_PICK(LLM_F32, LLM_BF16) KV_PICK(LLM_BF16, LLM_F32) KV_PICK(LLM_BF16, LLM_BF16)
    KV_PICK(LLM_I8, LLM_F32) KV_PICK(LLM_I8, LLM_BF16) KV_PICK(LLM_E4M3, LLM_F32) KV_PICK(LLM_E4M3, LLM_BF16)
#undef KV_PICK
    hipLaunchKernelGGL(kern, dim3((a.rows + 15) / 16, 2), dim3(256), 0, st, a);
    return hipGetLastError();
}

hipError_t launch_kv_keep(const llm_kv &c, int pos0, const uint8_t *path, int n, hipStream_t st) {
    const int cs = op_type_bytes(c.type);
    KeepArgs a;
    memset(&a, 0, sizeof a);
    a.side[0] = (uint8_t *)c.k, a.side[1] = (uint8_t *)c.v;
    a.scale[0] = c.k_scale, a.scale[1] = c.v_scale;
    a.layer = c.seq * cs, a.head = c.head * cs, a.pos = c.pos * cs;
    a.s_layer = c.s_seq, a.s_head = c.s_head, a.s_pos = c.s_pos;
    a.words = c.hs * cs / 4;
    a.pos0 = pos0;
    a.n = n;
    memcpy(a.path, path, n);
    hipLaunchKernelGGL(k_kv_keep, dim3(c.n_kv, c.n_seq, 2), dim3(64), 0, st, a);
    return hipGetLastError();
}

extern "C" int llm_kv_write(const llm_kv *c, const llm_rows *k, const llm_rows *v, const int *pos, const int *n, int max_n,
                            void *stream) {
    return kv_rows("llm_kv_write", true, c, k, v, pos, n, max_n, 0, stream);
}

extern "C" int llm_kv_read(const llm_kv *c, const llm_rows *k, const llm_rows *v, const int *pos, const int *n, int max_n,
                           int zero_rest, void *stream) {
    return kv_rows("llm_kv_read", false, c, k, v, pos, n, max_n, zero_rest, stream);
}
