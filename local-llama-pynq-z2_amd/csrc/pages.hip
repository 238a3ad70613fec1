// A cache in pages: rows written and read (llm_page_write, llm_page_read), pages shared, taken, freed and moved
// (llm_page_fork, llm_page_reserve, llm_page_compact).  The attention over pages is in page_attention.hip.
#include <string.h>

#include <algorithm>
#include <utility>

#include "device.h"
#include "operators.h"
#include "rows.h"

namespace {

// ---- rows -----------------------------------------------------------------------------------------------------------

struct RowArgs {
    uint8_t *c[2], *r[2];
    float *s[2];
    int64_t id, head, s_id, s_head;            // pool strides: codes, floats
    int64_t r_seq[2], r_tok[2], r_head[2];     // bytes
    const int *table, *refs, *pos, *n, *path;
    int per, n_pages, n_kv, hs, page, max_n, blocks, zero_rest;
    uint32_t units; // workgroups of a side; a row of the grid has GRID_ROW of them at most (2^32 threads would not fit)
};
constexpr uint32_t GRID_ROW = 1 << 22;
// The workgroup's, 0 behind the last (`over`: no branch, so that the arguments' loads stay together).
__device__ __forceinline__ uint32_t unit_id(const RowArgs &a, bool &over) {
    const uint32_t id = blockIdx.z * GRID_ROW + blockIdx.x;
    over = id >= a.units;
    return over ? 0 : id;
}

// Blocks that max_n tokens from any position on can reach.
__host__ __device__ __forceinline__ int blocks_of(int max_n) { return (max_n + PAGE_BLOCK - 2) / PAGE_BLOCK + 1; }

// Where a workgroup works: a block of 64 positions of a sequence's kv head, the offsets lo .. hi - 1 of its tokens in it.
struct Unit {
    int b, h, page, blk, lo, hi;
    int64_t first; // the token at offset 0 (below 0 if it is not of this call)
};
__device__ __forceinline__ bool find_unit(const RowArgs &a, Unit &u) {
    bool over;
    const uint32_t id = unit_id(a, over);
    u.h = id % a.n_kv;
    const uint32_t x = id / a.n_kv;
    u.b = x / a.blocks;
    const int nn = a.n ? min(max(a.n[u.b], 0), a.max_n) : a.max_n;
    const int64_t p0 = a.pos[u.b], end = min(p0 + nn, (int64_t)a.per * a.page);
    const int64_t at = (max(p0, (int64_t)0) / PAGE_BLOCK + x % a.blocks) * PAGE_BLOCK; // the block's first position
    const int64_t lo = max(p0, at), hi = min(end, at + PAGE_BLOCK);
    u.page = -1;
    if (over || lo >= hi) return false;
    u.lo = (int)(lo - at), u.hi = (int)(hi - at);
    u.first = at - p0;
    u.page = a.table[(int64_t)u.b * a.per + at / a.page];
    u.blk = (int)(at % a.page / PAGE_BLOCK);
    if ((uint32_t)u.page >= (uint32_t)a.n_pages) u.page = -1;
    return true;
}

template <int CT>
__device__ __forceinline__ uint8_t code_of(float q) { // |q| within the type's range, or NaN for e4m3
    if constexpr (CT == LLM_I8) return (uint8_t)(int)rintf(q);
    else return (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(q, q, 0, false);
}
template <int CT>
__device__ __forceinline__ uint32_t code4(const float (&q)[4]) {
    if constexpr (CT == LLM_E4M3)
        return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false), true);
    uint32_t w = 0;
#pragma unroll
    for (int k = 0; k < 4; k++) w |= (uint32_t)code_of<CT>(q[k]) << (8 * k);
    return w;
}
template <int CT>
__device__ __forceinline__ void value4(uint32_t w, float (&v)[4]) {
    if constexpr (CT == LLM_I8) {
#pragma unroll
        for (int k = 0; k < 4; k++) v[k] = (float)(int8_t)(w >> (8 * k));
    } else {
        const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
        v[0] = lo[0], v[1] = lo[1], v[2] = hi[0], v[3] = hi[1];
    }
}
template <int CT>
__device__ __forceinline__ float value_of(uint8_t c) {
    if constexpr (CT == LLM_I8) return (float)(int8_t)c;
    else return __builtin_amdgcn_cvt_f32_fp8((int)c, 0);
}

// Codes of values x / s (both scaled up as div_to_odd needs it; inv a rounded 1 / s): a product with the reciprocal is off by
// 2^-22 of itself at most (1 / s and the product are rounded, 2^-24 each), so it decides unless it falls that close to a border
// between two codes; then the exact quotient does.  Borders: int8 the halves, 127 2^-22 = 3e-5; e4m3 the middles between two
// neighbours, the 20 bits below its three at 0x80000, and anywhere below its normal values, 2^-6.
template <int CT>
__device__ __forceinline__ uint32_t codes_of(float4 x, float s, float inv, float sign) {
    constexpr float top = CT == LLM_I8 ? 127.0f : 448.0f;
    float v[4] = {x.x * sign, x.y * sign, x.z * sign, x.w * sign}, q[4];
    bool near = false;
#pragma unroll
    for (int k = 0; k < 4; k++) {
        q[k] = v[k] * inv;
        if constexpr (CT == LLM_I8) {
            near |= fabsf(fabsf(q[k] - rintf(q[k])) - 0.5f) < 1e-4f;
        } else {
            near |= ((__float_as_uint(q[k]) + 16u - 0x80000u) & 0xfffffu) < 32u;
            near |= fabsf(q[k]) < 0x1p-6f && q[k] != 0.0f;
        }
    }
    if (__any(near))
#pragma unroll
        for (int k = 0; k < 4; k++) q[k] = div_to_odd(v[k], s);
#pragma unroll
    for (int k = 0; k < 4; k++) q[k] = fminf(fmaxf(q[k], -top), top);
    return code4<CT>(q);
}

constexpr int WRITE_T = 512; // threads of a block's workgroup: few rows a thread, whose latencies count
constexpr int TURN = 68; // bytes from row to row of a turned block in LDS: rows of a wave's stores fall into 16 banks

// The rows of a block: their largest magnitude decides the scale, then their codes; a workgroup a block and side.  The rows are
// read once, all loads at once, and wait in registers; V's codes are turned in LDS.  2048 fp32 rows of 4 heads of 128, 8.4 MB:
// 8.6 us (16.3 with exact quotients for all and V stored byte by byte), bound by its phases one after another with a workgroup a
// CU: of a wave's 15k cycles it waits for 8.9k, vector instructions are issued in 28% of a SIMD's; one row: 4.2 us, dependent loads.
template <int CT, int RT>
__global__ void __launch_bounds__(WRITE_T) k_page_write(RowArgs a) {
    constexpr int RS = RT == LLM_F32 ? 4 : 2, ITEMS = 64 * 256 / 4 / WRITE_T; // of four values a thread
    __shared__ uint32_t sm_max[WRITE_T / 64];
    __shared__ __align__(4) uint8_t sm_v[256 * TURN];
    Unit u;
    if (!find_unit(a, u) || u.page < 0 || (a.refs && a.refs[u.page] != 1)) return;
    const int side = blockIdx.y, per_row = a.hs / 4, items = (u.hi - u.lo) * per_row;
    uint8_t *const dst = a.c[side] + u.page * a.id + u.h * a.head + u.blk * (PAGE_BLOCK * a.hs);
    float *const scale = a.s[side] + u.page * a.s_id + u.h * a.s_head + u.blk;
    const uint8_t *const src = a.r[side] + u.b * a.r_seq[side] + u.h * a.r_head[side];
    const float old = u.lo ? *scale : 0.0f;
    float4 x[ITEMS];
#pragma unroll
    for (int k = 0; k < ITEMS; k++) {
        const int i = threadIdx.x + WRITE_T * k;
        x[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (i < items) {
            int64_t t = u.first + u.lo + i / per_row;
            if (a.path) t = a.path[(int64_t)u.b * a.max_n + t];
            if ((uint64_t)t < (uint64_t)a.max_n) x[k] = row4<RT>(src + t * a.r_tok[side] + (size_t)(i % per_row) * 4 * RS);
        }
    }
    uint32_t m = 0;
#pragma unroll
    for (int k = 0; k < ITEMS; k++)
        for (float v : {x[k].x, x[k].y, x[k].z, x[k].w}) m = max(m, __float_as_uint(v) & 0x7fffffffu);
    m = umax16(m);
    for (int off = 16; off < 64; off <<= 1) m = max(m, (uint32_t)__shfl_xor((int)m, off));
    if ((threadIdx.x & 63) == 0) sm_max[threadIdx.x / 64] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < WRITE_T / 64; i++) m = max(m, sm_max[i]);
    const float top = CT == LLM_I8 ? 127.0f : 448.0f, want = __uint_as_float(m) / top;
    const bool bad = m >= 0x7f800000u || !(fabsf(old) < INFINITY);
    float s = fabsf(old), back = 1.0f; // the new scale's magnitude, and what takes the codes before lo to it
    if (s == 0.0f) s = want, back = 0.0f;
    else if (!bad)
        while (s < want) s *= 2.0f, back *= 0.5f;
    if (u.lo && !bad && back != 1.0f)
        for (int i = threadIdx.x; i < u.lo * a.hs; i += WRITE_T) {
            uint8_t *c = side ? dst + i / u.lo * PAGE_BLOCK + i % u.lo : dst + i;
            *c = back == 0.0f ? 0 : code_of<CT>(value_of<CT>(*c) * back);
        }
    const bool zero = bad || s == 0.0f;
    // (rows of tiny values: scaled by 2^80, their remainders would underflow; no code but 0 of a block without a scale)
    const float up = s < 0x1p-60f ? 0x1p80f : 1.0f, su = zero ? 1.0f : s * up, sign = old < 0.0f ? -up : up, inv = 1.0f / su;
#pragma unroll
    for (int k = 0; k < ITEMS; k++) {
        if (WRITE_T * k >= items) break;
        const int i = threadIdx.x + WRITE_T * k;
        if (i >= items) continue;
        const int o = u.lo + i / per_row, d = i % per_row * 4;
        uint32_t w = 0;
        if (!zero) w = codes_of<CT>(x[k], su, inv, sign); // (0 * infinity)
        if (side == 0) *(uint32_t *)(dst + o * a.hs + d) = w;
        else
#pragma unroll
            for (int e = 0; e < 4; e++) sm_v[(d + e) * TURN + o] = (uint8_t)(w >> (8 * e));
    }
    if (threadIdx.x == 0) *scale = bad ? __uint_as_float(0x7fc00000u) : old < 0.0f ? -s : s;
    if (side == 0) return;
    __syncthreads();
    // 16 positions of a dimension a thread: whole, or those of the call
    for (int i = threadIdx.x; i < a.hs * 4; i += WRITE_T) {
        const int d = i / 4, o = i % 4 * 16, lo = max(u.lo, o), hi = min(u.hi, o + 16);
        const uint8_t *from = sm_v + d * TURN;
        uint8_t *to = dst + d * PAGE_BLOCK;
        if (hi - lo == 16) {
            const uint32_t *w = (const uint32_t *)(from + o);
            *(uint4 *)(to + o) = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
            for (int k = lo; k < hi; k++) to[k] = from[k];
        }
    }
}

// The same the other way: a workgroup a block of the cache and side, its rows out of the block's codes (V's by LDS, whose rows of
// hs + 4 bytes spread over the banks).  7069 rows of 4 heads of 128, 29 MB of fp32 out of 7.2: 10.0
// us, 3.6 TB/s; of a wave's 14.5k cycles it waits for 9.2k, vector instructions are issued in a quarter of a SIMD's.
template <int CT, int RT>
__global__ void __launch_bounds__(256) k_page_read(RowArgs a) {
    constexpr int RS = RT == LLM_F32 ? 4 : 2;
    __shared__ __align__(4) uint8_t sm_v[PAGE_BLOCK * 260]; // V's codes by position
    bool over;
    const uint32_t id = unit_id(a, over);
    const int side = blockIdx.y, h = id % a.n_kv, x = id / a.n_kv, b = x / a.blocks;
    const int64_t p0 = a.pos[b], at = ((p0 >> 6) + x % a.blocks) * PAGE_BLOCK; // (rounded down, below 0 too)
    const int lo = (int)max((int64_t)0, p0 - at), hi = (int)min((int64_t)PAGE_BLOCK, p0 + a.max_n - at); // offsets that rows are for
    if (over || lo >= hi) return;
    const int nn = a.n ? min(max(a.n[b], 0), a.max_n) : a.max_n;
    int page = -1;
    if (at >= 0 && at < (int64_t)a.per * a.page) page = a.table[(int64_t)b * a.per + at / a.page];
    const int have = (uint32_t)page < (uint32_t)a.n_pages ? (int)min((int64_t)hi, p0 + nn - at) : lo; // offsets up to which there are
    uint8_t *const dst = a.r[side] + b * a.r_seq[side] + (at - p0) * a.r_tok[side] + h * a.r_head[side];
    const int per_row = a.hs / 4;
    if (a.zero_rest)
        for (int i = threadIdx.x; i < (hi - max(lo, have)) * per_row; i += 256)
            put4<RT>(dst + (max(lo, have) + i / per_row) * a.r_tok[side] + (size_t)(i % per_row) * 4 * RS, make_float4(0.0f, 0.0f, 0.0f, 0.0f));
    if (lo >= have) return;
    const int blk = (int)(at & (a.page - 1)) / PAGE_BLOCK;
    const uint8_t *const src = a.c[side] + page * a.id + h * a.head + blk * (PAGE_BLOCK * a.hs);
    const float s = a.s[side][page * a.s_id + h * a.s_head + blk];
    if (side) {
        uint4 w[4]; // 16 positions of a dimension each
#pragma unroll
        for (int k = 0; k < 4; k++)
            if ((int)threadIdx.x + 256 * k < a.hs * 4) w[k] = *(const uint4 *)(src + (threadIdx.x + 256 * k) * 16);
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int i = threadIdx.x + 256 * k, d = i / 4, o = i % 4 * 16;
            if (i >= a.hs * 4) break;
            const uint32_t q[4] = {w[k].x, w[k].y, w[k].z, w[k].w};
#pragma unroll
            for (int e = 0; e < 16; e++) sm_v[(o + e) * (a.hs + 4) + d] = (uint8_t)(q[e / 4] >> (8 * (e % 4)));
        }
        __syncthreads();
    }
#pragma unroll 4
    for (int i = threadIdx.x; i < (have - lo) * per_row; i += 256) {
        const int o = lo + i / per_row, d = i % per_row * 4;
        const uint32_t w = side ? *(const uint32_t *)(sm_v + o * (a.hs + 4) + d) : *(const uint32_t *)(src + o * a.hs + d);
        float v[4];
        value4<CT>(w, v);
        put4<RT>(dst + o * a.r_tok[side] + (size_t)d * RS, make_float4(v[0] * s, v[1] * s, v[2] * s, v[3] * s));
    }
}

int page_rows(const char *who, bool write, const llm_pages *c, const llm_rows *k, const llm_rows *v, int n_seq, const int *table,
              int per, const int *refs, const int *pos, const int *n, const int *path, int max_n, int zero_rest, void *stream) {
    if (!c || !k || !v || max_n < 0 || max_n > 1 << 30) { // (more than a table's positions)
        fprintf(stderr, "%s: bad arguments (%d rows a sequence)\n", who, max_n);
        return -1;
    }
    if (!op_check_pages(c, nullptr, who) || !op_check_table(table, n_seq, per, nullptr, who)) return -1;
    if (!write)
        for (const llm_rows *r : {k, v}) {
            const int count[] = {n_seq, max_n, c->n_kv};
            const int64_t stride[] = {r->seq, r->tok, r->head};
            if (!op_check_apart(who, "the rows", 3, count, stride)) return -1;
        }
    const int blocks = blocks_of(max_n);
    if ((int64_t)n_seq * blocks * c->n_kv > 0x7fffffffll) {
        fprintf(stderr, "%s: %d sequences of %d rows\n", who, n_seq, max_n);
        return -1;
    }
    OpDevice dev(who);
    if (!op_check_pages(c, &dev, who)) return -1;
    if (!max_n || !n_seq) return 0;
    if (!op_check_rows(k, "k", &dev, who) || !op_check_rows(v, "v", &dev, who) ||
        !op_check_table(table, n_seq, per, &dev, who) || !dev.holds(pos, "pos") || (refs && !dev.holds(refs, "refs")) ||
        (n && !dev.holds(n, "n")) || (path && !dev.holds(path, "path")))
        return -1;
    if (k->type != v->type) {
        fprintf(stderr, "%s: k and v rows of different types\n", who);
        return -1;
    }
    if (!dev.select()) return -1;
    const int rs = op_type_bytes(k->type);
    RowArgs a;
    memset(&a, 0, sizeof a);
    for (int i = 0; i < 2; i++) {
        const llm_rows *r = i ? v : k;
        a.c[i] = (uint8_t *)(i ? c->v : c->k), a.s[i] = i ? c->v_scale : c->k_scale;
        a.r[i] = (uint8_t *)r->p, a.r_seq[i] = r->seq * rs, a.r_tok[i] = r->tok * rs, a.r_head[i] = r->head * rs;
    }
    a.id = c->id, a.head = c->head, a.s_id = c->s_id, a.s_head = c->s_head;
    a.table = table, a.refs = refs, a.pos = pos, a.n = n, a.path = path;
    a.per = per, a.n_pages = c->n_pages, a.n_kv = c->n_kv, a.hs = c->hs, a.page = c->page, a.max_n = max_n;
    a.blocks = blocks, a.zero_rest = zero_rest;
    a.units = (uint32_t)(n_seq * blocks * c->n_kv);
    const dim3 grid(std::min(a.units, GRID_ROW), 2, (a.units + GRID_ROW - 1) / GRID_ROW);
    void (*kern)(RowArgs) = nullptr;
#define PAGE_PICK(C, R)                                                                   \
    if (c->type == C && k->type == R) kern = write ? k_page_write<C, R> : k_page_read<C, R>;
    PAGE_PICK(LLM_I8, LLM_F32) PAGE_PICK(LLM_I8, LLM_BF16) PAGE_PICK(LLM_E4M3, LLM_F32) PAGE_PICK(LLM_E4M3, LLM_BF16)
#undef PAGE_PICK
    hipLaunchKernelGGL(kern, grid, dim3(write ? WRITE_T : 256), 0, (hipStream_t)stream, a);
    HIP_OR_FAIL(who, hipGetLastError());
    return 0;
}

// ---- tables ---------------------------------------------------------------------------------------------------------

struct ForkArgs {
    int n_pages, page, n_seq, per, count;
    int *table, *lens, *refs;
    const int *to, *from;
    int *rows, *len; // work: the new rows of the table, their lengths (-1: the entry does nothing)
};

// The counts follow, and the new rows are laid by: tables are only read here, so that every entry sees them as they were.  The two
// launches are latency, 2 to 5 us each.
__global__ void __launch_bounds__(256) k_fork_count(ForkArgs a) {
    __shared__ int again;
    const int i = blockIdx.x, to = a.to[i], from = a.from[i];
    if (threadIdx.x == 0) again = 0;
    __syncthreads();
    bool later = false;
    for (int k = i + 1 + threadIdx.x; k < a.count; k += 256) later |= a.to[k] == to;
    if (later) again = 1;
    __syncthreads();
    const bool live = !again && (uint32_t)to < (uint32_t)a.n_seq, there = (uint32_t)from < (uint32_t)a.n_seq;
    const int len = there ? (int)min((int64_t)max(a.lens[from], 0), (int64_t)a.per * a.page) : 0;
    if (threadIdx.x == 0) a.len[i] = live ? len : -1;
    if (!live) return;
    const int need = (len + a.page - 1) / a.page;
    for (int j = threadIdx.x; j < a.per; j += 256) {
        const int old = a.table[(int64_t)to * a.per + j];
        int next = j < need ? a.table[(int64_t)from * a.per + j] : -1;
        if ((uint32_t)next >= (uint32_t)a.n_pages) next = -1;
        if (next >= 0) atomicAdd(&a.refs[next], 1);
        if ((uint32_t)old < (uint32_t)a.n_pages) atomicSub(&a.refs[old], 1);
        a.rows[(int64_t)i * a.per + j] = next;
    }
}
__global__ void __launch_bounds__(256) k_fork_write(ForkArgs a) {
    const int i = blockIdx.x, len = a.len[i];
    if (len < 0) return;
    const int to = a.to[i];
    for (int j = threadIdx.x; j < a.per; j += 256) a.table[(int64_t)to * a.per + j] = a.rows[(int64_t)i * a.per + j];
    if (threadIdx.x == 0) a.lens[to] = len;
}

constexpr int BOOK_T = 1024; // threads of the workgroup that keeps the books

// Inclusive sum over the block's threads of small counts; `total` gets the whole.
__device__ __forceinline__ int block_scan(int v, int *sm, int &total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x / 64;
    int x = v;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const int y = __shfl_up(x, off);
        x += lane >= off ? y : 0;
    }
    if (lane == 63) sm[wave] = x;
    __syncthreads();
    int before = 0;
    total = 0;
    for (int w = 0; w < BOOK_T / 64; w++) {
        before += w < wave ? sm[w] : 0;
        total += sm[w];
    }
    __syncthreads();
    return before + x;
}

struct ReserveArgs {
    int n_pages, page, n_seq, per, max_n, most; // most: pages that a sequence's tokens can reach
    int *table, *refs, *result;
    const int *lens, *n;
    int *claims, *last, *plan, *ids; // work: claims to a shared page, the last sequence with one; entries' plans; free pages
    int4 *copies;                    // of each sequence: from, to, blocks
};

constexpr int BOOK_PAGES = 8; // neighbouring pages that a thread of the books looks at
// Bits of the thread's pages from `first` on that are free (used: the others).
__device__ __forceinline__ uint32_t free_pages(const int *refs, int n_pages, int first, bool used) {
    typedef int i32x4 __attribute__((ext_vector_type(4), aligned(4)));
    uint32_t bits = 0;
    if (first + BOOK_PAGES <= n_pages) {
        const i32x4 a = *(const i32x4 *)(refs + first), b = *(const i32x4 *)(refs + first + 4);
#pragma unroll
        for (int k = 0; k < 4; k++) bits |= (uint32_t)((a[k] > 0) == used) << k | (uint32_t)((b[k] > 0) == used) << (k + 4);
    } else {
        for (int k = 0; first + k < n_pages; k++) bits |= (uint32_t)((refs[first + k] > 0) == used) << k;
    }
    return bits;
}

// The pages that each sequence needs, in the order of sequences and positions, one workgroup.  It is bound by the latency of
// loads that depend on each other: what the free pages are is asked for first, an entry's own loads are kept for the end, and the
// claims to shared pages are compared only where there are some.  5.6 us for 4 beams, 7.4 for 64 with shared pages.
__global__ void __launch_bounds__(BOOK_T) k_reserve(ReserveArgs a) {
    __shared__ int sm[BOOK_T / 64], misfit, any_shared;
    __shared__ int2 claim[BOOK_T];
    const int items = a.n_seq * a.most;
    struct Item {
        int b, e, len, refs;
        int64_t at;       // of the table
        bool fits, asked; // the sequence's tokens; a page that they are written to
    };
    auto item = [&](int i) {
        Item t;
        t.b = i / a.most;
        const int len = max(a.lens[t.b], 0), nn = a.n[t.b], j = len / a.page + i % a.most;
        t.len = len;
        t.fits = nn <= 0 || (nn <= a.max_n && (int64_t)len + nn <= (int64_t)a.per * a.page);
        t.asked = nn > 0 && t.fits && j <= (len + nn - 1) / a.page;
        t.at = (int64_t)t.b * a.per + j;
        t.e = t.asked ? a.table[t.at] : -1;
        if ((uint32_t)t.e >= (uint32_t)a.n_pages) t.e = -1;
        t.refs = t.e >= 0 ? a.refs[t.e] : 0;
        return t;
    };
    if (threadIdx.x == 0) misfit = any_shared = 0;
    uint32_t free = free_pages(a.refs, a.n_pages, BOOK_PAGES * (int)threadIdx.x, false);
    __syncthreads();
    Item mine; // of entry threadIdx.x
    int plan0 = 0, want = 0; // plan: 1 a page, 2 one in place of a shared one, 3 shared, not decided yet
    mine.e = -1, mine.len = 0, mine.at = 0, mine.b = 0;
    for (int i = threadIdx.x; i < items; i += BOOK_T) {
        const Item t = item(i);
        const int plan = !t.asked ? 0 : t.refs <= 0 ? 1 : t.refs > 1 ? 3 : 0;
        if (!t.fits) misfit = 1;
        if (plan == 3) any_shared = 1;
        if (i < BOOK_T) mine = t, plan0 = plan;
        else a.plan[i] = plan;
        want += plan == 1;
    }
    __syncthreads();
    if (any_shared && items <= BOOK_T) { // few: compared with each other in LDS
        int all;
        const int at = block_scan(plan0 == 3, sm, all) - 1;
        if (plan0 == 3) claim[at] = make_int2(mine.e, mine.b);
        __syncthreads();
        if (plan0 == 3) {
            int claims = 0;
            bool later = false;
            for (int k = 0; k < all; k++) {
                const int2 c = claim[k];
                claims += c.x == mine.e;
                later |= c.x == mine.e && c.y > mine.b;
            }
            plan0 = claims != mine.refs || later ? 2 : 0; // (all who have it want it: the last one keeps it)
            want += plan0 == 2;
        }
    } else if (any_shared) {
        for (int i = threadIdx.x; i < items; i += BOOK_T)
            if ((i < BOOK_T ? plan0 : a.plan[i]) == 3) {
                const Item t = i < BOOK_T ? mine : item(i);
                a.claims[t.e] = 0, a.last[t.e] = -1;
            }
        __threadfence();
        __syncthreads();
        for (int i = threadIdx.x; i < items; i += BOOK_T)
            if ((i < BOOK_T ? plan0 : a.plan[i]) == 3) {
                const Item t = i < BOOK_T ? mine : item(i);
                atomicAdd(&a.claims[t.e], 1);
                atomicMax(&a.last[t.e], t.b);
            }
        __threadfence();
        __syncthreads();
        for (int i = threadIdx.x; i < items; i += BOOK_T)
            if ((i < BOOK_T ? plan0 : a.plan[i]) == 3) {
                const Item t = i < BOOK_T ? mine : item(i);
                const int claims = __hip_atomic_load(&a.claims[t.e], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                const int last = __hip_atomic_load(&a.last[t.e], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                const int plan = claims != t.refs || last != t.b ? 2 : 0;
                if (i < BOOK_T) plan0 = plan;
                else a.plan[i] = plan;
                want += plan == 2;
            }
    }
    int total, found = 0;
    block_scan(want, sm, total);
    for (int base = 0; base < a.n_pages && found < total; base += BOOK_PAGES * BOOK_T) {
        const int first = base + BOOK_PAGES * (int)threadIdx.x;
        if (base) free = free_pages(a.refs, a.n_pages, first, false);
        int all, at = found + block_scan(__popc(free), sm, all) - __popc(free);
        for (uint32_t f = free; f && at < total; f &= f - 1) a.ids[at++] = first + __ffs(f) - 1;
        found += all;
    }
    const bool ok = found >= total && !misfit;
    if (threadIdx.x == 0) a.result[0] = ok, a.result[1] = total;
    for (int b = threadIdx.x; b < a.n_seq; b += BOOK_T) a.copies[b] = make_int4(-1, 0, 0, 0);
    if (!ok || !total) return;
    __syncthreads();
    int before = 0;
    for (int base = 0; base < items; base += BOOK_T) {
        const int i = base + threadIdx.x, plan = i >= items ? 0 : base ? a.plan[i] : plan0;
        int all;
        const int rank = before + block_scan(plan != 0, sm, all) - 1;
        before += all;
        if (!plan) continue;
        const Item t = base ? item(i) : mine;
        const int page = a.ids[rank];
        a.table[t.at] = page;
        a.refs[page] = 1;
        if (plan == 2) {
            atomicSub(&a.refs[t.e], 1);
            if (i % a.most == 0 && t.len % a.page)
                a.copies[t.b] = make_int4(t.e, page, (t.len % a.page + PAGE_BLOCK - 1) / PAGE_BLOCK, 0);
        }
    }
}

struct MoveArgs {
    uint8_t *c[2];
    float *s[2];
    int64_t layer, id, head, s_layer, s_id, s_head;
    int hs, n_kv, n_layers;
};
// `blocks` blocks of page `from` to page `to`, of one layer, head and side, by a wave: eight loads of 16 bytes a lane under way.
// Bound by memory: 424 MB moved in 171 us, 5.0 TB/s read and written.
__device__ __forceinline__ void move_blocks(const MoveArgs &a, uint32_t unit, int from, int to, int blocks) {
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    const int lane = threadIdx.x & 63, side = unit & 1, h = unit / 2 % a.n_kv, layer = unit / 2 / a.n_kv;
    const int64_t at = layer * a.layer + h * a.head, s_at = layer * a.s_layer + h * a.s_head;
    const u32x4 *src = (const u32x4 *)(a.c[side] + at + from * a.id);
    u32x4 *dst = (u32x4 *)(a.c[side] + at + to * a.id);
    const int count = blocks * (PAGE_BLOCK / 16) * a.hs;
    float s = 0.0f;
    if (lane < blocks) s = a.s[side][s_at + from * a.s_id + lane];
    for (int i = lane; i < count; i += 64 * 8) {
        u32x4 v[8];
#pragma unroll
        for (int k = 0; k < 8; k++)
            if (i + 64 * k < count) v[k] = src[i + 64 * k];
#pragma unroll
        for (int k = 0; k < 8; k++)
            if (i + 64 * k < count) dst[i + 64 * k] = v[k];
    }
    if (lane < blocks) a.s[side][s_at + to * a.s_id + lane] = s;
}
__global__ void __launch_bounds__(256) k_reserve_copy(MoveArgs a, const int4 *copies, uint32_t units) {
    const int4 c = copies[blockIdx.y];
    const uint32_t u = blockIdx.x * 4 + threadIdx.x / 64;
    if (c.x >= 0 && u < units) move_blocks(a, u, c.x, c.y, c.z);
}

struct CompactArgs {
    int n_pages, n_seq, per;
    int *table, *refs, *result;
    int *map, *hole, *far; // work: where pages from the u-th on went; the free numbers below, the used ones above
};
// Holes and what goes there, in order, by one workgroup.
__global__ void __launch_bounds__(BOOK_T) k_compact(CompactArgs a) {
    __shared__ int sm[BOOK_T / 64];
    constexpr int STEP = BOOK_PAGES * BOOK_T;
    const int mine = BOOK_PAGES * (int)threadIdx.x;
    const uint32_t first = free_pages(a.refs, a.n_pages, mine, true); // (of most pools these are all)
    int sum = __popc(first), u, holes = 0, fars = 0;
    for (int base = STEP; base < a.n_pages; base += STEP) sum += __popc(free_pages(a.refs, a.n_pages, base + mine, true));
    block_scan(sum, sm, u);
    for (int base = 0; base < a.n_pages; base += STEP) {
        const int at = base + mine, have = min(max(a.n_pages - at, 0), BOOK_PAGES), below = min(max(u - at, 0), have);
        const uint32_t used = base ? free_pages(a.refs, a.n_pages, at, true) : first;
        const uint32_t low = (1u << below) - 1, there = (1u << have) - 1;
        const uint32_t hole = ~used & low, far = used & there & ~low;
        int all; // (both counts in one sum: a pass has no more than 8192 of either)
        const int upto = block_scan(__popc(hole) | __popc(far) << 16, sm, all);
        int h = holes + (upto & 0xffff) - __popc(hole), f = fars + (upto >> 16) - __popc(far);
        holes += all & 0xffff;
        fars += all >> 16;
        for (uint32_t x = hole; x; x &= x - 1) a.hole[h++] = at + __ffs(x) - 1;
        for (int k = below; k < have; k++) {
            const bool moves = far >> k & 1;
            a.map[at + k] = moves ? f : -1;
            if (moves) a.far[f++] = at + k;
        }
    }
    if (threadIdx.x == 0) a.result[0] = u, a.result[1] = fars;
    __syncthreads();
    for (int k = threadIdx.x; k < fars; k += BOOK_T) {
        const int to = a.hole[k], from = a.far[k];
        a.refs[to] = a.refs[from];
        a.refs[from] = 0;
    }
}
// The pages' contents, and the tables: blocks from `movers` on take the latter.
__global__ void __launch_bounds__(256) k_compact_move(MoveArgs a, CompactArgs t, int blocks, int movers) {
    const int u = t.result[0], moves = t.result[1];
    if ((int)blockIdx.x >= movers) {
        const int64_t i = (int64_t)(blockIdx.x - movers) * 256 + threadIdx.x;
        if (i >= (int64_t)t.n_seq * t.per) return;
        const int e = t.table[i];
        if (e < u || e >= t.n_pages) return;
        const int k = t.map[e];
        t.table[i] = k < 0 ? -1 : t.hole[k];
        return;
    }
    const int64_t per = (int64_t)2 * a.n_kv * a.n_layers;
    for (int64_t i = blockIdx.x * 4 + threadIdx.x / 64; i < moves * per; i += 4 * movers) {
        const int k = (int)(i / per);
        move_blocks(a, (uint32_t)(i - k * per), t.far[k], t.hole[k], blocks);
    }
}

MoveArgs move_args(const llm_pages *c) {
    MoveArgs a;
    memset(&a, 0, sizeof a);
    a.c[0] = (uint8_t *)c->k, a.c[1] = (uint8_t *)c->v, a.s[0] = c->k_scale, a.s[1] = c->v_scale;
    a.layer = c->layer, a.id = c->id, a.head = c->head, a.s_layer = c->s_layer, a.s_id = c->s_id, a.s_head = c->s_head;
    a.hs = c->hs, a.n_kv = c->n_kv, a.n_layers = c->n_layers;
    return a;
}

constexpr int64_t MOST_UNITS = 1 << 25; // layers, heads and sides of a page: a wave each, and a grid has 2^32 threads

bool work_ok(const char *who, void *work, size_t have, size_t need, unsigned align, OpDevice &dev) {
    if (!need || (have >= need && !((uintptr_t)work & (align - 1)) && dev.holds(work, "the work memory"))) return true;
    fprintf(stderr, "%s: %zu bytes of work memory are needed, %u-byte aligned\n", who, need, align);
    return false;
}

int reach(int per, int page, int max_n) { // pages that max_n tokens can touch
    return (int)std::min<int64_t>(per, ((int64_t)max_n + page - 2) / page + 1);
}

} // namespace

bool op_check_pages(const llm_pages *c, OpDevice *dev, const char *who) {
    if (!op_scaled(c->type) || c->n_layers < 1 || c->n_pages < 1 || c->n_kv < 1 || c->hs < 16 || c->hs > 256 || c->hs % 16 ||
        (c->page != 64 && c->page != 128 && c->page != 256)) {
        fprintf(stderr, "%s: pages of type %d, %d layers of %d pages, %d heads of %d values, %d positions are not taken\n", who,
                c->type, c->n_layers, c->n_pages, c->n_kv, c->hs, c->page);
        return false;
    }
    // layers, pages and heads in the order of their strides: each lies behind what the ones before it take (of one there is no
    // next)
    auto apart = [&](int64_t least, int64_t layer, int64_t id, int64_t head) {
        std::pair<int64_t, int> dim[] = {{layer, c->n_layers}, {id, c->n_pages}, {head, c->n_kv}};
        std::sort(dim, dim + 3);
        __int128 extent = least;
        for (auto [stride, count] : dim) {
            if (count > 1 && stride < extent) return false;
            extent += (__int128)(count - 1) * stride;
        }
        return true;
    };
    if (!apart((int64_t)c->page * c->hs, c->layer, c->id, c->head) || !apart(c->page / PAGE_BLOCK, c->s_layer, c->s_id, c->s_head)) {
        fprintf(stderr, "%s: strides of the pages that lie on themselves\n", who);
        return false;
    }
    if (c->layer < 0 || c->id < 0 || c->head < 0 || c->s_layer < 0 || c->s_id < 0 || c->s_head < 0 ||
        ((c->layer | c->id | c->head) & 15) || (((uintptr_t)c->k | (uintptr_t)c->v) & 15) ||
        (((uintptr_t)c->k_scale | (uintptr_t)c->v_scale) & 3)) {
        fprintf(stderr, "%s: addresses and strides of the codes have to be multiples of 16, of the scales of 4 bytes\n", who);
        return false;
    }
    if (c->k == c->v || c->k_scale == c->v_scale) {
        fprintf(stderr, "%s: k and v are the same memory\n", who);
        return false;
    }
    if (!dev) return true;
    return dev->holds(c->k, "the K pages") && dev->holds(c->v, "the V pages") && dev->holds(c->k_scale, "the K scales") &&
           dev->holds(c->v_scale, "the V scales");
}

bool op_check_table(const int *table, int n_seq, int per, OpDevice *dev, const char *who) {
    if (n_seq < 0 || per < 1 || ((uintptr_t)table & 3)) {
        fprintf(stderr, "%s: a table of %d sequences, %d pages each\n", who, n_seq, per);
        return false;
    }
    if (per > (1 << 30) / 256) { // (positions stay within an int)
        fprintf(stderr, "%s: %d pages for a sequence\n", who, per);
        return false;
    }
    return !dev || dev->holds(table, "table");
}

extern "C" int llm_page_write(const llm_pages *c, const llm_rows *k, const llm_rows *v, int n_seq, const int *table, int per,
                              const int *refs, const int *pos, const int *n, const int *path, int max_n, void *stream) {
    return page_rows("llm_page_write", true, c, k, v, n_seq, table, per, refs, pos, n, path, max_n, 0, stream);
}

extern "C" int llm_page_read(const llm_pages *c, const llm_rows *k, const llm_rows *v, int n_seq, const int *table, int per,
                             const int *pos, const int *n, int max_n, int zero_rest, void *stream) {
    return page_rows("llm_page_read", false, c, k, v, n_seq, table, per, nullptr, pos, n, nullptr, max_n, zero_rest, stream);
}

extern "C" size_t llm_page_fork_work(int per, int count) {
    return per > 0 && count > 0 && count <= 65535 ? (size_t)count * ((size_t)per + 1) * 4 : 0;
}

extern "C" int llm_page_fork(int n_pages, int page, int n_seq, int *table, int per, int *lens, int *refs, const int *to,
                             const int *from, int count, void *work, size_t work_bytes, void *stream) {
    const char *who = "llm_page_fork";
    if (n_pages < 1 || (page != 64 && page != 128 && page != 256) || count < 0 || count > 65535) {
        fprintf(stderr, "%s: bad arguments (%d pages of %d positions, %d entries)\n", who, n_pages, page, count);
        return -1;
    }
    if (!op_check_table(table, n_seq, per, nullptr, who)) return -1;
    if (!count || !n_seq) return 0;
    OpDevice dev(who);
    if (!op_check_table(table, n_seq, per, &dev, who) || !dev.holds(lens, "lens") || !dev.holds(refs, "refs") ||
        !dev.holds(to, "to") || !dev.holds(from, "from") ||
        !work_ok(who, work, work_bytes, llm_page_fork_work(per, count), 4, dev) || !dev.select())
        return -1;
    const ForkArgs a = {n_pages, page, n_seq, per, count, table, lens, refs, to, from, (int *)work + count, (int *)work};
    hipLaunchKernelGGL(k_fork_count, dim3(count), dim3(256), 0, (hipStream_t)stream, a);
    HIP_OR_FAIL(who, hipGetLastError());
    hipLaunchKernelGGL(k_fork_write, dim3(count), dim3(256), 0, (hipStream_t)stream, a);
    HIP_OR_FAIL(who, hipGetLastError());
    return 0;
}

extern "C" size_t llm_page_reserve_work(const llm_pages *c, int n_seq, int per, int max_n) {
    if (!c || !op_scaled(c->type) || c->n_pages < 1 || c->page < 64 || n_seq < 1 || per < 1 || max_n < 1) return 0;
    const size_t items = (size_t)n_seq * reach(per, c->page, max_n);
    return (size_t)n_seq * 16 + 4 * (2 * (size_t)c->n_pages + 2 * items);
}

extern "C" int llm_page_reserve(const llm_pages *c, int n_seq, int *table, int per, int *refs, const int *lens, const int *n,
                                int max_n, int *result, void *work, size_t work_bytes, void *stream) {
    const char *who = "llm_page_reserve";
    if (!c || max_n < 0) {
        fprintf(stderr, "%s: bad arguments\n", who);
        return -1;
    }
    if (!op_check_pages(c, nullptr, who) || !op_check_table(table, n_seq, per, nullptr, who)) return -1;
    const int64_t units = (int64_t)2 * c->n_kv * c->n_layers;
    if ((int64_t)n_seq * reach(per, c->page, max_n) > 1 << 30 || n_seq > 65535 || units > MOST_UNITS) {
        fprintf(stderr, "%s: %d sequences of %d tokens, %d layers of %d heads\n", who, n_seq, max_n, c->n_layers, c->n_kv);
        return -1;
    }
    OpDevice dev(who);
    if (!op_check_pages(c, &dev, who)) return -1;
    const bool any = max_n && n_seq; // (else only the result is written)
    if (!dev.holds(refs, "refs") || !dev.holds(result, "result") ||
        (any && (!op_check_table(table, n_seq, per, &dev, who) || !dev.holds(lens, "lens") || !dev.holds(n, "n") ||
                 !work_ok(who, work, work_bytes, llm_page_reserve_work(c, n_seq, per, max_n), 16, dev))) ||
        !dev.select())
        return -1;
    ReserveArgs a;
    memset(&a, 0, sizeof a);
    a.n_pages = c->n_pages, a.page = c->page, a.n_seq = any ? n_seq : 0, a.per = per, a.max_n = max_n;
    a.most = reach(per, c->page, max_n);
    a.table = table, a.refs = refs, a.result = result, a.lens = lens, a.n = n;
    a.copies = (int4 *)work;
    a.claims = (int *)(a.copies + n_seq), a.last = a.claims + c->n_pages, a.plan = a.last + c->n_pages;
    a.ids = a.plan + (size_t)n_seq * a.most;
    hipLaunchKernelGGL(k_reserve, dim3(1), dim3(BOOK_T), 0, (hipStream_t)stream, a);
    HIP_OR_FAIL(who, hipGetLastError());
    if (!any) return 0;
    hipLaunchKernelGGL(k_reserve_copy, dim3((unsigned)((units + 3) / 4), n_seq), dim3(256), 0, (hipStream_t)stream, move_args(c),
                       (const int4 *)a.copies, (uint32_t)units);
    HIP_OR_FAIL(who, hipGetLastError());
    return 0;
}

extern "C" size_t llm_page_compact_work(const llm_pages *c) {
    return c && c->n_pages > 0 ? 4 * 3 * (size_t)c->n_pages : 0;
}

extern "C" int llm_page_compact(const llm_pages *c, int n_seq, int *table, int per, int *refs, int *result, void *work,
                                size_t work_bytes, void *stream) {
    const char *who = "llm_page_compact";
    if (!c) {
        fprintf(stderr, "%s: bad arguments\n", who);
        return -1;
    }
    if (!op_check_pages(c, nullptr, who) || !op_check_table(table, n_seq, per, nullptr, who)) return -1;
    const int64_t entries = (int64_t)n_seq * per;
    const int movers = 2048;
    if (entries > (int64_t)1 << 31) { // (a thread each, of 2^32; looked at before the first launch changes the counts)
        fprintf(stderr, "%s: a table of %d sequences, %d pages each\n", who, n_seq, per);
        return -1;
    }
    if ((int64_t)2 * c->n_kv * c->n_layers > MOST_UNITS) {
        fprintf(stderr, "%s: %d layers of %d heads\n", who, c->n_layers, c->n_kv);
        return -1;
    }
    OpDevice dev(who);
    if (!op_check_pages(c, &dev, who) || (n_seq && !op_check_table(table, n_seq, per, &dev, who)) || !dev.holds(refs, "refs") ||
        !dev.holds(result, "result") || !work_ok(who, work, work_bytes, llm_page_compact_work(c), 4, dev) || !dev.select())
        return -1;
    CompactArgs a;
    memset(&a, 0, sizeof a);
    a.n_pages = c->n_pages, a.n_seq = n_seq, a.per = per, a.table = table, a.refs = refs, a.result = result;
    a.map = (int *)work, a.hole = a.map + c->n_pages, a.far = a.hole + c->n_pages;
    hipLaunchKernelGGL(k_compact, dim3(1), dim3(BOOK_T), 0, (hipStream_t)stream, a);
    HIP_OR_FAIL(who, hipGetLastError());
    hipLaunchKernelGGL(k_compact_move, dim3(movers + (unsigned)((entries + 255) / 256)), dim3(256), 0, (hipStream_t)stream,
                       move_args(c), a, c->page / PAGE_BLOCK, movers);
    HIP_OR_FAIL(who, hipGetLastError());
    return 0;
}
