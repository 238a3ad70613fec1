// llm_logprobs: log probabilities of given tokens, entropy and the largest logits, one pass over the logits.
//
// A block walks a row (or a segment of it, where there are few rows) in steps of 16 values a thread.  Per thread: the running
// maximum m, s = sum e^(x - m) and t = sum e^(x - m) (x - m), joined at the end: lse = m + log s, entropy = log s - t / s.
// The largest logits: a value goes into the block's list in LDS only if it is above a bound that at least `top` values
// reach.  The bound starts as the top-th largest of a wave's 64 lane maxima (at least `top` values reach that), and becomes
// the list's own top-th value when the list is cut, so that after the first steps almost nothing is listed and the
// logits are read at the rate of memory: 1021 rows of 151936 fp32 logits 132 us, 4.7 TB/s.  Few rows are bound by what every
// segment begins with, the first bound's 32 dependent ballots and the first cut of the list, and by a second launch: one row of
// 65536 logits, top 20, 7.8 us and the segments' join 6.0; 37 of 151936 bf16 logits, top 5, 12.0 and 3.9 (vector instructions in
// 11k of the 20k cycles that a SIMD's waves live, with two steps a segment).
#include <string.h>

#include <algorithm>

#include "device.h"
#include "operators.h"

namespace {

constexpr int LP_T = 256, LP_E = 16, LP_STEP = LP_T * LP_E; // values a block takes at once
constexpr int LP_TOP = 32;                                  // most alternatives
constexpr int LP_KEEP = 256;                                // the list is cut when it holds more
constexpr int LP_CAP = LP_KEEP + LP_STEP;          // (a step adds no more than it has)
constexpr int LP_MAX_SEG = 64;

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct LpArgs {
    const uint8_t *x;
    int64_t stride; // bytes
    int rows, vocab, seg, per; // segments of a row, steps of each
    float inv_t;
    const int *tokens;
    int n_tokens, top;
    float *logp, *entropy, *lse, *top_logp;
    int *top_ids;
    float *part;     // [row][segment][4]: m, s, t
    uint64_t *list;  // [row][segment][top]
};

// Order-preserving key of a logit; NaN above all, -0 as +0.  An entry is key << 32 | ~index: the larger entry is the
// larger logit, the lower index among equals.
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);
    if (x != x) return 0xffffffffu;
    return u >> 31 ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) {
    return __uint_as_float(key == 0xffffffffu ? 0x7fc00000u : key >> 31 ? key & 0x7fffffffu : ~key);
}
__device__ __forceinline__ uint64_t entry_of(float x, int i) { return (uint64_t)key_of(x) << 32 | (uint32_t)~i; }

struct Stat {
    float m, s, t; // t over z = (x - m) log2(e) / T
};
// a and b with one maximum; c = log2(e) / T
__device__ __forceinline__ Stat join(Stat a, Stat b, float c) {
    Stat r;
    r.m = fmaxf(a.m, b.m);
    const float mu = r.m == -INFINITY ? 0.0f : r.m;
    auto add = [&](const Stat &o, float &s, float &t) {
        const float d = fmaxf((o.m - mu) * c, -300.0f), f = __builtin_amdgcn_exp2f(d); // (-300: factor 0)
        s += o.s * f;
        t += (o.t + d * o.s) * f;
    };
    r.s = r.t = 0.0f;
    add(a, r.s, r.t);
    add(b, r.s, r.t);
    return r;
}
__device__ __forceinline__ Stat wave_join(Stat v, float c) {
    Stat r;
    r.m = wave_max(v.m);
    const float mu = r.m == -INFINITY ? 0.0f : r.m;
    const float d = fmaxf((v.m - mu) * c, -300.0f), f = __builtin_amdgcn_exp2f(d);
    r.s = wave_sum(v.s * f);
    r.t = wave_sum((v.t + d * v.s) * f);
    return r;
}

// The k-th largest (k >= 1) of the 64 lanes' keys: the largest key that at least k lanes reach, bit by bit.
__device__ __forceinline__ uint32_t kth_of_wave(uint32_t key, int k) {
    uint32_t r = 0;
#pragma unroll
    for (int bit = 31; bit >= 0; bit--) {
        const uint32_t c = r | 1u << bit;
        if (__popcll(__ballot(key >= c)) >= k) r = c;
    }
    return r;
}

// The `top` largest of list[0 .. n) to its front in descending order (all of them, ordered, where n <= top), by the block.
// Distinct entries; scratch: LP_TOP entries.
__device__ void list_cut(uint64_t *list, int n, int top, uint64_t *scratch) {
    const int keep = min(n, top);
    if (n <= 2 * LP_KEEP) { // an entry's place is the number of larger ones
        for (int i = threadIdx.x; i < n; i += LP_T) {
            const uint64_t e = list[i];
            int r = 0, k = 0;
            for (; k + 8 <= n; k += 8) // (eight reads under way at once)
#pragma unroll
                for (int u = 0; u < 8; u++) r += list[k + u] > e;
            for (; k < n; k++) r += list[k] > e;
            if (r < keep) scratch[r] = e;
        }
        __syncthreads();
    } else { // many: the largest below the last one found, `keep` times
        __shared__ uint64_t best[LP_T / 64];
        uint64_t below = ~(uint64_t)0;
        for (int r = 0; r < keep; r++) {
            uint64_t b = 0;
            for (int i = threadIdx.x; i < n; i += LP_T) {
                const uint64_t e = list[i];
                if (e < below && e > b) b = e;
            }
            for (int off = 1; off < 64; off <<= 1) {
                const uint64_t o = __shfl_xor((unsigned long long)b, off);
                if (o > b) b = o;
            }
            if ((threadIdx.x & 63) == 0) best[threadIdx.x / 64] = b;
            __syncthreads();
            for (int w = 0; w < LP_T / 64; w++)
                if (best[w] > b) b = best[w];
            below = b;
            if (threadIdx.x == 0) scratch[r] = b;
            __syncthreads();
        }
    }
    for (int i = threadIdx.x; i < keep; i += LP_T) list[i] = scratch[i];
    __syncthreads();
}

// Results of a row from its statistics and its ordered list.
__device__ void finish(const LpArgs &a, int row, Stat st, const uint64_t *list) {
    const float ln2 = 0.69314718055994530942f, ls = logf(st.s);
    if (threadIdx.x == 0) {
        if (a.lse) a.lse[row] = st.m * a.inv_t + ls;
        if (a.entropy) a.entropy[row] = ls - ln2 * (st.t / st.s);
    }
    for (int i = threadIdx.x; i < a.top; i += LP_T) {
        const uint64_t e = list[i];
        a.top_ids[(int64_t)row * a.top + i] = (int)~(uint32_t)e;
        a.top_logp[(int64_t)row * a.top + i] = (value_of((uint32_t)(e >> 32)) - st.m) * a.inv_t - ls;
    }
}

template <int TY>
__device__ __forceinline__ float value_at(const uint8_t *row, int i) {
    if constexpr (TY == LLM_F32) return ((const float *)row)[i];
    return __uint_as_float((uint32_t)((const uint16_t *)row)[i] << 16);
}

// the logit of a row's i-th given token
template <int TY>
__device__ __forceinline__ float given_logit(const LpArgs &a, int row, int i) {
    const int tok = a.tokens[(int64_t)row * a.n_tokens + i];
    return tok >= 0 && tok < a.vocab ? value_at<TY>(a.x + row * a.stride, tok) : -INFINITY;
}
// their log probabilities; x the thread's first logit (an id out of range: -infinity whatever the row holds)
template <int TY>
__device__ __forceinline__ void given(const LpArgs &a, int row, Stat st, float x) {
    const float ls = logf(st.s);
    for (int i = threadIdx.x; i < a.n_tokens; i += LP_T) {
        const int tok = a.tokens[(int64_t)row * a.n_tokens + i];
        if (i >= LP_T) x = given_logit<TY>(a, row, i);
        a.logp[(int64_t)row * a.n_tokens + i] = tok >= 0 && tok < a.vocab ? (x - st.m) * a.inv_t - ls : -INFINITY;
    }
}

template <int TY>
__global__ void __launch_bounds__(LP_T) k_logprobs(LpArgs a) {
    constexpr int ES = TY == LLM_F32 ? 4 : 2, PER = 16 / ES, NL = LP_E / PER; // values a 16-byte load, loads a step
    __shared__ uint64_t list[LP_CAP];
    __shared__ uint64_t scratch[LP_TOP];
    __shared__ Stat sm_st[LP_T / 64];
    __shared__ uint32_t bound;
    __shared__ int count;
    const int row = blockIdx.x / a.seg, seg = blockIdx.x - row * a.seg, lane = threadIdx.x & 63;
    // The row from the 16-byte boundary at or before its start, to the one at or after its end: no load leaves a 16-byte
    // unit that holds some of the row.  Values are numbered from there; `lead` of them are not the row's.
    const uintptr_t start = (uintptr_t)(a.x + row * a.stride);
    const int lead = (int)(start & 15) / ES;
    const int64_t bytes = ((int64_t)(lead + a.vocab) * ES + 15) & ~(int64_t)15;
    const auto rs = __builtin_amdgcn_make_buffer_rsrc((void *)(start & ~(uintptr_t)15), 0, (int)bytes, 0x00020000);
    const int steps = (int)((bytes + 16 * NL * LP_T - 1) / (16 * NL * LP_T));
    const int first = seg * a.per, last = min(first + a.per, steps);
    const float c = a.inv_t * 1.44269504088896340736f;
    if (threadIdx.x == 0) bound = 0, count = 0;
    __syncthreads();
    u32x4 raw[NL];
    auto load = [&](int step) {
#pragma unroll
        for (int i = 0; i < NL; i++) {
            const uint32_t off = ((uint32_t)step * NL + i) * LP_T * 16 + threadIdx.x * 16;
            const auto v = __builtin_amdgcn_raw_buffer_load_b128(rs, (int)(step < last ? off : 0x80000000u), 0, 0);
            raw[i] = (u32x4){v[0], v[1], v[2], v[3]};
        }
    };
    Stat st = {-INFINITY, 0.0f, 0.0f};
    load(first);
    for (int step = first; step < last; step++) {
        float x[LP_E];
#pragma unroll
        for (int i = 0; i < NL; i++)
#pragma unroll
            for (int k = 0; k < PER; k++)
                x[i * PER + k] = TY == LLM_F32 ? __uint_as_float(raw[i][k])
                                               : __uint_as_float(k % 2 ? raw[i][k / 2] & 0xffff0000u : raw[i][k / 2] << 16);
        load(step + 1);
        // index of value i * PER + k of this thread in the row
        const int idx0 = (step * NL * LP_T + (int)threadIdx.x) * PER - lead;
        auto idx = [&](int e) { return idx0 + (e / PER) * LP_T * PER + e % PER; };
        const bool edge = step == 0 || step == steps - 1;
        if (edge)
#pragma unroll
            for (int e = 0; e < LP_E; e++)
                if ((uint32_t)idx(e) >= (uint32_t)a.vocab) x[e] = -INFINITY;
        float mx = x[0];
#pragma unroll
        for (int e = 1; e < LP_E; e++) mx = fmaxf(mx, x[e]);
        const float mn = fmaxf(st.m, mx), mu = mn == -INFINITY ? 0.0f : mn;
        {
            const float d = fmaxf((st.m - mu) * c, -300.0f), f = __builtin_amdgcn_exp2f(d);
            st.t = (st.t + d * st.s) * f;
            st.s *= f;
            st.m = mn;
        }
#pragma unroll
        for (int e = 0; e < LP_E; e++) {
            const float z = (x[e] - mu) * c, p = __builtin_amdgcn_exp2f(z);
            st.s += p;
            st.t += p * fmaxf(z, -300.0f);
        }
        if (a.top) {
            uint32_t km = key_of(mx);
            if (st.s != st.s) { // (NaN among the values: the maximum does not show it)
#pragma unroll
                for (int e = 0; e < LP_E; e++) km = max(km, key_of(x[e]));
            }
            uint32_t lim = bound; // values below lim, or equal to it behind a full list, are not among the top
            if (__popcll(__ballot(km > lim)) >= a.top) lim = max(lim, kth_of_wave(km, a.top) - 1);
            if (__any(km > lim)) { // places by one addition a wave
                uint64_t in[LP_E];
                int total = 0;
#pragma unroll
                for (int e = 0; e < LP_E; e++) {
                    in[e] = __ballot((!edge || (uint32_t)idx(e) < (uint32_t)a.vocab) && key_of(x[e]) > lim);
                    total += __popcll(in[e]);
                }
                int at = 0;
                if (lane == 0 && total) at = atomicAdd(&count, total);
                at = __builtin_amdgcn_readfirstlane(at);
#pragma unroll
                for (int e = 0; e < LP_E; e++) {
                    if (in[e] == 0) continue;
                    if ((in[e] >> lane) & 1)
                        list[at + __builtin_amdgcn_mbcnt_hi((uint32_t)(in[e] >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)in[e], 0))] =
                            entry_of(x[e], idx(e));
                    at += __popcll(in[e]);
                }
            }
            __syncthreads();
            const int have = count;
            if (step + 1 < last && (have > LP_KEEP || (!bound && have >= a.top))) {
                list_cut(list, have, a.top, scratch);
                if (threadIdx.x == 0) {
                    count = a.top;
                    bound = (uint32_t)(list[a.top - 1] >> 32);
                }
            }
            __syncthreads();
        }
    }
    st = wave_join(st, c);
    if (lane == 0) sm_st[threadIdx.x / 64] = st;
    __syncthreads();
    st = sm_st[0];
#pragma unroll
    for (int w = 1; w < LP_T / 64; w++) st = join(st, sm_st[w], c);
    int have = 0;
    if (a.top) {
        have = min(count, a.top);
        list_cut(list, count, a.top, scratch);
    }
    if (a.seg == 1) {
        finish(a, row, st, list);
        given<TY>(a, row, st, (int)threadIdx.x < a.n_tokens ? given_logit<TY>(a, row, threadIdx.x) : 0.0f);
    } else {
        const int64_t part = (int64_t)row * a.seg + seg;
        if (threadIdx.x == 0) {
            a.part[4 * part] = st.m;
            a.part[4 * part + 1] = st.s;
            a.part[4 * part + 2] = st.t;
        }
        for (int i = threadIdx.x; i < a.top; i += LP_T) a.list[part * a.top + i] = i < have ? list[i] : 0;
    }
}

// The segments of a row joined.
template <int TY>
__global__ void __launch_bounds__(LP_T) k_logprobs_join(LpArgs a) {
    __shared__ uint64_t list[LP_MAX_SEG * LP_TOP];
    __shared__ uint64_t scratch[LP_TOP];
    __shared__ int count;
    const int row = blockIdx.x, lane = threadIdx.x & 63;
    const float c = a.inv_t * 1.44269504088896340736f;
    const float *pt = a.part + 4 * (int64_t)row * a.seg;
    // every load that depends on no other first: the statistics, the lists, the given tokens' logits
    constexpr int NE = LP_MAX_SEG * LP_TOP / LP_T;
    const uint64_t *from = a.list + (int64_t)row * a.seg * a.top;
    Stat st = {-INFINITY, 0.0f, 0.0f};
    if (lane < a.seg) st = {pt[4 * lane], pt[4 * lane + 1], pt[4 * lane + 2]};
    uint64_t ent[NE], end = 0;
#pragma unroll
    for (int u = 0; u < NE; u++) ent[u] = (int)threadIdx.x + u * LP_T < a.seg * a.top ? from[threadIdx.x + u * LP_T] : 0;
    if (a.top && lane < a.seg) end = from[lane * a.top + a.top - 1];
    float x = 0.0f;
    if ((int)threadIdx.x < a.n_tokens) x = given_logit<TY>(a, row, threadIdx.x);
    if (threadIdx.x == 0) count = 0;
    __syncthreads();
    st = wave_join(st, c);
    if (a.top) {
        // the segments' last entries: `top` values reach the largest of them
        uint32_t lim = (uint32_t)(end >> 32);
        for (int off = 1; off < 64; off <<= 1) lim = max(lim, (uint32_t)__shfl_xor((int)lim, off));
#pragma unroll
        for (int u = 0; u < NE; u++)
            if (ent[u] && (uint32_t)(ent[u] >> 32) >= lim) list[atomicAdd(&count, 1)] = ent[u];
        __syncthreads();
        list_cut(list, count, a.top, scratch);
    }
    finish(a, row, st, list);
    given<TY>(a, row, st, x);
}

struct LpPlan {
    int seg, per;
    size_t bytes;
};

// Segments of a row: one where the rows alone fill the chip, else until the grid has four blocks a CU.
LpPlan lp_plan(int rows, int vocab, int top) {
    LpPlan p;
    const int steps = (int)(((int64_t)vocab + 7 + LP_STEP - 1) / LP_STEP); // (with the longest lead)
    int seg = rows >= 512 ? 1 : std::min({(1024 + rows - 1) / std::max(rows, 1), steps, LP_MAX_SEG});
    seg = std::max(seg, 1);
    p.per = (steps + seg - 1) / seg;
    p.seg = std::max(1, (steps + p.per - 1) / p.per);
    p.bytes = p.seg > 1 ? (size_t)rows * p.seg * (16 + 8 * (size_t)top) : 0;
    return p;
}

} // namespace

extern "C" size_t llm_logprobs_work(int rows, int vocab, int top) {
    return rows > 0 && vocab > 0 && top >= 0 && top <= LP_TOP ? lp_plan(rows, vocab, top).bytes : 0;
}

hipError_t launch_logprobs(const LogprobsCall &q, hipStream_t st) {
    const int es = op_type_bytes(q.type);
    const LpPlan p = lp_plan(q.rows, q.vocab, q.top);
    LpArgs a;
    memset(&a, 0, sizeof a);
    a.x = (const uint8_t *)q.logits;
    a.stride = q.stride * es;
    a.rows = q.rows, a.vocab = q.vocab, a.seg = p.seg, a.per = p.per;
    a.inv_t = 1.0f / q.temperature;
    a.tokens = q.tokens, a.n_tokens = q.n_tokens, a.top = q.top;
    a.logp = q.logp, a.entropy = q.entropy, a.lse = q.lse, a.top_ids = q.top_ids, a.top_logp = q.top_logp;
    a.part = (float *)q.work;
    a.list = (uint64_t *)((float *)q.work + (size_t)q.rows * p.seg * 4);
    const bool f32 = q.type == LLM_F32;
    hipLaunchKernelGGL(f32 ? k_logprobs<LLM_F32> : k_logprobs<LLM_BF16>, dim3(q.rows * p.seg), dim3(LP_T), 0, st, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.seg == 1) return e;
    hipLaunchKernelGGL(f32 ? k_logprobs_join<LLM_F32> : k_logprobs_join<LLM_BF16>, dim3(q.rows), dim3(LP_T), 0, st, a);
    return hipGetLastError();
}

extern "C" int llm_logprobs(const void *logits, int type, int rows, int vocab, int64_t stride, float temperature,
                            const int *tokens, int n_tokens, float *logp, float *entropy, float *lse, int top, int *top_ids,
                            float *top_logp, void *work, size_t work_bytes, void *stream) {
    const char *who = "llm_logprobs";
    const int es = op_type_bytes(type);
    if ((type != LLM_F32 && type != LLM_BF16) || rows < 0 || vocab < 1 || vocab > 1 << 28 || (stride < vocab && rows > 1) ||
        !(temperature >= 1e-30f && temperature <= 1e30f) || n_tokens < 0 || top < 0 || top > LP_TOP || top > vocab ||
        ((uintptr_t)logits & (es - 1))) {
        fprintf(stderr, "%s: bad arguments (type %d, %d rows of %d logits, temperature %g, %d tokens, top %d)\n", who, type,
                rows, vocab, temperature, n_tokens, top);
        return -1;
    }
    if (!rows) return 0;
    OpDevice dev(who);
    if (!dev.holds(logits, "logits") || (n_tokens && (!dev.holds(tokens, "tokens") || !dev.holds(logp, "logp"))) ||
        (entropy && !dev.holds(entropy, "entropy")) || (lse && !dev.holds(lse, "lse")) ||
        (top && (!dev.holds(top_ids, "top_ids") || !dev.holds(top_logp, "top_logp"))))
        return -1;
    const LpPlan p = lp_plan(rows, vocab, top);
    if (p.bytes && (work_bytes < p.bytes || ((uintptr_t)work & 15) || !dev.holds(work, "the work memory"))) {
        fprintf(stderr, "%s: %zu bytes of work memory are needed, 16-byte aligned\n", who, p.bytes);
        return -1;
    }
    if ((int64_t)rows * p.seg > 0x7fffffff) {
        fprintf(stderr, "%s: %d rows\n", who, rows);
        return -1;
    }
    if (!dev.select()) return -1;
    const LogprobsCall q = {logits, type, rows, vocab, stride, temperature, tokens, n_tokens,
                            logp, entropy, lse, top, top_ids, top_logp, work};
    HIP_OR_FAIL(who, launch_logprobs(q, (hipStream_t)stream));
    return 0;
}
