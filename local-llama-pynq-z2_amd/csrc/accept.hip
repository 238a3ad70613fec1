// llm_draft_accept: drafted tokens kept or turned down against the target's probabilities.
//
// Three launches.  k_accept_rows reads every row of logits once: a workgroup takes a segment of a row into registers, finds its
// largest value and the sum of e^((x - largest) / T).  k_accept_walk joins them, walks the tree and sums the weights of the last node's
// row, a workgroup a segment: every workgroup of a sequence walks by itself, which needs no wait between them.  k_accept_draw
// finds the segment and the token that the drawn point falls into.
//
// What is left of p after a child was turned down: max(0, w / z - q) in proportion, w = max(0, p - a q), z the sum of w.  That is
// max(0, p - (a + z) q) / z: one number, a, says all that the tokens turned down have changed.
//
// Sums and exponentials are in 64 bits: a token drawn in the tail of 150k stands between borders 1e-6 apart, which an error of
// 2^-24 in the likeliest token's weight would all move by 6e-8.
#include <string.h>

#include <algorithm>

#include "device.h"
#include "operators.h"

namespace {

constexpr int AC_T = 256, AC_E = 16, AC_SEG = AC_T * AC_E; // values of a segment
constexpr int AC_N = 64;                                   // most nodes

struct AcPart { // of a segment: largest value, its first place (temperature 0), sum relative to it
    float m;
    int best;
    double s;
};
struct AcEnd { // of a sequence: the last node, its row's statistics, what is left of it
    int node, turned;
    float m;
    int best;
    double s, a;
    int out[AC_N]; // tokens turned down (no draft probabilities)
};
struct AcArgs {
    const uint8_t *x, *q;
    int64_t seq, row, p_seq, p_row; // bytes
    int max_n, vocab, segs;
    double inv_t; // 0: temperature 0
    const int *tokens, *parents, *n;
    const float *coins;
    int *kept, *path, *next;
    float *logp;
    AcPart *part; // [seq][row][segment]
    AcEnd *end;   // [seq]
    double *sums; // [seq][segment]
};

template <int TY>
__device__ __forceinline__ float at(const uint8_t *row, int i) {
    if constexpr (TY == LLM_F32) return ((const float *)row)[i];
    return __uint_as_float((uint32_t)((const uint16_t *)row)[i] << 16);
}
__device__ __forceinline__ int nodes(const AcArgs &a, int b) { return a.n ? min(max(a.n[b], 0), a.max_n) : a.max_n; }

__device__ __forceinline__ double wave_add(double v) { // in a fixed order
    for (int off = 1; off < 64; off <<= 1) v += __shfl_xor(v, off);
    return v;
}
// e^(x / T) relative to the largest value m of a row; temperature 0: 1 at `best`
__device__ __forceinline__ double weight(const AcArgs &a, float x, float m, int i, int best) {
    if (a.inv_t == 0.0) return i == best ? 1.0 : 0.0;
    return exp(((double)x - (double)m) * a.inv_t);
}

template <int TY>
__global__ void __launch_bounds__(AC_T) k_accept_rows(AcArgs a) {
    __shared__ float sm_m[AC_T / 64];
    __shared__ int sm_i[AC_T / 64];
    __shared__ double sm_s[AC_T / 64];
    const int seg = blockIdx.x, r = blockIdx.y, b = blockIdx.z, lane = threadIdx.x & 63, wave = threadIdx.x / 64;
    if (r >= nodes(a, b)) return;
    const uint8_t *row = a.x + b * a.seq + r * a.row;
    float x[AC_E], m = -INFINITY;
    bool nan = false;
#pragma unroll
    for (int e = 0; e < AC_E; e++) {
        const int i = seg * AC_SEG + e * AC_T + threadIdx.x;
        x[e] = i < a.vocab ? at<TY>(row, i) : -INFINITY;
        m = fmaxf(m, x[e]);
        nan |= x[e] != x[e];
    }
    m = wave_max(m);
    if (lane == 0) sm_m[wave] = m;
    __syncthreads();
    m = fmaxf(fmaxf(sm_m[0], sm_m[1]), fmaxf(sm_m[2], sm_m[3]));
    double s = 0.0;
    int best = 0x7fffffff;
    if (a.inv_t == 0.0) {
#pragma unroll
        for (int e = AC_E - 1; e >= 0; e--)
            if (x[e] == m) best = seg * AC_SEG + e * AC_T + threadIdx.x;
        s = nan || m == INFINITY ? __builtin_nan("") : 0.0;
    } else if (m > -INFINITY) {
#pragma unroll
        for (int e = 0; e < AC_E; e++) s += exp(((double)x[e] - (double)m) * a.inv_t);
    } else if (nan) {
        s = __builtin_nan("");
    }
    s = wave_add(s);
    for (int off = 1; off < 64; off <<= 1) best = min(best, __shfl_xor(best, off));
    if (lane == 0) sm_s[wave] = s, sm_i[wave] = best;
    __syncthreads();
    if (threadIdx.x == 0) {
        AcPart &p = a.part[((int64_t)b * a.max_n + r) * a.segs + seg];
        p.m = m;
        p.best = min(min(sm_i[0], sm_i[1]), min(sm_i[2], sm_i[3]));
        p.s = (sm_s[0] + sm_s[1]) + (sm_s[2] + sm_s[3]);
    }
}

// A row's segments joined by a wave: largest value, its first place, the sum (NaN: the row has no probabilities).
__device__ __forceinline__ void row_stats(const AcArgs &a, int b, int r, float &m, int &best, double &s) {
    const AcPart *p = a.part + ((int64_t)b * a.max_n + r) * a.segs;
    const int lane = threadIdx.x & 63;
    m = -INFINITY;
    for (int k = lane; k < a.segs; k += 64) m = fmaxf(m, p[k].m);
    m = wave_max(m);
    s = 0.0;
    best = 0x7fffffff;
    for (int k = lane; k < a.segs; k += 64) {
        if (a.inv_t == 0.0) {
            s += p[k].s; // (0 or NaN)
            if (p[k].m == m) best = min(best, p[k].best);
        } else if (p[k].m > -INFINITY || p[k].s != p[k].s) {
            s += p[k].s * exp(((double)p[k].m - (double)m) * a.inv_t);
        }
    }
    s = wave_add(s);
    for (int off = 1; off < 64; off <<= 1) best = min(best, __shfl_xor(best, off));
    if (a.inv_t == 0.0) s = s == 0.0 && m > -INFINITY ? 1.0 : __builtin_nan("");
    else if (!(s > 0.0)) s = __builtin_nan("");
}

// The weights of the thread's AC_E neighbouring values of a segment, in order.
template <int TY, int PT>
__device__ __forceinline__ void left_of(const AcArgs &a, const uint8_t *row, const uint8_t *probs, const AcEnd &e, int first,
                                        double (&w)[AC_E]) {
#pragma unroll
    for (int k = 0; k < AC_E; k++) {
        const int i = first + k;
        w[k] = 0.0;
        if (i >= a.vocab) continue;
        w[k] = weight(a, at<TY>(row, i), e.m, i, e.best) / e.s;
        if (PT >= 0 && e.a != 0.0) w[k] = fmax(w[k] - e.a * (double)at<PT>(probs, i), 0.0);
        if (PT < 0)
            for (int t = 0; t < e.turned; t++)
                if (e.out[t] == i) w[k] = 0.0;
    }
}

template <int TY, int PT> // PT: the type of the draft's probabilities, -1: none
__global__ void __launch_bounds__(AC_T) k_accept_walk(AcArgs a) {
    constexpr int PQ = PT < 0 ? LLM_F32 : PT;
    __shared__ float sm_m[AC_N];
    __shared__ int sm_best[AC_N], sm_parent[AC_N], sm_token[AC_N], sm_path[AC_N];
    __shared__ double sm_s[AC_N], sm_p[AC_N], sm_q[AC_N], sm_sum[AC_T / 64];
    __shared__ AcEnd end;
    const int seg = blockIdx.x, b = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x / 64, nn = nodes(a, b);
    const int64_t at0 = (int64_t)b * a.max_n;
    if (nn == 0) {
        if (seg == 0) {
            for (int i = threadIdx.x; i < a.max_n; i += AC_T) a.path[at0 + i] = -1, a.logp[at0 + i] = 0.0f;
            if (threadIdx.x == 0) a.kept[b] = 0, a.next[b] = -1;
        }
        return;
    }
    for (int r = wave; r < nn; r += AC_T / 64) {
        float m;
        int best;
        double s;
        row_stats(a, b, r, m, best, s);
        if (lane == 0) sm_m[r] = m, sm_best[r] = best, sm_s[r] = s;
    }
    __syncthreads();
    const uint8_t *const x = a.x + b * a.seq, *const q = PT >= 0 ? a.q + b * a.p_seq : nullptr;
    for (int i = threadIdx.x; i < a.max_n; i += AC_T) {
        float lp = 0.0f;
        int parent = -1, token = -1;
        if (i > 0 && i < nn) {
            parent = a.parents ? a.parents[at0 + i] : i - 1;
            if (parent < 0 || parent >= i) parent = -1;
            token = a.tokens[at0 + i];
            if (token < 0 || token >= a.vocab) token = -1;
            double p = 0.0;
            if (parent >= 0) {
                lp = -INFINITY;
                if (token >= 0) {
                    const float y = at<TY>(x + parent * a.row, token);
                    p = weight(a, y, sm_m[parent], token, sm_best[parent]) / sm_s[parent];
                    if (a.inv_t == 0.0) lp = p != p ? NAN : p > 0.0 ? 0.0f : -INFINITY;
                    else lp = (float)(((double)y - (double)sm_m[parent]) * a.inv_t - log(sm_s[parent]));
                    if (PT >= 0) sm_q[i] = (double)at<PQ>(q + parent * a.p_row, token);
                }
            }
            sm_p[i] = p;
        }
        if (i < AC_N) sm_parent[i] = parent, sm_token[i] = token;
        if (seg == 0 && i > 0) a.logp[at0 + i] = lp;
    }
    __syncthreads();
    // the walk, by all threads alike
    int node = 0, kept = 1, turned = 0;
    double left = 1.0, aq = 0.0;
    for (int i = 1; i < nn; i++) {
        if (sm_parent[i] != node || sm_token[i] < 0) continue;
        const double u = (double)a.coins[at0 + i];
        double w = sm_p[i];
        bool takes;
        if (PT >= 0) {
            w = fmax(w - aq * sm_q[i], 0.0);
            takes = u * sm_q[i] * left < w;
        } else {
            for (int t = 0; t < turned; t++)
                if (end.out[t] == sm_token[i]) w = 0.0;
            takes = u * left < w;
        }
        if (takes) {
            if (threadIdx.x == 0) sm_path[kept] = i;
            node = i, left = 1.0, aq = 0.0, turned = 0;
            kept++;
            continue;
        }
        if (PT >= 0) {
            aq += left;
            bool more = false; // another child to hold against what is left
            for (int k = i + 1; k < nn; k++) more |= sm_parent[k] == node && sm_token[k] >= 0;
            if (more) {
                const uint8_t *row = x + node * a.row, *probs = q + node * a.p_row;
                double s = 0.0;
                for (int k = threadIdx.x; k < a.vocab; k += AC_T)
                    s += fmax(weight(a, at<TY>(row, k), sm_m[node], k, sm_best[node]) / sm_s[node] -
                                  aq * (double)at<PQ>(probs, k), 0.0);
                s = wave_add(s);
                __syncthreads();
                if (lane == 0) sm_sum[wave] = s;
                __syncthreads();
                left = (sm_sum[0] + sm_sum[1]) + (sm_sum[2] + sm_sum[3]);
            }
        } else {
            left = fmax(left - w, 0.0);
            __syncthreads();
            if (threadIdx.x == 0) end.out[turned] = sm_token[i];
            turned++;
            __syncthreads();
        }
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        sm_path[0] = 0;
        end.node = node, end.turned = turned, end.m = sm_m[node], end.best = sm_best[node], end.s = sm_s[node], end.a = aq;
    }
    __syncthreads();
    if (seg == 0) {
        for (int i = threadIdx.x; i < a.max_n; i += AC_T) a.path[at0 + i] = i < kept ? sm_path[i] : -1;
        if (threadIdx.x == 0) {
            a.kept[b] = kept;
            a.end[b] = end;
        }
    }
    double w[AC_E], s = 0.0;
    left_of<TY, PT>(a, x + node * a.row, PT >= 0 ? q + node * a.p_row : nullptr, end, seg * AC_SEG + threadIdx.x * AC_E, w);
#pragma unroll
    for (int k = 0; k < AC_E; k++) s += w[k];
    s = wave_add(s);
    if (lane == 0) sm_sum[wave] = s;
    __syncthreads();
    if (threadIdx.x == 0) a.sums[(int64_t)b * a.segs + seg] = (sm_sum[0] + sm_sum[1]) + (sm_sum[2] + sm_sum[3]);
}

template <int TY, int PT>
__global__ void __launch_bounds__(AC_T) k_accept_draw(AcArgs a) {
    __shared__ AcEnd end;
    __shared__ double sm_sum[AC_T / 64];
    __shared__ double sm_before;
    __shared__ int sm_seg, sm_at, sm_last;
    const int b = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x / 64;
    if (nodes(a, b) == 0) return;
    if (threadIdx.x == 0) end = a.end[b], sm_at = 0x7fffffff, sm_last = -1;
    __syncthreads();
    const int64_t at0 = (int64_t)b * a.max_n;
    const double *sums = a.sums + (int64_t)b * a.segs;
    const AcPart *part = a.part + (at0 + end.node) * a.segs;
    double u = 0.0;
    if (threadIdx.x == 0) {
        double all = 0.0;
        for (int k = 0; k < a.segs; k++) all += sums[k];
        bool whole = false; // nothing is left: the target's own row
        auto sum_of = [&](int k) {
            if (!whole) return sums[k];
            if (a.inv_t == 0.0) return end.best / AC_SEG == k ? 1.0 : 0.0;
            return part[k].m > -INFINITY ? part[k].s * exp(((double)part[k].m - (double)end.m) * a.inv_t) / end.s : 0.0;
        };
        if (all == 0.0) {
            whole = true;
            for (int k = 0; k < a.segs; k++) all += sum_of(k);
            end.a = 0.0, end.turned = 0;
        }
        double before = 0.0;
        int seg = -1;
        if (all > 0.0) {
            u = (double)a.coins[at0] * all;
            for (seg = 0; seg < a.segs - 1; seg++) {
                const double s = sum_of(seg);
                if (before + s > u) break;
                before += s;
            }
            while (seg > 0 && sum_of(seg) == 0.0) before -= sum_of(--seg); // (the last segments may have nothing)
        }
        sm_seg = seg;
        sm_before = before;
        sm_sum[0] = u;
    }
    __syncthreads();
    const int seg = sm_seg;
    u = sm_sum[0];
    if (seg < 0) {
        if (threadIdx.x == 0) a.next[b] = -1, a.logp[at0] = NAN;
        return;
    }
    __syncthreads();
    const uint8_t *row = a.x + b * a.seq + end.node * a.row;
    double w[AC_E], s = 0.0;
    const int first = seg * AC_SEG + threadIdx.x * AC_E;
    left_of<TY, PT>(a, row, PT >= 0 ? a.q + b * a.p_seq + end.node * a.p_row : nullptr, end, first, w);
#pragma unroll
    for (int k = 0; k < AC_E; k++) s += w[k];
    double upto = s;
    for (int off = 1; off < 64; off <<= 1) {
        const double y = __shfl_up(upto, off);
        upto += lane >= off ? y : 0.0;
    }
    if (lane == 63) sm_sum[wave] = upto;
    __syncthreads();
    double c = sm_before + (upto - s);
    for (int k = 0; k < wave; k++) c += sm_sum[k];
    int found = 0x7fffffff, last = -1;
#pragma unroll
    for (int k = 0; k < AC_E; k++) {
        c += w[k];
        if (w[k] > 0.0) {
            last = first + k;
            if (c > u && found == 0x7fffffff) found = first + k;
        }
    }
    if (found != 0x7fffffff) atomicMin(&sm_at, found);
    if (last >= 0) atomicMax(&sm_last, last);
    __syncthreads();
    if (threadIdx.x == 0) {
        const int token = sm_at != 0x7fffffff ? sm_at : sm_last; // (a point at the end, by rounding)
        a.next[b] = token;
        if (token < 0) { // (draft probabilities that are not finite)
            a.logp[at0] = NAN;
            return;
        }
        double lp = 0.0;
        if (a.inv_t != 0.0) lp = ((double)at<TY>(row, token) - (double)end.m) * a.inv_t - log(end.s);
        else if (token != end.best) lp = -INFINITY;
        a.logp[at0] = (float)lp;
    }
}

int64_t ac_segs(int vocab) { return ((int64_t)vocab + AC_SEG - 1) / AC_SEG; }

} // namespace

extern "C" size_t llm_draft_accept_work(int n_seq, int max_n, int vocab) {
    if (n_seq < 1 || max_n < 1 || max_n > AC_N || vocab < 1) return 0;
    const size_t segs = ac_segs(vocab);
    return (size_t)n_seq * (max_n * segs * sizeof(AcPart) + sizeof(AcEnd) + segs * sizeof(double));
}

extern "C" int llm_draft_accept(const void *logits, int type, int n_seq, int max_n, int vocab, int64_t seq, int64_t row,
                                float temperature, const void *probs, int p_type, int64_t p_seq, int64_t p_row,
                                const int *tokens, const int *parents, const int *n, const float *coins, int *kept, int *path,
                                int *next, float *logp, void *work, size_t work_bytes, void *stream) {
    const char *who = "llm_draft_accept";
    auto typed = [](int t) { return t == LLM_F32 || t == LLM_BF16; };
    if (!typed(type) || (probs && !typed(p_type)) || n_seq < 0 || n_seq > 65535 || max_n < 0 || max_n > AC_N || vocab < 1 ||
        vocab > 1 << 28 || !(temperature == 0.0f || (temperature >= 1e-30f && temperature <= 1e30f)) || seq < 0 || row < 0 ||
        (probs && (p_seq < 0 || p_row < 0)) || ((uintptr_t)logits & (op_type_bytes(type) - 1)) ||
        (probs && ((uintptr_t)probs & (op_type_bytes(p_type) - 1)))) {
        fprintf(stderr, "%s: bad arguments (type %d, %d sequences of %d nodes (at most %d), %d logits, temperature %g)\n", who,
                type, n_seq, max_n, AC_N, vocab, temperature);
        return -1;
    }
    if (!n_seq || !max_n) return 0;
    OpDevice dev(who);
    if (!dev.holds(logits, "logits") || (probs && !dev.holds(probs, "probs")) || !dev.holds(tokens, "tokens") ||
        (parents && !dev.holds(parents, "parents")) || (n && !dev.holds(n, "n")) || !dev.holds(coins, "coins") ||
        !dev.holds(kept, "kept") || !dev.holds(path, "path") || !dev.holds(next, "next") || !dev.holds(logp, "logp"))
        return -1;
    const size_t need = llm_draft_accept_work(n_seq, max_n, vocab);
    if (work_bytes < need || ((uintptr_t)work & 15) || !dev.holds(work, "the work memory")) {
        fprintf(stderr, "%s: %zu bytes of work memory are needed, 16-byte aligned\n", who, need);
        return -1;
    }
    if (!dev.select()) return -1;
    const int xs = op_type_bytes(type), ps = probs ? op_type_bytes(p_type) : 0;
    AcArgs a;
    memset(&a, 0, sizeof a);
    a.x = (const uint8_t *)logits, a.q = (const uint8_t *)probs;
    a.seq = seq * xs, a.row = row * xs, a.p_seq = p_seq * ps, a.p_row = p_row * ps;
    a.max_n = max_n, a.vocab = vocab, a.segs = (int)ac_segs(vocab);
    a.inv_t = temperature == 0.0f ? 0.0 : 1.0 / (double)temperature;
    a.tokens = tokens, a.parents = parents, a.n = n, a.coins = coins;
    a.kept = kept, a.path = path, a.next = next, a.logp = logp;
    a.part = (AcPart *)work;
    a.end = (AcEnd *)(a.part + (size_t)n_seq * max_n * a.segs);
    a.sums = (double *)(a.end + n_seq);
    hipStream_t st = (hipStream_t)stream;
    const bool f32 = type == LLM_F32;
    hipLaunchKernelGGL(f32 ? k_accept_rows<LLM_F32> : k_accept_rows<LLM_BF16>, dim3(a.segs, max_n, n_seq), dim3(AC_T), 0, st, a);
    HIP_OR_FAIL(who, hipGetLastError());
    void (*walk)(AcArgs) = nullptr, (*draw)(AcArgs) = nullptr;
    const int pt = probs ? p_type : -1;
#define ACCEPT_PICK(T, P) \
    if (type == T && pt == P) walk = k_accept_walk<T, P>, draw = k_accept_draw<T, P>;
    ACCEPT_PICK(LLM_F32, -1) ACCEPT_PICK(LLM_F32, LLM_F32) ACCEPT_PICK(LLM_F32, LLM_BF16)
    ACCEPT_PICK(LLM_BF16, -1) ACCEPT_PICK(LLM_BF16, LLM_F32) ACCEPT_PICK(LLM_BF16, LLM_BF16)
#undef ACCEPT_PICK
    hipLaunchKernelGGL(walk, dim3(a.segs, n_seq), dim3(AC_T), 0, st, a);
    HIP_OR_FAIL(who, hipGetLastError());
    hipLaunchKernelGGL(draw, dim3(n_seq), dim3(AC_T), 0, st, a);
    HIP_OR_FAIL(who, hipGetLastError());
    return 0;
}
