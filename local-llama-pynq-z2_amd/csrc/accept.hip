// llm_draft_accept: drafted tokens kept or turned down against the target's probabilities.
//
// k_accept_rows reads every row of logits once: a workgroup takes a segment of a row into registers, finds its largest value and
// the sum of e^((x - largest) / T).  k_accept_walk joins them, walks the tree and sums the weights of the last node's row, a
// workgroup a segment: every workgroup of a sequence walks by itself, which needs no wait between them, and the last one to be done
// finds the segment and the token that the drawn point falls into.
//
// What is left of p after a child was turned down: max(0, w / z - q) in proportion, w = max(0, p - a q), z the sum of w.  That is
// max(0, p - (a + z) q) / z: one number, a, says all that the tokens turned down have changed.
//
// Sums and exponentials that decide are in 64 bits: a token drawn in the tail of 150k stands between borders 1e-6 apart, which an
// error of 2^-24 in the likeliest token's weight would all move by 6e-8.
//
// What bounds it: the rows' bytes, read once.  16 trees of up to 37 rows of 151936 bf16 logits, 154 MB: 25.5 us, 6.0 TB/s, for
// the rows (the last call left a part of them in the caches) and 17.0 for the walk; a chain of 6 fp32 rows with draft
// probabilities: 4.1 and 10.7.  The walk is a chain of short steps (of that chain, in thousands of cycles: the parts' loads and
// join and the tokens' probabilities 5.6, the walk 1.5, a segment's sum 7.6, the count 1.6, the choice of a segment 2.2, of a
// token 3.5), each code that runs once: fetching it is a part of the time.  Trees with draft probabilities need a row's pass for
// each child with a later sibling that is turned down: see k_accept_ask; trees without where a likely one is: see rest_of.
#include <string.h>

#include <algorithm>

#include "device.h"
#include "operators.h"

namespace {

constexpr int AC_T = 256, AC_E = 16, AC_SEG = AC_T * AC_E; // values of a segment
constexpr int AC_N = 64;                                   // most nodes: a lane each
// Least vocabulary for k_accept_ask and k_accept_left, three launches of 7 us together: a single tree of 20 nodes over 32000
// logits 27 us with them and 19 (nothing is asked for) or 36 without, over 151936 33 and 95, 16 trees of 37 over 8192 logits 38
// and 28, over 16384 43 and 40, over 32000 60 and 79, over 151936 117 and 290 (all fp32).
constexpr int AC_ASK = 16384;

struct AcPart { // of a part of a row: largest value, its first place (temperature 0), sum relative to it
    float m;
    int best;
    double s;
};
struct AcEnd { // a sequence's last node, its row's statistics, what is left of it
    int node, turned;
    float m;
    int best;
    double s, inv, a; // inv: 1 / s
    int out[AC_N]; // tokens turned down (no draft probabilities)
};
struct AcAsk { // a node whose first child is turned down and not its last one; its row's statistics; the second child
    int node, more, best; // more: there is a third
    float m;
    double inv, p, q, coin;
};
struct AcArgs {
    const uint8_t *x, *q;
    int64_t seq, row, p_seq, p_row; // bytes
    int max_n, vocab, segs, parts; // parts: workgroups of a row in k_accept_rows
    double c; // log2(e) / T; 0: temperature 0
    const int *tokens, *parents, *n;
    const float *coins;
    int *kept, *path, *next;
    float *logp;
    AcPart *part; // [seq][row][part]
    double *sums, *shares; // [seq][segment], [seq][segment][thread]
    int *done;    // [seq]: segments that are summed
    AcAsk *asks;  // [seq][max_n]
    int *count;   // [seq]: of them
    double *left; // [seq][node][0, 1][segment]: what is left after the node's first and second child; NULL: not known
};

template <int TY>
__device__ __forceinline__ float at(const uint8_t *row, int i) {
    if constexpr (TY == LLM_F32) return ((const float *)row)[i];
    return __uint_as_float((uint32_t)((const uint16_t *)row)[i] << 16);
}
// Neighbouring values from i on (16 bytes; a row starts anywhere), `none` behind the row's end.
template <int TY>
constexpr int AC_V = TY == LLM_F32 ? 4 : 8;
template <int TY, bool ALL = false> // ALL: they are in the row, all of the wave's
__device__ __forceinline__ void values(const uint8_t *row, int i, int vocab, float none, float *x) {
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4), aligned(2)));
    constexpr int V = AC_V<TY>;
    if (ALL || i + V <= vocab) {
        const u32x4 u = *(const u32x4 *)(row + (size_t)i * (TY == LLM_F32 ? 4 : 2));
#pragma unroll
        for (int k = 0; k < V; k++)
            x[k] = TY == LLM_F32 ? __uint_as_float(u[k % 4]) : __uint_as_float(k % 2 ? u[k / 2] & 0xffff0000u : u[k / 2] << 16);
    } else {
#pragma unroll
        for (int k = 0; k < V; k++) x[k] = i + k < vocab ? at<TY>(row, i + k) : none;
    }
}
__device__ __forceinline__ int nodes(const AcArgs &a, int b) { return a.n ? min(max(a.n[b], 0), a.max_n) : a.max_n; }

// 2^y for y <= 0 (below -1020, and NaN: 2^-1020): y = n + f, f in [-1/2, 1/2], and 2^f = e^(f ln 2) by its series up to the tenth
// power, whose next term is below (ln 2 / 2)^11 / 11! = 2.2e-13.  Adding 1.5 2^52 rounds to whole numbers and leaves n in the sum's
// low bits, from where it goes into the exponent: no instruction of less than full rate.
__device__ __forceinline__ double exp2_of(double y) {
    constexpr double WHOLE = 6755399441055744.0, L = 0.693147180559945309417232121458;
    y = fmax(y, -1020.0);
    const double t = y + WHOLE, f = y - (t - WHOLE);
    constexpr double L2 = L * L, L4 = L2 * L2, L8 = L4 * L4;
    constexpr double k[] = {L8 * L / 362880.0, L8 / 40320.0, L4 * L2 * L / 5040.0, L4 * L2 / 720.0, L4 * L / 120.0, L4 / 24.0,
                            L2 * L / 6.0, L2 / 2.0, L, 1.0};
    double p = L8 * L2 / 3628800.0;
#pragma unroll
    for (double c : k) p = fma(p, f, c);
    const uint64_t u = __builtin_bit_cast(uint64_t, p);
    const uint32_t n = (uint32_t)__builtin_bit_cast(uint64_t, t);
    return __builtin_bit_cast(double, (uint64_t)((uint32_t)(u >> 32) + (n << 20)) << 32 | (uint32_t)u);
}
// e^(x / T) relative to the largest value m of a row, c = log2(e) / T.  A masked logit's is 0, not nearly 0: by a product, since a
// branch would keep the series of neighbouring values from being worked on together.
__device__ __forceinline__ double weight(float x, double m, double c) {
    const double y = ((double)x - m) * c; // (an exact difference: 1 / T may be large)
    return exp2_of(y) * (y >= -1020.0 ? 1.0 : 0.0);
}
// The same of one value; temperature 0: 1 at `best`.
__device__ __forceinline__ double weight_of(const AcArgs &a, float x, float m, int i, int best) {
    return a.c == 0.0 ? i == best ? 1.0 : 0.0 : weight(x, (double)m, a.c);
}

// A double through a DPP operand (lanes without a source, and rows that ROWS leaves out: 0).
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ double dpp64(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)u, CTRL, ROWS, 0xf, false);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(u >> 32), CTRL, ROWS, 0xf, false);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double lane_of(double v, int i) { // i: uniform
    const uint64_t w = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(double, (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(w >> 32), i) << 32 |
                                          (uint32_t)__builtin_amdgcn_readlane((int)w, i));
}
template <int W> // over W neighbouring lanes, 16 or 64, in a fixed order: lane ^ 1, ^ 2, mirrors of 8 and 16, then rows of 16
__device__ __forceinline__ double lanes_add(double v) {
    v += dpp64<0xB1>(v);
    v += dpp64<0x4E>(v);
    v += dpp64<0x141>(v);
    v += dpp64<0x140>(v);
    return W == 16 ? v : (lane_of(v, 0) + lane_of(v, 16)) + (lane_of(v, 32) + lane_of(v, 48));
}
__device__ __forceinline__ double block_add(double v, double *sm) {
    v = lanes_add<64>(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sm[threadIdx.x / 64] = v;
    __syncthreads();
    return (sm[0] + sm[1]) + (sm[2] + sm[3]);
}
__device__ __forceinline__ double upto(double v) { // inclusive sum over a wave: row_shr 1, 2, 4, 8, row_bcast 15, 31
    v += dpp64<0x111>(v);
    v += dpp64<0x112>(v);
    v += dpp64<0x114>(v);
    v += dpp64<0x118>(v);
    v += dpp64<0x142, 0xa>(v);
    v += dpp64<0x143, 0xc>(v);
    return v;
}

// PER segments of a row a workgroup: one where there are few rows, four else (the walk has a quarter to join).
// EXACT: exponentials in 64 bits, for draft probabilities, which are held against p itself; without them a row's sum only decides
// about its children and log probabilities, and it takes those of the hardware in 32 bits: off by 2^-18 of itself for rows up to
// 2^22 (three roundings of the exponent, the instruction's, eight chains of additions); what is drawn from is summed in 64 bits by
// the walk.  A call of 16 trees of 37 bf16 rows: 43 us, with the series in 64 bits 80.
template <int TY, int PER, bool EXACT>
__global__ void __launch_bounds__(AC_T) k_accept_rows(AcArgs a) {
    constexpr int V = AC_V<TY>, E = AC_E * PER;
    __shared__ float sm_m[AC_T / 64];
    __shared__ int sm_i[AC_T / 64];
    __shared__ double sm_s[AC_T / 64];
    const int seg = blockIdx.x, r = blockIdx.y, b = blockIdx.z, lane = threadIdx.x & 63, wave = threadIdx.x / 64;
    if (seg == 0 && r == 0 && threadIdx.x == 0) a.done[b] = 0;
    if (r >= nodes(a, b)) return;
    const uint8_t *row = a.x + b * a.seq + r * a.row;
    auto index = [&](int e) { return seg * (PER * AC_SEG) + (e / V * AC_T + (int)threadIdx.x) * V + e % V; };
    float x[E], m = -INFINITY;
    bool nan = false;
    if ((seg + 1) * (PER * AC_SEG) <= a.vocab)
#pragma unroll
        for (int e = 0; e < E; e += V) values<TY, true>(row, index(e), a.vocab, -INFINITY, x + e);
    else
#pragma unroll
        for (int e = 0; e < E; e += V) values<TY, false>(row, index(e), a.vocab, -INFINITY, x + e);
#pragma unroll
    for (int e = 0; e < E; e++) {
        m = fmaxf(m, x[e]);
        nan |= x[e] != x[e];
    }
    m = wave_max(m);
    if (lane == 0) sm_m[wave] = m;
    __syncthreads();
    m = fmaxf(fmaxf(sm_m[0], sm_m[1]), fmaxf(sm_m[2], sm_m[3]));
    double s = 0.0;
    int best = 0x7fffffff;
    if (a.c == 0.0) {
#pragma unroll
        for (int e = 0; e < E; e++)
            if (x[e] == m) best = min(best, index(e));
        for (int off = 1; off < 64; off <<= 1) best = min(best, __shfl_xor(best, off));
    } else if (m > -INFINITY && m < INFINITY) {
        if constexpr (EXACT) {
#pragma unroll
            for (int e = 0; e < E; e++) s += exp2_of(((double)x[e] - (double)m) * a.c);
        } else {
            const float c = (float)a.c;
            float f[8] = {}; // (eight chains: a sum is off by 2^-21 of itself at most)
#pragma unroll
            for (int e = 0; e < E; e++) f[e % 8] += __builtin_amdgcn_exp2f((x[e] - m) * c);
#pragma unroll
            for (int k = 0; k < 8; k++) s += (double)f[k];
        }
    }
    if (nan || m == INFINITY) s = __builtin_nan(""); // (the row has no probabilities)
    s = lanes_add<64>(s);
    if (lane == 0) sm_s[wave] = s, sm_i[wave] = best;
    __syncthreads();
    if (threadIdx.x == 0) {
        AcPart &p = a.part[((int64_t)b * a.max_n + r) * a.parts + seg];
        p.m = m;
        p.best = min(min(sm_i[0], sm_i[1]), min(sm_i[2], sm_i[3]));
        p.s = (sm_s[0] + sm_s[1]) + (sm_s[2] + sm_s[3]);
    }
}

// A row's parts joined by 16 neighbouring lanes: largest value, its first place, the sum (NaN: no probabilities).
struct AcRow {
    static constexpr int U = 4; // parts of a lane at once
    AcPart p[U];
    __device__ __forceinline__ void load(const AcArgs &a, int b, int r, int k0) {
        const AcPart *from = a.part + ((int64_t)b * a.max_n + r) * a.parts;
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int k = k0 + 16 * u + (threadIdx.x & 15);
            p[u] = from[min(k, a.parts - 1)];
            if (k >= a.parts) p[u].m = -INFINITY, p[u].s = 0.0, p[u].best = 0x7fffffff;
        }
    }
    __device__ __forceinline__ void join(const AcArgs &a, int b, int r, float &m, int &best, double &s) {
        m = -INFINITY, s = 0.0, best = 0x7fffffff;
        for (int k0 = 0;;) {
            float top = m;
#pragma unroll
            for (int u = 0; u < U; u++) top = fmaxf(top, p[u].m);
            top = max16(top);
            auto scaled = [&](float mk, double sk) { // (0 and NaN stay what they are)
                return a.c == 0.0 || !(mk > -INFINITY) ? sk : sk * exp2_of(((double)mk - (double)top) * a.c);
            };
            s = scaled(m, s);
            if (top != m) best = 0x7fffffff;
#pragma unroll
            for (int u = 0; u < U; u++) {
                s += scaled(p[u].m, p[u].s);
                if (p[u].m == top) best = min(best, p[u].best);
            }
            m = top;
            k0 += 16 * U;
            if (k0 >= a.parts) break;
            load(a, b, r, k0);
        }
        s = lanes_add<16>(s);
        if (a.c == 0.0) {
#pragma unroll
            for (int off = 1; off < 16; off <<= 1) best = min(best, __shfl_xor(best, off));
            s = s == 0.0 && m > -INFINITY ? 1.0 : __builtin_nan("");
        } else if (!(s > 0.0)) {
            s = __builtin_nan("");
        }
    }
};

// log2(s) for s >= 1: the hardware's, and what it is short of.
__device__ __forceinline__ double log2_of(double s) {
    const double l = (double)__builtin_amdgcn_logf((float)s);
    return l + (s * exp2_of(-l) - 1.0) * 1.44269504088896340736;
}

// What is left of N neighbouring values from `first` on: x their logits (-infinity behind the row), q the draft's probabilities.
// A draft probability that is not finite leaves 0 for the test of a child (Z), NaN for the draw, which then has none.
template <int PT, bool Z, int N>
__device__ __forceinline__ void left_of(const AcArgs &a, const AcEnd &e, const float *x, const float *q, int first, double (&w)[N]) {
    const double m = (double)e.m, inv = e.inv, aq = e.a;
    if (a.c == 0.0) {
#pragma unroll
        for (int k = 0; k < N; k++) w[k] = first + k == e.best ? inv : inv - inv; // (NaN: no probabilities)
    } else {
#pragma unroll
        for (int k = 0; k < N; k++) w[k] = weight(x[k], m, a.c) * inv;
    }
    if (PT >= 0 && aq != 0.0)
#pragma unroll
        for (int k = 0; k < N; k++) {
            const double d = w[k] - aq * (double)q[k];
            w[k] = Z ? fmax(d, 0.0) : d < 0.0 ? 0.0 : d;
        }
    if (PT < 0)
        for (int t = 0; t < e.turned; t++) {
            const int at = e.out[t] - first;
#pragma unroll
            for (int k = 0; k < N; k++) w[k] = at == k ? 0.0 : w[k];
        }
}
// Its sum over the thread's AC_E neighbouring values of a segment, in order.  All loads go out first; the weights are a loop of
// four at a time, whose values move up: straight code, and no more of it than is run often enough to have been worth fetching
// (sixteen values in a row with branches for their masks and borders: 4 us more for the walk of sixteen trees over 151936 bf16
// logits).
template <int TY, int PT, bool Z>
__device__ __forceinline__ double left_sum(const AcArgs &a, const uint8_t *row, const uint8_t *probs, const AcEnd &e, int seg) {
    constexpr int PQ = PT < 0 ? LLM_F32 : PT;
    const int first = seg * AC_SEG + threadIdx.x * AC_E;
    float x[AC_E], q[AC_E];
#pragma unroll
    for (int k = 0; k < AC_E; k++) q[k] = 0.0f;
    if ((seg + 1) * AC_SEG <= a.vocab) {
#pragma unroll
        for (int k = 0; k < AC_E; k += AC_V<TY>) values<TY, true>(row, first + k, a.vocab, -INFINITY, x + k);
        if (PT >= 0)
#pragma unroll
            for (int k = 0; k < AC_E; k += AC_V<PQ>) values<PQ, true>(probs, first + k, a.vocab, 0.0f, q + k);
    } else {
#pragma unroll
        for (int k = 0; k < AC_E; k += AC_V<TY>) values<TY, false>(row, first + k, a.vocab, -INFINITY, x + k);
        if (PT >= 0)
#pragma unroll
            for (int k = 0; k < AC_E; k += AC_V<PQ>) values<PQ, false>(probs, first + k, a.vocab, 0.0f, q + k);
    }
    double s = 0.0;
#pragma unroll 1
    for (int k = 0; k < AC_E; k += 4) {
        double w[4];
        left_of<PT, Z>(a, e, x, q, first + k, w);
#pragma unroll
        for (int j = 0; j < 4; j++) s += w[j];
#pragma unroll
        for (int j = 0; j < AC_E - 4; j++) {
            x[j] = x[j + 4];
            q[j] = q[j + 4];
        }
    }
    return s;
}

// What a lane knows of its node: every wave alike.
struct AcNode {
    int parent, token; // -1: none
    float y, u;        // the token's logit after its parent; the coin
    double q, p;       // its probabilities: the draft's, the target's
};
// Of nn nodes, and their rows' statistics in LDS.
template <int TY, int PT>
__device__ __forceinline__ AcNode node_of(const AcArgs &a, int b, int nn, const uint8_t *x, const uint8_t *q, float *sm_m,
                                          int *sm_best, double *sm_s) {
    constexpr int PQ = PT < 0 ? LLM_F32 : PT;
    const int lane = threadIdx.x & 63;
    const int64_t at0 = (int64_t)b * a.max_n;
    AcRow rows; // (every load that depends on no other first)
    rows.load(a, b, min((int)threadIdx.x / 16, nn - 1), 0);
    AcNode d = {-1, -1, 0.0f, 0.0f, 0.0, 0.0};
    if (lane < nn) {
        d.u = a.coins[at0 + lane];
        d.parent = a.parents ? a.parents[at0 + lane] : lane - 1;
        d.token = a.tokens[at0 + lane];
    }
    if (lane == 0 || d.parent < 0 || d.parent >= lane) d.parent = -1;
    if (lane == 0 || d.token < 0 || d.token >= a.vocab) d.token = -1;
    const bool is = d.parent >= 0 && d.token >= 0;
    if (is) {
        d.y = at<TY>(x + d.parent * a.row, d.token);
        if (PT >= 0) d.q = (double)at<PQ>(q + d.parent * a.p_row, d.token);
    }
    for (int r = threadIdx.x / 16; r - (int)threadIdx.x / 16 < nn; r += AC_T / 16) {
        float m;
        int best;
        double s;
        rows.join(a, b, min(r, nn - 1), m, best, s);
        if (r < nn && (threadIdx.x & 15) == 0) sm_m[r] = m, sm_best[r] = best, sm_s[r] = s;
        rows.load(a, b, min(r + AC_T / 16, nn - 1), 0);
    }
    __syncthreads();
    if (is) d.p = weight_of(a, d.y, sm_m[d.parent], d.token, sm_best[d.parent]) / sm_s[d.parent];
    return d;
}

// What was turned down of trees with draft probabilities changes what is left of its parent's row by the number of children
// alone: after the first a is 1, after the second 1 + z.  A pass over a row within the walk is every workgroup's own; so z of
// every row that the walk may need it of is summed before, a workgroup a segment: k_accept_ask lists the nodes that may be
// reached, whose first child is turned down and not the last, k_accept_left sums what is left after the first child and, launched
// again, after the second.  Third children's are left to the walk.
template <int TY, int PT>
__global__ void __launch_bounds__(AC_T) k_accept_ask(AcArgs a) {
    __shared__ float sm_m[AC_N];
    __shared__ int sm_best[AC_N];
    __shared__ double sm_s[AC_N];
    const int b = blockIdx.x, lane = threadIdx.x & 63, nn = nodes(a, b);
    if (nn == 0) {
        if (threadIdx.x == 0) a.count[b] = 0;
        return;
    }
    const AcNode d = node_of<TY, PT>(a, b, nn, a.x + b * a.seq, a.q + b * a.p_seq, sm_m, sm_best, sm_s);
    if (threadIdx.x >= 64) return;
    const bool is = d.parent >= 0 && d.token >= 0;
    // as the walk decides about a first child
    const uint64_t takes = __ballot(is && (double)d.u * d.q * 1.0 < fmax(d.p - 0.0 * d.q, 0.0)), all = __ballot(is);
    uint64_t kids = 0; // the node's
    for (uint64_t left = all; left; left &= left - 1) {
        const int i = __ffsll((unsigned long long)left) - 1;
        if (__builtin_amdgcn_readlane(d.parent, i) == lane) kids |= (uint64_t)1 << i;
    }
    const int first = kids ? __ffsll((unsigned long long)kids) - 1 : lane;
    const int eldest = __shfl(first, max(d.parent, 0)); // the first child of the node's parent
    const uint64_t ok = __ballot(is && ((takes >> eldest) & 1) == (uint64_t)(lane == eldest));
    uint64_t reach = 1;
    for (uint64_t left = ok; left; left &= left - 1) {
        const int i = __ffsll((unsigned long long)left) - 1;
        reach |= ((reach >> __builtin_amdgcn_readlane(d.parent, i)) & 1) << i;
    }
    const uint64_t others = kids & (kids - 1);
    const bool asks = others && !((takes >> first) & 1) && ((reach >> lane) & 1);
    const uint64_t list = __ballot(asks);
    const int second = others ? __ffsll((unsigned long long)others) - 1 : 0;
    const double p = __shfl(d.p, second), q = __shfl(d.q, second);
    const float coin = __shfl(d.u, second);
    if (asks) {
        AcAsk &k = a.asks[(int64_t)b * a.max_n + __popcll(list & (((uint64_t)1 << lane) - 1))];
        k = {lane, (others & (others - 1)) != 0, sm_best[lane], sm_m[lane], 1.0 / sm_s[lane], p, q, (double)coin};
    }
    if (lane == 0) a.count[b] = __popcll(list);
}

// z of a node after its first (round 0) or second (1) child, by a whole wave.
__device__ __forceinline__ double z_of(const AcArgs &a, int b, int node, int round) {
    const double *from = a.left + (((int64_t)b * a.max_n + node) * 2 + round) * a.segs;
    double z = 0.0;
    for (int k = threadIdx.x & 63; k < a.segs; k += 64) z += from[k];
    return lanes_add<64>(z);
}

template <int TY, int PT>
__global__ void __launch_bounds__(AC_T) k_accept_left(AcArgs a, int round) {
    __shared__ double sm_sum[AC_T / 64];
    const int seg = blockIdx.x, b = blockIdx.z, count = a.count[b];
    for (int i = blockIdx.y; i < count; i += gridDim.y) {
        const AcAsk &k = a.asks[(int64_t)b * a.max_n + i];
        const int node = k.node;
        AcEnd e;
        e.turned = 0, e.m = k.m, e.best = k.best, e.inv = k.inv, e.a = 1.0;
        if (round) {
            if (!k.more) continue;
            const double z = z_of(a, b, node, 0);
            if (k.coin * k.q * z < fmax(k.p - k.q, 0.0)) continue; // (as the walk decides)
            e.a += z;
        }
        const double s = block_add(left_sum<TY, PT, true>(a, a.x + b * a.seq + node * a.row, a.q + b * a.p_seq + node * a.p_row, e, seg), sm_sum);
        if (threadIdx.x == 0) a.left[(((int64_t)b * a.max_n + node) * 2 + round) * a.segs + seg] = s;
    }
}

// The sum of a row's weights without the tokens of the lanes in `gone`, by the whole workgroup.  1 less a likely token's probability
// would be off by as much as the row's sum, however little is left; this is off by 2^-17 of itself: hardware exponentials, their
// exponents (60 more, so that 2^-180 of the largest weight still counts) by 2^-19, and eight chains of additions.  A sequence's pass
// over 151936 fp32 logits: 12 us more for one, 24 for sixteen.
template <int TY>
__device__ __forceinline__ double rest_of(const AcArgs &a, const uint8_t *row, float m, int token, uint64_t gone, double *sm) {
    constexpr int V = AC_V<TY>, E = 32, STEP = AC_T * E;
    const float c = (float)a.c;
    double s = 0.0;
    for (int k = 0; k < a.vocab; k += STEP) {
        auto index = [&](int e) { return k + (e / V * AC_T + (int)threadIdx.x) * V + e % V; };
        float x[E], f[8] = {};
        if (k + STEP <= a.vocab)
#pragma unroll
            for (int e = 0; e < E; e += V) values<TY, true>(row, index(e), a.vocab, -INFINITY, x + e);
        else
#pragma unroll
            for (int e = 0; e < E; e += V) values<TY, false>(row, index(e), a.vocab, -INFINITY, x + e);
        for (uint64_t out = gone; out; out &= out - 1) {
            const int t = __builtin_amdgcn_readlane(token, __ffsll((unsigned long long)out) - 1);
            if (t >= k && t - k < STEP)
#pragma unroll
                for (int e = 0; e < E; e++) x[e] = t == index(e) ? -INFINITY : x[e];
        }
#pragma unroll
        for (int e = 0; e < E; e++) f[e % 8] += __builtin_amdgcn_exp2f(fmaf(x[e] - m, c, 60.0f));
#pragma unroll
        for (int i = 0; i < 8; i++) s += (double)f[i];
    }
    return block_add(s, sm) * 0x1p-60;
}

template <int TY, int PT> // PT: the type of the draft's probabilities, -1: none
__global__ void __launch_bounds__(AC_T) k_accept_walk(AcArgs a) {
    constexpr int PQ = PT < 0 ? LLM_F32 : PT;
    __shared__ float sm_m[AC_N];
    __shared__ int sm_best[AC_N];
    __shared__ double sm_s[AC_N], sm_sum[AC_T / 64], sm_before, sm_point;
    __shared__ AcEnd end;
    __shared__ int sm_seg, sm_at[AC_T / 64], sm_end[AC_T / 64], sm_last;
    const int seg = blockIdx.x, b = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x / 64, nn = nodes(a, b);
    const int64_t at0 = (int64_t)b * a.max_n;
    if (nn == 0) {
        if (seg == 0) {
            for (int i = threadIdx.x; i < a.max_n; i += AC_T) a.path[at0 + i] = -1, a.logp[at0 + i] = 0.0f;
            if (threadIdx.x == 0) a.kept[b] = 0, a.next[b] = -1;
        }
        return;
    }
    const uint8_t *const x = a.x + b * a.seq, *const q = PT >= 0 ? a.q + b * a.p_seq : nullptr;
    const AcNode d = node_of<TY, PT>(a, b, nn, x, q, sm_m, sm_best, sm_s);
    const int parent = d.parent, token = d.token;
    const float y = d.y, u = d.u;
    const double prob = d.q, p = d.p;
    if (seg == 0 && wave == 0 && lane > 0 && lane < a.max_n) {
        float lp = 0.0f;
        if (parent >= 0) {
            lp = -INFINITY;
            if (token >= 0 && a.c == 0.0) lp = p != p ? NAN : p > 0.0 ? 0.0f : -INFINITY;
            else if (token >= 0)
                lp = (float)((((double)y - (double)sm_m[parent]) * a.c - log2_of(sm_s[parent])) * 0.693147180559945309417);
        }
        a.logp[at0 + lane] = lp;
    }
    // the walk: from child to child, values of a lane read by all
    int node = 0;
    uint64_t kept = 1, gone = 0; // nodes on the way; children of the node that were turned down
    // Without draft probabilities `left` is 1 less what was turned down, as far off as the row's sum: where that has become a quarter
    // it is summed anew (rest_of), and again where three quarters of that are gone.
    double left = 1.0, aq = 0.0, sure = 0.25;
    uint64_t open = __ballot(parent == 0 && token >= 0);
    while (open) {
        const int c = __ffsll((unsigned long long)open) - 1;
        open &= open - 1;
        const double coin = (double)__uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(u), c));
        double w = lane_of(p, c);
        bool takes;
        if (PT >= 0) {
            const double qc = lane_of(prob, c);
            w = fmax(w - aq * qc, 0.0);
            takes = coin * qc * left < w;
        } else {
            if (__ballot(token == __builtin_amdgcn_readlane(token, c)) & gone) w = 0.0;
            takes = coin * left < w;
        }
        if (takes) {
            node = c, left = 1.0, aq = 0.0, sure = 0.25;
            kept |= (uint64_t)1 << c;
            gone = 0;
            open = __ballot(parent == node && token >= 0);
            continue;
        }
        gone |= (uint64_t)1 << c;
        if (PT < 0) left = fmax(left - w, 0.0);
        else aq += left;
        const int round = __popcll(gone) - 1;
        if (!open) continue;
        // another child to hold against what is left
        if (PT >= 0 && a.left && round < 2) {
            left = z_of(a, b, node, round);
        } else if (PT < 0) {
            if (left < sure && a.c != 0.0) {
                left = rest_of<TY>(a, x + node * a.row, sm_m[node], token, gone, sm_sum) / sm_s[node];
                sure = 0.25 * left;
            }
        } else {
            const uint8_t *row = x + node * a.row, *probs = q + node * a.p_row;
            double s = 0.0;
            const double inv = 1.0 / sm_s[node];
            const bool greedy = a.c == 0.0;
            const double m = (double)sm_m[node];
            const int best = sm_best[node];
            for (int k = threadIdx.x * 8; k < a.vocab; k += AC_T * 8) {
                float xv[8], qv[8];
#pragma unroll
                for (int e = 0; e < 8; e += AC_V<TY>) values<TY>(row, k + e, a.vocab, -INFINITY, xv + e);
#pragma unroll
                for (int e = 0; e < 8; e += AC_V<PQ>) values<PQ>(probs, k + e, a.vocab, 0.0f, qv + e);
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const double w = greedy ? k + e == best ? inv : 0.0 : weight(xv[e], m, a.c) * inv;
                    s += fmax(w - aq * (double)qv[e], 0.0);
                }
            }
            left = block_add(s, sm_sum);
        }
    }
    if (wave == 0) {
        if (lane == 0) {
            end.node = node, end.turned = PT < 0 ? __popcll(gone) : 0;
            end.m = sm_m[node], end.best = sm_best[node], end.s = sm_s[node], end.inv = 1.0 / sm_s[node], end.a = aq;
        }
        if ((gone >> lane) & 1) end.out[__popcll(gone & (((uint64_t)1 << lane) - 1))] = token;
        if (seg == 0) {
            const int count = __popcll(kept);
            if (lane >= count && lane < a.max_n) a.path[at0 + lane] = -1;
            if ((kept >> lane) & 1) a.path[at0 + __popcll(kept & (((uint64_t)1 << lane) - 1))] = lane;
            if (lane == 0) a.kept[b] = count;
        }
    }
    __syncthreads();
    const uint8_t *const row = x + node * a.row, *const probs = PT >= 0 ? q + node * a.p_row : nullptr;
    // Sums of segments through the same code: the workgroup's own; of the sequence's last workgroup, where nothing is left, those
    // of the target's own row too.  The threads' shares are kept for the draw, which would else read the segment and sum it again
    // (the walk of 16 trees of bf16 rows: 2.7 us less).
    double *const sums = a.sums + (int64_t)b * a.segs, *const shares = a.shares + (int64_t)b * a.segs * AC_T;
    // (through to where every XCD reads it)
    auto put = [](double *at, double v) { __hip_atomic_store(at, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
    auto get = [](double *at) { return __hip_atomic_load(at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
    auto sum_at = [&](int k) { return k < a.segs ? get(&sums[k]) : 0.0; };
    int now = seg, rest = -1; // rest: the next segment of the target's own row
#pragma unroll 1
    for (;;) {
        const double share = left_sum<TY, PT, false>(a, row, probs, end, now), all_s = block_add(share, sm_sum);
        put(&shares[now * AC_T + threadIdx.x], share);
        if (threadIdx.x == 0) put(&sums[now], all_s);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); // (there before it is counted)
        __syncthreads();
        if (threadIdx.x == 0 && rest < 0)
            sm_last = __hip_atomic_fetch_add(&a.done[b], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == a.segs - 1;
        __syncthreads();
        if (!sm_last) return;
        if (rest >= 0 && rest < a.segs) {
            now = rest++;
            continue;
        }
        double mine = sum_at(lane), all = mine;
        for (int k = lane + 64; k < a.segs; k += 64) all += sum_at(k);
        all = lanes_add<64>(all);
        if (all == 0.0 && rest < 0) {
            __syncthreads();
            if (threadIdx.x == 0) end.a = 0.0, end.turned = 0;
            __syncthreads();
            now = 0, rest = 1;
            continue;
        }
        if (wave == 0) { // the point, its segment, and the sum before that, segments in order
            const double point = (double)__uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(u), 0)) * all;
            int found = -1, last = -1; // the segment; the last one that has something (a point at the end, by rounding)
            double before = 0.0, start = 0.0, last_start = 0.0;
            if (all > 0.0)
                for (int k0 = 0; k0 < a.segs && found < 0; k0 += 64) {
                    if (k0) mine = sum_at(k0 + lane);
                    const double to = before + upto(mine);
                    const uint64_t over = __ballot(mine > 0.0 && to > point), some = __ballot(mine > 0.0);
                    if (over) found = __ffsll((unsigned long long)over) - 1, start = lane_of(to - mine, found), found += k0;
                    if (some) last = 63 - __clzll((long long)some), last_start = lane_of(to - mine, last), last += k0;
                    before = lane_of(to, 63);
                }
            if (lane == 0) {
                sm_seg = found >= 0 ? found : last;
                sm_before = found >= 0 ? start : last_start;
                sm_point = point;
            }
        }
        __syncthreads();
        if (sm_seg < 0) { // no probabilities, or a draft's that are not finite
            if (threadIdx.x == 0) a.next[b] = -1, a.logp[at0] = NAN;
            return;
        }
        break;
    }
    const double s = get(&shares[sm_seg * AC_T + threadIdx.x]);
    // the thread whose values the point falls into: the first with the sum up to its end above it (else, by rounding, the last one
    // that has something)
    const double to = upto(s);
    if (lane == 63) sm_sum[wave] = to;
    __syncthreads();
    double c = sm_before + (to - s);
    for (int k = 0; k < wave; k++) c += sm_sum[k];
    // (by ballots: atomics of a wave's lanes on one address are taken one lane after another, 4 us for two)
    {
        const uint64_t over = __ballot(s > 0.0 && c + s > sm_point), some = __ballot(s > 0.0);
        if (lane == 0) {
            sm_at[wave] = over ? wave * 64 + __ffsll((unsigned long long)over) - 1 : 0x7fffffff;
            sm_end[wave] = some ? wave * 64 + 63 - __clzll((long long)some) : -1;
        }
    }
    __syncthreads();
    const int first_at = min(min(sm_at[0], sm_at[1]), min(sm_at[2], sm_at[3]));
    const int thread = first_at != 0x7fffffff ? first_at : max(max(sm_end[0], sm_end[1]), max(sm_end[2], sm_end[3]));
    if ((int)threadIdx.x == thread) sm_before = c;
    __syncthreads();
    if (wave) return;
    // its values, a lane each
    const int i = sm_seg * AC_SEG + thread * AC_E + lane;
    float value = 0.0f;
    double w = 0.0;
    if (thread >= 0 && lane < AC_E && i < a.vocab) {
        value = at<TY>(row, i);
        float qi = 0.0f;
        if (PT >= 0) qi = at<PQ>(probs, i);
        double one[1];
        left_of<PT, false>(a, end, &value, &qi, i, one);
        w = one[0];
    }
    const double sum = upto(w);
    const uint64_t over = __ballot(w > 0.0 && sm_before + sum > sm_point), some = __ballot(w > 0.0);
    const int drawn = over ? __ffsll((unsigned long long)over) - 1 : 63 - __clzll((long long)some);
    if (some == 0) {
        if (lane == 0) a.next[b] = -1, a.logp[at0] = NAN;
    } else if (lane == drawn) {
        float lp = i == end.best ? 0.0f : -INFINITY;
        if (a.c != 0.0) lp = (float)((((double)value - (double)end.m) * a.c - log2_of(end.s)) * 0.693147180559945309417);
        a.next[b] = i;
        a.logp[at0] = lp;
    }
}

int64_t ac_segs(int vocab) { return ((int64_t)vocab + AC_SEG - 1) / AC_SEG; }

} // namespace

extern "C" size_t llm_draft_accept_work(int n_seq, int max_n, int vocab) {
    if (n_seq < 1 || max_n < 1 || max_n > AC_N || vocab < 1) return 0;
    const size_t segs = ac_segs(vocab);
    return (size_t)n_seq * (max_n * (segs * (sizeof(AcPart) + 2 * sizeof(double)) + sizeof(AcAsk)) +
                            segs * (1 + AC_T) * sizeof(double) + 2 * sizeof(int));
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
    const int per = (int64_t)n_seq * max_n * a.segs >= 4096 ? 4 : 1;
    a.parts = (a.segs + per - 1) / per;
    a.c = temperature == 0.0f ? 0.0 : 1.44269504088896340736 / (double)temperature;
    a.tokens = tokens, a.parents = parents, a.n = n, a.coins = coins;
    a.kept = kept, a.path = path, a.next = next, a.logp = logp;
    a.part = (AcPart *)work;
    a.sums = (double *)(a.part + (size_t)n_seq * max_n * a.segs);
    a.shares = a.sums + (size_t)n_seq * a.segs;
    a.asks = (AcAsk *)(a.shares + (size_t)n_seq * a.segs * AC_T);
    double *const z = (double *)(a.asks + (size_t)n_seq * max_n);
    a.done = (int *)(z + (size_t)n_seq * max_n * 2 * a.segs);
    a.count = a.done + n_seq;
    if (probs && parents && max_n > 2 && vocab >= AC_ASK) a.left = z;
    hipStream_t st = (hipStream_t)stream;
    void (*rows)(AcArgs) = nullptr;
#define ACCEPT_PICK(T, P, X) \
    if (type == T && per == P && (probs != nullptr) == X) rows = k_accept_rows<T, P, X>;
    ACCEPT_PICK(LLM_F32, 1, false) ACCEPT_PICK(LLM_F32, 4, false) ACCEPT_PICK(LLM_BF16, 1, false) ACCEPT_PICK(LLM_BF16, 4, false)
    ACCEPT_PICK(LLM_F32, 1, true) ACCEPT_PICK(LLM_F32, 4, true) ACCEPT_PICK(LLM_BF16, 1, true) ACCEPT_PICK(LLM_BF16, 4, true)
#undef ACCEPT_PICK
    hipLaunchKernelGGL(rows, dim3(a.parts, max_n, n_seq), dim3(AC_T), 0, st, a);
    HIP_OR_FAIL(who, hipGetLastError());
    void (*walk)(AcArgs) = nullptr, (*ask)(AcArgs) = nullptr, (*sum)(AcArgs, int) = nullptr;
    const int pt = probs ? p_type : -1;
#define ACCEPT_PICK(T, P) \
    if (type == T && pt == P) ask = k_accept_ask<T, P>, sum = k_accept_left<T, P>, walk = k_accept_walk<T, P>;
    ACCEPT_PICK(LLM_F32, LLM_F32) ACCEPT_PICK(LLM_F32, LLM_BF16) ACCEPT_PICK(LLM_BF16, LLM_F32) ACCEPT_PICK(LLM_BF16, LLM_BF16)
#undef ACCEPT_PICK
    if (pt < 0) walk = type == LLM_F32 ? k_accept_walk<LLM_F32, -1> : k_accept_walk<LLM_BF16, -1>;
    if (a.left) {
        hipLaunchKernelGGL(ask, dim3(n_seq), dim3(AC_T), 0, st, a);
        HIP_OR_FAIL(who, hipGetLastError());
        for (int round = 0; round < (max_n > 3 ? 2 : 1); round++) {
            hipLaunchKernelGGL(sum, dim3(a.segs, std::min(max_n / 2, 4), n_seq), dim3(AC_T), 0, st, a, round);
            HIP_OR_FAIL(who, hipGetLastError());
        }
    }
    hipLaunchKernelGGL(walk, dim3(a.segs, n_seq), dim3(AC_T), 0, st, a);
    HIP_OR_FAIL(who, hipGetLastError());
    return 0;
}
