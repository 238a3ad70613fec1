// Attention of drafted tokens over a cache, head sizes up to TREE_HSP (a multiple of 64; this file is compiled for each).
//
// The rows of a kv head are its query heads' tokens (row = token * group + head of the group), in tiles of 16 on the
// 16 x 16 matrix instructions, with one running maximum and sum a row over the positions:
//   scores  S^T = K Q^T: K rows are the A operand, the queries B.  A lane 16 j + n then owns the scores of row n at
//           positions 4 j + i of every 16.
//   values  O^T += V^T P^T: its own probabilities are the B operand as they are (eight positions: 4 j + i of two tiles of
//           16); V, A, has those positions of one dimension in a lane.
// k_tree_attention: the block's four waves share the positions; K and V go from memory to the registers where they are used,
// and blocks with other rows of the same heads find them in the L2.  k_tree_rows, for many rows over bf16 caches: the waves
// share the rows; each step's K and V are read by all from LDS.
//
// Operands.  int8 and e4m3 codes are exact in fp16, and the fp32 side is held in two fp16 pieces (22 bits): a query row is
// scaled by a power of two to the top of fp16's range first, and so are the weights p * V scale, by the largest V scale met
// (a running exponent, as the maximum is running).  bf16 caches: three bf16 pieces.  16-bit queries are one piece, exactly; their
// weights stay two pieces over 8-bit caches (one, 2^-12 off, changed the rounding of a tenth of a batch's outputs) and are two
// over bf16 ones (2^-16 off, against the output's 2^-8: one output in five hundred rounds otherwise).  fp32 caches:
// v_mfma_f32_16x16x4_f32.  Maxima, sums and outputs are fp32.
#include <limits.h>

#include <type_traits>

#include "device.h"
#include "tree_attention.h"

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

constexpr int HSP = TREE_HSP;
constexpr uint32_t OUT_OF_RANGE = 0x80000000u; // a buffer offset past every resource here: the load returns zero

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ uint32_t bf2(float x, float y) { // a float pair in bf16, rounded
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){x, y}, bf16x2));
}
__device__ __forceinline__ float lo16(uint32_t u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float hi16(uint32_t u) { return __uint_as_float(u & 0xffff0000u); }

// x and y as NP 16-bit pieces (bf16 caches: bf16, 8-bit caches: fp16), each word a pair
template <int CT, int NP>
__device__ __forceinline__ void split(float x, float y, uint32_t *p) {
#pragma unroll
    for (int i = 0; i < NP; i++) {
        if constexpr (CT == LLM_BF16) {
            p[i] = bf2(x, y);
            if (i + 1 < NP) x -= lo16(p[i]), y -= hi16(p[i]);
        } else {
            const f16x2 h = __builtin_convertvector((f32x2){x, y}, f16x2);
            p[i] = __builtin_bit_cast(uint32_t, h);
            if (i + 1 < NP) x = fmaf((float)h[0], -1.0f, x), y = fmaf((float)h[1], -1.0f, y);
        }
    }
}
// Two codes (word W of u: bytes 2 W and 2 W + 1) as an fp16 pair.  int8 (its sign bit flipped before, flip_sign): 0x64 over
// the byte is 1024 + code + 128.
template <int CT>
__device__ __forceinline__ uint32_t flip_sign(uint32_t u) { return CT == LLM_I8 ? u ^ 0x80808080u : u; }
template <int CT, int W>
__device__ __forceinline__ uint32_t codes2(uint32_t u) {
    if constexpr (CT == LLM_I8) {
        const uint32_t h = __builtin_amdgcn_perm(0x64646464u, u, W ? 0x04030402u : 0x04010400u);
        const f16x2 c = __builtin_bit_cast(f16x2, h) - (f16x2){(_Float16)1152.0f, (_Float16)1152.0f};
        return __builtin_bit_cast(uint32_t, c);
    } else {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)u, 1.0f, W));
    }
}
// The pairs (a0, a1) of bytes 2 H and 2 H + 1: pieces of V at two positions, by dimension.
template <int CT, int H>
__device__ __forceinline__ void pairs2(uint32_t a0, uint32_t a1, uint32_t *p) {
    const uint32_t m = flip_sign<CT>(__builtin_amdgcn_perm(a1, a0, H ? 0x07030602u : 0x05010400u));
    p[0] = codes2<CT, 0>(m);
    p[1] = codes2<CT, 1>(m);
}

// An operand of a product over 32 terms: eight values a lane.  fp32: as they are, else NP 16-bit pieces.
template <int CT, int NP>
struct Frag {
    typename std::conditional<CT == LLM_F32, float[8], u32x4[NP]>::type v;
};
template <int CT, int NP>
__device__ __forceinline__ f32x4 product(const Frag<CT, 1> &a, const Frag<CT, NP> &b, f32x4 d) {
    if constexpr (CT == LLM_F32) {
#pragma unroll
        for (int i = 0; i < 8; i++) d = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[i], b.v[i], d, 0, 0, 0);
    } else {
#pragma unroll
        for (int p = NP - 1; p >= 0; p--) { // smallest pieces first
            if constexpr (CT == LLM_BF16)
                d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a.v[0]),
                                                            __builtin_bit_cast(bf16x8, b.v[p]), d, 0, 0, 0);
            else
                d = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a.v[0]),
                                                           __builtin_bit_cast(f16x8, b.v[p]), d, 0, 0, 0);
        }
    }
    return d;
}
// Scores of 16 positions and 16 rows.  fp32: an instruction adds its four products one after another, so one chain over all
// dimensions would be off by up to twice as much as four do (and a score's error is the weight's).
template <int CT, int NP>
struct Scores {
    static constexpr int N = CT == LLM_F32 ? 4 : 1;
    f32x4 c[N] = {};
    __device__ __forceinline__ void add(const Frag<CT, 1> &a, const Frag<CT, NP> &b) {
        if constexpr (CT == LLM_F32) {
#pragma unroll
            for (int i = 0; i < 8; i++) c[i % 4] = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[i], b.v[i], c[i % 4], 0, 0, 0);
        } else {
            c[0] = product(a, b, c[0]);
        }
    }
    __device__ __forceinline__ f32x4 sum() const {
        if constexpr (CT == LLM_F32) return (c[0] + c[1]) + (c[2] + c[3]);
        else return c[0];
    }
};
template <int CT, int NP>
__device__ __forceinline__ void fill(Frag<CT, NP> &f, const float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        if constexpr (CT == LLM_F32) f.v[i] = x[i], f.v[i + 1] = x[i + 1];
        else {
            uint32_t p[NP];
            split<CT, NP>(x[i], x[i + 1], p);
#pragma unroll
            for (int k = 0; k < NP; k++) f.v[k][i / 2] = p[k];
        }
    }
}

// The power of two that takes a magnitude to [2^14, 2^15) (magnitudes below 2^-112 to less, infinities: 2^-127 and NaN), and
// its inverse, from the magnitude's exponent field.
__device__ __forceinline__ uint32_t exponent(float x) { return (__float_as_uint(x) >> 23) & 0xff; }
__device__ __forceinline__ float power_to(uint32_t e) { return __uint_as_float(min(268u - e, 253u) << 23); }
__device__ __forceinline__ float power_from(uint32_t e) { return __uint_as_float((254u - min(268u - e, 253u)) << 23); }

// Over the four lane groups (lanes l, l ^ 16, l ^ 32, l ^ 48).
template <typename F>
__device__ __forceinline__ float over_groups(float x, F &&f) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = f(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return f(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float fmax_(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ float fadd_(float a, float b) { return a + b; }

__device__ __forceinline__ void wave_lds_fence() { // this wave's LDS stores before its loads
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

template <int CT, int QT>
struct TreePieces {
    static constexpr int ES = CT == LLM_F32 ? 4 : CT == LLM_BF16 ? 2 : 1;
    static constexpr bool SCALED = ES == 1;
    static constexpr int Q = QT == LLM_BF16 ? 1 : SCALED ? 2 : 3; // of a query
    static constexpr int P = QT == LLM_BF16 || SCALED ? 2 : 3;    // of a weight
};

template <int QT>
__device__ __forceinline__ float4 load_query(const uint8_t *row, int d) {
    if constexpr (QT == LLM_F32) return *(const float4 *)(row + (size_t)d * 4);
    const uint2 u = *(const uint2 *)(row + (size_t)d * 2);
    return make_float4(lo16(u.x), hi16(u.x), lo16(u.y), hi16(u.y));
}

// The dimension of value i = 4 q4 .. 4 q4 + 3 of lane group j in product s: a lane has 16-byte pieces of a K row, piece j of
// every four (for bf16 that is the rows' order, which k_tree_rows' LDS keeps).
template <int CT>
__device__ __forceinline__ int dim_of(int s, int j, int q4) {
    if constexpr (CT == LLM_BF16) return 32 * s + 8 * j + 4 * q4;
    else if constexpr (CT == LLM_F32) return 32 * s + 16 * q4 + 4 * j;
    else return 64 * (s / 2) + 16 * j + 8 * (s % 2) + 4 * q4;
}

// Where a block works: sequence, kv head, slice (`id` of all), first row, and how many positions and rows there are.
struct Place {
    int b, h, split, id, row0, len, end, rows, slices, first, last;
};

// The slice `id`: its sequence, kv head and number there, the slices of that head and their steps.  A sequence of n steps
// has ceil(n / q) slices a head, the same q for all, so that long sequences do not outlast the others; q is about the least
// at which there are no more than a.cap in all.  Every block finds it from the lengths.
__device__ __forceinline__ bool find_slice(const TreeArgs &a, uint32_t id, Place &p, int &steps) {
    if (a.n_seq == 1) {
        p.b = 0;
        p.h = (int)id / a.each;
        p.split = (int)id - p.h * a.each;
        p.slices = tree_one(a, tree_steps(a, 0), steps);
        return p.split < p.slices;
    }
    const int lane = threadIdx.x & 63;
    constexpr int GROUPS = TREE_MAX_SEQS / 64;
    int all[GROUPS];
    float sum = 0.0f, most = 0.0f; // (a guess to begin with: rounded sums of steps do)
#pragma unroll
    for (int i = 0; i < GROUPS; i++) {
        all[i] = 0;
        if (64 * i < a.n_seq) {
            if (64 * i + lane < a.n_seq) all[i] = tree_steps(a, 64 * i + lane);
            sum += (float)all[i];
            most = fmaxf(most, (float)all[i]);
        }
    }
    const float kv = (float)a.n_kv;
    const int guess = __builtin_amdgcn_readfirstlane((int)(wave_sum(sum) * kv / (float)a.cap));
    const int longest = __builtin_amdgcn_readfirstlane((int)wave_max(most));
    steps = longest <= TREE_WHOLE * a.least ? longest : max(max(a.least, guess), longest / a.each + 1);
    int n[GROUPS];
    for (;; steps += (steps + 15) / 16) { // (ends: at the longest sequence's steps there is a slice a head)
        float total = 0.0f;
#pragma unroll
        for (int i = 0; i < GROUPS; i++) {
            n[i] = 0;
            if (64 * i < a.n_seq) {
                n[i] = (all[i] + steps - 1) / steps;
                total += (float)n[i];
            }
        }
        if (wave_sum(total) * kv <= (float)a.cap) break; // (exact up to 2^24)
    }
    int before = 0; // slices of a head of the sequences before
#pragma unroll
    for (int i = 0; i < GROUPS; i++)
        if (64 * i < a.n_seq) {
            int upto = n[i];
#pragma unroll
            for (int off = 1; off < 64; off <<= 1) {
                const int x = __shfl_up(upto, off);
                upto += lane >= off ? x : 0;
            }
            const int passed = __popcll(__ballot((before + upto) * a.n_kv <= (int)id));
            if (passed < 64) { // (a lane without a sequence has passed none that its neighbours have not)
                const int at = __builtin_amdgcn_readfirstlane(passed);
                p.b = 64 * i + at;
                p.slices = __builtin_amdgcn_readlane(n[i], at);
                const int rest = (int)id - (before + __builtin_amdgcn_readlane(upto, at) - p.slices) * a.n_kv;
                p.h = rest / p.slices;
                p.split = rest - p.h * p.slices;
                return true;
            }
            before += __builtin_amdgcn_readlane(upto, 63);
        }
    return false;
}

// Blocks go to the eight XCDs in turn.  The row blocks of a slice follow each other on one, whose L2 then holds the slice's
// rows for all of them.
template <int QT>
__device__ __forceinline__ bool place(const TreeArgs &a, int block_rows, Place &p) {
    const uint32_t k = blockIdx.x >> 3, kr = k / (uint32_t)a.row_blocks, id = kr * 8 + (blockIdx.x & 7);
    int steps = INT_MAX;
    if (a.cap) {
        if (id >= (uint32_t)a.cap || !find_slice(a, id, p, steps)) return false;
    } else {
        if (id >= (uint32_t)(a.n_seq * a.n_kv)) return false; // (the grid is rounded up to eight slices)
        p.b = (int)(id / (uint32_t)a.n_kv);
        p.h = (int)id - p.b * a.n_kv;
        p.split = 0;
        p.slices = 1;
    }
    p.id = (int)id;
    const int row0 = (int)(k - kr * a.row_blocks) * block_rows;
    if (a.cap && a.n_seq > 1 && p.split == 0 && row0 == 0 && threadIdx.x == 0) // (for the join)
        a.plan[p.b * a.n_kv + p.h] = make_int2((int)id, p.slices);
    p.row0 = row0;
    p.len = min(max(a.lens[p.b], 0), a.ctx);
    const int nn = a.n ? min(max(a.n[p.b], 0), a.max_n) : a.max_n;
    p.end = (int)min((int64_t)p.len + nn, (int64_t)a.ctx);
    p.rows = nn * a.group;
    if (a.zero_rest && p.split == 0 && row0 + block_rows > p.rows) { // the rows behind the last token
        for (int e = threadIdx.x * 4; e < block_rows * a.hs; e += 4 * blockDim.x) {
            const int row = row0 + e / a.hs, t = row / a.group, d = e - (row - row0) * a.hs;
            if (row < p.rows || row >= a.max_n * a.group) continue;
            uint8_t *op = a.o + p.b * a.o_seq + t * a.o_tok + (p.h * a.group + row - t * a.group) * a.o_head;
            if constexpr (QT == LLM_F32) *(float4 *)(op + (size_t)d * 4) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            else *(uint2 *)(op + (size_t)d * 2) = make_uint2(0, 0);
        }
    }
    const int all = (p.end + a.tp - 1) / a.tp;
    p.first = p.split ? p.split * steps : 0;
    p.last = (int)min((int64_t)p.first + steps, (int64_t)all);
    return row0 < p.rows;
}

// The queries of row `row` (none from p.rows on: zeros, nothing seen) as the operand of its scores.  Returns what takes a
// score to the exponent of 2.
template <int CT, int QT, int NP>
__device__ __forceinline__ float load_queries(const TreeArgs &a, const Place &p, int row, Frag<CT, NP> (&qf)[HSP / 32],
                                              uint64_t &sees) {
    const int j = (threadIdx.x & 63) >> 4, t = row / a.group, g = row - t * a.group;
    const bool ok = row < p.rows;
    sees = 0;
    if (ok) sees = a.mask ? a.mask[(int64_t)p.b * a.max_n + t] : ~(uint64_t)0 >> (63 - t);
    if (p.end - p.len < 64) sees &= ((uint64_t)1 << (p.end - p.len)) - 1; // (tokens that are there)
    const uint8_t *qp = a.q + p.b * a.q_seq + (ok ? t * a.q_tok + (p.h * a.group + g) * a.q_head : 0);
    // every load goes out before the first is used (what is not there reads the row's start): behind conditions each would
    // be waited for by itself
    float4 v[HSP / 32][2];
#pragma unroll
    for (int s = 0; s < HSP / 32; s++)
#pragma unroll
        for (int q4 = 0; q4 < 2; q4++) {
            const int d = dim_of<CT>(s, j, q4);
            v[s][q4] = load_query<QT>(qp, d < a.hs ? d : 0);
        }
    float x[HSP / 32][8], mx = 0.0f;
#pragma unroll
    for (int s = 0; s < HSP / 32; s++)
#pragma unroll
        for (int q4 = 0; q4 < 2; q4++) {
            const bool there = ok && dim_of<CT>(s, j, q4) < a.hs;
            const float y[4] = {v[s][q4].x, v[s][q4].y, v[s][q4].z, v[s][q4].w};
#pragma unroll
            for (int i = 0; i < 4; i++) {
                x[s][4 * q4 + i] = there ? y[i] : 0.0f;
                mx = fmaxf(mx, fabsf(x[s][4 * q4 + i]));
            }
        }
    float to = 1.0f, from = 1.0f;
    if constexpr (TreePieces<CT, QT>::SCALED) {
        const uint32_t e = exponent(over_groups(mx, fmax_));
        to = power_to(e);
        from = power_from(e);
    }
    to *= a.sign;
#pragma unroll
    for (int s = 0; s < HSP / 32; s++) {
#pragma unroll
        for (int i = 0; i < 8; i++) x[s][i] *= to;
        fill(qf[s], x[s]);
    }
    return fmaxf(a.c * from, 1e-45f); // (never 0: the scores of what is not seen are -infinity times this)
}

// What the row sees of a step's positions where new tokens or the end are among them: bit 4 t + i.  A lane's four neighbours at
// once: those of `sees` from the first one on, ones below the new tokens, zeros past 64 of them.
template <int N>
__device__ __forceinline__ uint32_t seen_bits(const Place &p, int p0, uint64_t sees) {
    const int j = (threadIdx.x & 63) >> 4;
    uint32_t vis = 0;
#pragma unroll
    for (int t = 0; t < N / 4; t++) {
        const int at = p0 + 16 * t + 4 * j - p.len;
        const uint32_t below = ((uint32_t)sees << 4 | 15u) >> (max(at + 4, 0) & 31);
        const uint32_t from = at < 64 ? (uint32_t)(sees >> (at & 63)) : 0u;
        vis |= ((at < 0 ? below : from) & 15u) << (4 * t);
    }
    return vis;
}

// x where the row sees position i, else `or_else`, through a word of ones or zeros: as conditions the masks of all positions would
// take more scalar registers than there are.
__device__ __forceinline__ float if_seen(uint32_t vis, int i, float x, float or_else) {
    const uint32_t m = (uint32_t)__builtin_amdgcn_sbfe((int)vis, i, 1);
    return __uint_as_float((__float_as_uint(x) & m) | (__float_as_uint(or_else) & ~m));
}

// A step's scores x (with the K scales, if any) into the weights of its values: the running maximum m (exponents of 2) and
// sum l of the row; o and l are rescaled when the maximum has moved.  8-bit caches: `sv` (in LDS) holds the V scales at
// 16 t + i, and `ve` is the row's running exponent of the weights.  Before the edge every row sees every position: `step_e` is the
// exponent for all, and the scales come times its power.  At the edge they come as they are, and a row takes the exponent of
// those that it sees: what a row does not see changes no bit of it.  fp32 and bf16 weights have the exponents to go on with an
// old maximum until it is passed by a factor of 2^8 (a batch of 64-token trees over bf16: 144 us with every new maximum, 139
// so); the fp16 pieces' range is used up.
template <int NT, int CT, int NPP, int DT>
__device__ __forceinline__ void weights(f32x4 (&x)[NT], float cq, const float *sv, bool edge, uint32_t vis, uint32_t step_e,
                                        uint32_t &ve, float &m, float &l, f32x4 (&o)[DT], Frag<CT, NPP> (&pf)[NT / 2]) {
    constexpr bool SCALED = CT == LLM_I8 || CT == LLM_E4M3;
    float oe = 1.0f, pw = 1.0f; // what takes the row's values so far to its new power, and the power at the edge
    if constexpr (SCALED) {
        uint32_t e = step_e;
        if (edge) {
            float big = 0.0f;
#pragma unroll
            for (int t = 0; t < NT; t++) {
                const f32x4 s4 = *(const f32x4 *)(sv + 16 * t);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float s = fabsf(if_seen(vis, 4 * t + i, s4[i], 0.0f));
                    big = fmaxf(big, s < INFINITY ? s : 0.0f);
                }
            }
            e = max(ve, exponent(over_groups(big, fmax_)));
            pw = power_to(e);
        }
        if (e != ve) oe = power_from(ve) * power_to(e);
        ve = e;
    }
    if (edge)
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) x[t][i] = if_seen(vis, 4 * t + i, x[t][i], -INFINITY);
    float mx = x[0][0];
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
        for (int i = 0; i < 4; i++) mx = fmaxf(mx, x[t][i]);
    mx = over_groups(mx, fmax_);
    constexpr float SLACK = SCALED ? 0.0f : 8.0f;
    float mn = fmaxf(m, mx * cq), mu = m == -INFINITY ? 0.0f : m;
    const bool moved = mn > m + SLACK;
    if (__any(moved || oe != 1.0f)) {
        if (SLACK > 0.0f) mn = moved ? mn : m; // (a row's own: the wave's other rows change no bit of it)
        mu = mn == -INFINITY ? 0.0f : mn;
        const float al = __builtin_amdgcn_exp2f(m - mu), ao = al * oe;
        l *= al;
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
            for (int i = 0; i < 4; i++) o[d][i] *= ao;
        m = mn;
    }
#pragma unroll
    for (int u = 0; u < NT / 2; u++) {
        float w[8];
        f32x4 s4;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int t = 2 * u + i / 4;
            w[i] = __builtin_amdgcn_exp2f(fmaf(x[t][i % 4], cq, -mu));
            l += w[i];
            if constexpr (SCALED) {
                if (i % 4 == 0) s4 = *(const f32x4 *)(sv + 16 * t);
                w[i] *= s4[i % 4];
            }
        }
        if (SCALED && edge) { // (0 * a scale that is not finite)
#pragma unroll
            for (int i = 0; i < 8; i++) w[i] = if_seen(vis, 8 * u + i, w[i] * pw, 0.0f);
        }
        fill(pf[u], w);
    }
}

// Sums of row `row` at dimensions d .. d + 3: the output where there is one slice, else this slice's partial sums.
template <int QT>
__device__ __forceinline__ void put_values(const TreeArgs &a, const Place &p, int row, int d, float4 y) {
    if (d >= a.hs) return;
    if (p.slices > 1) {
        const int64_t part = (int64_t)p.id * a.max_n * a.group + row;
        *(float4 *)(a.acc + part * a.hs + d) = y;
        return;
    }
    const int t = row / a.group, g = row - t * a.group;
    uint8_t *op = a.o + p.b * a.o_seq + t * a.o_tok + (p.h * a.group + g) * a.o_head;
    if constexpr (QT == LLM_F32) *(float4 *)(op + (size_t)d * 4) = y;
    else *(uint2 *)(op + (size_t)d * 2) = make_uint2(bf2(y.x, y.y), bf2(y.z, y.w));
}
__device__ __forceinline__ void put_sums(const TreeArgs &a, const Place &p, int row, float m, float l) {
    const int64_t part = (int64_t)p.id * a.max_n * a.group + row;
    a.ml[2 * part] = m;
    a.ml[2 * part + 1] = l;
}
// what takes the sums of a row to its output (a row that sees nothing has the sum 0)
__device__ __forceinline__ float to_output(const Place &p, float l) {
    return p.slices > 1 ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
}

// A step's rows through buffers that hold its positions and no more: what lies past them reads as zero.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t step_rsrc(const void *base, int64_t stride, int step, int tp,
                                                            const Place &p) {
    const int left = step < p.last ? min(tp, p.end - step * tp) : 0;
    return __builtin_amdgcn_make_buffer_rsrc((void *)((const uint8_t *)base + (int64_t)step * tp * stride), 0,
                                             (int)(left * stride), 0x00020000);
}

// ---- the waves share the positions

template <int CT, int QT, int R>
struct TreeShape {
    static constexpr int ES = TreePieces<CT, QT>::ES;
    static constexpr int TP = tree_positions(HSP, CT, 0, R), NT = TP / 16; // positions a step, their tiles of 16
    static constexpr int KL = HSP * ES / 64;                                // 16-byte pieces of a K row a lane
    static constexpr int KS = HSP / 32;                                     // products of a score
    static constexpr int VW = HSP % 128 ? 4 : 8;                            // neighbouring dimensions a lane of V
    static constexpr int VC = HSP / (16 * VW), VR = VW * ES / 4;            // runs of them, a run's registers
    static constexpr size_t LDS = (size_t)2 * R * (HSP / 16) * 64 * 16 + 4 * R * 16 * 8 + 4 * 2 * 64 * 4;
};

// K's lane 16 j + n has 16-byte pieces of position n (piece j of every four), so a row's bytes are read whole and once.  V's
// lane n reads 4 or 8 neighbouring dimensions of its eight positions and pairs the registers of two positions, which
// transposes for nothing.  The next step's loads go out as soon as a step's registers are used.  No wave waits for
// another before the end.
// What bounds it: for one token, memory (32 sequences of 0 to 8190 e4m3 positions, 4 kv heads of 128: 28 us, 4.8 TB/s), or
// where few steps are left for each block, the latency of a step (32.7k int8 positions of one sequence: 13 us, 2.7 TB/s).
// For trees over 8-bit caches the vector instructions (codes into fp16, weights) and each step's chain of products, maximum,
// exponentials and products again, which two waves a SIMD hide in part: a 37-token tree, 259 rows, over 12k int8 positions takes
// 37 us (171 TFLOP/s, 342 of issued products), and of the 60k cycles that a SIMD's waves live, vector instructions are issued
// in 34k and the matrix unit is busy in 14k.
template <int CT, int QT, int R>
__global__ void __launch_bounds__(256, CT != LLM_F32 && HSP <= 128 ? 2 : 1) k_tree_attention(TreeArgs a) {
    using Sh = TreeShape<CT, QT, R>;
    using Pc = TreePieces<CT, QT>;
    constexpr int ES = Sh::ES, TP = Sh::TP, NT = Sh::NT, KL = Sh::KL, KS = Sh::KS, VW = Sh::VW, VC = Sh::VC, VR = Sh::VR;
    constexpr bool SCALED = Pc::SCALED;
    extern __shared__ __align__(16) uint8_t lds[];
    f32x4 *const sm_o = (f32x4 *)lds;                                           // [2][R][HSP / 16][64]
    float *const sm_ml = (float *)(lds + (size_t)2 * R * (HSP / 16) * 64 * 16); // [4][R][16][2]
    float *const sm_s = sm_ml + 4 * R * 16 * 2;                                 // [4][2][64]

    const int lane = threadIdx.x & 63, n = lane & 15, j = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    float2 *const my_ml = (float2 *)sm_ml + wave * R * 16; // until the end: what the wave's rows see, needed in its last step only
    Place p;
    if (!place<QT>(a, 16 * R, p)) return;
    const int row0 = p.row0;

    const uint8_t *const kb = a.k + p.b * a.seq + p.h * a.head, *const vb = a.v + p.b * a.seq + p.h * a.head;
    const float *ksb = nullptr, *vsb = nullptr;
    if constexpr (SCALED) {
        ksb = a.ks + p.b * a.s_seq + p.h * a.s_head;
        vsb = a.vs + p.b * a.s_seq + p.h * a.s_head;
    }
    const uint32_t ps = (uint32_t)a.pos, hb = (uint32_t)(a.hs * ES);
    u32x4 kr[NT][KL];
    uint32_t vr[TP / 4][VC][VR];
    uint32_t skr = 0, svr = 0;
    auto load_k = [&](int step) {
        const auto rs = step_rsrc(kb, a.pos, step, TP, p);
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int i = 0; i < KL; i++) {
                const uint32_t at = 64 * i + 16 * j;
                const auto x = __builtin_amdgcn_raw_buffer_load_b128(
                    rs, (int)(at < hb ? (16 * t + n) * ps + at : OUT_OF_RANGE), 0, 0);
                kr[t][i] = (u32x4){x[0], x[1], x[2], x[3]};
            }
        if constexpr (SCALED)
            skr = __builtin_amdgcn_raw_buffer_load_b32(step_rsrc(ksb, a.s_pos * 4, step, TP, p),
                                                       (int)(lane * (uint32_t)a.s_pos * 4), 0, 0);
    };
    auto load_v = [&](int step) {
        const auto rs = step_rsrc(vb, a.pos, step, TP, p);
        if constexpr (SCALED)
            svr = __builtin_amdgcn_raw_buffer_load_b32(step_rsrc(vsb, a.s_pos * 4, step, TP, p),
                                                       (int)(lane * (uint32_t)a.s_pos * 4), 0, 0);
#pragma unroll
        for (int x = 0; x < TP / 4; x++)
#pragma unroll
            for (int c = 0; c < VC; c++) {
                const uint32_t at = (c * 16 * VW + VW * n) * ES;
                const uint32_t off = at < hb ? (16 * (x / 4) + 4 * j + x % 4) * ps + at : OUT_OF_RANGE;
                if constexpr (VR == 1) vr[x][c][0] = __builtin_amdgcn_raw_buffer_load_b32(rs, (int)off, 0, 0);
                else if constexpr (VR == 2) {
                    const auto u = __builtin_amdgcn_raw_buffer_load_b64(rs, (int)off, 0, 0);
                    vr[x][c][0] = u[0], vr[x][c][1] = u[1];
                } else {
#pragma unroll
                    for (int i = 0; i < VR / 4; i++) {
                        const auto u = __builtin_amdgcn_raw_buffer_load_b128(rs, (int)(off + 16 * i), 0, 0);
#pragma unroll
                        for (int k = 0; k < 4; k++) vr[x][c][4 * i + k] = u[k];
                    }
                }
            }
    };
    int step = p.first + wave;
    load_k(step); // (a wave without a step loads nothing)
    load_v(step);

    Frag<CT, Pc::Q> qf[R][KS];
    float cq[R], m[R], l[R];
    f32x4 o[R][VC * VW];
#pragma unroll
    for (int r = 0; r < R; r++) {
        uint64_t sees;
        cq[r] = load_queries<CT, QT>(a, p, row0 + 16 * r + n, qf[r], sees);
        if (j == 0) my_ml[16 * r + n] = make_float2(__uint_as_float((uint32_t)sees), __uint_as_float((uint32_t)(sees >> 32)));
        m[r] = -INFINITY;
        l[r] = 0.0f;
#pragma unroll
        for (int d = 0; d < VC * VW; d++) o[r][d] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
    }
    wave_lds_fence();
    auto row_sees = [&](int r) {
        const float2 x = my_ml[16 * r + n];
        return (uint64_t)__float_as_uint(x.y) << 32 | __float_as_uint(x.x);
    };
    float *const my_s = sm_s + wave * 128;
    // exponent field of the largest V scale's magnitude (at least 2^-107): of all before the edge, and of what a row sees
    uint32_t ve = 20, row_ve[R];
#pragma unroll
    for (int r = 0; r < R; r++) row_ve[r] = ve;

    for (; step < p.last; step += 4) {
        const int p0 = step * TP;
        const bool edge = p0 + TP > p.len; // new tokens or the end among the positions
        f32x4 x[R][NT];
#pragma unroll
        for (int t = 0; t < NT; t++) {
Scores<CT, Pc::Q> sums[R];
#pragma unroll
            for (int s = 0; s < KS; s++) {
                Frag<CT, 1> kf;
                if constexpr (CT == LLM_F32) {
#pragma unroll
                    for (int i = 0; i < 8; i++) kf.v[i] = __uint_as_float(kr[t][2 * s + i / 4][i % 4]);
                } else if constexpr (CT == LLM_BF16) {
                    kf.v[0] = kr[t][s];
                } else {
                    const uint32_t u0 = flip_sign<CT>(kr[t][s / 2][2 * (s % 2)]);
                    const uint32_t u1 = flip_sign<CT>(kr[t][s / 2][2 * (s % 2) + 1]);
                    kf.v[0] = (u32x4){codes2<CT, 0>(u0), codes2<CT, 1>(u0), codes2<CT, 0>(u1), codes2<CT, 1>(u1)};
                }
#pragma unroll
                for (int r = 0; r < R; r++) sums[r].add(kf, qf[r][s]);
            }
#pragma unroll
            for (int r = 0; r < R; r++) x[r][t] = sums[r].sum();
        }
        if constexpr (SCALED) {
            my_s[lane] = __uint_as_float(skr);
            float sv = __uint_as_float(svr);
            if (!edge) {
                ve = max(ve, exponent(wave_max(fabsf(sv) < INFINITY ? fabsf(sv) : 0.0f)));
                sv *= power_to(ve);
            }
            my_s[64 + lane] = sv;
            wave_lds_fence();
        }
        load_k(step + 4);

        uint64_t bad = 0; // edge: new tokens whose V row is not finite
        if (edge) {
            if constexpr (CT != LLM_I8) {
                // a value (8-bit caches: an e4m3 code that is NaN) that is not finite would reach the rows that do not see it
                // as 0 * inf: taken out here, and the rows that do see it become NaN
#pragma unroll
                for (int i = 0; i < TP / 4; i++) {
                    const int q = p0 + 16 * (i / 4) + i % 4; // of lane group 0
                    bool nf = false;
#pragma unroll
                    for (int c = 0; c < VC; c++)
#pragma unroll
                        for (int k = 0; k < VR; k++) {
                            const uint32_t u = vr[i][c][k];
                            if constexpr (CT == LLM_F32) nf |= (u & 0x7f800000u) == 0x7f800000u;
                            else if constexpr (CT == LLM_E4M3) nf |= (((u & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0; // 0x7f
                            else nf |= (u & 0x7f80u) == 0x7f80u || (u & 0x7f800000u) == 0x7f800000u;
                        }
                    nf = nf && q + 4 * j >= p.len;
                    const uint64_t any = __ballot(nf);
                    if (any) {
#pragma unroll
                        for (int g = 0; g < 4; g++)
                            if ((any >> (16 * g)) & 0xffff) bad |= (uint64_t)1 << (q + 4 * g - p.len);
                        if ((any >> (16 * j)) & 0xffff)
#pragma unroll
                            for (int c = 0; c < VC; c++)
#pragma unroll
                                for (int k = 0; k < VR; k++) vr[i][c][k] = 0;
                    }
                }
            }
        }

        if constexpr (SCALED)
#pragma unroll
            for (int t = 0; t < NT; t++) {
                const f32x4 sk = *(const f32x4 *)(my_s + 16 * t + 4 * j);
#pragma unroll
                for (int r = 0; r < R; r++)
#pragma unroll
                    for (int i = 0; i < 4; i++) x[r][t][i] *= sk[i];
            }
        Frag<CT, Pc::P> pf[R][NT / 2];
#pragma unroll
        for (int r = 0; r < R; r++) {
            uint32_t vis = 0;
            uint64_t sees = 0;
            if (edge) {
                sees = row_sees(r);
                vis = seen_bits<TP / 4>(p, p0, sees);
            }
            weights(x[r], cq[r], my_s + 64 + 4 * j, edge, vis, ve, row_ve[r], m[r], l[r], o[r], pf[r]);
            if (CT != LLM_I8 && (sees & bad)) l[r] = NAN;
        }

#pragma unroll
        for (int u = 0; u < NT / 2; u++)
#pragma unroll
            for (int c = 0; c < VC; c++) {
                Frag<CT, 1> vf[VW];
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    const uint32_t *v0 = vr[8 * u + i][c], *v1 = vr[8 * u + i + 1][c];
                    if constexpr (CT == LLM_F32) {
#pragma unroll
                        for (int e = 0; e < VW; e++)
                            vf[e].v[i] = __uint_as_float(v0[e]), vf[e].v[i + 1] = __uint_as_float(v1[e]);
                    } else if constexpr (CT == LLM_BF16) {
#pragma unroll
                        for (int e = 0; e < VW; e++)
                            vf[e].v[0][i / 2] = __builtin_amdgcn_perm(v1[e / 2], v0[e / 2], e % 2 ? 0x07060302 : 0x05040100);
                    } else {
#pragma unroll
                        for (int e = 0; e < VW; e += 4) {
                            uint32_t q[4];
                            pairs2<CT, 0>(v0[e / 4], v1[e / 4], q);
                            pairs2<CT, 1>(v0[e / 4], v1[e / 4], q + 2);
#pragma unroll
                            for (int k = 0; k < 4; k++) vf[e + k].v[0][i / 2] = q[k];
                        }
                    }
                }
#pragma unroll
                for (int e = 0; e < VW; e++)
#pragma unroll
                    for (int r = 0; r < R; r++) o[r][c * VW + e] = product(vf[e], pf[r][u], o[r][c * VW + e]);
            }
        load_v(step + 4);
    }

    // the four waves' sums joined: each scaled to the common maximum, waves 2 and 3 into 0 and 1, then 1 into 0
#pragma unroll
    for (int r = 0; r < R; r++) {
        l[r] = over_groups(l[r], fadd_);
        if (j == 0) {
            sm_ml[((wave * R + r) * 16 + n) * 2] = m[r];
            sm_ml[((wave * R + r) * 16 + n) * 2 + 1] = l[r];
        }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < R; r++) {
        float mw[4], lw[4];
#pragma unroll
        for (int w = 0; w < 4; w++) {
            mw[w] = sm_ml[((w * R + r) * 16 + n) * 2];
            lw[w] = sm_ml[((w * R + r) * 16 + n) * 2 + 1];
        }
        const float mn = fmaxf(fmaxf(mw[0], mw[1]), fmaxf(mw[2], mw[3])), mu = mn == -INFINITY ? 0.0f : mn;
        const float al = __builtin_amdgcn_exp2f(m[r] - mu) * (SCALED ? power_from(row_ve[r]) : 1.0f);
        l[r] = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; w++) l[r] += lw[w] * __builtin_amdgcn_exp2f(mw[w] - mu);
        m[r] = mn;
#pragma unroll
        for (int d = 0; d < VC * VW; d++)
#pragma unroll
            for (int i = 0; i < 4; i++) o[r][d][i] *= al;
    }
    auto slot = [&](int s, int r, int d) -> f32x4 & { return sm_o[((s * R + r) * (HSP / 16) + d) * 64 + lane]; };
#pragma unroll
    for (int half = 2; half; half >>= 1) {
        if (wave >= half && wave < 2 * half)
#pragma unroll
            for (int r = 0; r < R; r++)
#pragma unroll
                for (int d = 0; d < VC * VW; d++) slot(wave - half, r, d) = o[r][d];
        __syncthreads();
        if (wave < half)
#pragma unroll
            for (int r = 0; r < R; r++)
#pragma unroll
                for (int d = 0; d < VC * VW; d++) o[r][d] += slot(wave, r, d);
        __syncthreads();
    }
    if (wave) return;
#pragma unroll
    for (int r = 0; r < R; r++) {
        const int row = row0 + 16 * r + n;
        if (row >= p.rows) continue;
        const float il = to_output(p, l[r]);
        if (p.slices > 1 && j == 0) put_sums(a, p, row, m[r], l[r]);
#pragma unroll
        for (int c = 0; c < VC; c++)
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int e = 0; e < VW; e += 4) {
                    const f32x4 *y = &o[r][c * VW + e];
                    put_values<QT>(a, p, row, c * 16 * VW + VW * (4 * j + i) + e,
                                   make_float4(y[0][i] * il, y[1][i] * il, y[2][i] * il, y[3][i] * il));
                }
    }
}

// ---- many rows over bf16 caches: the waves share the rows

#if TREE_HSP == 128
// A step in LDS, 16-bit values in units of eight: K rows in order, V transposed, its positions in the order of the weights'
// lanes: unit 4 u + j of a V row's eight holds positions 4 j + i of tiles 2 u and 2 u + 1.  Sixteen units are all banks
// once; the units of a row change places by its number, so that the sixteen rows of a read are in different ones, and
// the runs of a write in half of them.
struct __align__(16) TreeStep {
    static constexpr int KU = 16; // units of a K row
    static_assert(HSP == 8 * KU, "rows of 128 values");
    uint4 k[64 * KU], v[HSP * 8];
    __device__ __forceinline__ static int k_at(int row, int unit) {
        return row * KU + (unit ^ (row & 15));
    }
    __device__ __forceinline__ static int v_at(int dim, int unit) { return dim * 8 + (unit ^ ((dim >> 1) & 7)); }
};

// A wave has R tiles of 16 rows and takes them through scores, softmax and values 32 positions at a time: few enough
// registers for four waves a SIMD at R = 1, which hide each other's LDS and product latencies.  A step of 64 positions is
// in LDS while the next one's loads are under way: one barrier a step.  LDS bounds it: 16 waves a CU read each step's 32 KB,
// 4096 cycles at 128 bytes a cycle, of about 5500 (448 rows over eight sequences of 0 to 16k positions, 4 kv heads of 128: 121
// us, 358 TFLOP/s, 537 of issued products.  Two tiles in each of four waves read half, with two waves a SIMD: 144 a call
// against 128).
template <int QT, int NW, int R>
__global__ void __launch_bounds__(64 * NW, NW == 4 ? 2 : 4) k_tree_rows(TreeArgs a) {
    constexpr int CT = LLM_BF16;
    using Pc = TreePieces<CT, QT>;
    constexpr int KS = HSP / 32, DT = HSP / 16;
    constexpr bool APART = NW == 8; // waves 4 to 7 fetch K, 0 to 3 V; four waves fetch both
    constexpr int KN = HSP / 8, KL = 64 * KN / 256; // 16-byte pieces of a K row, of a thread
    constexpr int VN = HSP / 4;                     // runs of four dimensions: a thread takes one, at eight positions
    constexpr int VAT = APART ? 0 : 4 * KL, NR = APART ? 16 : 4 * KL + 16;
    __shared__ TreeStep sm[2];
    __shared__ uint32_t sm_bad[2]; // new tokens whose V row is not finite

    const int lane = threadIdx.x & 63, n = lane & 15, j = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Place p;
    if (!place<QT>(a, a.block_rows, p)) return;

    const int row0 = p.row0 + wave * 16 * R;
    const bool works = wave * 16 * R < a.block_rows && row0 < p.rows; // (a wave without rows still fetches)
    const bool does_k = !APART || wave >= 4, does_v = !APART || wave < 4;
    const uint32_t hb = (uint32_t)(a.hs * 2);
    const int64_t at0 = p.b * a.seq + p.h * a.head + (int64_t)p.first * 64 * a.pos;
    const uint8_t *kp = a.k + at0, *vp = a.v + at0;
    int left = min(p.end, p.last * 64) - p.first * 64; // positions not fetched yet
    uint32_t raw[NR];
    // Addresses are formed again at every use, from values that the compiler cannot see through: kept across the loop they
    // would cost the registers that keep it free of spills (a reload waits for the loads under way).
    auto again = [](uint32_t x) {
        asm volatile("" : "+v"(x));
        return x;
    };
    auto load = [&] {
        const uint32_t tid = again(threadIdx.x & 255), ps = a.pos;
        const int here = max(min(left, 64), 0);
        if (does_k) {
            const auto rk = __builtin_amdgcn_make_buffer_rsrc((void *)kp, 0, (int)(here * a.pos), 0x00020000);
#pragma unroll
            for (int i = 0; i < KL; i++) {
                const uint32_t piece = tid + 256 * i, at = piece % KN * 16;
                const auto x = __builtin_amdgcn_raw_buffer_load_b128(rk, (int)(at < hb ? piece / KN * ps + at : OUT_OF_RANGE), 0, 0);
#pragma unroll
                for (int k = 0; k < 4; k++) raw[4 * i + k] = x[k];
            }
        }
        if (does_v) {
            const auto rv = __builtin_amdgcn_make_buffer_rsrc((void *)vp, 0, (int)(here * a.pos), 0x00020000);
            const uint32_t vu = tid / VN, vc = tid % VN; // unit and run
            const uint32_t vo = 8 * vc < hb ? (32 * (vu / 4) + 4 * (vu % 4)) * ps + 8 * vc : OUT_OF_RANGE;
#pragma unroll
            for (int i = 0; i < 8; i++) { // (out of range stays so)
                const auto x = __builtin_amdgcn_raw_buffer_load_b64(rv, (int)(vo + (16 * (i / 4) + i % 4) * ps), 0, 0);
                raw[VAT + 2 * i] = x[0], raw[VAT + 2 * i + 1] = x[1];
            }
        }
        kp += 64 * a.pos;
        vp += 64 * a.pos;
        left -= 64;
    };
    auto store = [&](int step, TreeStep &st) {
        const uint32_t tid = again(threadIdx.x & 255), vu = tid / VN, vc = tid % VN;
        if (does_k)
#pragma unroll
            for (int i = 0; i < KL; i++) {
                const uint32_t piece = tid + 256 * i;
                st.k[st.k_at(piece / KN, piece % KN)] = make_uint4(raw[4 * i], raw[4 * i + 1], raw[4 * i + 2], raw[4 * i + 3]);
            }
        if (does_v) {
            uint32_t *vr = raw + VAT;
            if (step * 64 + 64 > p.len) { // values that are not finite among the new tokens: see k_tree_attention
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const int at = step * 64 + (int)(32 * (vu / 4) + 4 * (vu % 4)) + 16 * (i / 4) + i % 4 - p.len;
                    bool nf = false;
#pragma unroll
                    for (int k = 0; k < 2; k++) {
                        const uint32_t u = vr[2 * i + k];
                        nf |= (u & 0x7f80u) == 0x7f80u || (u & 0x7f800000u) == 0x7f800000u;
                    }
                    if (nf && at >= 0) { // (the row's other values may stay: who sees them becomes NaN)
                        atomicOr(&sm_bad[at / 32], 1u << (at % 32));
                        vr[2 * i] = vr[2 * i + 1] = 0;
                    }
                }
            }
            u32x4 w[4];
#pragma unroll
            for (int i = 0; i < 8; i += 2)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    w[e][i / 2] = __builtin_amdgcn_perm(vr[2 * i + 2 + e / 2], vr[2 * i + e / 2], e % 2 ? 0x07060302 : 0x05040100);
#pragma unroll
            for (int e = 0; e < 4; e++) st.v[st.v_at(4 * vc + e, vu)] = make_uint4(w[e][0], w[e][1], w[e][2], w[e][3]);
        }
    };

    load();
    if (threadIdx.x < 2) sm_bad[threadIdx.x] = 0;
    Frag<CT, Pc::Q> qf[R][KS];
    uint64_t sees[R];
    float cq[R], m[R], l[R];
    f32x4 o[R][DT];
#pragma unroll
    for (int r = 0; r < R; r++) {
        cq[r] = load_queries<CT, QT>(a, p, row0 + 16 * r + n, qf[r], sees[r]);
        m[r] = -INFINITY;
        l[r] = 0.0f;
#pragma unroll
        for (int d = 0; d < DT; d++) o[r][d] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
    }
    __syncthreads();
    store(p.first, sm[0]);
    load();
    __syncthreads();

    for (int step = p.first; step < p.last; step++) {
        const TreeStep &st = sm[(step - p.first) & 1];
        if (works) {
            const bool edge = step * 64 + 64 > p.len;
#pragma unroll 1
            for (int u = 0; u < 2; u++) { // 32 positions
                const int n = again(threadIdx.x & 15), j = again(threadIdx.x & 63) >> 4;
                f32x4 x[R][2];
#pragma unroll
                for (int r = 0; r < R; r++)
#pragma unroll
                    for (int t = 0; t < 2; t++) x[r][t] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int s = 0; s < KS; s++)
#pragma unroll
                    for (int t = 0; t < 2; t++) {
                        Frag<CT, 1> kf;
                        kf.v[0] = *(const u32x4 *)&st.k[st.k_at(32 * u + 16 * t + n, 4 * s + j)];
#pragma unroll
                        for (int r = 0; r < R; r++) x[r][t] = product(kf, qf[r][s], x[r][t]);
                    }
                Frag<CT, Pc::P> pf[R][1];
#pragma unroll
                for (int r = 0; r < R; r++) {
                    uint32_t vis = 0, none = 0;
                    if (edge) vis = seen_bits<8>(p, step * 64 + 32 * u, sees[r]);
                    weights(x[r], cq[r], nullptr, edge, vis, 0, none, m[r], l[r], o[r], pf[r]);
                }
#pragma unroll
                for (int d = 0; d < DT; d++) {
                    Frag<CT, 1> vf;
                    vf.v[0] = *(const u32x4 *)&st.v[st.v_at(16 * d + n, 4 * u + j)];
#pragma unroll
                    for (int r = 0; r < R; r++) o[r][d] = product(vf, pf[r][0], o[r][d]);
                }
            }
        }
        store(step + 1, sm[(step + 1 - p.first) & 1]);
        load();
        __syncthreads();
    }
    if (!works) return;
#pragma unroll
    for (int r = 0; r < R; r++) {
        const int row = row0 + 16 * r + n;
        l[r] = over_groups(l[r], fadd_);
        if (sees[r] & ((uint64_t)sm_bad[1] << 32 | sm_bad[0])) l[r] = NAN;
        if (row >= p.rows) continue;
        const float il = to_output(p, l[r]);
        if (p.slices > 1 && j == 0) put_sums(a, p, row, m[r], l[r]);
#pragma unroll
        for (int d = 0; d < DT; d++)
            put_values<QT>(a, p, row, 16 * d + 4 * j,
                           make_float4(o[r][d][0] * il, o[r][d][1] * il, o[r][d][2] * il, o[r][d][3] * il));
    }
}
#endif

} // namespace

#define TREE_NAME2(n) tree_kernel_##n
#define TREE_NAME(n) TREE_NAME2(n)

TreeKernel TREE_NAME(TREE_HSP)(int type, int q_type, int tiles, int many, size_t *lds) {
#define TREE_PICK(C, Q, T)                                 \
    if (!many && type == C && q_type == Q && tiles == T) { \
        *lds = TreeShape<C, Q, T>::LDS;                    \
        return k_tree_attention<C, Q, T>;                  \
    }
#define TREE_PICK_Q(C, T) TREE_PICK(C, LLM_F32, T) TREE_PICK(C, LLM_BF16, T)
    TREE_PICK_Q(LLM_F32, 1) TREE_PICK_Q(LLM_BF16, 1) TREE_PICK_Q(LLM_I8, 1) TREE_PICK_Q(LLM_E4M3, 1)
#if TREE_HSP <= 128
    TREE_PICK_Q(LLM_I8, 2) TREE_PICK_Q(LLM_E4M3, 2) TREE_PICK(LLM_BF16, LLM_BF16, 2)
#endif
#if TREE_HSP == 128
    *lds = 0;
    if (many == 8 && tiles == 1 && type == LLM_BF16 && q_type == LLM_BF16) return k_tree_rows<LLM_BF16, 8, 1>;
    if (many == 4 && tiles == 2 && type == LLM_BF16 && q_type == LLM_F32) return k_tree_rows<LLM_F32, 4, 2>;
#endif
    return nullptr;
}
