// Attention of drafted tokens over a cache, head sizes up to TREE_HSP (a multiple of 64; this file is compiled for each).
//
// The rows of a kv head are its query heads' tokens (row = token * group + head of the group), in tiles of 16; a wave takes
// one or two tiles over every fourth step of TP positions of its block's slice, with one running maximum and sum a row.
// Everything stays in registers, nothing crosses lanes but the maximum:
//   scores  S^T = K Q^T: K rows are the A operand, lane 16 j + n has 16-byte pieces of position n (piece j of every four),
//           so a row's bytes are read whole and once; Q's lanes hold the same values of row n.  The lane then owns the
//           scores of row n at positions 4 j + i of every 16.
//   values  O^T += V^T P^T: its own probabilities are the B operand as they are (eight positions: 4 j + i of two tiles of
//           16).  A's lane n needs those positions of one dimension: it reads 4 or 8 neighbouring dimensions of each of the
//           positions and pairs the registers of two positions, which transposes for nothing.
// int8 and e4m3 codes and bf16 values are exact in bf16, so the products run on v_mfma_f32_16x16x32_bf16 with the fp32 side
// (queries, probabilities * V scale) in bf16 pieces: three hold all 24 bits; 16-bit queries are one, their probabilities
// two (2^-16, against the output's 2^-9).  fp32 caches take v_mfma_f32_16x16x4_f32.
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

// a float pair in bf16, rounded; exact for codes
__device__ __forceinline__ uint32_t bf2(float x, float y) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){x, y}, bf16x2));
}
__device__ __forceinline__ float lo16(uint32_t u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float hi16(uint32_t u) { return __uint_as_float(u & 0xffff0000u); }
// x and y as NP bf16 pieces, each word a pair
template <int NP>
__device__ __forceinline__ void split(float x, float y, uint32_t *p) {
#pragma unroll
    for (int i = 0; i < NP; i++) {
        p[i] = bf2(x, y);
        if (i + 1 < NP) x -= lo16(p[i]), y -= hi16(p[i]);
    }
}
template <int CT, int BYTE>
__device__ __forceinline__ float code(uint32_t w) { // byte BYTE's value
    if constexpr (CT == LLM_I8) return (float)(int8_t)(w >> (8 * BYTE));
    else {
        const auto f = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, BYTE >= 2);
        return f[BYTE & 1];
    }
}
template <int CT>
__device__ __forceinline__ void codes4(uint32_t w, uint32_t *p) { // four codes as two bf16 pairs
    p[0] = bf2(code<CT, 0>(w), code<CT, 1>(w));
    p[1] = bf2(code<CT, 2>(w), code<CT, 3>(w));
}

// An operand of a product over 32 terms: eight values a lane.  fp32: as they are, else NP bf16 pieces.
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
        for (int p = NP - 1; p >= 0; p--) // smallest pieces first
            d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a.v[0]),
                                                        __builtin_bit_cast(bf16x8, b.v[p]), d, 0, 0, 0);
    }
    return d;
}
template <int CT, int NP>
__device__ __forceinline__ void fill(Frag<CT, NP> &f, const float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        if constexpr (CT == LLM_F32) f.v[i] = x[i], f.v[i + 1] = x[i + 1];
        else {
            uint32_t p[NP];
            split<NP>(x[i], x[i + 1], p);
#pragma unroll
            for (int k = 0; k < NP; k++) f.v[k][i / 2] = p[k];
        }
    }
}

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

template <int CT, int QT, int R>
struct TreeShape {
    static constexpr int ES = CT == LLM_F32 ? 4 : CT == LLM_BF16 ? 2 : 1;
    static constexpr int TP = tree_positions(HSP, CT), NT = TP / 16; // positions a step, their tiles of 16
    static constexpr int KL = HSP * ES / 64;                         // 16-byte pieces of a K row a lane
    static constexpr int KS = HSP / 32;                              // products of a score
    static constexpr int VW = HSP % 128 ? 4 : 8;                     // neighbouring dimensions a lane of V
    static constexpr int VC = HSP / (16 * VW), VR = VW * ES / 4;     // runs of them, a run's registers
    static constexpr int NPQ = QT == LLM_BF16 ? 1 : 3, NPP = QT == LLM_BF16 ? 2 : 3;
    static constexpr size_t LDS = (size_t)2 * R * (HSP / 16) * 64 * 16 + 4 * R * 16 * 8 + 4 * 2 * 64 * 4;
};

template <int CT, int QT, int R>
__global__ void __launch_bounds__(256) k_tree_attention(TreeArgs a) {
    using Sh = TreeShape<CT, QT, R>;
    constexpr int ES = Sh::ES, TP = Sh::TP, NT = Sh::NT, KL = Sh::KL, KS = Sh::KS, VW = Sh::VW, VC = Sh::VC, VR = Sh::VR;
    constexpr int NPQ = Sh::NPQ, NPP = Sh::NPP;
    constexpr bool SCALED = ES == 1;
    extern __shared__ __align__(16) uint8_t lds[];
    f32x4 *const sm_o = (f32x4 *)lds;                                        // [2][R][HSP / 16][64]
    float *const sm_ml = (float *)(lds + (size_t)2 * R * (HSP / 16) * 64 * 16); // [4][R][16][2]
    float *const sm_s = sm_ml + 4 * R * 16 * 2;                              // [4][2][64]

    const int lane = threadIdx.x & 63, n = lane & 15, j = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int id = blockIdx.x;
    const int split_id = id % a.splits;
    id /= a.splits;
    const int h = id % a.n_kv, b = id / a.n_kv;
    const int len = min(max(a.lens[b], 0), a.ctx);
    const int nn = a.n ? min(max(a.n[b], 0), a.max_n) : a.max_n;
    const int end = min((int64_t)len + nn, (int64_t)a.ctx), rows = nn * a.group, row0 = blockIdx.y * 16 * R;
    int steps;
    const int slices = tree_slices(end, TP, a.splits, &steps);
    if (a.zero_rest && split_id == 0) { // the rows behind the last token
        for (int e = threadIdx.x * 4; e < 16 * R * a.hs; e += 1024) {
            const int row = row0 + e / a.hs, t = row / a.group, d = e - (row - row0) * a.hs;
            if (row < rows || row >= a.max_n * a.group) continue;
            uint8_t *op = a.o + b * a.o_seq + t * a.o_tok + (h * a.group + row - t * a.group) * a.o_head;
            if constexpr (QT == LLM_F32) *(float4 *)(op + (size_t)d * 4) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            else *(uint2 *)(op + (size_t)d * 2) = make_uint2(0, 0);
        }
    }
    if (row0 >= rows || split_id >= slices) return;
    const int all = (end + TP - 1) / TP, first = split_id * steps, last = min(first + steps, all);

    // the rows of this wave's tiles: queries, and what each sees among the new tokens
    Frag<CT, NPQ> qf[R][KS];
    uint64_t sees[R];
#pragma unroll
    for (int r = 0; r < R; r++) {
        const int row = row0 + 16 * r + n, t = row / a.group, g = row - t * a.group;
        const bool ok = row < rows;
        sees[r] = 0;
        if (ok) sees[r] = a.mask ? a.mask[(int64_t)b * a.max_n + t] : ~(uint64_t)0 >> (63 - t);
        const uint8_t *qp = a.q + b * a.q_seq + (ok ? t * a.q_tok + (h * a.group + g) * a.q_head : 0);
#pragma unroll
        for (int s = 0; s < KS; s++) {
            float x[8];
#pragma unroll
            for (int q4 = 0; q4 < 2; q4++) {
                // the lane's values of product s are those of its pieces of K
                const int d = CT == LLM_F32 ? 32 * s + 16 * q4 + 4 * j
                              : CT == LLM_BF16 ? 32 * s + 8 * j + 4 * q4 : 64 * (s / 2) + 16 * j + 8 * (s % 2) + 4 * q4;
                float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (ok && d < a.hs) {
                    if constexpr (QT == LLM_F32) v = *(const float4 *)(qp + (size_t)d * 4);
                    else {
                        const uint2 u = *(const uint2 *)(qp + (size_t)d * 2);
                        v = make_float4(lo16(u.x), hi16(u.x), lo16(u.y), hi16(u.y));
                    }
                }
                x[4 * q4] = v.x, x[4 * q4 + 1] = v.y, x[4 * q4 + 2] = v.z, x[4 * q4 + 3] = v.w;
            }
            fill(qf[r][s], x);
        }
    }

    const uint8_t *const kb = a.k + b * a.seq + h * a.head, *const vb = a.v + b * a.seq + h * a.head;
    const float *ksb = nullptr, *vsb = nullptr;
    if constexpr (SCALED) {
        ksb = a.ks + b * a.s_seq + h * a.s_head;
        vsb = a.vs + b * a.s_seq + h * a.s_head;
    }
    const uint32_t ps = (uint32_t)a.pos, hb = (uint32_t)(a.hs * ES);
    u32x4 kr[NT][KL];
    uint32_t vr[TP / 4][VC][VR];
    uint32_t skr = 0, svr = 0;

    // A step's rows through buffers that hold its positions and no more: what lies past them reads as zero.
    auto rsrc = [&](const void *p, int64_t stride, int step) {
        const int left = step < last ? min(TP, end - step * TP) : 0;
        return __builtin_amdgcn_make_buffer_rsrc((void *)((const uint8_t *)p + (int64_t)step * TP * stride), 0,
                                                 (int)(left * stride), 0x00020000);
    };
    auto load_k = [&](int step) {
        const auto rs = rsrc(kb, a.pos, step);
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int p = 0; p < KL; p++) {
                const uint32_t at = 64 * p + 16 * j;
                const auto x = __builtin_amdgcn_raw_buffer_load_b128(
                    rs, (int)(at < hb ? (16 * t + n) * ps + at : OUT_OF_RANGE), 0, 0);
                kr[t][p] = (u32x4){x[0], x[1], x[2], x[3]};
            }
        if constexpr (SCALED)
            skr = __builtin_amdgcn_raw_buffer_load_b32(rsrc(ksb, a.s_pos * 4, step), (int)(lane * (uint32_t)a.s_pos * 4), 0, 0);
    };
    auto load_v = [&](int step) {
        const auto rs = rsrc(vb, a.pos, step);
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
                    for (int p = 0; p < VR / 4; p++) {
                        const auto u = __builtin_amdgcn_raw_buffer_load_b128(rs, (int)(off + 16 * p), 0, 0);
#pragma unroll
                        for (int k = 0; k < 4; k++) vr[x][c][4 * p + k] = u[k];
                    }
                }
            }
        if constexpr (SCALED)
            svr = __builtin_amdgcn_raw_buffer_load_b32(rsrc(vsb, a.s_pos * 4, step), (int)(lane * (uint32_t)a.s_pos * 4), 0, 0);
    };

    f32x4 o[R][VC][VW];
    float m[R], l[R];
#pragma unroll
    for (int r = 0; r < R; r++) {
        m[r] = -INFINITY;
        l[r] = 0.0f;
#pragma unroll
        for (int c = 0; c < VC; c++)
#pragma unroll
            for (int e = 0; e < VW; e++) o[r][c][e] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
    }
    float *const my_s = sm_s + wave * 128;

    int step = first + wave;
    if (step < last) {
        load_k(step);
        load_v(step);
    }
    for (; step < last; step += 4) {
        const int p0 = step * TP;
        const bool edge = p0 + TP > len; // new tokens or the end among the positions
        if constexpr (SCALED) {
            my_s[lane] = __uint_as_float(skr);
            my_s[64 + lane] = __uint_as_float(svr);
            wave_lds_fence();
        }
        f32x4 x[R][NT];
#pragma unroll
        for (int t = 0; t < NT; t++) {
#pragma unroll
            for (int r = 0; r < R; r++) x[r][t] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int s = 0; s < KS; s++) {
                Frag<CT, 1> kf;
                if constexpr (CT == LLM_F32) {
#pragma unroll
                    for (int i = 0; i < 8; i++) kf.v[i] = __uint_as_float(kr[t][2 * s + i / 4][i % 4]);
                } else if constexpr (CT == LLM_BF16) {
                    kf.v[0] = kr[t][s];
                } else {
                    uint32_t p[4];
                    codes4<CT>(kr[t][s / 2][2 * (s % 2)], p);
                    codes4<CT>(kr[t][s / 2][2 * (s % 2) + 1], p + 2);
                    kf.v[0] = (u32x4){p[0], p[1], p[2], p[3]};
                }
#pragma unroll
                for (int r = 0; r < R; r++) x[r][t] = product(kf, qf[r][s], x[r][t]);
            }
        }
        load_k(step + 4);

        uint32_t vis[R]; // edge: bit 4 t + i, whether the row sees the position
        uint64_t bad = 0; // edge, fp32 and bf16: new tokens whose V row is not finite
#pragma unroll
        for (int r = 0; r < R; r++) vis[r] = 0;
        if (edge) {
#pragma unroll
            for (int r = 0; r < R; r++)
#pragma unroll
                for (int i = 0; i < TP / 4; i++) {
                    const int p = p0 + 16 * (i / 4) + 4 * j + i % 4;
                    const bool v = p < len || (p < end && ((sees[r] >> (p - len)) & 1));
                    vis[r] |= (uint32_t)v << i;
                }
            if constexpr (!SCALED) {
                // a value that is not finite would reach the rows that do not see it as 0 * inf: taken out here, and
                // the rows that do see it become NaN at the end
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
                            else nf |= (u & 0x7f80u) == 0x7f80u || (u & 0x7f800000u) == 0x7f800000u;
                        }
                    nf = nf && q + 4 * j >= len;
                    const uint64_t any = __ballot(nf);
                    if (any) {
#pragma unroll
                        for (int g = 0; g < 4; g++)
                            if ((any >> (16 * g)) & 0xffff) bad |= (uint64_t)1 << (q + 4 * g - len);
                        if ((any >> (16 * j)) & 0xffff)
#pragma unroll
                            for (int c = 0; c < VC; c++)
#pragma unroll
                                for (int k = 0; k < VR; k++) vr[i][c][k] = 0;
                    }
                }
            }
        }

        Frag<CT, NPP> pf[R][NT / 2];
#pragma unroll
        for (int r = 0; r < R; r++) {
            float mx = -INFINITY;
#pragma unroll
            for (int t = 0; t < NT; t++) {
                f32x4 sk = (f32x4){a.c, a.c, a.c, a.c};
                if constexpr (SCALED) {
                    const f32x4 s4 = *(const f32x4 *)(my_s + 16 * t + 4 * j);
#pragma unroll
                    for (int i = 0; i < 4; i++) sk[i] = s4[i] * a.c;
                }
#pragma unroll
                for (int i = 0; i < 4; i++) x[r][t][i] *= sk[i];
                if (edge)
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (!((vis[r] >> (4 * t + i)) & 1)) x[r][t][i] = -INFINITY;
#pragma unroll
                for (int i = 0; i < 4; i++) mx = fmaxf(mx, x[r][t][i]);
            }
            mx = over_groups(mx, fmax_);
            const float mn = fmaxf(m[r], mx), mu = mn == -INFINITY ? 0.0f : mn;
            if (__any(mn > m[r])) {
                const float al = __builtin_amdgcn_exp2f(m[r] - mu);
                l[r] *= al;
#pragma unroll
                for (int c = 0; c < VC; c++)
#pragma unroll
                    for (int e = 0; e < VW; e++)
#pragma unroll
                        for (int i = 0; i < 4; i++) o[r][c][e][i] *= al;
                m[r] = mn;
            }
            float w[TP / 4];
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    w[4 * t + i] = __builtin_amdgcn_exp2f(x[r][t][i] - mu);
                    l[r] += w[4 * t + i];
                }
            if constexpr (SCALED) {
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    const f32x4 s4 = *(const f32x4 *)(my_s + 64 + 16 * t + 4 * j);
#pragma unroll
                    for (int i = 0; i < 4; i++) w[4 * t + i] *= s4[i];
                }
                if (edge) // (0 * a scale that is not finite)
#pragma unroll
                    for (int i = 0; i < TP / 4; i++)
                        if (!((vis[r] >> i) & 1)) w[i] = 0.0f;
            }
#pragma unroll
            for (int u = 0; u < NT / 2; u++) {
                float y[8];
#pragma unroll
                for (int i = 0; i < 8; i++) y[i] = w[8 * u + i];
                fill(pf[r][u], y);
            }
            if (!SCALED && (sees[r] & bad)) l[r] = NAN;
        }

#pragma unroll
        for (int u = 0; u < NT / 2; u++)
#pragma unroll
            for (int c = 0; c < VC; c++)
#pragma unroll
                for (int e = 0; e < VW; e++) {
                    Frag<CT, 1> vf;
#pragma unroll
                    for (int i = 0; i < 8; i += 2) {
                        const uint32_t *v0 = vr[8 * u + i][c], *v1 = vr[8 * u + i + 1][c];
                        if constexpr (CT == LLM_F32) {
                            vf.v[i] = __uint_as_float(v0[e]), vf.v[i + 1] = __uint_as_float(v1[e]);
                        } else if constexpr (CT == LLM_BF16) {
                            vf.v[0][i / 2] = e % 2 ? __builtin_amdgcn_perm(v1[e / 2], v0[e / 2], 0x07060302)
                                                   : __builtin_amdgcn_perm(v1[e / 2], v0[e / 2], 0x05040100);
                        } else {
                            const uint32_t a0 = v0[e / 4], a1 = v1[e / 4];
                            vf.v[0][i / 2] = e % 4 == 0   ? bf2(code<CT, 0>(a0), code<CT, 0>(a1))
                                             : e % 4 == 1 ? bf2(code<CT, 1>(a0), code<CT, 1>(a1))
                                             : e % 4 == 2 ? bf2(code<CT, 2>(a0), code<CT, 2>(a1))
                                                          : bf2(code<CT, 3>(a0), code<CT, 3>(a1));
                        }
                    }
#pragma unroll
                    for (int r = 0; r < R; r++) o[r][c][e] = product(vf, pf[r][u], o[r][c][e]);
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
        const float al = __builtin_amdgcn_exp2f(m[r] - mu);
        l[r] = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; w++) l[r] += lw[w] * __builtin_amdgcn_exp2f(mw[w] - mu);
        m[r] = mn;
#pragma unroll
        for (int c = 0; c < VC; c++)
#pragma unroll
            for (int e = 0; e < VW; e++)
#pragma unroll
                for (int i = 0; i < 4; i++) o[r][c][e][i] *= al;
    }
    auto slot = [&](int s, int r, int c, int e) -> f32x4 & { return sm_o[((s * R + r) * (HSP / 16) + c * VW + e) * 64 + lane]; };
#pragma unroll
    for (int half = 2; half; half >>= 1) {
        if (wave >= half && wave < 2 * half)
#pragma unroll
            for (int r = 0; r < R; r++)
#pragma unroll
                for (int c = 0; c < VC; c++)
#pragma unroll
                    for (int e = 0; e < VW; e++) slot(wave - half, r, c, e) = o[r][c][e];
        __syncthreads();
        if (wave < half)
#pragma unroll
            for (int r = 0; r < R; r++)
#pragma unroll
                for (int c = 0; c < VC; c++)
#pragma unroll
                    for (int e = 0; e < VW; e++) o[r][c][e] += slot(wave, r, c, e);
        __syncthreads();
    }
    if (wave) return;
#pragma unroll
    for (int r = 0; r < R; r++) {
        const int row = row0 + 16 * r + n, t = row / a.group, g = row - t * a.group;
        if (row >= rows) continue;
        // a row that sees nothing has the sum 0
        const float il = slices > 1 ? 1.0f : l[r] == 0.0f ? 0.0f : 1.0f / l[r];
        const int64_t part = (((int64_t)b * a.n_kv + h) * a.splits + split_id) * a.max_n * a.group + row;
        if (slices > 1 && j == 0) {
            a.ml[2 * part] = m[r];
            a.ml[2 * part + 1] = l[r];
        }
        uint8_t *op = a.o + b * a.o_seq + t * a.o_tok + (h * a.group + g) * a.o_head;
#pragma unroll
        for (int c = 0; c < VC; c++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int d = c * 16 * VW + VW * (4 * j + i);
                if (d >= a.hs) continue;
#pragma unroll
                for (int e = 0; e < VW; e += 4) {
                    const float4 y = make_float4(o[r][c][e][i] * il, o[r][c][e + 1][i] * il, o[r][c][e + 2][i] * il,
                                                 o[r][c][e + 3][i] * il);
                    if (slices > 1) *(float4 *)(a.acc + part * a.hs + d + e) = y;
                    else if constexpr (QT == LLM_F32) *(float4 *)(op + (size_t)(d + e) * 4) = y;
                    else *(uint2 *)(op + (size_t)(d + e) * 2) = make_uint2(bf2(y.x, y.y), bf2(y.z, y.w));
                }
            }
    }
}

} // namespace

#define TREE_NAME2(n) tree_kernel_##n
#define TREE_NAME(n) TREE_NAME2(n)

TreeKernel TREE_NAME(TREE_HSP)(int type, int q_type, int tiles, size_t *lds) {
#define TREE_PICK(C, Q, T)                           \
    if (type == C && q_type == Q && tiles == T) {    \
        *lds = TreeShape<C, Q, T>::LDS;              \
        return k_tree_attention<C, Q, T>;            \
    }
#define TREE_PICK_Q(C, T) TREE_PICK(C, LLM_F32, T) TREE_PICK(C, LLM_BF16, T)
    TREE_PICK_Q(LLM_F32, 1) TREE_PICK_Q(LLM_BF16, 1) TREE_PICK_Q(LLM_I8, 1) TREE_PICK_Q(LLM_E4M3, 1)
#if TREE_HSP <= 128
    TREE_PICK_Q(LLM_F32, 2) TREE_PICK_Q(LLM_BF16, 2) TREE_PICK_Q(LLM_I8, 2) TREE_PICK_Q(LLM_E4M3, 2)
#endif
    return nullptr;
#undef TREE_PICK
#undef TREE_PICK_Q
}
