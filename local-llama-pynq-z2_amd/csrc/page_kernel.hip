// Attention of the newest tokens over a cache in pages and over their own rows, head sizes up to PAGE_HSP (a multiple of 64; this
// file is compiled for each).
//
// The rows of a kv head are its query heads' tokens (row = token * group + head of the group), in tiles of 16 on the 16 x 16
// matrix instructions.  A step is a block of 64 positions, with one scale for its K codes and one for its V codes:
//   scores  S^T = K Q^T: K's codes are the A operand, the queries B.  Row r of tile t of K is position 16 (r / 4) + 4 t + r % 4
//           of the block, so that lane 16 j + n owns the scores of row n at positions 16 j .. 16 j + 15.
//   values  O^T += V^T P^T: those are the positions that lane 16 j + n of the A operand has of dimension n of a tile, 16 bytes
//           of a row of the turned V as they lie in the page; the lane's own weights are the B operand as they are.
// Nothing is shuffled or passed through LDS on the way.
//
// A block's weights are taken relative to the row's own largest score in the block: 2^15 at most, fp16 pieces of which hold
// them to 2^-39 of the largest whatever the scales of other blocks are.  The block's products then join the running sums with one
// factor a row, which carries the V scale too: o = o * f + (V^T P^T) * g.
//
// Operands.  int8 and e4m3 codes are exact in fp16.  A query row is scaled by a power of two to the top of fp16's range: fp32
// ones are two pieces (22 bits), bf16 ones one (their 8 bits down to 2^-39 of the largest).  Weights are two pieces.  The new
// tokens' rows go through v_mfma_f32_16x16x4_f32 with fp32 queries and weights.  Maxima, sums and outputs are fp32.
#include "device.h"
#include "page_attention.h"

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

constexpr int HSP = PAGE_HSP;
constexpr int KL = HSP / 64;                   // 16-byte pieces of a K row a lane
constexpr int DT = HSP / 16;                   // tiles of 16 dimensions
constexpr uint32_t OUT_OF_RANGE = 0x80000000u; // a buffer offset past every resource here: the load returns zero

__device__ __forceinline__ uint32_t bf2(float x, float y) { // a float pair in bf16, rounded
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){x, y}, bf16x2));
}
__device__ __forceinline__ float lo16(uint32_t u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float hi16(uint32_t u) { return __uint_as_float(u & 0xffff0000u); }

// x and y as NP fp16 pieces, each word a pair
template <int NP>
__device__ __forceinline__ void split(float x, float y, uint32_t *p) {
#pragma unroll
    for (int i = 0; i < NP; i++) {
        const f16x2 h = __builtin_convertvector((f32x2){x, y}, f16x2);
        p[i] = __builtin_bit_cast(uint32_t, h);
        if (i + 1 < NP) x = fmaf((float)h[0], -1.0f, x), y = fmaf((float)h[1], -1.0f, y);
    }
}
// Eight codes (two words) as fp16.  int8: 0x64 over the byte with its sign bit flipped is 1024 + code + 128.
template <int CT>
__device__ __forceinline__ f16x8 codes8(uint32_t a, uint32_t b) {
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t u = i < 2 ? a : b;
        if constexpr (CT == LLM_I8) {
            const uint32_t h = __builtin_amdgcn_perm(0x64646464u, u ^ 0x80808080u, i % 2 ? 0x04030402u : 0x04010400u);
            r[i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, h) - (f16x2){(_Float16)1152.0f, (_Float16)1152.0f});
        } else {
            r[i] = __builtin_bit_cast(uint32_t, i % 2 ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)u, 1.0f, 1)
                                                      : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)u, 1.0f, 0));
        }
    }
    return __builtin_bit_cast(f16x8, r);
}
__device__ __forceinline__ f32x4 product(f16x8 a, u32x4 b, f32x4 d) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, __builtin_bit_cast(f16x8, b), d, 0, 0, 0);
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

template <int T>
__device__ __forceinline__ float4 load4(const uint8_t *row, int d) { // four values of a row of activations
    if constexpr (T == LLM_F32) return *(const float4 *)(row + (size_t)d * 4);
    const uint2 u = *(const uint2 *)(row + (size_t)d * 2);
    return make_float4(lo16(u.x), hi16(u.x), lo16(u.y), hi16(u.y));
}
template <int T>
__device__ __forceinline__ float load1(const uint8_t *row, int d) {
    if constexpr (T == LLM_F32) return *(const float *)(row + (size_t)d * 4);
    return __uint_as_float((uint32_t)*(const uint16_t *)(row + (size_t)d * 2) << 16);
}
template <int T>
__device__ __forceinline__ void store4(uint8_t *row, int d, float4 y) {
    if constexpr (T == LLM_F32) *(float4 *)(row + (size_t)d * 4) = y;
    else *(uint2 *)(row + (size_t)d * 2) = make_uint2(bf2(y.x, y.y), bf2(y.z, y.w));
}

template <int QT>
struct Pieces {
    static constexpr int Q = QT == LLM_BF16 ? 1 : 2, P = 2; // of a query, of a weight
};

// The running state of a row: the exponent of 2 that its weights are relative to, the lane's part of their sum, the sums of values
// (dimension 16 d + 4 j + i).
struct State {
    float m, l;
    f32x4 o[DT];
};
// What takes the sums so far (f) and a step whose weights are relative to ms (g) to a common exponent.
__device__ __forceinline__ void join(State &s, float ms, float &f, float &g) {
    const float mn = fmaxf(s.m, ms), mu = mn == -INFINITY ? 0.0f : mn;
    f = __builtin_amdgcn_exp2f(s.m - mu);
    g = __builtin_amdgcn_exp2f(ms - mu);
    s.m = mn;
    s.l *= f;
    if (__any(f != 1.0f))
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
            for (int i = 0; i < 4; i++) s.o[d][i] *= f;
}

template <int CT, int QT>
__global__ void __launch_bounds__(256, HSP <= 128 ? 2 : 1) k_page_attention(PageArgs a) {
    using Pc = Pieces<QT>;
    extern __shared__ __align__(16) uint8_t lds[];
    f32x4 *const sm_o = (f32x4 *)lds;                            // [2][DT][64]
    float2 *const sm_ml = (float2 *)(lds + (size_t)2 * DT * 64 * 16); // [4][16]
    const int lane = threadIdx.x & 63, n = lane & 15, j = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int row0 = blockIdx.x * 16, h = blockIdx.y, b = blockIdx.z;
    const int nn = a.n ? min(max(a.n[b], 0), a.max_n) : a.max_n, rows = nn * a.group;
    const int len = (int)min((int64_t)max(a.lens[b], 0), (int64_t)a.per * a.page), steps = (len + PAGE_BLOCK - 1) / PAGE_BLOCK;
    if (a.zero_rest && row0 + 16 > rows) // the rows behind the last token
        for (int e = threadIdx.x * 4; e < 16 * a.hs; e += 1024) {
            const int row = row0 + e / a.hs, t = row / a.group, d = e % a.hs;
            if (row >= rows && row < a.max_n * a.group)
                store4<QT>(a.o + b * a.o_seq + t * a.o_tok + (h * a.group + row - t * a.group) * a.o_head, d,
                           make_float4(0.0f, 0.0f, 0.0f, 0.0f));
        }
    if (row0 >= rows) return;

    // the queries: value e of product s is dimension 64 (s / 2) + 16 j + 8 (s % 2) + e
    const int row = row0 + n, tok = row / a.group;
    const bool ok = row < rows;
    const uint8_t *const qp = a.q + b * a.q_seq + (ok ? tok * a.q_tok + (h * a.group + row - tok * a.group) * a.q_head : 0);
    u32x4 qf[2 * KL][Pc::Q];
    float cq;
    {
        float x[2 * KL][8], mx = 0.0f;
#pragma unroll
        for (int s = 0; s < 2 * KL; s++)
#pragma unroll
            for (int q4 = 0; q4 < 2; q4++) {
                const int d = 64 * (s / 2) + 16 * j + 8 * (s % 2) + 4 * q4;
                const float4 y = ok && d < a.hs ? load4<QT>(qp, d) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                x[s][4 * q4] = y.x, x[s][4 * q4 + 1] = y.y, x[s][4 * q4 + 2] = y.z, x[s][4 * q4 + 3] = y.w;
                mx = fmaxf(mx, fmaxf(fmaxf(fabsf(y.x), fabsf(y.y)), fmaxf(fabsf(y.z), fabsf(y.w))));
            }
        const uint32_t e = exponent(over_groups(mx, fmax_));
        const float to = power_to(e) * a.sign;
        cq = a.c * power_from(e);
#pragma unroll
        for (int s = 0; s < 2 * KL; s++)
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                uint32_t p[Pc::Q];
                split<Pc::Q>(x[s][i] * to, x[s][i + 1] * to, p);
#pragma unroll
                for (int k = 0; k < Pc::Q; k++) qf[s][k][i / 2] = p[k];
            }
    }

    State st;
    st.m = -INFINITY, st.l = 0.0f;
#pragma unroll
    for (int d = 0; d < DT; d++) st.o[d] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
    const uint32_t bytes = PAGE_BLOCK * a.hs;
    for (int step = wave; step < steps; step += 4) {
        const int at = step * PAGE_BLOCK;
        const int page = __builtin_amdgcn_readfirstlane(a.table[(int64_t)b * a.per + at / a.page]), blk = at % a.page / PAGE_BLOCK;
        if ((uint32_t)page >= (uint32_t)a.n_pages) continue;
        const int64_t base = page * a.id + h * a.head + blk * (int64_t)bytes, s_at = page * a.s_id + h * a.s_head + blk;
        const auto rk = __builtin_amdgcn_make_buffer_rsrc((void *)(a.k + base), 0, (int)bytes, 0x00020000);
        const auto rv = __builtin_amdgcn_make_buffer_rsrc((void *)(a.v + base), 0, (int)bytes, 0x00020000);
        const float ks = a.ks[s_at] * cq, vs = a.vs[s_at];
        f32x4 x[4];
        float ms = -INFINITY;
        const int left = len - at; // positions of the block that are there
#pragma unroll
        for (int t = 0; t < 4; t++) {
            x[t] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < KL; i++) {
                const uint32_t d = 64 * i + 16 * j, off = (16 * (n >> 2) + 4 * t + (n & 3)) * a.hs + d;
                const auto c = __builtin_amdgcn_raw_buffer_load_b128(rk, (int)(d < (uint32_t)a.hs ? off : OUT_OF_RANGE), 0, 0);
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const f16x8 kf = codes8<CT>(c[2 * u], c[2 * u + 1]);
#pragma unroll
                    for (int p = Pc::Q - 1; p >= 0; p--) x[t] = product(kf, qf[2 * i + u][p], x[t]); // smallest pieces first
                }
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
                x[t][i] = 16 * j + 4 * t + i < left ? x[t][i] * ks : -INFINITY;
                ms = fmaxf(ms, x[t][i]);
            }
        }
        ms = over_groups(ms, fmax_);
        // A step's largest weight is 2^15, the top of fp16's range.  Scores from 2^23 on have steps of 1 or more, and the
        // difference could be 16: those weights are few and far apart, and their largest is 1.
        ms -= fabsf(ms) < 0x1p23f ? 15.0f : 0.0f;
        const float mu = ms == -INFINITY ? 0.0f : ms;
        float f, g, l = 0.0f;
        u32x4 pf[2][Pc::P];
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                const float w0 = __builtin_amdgcn_exp2f(x[2 * u + e / 4][e % 4] - mu);
                const float w1 = __builtin_amdgcn_exp2f(x[2 * u + e / 4][e % 4 + 1] - mu);
                l += w0;
                l += w1;
                uint32_t p[Pc::P];
                split<Pc::P>(w0, w1, p);
#pragma unroll
                for (int k = 0; k < Pc::P; k++) pf[u][k][e / 2] = p[k];
            }
        join(st, ms, f, g);
        st.l += l * g;
        const float gv = g * vs;
#pragma unroll
        for (int d = 0; d < DT; d++) {
            if (16 * d >= a.hs) break;
            const auto c = __builtin_amdgcn_raw_buffer_load_b128(rv, (16 * d + n) * PAGE_BLOCK + 16 * j, 0, 0);
            uint32_t w[4] = {c[0], c[1], c[2], c[3]};
            if (CT == LLM_E4M3 && left < PAGE_BLOCK) // codes past the end may be NaN: 0 * NaN
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const int have = min(max(left - 16 * j - 4 * k, 0), 4);
                    w[k] &= have == 4 ? 0xffffffffu : (1u << (8 * have)) - 1;
                }
            f32x4 y = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const f16x8 vf = codes8<CT>(w[2 * u], w[2 * u + 1]);
#pragma unroll
                for (int p = Pc::P - 1; p >= 0; p--) y = product(vf, pf[u][p], y);
            }
#pragma unroll
            for (int i = 0; i < 4; i++) st.o[d][i] = fmaf(y[i], gv, st.o[d][i]);
        }
    }

    // the new tokens' own rows, by the wave with the fewest steps: tiles of 16 tokens, all in fp32
    if (a.kr && wave == (steps & 3)) {
        uint64_t sees = 0;
        if (ok) sees = a.mask ? a.mask[(int64_t)b * a.max_n + tok] : ~(uint64_t)0 >> (63 - tok);
        if (nn < 64) sees &= ((uint64_t)1 << nn) - 1;
        const uint8_t *const kp = a.kr + b * a.k_seq + h * a.k_head, *const vp = a.vr + b * a.v_seq + h * a.v_head;
        const int part = a.hs / 4; // dimension part * j + 4 s + i is term j of product 4 s + i
        float c = a.c * a.sign;
        for (int t = 0; t < (nn + 15) / 16; t++) {
            f32x4 y[4];
#pragma unroll
            for (int i = 0; i < 4; i++) y[i] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
            const bool there = 16 * t + n < nn;
            for (int s = 0; s < part; s += 4) { // (four chains: a score is off by half as much as one would be)
                const float4 none = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                const float4 kx = there ? load4<QT>(kp + (16 * t + n) * a.k_tok, part * j + s) : none;
                const float4 qx = ok ? load4<QT>(qp, part * j + s) : none;
                y[0] = __builtin_amdgcn_mfma_f32_16x16x4f32(kx.x, qx.x, y[0], 0, 0, 0);
                y[1] = __builtin_amdgcn_mfma_f32_16x16x4f32(kx.y, qx.y, y[1], 0, 0, 0);
                y[2] = __builtin_amdgcn_mfma_f32_16x16x4f32(kx.z, qx.z, y[2], 0, 0, 0);
                y[3] = __builtin_amdgcn_mfma_f32_16x16x4f32(kx.w, qx.w, y[3], 0, 0, 0);
            }
            const f32x4 sum = (y[0] + y[1]) + (y[2] + y[3]);
            float x[4], ms = -INFINITY;
#pragma unroll
            for (int i = 0; i < 4; i++) { // token 16 t + 4 j + i
                x[i] = (sees >> (16 * t + 4 * j + i)) & 1 ? sum[i] * c : -INFINITY;
                ms = fmaxf(ms, x[i]);
            }
            ms = over_groups(ms, fmax_);
            const float mu = ms == -INFINITY ? 0.0f : ms;
            float f, g, l = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                x[i] = __builtin_amdgcn_exp2f(x[i] - mu);
                l += x[i];
            }
            join(st, ms, f, g);
            uint64_t bad = 0; // tokens whose V row is not finite: who sees them becomes NaN, to the others they are zero
            f32x4 z[DT];
#pragma unroll
            for (int d = 0; d < DT; d++) z[d] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int at = 16 * t + 4 * j + i;
                bool nf = false;
#pragma unroll
                for (int d = 0; d < DT; d++) {
                    if (16 * d >= a.hs) break;
                    float v = at < nn ? load1<QT>(vp + at * a.v_tok, 16 * d + n) : 0.0f;
                    if (!(fabsf(v) < INFINITY)) nf = true, v = 0.0f;
                    z[d] = __builtin_amdgcn_mfma_f32_16x16x4f32(v, x[i], z[d], 0, 0, 0);
                }
                const uint64_t any = __ballot(nf);
#pragma unroll
                for (int k = 0; k < 4; k++)
                    if ((any >> (16 * k)) & 0xffff) bad |= (uint64_t)1 << (16 * t + 4 * k + i);
            }
            st.l = sees & bad ? NAN : st.l + l * g;
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int i = 0; i < 4; i++) st.o[d][i] = fmaf(z[d][i], g, st.o[d][i]);
        }
    }

    // the four waves' sums joined: each scaled to the common maximum, waves 2 and 3 into 0 and 1, then 1 into 0
    st.l = over_groups(st.l, fadd_);
    if (j == 0) sm_ml[wave * 16 + n] = make_float2(st.m, st.l);
    __syncthreads();
    float mn = -INFINITY, l = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; w++) mn = fmaxf(mn, sm_ml[w * 16 + n].x);
    const float mu = mn == -INFINITY ? 0.0f : mn;
#pragma unroll
    for (int w = 0; w < 4; w++) l += sm_ml[w * 16 + n].y * __builtin_amdgcn_exp2f(sm_ml[w * 16 + n].x - mu);
    const float al = __builtin_amdgcn_exp2f(st.m - mu);
#pragma unroll
    for (int d = 0; d < DT; d++)
#pragma unroll
        for (int i = 0; i < 4; i++) st.o[d][i] *= al;
#pragma unroll
    for (int half = 2; half; half >>= 1) {
        if (wave >= half && wave < 2 * half)
#pragma unroll
            for (int d = 0; d < DT; d++) sm_o[((wave - half) * DT + d) * 64 + lane] = st.o[d];
        __syncthreads();
        if (wave < half)
#pragma unroll
            for (int d = 0; d < DT; d++) st.o[d] += sm_o[(wave * DT + d) * 64 + lane];
        __syncthreads();
    }
    if (wave || !ok) return;
    const float il = l == 0.0f ? 0.0f : 1.0f / l;
    uint8_t *const op = a.o + b * a.o_seq + tok * a.o_tok + (h * a.group + row - tok * a.group) * a.o_head;
#pragma unroll
    for (int d = 0; d < DT; d++)
        if (16 * d < a.hs)
            store4<QT>(op, 16 * d + 4 * j, make_float4(st.o[d][0] * il, st.o[d][1] * il, st.o[d][2] * il, st.o[d][3] * il));
}

} // namespace

#define PAGE_NAME2(n) page_kernel_##n
#define PAGE_NAME(n) PAGE_NAME2(n)

PageKernel PAGE_NAME(PAGE_HSP)(int type, int q_type, size_t *lds) {
    *lds = (size_t)2 * DT * 64 * 16 + 4 * 16 * 8;
    if (type == LLM_I8) return q_type == LLM_F32 ? k_page_attention<LLM_I8, LLM_F32> : k_page_attention<LLM_I8, LLM_BF16>;
    return q_type == LLM_F32 ? k_page_attention<LLM_E4M3, LLM_F32> : k_page_attention<LLM_E4M3, LLM_BF16>;
}
