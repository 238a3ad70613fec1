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
// ones are two pieces (22 bits), bf16 ones one (their 8 bits down to 2^-39 of the largest).  Weights are two pieces, of bf16 rows
// too: one (11 bits) gave 3% of a batch's bf16 outputs another rounding than the exact result, two give 0.1%, at the price of 16 us in
// 138 for eight trees of 64 over int8 pages.  The new tokens' rows go through v_mfma_f32_16x16x4_f32 with fp32 queries and weights.
// Maxima, sums and outputs are fp32.
//
// What bounds it.  Few rows: memory (32 decode steps of 7 query heads a kv head over 131 MB of e4m3 pages: 27.4 us, 4.8 TB/s), or
// with few positions a chain of dependent loads (arguments, length, page, codes, the new row: 7.0 us for 203 positions of heads
// of 64, 5.6 of it with none).  Many rows: vector instructions, which turn codes into fp16 and make the weights (a step of two
// tiles of bf16 rows over int8 pages: 676, of which 320 are for the codes, beside 104 products); 448 rows of each of eight
// sequences over up to 16k positions: 139 us, 312 TFLOP/s.
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
// Eight codes (two words) as fp16.  int8, its sign bit flipped, is code + 128 in a byte: 0x64 over it is 1024 + code + 128, from
// which 1152 is taken.
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

// an operand of ones
__device__ __forceinline__ f16x8 ones() {
    const uint32_t u = 0x3c003c00u;
    return __builtin_bit_cast(f16x8, (u32x4){u, u, u, u});
}

// The exponent field of a power of two that takes a magnitude to [2^14, 2^15) (magnitudes below 2^-112 to less, but all of
// their bits into fp16's range; infinities stay).
__device__ __forceinline__ uint32_t power_to(float x) { return min(268u - ((__float_as_uint(x) >> 23) & 0xff), 253u); }

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

// Pieces of a query (16-bit ones are exact in one) and of a weight.
template <int QT>
constexpr int Q_PIECES = QT == LLM_BF16 ? 1 : 2;
constexpr int P_PIECES = 2;

// The running state of a row: the exponent of 2 that its weights are relative to, their sum, the sums of values (dimension
// 16 d + 4 j + i).
struct State {
    float m, l;
    f32x4 o[DT];
};
// What takes the sums so far (f) and a step whose weights are relative to ms (g) to a common exponent.  It is set so that the step's
// largest weight, 2^15, counts as 2^-8, and stays until one would count as more than 1: few steps do, and the factor 1 is not
// multiplied by.  (Sums of weights up to 1 overflow where the values' own would.)
__device__ __forceinline__ void join(State &s, float ms, float &f, float &g) {
    const float mn = ms > s.m - 15.0f ? ms + 23.0f : s.m, mu = mn == -INFINITY ? 0.0f : mn;
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

// A value that the wave's lanes share and nothing writes while the kernel runs, through the scalar unit.
template <typename T>
__device__ __forceinline__ T uniform(const T *p) {
    return *(const __attribute__((address_space(4))) T *)(uintptr_t)p;
}

// Where a workgroup works: sequence, kv head, slice (`id` of all), first row; the slice's blocks and whether the
// new tokens' rows are its, the sequence's positions and rows.
struct Place {
    int b, h, split, id, row0, len, nn, rows, slices, first, last;
    bool fresh;
};

// Blocks go to the eight XCDs in turn.  The row blocks of a slice follow each other on one, whose L2 then holds the slice's
// pages for all of them.
template <int QT>
__device__ __forceinline__ bool place(const PageArgs &a, int block_rows, Place &p) {
    const uint32_t k = blockIdx.x >> 3, kr = k / (uint32_t)a.row_blocks, id = kr * 8 + (blockIdx.x & 7);
    int steps = 0x7fffffff;
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
    p.row0 = (int)(k - kr * a.row_blocks) * block_rows;
    if (a.cap && a.n_seq > 1 && p.split == 0 && p.row0 == 0 && threadIdx.x == 0) // (for the join)
        a.plan[p.b * a.n_kv + p.h] = make_int2((int)id, p.slices);
    p.nn = a.n ? min(max(a.n[p.b], 0), a.max_n) : a.max_n;
    p.rows = p.nn * a.group;
    if (a.zero_rest && p.split == 0 && p.rows < a.max_n * a.group && p.row0 + block_rows > p.rows) // the rows behind the last token
        for (int e = threadIdx.x * 4; e < block_rows * a.hs; e += 1024) {
            const int row = p.row0 + e / a.hs, t = row / a.group, d = e % a.hs;
            if (row >= p.rows && row < a.max_n * a.group)
                store4<QT>(a.o + p.b * a.o_seq + t * a.o_tok + (p.h * a.group + row - t * a.group) * a.o_head, d,
                           make_float4(0.0f, 0.0f, 0.0f, 0.0f));
        }
    p.len = page_len(a, p.b);
    const int all = (p.len + PAGE_BLOCK - 1) / PAGE_BLOCK, end = (int)min((int64_t)(p.split + 1) * steps, (int64_t)0x7fffffff);
    p.first = p.split ? min(p.split * steps, all) : 0;
    p.last = min(end, all);
    p.fresh = new_steps(a, p.nn) && p.split == p.slices - 1; // (the steps behind the blocks)
    return p.row0 < p.rows;
}

// Sums of row `row` at dimensions d .. d + 3: the output where there is one slice, else this slice's partial sums.
template <int QT>
__device__ __forceinline__ void put_values(const PageArgs &a, const Place &p, int row, int d, float4 y) {
    if (d >= a.hs) return;
    if (p.slices > 1) {
        const int64_t part = (int64_t)p.id * a.max_n * a.group + row;
        *(float4 *)(a.acc + part * a.hs + d) = y;
        return;
    }
    const int t = row / a.group;
    store4<QT>(a.o + p.b * a.o_seq + t * a.o_tok + (p.h * a.group + row - t * a.group) * a.o_head, d, y);
}
template <int QT>
__device__ __forceinline__ void put_row(const PageArgs &a, const Place &p, int row, int j, const State &s, float l) {
    if (p.slices > 1 && j == 0) {
        const int64_t part = (int64_t)p.id * a.max_n * a.group + row;
        a.ml[2 * part] = s.m;
        a.ml[2 * part + 1] = l;
    }
    const float il = p.slices > 1 ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l; // (a row that sees nothing has the sum 0)
#pragma unroll
    for (int d = 0; d < DT; d++)
        put_values<QT>(a, p, row, 16 * d + 4 * j,
                       make_float4(s.o[d][0] * il, s.o[d][1] * il, s.o[d][2] * il, s.o[d][3] * il));
}

// The new tokens' own rows, all in fp32: tiles of 16 tokens, from `first` on every `stride`-th.  A tile's K and V values are
// loaded while the one before is worked on; what is not there reads a row that is.  EARLY: the first one's before it is known
// whether the rows see it (one decode step of heads of 128 over 200 positions: 9.6 us instead of 10.6; two tiles would spill).
template <int QT, bool EARLY>
__device__ __forceinline__ void new_rows(const PageArgs &a, const Place &p, int first, int stride, const uint8_t *qp, bool ok, int tok,
                                         State &st) {
    const int lane = threadIdx.x & 63, n = lane & 15, j = lane >> 4, nn = p.nn, tiles = (nn + 15) / 16;
    const uint8_t *const kp = a.kr + p.b * a.k_seq + p.h * a.k_head, *const vp = a.vr + p.b * a.v_seq + p.h * a.v_head;
    const int part = a.hs / 4; // dimension part * j + 4 s + i is term j of product 4 s + i
    const float c = a.c * a.sign;
    float4 kx[HSP / 16], qx[HSP / 16];
    float v[4][DT];
    auto load = [&](int t) {
        const uint8_t *const krow = kp + min(16 * t + n, nn - 1) * a.k_tok;
#pragma unroll
        for (int s = 0; s < HSP / 16; s++) kx[s] = load4<QT>(krow, part * j + (4 * s < part ? 4 * s : 0));
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (16 * t + i >= nn) break; // (tokens 16 t + 4 j + i, of all lane groups)
            const uint8_t *const vrow = vp + min(16 * t + 4 * j + i, nn - 1) * a.v_tok;
#pragma unroll
            for (int d = 0; d < DT; d++) v[i][d] = load1<QT>(vrow, (16 * d < a.hs ? 16 * d : 0) + n);
        }
    };
    auto load_q = [&] {
#pragma unroll
        for (int s = 0; s < HSP / 16; s++) {
            qx[s] = load4<QT>(qp, part * j + (4 * s < part ? 4 * s : 0));
            if (!ok || 4 * s >= part) qx[s] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
    };
    if (first >= tiles) return;
    if (EARLY) {
        load(first);
        load_q();
    }
    uint64_t sees = 0;
    if (ok) sees = a.mask ? a.mask[(int64_t)p.b * a.max_n + tok] : ~(uint64_t)0 >> (63 - tok);
    if (nn < 64) sees &= ((uint64_t)1 << nn) - 1;
    // (tiles of which no row sees a token are left out)
    auto next = [&](int t) {
        while (t < tiles && !__any((int)(sees >> 16 * t) & 0xffff)) t += stride;
        return t;
    };
    int t = next(first);
    if (t >= tiles) return;
    if (!EARLY || t != first) load(t);
    if (!EARLY) load_q();
    for (;;) {
        f32x4 y[4];
#pragma unroll
        for (int i = 0; i < 4; i++) y[i] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int s = 0; s < HSP / 16; s++) // (four chains: a score is off by half as much as one would be)
            if (4 * s < part) {
                y[0] = __builtin_amdgcn_mfma_f32_16x16x4f32(kx[s].x, qx[s].x, y[0], 0, 0, 0);
                y[1] = __builtin_amdgcn_mfma_f32_16x16x4f32(kx[s].y, qx[s].y, y[1], 0, 0, 0);
                y[2] = __builtin_amdgcn_mfma_f32_16x16x4f32(kx[s].z, qx[s].z, y[2], 0, 0, 0);
                y[3] = __builtin_amdgcn_mfma_f32_16x16x4f32(kx[s].w, qx[s].w, y[3], 0, 0, 0);
            }
        const f32x4 sum = (y[0] + y[1]) + (y[2] + y[3]);
        const uint32_t mine = (uint32_t)(sees >> (16 * t + 4 * j));
        float x[4], ms = -INFINITY;
#pragma unroll
        for (int i = 0; i < 4; i++) { // token 16 t + 4 j + i
            x[i] = mine & (1u << i) ? sum[i] * c : -INFINITY;
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
        l = over_groups(l, fadd_);
        join(st, ms, f, g);
        bool nf[4] = {false, false, false, false};
        f32x4 z[DT];
#pragma unroll
        for (int d = 0; d < DT; d++) z[d] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (16 * t + i >= nn) break;
#pragma unroll
            for (int d = 0; d < DT; d++) { // a value that is not finite is zero here
                const bool bad = !(fabsf(v[i][d]) < INFINITY);
                nf[i] |= bad;
                z[d] = __builtin_amdgcn_mfma_f32_16x16x4f32(bad ? 0.0f : v[i][d], x[i], z[d], 0, 0, 0);
            }
        }
        const int now = t;
        t = next(t + stride);
        if (t < tiles) load(t);
        st.l = fmaf(l, g, st.l);
        if (__any(nf[0] | nf[1] | nf[2] | nf[3])) { // and who sees its token becomes NaN
            uint64_t bad = 0;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint64_t any = __ballot(nf[i] && 16 * now + 4 * j + i < nn);
#pragma unroll
                for (int k = 0; k < 4; k++)
                    if ((any >> (16 * k)) & 0xffff) bad |= (uint64_t)1 << (16 * now + 4 * k + i);
            }
            if (sees & bad) st.l = NAN;
        }
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
            for (int i = 0; i < 4; i++) st.o[d][i] = fmaf(z[d][i], g, st.o[d][i]);
        if (t >= tiles) return;
    }
}

// LDS: 16-byte values a lane of a wave with two tiles (their queries, later a tile's sums), and bytes in all (later what joins
// the waves).
template <int R, int Q>
constexpr int page_wave_lds() {
    const int q = R * 2 * KL * Q;
    return R == 1 ? 0 : q > DT ? q : DT;
}
template <int R, bool ROWS, int Q>
constexpr size_t page_lds() {
    const size_t q = (size_t)4 * page_wave_lds<R, Q>() * 64 * 16, o = ROWS ? 0 : (size_t)2 * R * DT * 64 * 16 + 4 * R * 16 * 8;
    return q > o ? q : o;
}

// A wave has R tiles of 16 rows.  ROWS: the workgroup's four waves have other rows of the same positions each; else they share the
// rows and take every fourth step, and are joined at the end.  A step's codes are converted once for the R tiles; the next step's
// loads go out as soon as a step's registers are used, its page's number a step before.
template <int CT, int QT, int R, bool ROWS>
__global__ void __launch_bounds__(256, (HSP <= 128 ? 2 : 1)) k_page_attention(PageArgs a) {
    constexpr int NQ = Q_PIECES<QT>, NP = P_PIECES, WAVE_LDS = page_wave_lds<R, NQ>();
    constexpr int STRIDE = ROWS ? 1 : 4, BLOCK_ROWS = 16 * R * (ROWS ? 4 : 1);
    extern __shared__ __align__(16) uint8_t lds[];
    const int lane = threadIdx.x & 63, n = lane & 15, j = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Place p;
    if (!place<QT>(a, BLOCK_ROWS, p)) return;
    const int row0 = p.row0 + (ROWS ? wave * 16 * R : 0);
    if (ROWS && row0 >= p.rows) return; // (no wave waits for another)

    const uint32_t bytes = PAGE_BLOCK * a.hs;
    const int *const table = a.table + (int64_t)p.b * a.per;
    const int shift = __builtin_ctz(a.page); // (a power of two)
    auto page_of = [&](int step) { // -1: none
        int page = -1;
        if (step < p.last) page = uniform(table + (step * PAGE_BLOCK >> shift));
        return (uint32_t)page < (uint32_t)a.n_pages ? page : -1;
    };
    // Offsets are formed again at every use, from values that the compiler cannot see through: all of them kept across the loop
    // take registers that spill, and a reload waits for the loads under way.
    auto again = [](uint32_t x) {
        asm volatile("" : "+v"(x));
        return x;
    };
    const uint32_t k_at = (16 * (n >> 2) + (n & 3)) * a.hs + 16 * j, k_last = 64 * (KL - 1) + 16 * j < a.hs ? k_at : OUT_OF_RANGE;
    u32x4 kr[4][KL], vr[DT];
    float ks = 0.0f, vs = 0.0f; // (no page: nothing of the step is seen, and zero scales keep it finite)
    auto load_k = [&](int step, int page) {
        const int blk = (step * PAGE_BLOCK & (a.page - 1)) / PAGE_BLOCK;
        const uint8_t *base = a.k;
        ks = 0.0f;
        if (page >= 0) {
            base += page * a.id + p.h * a.head + blk * (int64_t)bytes;
            ks = uniform(a.ks + (page * a.s_id + p.h * a.s_head + blk));
        }
        const auto rs = __builtin_amdgcn_make_buffer_rsrc((void *)base, 0, page >= 0 ? (int)bytes : 0, 0x00020000);
        const uint32_t at = again(k_at), last = again(k_last);
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int i = 0; i < KL; i++) {
                const auto c = __builtin_amdgcn_raw_buffer_load_b128(rs, (int)((i < KL - 1 ? at : last) + 4 * t * a.hs + 64 * i), 0, 0);
                kr[t][i] = (u32x4){c[0], c[1], c[2], c[3]};
            }
    };
    auto load_v = [&](int step, int page) {
        const int blk = (step * PAGE_BLOCK & (a.page - 1)) / PAGE_BLOCK;
        const uint8_t *base = a.v;
        vs = 0.0f;
        if (page >= 0) {
            base += page * a.id + p.h * a.head + blk * (int64_t)bytes;
            vs = uniform(a.vs + (page * a.s_id + p.h * a.s_head + blk));
        }
        const auto rs = __builtin_amdgcn_make_buffer_rsrc((void *)base, 0, page >= 0 ? (int)bytes : 0, 0x00020000);
        const uint32_t at = again(n * PAGE_BLOCK + 16 * j);
#pragma unroll
        for (int d = 0; d < DT; d++) { // (dimensions from hs on lie past the block)
            const auto c = __builtin_amdgcn_raw_buffer_load_b128(rs, (int)(at + 16 * d * PAGE_BLOCK), 0, 0);
            vr[d] = (u32x4){c[0], c[1], c[2], c[3]};
        }
    };
    u32x4 *const mine_ = (u32x4 *)lds + wave * WAVE_LDS * 64 + lane; // [WAVE_LDS][64], a lane's own
    auto park = [&](State &s, bool out) {
        f32x4 *const at = (f32x4 *)mine_;
#pragma unroll
        for (int d = 0; d < DT; d++) {
            if (out) at[d * 64] = s.o[d];
            else s.o[d] = at[d * 64];
        }
    };
    int step = p.first + (ROWS ? 0 : wave);
    int page = page_of(step), next = page_of(step + STRIDE);
    // of row `row` of the wave's tile r, as they lie (what is not there reads the row's start: no load waits behind a condition)
    float x[2 * KL][8];
    auto load_q = [&](int r) {
        const int row = row0 + 16 * r + n, tok = row / a.group;
        const uint8_t *const qp = a.q + p.b * a.q_seq + (row < p.rows ? tok * a.q_tok + (p.h * a.group + row - tok * a.group) * a.q_head : 0);
#pragma unroll
        for (int s = 0; s < 2 * KL; s++)
#pragma unroll
            for (int q4 = 0; q4 < 2; q4++) {
                const int d = 64 * (s / 2) + 16 * j + 8 * (s % 2) + 4 * q4;
                const float4 y = load4<QT>(qp, d < a.hs ? d : 0);
                x[s][4 * q4] = y.x, x[s][4 * q4 + 1] = y.y, x[s][4 * q4 + 2] = y.z, x[s][4 * q4 + 3] = y.w;
            }
    };
    if (R == 1) { // (with more rows their queries' values take the registers)
        load_q(0);
        load_k(step, page);
        load_v(step, page);
    }

    // the queries: value e of product s is dimension 64 (s / 2) + 16 j + 8 (s % 2) + e
    // (two tiles' queries wait in LDS, a lane's own: in registers they would spill)
    u32x4 qf[R > 1 ? 1 : R][2 * KL][NQ];
    u32x4 *const sm_q = mine_; // [R][2 KL][Q]
    // A score is a product of the pieces times the softmax scale, the block's and what the queries were divided by: mantissas and
    // exponents apart, so that nothing leaves fp32's range on the way
    const float cm = __builtin_amdgcn_frexp_mantf(a.c);
    int cq[R];
    State st[R];
#pragma unroll
    for (int r = 0; r < R; r++) {
        const bool ok = row0 + 16 * r + n < p.rows;
        float mx = 0.0f;
        if (R > 1) load_q(r);
#pragma unroll
        for (int s = 0; s < 2 * KL; s++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                if (!ok || 64 * (s / 2) + 16 * j + 8 * (s % 2) >= a.hs) x[s][e] = 0.0f;
                mx = fmaxf(mx, fabsf(x[s][e]));
            }
        const uint32_t e = power_to(over_groups(mx, fmax_));
        const float to = __uint_as_float(e << 23) * a.sign;
        cq[r] = __builtin_amdgcn_frexp_expf(a.c) + 127 - (int)e;
#pragma unroll
        for (int s = 0; s < 2 * KL; s++)
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                uint32_t w[NQ];
                split<NQ>(x[s][i] * to, x[s][i + 1] * to, w);
#pragma unroll
                for (int k = 0; k < NQ; k++) qf[R > 1 ? 0 : r][s][k][i / 2] = w[k];
            }
        if (R > 1)
#pragma unroll
            for (int s = 0; s < 2 * KL; s++)
#pragma unroll
                for (int k = 0; k < NQ; k++) sm_q[((r * 2 * KL + s) * NQ + k) * 64] = qf[0][s][k];
        st[r].m = -INFINITY, st[r].l = 0.0f;
#pragma unroll
        for (int d = 0; d < DT; d++) st[r].o[d] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
    }
    if (R > 1) {
        load_k(step, page);
        load_v(step, page);
    }
    for (; step < p.last; step += STRIDE) {
        const int left = page < 0 ? 0 : p.len - step * PAGE_BLOCK; // positions of the block that are seen
        const int mine = left - (int)again(16 * j);                // of the lane's 16
        // (products first: of a SIMD's two waves the one that makes weights then fills in.  Eight trees of 64 fp32 rows over up to
        // 16k int8 positions: 164 us without, 156 with it, bf16 rows 145 and 139; two over e4m3 77 and 74, 69 and 66)
        __builtin_amdgcn_s_setprio(1);
        f32x4 x[R][4];
#pragma unroll
        for (int r = 0; r < R; r++)
#pragma unroll
            for (int t = 0; t < 4; t++) x[r][t] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int s = 0; s < 2 * KL; s++) {
            u32x4 q[R][NQ];
#pragma unroll
            for (int r = 0; r < R; r++)
#pragma unroll
                for (int k = 0; k < NQ; k++) q[r][k] = R > 1 ? sm_q[((r * 2 * KL + s) * NQ + k) * 64] : qf[r % (R > 1 ? 1 : R)][s][k];
#pragma unroll
            for (int t = 0; t < 4; t++) {
                const f16x8 kf = codes8<CT>(kr[t][s / 2][2 * (s % 2)], kr[t][s / 2][2 * (s % 2) + 1]);
#pragma unroll
                for (int r = 0; r < R; r++)
#pragma unroll
                    for (int k = NQ - 1; k >= 0; k--) x[r][t] = product(kf, q[r][k], x[r][t]); // smallest pieces first
            }
        }
        __builtin_amdgcn_s_setprio(0);
        // a scale below zero turns the scores round; one that is not finite, of K or V, makes every row NaN through its values
        if (ks < 0.0f)
#pragma unroll
            for (int r = 0; r < R; r++)
#pragma unroll
                for (int t = 0; t < 4; t++) x[r][t] = -x[r][t];
        const float size = fabsf(ks) < INFINITY ? fabsf(ks) : 0.0f, v_size = fabsf(ks) < INFINITY ? vs : NAN;
        const float sm = __builtin_amdgcn_frexp_mantf(size) * cm;
        const int se = __builtin_amdgcn_frexp_expf(size);
        u32x4 pf[R][2][NP];
        float gv[R];
#pragma unroll
        for (int r = 0; r < R; r++) {
            // (neither 0 nor infinite: what is not seen is -infinity times it, and a score may be 0)
            float c = __builtin_amdgcn_fmed3f(__builtin_amdgcn_ldexpf(sm, cq[r] + se), 1e-45f, 3.4e38f), ms = -INFINITY;
            if (left < PAGE_BLOCK)
#pragma unroll
                for (int t = 0; t < 4; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (4 * t + i >= mine) x[r][t][i] = -INFINITY;
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int i = 0; i < 4; i++) ms = fmaxf(ms, x[r][t][i]);
            ms = over_groups(ms, fmax_) * c;
            // A step's largest weight is 2^15, the top of fp16's range.  Scores from 2^23 on have steps of 1 or more, and the
            // difference could be 16: those weights are few and far apart, their largest is 1, and it takes scores rounded alike.
            if (__any(fabsf(ms) >= 0x1p23f && ms != -INFINITY)) {
#pragma unroll
                for (int t = 0; t < 4; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++) x[r][t][i] *= c;
                c = 1.0f;
            }
            ms -= fabsf(ms) < 0x1p23f ? 15.0f : 0.0f;
            const float mu = ms == -INFINITY ? 0.0f : -ms;
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    uint32_t w[NP];
                    split<NP>(__builtin_amdgcn_exp2f(fmaf(x[r][2 * u + e / 4][e % 4], c, mu)),
                                 __builtin_amdgcn_exp2f(fmaf(x[r][2 * u + e / 4][e % 4 + 1], c, mu)), w);
#pragma unroll
                    for (int k = 0; k < NP; k++) pf[r][u][k][e / 2] = w[k];
                }
            // the sum of the weights as the products take them
            f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int k = NP - 1; k >= 0; k--)
#pragma unroll
                for (int u = 0; u < 2; u++) sum = product(ones(), pf[r][u][k], sum);
            float f, g;
            join(st[r], ms, f, g);
            gv[r] = g * (v_size + (v_size - v_size)); // (an infinite one is NaN; looked at here, not before the scores: 0.3 us a call)
            st[r].l = fmaf(sum[0], g, st[r].l);
        }
        load_k(step + STRIDE, next);
        if (CT == LLM_E4M3 && left < PAGE_BLOCK) // codes past the end may be NaN: 0 * NaN
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const int have = min(max(mine - 4 * k, 0), 4);
                const uint32_t keep = have == 4 ? 0xffffffffu : (1u << (8 * have)) - 1;
#pragma unroll
                for (int d = 0; d < DT; d++) vr[d][k] &= keep;
            }
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int d = 0; d < DT; d++) {
            f16x8 vf[2];
#pragma unroll
            for (int u = 0; u < 2; u++) vf[u] = codes8<CT>(vr[d][2 * u], vr[d][2 * u + 1]);
#pragma unroll
            for (int r = 0; r < R; r++) {
                f32x4 y = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int k = NP - 1; k >= 0; k--)
#pragma unroll
                    for (int u = 0; u < 2; u++) y = product(vf[u], pf[r][u][k], y);
#pragma unroll
                for (int i = 0; i < 4; i++) st[r].o[d][i] = fmaf(y[i], gv[r], st[r].o[d][i]);
            }
        }
        __builtin_amdgcn_s_setprio(0);
        load_v(step + STRIDE, next);
        page = next;
        next = page_of(step + 2 * STRIDE);
    }

    // the new tokens' rows; waves that share the rows take a tile each, from the one with the fewest steps on
#pragma unroll
    for (int r = 0; r < R; r++) {
        const int row = row0 + 16 * r + n, tok = row / a.group;
        const bool ok = row < p.rows;
        const uint8_t *const qp = a.q + p.b * a.q_seq + (ok ? tok * a.q_tok + (p.h * a.group + row - tok * a.group) * a.q_head : 0);
        if (!p.fresh || row0 + 16 * r >= p.rows) break;
        if (R > 1) park(st[R - 1 - r], true); // (the other tile's sums out of the way, over the queries)
        new_rows<QT, R == 1>(a, p, ROWS ? 0 : (wave - (p.last - p.first)) & 3, ROWS ? 1 : 4, qp, ok, tok, st[r]);
        if (R > 1) park(st[R - 1 - r], false);
    }
    if constexpr (!ROWS) { // the four waves' sums joined: each scaled to a common exponent, waves 2 and 3 into 0 and 1, then 1 into 0
        f32x4 *const sm_o = (f32x4 *)lds;                                     // [2][R][DT][64]
        float2 *const sm_ml = (float2 *)(lds + (size_t)2 * R * DT * 64 * 16); // [4][R][16]
        __syncthreads(); // (their queries may lie there)
        if (j == 0)
#pragma unroll
            for (int r = 0; r < R; r++) sm_ml[(wave * R + r) * 16 + n] = make_float2(st[r].m, st[r].l);
        __syncthreads();
#pragma unroll
        for (int r = 0; r < R; r++) {
            float mn = -INFINITY, l = 0.0f;
#pragma unroll
            for (int w = 0; w < 4; w++) mn = fmaxf(mn, sm_ml[(w * R + r) * 16 + n].x);
            const float mu = mn == -INFINITY ? 0.0f : mn, al = __builtin_amdgcn_exp2f(st[r].m - mu);
#pragma unroll
            for (int w = 0; w < 4; w++) {
                const float2 ml = sm_ml[(w * R + r) * 16 + n];
                l += ml.y * __builtin_amdgcn_exp2f(ml.x - mu);
            }
            st[r].m = mn, st[r].l = l;
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int i = 0; i < 4; i++) st[r].o[d][i] *= al;
        }
#pragma unroll
        for (int half = 2; half; half >>= 1) {
            if (wave >= half && wave < 2 * half)
#pragma unroll
                for (int r = 0; r < R; r++)
#pragma unroll
                    for (int d = 0; d < DT; d++) sm_o[(((wave - half) * R + r) * DT + d) * 64 + lane] = st[r].o[d];
            __syncthreads();
            if (wave < half)
#pragma unroll
                for (int r = 0; r < R; r++)
#pragma unroll
                    for (int d = 0; d < DT; d++) st[r].o[d] += sm_o[((wave * R + r) * DT + d) * 64 + lane];
            __syncthreads();
        }
        if (wave) return;
    }
#pragma unroll
    for (int r = 0; r < R; r++) {
        const int row = row0 + 16 * r + n;
        if (row < p.rows) put_row<QT>(a, p, row, j, st[r], st[r].l);
    }
}

} // namespace

#define PAGE_NAME2(n) page_kernel_##n
#define PAGE_NAME(n) PAGE_NAME2(n)

PageKernel PAGE_NAME(PAGE_HSP)(int type, int q_type, int tiles, int rows, size_t *lds) {
#define PAGE_PICK(C, QY, T, W)                                                   \
    if (type == C && q_type == QY && tiles == T && (rows != 0) == W) {            \
        *lds = page_lds<T, W, Q_PIECES<QY>>();                                 \
        return k_page_attention<C, QY, T, W>;                                    \
    }
#define PAGE_PICK_T(T, W)                                                        \
    PAGE_PICK(LLM_I8, LLM_F32, T, W) PAGE_PICK(LLM_I8, LLM_BF16, T, W)           \
    PAGE_PICK(LLM_E4M3, LLM_F32, T, W) PAGE_PICK(LLM_E4M3, LLM_BF16, T, W)
    PAGE_PICK_T(1, false)
#if PAGE_HSP <= 128
    PAGE_PICK_T(2, false) PAGE_PICK_T(2, true)
#endif
    return nullptr;
}
