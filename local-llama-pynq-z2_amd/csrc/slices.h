// Attention whose positions are cut into slices: which block takes what, and the join (internal header).  A call's arguments A
// have n_seq, n_kv, hs, group, max_n, n, cap (most slices in all, 0: none), each (of a head), least (their steps), acc, ml, plan and
// the output's address and strides, and steps_of(A, sequence) gives the steps of a sequence.
#pragma once
#include "device.h"

constexpr int MAX_SLICES = 128; // of a sequence's kv head
constexpr int MAX_CUT_SEQS = 512;   // of a call whose positions are cut
// A sequence of so many times the least steps stays whole: cutting it costs the join (7 rows over 300 int8 positions: 11.0 us
// whole, 12.4 in two slices; over 800, four times the least: 14.8 and 12.4).
constexpr int WHOLE_STEPS = 3;

// Slices of the only sequence of a call, of `all` steps: head h has numbers h * each and on.
template <typename A>
__device__ __forceinline__ int slices_of_one(const A &a, int all, int &steps) {
    steps = all <= WHOLE_STEPS * a.least ? all : max(a.least, (all + a.each - 1) / a.each);
    return (all + steps - 1) / steps;
}

// Inclusive sum over a wave: within rows of 16 lanes, then of the rows before (DPP: row_shr 1, 2, 4, 8, row_bcast 15, 31).
__device__ __forceinline__ int wave_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
    return v;
}

// The slice `id`: its sequence, kv head and number there, the slices of that head and their steps.  A sequence of n steps
// has ceil(n / q) slices a head, the same q for all, so that long sequences do not outlast the others; q is about the least
// at which there are no more than a.cap in all.  Every block finds it from the lengths.
template <typename A, typename P>
__device__ __forceinline__ bool find_slice(const A &a, uint32_t id, P &p, int &steps) {
    if (a.n_seq == 1) {
        p.b = 0;
        p.h = (int)id / a.each;
        p.split = (int)id - p.h * a.each;
        p.slices = slices_of_one(a, steps_of(a, 0), steps);
        return p.split < p.slices;
    }
    const int lane = threadIdx.x & 63;
    constexpr int GROUPS = MAX_CUT_SEQS / 64;
    int all[GROUPS];
    float sum = 0.0f, most = 0.0f; // (a guess to begin with: rounded sums of steps do)
#pragma unroll
    for (int i = 0; i < GROUPS; i++) {
        all[i] = 0;
        if (64 * i < a.n_seq) {
            if (64 * i + lane < a.n_seq) all[i] = steps_of(a, 64 * i + lane);
            sum += (float)all[i];
            most = fmaxf(most, (float)all[i]);
        }
    }
    const float kv = (float)a.n_kv;
    const int guess = __builtin_amdgcn_readfirstlane((int)(wave_sum(sum) * kv / (float)a.cap));
    const int longest = __builtin_amdgcn_readfirstlane((int)wave_max(most));
    steps = longest <= WHOLE_STEPS * a.least ? longest : max(max(a.least, guess), longest / a.each + 1);
    // Four lengths at once, each a sixteenth above the one before, whose chains of instructions overlap; the first at which there
    // are few enough slices (32 sequences: 3.7k cycles for the whole function; 5.5k one after another, with the scan through LDS).
    constexpr int AT_ONCE = 4;
    for (bool fits = false; !fits;) { // (ends: at the longest sequence's steps there is a slice a head)
        int q[AT_ONCE];
        float total[AT_ONCE];
#pragma unroll
        for (int u = 0; u < AT_ONCE; u++) {
            q[u] = u ? q[u - 1] + (q[u - 1] + 15) / 16 : steps;
            total[u] = 0.0f;
        }
#pragma unroll
        for (int i = 0; i < GROUPS; i++)
            if (64 * i < a.n_seq)
#pragma unroll
                for (int u = 0; u < AT_ONCE; u++) total[u] += (float)((all[i] + q[u] - 1) / q[u]);
#pragma unroll
        for (int u = 0; u < AT_ONCE; u++) total[u] = wave_sum(total[u]) * kv; // (exact up to 2^24)
#pragma unroll
        for (int u = 0; u < AT_ONCE; u++)
            if (!fits) {
                steps = q[u];
                fits = total[u] <= (float)a.cap;
            }
        if (!fits) steps += (steps + 15) / 16;
    }
    steps = __builtin_amdgcn_readfirstlane(steps);
    int before = 0; // slices of a head of the sequences before
#pragma unroll
    for (int i = 0; i < GROUPS; i++)
        if (64 * i < a.n_seq) {
            const int n = (all[i] + steps - 1) / steps, upto = wave_scan(n);
            const int passed = __popcll(__ballot((before + upto) * a.n_kv <= (int)id));
            if (passed < 64) { // (a lane without a sequence has passed none that its neighbours have not)
                const int at = __builtin_amdgcn_readfirstlane(passed);
                p.b = 64 * i + at;
                p.slices = __builtin_amdgcn_readlane(n, at);
                const int rest = (int)id - (before + __builtin_amdgcn_readlane(upto, at) - p.slices) * a.n_kv;
                p.h = rest / p.slices;
                p.split = rest - p.h * p.slices;
                return true;
            }
            before += __builtin_amdgcn_readlane(upto, 63);
        }
    return false;
}

// A row's slices joined: weights exp2(max_s - max).  W waves a row (the block has four): a thread takes four values of
// every (64 W / (hs / 4))-th slice, eight slices' loads at once.
template <typename A, int QT, int W>
__global__ void __launch_bounds__(256) k_join_slices(A a) {
    __shared__ float sm_f[4 / W][MAX_SLICES + 64]; // (a group's last loads may be past the last slice: weight 0)
    __shared__ float4 sm_o[256];
    constexpr int T = 64 * W;
    const int lane = threadIdx.x & 63, part = threadIdx.x / T, tid = threadIdx.x % T;
    const int row = blockIdx.x * (4 / W) + part, h = blockIdx.y, b = blockIdx.z;
    const int nn = a.n ? min(max(a.n[b], 0), a.max_n) : a.max_n;
    int slices, first;
    if (a.n_seq == 1) {
        int steps;
        slices = slices_of_one(a, steps_of(a, 0), steps);
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
    float m[MAX_SLICES / 64], l[MAX_SLICES / 64], mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < MAX_SLICES / 64; i++) {
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
    for (int i = 0; i < MAX_SLICES / 64; i++) {
        const float f = __builtin_amdgcn_exp2f(m[i] - mu);
        sum += l[i] * f;
        if (tid < 64) sm_f[part][lane + 64 * i] = f;
    }
    sum = wave_sum(sum);
    if (tid < 64) sm_f[part][lane + MAX_SLICES] = 0.0f;
    __syncthreads();
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int s0 = g; s0 < slices; s0 += U * groups) {
        if (s0 != g) load(s0);
#pragma unroll
        for (int u = 0; u < U; u++) {
            const float f = sm_f[part][min(s0 + u * groups, MAX_SLICES)];
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
