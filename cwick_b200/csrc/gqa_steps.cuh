// gqa_steps.cuh -- what the streaming GQA decode kernels (gqa_decode.cu: bf16 cache, kv8_decode.cu: 8-bit cache) share: the steps of
// all sequences dealt out to the blocks in equal contiguous ranges, worked out from the lengths on the device, and the merge of the
// records that a sequence's blocks leave.
#pragma once
#include "cwk_common.cuh"

namespace {

// The list of all steps: sequence after sequence, in each one head group after the other, in each `keys` cached rows a step.
struct GqaSteps {
    const int32_t *kv_len;                    // [B]; NULL: every sequence has `most` rows
    int B, groups, keys;
    int most;                                 // a length beyond this counts as this (the rows that there are)
    int2 *meta;                               // [B][groups]: first record slot, number of slots
};
__device__ __forceinline__ int length_of(const GqaSteps &p, int b) { return p.kv_len ? min(max(p.kv_len[b], 0), p.most) : p.most; }

// A block's place in the list of all steps: sequence, group of KV heads, step within it.
struct GqaPlace {
    int b, hg, step, steps, len;      // steps: of this sequence (and head group)
};
__device__ __forceinline__ int steps_of(const GqaSteps &p, int b) { return b < p.B ? (length_of(p, b) + p.keys - 1) / p.keys : 0; }

// This block's range [lo, hi) of all steps, and where it begins. Every warp works it out for itself; the first one notes, for
// every (sequence, head group) whose first step is in the range, its first record slot (slots are numbered by head group
// plus block: one of the two grows from record to record) and their number.
__device__ __forceinline__ int gqa_range(const GqaSteps &p, int lane, bool note, GqaPlace &at) {
    const int nhg = p.groups;
    int64_t total = 0;
    for (int b0 = 0; b0 < p.B; b0 += 32) {
        int v = steps_of(p, b0 + lane);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        total += v;
    }
    total *= nhg;
    const int64_t G = max((int64_t)1, min((int64_t)gridDim.x, total)), g = blockIdx.x;      // no block between two others is left without a step
    const int64_t lo = g < G ? total * g / G : total, hi = g < G ? total * (g + 1) / G : total;
    int64_t before = 0;
    for (int b0 = 0; b0 < p.B; b0 += 32) {
        const int mine = steps_of(p, b0 + lane);
        int v = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += u;
        }
        const int64_t s0 = (before + v - mine) * nhg, s1 = s0 + (int64_t)mine * nhg;       // this lane's sequence: steps [s0, s1)
        const bool here = mine > 0 && s0 <= lo && lo < s1 && lo < hi;
        const uint32_t who = __ballot_sync(0xffffffffu, here);
        if (who) {
            const int src = __ffs(who) - 1;
            at.b = b0 + src;
            at.steps = __shfl_sync(0xffffffffu, mine, src);
            const int off = (int)__shfl_sync(0xffffffffu, (int)(lo - s0), src);
            at.hg = off / at.steps;
            at.step = off % at.steps;
        }
        if (note && b0 + lane < p.B) {
            if (mine == 0) {
                if (s0 > 0 ? (lo < s0 && s0 <= hi) : g == 0)
                    for (int h = 0; h < nhg; h++) p.meta[(b0 + lane) * nhg + h] = make_int2(0, 0);
            } else if (s0 < hi && s1 > lo) {
                const int64_t h0 = lo > s0 ? (lo - s0 + mine - 1) / mine : 0;              // first head group that begins here
                for (int64_t h = h0; h < nhg && s0 + h * mine < hi; h++) {
                    const int64_t g1 = ((s0 + (h + 1) * mine) * G - 1) / total;              // the block with its last step
                    p.meta[(b0 + lane) * nhg + h] = make_int2((int)((b0 + lane) * nhg + h + g), (int)(g1 - g + 1));
                }
            }
        }
        before += __shfl_sync(0xffffffffu, v, 31);
    }
    return (int)(hi - lo);
}
__device__ __forceinline__ void gqa_advance(const GqaSteps &p, GqaPlace &at) {      // to the next step; there is one
    if (++at.step < at.steps) return;
    at.step = 0;
    if (++at.hg < p.groups) return;
    at.hg = 0;
    do {
        at.b++;
        at.len = length_of(p, at.b);
    } while (at.len <= 0);
    at.steps = steps_of(p, at.b);
}

// The merge of `cnt` records of one query row, at(i) its i-th {m, l, o[HD]}: (HD / 2) x GROUPS threads, two columns each, the
// records dealt out to the groups (one sequence has a record from every block: 148 in a row are 20 us of loads for one group of
// threads). True for the threads of group 0, which get the joined columns x, y (not yet divided) and the sum `den`.
template <int HD, int GROUPS, class At>
__device__ __forceinline__ bool gqa_merge_records(int cnt, At at, float &den, float &x, float &y) {
    constexpr int NT = HD / 2;
    __shared__ float s_m[GROUPS], s_l[GROUPS];
    __shared__ float2 s_o[GROUPS][NT];
    const int g = threadIdx.x / NT, tid = threadIdx.x % NT;
    float M = -INFINITY;
    den = x = y = 0.f;
    for (int i0 = g; i0 < cnt; i0 += 8 * GROUPS) {         // eight records' loads at once; the running maximum as the scores'
        float m[8], l[8];
        float2 o[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int i = i0 + j * GROUPS;
            const float *r = at(min(i, cnt - 1));
            m[j] = i < cnt ? r[0] : -INFINITY;
            l[j] = r[1];
            o[j] = *reinterpret_cast<const float2 *>(r + 2 + 2 * tid);
        }
        float mx = M;
#pragma unroll
        for (int j = 0; j < 8; j++) mx = fmaxf(mx, m[j]);
        if (mx == -INFINITY) continue;
        const float a = exp2f(M - mx);
        den *= a; x *= a; y *= a;
        M = mx;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float w = exp2f(m[j] - M);
            den += w * l[j]; x += w * o[j].x; y += w * o[j].y;
        }
    }
    if (GROUPS > 1) {
        if (tid == 0) { s_m[g] = M; s_l[g] = den; }
        s_o[g][tid] = make_float2(x, y);
        __syncthreads();
        if (g > 0) return false;
        float mx = -INFINITY;
#pragma unroll
        for (int j = 0; j < GROUPS; j++) mx = fmaxf(mx, s_m[j]);
        den = x = y = 0.f;
#pragma unroll
        for (int j = 0; j < GROUPS; j++) {
            const float w = s_m[j] == -INFINITY ? 0.f : exp2f(s_m[j] - mx);
            den += w * s_l[j]; x += w * s_o[j][tid].x; y += w * s_o[j][tid].y;
        }
    }
    return true;
}

}  // namespace
