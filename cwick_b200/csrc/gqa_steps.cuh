// gqa_steps.cuh -- what the streaming GQA decode kernels (gqa_decode.cu: bf16 cache, kv8_decode.cu: 8-bit cache) share: the steps of
// all sequences dealt out to the blocks in equal contiguous ranges, worked out from the lengths on the device. (Their records, and the
// merges of these, are each kernel's own.)
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

// What a warp knows of the list: its sequence's steps (sequence 32 i + lane), and those up to and with it among the 32; all steps, groups
// included. One round of up to 32 sequences is kept, more are walked over again: the start of a block is code that runs once, with
// nothing in flight yet, so what counts is that it is little (divisions in 64 bits, a second walk and the note in front of the first
// copies were 4 us of a step of 16 sequences).
struct GqaList {
    int mine, upto;
    int64_t total, lo, hi;                    // lo, hi: the block's steps
};
__device__ __forceinline__ void gqa_round(const GqaSteps &p, int b0, int lane, GqaList &s) {
    s.mine = steps_of(p, b0 + lane);
    s.upto = s.mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, s.upto, o);
        if (lane >= o) s.upto += u;
    }
}
__device__ __forceinline__ GqaList gqa_list(const GqaSteps &p, int lane) {
    GqaList s;
    gqa_round(p, 0, lane, s);
    s.total = __shfl_sync(0xffffffffu, s.upto, 31);
    if (p.B > 32) {
        const int mine = s.mine, upto = s.upto;
#pragma unroll 1
        for (int b0 = 32; b0 < p.B; b0 += 32) {
            gqa_round(p, b0, lane, s);
            s.total += __shfl_sync(0xffffffffu, s.upto, 31);
        }
        s.mine = mine; s.upto = upto;
    }
    s.total *= p.groups;
    return s;
}
// body(first sequence of the round, this lane's steps, the steps in front of them, groups included); it is given GqaList's first round
template <class U, class F>
__device__ __forceinline__ void gqa_walk(const GqaSteps &p, GqaList s, int lane, F &&body) {
    U before = 0;
#pragma unroll 1
    for (int b0 = 0;;) {
        body(b0, s.mine, (before + s.upto - s.mine) * (U)p.groups);
        if ((b0 += 32) >= p.B) return;
        before += __shfl_sync(0xffffffffu, s.upto, 31);
        gqa_round(p, b0, lane, s);
    }
}
// The block's range [lo, hi) of `total` steps: all blocks the same number, but for one; no block between two others is left without a step.
// U: an unsigned type that total * (blocks + 1) fits.
template <class U> __device__ __forceinline__ U gqa_blocks(U total) { return max((U)1, min((U)gridDim.x, total)); }
template <class U> __device__ __forceinline__ U gqa_from(U total, U g) {
    const U G = gqa_blocks(total);
    return g >= G ? total : G == total ? g : total * g / G;
}
template <class U>
__device__ __forceinline__ int gqa_share(const GqaSteps &p, GqaList &s, int lane, GqaPlace &at) {
    const U total = (U)s.total, lo = gqa_from<U>(total, blockIdx.x), hi = gqa_from<U>(total, blockIdx.x + 1);
    s.lo = lo; s.hi = hi;
    gqa_walk<U>(p, s, lane, [&](int b0, int mine, U s0) {
        const uint32_t who = __ballot_sync(0xffffffffu, mine > 0 && s0 <= lo && lo < s0 + (U)mine * (U)p.groups && lo < hi);
        if (who) {
            const int src = __ffs(who) - 1;
            at.b = b0 + src;
            at.steps = __shfl_sync(0xffffffffu, mine, src);
            const uint32_t off = __shfl_sync(0xffffffffu, (uint32_t)(lo - s0), src);
            at.hg = p.groups == 1 ? 0 : off / (uint32_t)at.steps;
            at.step = off - at.hg * at.steps;
        }
    });
    return (int)(hi - lo);
}
// Where the block begins, and how many steps it has; the list is for gqa_note.
__device__ __forceinline__ int gqa_range(const GqaSteps &p, int lane, GqaList &s, GqaPlace &at) {
    if (p.B == 1) {                                        // nothing to add up or to look for
        s.mine = s.upto = steps_of(p, 0);
        s.total = (int64_t)s.mine * p.groups;
        if (s.total * (gridDim.x + 1) < (1ll << 32)) {
            const uint32_t lo = gqa_from<uint32_t>((uint32_t)s.total, blockIdx.x), hi = gqa_from<uint32_t>((uint32_t)s.total, blockIdx.x + 1);
            s.lo = lo; s.hi = hi;
            at.steps = s.mine;
            at.hg = p.groups == 1 || lo == hi ? 0 : lo / (uint32_t)s.mine;
            at.step = (int)lo - at.hg * s.mine;
            return (int)(hi - lo);
        }
    }
    s = gqa_list(p, lane);
    if (s.total * (gridDim.x + 1) < (1ll << 32)) return gqa_share<uint32_t>(p, s, lane, at);
    return gqa_share<uint64_t>(p, s, lane, at);
}
// One warp of the block notes, for every (sequence, head group) whose first step is in the block's range, its first record slot (slots
// are numbered by head group plus block: one of the two grows from record to record) and their number.
template <class U>
__device__ __forceinline__ void gqa_note_as(const GqaSteps &p, const GqaList &s, int lane) {
    const U total = (U)s.total, nhg = p.groups, G = gqa_blocks(total), g = blockIdx.x, lo = (U)s.lo, hi = (U)s.hi;
    gqa_walk<U>(p, s, lane, [&](int b0, int mine, U s0) {
        const int b = b0 + lane;
        if (b >= p.B) return;
        if (mine == 0) {
            if (s0 > 0 ? (lo < s0 && s0 <= hi) : g == 0)
                for (int h = 0; h < p.groups; h++) p.meta[b * p.groups + h] = make_int2(0, 0);
        } else if (s0 < hi && s0 + (U)mine * nhg > lo) {
            const U h0 = lo <= s0 ? 0 : nhg == 1 ? 1 : (lo - s0 + mine - 1) / (U)mine;      // first head group that begins here
#pragma unroll 1
            for (U h = h0; h < nhg && s0 + h * mine < hi; h++) {
                const U last = s0 + (h + 1) * mine, g1 = last <= hi ? g : G == total ? last - 1 : (last * G - 1) / total;      // the block with its last step
                p.meta[b * p.groups + (int)h] = make_int2(b * p.groups + (int)(h + g), (int)(g1 - g + 1));
            }
        }
    });
}
__device__ __forceinline__ void gqa_note(const GqaSteps &p, GqaList s, int lane) {
    if (p.B == 1) {
        if (p.groups == 1) {
            if (blockIdx.x == 0 && lane == 0) p.meta[0] = make_int2(0, (int)min((int64_t)gridDim.x, s.total));
            return;
        }
        if (lane > 0) s.mine = 0;                          // (gqa_range may have left the one sequence's steps in every lane)
    }
    if (s.total * (gridDim.x + 1) < (1ll << 32)) gqa_note_as<uint32_t>(p, s, lane);
    else gqa_note_as<uint64_t>(p, s, lane);
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

}  // namespace
