// kv8.cuh -- the GQA cache held in 8 bits: its codes, its scales, and the check of a descriptor (cwk_kv8, cwk_attn.h).
//
// A block of 32, 64 or 128 rows of one KV head shares one scale 2^e, for K and for V each: value = code * 2^e. Powers of two,
// because rows arrive one at a time: when a later row of an open block is too large for its scale, the codes in front of it move
// to the new scale by an exponent shift, exactly (E4M3, but for values that become subnormal) or with one more rounding (INT8), and a value read
// back is exact in bf16. What it costs: up to a factor of two of the scale's range, nothing for E4M3's relative precision.
#pragma once
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "cwk_common.cuh"

// CWK_OK, or an error with its text: everything of a descriptor that the host can see.
int cwk_kv8_check(cwk_ctx *ctx, const cwk_kv8 *c, const char *who);
// Rows row0 .. row0 + n - 1 of the slot at `c` widened to bf16 [n][nkv][hd], K and V (row0 + n <= c.rows).
int cwk_kv8_widen(cwk_ctx *ctx, const cwk_kv8 &c, int64_t row0, int64_t n, void *k, void *v);
// Query rows of `n` tokens per sequence over the cache of slots 0 .. B - 1 (kv8_decode.cu); the caller has checked everything.
// kv_len NULL: every sequence has max_kv_len rows.
int cwk_kv8_streams(cwk_ctx *ctx, const void *q, const cwk_kv8 &c, const int32_t *kv_len, int max_kv_len, int B, int n, int nh, float scale,
                    void *out, int max_blocks);

namespace {

constexpr int KV8_LOW = -100, KV8_HIGH_E4M3 = 119, KV8_HIGH_INT8 = 121;      // exponents that a scale can have: no value leaves bf16's normal range
constexpr float KV8_MAX_E4M3 = 448.f, KV8_MAX_INT8 = 127.f;

__host__ __device__ __forceinline__ constexpr int kv8_high(bool i8) { return i8 ? KV8_HIGH_INT8 : KV8_HIGH_E4M3; }
// 2^e for e in [-126, 127]
__device__ __forceinline__ float kv8_two(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
// what a stored scale stands for
__device__ __forceinline__ float kv8_scale(uint32_t byte) { return __uint_as_float(byte << 23); }
// least e with amax <= 448 * 2^e (E4M3) or 127 * 2^e (INT8), within the limits; amax finite, >= 0. amax = 1.f * 2^a: 448 = 1.75 * 2^8, 127 = 1.984375 * 2^6.
__device__ __forceinline__ int kv8_exponent(float amax, bool i8) {
    const uint32_t u = __float_as_uint(amax);
    const int a = (int)(u >> 23) - 127;
    const int e = i8 ? a - 6 + ((u & 0x7FFFFFu) > 0x7E0000u) : a - 8 + ((u & 0x7FFFFFu) > 0x600000u);
    return min(max(e, KV8_LOW), kv8_high(i8));
}
// y (in units of the scale) -> code, to nearest even, saturating. NaN is E4M3's NaN (INT8 has none: 0).
__device__ __forceinline__ uint32_t kv8_encode_e4m3x2(float lo, float hi) {
    return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ uint32_t kv8_encode_i8(float y) {
    return (uint32_t)__float2int_rn(fminf(fmaxf(y == y ? y : 0.f, -KV8_MAX_INT8), KV8_MAX_INT8)) & 255u;
}
// four values -> four codes, the first in the lowest byte
template <bool I8>
__device__ __forceinline__ uint32_t kv8_encode4(const float (&y)[4]) {
    if constexpr (I8) return kv8_encode_i8(y[0]) | kv8_encode_i8(y[1]) << 8 | kv8_encode_i8(y[2]) << 16 | kv8_encode_i8(y[3]) << 24;
    else return kv8_encode_e4m3x2(y[0], y[1]) | kv8_encode_e4m3x2(y[2], y[3]) << 16;
}
// two E4M3 codes (low half of `two`) -> two f16, exactly
__device__ __forceinline__ uint32_t kv8_e4m3_f16x2(uint32_t two) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)two));
    return r;
}
// two INT8 codes -> two f16, exactly: `biased` holds code + 128 in its bytes; with 0x64 above it a byte b is the f16 number 1024 + b
template <uint32_t SEL>
__device__ __forceinline__ uint32_t kv8_i8_f16x2(uint32_t biased) {
    const uint32_t x = __byte_perm(biased, 0x64646464u, SEL);
    const __half2 h = __hsub2(*reinterpret_cast<const __half2 *>(&x), __half2half2(__ushort_as_half((unsigned short)0x6480)));
    return *reinterpret_cast<const uint32_t *>(&h);
}
// four codes (bytes 0..3) -> f16 pairs (0, 1) and (2, 3)
template <bool I8>
__device__ __forceinline__ void kv8_decode4(uint32_t codes, uint32_t &p01, uint32_t &p23) {
    if constexpr (I8) {
        const uint32_t b = codes ^ 0x80808080u;
        p01 = kv8_i8_f16x2<0x4140>(b);
        p23 = kv8_i8_f16x2<0x4342>(b);
    } else {
        p01 = kv8_e4m3_f16x2(codes);
        p23 = kv8_e4m3_f16x2(codes >> 16);
    }
}
// the same for the pairs (0, 2) and (1, 3)
template <bool I8>
__device__ __forceinline__ void kv8_decode4_even_odd(uint32_t codes, uint32_t &p02, uint32_t &p13) {
    if constexpr (I8) {
        const uint32_t b = codes ^ 0x80808080u;
        p02 = kv8_i8_f16x2<0x4240>(b);
        p13 = kv8_i8_f16x2<0x4341>(b);
    } else {
        const uint32_t x = __byte_perm(codes, 0u, 0x3120);
        p02 = kv8_e4m3_f16x2(x);
        p13 = kv8_e4m3_f16x2(x >> 16);
    }
}

}  // namespace
