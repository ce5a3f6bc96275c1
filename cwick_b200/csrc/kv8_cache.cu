// kv8_cache.cu -- writing and reading the GQA cache held in 8 bits (format: kv8.cuh), compiled without fast-math.
//
// Writing. A task is one block of rows of one KV head, K or V: its new rows are read once into registers (a warp has four or eight rows in a
// row, a lane hd / 32 neighbouring values of each), the largest magnitude is found over the task, then the codes go out; an open block
// whose scale grows has the codes in front of the new rows rewritten. In front of the quantisation, for cwk_gqa_qk_prep_kv8, keys get
// their RMS norm and rotation (src/q35_model.c:112-122, :144-153, :459-477), and query heads the same on blocks of their own. Bound: the store by
// HBM, 16,381 rows of 4 KV heads of 256, bf16 to INT8 (101 MB) 17.8 us = 5.7 TB/s, E4M3 19.0, from f32 28.4 (5.9 TB/s); one row of 64 slots by
// latency, 2.6 us. The preparation by the instructions of the keys: 7 x 300 rows and 16 query heads (64 MB) 20.1 us, 512 rows 8.2, one
// of 64 slots 4.3.
//
// Reading is a conversion on the way: the same 16,381 rows to bf16 18.9 us = 5.3 TB/s.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "kv8.cuh"

namespace {

enum { SRC_BF16 = 0, SRC_F32 = 1 };

struct Kv8StoreParams {
    const void *k, *v;                         // [B][n][nkv][hd]
    const int32_t *pos, *count;                // [B]; count NULL: n
    uint8_t *kc, *vc, *ks, *vs;
    int64_t rows;                              // per slot
    int B, n, nkv, lb;                         // block = 1 << lb
    int window;                                // blocks that n rows can touch
};
struct Kv8PrepParams : Kv8StoreParams {
    int nh, rot, heads;                        // heads: query heads per warp
    float eps;
    const float *qg, *q_norm, *k_norm;
    uint16_t *q_out;
    int64_t tasks;                             // K and V tasks; the blocks behind them have query rows
    double octaves;                            // angle per position of pair i: 2^(-i * octaves)
};
static_assert(sizeof(Kv8StoreParams) <= 128, "kernel parameters: more than 128 bytes of them come later");
constexpr int KQ_HEADS = 8;                    // most query heads of a warp

// new rows of slot b: positions pos .. pos + the result - 1, all inside the slot
__device__ __forceinline__ int new_rows(const Kv8StoreParams &p, int b, int64_t &pos) {
    pos = p.pos[b];
    const int64_t c = p.count ? min(p.count[b], p.n) : p.n;
    return pos < 0 ? 0 : (int)max((int64_t)0, min(c, p.rows - pos));
}

// A lane's V values of a row, as they lie in memory (two bf16 or one f32 a word).
template <int V, int SRC>
struct Raw {
    static constexpr int W = SRC == SRC_BF16 ? V / 2 : V;
    uint32_t w[W];
    __device__ __forceinline__ void load(const void *src, int64_t row, int lane) {
        const uint32_t *s = (const uint32_t *)src + (row * 32 + lane) * W;
        if constexpr (W == 2) { const uint2 u = *reinterpret_cast<const uint2 *>(s); w[0] = u.x; w[1] = u.y; }
        else {
#pragma unroll
            for (int i = 0; i < W / 4; i++) {
                const uint4 u = reinterpret_cast<const uint4 *>(s)[i];
                w[4 * i] = u.x; w[4 * i + 1] = u.y; w[4 * i + 2] = u.z; w[4 * i + 3] = u.w;
            }
        }
    }
    __device__ __forceinline__ float operator[](int i) const {
        if constexpr (SRC == SRC_BF16) return __uint_as_float(i & 1 ? w[i >> 1] & 0xFFFF0000u : w[i >> 1] << 16);
        else return __uint_as_float(w[i]);
    }
    // bits of the largest magnitude; 0x7F800000 and up: there is a value that is not finite
    __device__ __forceinline__ uint32_t magnitude() const {
        if constexpr (SRC == SRC_BF16) {                   // two at a time (a NaN wins)
            __nv_bfloat162 m = __habs2(*reinterpret_cast<const __nv_bfloat162 *>(&w[0]));
#pragma unroll
            for (int i = 1; i < W; i++) m = __hmax2_nan(m, __habs2(*reinterpret_cast<const __nv_bfloat162 *>(&w[i])));
            const uint32_t u = *reinterpret_cast<const uint32_t *>(&m);
            return max(u & 0x7FFF0000u, (u << 16) & 0x7FFF0000u);
        }
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < V; i++) m = max(m, __float_as_uint((*this)[i]) & 0x7FFFFFFFu);
        return m;
    }
};
__device__ __forceinline__ uint32_t finite_magnitude(float x) {
    const uint32_t u = __float_as_uint(x) & 0x7FFFFFFFu;
    return u < 0x7F800000u ? u : 0u;
}

// float -> double in integer work: the conversion instructions of 64-bit types run at a small part of the rate of the arithmetic (with
// them the keys of 2100 tokens took 38 us, most of the time in conversions). Not for subnormals.
__device__ __forceinline__ double wide(float x) {
    const uint32_t u = __float_as_uint(x), e = u & 0x7F800000u;
    const uint32_t hi = (u & 0x80000000u) | (((u & 0x7FFFFFFFu) >> 3) + 0x38000000u) | (e == 0x7F800000u ? 0x7FF00000u : 0u);
    return __hiloint2double((int)(e ? hi : u), (int)(e ? u << 29 : 0u));
}
__device__ __forceinline__ bool subnormal(float x) {
    const uint32_t u = __float_as_uint(x) & 0x7FFFFFFFu;
    return u - 1u < 0x7FFFFFu;
}

// The angle of pair i per position.
__device__ __forceinline__ double frequency(double octaves, int i) { return exp2(-(double)i * octaves); }
// cos and sin of the angles at positions pos .. pos + rows - 1 by a warp, [rows][pairs]: the angle taken into [-pi, pi] in double, then
// rounded to float (2^-22); the sum with 1.5 * 2^52 is the nearest whole number of turns. (Not unrolled: the copies of the code that
// forms a cosine would not stay in the instruction cache.)
__device__ __forceinline__ void angles(double octaves, int pairs, int64_t pos, int rows, int lane, float2 *cs) {
#pragma unroll 1
    for (int i = lane; i < pairs; i += 32) {
        const double f = frequency(octaves, i);
#pragma unroll 1
        for (int r = 0; r < rows; r++) {
            const double a = (double)(pos + r) * f, turns = (a * 0.15915494309189533577 + 6755399441055744.0) - 6755399441055744.0;
            float s, c;
            sincosf((float)fma(-turns, 6.283185307179586477, a), &s, &c);
            cs[r * pairs + i] = make_float2(c, s);
        }
    }
    __syncwarp();
}
// the same of one position in double
__device__ __forceinline__ void angles(double octaves, int pairs, int64_t pos, int lane, double2 *cs) {
    __syncwarp();
#pragma unroll 1
    for (int i = lane; i < pairs; i += 32) {
        double c, s;
        sincos((double)pos * frequency(octaves, i), &s, &c);
        cs[i] = make_double2(c, s);
    }
    __syncwarp();
}

// A row's norm and rotation by a warp: y = x * rstd * (1 + w), the first `rot` values turned in pairs (i, i + rot / 2). Errors of a value in
// float, in units of 2^-24: sum of squares 8 roundings, in its root half of that, rsqrtf 4 (two units in the last place), its argument 1, 1 + w 1,
// two products 2, in all 12 of the value's size: < 2^-20. A turned one: angle 4 (rounded from [-pi, pi]), cos and sin 2 (an ulp or two),
// turn 3, in all 21 of the pair's size, which is at most sqrt 2 times the result's |y| + |other|: < 2^-19 of that.
constexpr float KEY_ERR = 0x1p-20f, KEY_ERR_TURNED = 0x1p-19f;
// the lane with the other values of this lane's pairs (itself where it has none)
template <int V>
__device__ __forceinline__ int partner(int rot, int lane) {
    const int d0 = lane * V, shift = rot / 2 / V;
    return d0 < rot / 2 ? lane + shift : d0 < rot ? lane - shift : lane;
}
template <int V, class T, class X, class CS>
__device__ __forceinline__ void norm_rotate(const X &x, T rstd, const T (&w1)[V], int rot, int lane, const CS *cs, T (&y)[V]) {
#pragma unroll
    for (int i = 0; i < V; i++) y[i] = x[i] * rstd * w1[i];
    if (rot == 0) return;
    const int d0 = lane * V, from = partner<V>(rot, lane), pair = d0 < rot / 2 ? d0 : d0 - rot / 2;
    const bool lo = d0 < rot / 2, hi = !lo && d0 < rot;
#pragma unroll
    for (int i = 0; i < V; i++) {
        const T other = __shfl_sync(0xffffffffu, y[i], from);
        if (lo || hi) {
            const CS t = cs[pair + i];
            y[i] = y[i] * t.x + other * (lo ? -t.y : t.y);
        }
    }
}
// this lane's part of a row's sum of squares, and the sum over the warp
template <int V, class T, class X>
__device__ __forceinline__ T squares(const X &x) {
    T sum = 0;
#pragma unroll
    for (int i = 0; i < V; i += 4) {
        const T a = x[i], b = x[i + 1], c = x[i + 2], d = x[i + 3];
        sum += (a * a + b * b) + (c * c + d * d);
    }
    return sum;
}
template <class T>
__device__ __forceinline__ T warp_sum(T sum) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    return sum;
}

// double -> float for a second rounding to few bits: cut off, the last bit set where anything was, so that the second rounding sees
// on which side of a tie the value is. Integer work (conversions run at a quarter of its rate); below 2^-126 it is zero.
__device__ __forceinline__ float to_odd(double y) {
    const uint32_t hi = (uint32_t)__double2hiint(y), lo = (uint32_t)__double2loint(y), mag = hi & 0x7FFFFFFFu;
    const uint32_t f = (mag - 0x38000000u) << 3 | lo >> 29 | (lo << 3 != 0u ? 1u : 0u);
    return __uint_as_float((hi & 0x80000000u) | (mag < 0x38100000u ? 0u : mag >= 0x47F00000u ? (mag > 0x7FF00000u || (mag == 0x7FF00000u && lo) ? 0x7FC00000u : 0x7F800000u) : f));
}

template <int V>
__device__ __forceinline__ void store_words(uint8_t *dst, const uint32_t (&w)[V / 4]) {
    if constexpr (V == 8) *reinterpret_cast<uint2 *>(dst) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<uint32_t *>(dst) = w[0];
}
__device__ __forceinline__ uint32_t low_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}
// Codes of values in units of the scale. careful: some are not finite, or larger than the largest code.
template <int V, bool I8>
__device__ __forceinline__ void codes_of(const float (&y)[V], bool careful, bool is_v, uint32_t (&w)[V / 4]) {
#pragma unroll
    for (int i = 0; i < V / 4; i++) {
        float t[4] = {y[4 * i], y[4 * i + 1], y[4 * i + 2], y[4 * i + 3]};
        if (careful) {
            // A NaN among keys shows in the scores of the queries that see it. Among values it would reach queries that do not: their
            // probability of it is zero, but the product is not. So values take zero in its place.
#pragma unroll
            for (int j = 0; j < 4; j++) if (is_v && t[j] != t[j]) t[j] = 0.f;
            w[i] = kv8_encode4<I8>(t);
        } else if constexpr (I8) {
            uint32_t u[4];                     // plus 1.5 * 2^23: the nearest whole number (ties to even) in the low bits
#pragma unroll
            for (int j = 0; j < 4; j++) u[j] = __float_as_uint(t[j] + 12582912.f);
            w[i] = low_bytes(u[0], u[1], u[2], u[3]);
        } else w[i] = kv8_encode4<I8>(t);
    }
}
// The same of x * f, f a power of two: the product is exact, so it goes with the addition.
template <int V, bool I8, class X>
__device__ __forceinline__ void store_scaled(uint8_t *dst, const X &x, float f, bool careful, bool is_v) {
    uint32_t w[V / 4];
    if (I8 && !careful) {
        uint32_t u[V];
#pragma unroll
        for (int j = 0; j < V; j++) u[j] = __float_as_uint(__fmaf_rn(x[j], f, 12582912.f));
#pragma unroll
        for (int i = 0; i < V / 4; i++) w[i] = low_bytes(u[4 * i], u[4 * i + 1], u[4 * i + 2], u[4 * i + 3]);
    } else {
        float y[V];
#pragma unroll
        for (int j = 0; j < V; j++) y[j] = x[j] * f;
        codes_of<V, I8>(y, careful, is_v, w);
    }
    store_words<V>(dst, w);
}
template <int V, bool I8>
__device__ __forceinline__ void store_codes(uint8_t *dst, const float (&y)[V], bool careful, bool is_v) {
    uint32_t w[V / 4];
    codes_of<V, I8>(y, careful, is_v, w);
    store_words<V>(dst, w);
}

// Rows r0 .. r0 + lead - 1 of an open block move from scale 2^was to 2^e, e > was: 16 codes a thread, two such pieces in flight (one warp
// may have 127 rows to move).
template <int HD, bool I8>
__device__ __forceinline__ void rescale(uint8_t *codes, int64_t ld, int lead, int was, int e, bool is_v) {
    constexpr int CH = HD / 16, U = 2;
    const float f = was - e < -126 ? 0.f : kv8_two(was - e);
    for (int i0 = threadIdx.x; i0 < lead * CH; i0 += U * blockDim.x) {
        uint4 c[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int i = i0 + u * blockDim.x;
            if (i < lead * CH) c[u] = *reinterpret_cast<const uint4 *>(codes + (i / CH) * ld + (i % CH) * 16);
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int i = i0 + u * blockDim.x;
            if (i >= lead * CH) break;
            uint8_t *at = codes + (i / CH) * ld + (i % CH) * 16;
            const uint32_t w[4] = {c[u].x, c[u].y, c[u].z, c[u].w};
#pragma unroll
            for (int k = 0; k < 4; k += 2) {
                float y[8];
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    uint32_t a, b;
                    kv8_decode4<I8>(w[k + h], a, b);
                    const float2 v0 = __half22float2(*reinterpret_cast<const __half2 *>(&a)), v1 = __half22float2(*reinterpret_cast<const __half2 *>(&b));
                    y[4 * h] = v0.x * f; y[4 * h + 1] = v0.y * f; y[4 * h + 2] = v1.x * f; y[4 * h + 3] = v1.y * f;
                }
                store_codes<8, I8>(at + 4 * k, y, true, is_v);
            }
        }
    }
}

// A reciprocal root in float of squares that leave float's range, or are so small that they have few bits: below 1e17 the sum of 128 squares
// or more is above 2^-106, and what each loses below 2^-149 is nothing beside it.
__device__ __forceinline__ bool out_of_range(float rstd) { return !(rstd > 1e-15f && rstd < 1e17f); }
template <int V>
__device__ __forceinline__ void store_query(uint16_t *dst, const float (&y)[V]) {
    uint32_t o[V / 2];
#pragma unroll
    for (int k = 0; k < V / 2; k++) o[k] = pack_bf16x2(y[2 * k], y[2 * k + 1]);
    if constexpr (V == 8) *reinterpret_cast<uint4 *>(dst) = make_uint4(o[0], o[1], o[2], o[3]);
    else *reinterpret_cast<uint2 *>(dst) = make_uint2(o[0], o[1]);
}
// Those of query heads h0 .. h0 + heads - 1 of a token again, multiplied by a power of two first, and epsilon by its square: large rows (root of the
// mean 2^49 and up) come below 2^48, small ones are at most 2^44, the least subnormal 2^-49. (Not inlined: to 7 x 300 rows that
// have no use for it, 19.6 us, it adds 0.9 in line and so 0.4 to 0.5.)
template <int V>
__device__ __noinline__ void query_rows_out_of_range(const Kv8PrepParams &p, int64_t t, int h0, int heads, int lane, const float2 *csf) {
    constexpr int HD = 32 * V;
    Raw<V, SRC_F32> w;
    w.load(p.q_norm, 0, lane);
    float w1[V];
#pragma unroll
    for (int i = 0; i < V; i++) w1[i] = 1.f + w[i];
#pragma unroll 1
    for (int i = 0; i < heads; i++) {
        Raw<V, SRC_F32> x;
        x.load(p.qg, (t * p.nh + h0 + i) * 2, lane);
        const float sum = warp_sum(squares<V, float>(x)), unit = sum > 1.f ? 0x1p-80f : 0x1p100f;
        if (!out_of_range(rsqrtf(sum * (1.f / HD) + p.eps))) continue;
        float z[V], y[V];
#pragma unroll
        for (int k = 0; k < V; k++) z[k] = x[k] * unit;
        norm_rotate<V, float>(z, rsqrtf(warp_sum(squares<V, float>(z)) * (1.f / HD) + p.eps * unit * unit), w1, p.rot, lane, csf, y);
        store_query<V>(p.q_out + (t * p.nh + h0 + i) * HD + lane * V, y);
    }
}

// V: values of a row per lane (head dim / 32); ROWS: rows of a warp. PREP: f32 rows, keys normed and rotated; blocks from p.tasks on have
// query rows.
template <int V, int SRC, bool I8, class PARAMS, int ROWS>
__global__ void __launch_bounds__(512, SRC == SRC_BF16 ? 2 : 1) kv8_write_kernel(const __grid_constant__ PARAMS p) {
    constexpr bool PREP = std::is_same<PARAMS, Kv8PrepParams>::value;
    constexpr int HD = 32 * V;
    extern __shared__ double2 s_cs[];                      // PREP: of a warp, [ROWS][rot / 2] cos and sin in float, or [rot / 2] in double
    __shared__ uint32_t s_max[16];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    cwk_pdl_launch();
    cwk_pdl_wait();
    if constexpr (PREP) if (blockIdx.x >= p.tasks) {
        const int pairs = p.rot / 2;
        float2 *csf = reinterpret_cast<float2 *>(s_cs) + warp * ROWS * pairs;
        // ---- query rows: a warp has `heads` heads of one token
        const int parts = (p.nh + p.heads - 1) / p.heads;
        const int64_t id = ((int64_t)blockIdx.x - p.tasks) * warps + warp, t = id / parts;
        if (t >= (int64_t)p.B * p.n) return;
        const int b = (int)(t / p.n), j = (int)(t % p.n), h0 = (int)(id % parts) * p.heads, heads = min(p.heads, p.nh - h0);
        Raw<V, SRC_F32> x[KQ_HEADS], w;
        w.load(p.q_norm, 0, lane);
#pragma unroll
        for (int i = 0; i < KQ_HEADS; i++)
            if (i < heads) x[i].load(p.qg, (t * p.nh + h0 + i) * 2, lane);      // rows [q | gate] of 2 * hd
        int64_t pos;
        if (j >= new_rows(p, b, pos)) return;
        angles(p.octaves, pairs, pos + j, 1, lane, csf);
        float w1[V];
#pragma unroll
        for (int i = 0; i < V; i++) w1[i] = 1.f + w[i];
        float least = 1.f, most = 1.f;                     // of the reciprocal roots
#pragma unroll
        for (int i = 0; i < KQ_HEADS; i++) {
            if (i >= heads) break;
            const float r = rsqrtf(warp_sum(squares<V, float>(x[i])) * (1.f / HD) + p.eps);
            least = fminf(least, r);
            most = fmaxf(most, r);
            float y[V];
            norm_rotate<V, float>(x[i], r, w1, p.rot, lane, csf, y);
            store_query<V>(p.q_out + (t * p.nh + h0 + i) * HD + lane * V, y);
        }
        if (least <= 1e-15f || most >= 1e17f) query_rows_out_of_range<V>(p, t, h0, heads, lane, csf);
        return;
    }
    uint32_t id = blockIdx.x;
    const int head = (int)(id % p.nkv); id /= p.nkv;
    const int win = (int)(id % p.window); id /= p.window;
    const int b = (int)(id % p.B);
    const bool is_v = id / p.B != 0;                       // (all keys first: their tasks are the longer ones)
    int64_t pos;
    const int cnt = new_rows(p, b, pos);
    const int64_t blk = (pos >> p.lb) + win, r0 = blk << p.lb;
    const int64_t lo = max(r0, pos), hi = min(r0 + (1 << p.lb), pos + cnt);
    if (lo >= hi) return;
    uint8_t *codes = (is_v ? p.vc : p.kc) + (((int64_t)b * p.rows + r0) * p.nkv + head) * HD;
    uint8_t *scale = (is_v ? p.vs : p.ks) + ((int64_t)b * (p.rows >> p.lb) + blk) * p.nkv + head;
    const int64_t ld = (int64_t)p.nkv * HD;
    const int lead = (int)(lo - r0), many = (int)(hi - lo);
    const int was_byte = lead > 0 ? (int)*scale : 0;
    const int first = warp * ROWS, mine = min(ROWS, many - first);      // this warp's rows: lo + first .. (none: <= 0)
    const void *src = is_v ? p.v : p.k;
    const int64_t row = ((int64_t)b * p.n + (lo - pos) + first) * p.nkv + head;
    // over the task: the largest of a value's bits
    auto task_max = [&](uint32_t m) {
        m = __reduce_max_sync(0xffffffffu, m);
        if (lane == 0) s_max[warp] = m;
        __syncthreads();
        for (int i = 0; i < warps; i++) m = max(m, s_max[i]);
        return m;
    };
    int e;
    bool careful;                                          // some values are not finite, or larger than the largest code
    auto settle = [&](uint32_t amax, bool odd) {
        e = kv8_exponent(__uint_as_float(amax), I8);
        careful = odd || e == kv8_high(I8);
        if (lead > 0) {
            const int was = min(max(was_byte - 127, KV8_LOW), kv8_high(I8));
            if (was >= e) e = was;
            else rescale<HD, I8>(codes, ld, lead, was, e, is_v);
        }
        if (threadIdx.x == 0) *scale = (uint8_t)(e + 127);
    };
    uint8_t *dst = codes + (lead + first) * ld + lane * V;
    Raw<V, SRC> x[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; i++)
        if (i < mine) x[i].load(src, row + i * p.nkv, lane);
    if constexpr (PREP) if (!is_v) {
        const int pairs = p.rot / 2;
        float2 *csf = reinterpret_cast<float2 *>(s_cs) + warp * ROWS * pairs;
        double2 *cs = reinterpret_cast<double2 *>(csf);    // (one of them at a time)
        // ---- keys. A code is that of the value in 64 bits, formed in float: where a float's error could change the code (or the
        // exponent), the row (or the largest magnitude) is formed again in double. That is one row in thirty or less, and double, with its
        // conversions, is some eight times the work: 512 tokens 20 us with all rows in double.
        Raw<V, SRC_F32> w;
        w.load(p.k_norm, 0, lane);
        auto row64 = [&](int r, double (&y)[V]) {
            Raw<V, SRC> z;
            z.load(src, row + r * p.nkv, lane);
            double x64[V], w1[V];
            bool some = false;
#pragma unroll
            for (int i = 0; i < V; i++) {
                x64[i] = wide(z[i]);
                w1[i] = 1.0 + wide(w[i]);
                some |= subnormal(z[i]);
            }
            if (some)                                      // (an ordinary row has none)
#pragma unroll
                for (int i = 0; i < V; i++) x64[i] = (double)z[i];
            angles(p.octaves, pairs, lo + first + r, lane, cs);
            norm_rotate<V, double>(x64, rsqrt(warp_sum(squares<V, double>(x64)) / (double)HD + (double)p.eps), w1, p.rot, lane, cs, y);
        };
        float y[ROWS][V];
        uint32_t amax = 0;
        bool unsure = false;
        angles(p.octaves, pairs, lo + first, max(mine, 0), lane, csf);
        {
            float w1[V];
#pragma unroll
            for (int i = 0; i < V; i++) w1[i] = 1.f + w[i];
#pragma unroll
            for (int i = 0; i < ROWS; i++) {
                if (i >= mine) break;
                const float r = rsqrtf(warp_sum(squares<V, float>(x[i])) * (1.f / HD) + p.eps);
                unsure |= out_of_range(r);
                norm_rotate<V, float>(x[i], r, w1, p.rot, lane, csf + i * pairs, y[i]);
#pragma unroll
                for (int j = 0; j < V; j++) amax = max(amax, __float_as_uint(y[i][j]) & 0x7FFFFFFFu);
            }
        }
        amax = task_max(amax);
        const float top = __uint_as_float(amax);
        bool odd = false;
        unsure |= amax >= 0x7F800000u;
        const bool all64 = __syncthreads_or(unsure);       // no row's float values are good
        if (all64 || kv8_exponent(top * (1.f - 4.f * KEY_ERR_TURNED), I8) != kv8_exponent(top * (1.f + 4.f * KEY_ERR_TURNED), I8)) {
            uint32_t finite = 0, all = 0;
#pragma unroll 1
            for (int r = 0; r < mine; r++) {
                double z[V];
                row64(r, z);
#pragma unroll
                for (int j = 0; j < V; j++) {
                    const float up = __double2float_ru(fabs(z[j]));      // never below the value
                    finite = max(finite, finite_magnitude(up));
                    all = max(all, __float_as_uint(up) & 0x7FFFFFFFu);
                }
            }
            odd = __syncthreads_or(all >= 0x7F800000u);
            amax = task_max(finite);
        }
        settle(amax, odd);
        const float f = kv8_two(-e);
        uint32_t again = 0;                                // rows of which some value's code is not certain
        const int from = partner<V>(p.rot, lane);
        const bool turned = lane * V < p.rot;
#pragma unroll
        for (int i = 0; i < ROWS; i++) {
            if (i >= mine) break;
            float a[V], b[V];
#pragma unroll
            for (int j = 0; j < V; j++) {
                const float other = __shfl_sync(0xffffffffu, y[i][j], from);
                const float err = turned ? (fabsf(y[i][j]) + fabsf(other)) * KEY_ERR_TURNED : fabsf(y[i][j]) * KEY_ERR;
                a[j] = (y[i][j] - err) * f;
                b[j] = (y[i][j] + err) * f;
            }
            // what lies between two values of one code has that code
            uint32_t wa[V / 4], wb[V / 4], differ = 0;
            codes_of<V, I8>(a, careful, false, wa);
            codes_of<V, I8>(b, careful, false, wb);
#pragma unroll
            for (int j = 0; j < V / 4; j++) differ |= wa[j] ^ wb[j];
            if (all64 || __any_sync(0xffffffffu, differ != 0)) again |= 1u << i;
            else store_words<V>(dst + i * ld, wa);
        }
        const double f64 = wide(f);
#pragma unroll 1
        for (; again; again &= again - 1) {
            const int r = __ffs(again) - 1;
            double z[V];
            row64(r, z);
            float q[V];
            // INT8: the nearest whole number, as a float; E4M3: to odd, then (in codes_of) to nearest
#pragma unroll
            for (int j = 0; j < V; j++) {
                if constexpr (I8) q[j] = z[j] == z[j] ? (float)rint(fmin(fmax(z[j] * f64, -127.0), 127.0)) : 0.f;
                else q[j] = to_odd(z[j] * f64);
            }
            store_codes<V, I8>(dst + r * ld, q, true, false);
        }
        return;
    }
    uint32_t all = 0;
#pragma unroll
    for (int i = 0; i < ROWS; i++)
        if (i < mine) all = max(all, x[i].magnitude());
    uint32_t amax = all;
    if (all >= 0x7F800000u) {                              // an infinity saturates and does not set the scale; nor does a NaN
        amax = 0;
#pragma unroll
        for (int i = 0; i < ROWS; i++)
#pragma unroll
            for (int j = 0; j < V; j++)
                if (i < mine) amax = max(amax, finite_magnitude(x[i][j]));
    }
    const bool odd = __syncthreads_or(all >= 0x7F800000u);
    settle(task_max(amax), odd);
    const float f = kv8_two(-e);
#pragma unroll
    for (int i = 0; i < ROWS; i++, dst += ld) {
        if (i >= mine) break;
        store_scaled<V, I8>(dst, x[i], f, careful, is_v);
    }
}

// Codes -> values. pos[b] + j for j < count[b] (cwk_kv8_load), or one slot's rows from row0 on (cwk_kv8_widen, pos NULL).
struct Kv8ReadParams {
    const uint8_t *kc, *vc, *ks, *vs;
    int64_t rows, row0;
    const int32_t *pos, *count;
    int B, nkv, lb;
    int64_t n;
    void *k, *v;
};
constexpr int KR_THREADS = 128, KR_ROWS = 4;

// A thread has eight codes (head, place in it) of every `step`-th row of a slot, KR_ROWS rows in flight. grid (chunks of rows, slot, K or V)
template <int HD, bool I8, bool F32>
__global__ void __launch_bounds__(KR_THREADS) kv8_read_kernel(const Kv8ReadParams p) {
    constexpr int PER = 8, CH = HD / PER;                  // codes per thread and row; such pieces of a head
    cwk_pdl_launch();
    const int b = blockIdx.y, pieces = p.nkv * CH;         // of a row
    // rows that the block's threads have at once; a row wider than the block is done in parts
    const int step = max(KR_THREADS / pieces, 1), r = (int)threadIdx.x / pieces, at0 = (int)threadIdx.x % pieces;
    if (r >= step) return;
    cwk_pdl_wait();
    const uint8_t *codes = (blockIdx.z ? p.vc : p.kc) + (int64_t)b * p.rows * p.nkv * HD, *scales = (blockIdx.z ? p.vs : p.ks) + (int64_t)b * (p.rows >> p.lb) * p.nkv;
    uint8_t *out = (uint8_t *)(blockIdx.z ? p.v : p.k) + (int64_t)b * p.n * p.nkv * HD * (F32 ? 4 : 2);
    const int64_t pos = p.pos ? (int64_t)p.pos[b] : p.row0;
    const int64_t end = pos < 0 ? 0 : min(min(p.n, p.count ? (int64_t)p.count[b] : p.n), p.rows - pos), j0 = (int64_t)blockIdx.x * (step * KR_ROWS) + r;
    for (int at = at0; at < pieces; at += KR_THREADS) {
        const int head = at / CH;
        uint2 c[KR_ROWS];
        uint32_t s[KR_ROWS];
#pragma unroll
        for (int u = 0; u < KR_ROWS; u++) {
            const int64_t j = j0 + u * step, row = pos + j;
            if (j >= end) continue;
            c[u] = *reinterpret_cast<const uint2 *>(codes + (row * pieces + at) * PER);
            s[u] = scales[(row >> p.lb) * p.nkv + head];
        }
#pragma unroll
        for (int u = 0; u < KR_ROWS; u++) {
            const int64_t j = j0 + u * step;
            if (j >= end) continue;
            const float f = kv8_scale(s[u]);
            uint32_t h[4];
            kv8_decode4<I8>(c[u].x, h[0], h[1]);
            kv8_decode4<I8>(c[u].y, h[2], h[3]);
            float2 y[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                y[i] = __half22float2(*reinterpret_cast<const __half2 *>(&h[i]));
                y[i].x *= f; y[i].y *= f;
            }
            if constexpr (F32) {
                float4 *o = reinterpret_cast<float4 *>(out + (j * pieces + at) * PER * 4);
                o[0] = make_float4(y[0].x, y[0].y, y[1].x, y[1].y);
                o[1] = make_float4(y[2].x, y[2].y, y[3].x, y[3].y);
            } else {
                uint32_t w[4];
#pragma unroll
                for (int i = 0; i < 4; i++) w[i] = pack_bf16x2(y[i].x, y[i].y);       // exact
                *reinterpret_cast<uint4 *>(out + (j * pieces + at) * PER * 2) = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
    }
}

int log2_of(int block) { return block == 32 ? 5 : block == 64 ? 6 : 7; }

int launch_read(cwk_ctx *ctx, const Kv8ReadParams &p, int hd, bool i8, bool f32) {
    const int per_block = std::max(KR_THREADS / (p.nkv * (hd / 8)), 1) * KR_ROWS;
    const int64_t chunks = (p.n + per_block - 1) / per_block;
    if (chunks > 0x7FFFFFFF || p.B > 65535) return cwk_fail(ctx, CWK_ERR_ARGUMENT, "kv8_load: too many rows or slots in one call");
    void (*kern)(Kv8ReadParams);
    if (hd == 256) kern = i8 ? (f32 ? kv8_read_kernel<256, true, true> : kv8_read_kernel<256, true, false>)
                             : (f32 ? kv8_read_kernel<256, false, true> : kv8_read_kernel<256, false, false>);
    else kern = i8 ? (f32 ? kv8_read_kernel<128, true, true> : kv8_read_kernel<128, true, false>)
                   : (f32 ? kv8_read_kernel<128, false, true> : kv8_read_kernel<128, false, false>);
    CWK_CUDA(ctx, cwk_launch_early(kern, dim3((unsigned)chunks, p.B, 2), dim3(KR_THREADS), 0, ctx->stream, p));
    ctx->launches++;
    return CWK_OK;
}

template <int V, int SRC, int ROWS, class PARAMS>
int launch_write_rows(cwk_ctx *ctx, PARAMS &p, int type) {
    const int block = 1 << p.lb, warps = (std::min(block, p.n) + ROWS - 1) / ROWS;
    p.window = (int)(((int64_t)p.n + block - 2) / block + 1);
    const int64_t tasks = (int64_t)2 * p.B * p.window * p.nkv;
    int64_t blocks = tasks;
    size_t smem = 0;
    auto kern = type == CWK_KV8_INT8 ? kv8_write_kernel<V, SRC, true, PARAMS, ROWS> : kv8_write_kernel<V, SRC, false, PARAMS, ROWS>;
    if constexpr (std::is_same<PARAMS, Kv8PrepParams>::value) {
        p.tasks = tasks;
        // Query heads of a token that share its angles and are on their way together; few rows: a warp each. A warp for one / for eight, 16 heads
        // of 256, replayed: 64 slots 4.4 / 5.0 us, 128 slots 4.6 / 5.3, 256 slots 7.7 / 6.8, 512 tokens of one 11.1 / 9.1.
        p.heads = p.n * (int64_t)p.B * p.nh <= 2048 ? 1 : KQ_HEADS;
        blocks += ((int64_t)p.B * p.n * ((p.nh + p.heads - 1) / p.heads) + warps - 1) / warps;
        smem = (size_t)(p.rot / 2) * warps * ROWS * sizeof(float2);      // 128 KB at most (32 KB for 64 values in blocks of 128 rows)
        static bool attr_set[2][16] = {};
        bool &set = attr_set[type == CWK_KV8_INT8][ctx->device & 15];
        if (!set) CWK_CUDA(ctx, cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 128 << 10));
        set = true;
    }
    if (blocks > 0x7FFFFFFF) return cwk_fail(ctx, CWK_ERR_ARGUMENT, "kv8 write: too many rows in one call");
    CWK_CUDA(ctx, cwk_launch_early(kern, dim3((unsigned)blocks), dim3(32 * warps), smem, ctx->stream, p));
    ctx->launches++;
    return CWK_OK;
}
// Rows of a warp: eight, and four for the preparation of shorter blocks, whose keys go from row to row.
template <int V, int SRC>
int launch_write(cwk_ctx *ctx, Kv8StoreParams &p, int type) { return launch_write_rows<V, SRC, 8>(ctx, p, type); }
template <int V, int SRC>
int launch_write(cwk_ctx *ctx, Kv8PrepParams &p, int type) {
    return p.lb == 7 ? launch_write_rows<V, SRC, 8>(ctx, p, type) : launch_write_rows<V, SRC, 4>(ctx, p, type);
}

void describe(Kv8StoreParams &p, const cwk_kv8 *c, const void *k, const void *v, const int32_t *pos, const int32_t *count, int B, int n) {
    p.k = k; p.v = v; p.pos = pos; p.count = count; p.B = B; p.n = n; p.nkv = c->nkv; p.lb = log2_of(c->block); p.rows = c->rows;
    p.kc = (uint8_t *)c->k; p.vc = (uint8_t *)c->v; p.ks = c->k_scale; p.vs = c->v_scale;
}

bool aligned(const void *a, const void *b) { return (((uintptr_t)a | (uintptr_t)b) & 15) == 0; }

}  // namespace

int cwk_kv8_check(cwk_ctx *ctx, const cwk_kv8 *c, const char *who) {
    if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale) return cwk_fail(ctx, CWK_ERR_ARGUMENT, "%s: null cache", who);
    if (c->hd != 128 && c->hd != 256) return cwk_fail(ctx, CWK_ERR_UNSUPPORTED, "%s: head_dim %d not built (128 or 256)", who, c->hd);
    if (c->block != 32 && c->block != 64 && c->block != 128)
        return cwk_fail(ctx, CWK_ERR_UNSUPPORTED, "%s: blocks of %d rows not built (32, 64 or 128)", who, c->block);
    if (c->type != CWK_KV8_E4M3 && c->type != CWK_KV8_INT8) return cwk_fail(ctx, CWK_ERR_UNSUPPORTED, "%s: unknown code type %d", who, c->type);
    if (c->slots <= 0 || c->nkv <= 0 || c->nkv > 65535 || c->rows <= 0 || c->rows % c->block != 0 || c->rows > 0x7FFFFF00)
        return cwk_fail(ctx, CWK_ERR_ARGUMENT, "%s: bad cache dimensions (rows: a multiple of the block, below 2^31 - 256)", who);
    if (!aligned(c->k, c->v)) return cwk_fail(ctx, CWK_ERR_ARGUMENT, "%s: the codes must be 16-byte aligned", who);
    return CWK_OK;
}

int cwk_kv8_widen(cwk_ctx *ctx, const cwk_kv8 &c, int64_t row0, int64_t n, void *k, void *v) {
    Kv8ReadParams p{};
    p.kc = (const uint8_t *)c.k; p.vc = (const uint8_t *)c.v; p.ks = c.k_scale; p.vs = c.v_scale;
    p.rows = c.rows; p.row0 = row0; p.B = 1; p.nkv = c.nkv; p.lb = log2_of(c.block); p.n = n; p.k = k; p.v = v;
    return launch_read(ctx, p, c.hd, c.type == CWK_KV8_INT8, false);
}

extern "C" {

int cwk_kv8_store(cwk_ctx *ctx, const cwk_kv8 *c, const void *k, const void *v, int f32, const int32_t *pos, const int32_t *count, int B, int n) {
    int s = cwk_kv8_check(ctx, c, "kv8_store");
    if (s != CWK_OK) return s;
    if (!ctx || !k || !v || !pos) return cwk_fail(ctx, CWK_ERR_ARGUMENT, "kv8_store: null argument");
    if (B <= 0 || n <= 0 || B > c->slots) return cwk_fail(ctx, CWK_ERR_ARGUMENT, "kv8_store: bad dimensions (%d slots, %d rows)", B, n);
    if (!aligned(k, v)) return cwk_fail(ctx, CWK_ERR_ARGUMENT, "kv8_store: pointers must be 16-byte aligned");
    CWK_CUDA(ctx, cudaSetDevice(ctx->device));
    Kv8StoreParams p{};
    describe(p, c, k, v, pos, count, B, n);
    CwkKernelTimer timer(ctx);
    if (c->hd == 256) return f32 ? launch_write<8, SRC_F32>(ctx, p, c->type) : launch_write<8, SRC_BF16>(ctx, p, c->type);
    return f32 ? launch_write<4, SRC_F32>(ctx, p, c->type) : launch_write<4, SRC_BF16>(ctx, p, c->type);
}

int cwk_kv8_load(cwk_ctx *ctx, const cwk_kv8 *c, const int32_t *pos, const int32_t *count, int B, int n, void *k, void *v, int f32) {
    int s = cwk_kv8_check(ctx, c, "kv8_load");
    if (s != CWK_OK) return s;
    if (!ctx || !k || !v || !pos) return cwk_fail(ctx, CWK_ERR_ARGUMENT, "kv8_load: null argument");
    if (B <= 0 || n <= 0 || B > c->slots) return cwk_fail(ctx, CWK_ERR_ARGUMENT, "kv8_load: bad dimensions (%d slots, %d rows)", B, n);
    if (!aligned(k, v)) return cwk_fail(ctx, CWK_ERR_ARGUMENT, "kv8_load: pointers must be 16-byte aligned");
    CWK_CUDA(ctx, cudaSetDevice(ctx->device));
    Kv8ReadParams p{};
    p.kc = (const uint8_t *)c->k; p.vc = (const uint8_t *)c->v; p.ks = c->k_scale; p.vs = c->v_scale;
    p.rows = c->rows; p.pos = pos; p.count = count; p.B = B; p.nkv = c->nkv; p.lb = log2_of(c->block); p.n = n; p.k = k; p.v = v;
    CwkKernelTimer timer(ctx);
    return launch_read(ctx, p, c->hd, c->type == CWK_KV8_INT8, f32 != 0);
}

int cwk_gqa_qk_prep_kv8(cwk_ctx *ctx, const float *qg, const float *k, const float *v, const float *q_norm, const float *k_norm, float eps, int rot,
                        double theta, const int32_t *pos, const int32_t *count, int B, int n, int nh, void *q_out, const cwk_kv8 *c) {
    int s = cwk_kv8_check(ctx, c, "gqa_qk_prep_kv8");
    if (s != CWK_OK) return s;
    if (!ctx || !qg || !k || !v || !q_norm || !k_norm || !pos || !q_out) return cwk_fail(ctx, CWK_ERR_ARGUMENT, "gqa_qk_prep_kv8: null argument");
    if (B <= 0 || n <= 0 || nh <= 0 || B > c->slots) return cwk_fail(ctx, CWK_ERR_ARGUMENT, "gqa_qk_prep_kv8: bad dimensions");
    if (rot < 0 || rot > c->hd || (rot > 0 && !(theta > 0.0))) return cwk_fail(ctx, CWK_ERR_ARGUMENT, "gqa_qk_prep_kv8: bad rotation (%d of %d, base %g)", rot, c->hd, theta);
    if (rot % 16 != 0) return cwk_fail(ctx, CWK_ERR_UNSUPPORTED, "gqa_qk_prep_kv8: rotation of %d values not built (a multiple of 16)", rot);
    if (!aligned(k, v) || !aligned(qg, q_out) || !aligned(q_norm, k_norm))
        return cwk_fail(ctx, CWK_ERR_ARGUMENT, "gqa_qk_prep_kv8: pointers must be 16-byte aligned");
    CWK_CUDA(ctx, cudaSetDevice(ctx->device));
    Kv8PrepParams p{};
    describe(p, c, k, v, pos, count, B, n);
    p.qg = qg; p.q_norm = q_norm; p.k_norm = k_norm; p.q_out = (uint16_t *)q_out; p.nh = nh; p.rot = rot; p.eps = eps;
    p.octaves = rot > 0 ? 2.0 * log2(theta) / rot : 0.0;
    CwkKernelTimer timer(ctx);
    return c->hd == 256 ? launch_write<8, SRC_F32>(ctx, p, c->type) : launch_write<4, SRC_F32>(ctx, p, c->type);
}

}  // extern "C"
