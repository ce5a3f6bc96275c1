// kv8_decode.cu -- GQA decode over a cache held in 8 bits (kv8.cuh), for a batch of sequences with lengths of their own and one or a few
// query tokens each, and the entry of the prompt chunk over such a cache.
//
// The streams of gqa_decode.cu over half the bytes: no warp waits for another one, every warp has a ring of its own (32 keys a stage, K and V
// codes, filled by asynchronous copies), its own running maximum, sum and output, and the steps of all sequences are dealt out in equal
// contiguous ranges (gqa_steps.cuh). Codes become f16 in registers, exactly, on the way into mma.m16n8k16 (f16 operands, f32 sums), keys or
// value columns as its sixteen rows, query rows as its eight columns:
//   scores   a lane's 4 neighbouring bytes of a key are the MMA's k positions 2t, 2t+1, 2t+8, 2t+9: the dims are only renumbered, for
//            the queries alike, and no byte moves.
//   values   ldmatrix.trans on pairs of bytes gives a lane two keys of two neighbouring columns; one byte permutation pairs the keys, and
//            the even column goes to row g of the MMA, the odd one to row g + 8.
// The queries go to f16 too: each row divided by a power of two that brings its largest value into [1, 2), so what is lost is below
// 2^-25 of that value, 2^-16 of a bf16 step. Probabilities are f16 in [0, 2^8], three bits finer than bf16's from 2^-14 up; below, the
// step stays 2^-24, and one under 2^-25 is zero in the product while the f32 sum counts it: 10,000 such keys of a warp are 3e-4 of its
// largest, a thirteenth of the result's own rounding. The sums are f32. The scales are powers of two: a step's 32 keys are in one
// block, the key scale multiplies its scores and the value scale its product on the way into the f32 accumulators, so no code's value
// is ever rounded or out of f16's range.
//
// What bounds it: a batch by HBM, 64 sequences of 4096 rows (16 heads, 4 KV heads of 256, 537 MB) 91 us = 5.9 TB/s, INT8 the same, four tokens each 110;
// less by the start and the end of the streams, 16 sequences 32 us, one 8.4, of 32768 rows 21 (replayed); short caches by a warp's chain of steps,
// 1.4 us for 32 keys (2.1 with sixteen query rows), 16 sequences of 128 rows 5.1.
#include <algorithm>

#include "gqa_steps.cuh"
#include "kv8.cuh"

namespace {

constexpr int GW = 4;                 // warps per block
constexpr int GK = 32;                // keys per warp and step; every block of the cache is a multiple of it
constexpr float GQ_LAZY = 8.f;        // a score may outrun the reference exponent by 2^8 before a rescale

struct Kv8DecodeParams {
    const uint16_t *q;                // bf16 [B][n][nh][hd]
    const uint8_t *k, *v, *ks, *vs;
    int64_t rows;                     // per slot
    uint16_t *out;                    // bf16 [B][n][nh][hd]
    float *rec;                       // [slot][warp]: o [per * group][hd], then {m, l} [per * group]
    GqaSteps steps;                   // groups: (nkv / hb) * parts, the parts of the same keys next to each other; keys: GK * (GW / hb)
    int n, nkv, group, hb, lb;        // hb: KV heads a block works on at once (4, 2 or 1); block = 1 << lb
    int per, parts;                   // query tokens whose heads share the MMA columns; parts = ceil(n / per)
    float scale_log2;
    __host__ __device__ int nh() const { return nkv * group; }
};

// (Parameters of more than 128 bytes, or of bytes, come later: with eight bytes more a step of one sequence of 4096 rows took 9.3 us instead
// of 8.2, with heads and shifts as bytes 8.9.)
static_assert(sizeof(Kv8DecodeParams) <= 128, "kernel parameters");

__device__ __forceinline__ void mma_f16_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16_16816_zero(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {      // the first of a sum
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}

// floats of a warp's record: o [cols][HD], {m, l} [cols], a multiple of 16 bytes. Of 32 columns of o, those that one lane has are next to each other,
// 2 g, 2 g + 1, 16 + 2 g, 17 + 2 g, so that a record goes out in whole lines (four
// tokens of 16 sequences of 4096 rows, 19 MB of records, 46 -> 42 us).
__host__ __device__ __forceinline__ constexpr int kv8_record(int cols, int hd) { return cols * hd + ((2 * cols + 3) & ~3); }

// Places of a warp's ring, each the K or the V of a step: 24 KB a warp, so that two blocks of four warps are on an SM and a scheduler has
// two of these chains of dependent instructions to choose from. Sixteen query rows of 256 leave no registers for the query fragments
// beside the accumulators: they take the third place of the ring (4 tokens of 64 sequences of 4096 rows 124 -> 107 us).
template <int HD, int NB> constexpr bool KV8_Q_SHARED = HD == 256 && NB == 2;
template <int HD, int NB> constexpr int KV8_RING = KV8_Q_SHARED<HD, NB> ? 2 : HD == 256 ? 3 : 6;

// A running softmax sum of one query row, four columns of it.
struct Kv8Sum {
    float M = -INFINITY, den = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    __device__ __forceinline__ void add(float w, float l, const float4 &v) {
        den += w * l; o.x += w * v.x; o.y += w * v.y; o.z += w * v.z; o.w += w * v.w;
    }
    __device__ __forceinline__ void raise(float to) {      // to a reference exponent that is not lower
        const float a = exp2f(M - to);
        den *= a; o.x *= a; o.y *= a; o.z *= a; o.w *= a;
        M = to;
    }
    // out: the row, place: of the four columns in a record
    __device__ __forceinline__ void write(uint16_t *out, int place) const {
        const float inv = den != 0.f ? 1.f / den : 0.f;
        out += place / 32 * 32 + place % 32 / 2;
        *reinterpret_cast<uint32_t *>(out) = pack_bf16x2(o.x * inv, o.y * inv);
        *reinterpret_cast<uint32_t *>(out + 16) = pack_bf16x2(o.z * inv, o.w * inv);
    }
};

// NB: groups of eight MMA columns (query rows). WHOLE: a block has one head group of one sequence from its first row to its last, joins its
// own warps' records in shared memory and writes the output; otherwise its share of all steps, and records for the merge.
template <int HD, int NB, bool I8, bool WHOLE>
__global__ void __launch_bounds__(32 * GW, 2) kv8_decode_kernel(const Kv8DecodeParams p) {
    constexpr int CH = HD / 16;                           // 16-byte pieces per row
    constexpr int RING = KV8_RING<HD, NB>;
    constexpr bool QS = KV8_Q_SHARED<HD, NB>;
    constexpr int KB = GK * HD;                           // bytes of a place of the ring
    extern __shared__ __align__(128) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, lg = lane >> 2, lt = lane & 3;
    const uint32_t ring = smem_u32(smem) + warp * (RING + (QS ? 1 : 0)) * KB;
    uint4 *qs = reinterpret_cast<uint4 *>(smem + (warp * (RING + 1) + RING) * KB) + lane;      // QS: [HD / 16][lane]
    static_assert(!QS || HD / 16 * 32 * 16 <= KB, "query fragments");
    const int sub = warp / p.hb, wh = warp % p.hb;        // which 32 keys of a step, which KV head of the group
    const int keys = p.steps.keys, cols = p.per * p.group;
    GqaPlace at{0, 0, 0, 0, 0};
    cwk_pdl_launch();
    // (into L2 only, where the kernel before may still write them: what is spared is the way there)
    if (p.steps.kv_len && lane < p.steps.B) asm volatile("prefetch.global.L2 [%0];" ::"l"(p.steps.kv_len + lane));
    cwk_pdl_wait();
    GqaList list;
    int n;
    if constexpr (WHOLE) {
        at.b = (int)blockIdx.x / p.steps.groups;
        at.hg = (int)blockIdx.x % p.steps.groups;
        at.len = length_of(p.steps, at.b);
        at.steps = n = (at.len + keys - 1) / keys;
    } else {
        n = gqa_range(p.steps, lane, list, at);
        if (n <= 0) {
            if (warp == 0) gqa_note(p.steps, list, lane);
            return;
        }
        at.len = length_of(p.steps, at.b);
    }
    GqaPlace ld = at;                                     // the step being loaded
    auto head_of = [&](const GqaPlace &x) { return (x.hg / p.parts) * p.hb + wh; };
    auto query = [&](const GqaPlace &x, int col, bool &on) {      // row `col` of the place's queries
        const int tok = x.hg % p.parts * p.per + col / p.group;
        on = col < cols && tok < p.n;
        return p.q + ((((int64_t)x.b * p.n + tok) * p.nkv + head_of(x)) * p.group + col % p.group) * HD;
    };
    {   // on their way while the first copies are asked for
        bool on;
        const uint16_t *qr = query(at, lane / (HD / 64), on) + lane % (HD / 64) * 64;
        if (on) asm volatile("prefetch.global.L1 [%0];" ::"l"(qr));
    }
    int halves = 2 * n, ld_place = 0;                     // halves of steps (K, then V) still to be asked for; the place of the next one
    const int64_t row = (int64_t)p.nkv * HD;
    const int ld_c = lane % CH, ld_r = lane / CH;         // this lane's piece of a row, and which of the rows that one instruction copies
    int64_t ld_at = 0;                                    // where they are, for the step being loaded
    auto load_next = [&]() {
        if (halves > 0) {
            constexpr int RPI = 32 / CH;                  // rows per instruction: 2 or 4
            const int j0 = ld.step * keys + sub * GK;
            if (!(halves & 1)) ld_at = ((int64_t)ld.b * p.rows + j0 + ld_r) * row + head_of(ld) * HD + ld_c * 16;
            const uint8_t *src = ((halves & 1) ? p.v : p.k) + ld_at;
            const uint32_t dst = ring + ld_place * KB + ld_r * HD;
            if (j0 + GK <= ld.len) {
#pragma unroll
                for (int i = 0; i < GK / RPI; i++, src += RPI * row)
                    cp_async16(dst + i * RPI * HD + ((ld_c ^ ((i * RPI + ld_r) & 7)) << 4), src, true);
            } else {                                      // (rows behind the last are not read: zeros in their place)
#pragma unroll
                for (int i = 0; i < GK / RPI; i++, src += RPI * row) {
                    const bool ok = j0 + i * RPI + ld_r < ld.len;
                    cp_async16(dst + i * RPI * HD + ((ld_c ^ ((i * RPI + ld_r) & 7)) << 4), ok ? src : p.k, ok);
                }
            }
            halves--;
            ld_place = ld_place + 1 == RING ? 0 : ld_place + 1;
            if (halves > 0 && !(halves & 1)) gqa_advance(p.steps, ld);
        }
        cp_async_commit();
    };
    // the two scales of this warp's keys at a place (any value where it has no key there), not joined: that would wait for them
    auto scales = [&](const GqaPlace &x, uint32_t &ks, uint32_t &vs) {
        const int j0 = x.step * keys + sub * GK;
        ks = vs = 127;
        if (j0 >= x.len) return;
        const int64_t i = ((int64_t)x.b * (p.rows >> p.lb) + (j0 >> p.lb)) * p.nkv + head_of(x);
        ks = p.ks[i];
        vs = p.vs[i];
    };
    uint32_t ks, vs;
    scales(at, ks, vs);
#pragma unroll
    for (int i = 0; i < RING - 1; i++) load_next();
    if (!WHOLE && warp == 0) gqa_note(p.steps, list, lane);
    uint32_t bq[QS ? 1 : HD / 16][NB][2];                 // the query rows, as the score MMAs' second operand
    float acc[HD / 16][NB][4];                            // value columns 16 i + 2 lg (+ 1) of query rows 8 nb + 2 lt, + 1
    float m[NB][2], l[NB][2], unit[NB][2];                // unit: what a score MMA's result is multiplied by, besides the key scale
    int limit[NB][2];                                     // rows that the query row sees
    bool fresh = true;
    int place = 0;                                        // of the half in use
    for (int s = 0; s < n; s++) {
        if (fresh) {
            const int part = at.hg % p.parts;
#pragma unroll
            for (int nb = 0; nb < NB; nb++) {
                // this lane's dims of query row 8 nb + lg: 16 i + 4 lt .. + 3
                bool on;
                const uint16_t *qr = query(at, nb * 8 + lg, on) + 4 * lt;
                uint2 u[HD / 16];
                __nv_bfloat162 top = __float2bfloat162_rn(0.f);
#pragma unroll
                for (int i = 0; i < HD / 16; i++) u[i] = on ? *reinterpret_cast<const uint2 *>(qr + i * 16) : make_uint2(0u, 0u);
#pragma unroll
                for (int i = 0; i < HD / 16; i++) {
                    top = __hmax2(top, __habs2(*reinterpret_cast<const __nv_bfloat162 *>(&u[i].x)));
                    top = __hmax2(top, __habs2(*reinterpret_cast<const __nv_bfloat162 *>(&u[i].y)));
                }
                float big = fmaxf(__low2float(top), __high2float(top));
                big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
                big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
                const int e = min(max((int)(__float_as_uint(big) >> 23) - 127, -100), 120);
                const float down = kv8_two(-e);
#pragma unroll
                for (int i = 0; i < HD / 16; i++) {
                    const uint32_t q0 = pack_f16x2(__uint_as_float(u[i].x << 16) * down, __uint_as_float(u[i].x & 0xFFFF0000u) * down);
                    const uint32_t q1 = pack_f16x2(__uint_as_float(u[i].y << 16) * down, __uint_as_float(u[i].y & 0xFFFF0000u) * down);
                    if constexpr (QS) reinterpret_cast<uint2 *>(qs + i * 32)[nb] = make_uint2(q0, q1);      // (read by this lane alone)
                    else { bq[i][nb][0] = q0; bq[i][nb][1] = q1; }
                    acc[i][nb][0] = acc[i][nb][1] = acc[i][nb][2] = acc[i][nb][3] = 0.f;
                }
                // the two rows whose scores this lane gets are those of lanes with lg = 2 lt, 2 lt + 1
                const float up = kv8_two(e) * p.scale_log2;
#pragma unroll
                for (int x = 0; x < 2; x++) {
                    unit[nb][x] = __shfl_sync(0xffffffffu, up, (2 * lt + x) * 4);
                    limit[nb][x] = at.len - (p.n - 1 - (part * p.per + (nb * 8 + 2 * lt + x) / p.group));
                    l[nb][x] = 0.f;
                }
            }
        }
        cp_async_wait<RING - 2>();
        __syncwarp();                                     // every lane's copies of these keys have landed; the place before has been read
        load_next();
        GqaPlace next = at;                               // its scales are asked for a step ahead
        uint32_t ks_next = 0, vs_next = 0;
        if (s + 1 < n) {
            gqa_advance(p.steps, next);
            scales(next, ks_next, vs_next);
        }
        const uint32_t tK = ring + place * KB;
        place = place + 1 == RING ? 0 : place + 1;
        const uint32_t key = lane * HD, x7 = lane & 7;    // ldmatrix: a lane's address is key `lane`'s
        const float kscale = kv8_scale(ks), vscale = kv8_scale(vs);
        float c[2][NB][4];                                // scores of keys 16 h + lg, + 8
#pragma unroll
        for (int i = 0; i < HD / 16; i++) {
            uint32_t r[4], a[2][4];
            ldmatrix_x4(r[0], r[1], r[2], r[3], tK + key + ((i ^ x7) << 4));
            uint32_t q[NB][2];
            if constexpr (QS) {
                const uint4 v = qs[i * 32];
                q[0][0] = v.x; q[0][1] = v.y; q[NB - 1][0] = v.z; q[NB - 1][1] = v.w;
            } else {
#pragma unroll
                for (int nb = 0; nb < NB; nb++) { q[nb][0] = bq[i][nb][0]; q[nb][1] = bq[i][nb][1]; }
            }
#pragma unroll
            for (int h = 0; h < 2; h++) {
                kv8_decode4<I8>(r[2 * h], a[h][0], a[h][2]);
                kv8_decode4<I8>(r[2 * h + 1], a[h][1], a[h][3]);
#pragma unroll
                for (int nb = 0; nb < NB; nb++) {
                    if (i == 0) mma_f16_16816_zero(c[h][nb], a[h], q[nb][0], q[nb][1]);
                    else mma_f16_16816(c[h][nb], a[h], q[nb][0], q[nb][1]);
                }
            }
        }
        const int j0 = at.step * keys + sub * GK + lg;    // this lane's keys: j0, + 8, + 16, + 24
        uint32_t b[2][NB][2];                             // the probabilities, as the value MMAs' second operand
#pragma unroll
        for (int nb = 0; nb < NB; nb++) {
            float t[4][2];
#pragma unroll
            for (int x = 0; x < 2; x++)
#pragma unroll
                for (int k = 0; k < 4; k++)               // (one factor after the other: their product alone may be out of range)
                    t[k][x] = j0 + 8 * k < limit[nb][x] ? c[k >> 1][nb][(k & 1) * 2 + x] * unit[nb][x] * kscale : -INFINITY;
            float big[2];
#pragma unroll
            for (int x = 0; x < 2; x++) big[x] = fmaxf(fmaxf(t[0][x], t[1][x]), fmaxf(t[2][x], t[3][x]));
            if (fresh || __any_sync(0xffffffffu, big[0] > m[nb][0] + GQ_LAZY || big[1] > m[nb][1] + GQ_LAZY)) {
#pragma unroll
                for (int x = 0; x < 2; x++)
#pragma unroll
                    for (int o = 4; o < 32; o <<= 1) big[x] = fmaxf(big[x], __shfl_xor_sync(0xffffffffu, big[x], o));
                if (fresh) {
                    // A row that sees none of these keys sees none behind them: any exponent will do. And where all that it sees is NaN: its sum
                    // is NaN, which the merge keeps, but a NaN for exponent would lose against any other, or -infinity.
                    m[nb][0] = big[0] > -INFINITY ? big[0] : 0.f;
                    m[nb][1] = big[1] > -INFINITY ? big[1] : 0.f;
                } else {
                    float f[2];
#pragma unroll
                    for (int x = 0; x < 2; x++) {
                        const float to = fmaxf(m[nb][x], big[x]);
                        f[x] = exp2f(m[nb][x] - to);
                        m[nb][x] = to;
                        l[nb][x] *= f[x];
                    }
#pragma unroll
                    for (int i = 0; i < HD / 16; i++) { acc[i][nb][0] *= f[0]; acc[i][nb][1] *= f[1]; acc[i][nb][2] *= f[0]; acc[i][nb][3] *= f[1]; }
                }
            }
#pragma unroll
            for (int x = 0; x < 2; x++) {
#pragma unroll
                for (int k = 0; k < 4; k++) t[k][x] = exp2f(t[k][x] - m[nb][x]);
                l[nb][x] += (t[0][x] + t[1][x]) + (t[2][x] + t[3][x]);
            }
#pragma unroll
            for (int k = 0; k < 4; k++) {                 // [8 keys][8 rows] each -> [8 rows][8 keys]
                uint32_t &w = b[k >> 1][nb][k & 1];
                w = pack_f16x2(t[k][0], t[k][1]);
                asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %0;" : "+r"(w));
            }
        }
        cp_async_wait<RING - 2>();                        // the same for the values
        __syncwarp();
        load_next();
        const uint32_t tV = ring + place * KB;
        place = place + 1 == RING ? 0 : place + 1;
#pragma unroll
        for (int i = 0; i < HD / 16; i++) {
            uint32_t r[4], a[2][4];
            ldmatrix_x4_trans(r[0], r[1], r[2], r[3], tV + key + ((i ^ x7) << 4));
            float d[NB][4];
#pragma unroll
            for (int h = 0; h < 2; h++) {
                kv8_decode4_even_odd<I8>(r[2 * h], a[h][0], a[h][1]);
                kv8_decode4_even_odd<I8>(r[2 * h + 1], a[h][2], a[h][3]);
#pragma unroll
                for (int nb = 0; nb < NB; nb++) {
                    if (h == 0) mma_f16_16816_zero(d[nb], a[h], b[h][nb][0], b[h][nb][1]);
                    else mma_f16_16816(d[nb], a[h], b[h][nb][0], b[h][nb][1]);
                }
            }
#pragma unroll
            for (int nb = 0; nb < NB; nb++)
#pragma unroll
                for (int x = 0; x < 4; x++) acc[i][nb][x] = fmaf(d[nb][x], vscale, acc[i][nb][x]);
        }
        fresh = at.step + 1 == at.steps;
        if (fresh || s + 1 == n) {                        // the end of what this block has of the sequence's head group: its record
            float *rec;
            if constexpr (WHOLE) rec = reinterpret_cast<float *>(smem + warp * (RING + (QS ? 1 : 0)) * KB);
            else rec = p.rec + (((int64_t)at.b * p.steps.groups + at.hg + blockIdx.x) * GW + warp) * kv8_record(cols, HD);
            static_assert(kv8_record(8 * NB, HD) * 4 <= (RING + (QS ? 1 : 0)) * KB, "a record in the place of the ring");
            if (WHOLE) __syncwarp();                      // every lane has read its last values
#pragma unroll
            for (int nb = 0; nb < NB; nb++)
#pragma unroll
                for (int x = 0; x < 2; x++) {
                    float sum = l[nb][x];
#pragma unroll
                    for (int o = 4; o < 32; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                    const int col = nb * 8 + 2 * lt + x;
                    if (col >= cols) continue;
                    if (WHOLE && p.hb == GW) {            // the warp has all of the rows' keys
                        const int tok = at.hg % p.parts * p.per + col / p.group;
                        if (tok >= p.n) continue;
                        const float inv = sum != 0.f ? 1.f / sum : 0.f;
                        uint16_t *dst = p.out + (((int64_t)at.b * p.n + tok) * p.nh() + head_of(at) * p.group + col % p.group) * HD + 2 * lg;
#pragma unroll
                        for (int i = 0; i < HD / 16; i++)
                            *reinterpret_cast<uint32_t *>(dst + i * 16) = pack_bf16x2(acc[i][nb][x] * inv, acc[i][nb][2 + x] * inv);
                        continue;
                    }
                    float *o = rec + col * HD;
                    if (lg == 0) *reinterpret_cast<float2 *>(rec + cols * HD + col * 2) = make_float2(sum != 0.f ? m[nb][x] : -INFINITY, sum);
#pragma unroll
                    for (int i = 0; i < HD / 16; i += 2)
                        *reinterpret_cast<float4 *>(o + i * 16 + 4 * lg) = make_float4(acc[i][nb][x], acc[i][nb][2 + x], acc[i + 1][nb][x], acc[i + 1][nb][2 + x]);
                }
        }
        at = next;
        ks = ks_next; vs = vs_next;
    }
    cp_async_wait<0>();
    if constexpr (WHOLE) {
        if (p.hb == GW && n > 0) return;
        __syncthreads();
        // the warps take the query rows of the block's KV heads in turn; no rows in the cache: zeros
        const int b = (int)blockIdx.x / p.steps.groups, hg = (int)blockIdx.x % p.steps.groups;
#pragma unroll 1
        for (int row = warp; row < p.hb * cols; row += GW) {
            const int w = row / cols, col = row % cols, tok = hg % p.parts * p.per + col / p.group;
            if (tok >= p.n) continue;
            Kv8Sum s[HD / 128];
            for (int k = w; k < GW && n > 0; k += p.hb) {
                const float *rec = reinterpret_cast<const float *>(smem + k * (RING + (QS ? 1 : 0)) * KB);
                const float2 ml = *reinterpret_cast<const float2 *>(rec + cols * HD + col * 2);
                if (ml.x == -INFINITY) continue;
#pragma unroll
                for (int j = 0; j < HD / 128; j++) {
                    if (ml.x > s[j].M) s[j].raise(ml.x);
                    s[j].add(exp2f(ml.x - s[j].M), ml.y, *reinterpret_cast<const float4 *>(rec + col * HD + j * 128 + lane * 4));
                }
            }
            uint16_t *dst = p.out + (((int64_t)b * p.n + tok) * p.nh() + (hg / p.parts * p.hb + w) * p.group + col % p.group) * HD;
#pragma unroll
            for (int j = 0; j < HD / 128; j++) s[j].write(dst, j * 128 + lane * 4);
        }
    }
}

// The records of one query row (token x head of sequence b): cnt of them, {m, l} and o of the i-th at ml(i) and o(i).
struct Kv8Records {
    const float *base;
    int64_t rsz;
    int cnt, ks, hb, ml, o;
    __device__ __forceinline__ Kv8Records(const Kv8DecodeParams &p, int hd, int b, int tok, int h) {
        const int kvh = h / p.group, cols = p.per * p.group, col = tok % p.per * p.group + h % p.group;
        const int2 meta = p.steps.meta[b * p.steps.groups + (kvh / p.hb) * p.parts + tok / p.per];
        hb = p.hb; ks = GW / hb; cnt = meta.y * ks;
        rsz = kv8_record(cols, hd);
        ml = cols * hd + col * 2; o = col * hd;
        base = p.rec + ((int64_t)meta.x * GW + kvh % hb) * rsz;
    }
    // slot first + i / ks, warp (i % ks) * hb + kvh % hb
    __device__ __forceinline__ const float *at(int i) const { return base + (ks == 1 ? (int64_t)i * GW : (int64_t)(i / ks) * GW + (i % ks) * hb) * rsz; }
};
// The records first, first + stride, .., eight records' loads at once; the running maximum as the scores'.
__device__ __forceinline__ void kv8_add_records(Kv8Sum &s, const Kv8Records &r, int column, int first, int stride) {
    for (int i0 = first; i0 < r.cnt; i0 += 8 * stride) {
        float2 ml[8];
        float4 v[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float *at = r.at(min(i0 + j * stride, r.cnt - 1));
            ml[j] = *reinterpret_cast<const float2 *>(at + r.ml);
            v[j] = *reinterpret_cast<const float4 *>(at + r.o + column);
            if (i0 + j * stride >= r.cnt) ml[j].x = -INFINITY;
        }
        float to = s.M;
#pragma unroll
        for (int j = 0; j < 8; j++) to = fmaxf(to, ml[j].x);
        if (to == -INFINITY) continue;
        s.raise(to);
#pragma unroll
        for (int j = 0; j < 8; j++) s.add(exp2f(ml[j].x - to), ml[j].y, v[j]);
    }
}

// Few records a row: 256 threads have the rows of a sequence one after another, four columns each. grid (parts of n * nh rows, sequence)
template <int HD>
__global__ void __launch_bounds__(256) kv8_merge_few_kernel(const Kv8DecodeParams p) {
    const int row = blockIdx.x * (1024 / HD) + threadIdx.x / (HD / 4), column = threadIdx.x % (HD / 4) * 4, b = blockIdx.y;
    cwk_pdl_launch();
    cwk_pdl_wait();
    if (row >= p.n * p.nh()) return;
    Kv8Sum s;
    kv8_add_records(s, Kv8Records(p, HD, b, row / p.nh(), row % p.nh()), column, 0, 1);
    s.write(p.out + ((int64_t)b * p.n * p.nh() + row) * HD, column);
}
// Many: 64 columns of a row to a block, its records dealt out to GROUPS groups of 16 threads: what counts is that all are asked for at
// once (one sequence of 4096 rows has 128 records a row). grid (row, sequence, HD / 64)
template <int HD, int GROUPS>
__global__ void __launch_bounds__(16 * GROUPS) kv8_merge_kernel(const Kv8DecodeParams p) {
    __shared__ float s_m[GROUPS], s_l[GROUPS];
    __shared__ float4 s_o[GROUPS][16];
    const int row = blockIdx.x, b = blockIdx.y, g = threadIdx.x / 16, t = threadIdx.x % 16, column = blockIdx.z * 64 + t * 4;
    cwk_pdl_launch();
    cwk_pdl_wait();
    Kv8Sum s;
    kv8_add_records(s, Kv8Records(p, HD, b, row / p.nh(), row % p.nh()), column, g, GROUPS);
    if (t == 0) { s_m[g] = s.M; s_l[g] = s.den; }
    s_o[g][t] = s.o;
    __syncthreads();
    if (g > 0) return;
    Kv8Sum all;
#pragma unroll
    for (int j = 0; j < GROUPS; j++) all.M = fmaxf(all.M, s_m[j]);
#pragma unroll
    for (int j = 0; j < GROUPS; j++) all.add(s_m[j] == -INFINITY ? 0.f : exp2f(s_m[j] - all.M), s_l[j], s_o[j][t]);
    all.write(p.out + ((int64_t)b * p.n * p.nh() + row) * HD, column);
}

template <int HD, int NB, bool WHOLE>
int launch(cwk_ctx *ctx, const Kv8DecodeParams &p, int type, int blocks) {
    constexpr int SMEM = GW * (KV8_RING<HD, NB> + (KV8_Q_SHARED<HD, NB> ? 1 : 0)) * GK * HD;      // 96 KB
    const bool i8 = type == CWK_KV8_INT8;
    auto kern = i8 ? kv8_decode_kernel<HD, NB, true, WHOLE> : kv8_decode_kernel<HD, NB, false, WHOLE>;
    static bool attr_set[2][16] = {};
    if (!attr_set[i8][ctx->device & 15]) {
        CWK_CUDA(ctx, cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM));
        attr_set[i8][ctx->device & 15] = true;
    }
    {
        CwkKernelTimer timer(ctx);
        CWK_CUDA(ctx, cwk_launch_early(kern, dim3(blocks), dim3(32 * GW), SMEM, ctx->stream, p));
        ctx->launches++;
    }
    if (WHOLE) return CWK_OK;
    // Records per query row; the threads that a group of 16 for every 64 columns of a row makes. Groups as long as there are records for them
    // and the SMs are not filled more than once (37 tokens of 32 heads after 300 rows, 222 blocks, 12 records a row, 1184 rows: 26.8 us with eight
    // groups a row, 15.2 with one).
    const int64_t each = (int64_t)blocks * (GW / p.hb) / ((int64_t)p.steps.B * p.steps.groups), rows = p.n * p.nh(), threads = rows * p.steps.B * (HD / 4);
    const int64_t room = std::min<int64_t>((int64_t)ctx->sm_count * 1536 / threads, each / 2);
    if (each > 8 && room >= 4) {
        const int groups = room >= 16 ? 16 : room >= 8 ? 8 : 4;
        CWK_CUDA(ctx, cwk_launch_early(groups == 16 ? kv8_merge_kernel<HD, 16> : groups == 8 ? kv8_merge_kernel<HD, 8> : kv8_merge_kernel<HD, 4>,
                                       dim3((unsigned)rows, p.steps.B, HD / 64), dim3(16 * groups), 0, ctx->stream, p));
    } else CWK_CUDA(ctx, cwk_launch_early(kv8_merge_few_kernel<HD>, dim3((unsigned)((rows + 1024 / HD - 1) / (1024 / HD)), p.steps.B), dim3(256), 0, ctx->stream, p));
    ctx->launches++;
    return CWK_OK;
}

}  // namespace

namespace {

// The shape of a pass over `B` sequences of up to `len` rows, and what it takes.
//
// Whole: a block for each head group of each sequence, no records, no merge and its launch; of one KV head, four or two, whichever gives the
// sooner end. Otherwise equal shares of all steps. By a cost of each side, in us a call replayed, fitted to 1 to 140 sequences of 20 to 4096
// rows, one and four tokens (and in shares to 580 chunks of 4 to 300 tokens after 0 to 12000 rows): steps one after another, or the bytes
// at 7 TB/s (shares 6.5) where there are many blocks. The host knows the longest length only. Shares even out what is shorter, whole blocks do not:
// so the shares count with five sixths of the rows (half ragged), and whole blocks are for lengths whose steps alone take no more than twice what
// shares of next to nothing take (one long sequence among short ones). A launch less is worth a microsecond to whoever launches.
// Whole / shares, 16 heads, 4 KV heads of 256: one sequence of 100 rows 4.9 / 7.4, of 600 10.6 / 7.5; 16 of 128 5.1 / 8.9, of 500 9.8 / 12.0, of 2000
// 27 / 21; 64 of 300 12.0 / 18.8, of 1200 28.7 / 36.7 (ragged from half to that 26 / 30; one of them and 63 of 100 rows 19 / 14), of 4096 80 / 92 (73 / 71); 80 of 1200, two more blocks
// than two for each SM, 51 / 44. Four tokens: 16 of 500 15.6 / 15.0, 64 of 1200 38 / 54 (37 / 46).
struct Kv8Shape {
    int hb, per, parts, keys, cols, blocks;
    int64_t groups;
    int64_t places;       // for records, a block's warps each, if the steps go out in shares
    bool whole;
    double us;
    Kv8Shape(int sm_count, int B, int64_t len, int n, int nh, int nkv, int hd, int max_blocks) {
        const int group = nh / nkv;
        per = std::min(n, std::max(1, 16 / group));
        parts = (n + per - 1) / per;
        cols = per * group;
        const bool wide = hd == 256, two = cols > 8;
        const int64_t sms = sm_count, slots = 2 * sms;
        const auto deal = [&](int heads) {
            hb = heads;
            keys = GK * (GW / hb);
            groups = (int64_t)(nkv / hb) * parts;
            return (len + keys - 1) / keys;
        };
        double one = 1e30, alone = 0;
        int best = 1;
        for (int h = 4; h >= 1; h /= 2) {
            if (nkv % h != 0) continue;
            const int64_t each = deal(h), all = B * groups, rounds = (all + slots - 1) / slots;
            if (all >= 1 << 30) continue;
            const auto step = [&](int64_t blocks) {       // of a block with so many beside it
                const double chain = (two ? (wide ? 2.05 : 1.2) : (wide ? 1.42 : 1.02)) * (blocks > sms ? 1.4 : 1.0);
                return std::max(chain, (double)(blocks * 2 * GW * GK * hd / parts) / 7e6);
            };
            const double ends = (two ? (wide ? 5.7 : 4.8) : (wide ? 3.9 : 3.2)) + (h < GW ? 0.3 + 0.3 * h * cols / GW : 0.0);
            const double x = each * ((rounds - 1) * step(slots) + step(all - (rounds - 1) * slots)) + 4.0 * (rounds - 1) + ends;
            if (x < one) { one = x; alone = each * step(1) + ends; best = h; }
        }
        const int64_t each = deal(nkv % 4 == 0 ? 4 : nkv % 2 == 0 ? 2 : 1), steps = B * groups * each;
        places = B * groups + slots;
        // as many blocks as there can be steps, at most two per SM
        blocks = (int)std::min<int64_t>(std::max<int64_t>(1, steps), max_blocks > 0 ? std::min<int64_t>(max_blocks, slots) : slots);
        const double turns = (double)((steps + blocks - 1) / blocks), records = (double)blocks * GW * cols * hd * 4e-6;
        const double stream = std::max(turns * (two ? (wide ? 3.1 : 1.85) : (wide ? 0.94 : 0.82)), (double)B * len * nkv * hd * 2 / 6.5e6);
        const double shares = (wide ? 6.8 : 6.0) + (B > 1 ? 1.5 : 0.0) + 0.65 * records;
        whole = max_blocks == 0 && one <= shares + stream * (B > 1 ? 5.0 / 6 : 1.0) + 1.0 && (B == 1 || alone <= 2 * shares);
        if (whole) {
            deal(best);
            blocks = (int)(B * groups);
        }
        us = whole ? one : shares + stream;
    }
};

// Which way a chunk goes. The streams read the codes once for every 16 query rows, every row over all keys; the tensor-core kernel has 128
// query tokens of a head in a tile, but wants the cache widened and three or four launches. Its cost fitted to the same 580 chunks ((16, 4), (8, 1),
// (8, 8), (32, 2), (24, 3) and (16, 2) heads). Streams / tensor cores, 16 heads, 4 KV heads of 256: 4 tokens after 2000 rows 11 / 37, 37 after
// 2500 26 / 38, 128 after 2000 45 / 41, 64 after 12000 71 / 65; of 128: 64 after 2000 17 / 30, 200 after 12000 115 / 55.
bool kv8_streams_sooner(int sm_count, int64_t pos, int n, int nh, int nkv, int hd) {
    if (nh / nkv > 16) return false;
    const int64_t T = pos + n;
    const bool wide = hd == 256;
    // items of 128 tokens x one head, 64 keys a tile; where the longest block has many tiles above an equal share they are dealt out in shares and joined
    const int64_t items = (int64_t)((n + 127) / 128) * nh;
    const auto tiles = [&](int64_t last) { return (last + 63) / 64; };
    int64_t all = 0;
    for (int64_t q = 0; q < n; q += 128) all += tiles(pos + std::min<int64_t>(q + 128, n)) * nh;
    const int64_t share = (all + sm_count - 1) / sm_count, idle = ((items + sm_count - 1) / sm_count) * sm_count - items;
    const int64_t dealt = std::max(tiles(T), share + idle * tiles(pos + std::min(128, n)) / sm_count);
    const bool shared = dealt > share + 28;
    const double tensor = (wide ? 15.5 : 14.3) + (double)(shared ? share : dealt) * (wide ? 0.64 : 0.54) + (shared ? (wide ? 17.4 : 14.0) : 0.0) + (double)T * nkv * hd * 6 * 0.256e-6;
    return Kv8Shape(sm_count, 1, T, n, nh, nkv, hd, 0).us < tensor;
}

}  // namespace

int cwk_kv8_streams(cwk_ctx *ctx, const void *q, const cwk_kv8 &c, const int32_t *kv_len, int max_kv_len, int B, int n, int nh, float scale,
                    void *out, int max_blocks) {
    Kv8DecodeParams p{};
    p.q = (const uint16_t *)q; p.k = (const uint8_t *)c.k; p.v = (const uint8_t *)c.v; p.ks = c.k_scale; p.vs = c.v_scale; p.rows = c.rows;
    const Kv8Shape shape(ctx->sm_count, B, max_kv_len, n, nh, c.nkv, c.hd, max_blocks);
    const int blocks = shape.blocks;
    p.n = n; p.nkv = c.nkv; p.parts = shape.parts;
    p.group = nh / c.nkv; p.hb = shape.hb; p.per = shape.per;
    p.lb = c.block == 32 ? 5 : c.block == 64 ? 6 : 7;
    p.scale_log2 = scale * 1.4426950408889634f;
    if (shape.groups > 0x7FFFFFFF) return cwk_fail(ctx, CWK_ERR_ARGUMENT, "gqa_decode_kv8: too many query tokens");
    p.out = (uint16_t *)out;
    p.steps = GqaSteps{kv_len, B, (int)shape.groups, shape.keys, kv_len ? (int)c.rows : max_kv_len, nullptr};
    const bool two = shape.cols > 8;
    // Whole blocks have no records. Their room is there all the same, so that it grows with the sequences and the tokens alone: a context that
    // has done the largest of its steps has it for every smaller one, captured or not.
    const size_t rec_bytes = (size_t)shape.places * GW * kv8_record(shape.cols, c.hd) * sizeof(float);
    const int s = cwk_reserve_scratch(ctx, rec_bytes + (size_t)shape.places * sizeof(int2));
    if (s != CWK_OK) return s;
    if (shape.whole) {
        if (c.hd == 256) return two ? launch<256, 2, true>(ctx, p, c.type, blocks) : launch<256, 1, true>(ctx, p, c.type, blocks);
        return two ? launch<128, 2, true>(ctx, p, c.type, blocks) : launch<128, 1, true>(ctx, p, c.type, blocks);
    }
    p.rec = ctx->scratch;
    p.steps.meta = (int2 *)((uint8_t *)ctx->scratch + rec_bytes);
    if (c.hd == 256) return two ? launch<256, 2, false>(ctx, p, c.type, blocks) : launch<256, 1, false>(ctx, p, c.type, blocks);
    return two ? launch<128, 2, false>(ctx, p, c.type, blocks) : launch<128, 1, false>(ctx, p, c.type, blocks);
}

// mla_prefill_attn.cu
int cwk_gqa_prefill_tc(cwk_ctx *ctx, const void *Q, const void *K, const void *V, int64_t pos, int n, int nh, int nkv, int hd,
                       float scale, void *out, int *flags, int spread);

extern "C" {

int cwk_gqa_decode_kv8(cwk_ctx *ctx, const void *q, const cwk_kv8 *c, const int32_t *kv_len, int max_kv_len, int B, int n, int nh, float scale,
                       void *out, int n_splits) {
    int s = cwk_kv8_check(ctx, c, "gqa_decode_kv8");
    if (s != CWK_OK) return s;
    if (!ctx || !q || !kv_len || !out) return cwk_fail(ctx, CWK_ERR_ARGUMENT, "gqa_decode_kv8: null argument");
    if (B <= 0 || B > 65535 || B > c->slots || n <= 0 || nh <= 0 || nh % c->nkv != 0 || max_kv_len < 0 || max_kv_len > c->rows)
        return cwk_fail(ctx, CWK_ERR_ARGUMENT, "gqa_decode_kv8: bad dimensions");
    if (nh / c->nkv > 16) return cwk_fail(ctx, CWK_ERR_UNSUPPORTED, "gqa_decode_kv8: group %d not built (up to 16)", nh / c->nkv);
    if ((((uintptr_t)q | (uintptr_t)out) & 15) != 0) return cwk_fail(ctx, CWK_ERR_ARGUMENT, "gqa_decode_kv8: pointers must be 16-byte aligned");
    CWK_CUDA(ctx, cudaSetDevice(ctx->device));
    return cwk_kv8_streams(ctx, q, *c, kv_len, max_kv_len, B, n, nh, scale, out,
                           n_splits > 0 ? (int)std::min<int64_t>((int64_t)n_splits * B * c->nkv, 1 << 20) : 0);
}

int cwk_gqa_prefill_kv8(cwk_ctx *ctx, const void *Q, const cwk_kv8 *c, int slot, int64_t pos, int n, int nh, float scale, void *out) {
    int s = cwk_kv8_check(ctx, c, "gqa_prefill_kv8");
    if (s != CWK_OK) return s;
    if (!ctx || !Q || !out) return cwk_fail(ctx, CWK_ERR_ARGUMENT, "gqa_prefill_kv8: null argument");
    if (slot < 0 || slot >= c->slots || n <= 0 || pos < 0 || pos > c->rows - n || nh <= 0 || nh % c->nkv != 0)
        return cwk_fail(ctx, CWK_ERR_ARGUMENT, "gqa_prefill_kv8: bad dimensions");
    if ((((uintptr_t)Q | (uintptr_t)out) & 15) != 0) return cwk_fail(ctx, CWK_ERR_ARGUMENT, "gqa_prefill_kv8: pointers must be 16-byte aligned");
    CWK_CUDA(ctx, cudaSetDevice(ctx->device));
    cwk_kv8 at = *c;
    const int64_t T = pos + n, row = (int64_t)c->nkv * c->hd;
    at.k = (uint8_t *)c->k + slot * c->rows * row; at.v = (uint8_t *)c->v + slot * c->rows * row;
    at.k_scale = c->k_scale + slot * (c->rows / c->block) * c->nkv; at.v_scale = c->v_scale + slot * (c->rows / c->block) * c->nkv;
    if (kv8_streams_sooner(ctx->sm_count, pos, n, nh, c->nkv, c->hd)) return cwk_kv8_streams(ctx, Q, at, nullptr, (int)T, 1, n, nh, scale, out, 0);
    // The slot's rows widened, exactly, behind the flags that the bf16 kernel keeps at the start of the workspace (a word per item and SM).
    // It grows by doubling, up to all of the slot's rows: a prompt's chunks ask for a little more every time (40 chunks of 512 in a
    // context that has no workspace yet 182 ms with a buffer of its own size for each, 5 to 8).
    const size_t flags = ((((size_t)((n + 127) / 128) * nh + ctx->sm_count + 3) * sizeof(int)) + 255) & ~(size_t)255, half = (size_t)T * row * 2;
    s = cwk_reserve_work_growing(ctx, flags + 2 * half, flags + (size_t)c->rows * row * 4);
    if (s != CWK_OK) return s;
    uint8_t *wk = (uint8_t *)ctx->work + flags;
    s = cwk_kv8_widen(ctx, at, 0, T, wk, wk + half);
    if (s != CWK_OK) return s;
    s = cwk_gqa_prefill_tc(ctx, Q, wk, wk + half, pos, n, nh, c->nkv, c->hd, scale, out, (int *)ctx->work, 2 * half <= (size_t)64 << 20);
    return s == CWK_ERR_UNSUPPORTED ? cwk_fail(ctx, s, "gqa_prefill_kv8: tensor maps are not available") : s;
}

}  // extern "C"
