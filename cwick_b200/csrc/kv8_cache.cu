// kv8_cache.cu -- writing and reading the GQA cache held in 8 bits (format: kv8.cuh), compiled without fast-math.
//
// Writing. A task is one block of rows of one KV head, K or V: its new rows are read once into registers (a warp has up to eight of them, a
// lane hd / 32 neighbouring values of each), the largest magnitude is found over the task, then the codes go out; an open block whose
// scale grows has the codes in front of the new rows rewritten. In front of the quantisation, for cwk_gqa_qk_prep_kv8, keys get
// their RMS norm and rotation (src/q35_model.c:112-122, :144-153, :459-477), and query heads the same on blocks of their own.
#include <algorithm>
#include <cmath>

#include "kv8.cuh"

namespace {

constexpr int KW_ROWS = 8;                     // rows per warp

enum { SRC_BF16 = 0, SRC_F32 = 1 };

struct Kv8WriteParams {
    const void *k, *v;                         // [B][n][nkv][hd]
    const int32_t *pos, *count;                // [B]; count NULL: n
    uint8_t *kc, *vc, *ks, *vs;
    int64_t rows;                              // per slot
    int B, n, nkv, lb;                         // block = 1 << lb
    int window;                                // blocks that n rows can touch
    // preparation
    const float *qg, *q_norm, *k_norm;
    uint16_t *q_out;
    int nh, rot;
    float eps;
    int64_t tasks;                             // K and V tasks; the blocks behind them have query rows
    int heads;                                 // query heads per warp
    double inv_freq[128];
};

// new rows of slot b: positions pos .. pos + the result - 1, all inside the slot
__device__ __forceinline__ int new_rows(const Kv8WriteParams &p, int b, int64_t &pos) {
    pos = p.pos[b];
    const int64_t c = p.count ? min(p.count[b], p.n) : p.n;
    return pos < 0 ? 0 : (int)max((int64_t)0, min(c, p.rows - pos));
}

template <int V, int SRC>
__device__ __forceinline__ void load_row(const void *src, int64_t row, int lane, float (&x)[V]) {
    if constexpr (SRC == SRC_BF16) {
        const uint16_t *s = (const uint16_t *)src + row * (32 * V) + lane * V;
        if constexpr (V == 8) {
            const uint4 u = *reinterpret_cast<const uint4 *>(s);
            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int i = 0; i < 4; i++) { x[2 * i] = __uint_as_float(w[i] << 16); x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u); }
        } else {
            const uint2 u = *reinterpret_cast<const uint2 *>(s);
            const uint32_t w[2] = {u.x, u.y};
#pragma unroll
            for (int i = 0; i < 2; i++) { x[2 * i] = __uint_as_float(w[i] << 16); x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u); }
        }
    } else {
        const float4 *s = reinterpret_cast<const float4 *>((const float *)src + row * (32 * V) + lane * V);
#pragma unroll
        for (int i = 0; i < V / 4; i++) {
            const float4 f = s[i];
            x[4 * i] = f.x; x[4 * i + 1] = f.y; x[4 * i + 2] = f.z; x[4 * i + 3] = f.w;
        }
    }
}

// finite magnitudes only: an infinity saturates and does not set the scale
__device__ __forceinline__ float magnitude(float x) {
    const float a = fabsf(x);
    return a <= 3.4028235e38f ? a : 0.f;       // (false for NaN too)
}

// cos and sin of a position's angles, for the rot / 2 pairs of a head, by a warp into its share of shared memory
__device__ __forceinline__ void angles(const Kv8WriteParams &p, int64_t pos, int lane, double2 *cs) {
    for (int i = lane; i < p.rot / 2; i += 32) {
        double c, s;
        sincos((double)pos * p.inv_freq[i], &s, &c);
        cs[i] = make_double2(c, s);
    }
    __syncwarp();
}

// A row's norm and rotation by a warp: y = x * rstd * (1 + w), the first `rot` values turned in pairs (i, i + rot / 2). Keys in T = double:
// a code hangs on which side of a border a value is, and this way it is the definition's; queries, which are rounded to bf16, in float.
template <int V, class T>
__device__ __forceinline__ void norm_rotate(const float (&x)[V], T rstd, const float (&w)[V], int rot, int lane, const double2 *cs, T (&y)[V]) {
#pragma unroll
    for (int i = 0; i < V; i++) y[i] = (T)x[i] * rstd * ((T)1 + (T)w[i]);
    if (rot == 0) return;
    const int d0 = lane * V, shift = rot / 2 / V;
    const bool lo = d0 < rot / 2, hi = !lo && d0 < rot;
    const int from = lo ? lane + shift : hi ? lane - shift : lane, pair = lo ? d0 : hi ? d0 - rot / 2 : 0;
#pragma unroll
    for (int i = 0; i < V; i++) {
        const T other = __shfl_sync(0xffffffffu, y[i], from);
        if (lo || hi) {
            const double2 t = cs[pair + i];
            const T c = (T)t.x, s = (T)t.y;
            y[i] = lo ? y[i] * c - other * s : y[i] * c + other * s;
        }
    }
}
template <int V, class T>
__device__ __forceinline__ T row_rstd(const float (&x)[V], float eps) {
    T sum = 0;
#pragma unroll
    for (int i = 0; i < V; i++) sum += (T)x[i] * (T)x[i];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    return (T)1 / sqrt(sum / (T)(32 * V) + (T)eps);
}

// double -> float for a second rounding to few bits: towards zero, the last bit set where anything was cut off, so that the
// second rounding sees on which side of a tie the value is
__device__ __forceinline__ float to_odd(double y) {
    const float f = __double2float_rz(y);
    return (double)f != y && y == y ? __uint_as_float(__float_as_uint(f) | 1u) : f;
}

template <int V, bool I8>
__device__ __forceinline__ void store_codes(uint8_t *dst, const float (&y)[V]) {
    uint32_t w[V / 4];
#pragma unroll
    for (int i = 0; i < V / 4; i++) {
        const float t[4] = {y[4 * i], y[4 * i + 1], y[4 * i + 2], y[4 * i + 3]};
        w[i] = kv8_encode4<I8>(t);
    }
    if constexpr (V == 8) *reinterpret_cast<uint2 *>(dst) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<uint32_t *>(dst) = w[0];
}

// A NaN among keys shows in the scores of the queries that see it. Among values it would reach queries that do not: their
// probability of it is zero, but the product is not. So values take zero in its place.
template <int V>
__device__ __forceinline__ void no_nan(float (&y)[V]) {
#pragma unroll
    for (int j = 0; j < V; j++) if (y[j] != y[j]) y[j] = 0.f;
}

// Rows r0 .. r0 + lead - 1 of an open block move from scale 2^was to 2^e, e > was.
template <int V, bool I8>
__device__ __forceinline__ void rescale(uint8_t *codes, int64_t ld, int lead, int was, int e, bool is_v, int warp, int warps, int lane) {
    const float f = was - e < -126 ? 0.f : kv8_two(was - e);
    for (int r = warp; r < lead; r += warps) {
        uint8_t *at = codes + r * ld + lane * V;
        float y[V];
#pragma unroll
        for (int i = 0; i < V / 4; i++) {
            uint32_t a, b;
            kv8_decode4<I8>(*reinterpret_cast<const uint32_t *>(at + 4 * i), a, b);
            const float2 u = __half22float2(*reinterpret_cast<const __half2 *>(&a)), v = __half22float2(*reinterpret_cast<const __half2 *>(&b));
            y[4 * i] = u.x * f; y[4 * i + 1] = u.y * f; y[4 * i + 2] = v.x * f; y[4 * i + 3] = v.y * f;
        }
        if (is_v) no_nan(y);
        store_codes<V, I8>(at, y);
    }
}

// V: values of a row per lane (head dim / 32). PREP: f32 rows, keys normed and rotated; blocks from p.tasks on have query rows.
template <int V, int SRC, bool I8, bool PREP>
__global__ void __launch_bounds__(512) kv8_write_kernel(const __grid_constant__ Kv8WriteParams p) {
    constexpr int HD = 32 * V;
    extern __shared__ double2 s_cs[];                      // PREP: [warp][rot / 2]
    __shared__ float s_max[16];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    cwk_pdl_launch();
    cwk_pdl_wait();
    double2 *cs = s_cs + warp * (p.rot / 2);
    if (PREP && blockIdx.x >= p.tasks) {
        // ---- query rows: a warp has `heads` heads of one token
        const int parts = (p.nh + p.heads - 1) / p.heads;
        const int64_t id = ((int64_t)blockIdx.x - p.tasks) * warps + warp, t = id / parts;
        if (t >= (int64_t)p.B * p.n) return;
        const int b = (int)(t / p.n), j = (int)(t % p.n), h0 = (int)(id % parts) * p.heads;
        int64_t pos;
        if (j >= new_rows(p, b, pos)) return;
        angles(p, pos + j, lane, cs);
        float w[V];
        load_row<V, SRC_F32>(p.q_norm, 0, lane, w);
        for (int h = h0; h < min(h0 + p.heads, p.nh); h++) {
            float x[V], y[V];
            load_row<V, SRC_F32>(p.qg, (t * p.nh + h) * 2, lane, x);      // rows [q | gate] of 2 * hd
            norm_rotate<V, float>(x, row_rstd<V, float>(x, p.eps), w, p.rot, lane, cs, y);
            uint32_t o[V / 2];
#pragma unroll
            for (int i = 0; i < V / 2; i++) o[i] = pack_bf16x2(y[2 * i], y[2 * i + 1]);
            uint16_t *dst = p.q_out + (t * p.nh + h) * HD + lane * V;
            if constexpr (V == 8) *reinterpret_cast<uint4 *>(dst) = make_uint4(o[0], o[1], o[2], o[3]);
            else *reinterpret_cast<uint2 *>(dst) = make_uint2(o[0], o[1]);
        }
        return;
    }
    int64_t id = blockIdx.x;
    const int head = (int)(id % p.nkv); id /= p.nkv;
    const int win = (int)(id % p.window); id /= p.window;
    const int b = (int)(id % p.B);
    const bool is_v = id / p.B != 0;                       // (all keys first: their tasks are the longer ones)
    int64_t pos;
    const int cnt = new_rows(p, b, pos);
    const int64_t blk = (pos >> p.lb) + win, r0 = blk << p.lb;
    const int64_t lo = max(r0, pos), hi = min(r0 + (1 << p.lb), pos + cnt);
    if (lo >= hi) return;
    const bool norm = PREP && !is_v;
    const void *src = is_v ? p.v : p.k;
    uint8_t *codes = (is_v ? p.vc : p.kc) + (((int64_t)b * p.rows + r0) * p.nkv + head) * HD;
    uint8_t *scale = (is_v ? p.vs : p.ks) + ((int64_t)b * (p.rows >> p.lb) + blk) * p.nkv + head;
    const int64_t ld = (int64_t)p.nkv * HD;
    const int lead = (int)(lo - r0);
    const int was_byte = lead > 0 ? (int)*scale : 0;
    float x[KW_ROWS][V], w[V];
    double rstd[KW_ROWS];
    float amax = 0.f;
    // row i of this warp: lo + warp + i * warps
#pragma unroll
    for (int i = 0; i < KW_ROWS; i++) {
        const int64_t r = lo + warp + i * warps;
        if (r < hi) load_row<V, SRC>(src, ((int64_t)b * p.n + (r - pos)) * p.nkv + head, lane, x[i]);
    }
    if (norm) load_row<V, SRC_F32>(p.k_norm, 0, lane, w);
#pragma unroll
    for (int i = 0; i < KW_ROWS; i++) {
        const int64_t r = lo + warp + i * warps;
        if (r >= hi) continue;                             // (the same for the whole warp)
        if (norm) {
            double y[V];
            rstd[i] = row_rstd<V, double>(x[i], p.eps);
            angles(p, r, lane, cs);
            norm_rotate<V, double>(x[i], rstd[i], w, p.rot, lane, cs, y);
#pragma unroll
            for (int j = 0; j < V; j++) amax = fmaxf(amax, magnitude(__double2float_ru(fabs(y[j]))));      // rounded up: never below the value
            __syncwarp();
        } else {
#pragma unroll
            for (int j = 0; j < V; j++) amax = fmaxf(amax, magnitude(x[i][j]));
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if (lane == 0) s_max[warp] = amax;
    __syncthreads();
    for (int i = 0; i < warps; i++) amax = fmaxf(amax, s_max[i]);
    int e = kv8_exponent(amax, I8);
    if (lead > 0) {
        const int was = min(max(was_byte - 127, KV8_LOW), kv8_high(I8));
        if (was >= e) e = was;
        else rescale<V, I8>(codes, ld, lead, was, e, is_v, warp, warps, lane);
    }
    if (threadIdx.x == 0) *scale = (uint8_t)(e + 127);
    const float f = kv8_two(-e);
#pragma unroll
    for (int i = 0; i < KW_ROWS; i++) {
        const int64_t r = lo + warp + i * warps;
        if (r >= hi) continue;
        float y[V];
        if (norm) {
            double z[V];
            angles(p, r, lane, cs);
            norm_rotate<V, double>(x[i], rstd[i], w, p.rot, lane, cs, z);
            __syncwarp();
            // INT8: one rounding of the double; E4M3: to odd, then to nearest
#pragma unroll
            for (int j = 0; j < V; j++) y[j] = I8 ? (float)rint(fmin(fmax(z[j] * (double)f, -127.0), 127.0)) : to_odd(z[j] * (double)f);
            // (a NaN goes through fmin and fmax as -127 or 127)
#pragma unroll
            for (int j = 0; j < V; j++) if (z[j] != z[j]) y[j] = NAN;
        } else {
#pragma unroll
            for (int j = 0; j < V; j++) y[j] = x[i][j] * f;
        }
        if (is_v) no_nan(y);
        store_codes<V, I8>(codes + (r - r0) * ld + lane * V, y);
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
constexpr int KR_THREADS = 256, KR_UNROLL = 4;

template <int HD, bool I8, bool F32>
__global__ void __launch_bounds__(KR_THREADS) kv8_read_kernel(const Kv8ReadParams p) {
    constexpr int PER = 8, CH = HD / PER;                  // values per thread and piece; pieces per head row
    cwk_pdl_launch();
    cwk_pdl_wait();
    const uint8_t *codes = blockIdx.y ? p.vc : p.kc, *scales = blockIdx.y ? p.vs : p.ks;
    uint8_t *out = (uint8_t *)(blockIdx.y ? p.v : p.k);
    const int64_t total = (int64_t)p.B * p.n * p.nkv * CH;
    const int64_t first = (int64_t)blockIdx.x * (KR_THREADS * KR_UNROLL) + threadIdx.x;
    uint2 c[KR_UNROLL];
    uint32_t s[KR_UNROLL];
    bool on[KR_UNROLL];
#pragma unroll
    for (int u = 0; u < KR_UNROLL; u++) {
        const int64_t id = first + u * KR_THREADS;
        on[u] = id < total;
        if (!on[u]) continue;
        const int piece = (int)(id % CH);
        const int64_t rh = id / CH;
        const int head = (int)(rh % p.nkv);
        const int64_t row = rh / p.nkv, j = row % p.n;
        const int b = (int)(row / p.n);
        const int64_t r = (p.pos ? (int64_t)p.pos[b] : p.row0) + j;
        on[u] = r >= 0 && r < p.rows && (!p.count || j < p.count[b]);
        if (!on[u]) continue;
        c[u] = *reinterpret_cast<const uint2 *>(codes + (((int64_t)b * p.rows + r) * p.nkv + head) * HD + piece * PER);
        s[u] = scales[((int64_t)b * (p.rows >> p.lb) + (r >> p.lb)) * p.nkv + head];
    }
#pragma unroll
    for (int u = 0; u < KR_UNROLL; u++) {
        if (!on[u]) continue;
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
        const int64_t id = first + u * KR_THREADS;
        if constexpr (F32) {
            float4 *o = reinterpret_cast<float4 *>(out + id * PER * 4);
            o[0] = make_float4(y[0].x, y[0].y, y[1].x, y[1].y);
            o[1] = make_float4(y[2].x, y[2].y, y[3].x, y[3].y);
        } else {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; i++) w[i] = pack_bf16x2(y[i].x, y[i].y);       // exact
            *reinterpret_cast<uint4 *>(out + id * PER * 2) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
}

int log2_of(int block) { return block == 32 ? 5 : block == 64 ? 6 : 7; }

int launch_read(cwk_ctx *ctx, const Kv8ReadParams &p, int hd, bool i8, bool f32) {
    const int64_t pieces = (int64_t)p.B * p.n * p.nkv * (hd / 8);
    const int64_t blocks = (pieces + KR_THREADS * KR_UNROLL - 1) / (KR_THREADS * KR_UNROLL);
    if (blocks > 0x7FFFFFFF) return cwk_fail(ctx, CWK_ERR_ARGUMENT, "kv8_load: too many rows in one call");
    void (*kern)(Kv8ReadParams);
    if (hd == 256) kern = i8 ? (f32 ? kv8_read_kernel<256, true, true> : kv8_read_kernel<256, true, false>)
                             : (f32 ? kv8_read_kernel<256, false, true> : kv8_read_kernel<256, false, false>);
    else kern = i8 ? (f32 ? kv8_read_kernel<128, true, true> : kv8_read_kernel<128, true, false>)
                   : (f32 ? kv8_read_kernel<128, false, true> : kv8_read_kernel<128, false, false>);
    CWK_CUDA(ctx, cwk_launch_early(kern, dim3((unsigned)blocks, 2), dim3(KR_THREADS), 0, ctx->stream, p));
    ctx->launches++;
    return CWK_OK;
}

template <int V, int SRC, bool PREP>
int launch_write(cwk_ctx *ctx, Kv8WriteParams &p, int type) {
    const int block = 1 << p.lb, warps = (std::min(block, p.n) + KW_ROWS - 1) / KW_ROWS;
    p.window = (int)(((int64_t)p.n + block - 2) / block + 1);
    p.tasks = (int64_t)2 * p.B * p.window * p.nkv;
    int64_t blocks = p.tasks;
    size_t smem = 0;
    if (PREP) {
        p.heads = p.n * (int64_t)p.B * p.nh <= 16 * 1024 ? 1 : 4;      // query heads that share a token's angles; few rows: one warp each
        blocks += ((int64_t)p.B * p.n * ((p.nh + p.heads - 1) / p.heads) + warps - 1) / warps;
        smem = (size_t)warps * (p.rot / 2) * sizeof(double2);
    }
    if (blocks > 0x7FFFFFFF) return cwk_fail(ctx, CWK_ERR_ARGUMENT, "kv8 write: too many rows in one call");
    auto kern = type == CWK_KV8_INT8 ? kv8_write_kernel<V, SRC, true, PREP> : kv8_write_kernel<V, SRC, false, PREP>;
    CWK_CUDA(ctx, cwk_launch_early(kern, dim3((unsigned)blocks), dim3(32 * warps), smem, ctx->stream, p));
    ctx->launches++;
    return CWK_OK;
}

void describe(Kv8WriteParams &p, const cwk_kv8 *c, const void *k, const void *v, const int32_t *pos, const int32_t *count, int B, int n) {
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
    Kv8WriteParams p{};
    describe(p, c, k, v, pos, count, B, n);
    CwkKernelTimer timer(ctx);
    if (c->hd == 256) return f32 ? launch_write<8, SRC_F32, false>(ctx, p, c->type) : launch_write<8, SRC_BF16, false>(ctx, p, c->type);
    return f32 ? launch_write<4, SRC_F32, false>(ctx, p, c->type) : launch_write<4, SRC_BF16, false>(ctx, p, c->type);
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
    Kv8WriteParams p{};
    describe(p, c, k, v, pos, count, B, n);
    p.qg = qg; p.q_norm = q_norm; p.k_norm = k_norm; p.q_out = (uint16_t *)q_out; p.nh = nh; p.rot = rot; p.eps = eps;
    for (int i = 0; i < rot / 2; i++) p.inv_freq[i] = pow(theta, -2.0 * i / rot);
    CwkKernelTimer timer(ctx);
    return c->hd == 256 ? launch_write<8, SRC_F32, true>(ctx, p, c->type) : launch_write<4, SRC_F32, true>(ctx, p, c->type);
}

}  // extern "C"
