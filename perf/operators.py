"""Performance cases of the GQA cache held in 8 bits: writing it (with and without the norms and the rotation in front),
reading it back, a decode step over it, a prompt chunk over it.

The cache of a slot holds K and V as 8-bit codes (E4M3, or two's complement INT8), [rows][kv heads][head dim], and a
power-of-two scale for each block of rows and KV head, as a biased exponent byte: value = code * 2^(byte - 127). Widths
are those of the repository's GQA layers (16 query heads, 4 KV heads of 256; rotation of the first 64 of a head, base
1e7) and the other groupings and head dimensions its GQA kernels are tested with.
"""
import math
from types import SimpleNamespace

import torch

own = False

DEV = "cuda:0"
EPS, ROT, THETA = 1e-6, 64, 1e7
LOW, HIGH = -100, {"e4m3": 119, "int8": 121}        # the least and the largest exponent of a scale
MOST = {"e4m3": 448.0, "int8": 127.0}


def listed():
    full = {"nh": 16, "nkv": 4, "hd": 256}
    return [
        # one user's next token at 4096 cached: latency
        {"name": "decode_1x4096", "kind": "decode", "batch": 1, "cached": 4096, "ragged": False, "tokens": 1, **full, "type": "e4m3", "block": 64},
        # an ordinary serving batch, every slot at its own length: cache bandwidth
        {"name": "decode_64x4096_ragged", "kind": "decode", "batch": 64, "cached": 4096, "ragged": True, "tokens": 1, **full, "type": "e4m3",
         "block": 64},
        # long contexts in INT8, heads of 128, eight query heads to a KV head
        {"name": "decode_6x30011_int8", "kind": "decode", "batch": 6, "cached": 30011, "ragged": True, "tokens": 1, "nh": 16, "nkv": 2, "hd": 128,
         "type": "int8", "block": 128},
        # three drafted tokens behind each slot's last one, checked in one step
        {"name": "decode_8x4_drafted", "kind": "decode", "batch": 8, "cached": 5003, "ragged": True, "tokens": 4, **full, "type": "e4m3", "block": 32},
        # a 512-position block of a long prompt (11,000 keys)
        {"name": "chunk_512_after_10488", "kind": "chunk", "tokens": 512, "before": 10488, **full, "type": "e4m3", "block": 64},
        # the odd-sized tail of a prompt behind a shared prefix, INT8
        {"name": "chunk_37_after_2501_int8", "kind": "chunk", "tokens": 37, "before": 2501, **full, "type": "int8", "block": 64},
        # a whole prompt, heads of 128
        {"name": "chunk_2000_hd128", "kind": "chunk", "tokens": 2000, "before": 0, "nh": 24, "nkv": 3, "hd": 128, "type": "e4m3", "block": 64},
        # the rows of one decode step of 64 slots, written and read back
        {"name": "write_64x1", "kind": "write", "batch": 64, "tokens": 1, "before": 2000, "ragged": False, "back": False, "nkv": 4, "hd": 256,
         "type": "e4m3", "block": 64, "f32": False},
        # a prefix of 16,381 rows moved into the cache and out again (blocks open at both ends)
        {"name": "write_16381_int8", "kind": "write", "batch": 1, "tokens": 16381, "before": 19, "ragged": False, "back": True, "nkv": 4, "hd": 256,
         "type": "int8", "block": 64, "f32": False},
        # what stands in front of a decode step's attention: q and k of 64 slots normed and rotated, the rows written
        {"name": "prep_64x1", "kind": "prep", "batch": 64, "tokens": 1, "before": 4000, "ragged": False, "back": False, **full, "type": "e4m3",
         "block": 64},
        # the same for a 512-position block of a prompt far into its context
        {"name": "prep_1x512_far", "kind": "prep", "batch": 1, "tokens": 512, "before": 99990, "ragged": False, "back": True, **full, "type": "e4m3",
         "block": 64},
        # chunks of ragged lengths of several slots, INT8
        {"name": "prep_7x300_ragged_int8", "kind": "prep", "batch": 7, "tokens": 300, "before": 1000, "ragged": True, "back": True, **full,
         "type": "int8", "block": 128},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    kind = rng.choice(["decode", "decode", "chunk", "chunk", "write", "prep"])
    nh, nkv = rng.choice([(16, 4), (16, 4), (16, 2), (8, 1), (8, 8), (24, 3), (32, 8), (32, 2)])
    c = {"kind": kind, "nh": nh, "nkv": nkv, "hd": rng.choice([128, 256]), "type": rng.choice(["e4m3", "int8"]), "block": rng.choice([32, 64, 128])}
    row = nkv * c["hd"]
    if kind == "decode":
        # up to the cache of the largest listed step (64 x 4096 rows of 1024 values)
        c["cached"] = _log(rng, 1, 40000)
        c["batch"] = _log(rng, 1, max(1, min(64, (64 * 4096 * 1024) // (c["cached"] * row))))
        c["tokens"] = min(c["cached"], rng.choice([1, 1, 1, 2, 3, 5]))
        c["ragged"] = rng.random() < 0.7
    elif kind == "chunk":
        c["tokens"] = _log(rng, 1, 2048)
        # up to the products of the largest listed chunk
        room = min(16000, 512 * 10744 * 16 * 256 // (c["tokens"] * nh * c["hd"]) - c["tokens"] // 2)
        c["before"] = 0 if rng.random() < 0.25 else _log(rng, 1, max(1, room))
    else:
        rows = _log(rng, 1, 12000 * 1024 // row if kind == "write" else 1800 * 16 // max(16, nh))
        c["batch"] = _log(rng, 1, min(64, rows))
        c["tokens"] = max(1, rows // c["batch"])
        c["before"] = 0 if rng.random() < 0.2 else _log(rng, 1, 30000 if c["batch"] <= 8 else 4000)
        c["ragged"], c["back"] = rng.random() < 0.5, rng.random() < 0.5
        if kind == "write":
            del c["nh"]
            c["f32"] = rng.random() < 0.3
    return c


# ---- the format -----------------------------------------------------------------------------------------------------------------

def _exponent(amax, kind):
    """Least e with amax <= MOST * 2^e, within the limits; amax is zero where there is nothing."""
    m, a = torch.frexp(amax)                                # amax = m * 2^a, m in [0.5, 1)
    e = (a - 9) + (m > 0.875) if kind == "e4m3" else (a - 7) + (m > 0.9921875)
    return torch.where(amax > 0, e, LOW).clamp(LOW, HIGH[kind]).to(torch.int32)


def _two(e):
    """2^e in f32, exactly (a power computed by the device may be off in its last place)."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _to_e4m3(y):
    """Nearest E4M3, ties to even. From 64 bits by way of 32: towards zero, with the last bit set where anything was cut
    off, so that the second rounding sees on which side of a tie the value is."""
    if y.dtype == torch.float64:
        near = y.float()
        bits = near.view(torch.int32)
        bits = bits - (near.double().abs() > y.abs()).to(torch.int32)
        y = (bits | (bits.view(torch.float32).double() != y).to(torch.int32)).view(torch.float32)
    return y.to(torch.float8_e4m3fn)


def _encode(x, e, kind):
    """Values -> codes as bytes; e broadcasts."""
    y = (x * _two(-e)).clamp(-MOST[kind], MOST[kind])
    return _to_e4m3(y).view(torch.uint8) if kind == "e4m3" else torch.round(y).to(torch.int8).view(torch.uint8)


def _decode(codes, e, kind):
    y = codes.view(torch.float8_e4m3fn if kind == "e4m3" else torch.int8).float()
    return y * _two(e)


def _blocks(x, block):
    """[B][rows][H][hd] -> [B][rows / block][block][H][hd]"""
    return x.view(x.shape[0], -1, block, *x.shape[2:])


def _encode_all(x, block, kind):
    """A whole cache from its rows: codes [B][rows][H][hd] and scale bytes [B][rows / block][H]."""
    y = _blocks(x, block)
    e = _exponent(y.abs().amax(dim=(2, 4)), kind)
    return _encode(y, e[:, :, None, :, None], kind).view(x.shape), (e + 127).to(torch.uint8)


def _decode_all(codes, scale, block, kind):
    return _decode(_blocks(codes, block), scale.to(torch.int32)[:, :, None, :, None] - 127, kind).view(codes.shape)


# ---- inputs ---------------------------------------------------------------------------------------------------------------------

def _lengths(case):
    """Cached rows of each slot: all alike, or spread over the upper half of the range (part of the case, not of the seed)."""
    B, T = case["batch"], case["cached"]
    if not case["ragged"]:
        return [T] * B
    g = torch.Generator().manual_seed(1000 * B + T)
    spread = torch.randint(max(case["tokens"], T // 2), T + 1, (B,), generator=g)
    spread[-1] = T
    return spread.tolist()


def _rows(gen, *shape, std=1.0):
    """K or V rows: some channels of a head are wider than others, as projections make them."""
    x = torch.randn(*shape, device=DEV, generator=gen)
    return x * (std * torch.exp(0.4 * torch.randn(*shape[-2:], device=DEV, generator=gen)))


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    s = SimpleNamespace(**{k: v for k, v in case.items() if k != "name"})
    nkv, hd, block = s.nkv, s.hd, s.block
    if s.kind in ("decode", "chunk"):
        B = s.batch if s.kind == "decode" else 1
        longest = s.cached if s.kind == "decode" else s.before + s.tokens
        s.rows = -(-longest // block) * block
        s.k, s.ks = _encode_all(_rows(gen, B, s.rows, nkv, hd), block, s.type)
        s.v, s.vs = _encode_all(_rows(gen, B, s.rows, nkv, hd), block, s.type)
        if s.kind == "decode":
            s.q = torch.randn(B, s.tokens, s.nh, hd, device=DEV, generator=gen).to(torch.bfloat16)
            s.kv_len, s.longest = torch.tensor(_lengths(case), dtype=torch.int32, device=DEV), longest
        else:
            s.q = torch.randn(s.tokens, s.nh, hd, device=DEV, generator=gen).to(torch.bfloat16)
        return s
    B, n = s.batch, s.tokens
    g = torch.Generator().manual_seed(100 * B + n)
    pos = torch.full((B,), s.before) if not s.ragged else torch.randint(s.before // 2, s.before + 1, (B,), generator=g)
    count = torch.randint((n + 1) // 2, n + 1, (B,), generator=g) if s.ragged else None
    window = ((n + block - 1) // block + 1) * block                       # rows of the blocks that n rows can lie in
    s.rows = (s.before // block) * block + window
    s.pos = pos.to(torch.int32).to(DEV)
    s.count = None if count is None else count.to(torch.int32).to(DEV)
    s.window = window
    # the slots hold rows already; the new ones are a little wider, so that open blocks meet scales that grow
    slot, first = torch.arange(B, device=DEV), (pos // block).to(DEV)
    held = (slot[:, None], (first * block)[:, None] + torch.arange(block, device=DEV))
    s.k, s.v = (torch.zeros(B, s.rows, nkv, hd, dtype=torch.uint8, device=DEV) for _ in range(2))
    s.ks, s.vs = (torch.full((B, s.rows // block, nkv), 127 - 9, dtype=torch.uint8, device=DEV) for _ in range(2))
    for codes, scale in ((s.k, s.ks), (s.v, s.vs)):
        c, e = _encode_all(_rows(gen, B, block, nkv, hd, std=0.5), block, s.type)
        codes[held], scale[slot, first] = c, e[:, 0]
    if s.kind == "write":
        dtype = torch.float32 if s.f32 else torch.bfloat16
        s.xk, s.xv = _rows(gen, B, n, nkv, hd).to(dtype), _rows(gen, B, n, nkv, hd).to(dtype)
    else:
        s.qg = torch.randn(B, n, s.nh, 2 * hd, device=DEV, generator=gen)
        s.xk, s.xv = _rows(gen, B, n, nkv, hd), _rows(gen, B, n, nkv, hd)
        s.q_norm, s.k_norm = (0.1 * torch.randn(hd, device=DEV, generator=gen) for _ in range(2))
        s.q_out = torch.zeros(B, n, s.nh, hd, dtype=torch.bfloat16, device=DEV)
    # what is read back: the new rows, or from the start of the block that the first of them is in
    lead = (pos % block if s.back else torch.zeros_like(pos)).to(torch.int32).to(DEV)
    s.from_row = s.pos - lead
    s.many = n + (block - 1 if s.back else 0)
    s.read = lead + (s.count if s.count is not None else n)
    s.k_back, s.v_back = (torch.zeros(B, s.many, nkv, hd, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    return s


# ---- the plain forms ------------------------------------------------------------------------------------------------------------

def _attend(q, k, v, limit):
    """q [B][n][nh][hd], k, v f32 [B][T][nkv][hd], limit [B][n]: query i of slot b sees its first limit rows."""
    B, n, nh, hd = q.shape
    T, nkv = k.shape[1:3]
    rows = q.float().view(B, n, nkv, nh // nkv, hd).permute(0, 2, 3, 1, 4).reshape(B, nkv, -1, hd)           # [B][nkv][group n][hd]
    sc = torch.matmul(rows, k.permute(0, 2, 3, 1)).view(B, nkv, nh // nkv, n, T) / math.sqrt(hd)
    seen = (torch.arange(T, device=DEV) < limit[:, :, None])[:, None, None]
    sc = torch.where(seen, sc, -torch.inf)
    p = torch.exp(sc - sc.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(B, nkv, -1, T), v.permute(0, 2, 1, 3))
    return out.view(B, nkv, nh // nkv, n, hd).permute(0, 3, 1, 2, 4).reshape(B, n, nh, hd).to(torch.bfloat16)


def _plain_decode(s):
    k, v = _decode_all(s.k, s.ks, s.block, s.type), _decode_all(s.v, s.vs, s.block, s.type)
    return _attend(s.q, k, v, s.kv_len[:, None] - s.tokens + 1 + torch.arange(s.tokens, device=DEV))


def _plain_chunk(s):
    k, v = _decode_all(s.k, s.ks, s.block, s.type), _decode_all(s.v, s.vs, s.block, s.type)
    return _attend(s.q[None], k, v, s.before + 1 + torch.arange(s.tokens, device=DEV)[None])[0]


def _put(s, x, codes, scale):
    """The new rows x [B][n][H][hd] into a cache, in place."""
    B, n = x.shape[:2]
    slot = torch.arange(B, device=DEV)[:, None]
    first = s.pos // s.block
    rows = (first * s.block)[:, None] + torch.arange(s.window, device=DEV)                    # [B][window]
    blocks = first[:, None] + torch.arange(s.window // s.block, device=DEV)
    count = s.count if s.count is not None else torch.full_like(s.pos, n)
    new = (rows >= s.pos[:, None]) & (rows < (s.pos + count)[:, None])
    old = (rows < s.pos[:, None]) & (count > 0)[:, None]
    xn = torch.where(new[:, :, None, None], x[slot, (rows - s.pos[:, None]).clamp(0, n - 1)], 0.0)
    was = scale[slot, blocks].to(torch.int32) - 127                                          # [B][blocks][H]
    e = _exponent(_blocks(xn, s.block).abs().amax(dim=(2, 4)), s.type)
    open_ = _blocks(old, s.block).any(2)[:, :, None]
    e = torch.where(open_, torch.maximum(e, was), e)
    held = codes[slot, rows]
    value = torch.where(old[:, :, None, None], _decode(_blocks(held, s.block), was[:, :, None, :, None], s.type).view(xn.shape).to(xn.dtype), xn)
    got = _encode(_blocks(value, s.block), e[:, :, None, :, None], s.type).view(held.shape)
    codes[slot, rows] = torch.where((new | old)[:, :, None, None], got, held)
    touched = _blocks(new, s.block).any(2)[:, :, None]
    scale[slot, blocks] = torch.where(touched, e + 127, was + 127).to(torch.uint8)


def _get(s, codes, scale, back):
    """Rows from_row .. of a cache as bf16; rows behind `read` stay as they are."""
    slot = torch.arange(codes.shape[0], device=DEV)[:, None]
    j = torch.arange(s.many, device=DEV)
    rows = (s.from_row[:, None] + j).clamp(max=s.rows - 1)
    y = _decode(codes[slot, rows], (scale[slot, rows // s.block].to(torch.int32) - 127)[..., None], s.type)
    back.copy_(torch.where((j < s.read[:, None])[:, :, None, None], y.to(torch.bfloat16), back))
    return back


def _norm_rotate(x, w, angle):
    """x [B][n][H][hd]: RMS norm with (1 + w), rotate-half on the first ROT values by angle f64 [B][n][ROT / 2]."""
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * (1 + w.to(x.dtype))
    c, d = torch.cos(angle).to(x.dtype)[:, :, None], torch.sin(angle).to(x.dtype)[:, :, None]
    lo, hi = y[..., :ROT // 2], y[..., ROT // 2:ROT]
    return torch.cat([lo * c - hi * d, hi * c + lo * d, y[..., ROT:]], -1)


def _plain_write(s):
    if s.kind == "write":
        q, k, v = None, s.xk.float(), s.xv.float()
    else:
        place = (s.pos[:, None] + torch.arange(s.tokens, device=DEV)).double()
        angle = place[:, :, None] * THETA ** (-torch.arange(0, ROT, 2, device=DEV, dtype=torch.float64) / ROT)
        q = _norm_rotate(s.qg[..., :s.hd], s.q_norm, angle).to(torch.bfloat16)
        if s.count is not None:
            q = torch.where((torch.arange(s.tokens, device=DEV) < s.count[:, None])[:, :, None, None], q, s.q_out)
        k, v = _norm_rotate(s.xk.double(), s.k_norm, angle), s.xv        # keys in 64 bits: a code hangs on which side of a border a value is
    _put(s, k, s.k, s.ks)
    _put(s, v, s.v, s.vs)
    back = {"k": _get(s, s.k, s.ks, s.k_back), "v": _get(s, s.v, s.vs, s.v_back)}
    return back if q is None else {"q": q, **back}


# ---- the framework's calls --------------------------------------------------------------------------------------------------------

_attn = None


def _own(s):
    global _attn
    from cwick_b200.ops import Attn, Kv8Cache
    if _attn is None:
        _attn = Attn(0)
    if not hasattr(s, "cache"):                             # the handle that a program keeps beside its buffers
        s.cache = Kv8Cache(s.k, s.v, s.ks, s.vs, s.block, s.type)
    if s.kind == "decode":
        return _attn.gqa_decode_kv8(s.q, s.cache, s.kv_len, max_kv_len=s.longest)
    if s.kind == "chunk":
        return _attn.gqa_prefill_kv8(s.q, s.cache, s.before)
    if s.kind == "write":
        _attn.kv8_store(s.cache, s.xk, s.xv, s.pos, s.count)
        k, v = _attn.kv8_load(s.cache, s.from_row, s.many, s.read, out=(s.k_back, s.v_back))
        return {"k": k, "v": v}
    q = _attn.gqa_qk_prep_kv8(s.cache, s.qg, s.xk, s.xv, s.q_norm, s.k_norm, EPS, ROT, THETA, s.pos, s.count, q_out=s.q_out)
    k, v = _attn.kv8_load(s.cache, s.from_row, s.many, s.read, out=(s.k_back, s.v_back))
    return {"q": q, "k": k, "v": v}


def run(state):
    if own:
        return _own(state)
    return {"decode": _plain_decode, "chunk": _plain_chunk, "write": _plain_write, "prep": _plain_write}[state.kind](state)


def work(case):
    c = SimpleNamespace(**case)
    row = c.nkv * c.hd
    if c.kind == "decode":
        lens = _lengths(case)
        seen = sum(n - c.tokens + 1 + i for n in lens for i in range(c.tokens))
        scales = sum(-(-n // c.block) for n in lens) * 2 * c.nkv
        return {"bytes": 2 * row * sum(lens) + scales + 4 * c.batch * c.tokens * c.nh * c.hd + 4 * c.batch, "flops": 4 * c.hd * c.nh * seen}
    if c.kind == "chunk":
        T = c.before + c.tokens
        seen = sum(c.before + 1 + i for i in range(c.tokens))
        return {"bytes": 2 * row * T + -(-T // c.block) * 2 * c.nkv + 4 * c.tokens * c.nh * c.hd, "flops": 4 * c.hd * c.nh * seen}
    B, n = c.batch, c.tokens
    new = B * n
    if c.ragged:                                            # as prepare() draws them
        g = torch.Generator().manual_seed(100 * B + n)
        pos = torch.randint(c.before // 2, c.before + 1, (B,), generator=g)
        new = int(torch.randint((n + 1) // 2, n + 1, (B,), generator=g).sum())
    else:
        pos = torch.full((B,), c.before)
    lead = int((pos % c.block).sum()) if c.back else 0
    size = 4 if c.kind == "prep" or c.f32 else 2
    # rows in, codes out; codes in again with the rows before them, values out
    total = 2 * row * (new * (size + 1) + (new + lead) * 3)
    flops = 2 * row * (new * 3 + (new + lead))
    if c.kind == "prep":
        total += new * c.nh * c.hd * 6 + 8 * c.hd
        flops += new * (c.nh * c.hd + row) * 8
    return {"bytes": total, "flops": flops}


# ---- from the definition, in 64 bits ----------------------------------------------------------------------------------------------

def _values64(kind):
    """What each of the 256 codes stands for."""
    if kind == "int8":
        return [float(b - 256 if b > 127 else b) for b in range(256)]

    def one(b):
        sign, e, m = (-1.0 if b & 128 else 1.0), (b >> 3) & 15, b & 7
        if e == 15 and m == 7:
            return math.nan
        return sign * (m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10))
    return [one(b) for b in range(256)]


def _two64(e):
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _cache64(codes, scale, block, kind):
    table = torch.tensor(_values64(kind), dtype=torch.float64, device=DEV)
    unit = _two64(scale.long() - 127).repeat_interleave(block, dim=1)
    return table[codes.long()] * unit[..., None]


def _round64(y, kind):
    """The code's value nearest to y (ties to the even code), y in units of the scale."""
    top = MOST[kind]
    if kind == "int8":
        return torch.round(y).clamp(-top, top)
    step = _two64(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    # log2 may be a hair off next to a power of two: the step is a power of two with |y| / step in [8, 16)
    step = torch.where(y.abs() >= 16 * step, 2 * step, torch.where((y.abs() < 8 * step) & (step > 2.0 ** -9), step / 2, step))
    return (torch.round(y / step) * step).clamp(-top, top)


def exact(case, seed):
    s = prepare(case, seed)
    if s.kind in ("decode", "chunk"):
        B = s.k.shape[0]
        q = (s.q if s.kind == "decode" else s.q[None]).double()
        lens = _lengths(case) if s.kind == "decode" else [s.before + s.tokens]
        n, group, want = q.shape[1], s.nh // s.nkv, torch.empty(q.shape, dtype=torch.float64, device=DEV)
        for b in range(B):
            T = lens[b]
            k = _cache64(s.k[b:b + 1], s.ks[b:b + 1], s.block, s.type)[0, :T]
            v = _cache64(s.v[b:b + 1], s.vs[b:b + 1], s.block, s.type)[0, :T]
            hidden = torch.arange(T, device=DEV)[None] > T - n + torch.arange(n, device=DEV)[:, None]
            for h in range(s.nh):
                sc = (q[b, :, h] @ k[:, h // group].T / math.sqrt(s.hd)).masked_fill(hidden, -math.inf)
                want[b, :, h] = torch.softmax(sc, -1) @ v[:, h // group]
        return want if s.kind == "decode" else want[0]
    B, n = s.batch, s.tokens
    k, v, out = s.xk.double(), s.xv.double(), {}
    counts = [n] * B if s.count is None else s.count.tolist()
    pos = s.pos.tolist()
    if s.kind == "prep":
        freq = torch.tensor([THETA ** (-2.0 * i / ROT) for i in range(ROT // 2)], dtype=torch.float64, device=DEV)
        turn = torch.stack([torch.arange(p, p + n, device=DEV) for p in pos]).double()[..., None] * freq
        turn = torch.polar(torch.ones_like(turn), turn)[:, :, None]

        def head(x, w):
            y = x / torch.sqrt(x.square().sum(-1, keepdim=True) / s.hd + EPS) * (1.0 + w.double())
            z = torch.complex(y[..., :ROT // 2].contiguous(), y[..., ROT // 2:ROT].contiguous()) * turn
            return torch.cat([z.real, z.imag, y[..., ROT:]], dim=-1)
        q = head(s.qg[..., :s.hd].double(), s.q_norm)
        for b in range(B):
            q[b, counts[b]:] = 0
        out["q"], k = q, head(k, s.k_norm)
    for name, x, codes, scale in (("k", k, s.k, s.ks), ("v", v, s.v, s.vs)):
        held = _cache64(codes, scale, s.block, s.type)
        back = torch.zeros(B, s.many, s.nkv, s.hd, dtype=torch.float64, device=DEV)
        for b in range(B):
            first, last = pos[b] // s.block, (pos[b] + counts[b] - 1) // s.block
            lo = first * s.block
            row = torch.zeros((last - first + 1) * s.block, s.nkv, s.hd, dtype=torch.float64, device=DEV)
            lead = pos[b] - lo
            row[lead:lead + counts[b]] = x[b, :counts[b]]
            top = row.view(-1, s.block, s.nkv, s.hd).abs().amax(dim=(1, 3))
            e = torch.ceil(torch.log2(top.clamp(min=2.0 ** -200) / MOST[s.type]))
            e = torch.where(top > MOST[s.type] * _two64(e), e + 1, torch.where(top <= MOST[s.type] * _two64(e - 1), e - 1, e))
            e = e.clamp(LOW, HIGH[s.type])
            if lead:
                e[0] = torch.maximum(e[0], scale[b, first].double() - 127)
                row[:lead] = held[b, lo:pos[b]]
            unit = _two64(e).repeat_interleave(s.block, dim=0)[..., None]
            value = _round64(row / unit, s.type) * unit
            start = lead if not s.back else 0
            m = counts[b] + lead - start
            back[b, :m] = value[start:start + m]
        out[name] = back
    return out
