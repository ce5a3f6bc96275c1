"""The GQA cache held in 8 bits: writing, reading back, norms and rotation in front of it, decode and prompt chunks over it, and a layer's
steps as they are used together. Against kv8_plain.py."""
import ctypes as C

import numpy as np
import pytest
import torch

import kv8_plain as plain
from cwick_b200 import lib as cl

pytestmark = pytest.mark.gpu
F16, BF16 = 2.0 ** -11, 2.0 ** -8          # half a step, relative


@pytest.fixture(scope="module")
def attn():
    from cwick_b200.ops import Attn
    return Attn(0)


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def cache_of(slots, rows, nkv, hd, block, kind, seed=0):
    """A cache whose every byte is some other slot's past: codes of all kinds (E4M3's NaN among them), scales of any size."""
    from cwick_b200.ops import Kv8Cache
    c = Kv8Cache.empty(slots, rows, nkv, hd, block, kind)
    g = gen(seed)
    for t in (c.k, c.v):
        t.copy_(torch.randint(0, 256, t.shape, device="cuda", generator=g, dtype=torch.uint8))
    for t in (c.k_scale, c.v_scale):
        t.copy_(torch.randint(100, 130, t.shape, device="cuda", generator=g, dtype=torch.uint8))
    return c


def plain_of(c):
    return [plain.Plain(t.cpu().numpy(), s.cpu().numpy(), c.block, c.type, is_v)
            for t, s, is_v in ((c.k, c.k_scale, False), (c.v, c.v_scale, True))]


def same(c, want):
    for t, s, w in ((c.k, c.k_scale, want[0]), (c.v, c.v_scale, want[1])):
        for got, bytes_ in ((s, w.scale), (t, w.codes)):
            off = np.argwhere(got.cpu().numpy() != bytes_)
            assert not len(off), (len(off), off[:3].tolist())


def rows_of(seed, shape, dtype, spread=1.0):
    """Rows whose magnitudes go up and down over positions and heads."""
    g = gen(seed)
    x = torch.randn(shape, device="cuda", generator=g) * torch.exp(spread * torch.randn(shape[:-1], device="cuda", generator=g))[..., None]
    return x.to(dtype)


# ---- writing and reading ------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("block,hd,nkv,dtype", [(32, 128, 3, torch.bfloat16), (64, 256, 4, torch.float32), (128, 256, 1, torch.bfloat16)])
@pytest.mark.parametrize("n,pos,count", [(1, [0, 31, 64], None), (1, [127, 5, 383], None), (33, [0, 31, 100], [33, 0, 7]), (200, [1, 60, 128], None),
                                         (130, [254, 300, 383], [130, 84, 1])])
def test_store_writes_the_definitions_bytes(attn, kind, block, hd, nkv, dtype, n, pos, count):
    rows = 384
    c = cache_of(3, rows, nkv, hd, block, kind, seed=n)
    want = plain_of(c)
    k, v = rows_of(n, (3, n, nkv, hd), dtype), rows_of(n + 1, (3, n, nkv, hd), dtype)
    attn.kv8_store(c, k, v, i32(pos), None if count is None else i32(count))
    for w, x in zip(want, (k, v)):
        w.store(x.double().cpu().numpy(), pos, [n] * 3 if count is None else count)
    same(c, want)


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_store_row_by_row_meets_growing_scales(attn, kind):
    """Rows one at a time into an open block, each larger than the last: every one moves the codes in front of it."""
    c = cache_of(2, 64, 2, 128, 32, kind)
    want = plain_of(c)
    for r in range(40):
        k, v = (rows_of(10 * r + i, (2, 1, 2, 128), torch.bfloat16) * (1.0 + 0.3 * r) for i in range(2))
        attn.kv8_store(c, k, v, i32([r, r]))
        for w, x in zip(want, (k, v)):
            w.store(x.double().cpu().numpy(), [r, r], [1, 1])
    same(c, want)
    # the same rows at once: the same scales, and each value within the two roundings of the final scale's step
    d = cache_of(2, 64, 2, 128, 32, kind)
    k = torch.cat([rows_of(10 * r, (2, 1, 2, 128), torch.bfloat16) * (1.0 + 0.3 * r) for r in range(40)], 1)
    attn.kv8_store(d, k, k, i32([0, 0]))
    assert torch.equal(c.k_scale, d.k_scale)
    one, all_ = (plain.Plain(x.k.cpu().numpy(), x.k_scale.cpu().numpy(), 32, kind, False).values()[:, :40] for x in (c, d))
    unit = np.ldexp(1.0, d.k_scale.cpu().numpy().astype(np.int64) - 127).repeat(32, 1)[:, :40, :, None]
    step = unit if kind == "int8" else unit * 2.0 ** -9       # E4M3: only subnormals round again
    assert np.all(np.abs(one - all_) <= step)


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_store_of_extreme_values(attn, kind, dtype):
    rows = [0.0, -0.0, float("inf"), float("-inf"), float("nan"), 3.3e38, -3.3e38, 1e-38, 1e-30, 448.0, 464.0, 127.0, 127.5, 2.0 ** -100, 1.0, 0.0625]
    c = cache_of(1, 64 * 16, 1, 128, 64, kind)
    want = plain_of(c)
    k = torch.zeros(1, 64 * 16, 1, 128, device="cuda")
    for i, x in enumerate(rows):                              # a block for each: alone, then with values around it
        k[0, 64 * i, 0, 3] = x
        k[0, 64 * i + 1, 0, 5] = 1.5 if i % 2 else 0.0
    k = k.to(dtype)
    attn.kv8_store(c, k, k, i32([0]))
    for w in want:
        w.store(k.double().cpu().numpy(), [0], [64 * 16])
    same(c, want)
    assert np.isfinite(want[1].values()).all()                # no value that is not finite among the values
    assert np.isnan(want[0].values()).sum() == (1 if kind == "e4m3" else 0)


def test_store_leaves_out_what_is_outside_the_slot(attn):
    c = cache_of(4, 128, 2, 128, 64, "e4m3")
    want = plain_of(c)
    k = rows_of(3, (4, 50, 2, 128), torch.bfloat16)
    pos, count = [100, -3, 128, 2 ** 31 - 10], [70, 50, 50, 50]
    attn.kv8_store(c, k, k, i32(pos), i32(count))
    for w in want:
        w.store(k.double().cpu().numpy(), pos, count)
    same(c, want)


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hd,nkv", [(128, 3), (256, 4)])
def test_load_gives_every_value_exactly(attn, kind, dtype, hd, nkv):
    c = cache_of(3, 256, nkv, hd, 64, kind)
    vals = [w.values() for w in plain_of(c)]
    pos, count, n = [0, 63, 200], [100, 5, 100], 100
    out = tuple(torch.full((3, n, nkv, hd), -7.0, device="cuda", dtype=dtype) for _ in range(2))
    attn.kv8_load(c, i32(pos), n, i32(count), out=out)
    for o, w in zip(out, vals):
        o = o.double().cpu().numpy()
        for b in range(3):
            m = min(count[b], 256 - pos[b])
            assert np.array_equal(o[b, :m], w[b, pos[b]:pos[b] + m], equal_nan=True)
            assert (o[b, m:] == -7.0).all()
    k, v = attn.kv8_load(c, i32([256, -1, 255]), 1, dtype=dtype)
    assert np.array_equal(v[2, 0].double().cpu().numpy(), vals[1][2, 255], equal_nan=True)


def test_load_of_a_negative_position_writes_nothing(attn):
    c = cache_of(3, 128, 2, 128, 64, "int8")
    want = plain_of(c)[1].values()
    out = tuple(torch.full((3, 9, 2, 128), -7.0, device="cuda") for _ in range(2))
    attn.kv8_load(c, i32([-4, 0, -(2 ** 31)]), 9, out=out)
    assert (out[1][0] == -7.0).all() and (out[1][2] == -7.0).all()
    assert np.array_equal(out[1][1].double().cpu().numpy(), want[1, :9])


def test_offsets_beyond_32_bits(attn):
    """A cache of 2.6 GB a tensor: rows of the last slot, and of the end of the first one."""
    from cwick_b200.ops import Kv8Cache
    rows, nkv, hd = 1302528, 4, 256
    c = Kv8Cache.empty(2, rows, nkv, hd, 64, "int8")
    k, v = rows_of(1, (2, 70, nkv, hd), torch.bfloat16), rows_of(2, (2, 70, nkv, hd), torch.bfloat16)
    pos = i32([rows - 70, rows - 100])
    c.k_scale.fill_(60), c.v_scale.fill_(60)
    attn.kv8_store(c, k, v, pos)
    gk, gv = attn.kv8_load(c, pos, 70, dtype=torch.float32)
    for got, x, s in ((gk, k, c.k_scale), (gv, v, c.v_scale)):
        unit = torch.stack([torch.pow(2.0, s[b, (int(pos[b]) + torch.arange(70, device="cuda")) // 64].double() - 127) for b in range(2)])
        assert float(((got.double() - x.double()).abs() / unit[..., None]).max()) <= 0.5 * (1 + 2.0 ** -20)
    # decode over the last rows only is not a call there is; a short slot behind a long one is
    c.k[1, :64].copy_(c.k[1, rows - 64:]), c.v[1, :64].copy_(c.v[1, rows - 64:])
    c.k_scale[1, 0], c.v_scale[1, 0] = c.k_scale[1, -1], c.v_scale[1, -1]
    q = torch.randn(2, 8, hd, device="cuda", generator=gen(4)).to(torch.bfloat16)
    got = attn.gqa_decode_kv8(q, c, i32([0, 30]), max_kv_len=64)
    kk, vv = (torch.tensor(plain.VALUES["int8"], device="cuda")[t[1, :30].long()] * torch.pow(2.0, s[1, 0].double() - 127)[None, :, None]
              for t, s in ((c.k, c.k_scale), (c.v, c.v_scale)))
    want, tol = plain.attend(q[1:].double(), kk, vv, i32([30]), hd ** -0.5, F16)
    assert not got[0].any() and bool(((got[1:].double() - want).abs() <= tol).all())


# ---- norms and rotation -------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("n,pos,count", [(1, [0, 31, 100000], None), (70, [3, 60, 7], [70, 0, 33]), (200, [64, 1, 55], None)])
@pytest.mark.parametrize("nh,nkv,hd,rot,block", [(16, 4, 256, 64, 64), (6, 2, 128, 128, 32), (5, 1, 256, 256, 128), (3, 3, 128, 16, 64), (2, 1, 256, 0, 64)])
def test_prep_against_64_bits(attn, kind, n, pos, count, nh, nkv, hd, rot, block):
    rows, theta, eps = 100096, 1e7, 1e-6
    g = gen(n + hd)
    qg = torch.randn(3, n, nh, 2 * hd, device="cuda", generator=g)
    k, v = rows_of(n, (3, n, nkv, hd), torch.float32), rows_of(n + 1, (3, n, nkv, hd), torch.float32)
    qn, kn = (0.1 * torch.randn(hd, device="cuda", generator=g) for _ in range(2))
    from cwick_b200.ops import Kv8Cache
    c = Kv8Cache.empty(3, rows, nkv, hd, block, kind)
    for t in (c.k_scale, c.v_scale):
        t.fill_(100)
    for t in (c.k, c.v):
        t.fill_(0x35)
    q_out = torch.full((3, n, nh, hd), 9.0, dtype=torch.bfloat16, device="cuda")
    attn.gqa_qk_prep_kv8(c, qg, k, v, qn, kn, eps, rot, theta, i32(pos), None if count is None else i32(count), q_out=q_out)
    counts = [n] * 3 if count is None else count
    for b in range(3):
        p, m = pos[b], counts[b]
        at = p + np.arange(n)
        want = plain.norm_rotate(qg[b, ..., :hd].double().cpu().numpy(), qn.cpu().numpy(), eps, rot, theta, at)[:m]
        got = q_out[b, :m].double().cpu().numpy()
        # bf16's half step; f32 norm and rotation: a pair's members mix, each within a few 2^-24 of the larger
        size = np.abs(want).max(-1, keepdims=True) if m else 0
        assert np.all(np.abs(got - want) <= 2.0 ** -8 * np.abs(want) + 2.0 ** -20 * size)
        assert bool((q_out[b, m:] == 9.0).all())
        # the slot's touched rows, in whole blocks
        first, last = p // block * block, -(-(p + max(m, 1)) // block) * block
        kk = plain.norm_rotate(k[b].double().cpu().numpy(), kn.cpu().numpy(), eps, rot, theta, at)
        for t, s, x, is_v in ((c.k, c.k_scale, kk, False), (c.v, c.v_scale, v[b].double().cpu().numpy(), True)):
            w = plain.Plain(np.full((1, last - first, nkv, hd), 0x35, np.uint8), np.full((1, (last - first) // block, nkv), 100, np.uint8), block, kind, is_v)
            w.store(x[None], [p - first], [m])
            assert np.array_equal(s[b, first // block:last // block].cpu().numpy(), w.scale[0])
            assert np.array_equal(t[b, first:last].cpu().numpy(), w.codes[0])


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("eps", [1e-6, 0.0])
def test_prep_of_extreme_rows(attn, kind, eps):
    """Rows whose squares leave float's range at either end, zero rows, infinities and NaN, next to ordinary ones: the float pass cannot
    be trusted there, and codes and scales are still the definition's."""
    nh, nkv, hd, rot, block, theta, n = 2, 2, 256, 64, 32, 1e4, 96
    g = gen(5)
    k, v = (torch.randn(1, n, nkv, hd, device="cuda", generator=g) for _ in range(2))
    size = torch.ones(n, device="cuda")
    size[3], size[4], size[40], size[41], size[42] = 1e30, 1e-30, 3e37, 1e-42, 0.0
    k *= size[None, :, None, None]
    v *= size[None, :, None, None]
    k[0, 70, 0, 9], k[0, 71, 1, 200], v[0, 72, 0, 3], v[0, 73, 1, 4] = float("inf"), float("nan"), float("-inf"), float("nan")
    qn, kn = (0.1 * torch.randn(hd, device="cuda", generator=g) for _ in range(2))
    kn[100] = 1e6                                     # one channel far above the rest
    c = cache_of(1, 128, nkv, hd, block, kind)
    want = plain_of(c)
    qg = torch.randn(1, n, nh, 2 * hd, device="cuda", generator=g)
    attn.gqa_qk_prep_kv8(c, qg, k, v, qn, kn, eps, rot, theta, i32([7]))
    with np.errstate(all="ignore"):
        want[0].store(plain.norm_rotate(k[0].double().cpu().numpy(), kn.cpu().numpy(), eps, rot, theta, 7 + np.arange(n))[None], [7], [n])
        want[1].store(v.double().cpu().numpy(), [7], [n])
    same(c, want)


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("eps", [0.0, float(np.float32(1e-40)), float(np.float32(1e-32))])
@pytest.mark.parametrize("hd,alone", [(256, True), (128, True), (256, False)])
def test_prep_of_keys_whose_squares_are_subnormal(attn, kind, eps, hd, alone):
    """Without an epsilon that outweighs them, rows down to 1e-23 have a sum of squares in float that is not zero and has few bits: a block for
    each size, in which one row is that small (no other row casts doubt on the block) or all are."""
    sizes = [1e-15, 1e-16, 1e-17, 1e-18, 1e-19, 1e-20, 1e-21, 1e-22, 3e-23, 1e-23]
    nh, nkv, rot, block, theta, n = 1, 2, 64, 32, 1e4, 32 * len(sizes)
    g = gen(11)
    qg = torch.randn(1, n, nh, 2 * hd, device="cuda", generator=g)
    k, v = (torch.randn(1, n, nkv, hd, device="cuda", generator=g) for _ in range(2))
    for i, size in enumerate(sizes):
        k[:, 32 * i + 13:32 * i + 14 if alone else 32 * i + 32] *= size
    qn, kn = (0.1 * torch.randn(hd, device="cuda", generator=g) for _ in range(2))
    c = cache_of(1, n, nkv, hd, block, kind)
    want = plain_of(c)
    attn.gqa_qk_prep_kv8(c, qg, k, v, qn, kn, eps, rot, theta, i32([0]))
    want[0].store(plain.norm_rotate(k[0].double().cpu().numpy(), kn.cpu().numpy(), eps, rot, theta, np.arange(n))[None], [0], [n])
    want[1].store(v.double().cpu().numpy(), [0], [n])
    same(c, want)


@pytest.mark.parametrize("eps", [0.0, float(np.float32(1e-40)), 1e-6])
@pytest.mark.parametrize("hd,nh,n", [(256, 3, 90), (128, 10, 300)])
def test_prep_of_query_rows_of_any_size(attn, eps, hd, nh, n):
    """Query rows whose squares leave float's range at either end, or have few bits there, beside ordinary heads of the same token."""
    sizes = [1.0, 1e-10, 1e-15, 1e-17, 1e-18, 1e-19, 1e-20, 1e-21, 1e-22, 3e-23, 1e-30, 1e-37, 1e-42, 1e12, 1e15, 1e17, 1e18, 1e19, 1e25, 1e33, 5e37]
    nkv, rot, theta, pos = 1, 64, 1e4, 77
    g = gen(n)
    size = torch.tensor(sizes, device="cuda")[torch.arange(n * nh, device="cuda") % len(sizes)].view(n, nh, 1)
    qg = torch.randn(1, n, nh, 2 * hd, device="cuda", generator=g) * size
    k, v = (torch.randn(1, n, nkv, hd, device="cuda", generator=g) for _ in range(2))
    qn, kn = (0.1 * torch.randn(hd, device="cuda", generator=g) for _ in range(2))
    c = cache_of(1, 512, nkv, hd, 64, "e4m3")
    got = attn.gqa_qk_prep_kv8(c, qg, k, v, qn, kn, eps, rot, theta, i32([pos]))[0].double().cpu().numpy()
    want = plain.norm_rotate(qg[0, ..., :hd].double().cpu().numpy(), qn.cpu().numpy(), float(np.float32(eps)), rot, theta, pos + np.arange(n))
    # bf16's half step (of its least normal number below that); f32 norm and rotation as in test_prep_against_64_bits
    size = np.abs(want).max(-1, keepdims=True)
    assert np.all(np.abs(got - want) <= 2.0 ** -8 * np.abs(want) + 2.0 ** -20 * size + 2.0 ** -134)


# ---- decode -------------------------------------------------------------------------------------------------------------------

def filled(attn, slots, rows, nkv, hd, block, kind, seed, climb=False):
    """A cache with rows everywhere, and its values."""
    c = cache_of(slots, rows, nkv, hd, block, kind, seed)
    k, v = rows_of(seed, (slots, rows, nkv, hd), torch.float32, 0.3), rows_of(seed + 1, (slots, rows, nkv, hd), torch.float32, 0.3)
    if climb:
        k = 0.3 * k + torch.linspace(0, 6, rows, device="cuda")[:, None, None] * torch.sign(k[:, -1:])
    attn.kv8_store(c, k, v, i32([0] * slots))
    table = torch.tensor(plain.VALUES[kind], device="cuda")
    return c, *((table[t.long()] * torch.pow(2.0, s.double() - 127).repeat_interleave(block, 1)[..., None]) for t, s in ((c.k, c.k_scale), (c.v, c.v_scale)))


def spoil(c, lens):
    """Behind a slot's rows: E4M3's NaN, and scales that stand for infinity."""
    for b, n in enumerate(lens):
        c.k[b, n:] = 127
        c.v[b, n:] = 255
        for s in (c.k_scale, c.v_scale):
            s[b, -(-n // c.block):] = 255


def check_decode(attn, c, k, v, q, lens, scale=None, n_splits=0):
    B, n, nh, hd = q.shape
    spoil(c, lens)
    got = attn.gqa_decode_kv8(q, c, i32(lens), scale, max_kv_len=max(lens), n_splits=n_splits)
    attn.ctx.sync()
    for b in range(B):
        limits = (lens[b] - n + 1 + torch.arange(n, device="cuda")).clamp(min=0)
        want, tol = plain.attend(q[b].double(), k[b, :lens[b]], v[b, :lens[b]], limits, hd ** -0.5 if scale is None else scale, F16)
        off = (got[b].double() - want).abs()
        assert bool((off <= tol).all()), (b, float((off / tol.clamp(min=1e-30)).max()))
    return got


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("hd", [128, 256])
@pytest.mark.parametrize("nh,nkv", [(16, 4), (8, 1), (6, 2), (24, 3), (8, 8), (32, 2), (12, 1)])
@pytest.mark.parametrize("lens", [[0, 17, 0, 1, 2500, 64, 0], [3, 3, 3], [5000]])
def test_decode_of_ragged_batches(attn, kind, hd, nh, nkv, lens):
    rows = -(-max(lens) // 64) * 64
    c, k, v = filled(attn, len(lens), rows, nkv, hd, 64, kind, seed=nh + rows)
    q = torch.randn(len(lens), 1, nh, hd, device="cuda", generator=gen(nh)).to(torch.bfloat16)
    check_decode(attn, c, k, v, q, lens)


@pytest.mark.parametrize("n,hd,kind", [(1, 256, "e4m3"), (1, 128, "int8"), (4, 256, "int8")])
@pytest.mark.parametrize("B,most,nh,nkv", [(5, 130, 16, 4), (40, 300, 16, 4), (90, 300, 16, 4), (100, 60, 8, 2), (40, 300, 32, 8), (160, 200, 16, 4)])
def test_decode_of_many_short_sequences(attn, n, hd, kind, B, most, nh, nkv):
    """Blocks of one, two and four KV heads that have a sequence to themselves, one round of them and more."""
    rows = -(-most // 32) * 32
    c, k, v = filled(attn, B, rows, nkv, hd, 32, kind, seed=B + n)
    lens = torch.randint(0, most + 1, (B,), generator=torch.Generator().manual_seed(B)).tolist()
    lens[:5] = [most, 0, 1, 33, 32]
    q = torch.randn(B, n, nh, hd, device="cuda", generator=gen(B)).to(torch.bfloat16)
    check_decode(attn, c, k, v, q, lens)


@pytest.mark.parametrize("block", [32, 128])
@pytest.mark.parametrize("n,nh,nkv", [(2, 16, 4), (4, 16, 4), (5, 16, 4), (3, 6, 2), (2, 24, 3), (17, 8, 8), (3, 16, 1)])
@pytest.mark.parametrize("hd,lens", [(256, [700, 0, 1, 33]), (128, [2, 1031])])
def test_decode_of_several_tokens(attn, block, n, nh, nkv, hd, lens):
    """Fewer, as many and more tokens than share a pass; sequences shorter than the tokens: what sees no row is zero."""
    rows = -(-max(lens) // block) * block
    c, k, v = filled(attn, len(lens), rows, nkv, hd, block, "e4m3", seed=n)
    q = torch.randn(len(lens), n, nh, hd, device="cuda", generator=gen(n)).to(torch.bfloat16)
    got = check_decode(attn, c, k, v, q, lens)
    for b, m in enumerate(lens):
        assert not got[b, :max(0, n - m)].any()


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("n_splits", [0, 1, 3])
def test_decode_of_climbing_scores(attn, kind, n_splits):
    """Later keys lean further and further: the running maximum is outrun many times."""
    c, k, v = filled(attn, 2, 3200, 4, 256, 64, kind, seed=5, climb=True)
    q = (2 * torch.sign(k[:, -1]).repeat_interleave(4, 1)[:, None] + 0.1).to(torch.bfloat16)
    check_decode(attn, c, k, v, q, [3200, 1999], n_splits=n_splits)


def test_decode_of_queries_and_scales_far_from_one(attn):
    """Queries of 2^-40 to 2^30, blocks whose scales differ by 2^60, an all-zero block: nothing leaves the formats' range."""
    hd, nkv = 256, 2
    c = cache_of(1, 256, nkv, hd, 32, "e4m3")
    size = torch.tensor([1.0, 2.0 ** 30, 2.0 ** -30, 0.0, 1.0, 2.0 ** -60, 4.0, 1.0], device="cuda").repeat_interleave(32)[None, :, None, None]
    k, v = rows_of(1, (1, 256, nkv, hd), torch.float32, 0.0), rows_of(2, (1, 256, nkv, hd), torch.float32, 0.0) * size
    attn.kv8_store(c, k, v, i32([0]))
    table = torch.tensor(plain.VALUES["e4m3"], device="cuda")
    k, v = ((table[t.long()] * torch.pow(2.0, s.double() - 127).repeat_interleave(32, 1)[..., None]) for t, s in ((c.k, c.k_scale), (c.v, c.v_scale)))
    for f in (2.0 ** -40, 1.0, 2.0 ** 30):
        q = (torch.randn(1, 1, 4, hd, device="cuda", generator=gen(3)) * f).to(torch.bfloat16)
        for lens in ([256], [31], [100]):
            c2 = type(c)(c.k.clone(), c.v.clone(), c.k_scale.clone(), c.v_scale.clone(), 32, "e4m3")
            check_decode(attn, c2, k, v, q, lens, scale=hd ** -0.5 / f)


def test_decode_of_nan_rows(attn):
    """A NaN row reaches the tokens that see it and no other, of its own sequence or another."""
    c = cache_of(2, 128, 1, 256, 64, "e4m3")
    k, v = rows_of(1, (2, 100, 1, 256), torch.bfloat16), rows_of(2, (2, 100, 1, 256), torch.bfloat16)
    k[0, 98], v[0, 98] = float("nan"), float("nan")
    attn.kv8_store(c, k, v, i32([0, 0]))
    q = torch.randn(2, 3, 4, 256, device="cuda", generator=gen(1)).to(torch.bfloat16)
    got = attn.gqa_decode_kv8(q, c, i32([100, 100]), max_kv_len=100)
    assert bool(got[0, 0].isfinite().all()) and bool(got[1].isfinite().all())
    assert bool(got[0, 1:].isnan().all())


@pytest.mark.parametrize("n", [1, 4])
@pytest.mark.parametrize("lens,n_splits", [([4096], 0), ([4096], 5), ([4096, 700], 0), ([90] * 40, 0), ([300] * 90, 0), ([2500] + [40] * 70, 0)])
def test_decode_of_sequences_of_nan_rows(attn, n, lens, n_splits):
    """Sequences of NaN keys alone, and of 128 at the front: what warps leave of them has no score to be the reference exponent, and every query
    row shows it, however the rows are dealt out and joined. A sequence beside them does not."""
    nh, nkv, hd = 16, 4, 256
    rows = -(-max(lens) // 64) * 64
    for bad in (rows, 128):
        c = cache_of(len(lens), rows, nkv, hd, 64, "e4m3")
        k, v = (rows_of(i, (len(lens), rows, nkv, hd), torch.bfloat16) for i in range(2))
        k[0, :bad] = float("nan")
        attn.kv8_store(c, k, v, i32([0] * len(lens)))
        q = torch.randn(len(lens), n, nh, hd, device="cuda", generator=gen(1)).to(torch.bfloat16)
        got = attn.gqa_decode_kv8(q, c, i32(lens), max_kv_len=max(lens), n_splits=n_splits)
        assert bool(got[0].isnan().all())
        assert bool(got[1:].isfinite().all())



@pytest.mark.parametrize("expected", [0, 32, 1024])
@pytest.mark.parametrize("B,n,n_splits", [(3, 1, 0), (3, 5, 0), (3, 1, 2), (70, 1, 0)])
def test_decode_of_lengths_beyond_what_was_expected(attn, B, n, n_splits, expected):
    """max_kv_len shapes the launch only: longer sequences are read to their end, and a length beyond the slot's rows is the slot's."""
    nh, nkv, hd, rows = 16, 4, 256, 1024
    c, k, v = filled(attn, B, rows, nkv, hd, 64, "int8", seed=6)
    q = torch.randn(B, n, nh, hd, device="cuda", generator=gen(6)).to(torch.bfloat16)
    lens = [1000, 2 ** 31 - 1, 7, 1025, -3] * 14
    got = attn.gqa_decode_kv8(q, c, i32(lens[:B]), max_kv_len=expected, n_splits=n_splits)
    attn.ctx.sync()
    for b in range(B):
        m = min(max(lens[b], 0), rows)
        want, tol = plain.attend(q[b].double(), k[b, :m], v[b, :m], (m - n + 1 + torch.arange(n, device="cuda")).clamp(min=0), hd ** -0.5, F16)
        assert bool(((got[b].double() - want).abs() <= tol).all()), b



@pytest.mark.parametrize("largest,smaller", [((64, 1200, 1), [(16, 1200, 1), (16, 2000, 1)]), ((16, 500, 4), [(1, 4000, 4), (12, 900, 3), (2, 3000, 1)])])
def test_decode_captured_after_the_largest_step(attn, largest, smaller):
    """A context that has done the largest step has room for smaller ones, although the largest takes a form without records: their capture
    takes no memory, and one's replay holds after the others."""
    from cwick_b200.ops import Attn
    nh, nkv, hd = 16, 4, 256
    rows = max(x[1] for x in [largest] + smaller)
    rows = -(-rows // 64) * 64
    c, _, _ = filled(attn, largest[0], rows, nkv, hd, 64, "e4m3", seed=9)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()

    def query(B, n):
        return torch.randn(B, n, nh, hd, device="cuda", generator=gen(B)).to(torch.bfloat16)
    with torch.cuda.stream(side):
        a = Attn(0)
        before = a.ctx.launches
        a.gqa_decode_kv8(query(largest[0], largest[2]), c, i32([largest[1]] * largest[0]), max_kv_len=largest[1])
        assert a.ctx.launches - before == 1               # whole blocks
        graphs = []
        for B, length, n in smaller:
            q, lens = query(B, n), i32([length] * B)
            torch.cuda.synchronize()                      # (the other context is on another stream)
            out, want = torch.empty_like(q), attn.gqa_decode_kv8(q, c, lens, max_kv_len=length)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                a.gqa_decode_kv8(q, c, lens, max_kv_len=length, out=out)
            graphs.append((graph, out, want, q, lens))    # (the graph reads these two)
        for graph, out, want, *_ in graphs + graphs[::-1]:
            out.zero_()
            graph.replay()
            side.synchronize()
            assert torch.equal(out, want)
    del graphs, graph


def test_decode_gives_the_same_bits_again(attn):
    c, k, v = filled(attn, 3, 1024, 4, 256, 64, "e4m3", seed=8)
    q = torch.randn(3, 16, 256, device="cuda", generator=gen(2)).to(torch.bfloat16)
    lens = i32([1000, 17, 1024])
    first = attn.gqa_decode_kv8(q, c, lens)
    for _ in range(3):
        assert torch.equal(attn.gqa_decode_kv8(q, c, lens), first)


@pytest.mark.parametrize("B,length,n,nh,nkv,hd,launches", [(1, 100, 1, 16, 4, 256, 1), (1, 4000, 1, 16, 4, 256, 2), (16, 128, 1, 16, 4, 256, 1), (64, 4000, 1, 16, 4, 256, 2),
                                                           (64, 1200, 4, 16, 4, 256, 1), (2, 3000, 4, 16, 2, 128, 2)])
def test_decode_takes_the_form_it_is_tested_in(attn, B, length, n, nh, nkv, hd, launches):
    """Whole blocks are one launch, shares and their merge two: lengths far from where the cost changes sides."""
    rows = -(-length // 64) * 64
    c, k, v = filled(attn, B, rows, nkv, hd, 64, "int8", seed=B)
    q = torch.randn(B, n, nh, hd, device="cuda", generator=gen(B)).to(torch.bfloat16)
    lens = [length - b for b in range(B)]
    before = attn.ctx.launches
    check_decode(attn, c, k, v, q, lens)
    assert attn.ctx.launches - before == launches


# ---- prompt chunks --------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("n,pos,nh,nkv,hd", [(1, 0, 4, 1, 256), (1, 700, 16, 4, 256), (3, 500, 16, 4, 128), (17, 300, 8, 8, 256), (64, 0, 16, 1, 256),
                                             (200, 37, 16, 4, 256), (129, 0, 16, 4, 128), (257, 1300, 8, 2, 256), (300, 1, 4, 4, 128),
                                             (700, 0, 24, 3, 128), (150, 3000, 16, 2, 128), (520, 2800, 6, 2, 128), (130, 700, 20, 1, 256), (5, 70, 20, 1, 128)])
def test_prefill_against_64_bits(attn, kind, n, pos, nh, nkv, hd):
    T = pos + n
    rows = -(-T // 64) * 64
    c, k, v = filled(attn, 3, rows, nkv, hd, 64, kind, seed=n)
    spoil(c, [0, T, 0])
    Q = torch.randn(n, nh, hd, device="cuda", generator=gen(n)).to(torch.bfloat16)
    got = attn.gqa_prefill_kv8(Q, c, pos, slot=1)
    attn.ctx.sync()
    want, tol = plain.attend(Q.double(), k[1, :T], v[1, :T], pos + 1 + torch.arange(n, device="cuda"), hd ** -0.5, BF16)
    off = (got.double() - want).abs()
    assert bool((off <= tol).all()), float((off / tol).max())


@pytest.mark.parametrize("n,pos,nh,nkv,hd", [(5, 1000, 16, 4, 256), (300, 0, 16, 4, 256), (257, 3000, 8, 2, 256), (300, 0, 24, 3, 128), (150, 3000, 16, 2, 128)])
@pytest.mark.parametrize("bad", ["front", "last"])
def test_prefill_of_nan_rows(attn, n, pos, nh, nkv, hd, bad):
    """NaN keys reach the queries that see them and no other, by streams and by tensor cores, in shares or not."""
    T = pos + n
    rows = -(-T // 64) * 64
    c = cache_of(1, rows, nkv, hd, 64, "e4m3")
    k, v = (rows_of(i, (1, rows, nkv, hd), torch.bfloat16) for i in range(2))
    if bad == "front":
        k[0, :128] = float("nan")
    else:
        k[0, T - 3] = float("nan")
    attn.kv8_store(c, k, v, i32([0]))
    got = attn.gqa_prefill_kv8(torch.randn(n, nh, hd, device="cuda", generator=gen(n)).to(torch.bfloat16), c, pos)
    attn.ctx.sync()
    if bad == "front":
        assert bool(got.isnan().all())
    else:
        assert bool(got[:n - 3].isfinite().all()) and bool(got[n - 3:].isnan().all())


@pytest.mark.parametrize("climb", [False, True])
@pytest.mark.parametrize("n,pos,nh,nkv,launches", [(700, 0, 24, 3, 3), (512, 0, 32, 4, 3), (520, 1000, 20, 1, 3), (385, 700, 24, 6, 3), (256, 6000, 16, 2, 4), (520, 4800, 6, 2, 4),
                                                           (640, 6000, 16, 2, 4)])
def test_prefill_of_heads_of_128_and_climbing_scores(attn, n, pos, nh, nkv, launches, climb):
    """The tensor-core kernel at head dim 128, item by item (3 launches: the rows widened, the fast form, the exact form) and in shares (4: their
    merge), with scores that climb along the prompt by more than the fast form covers: the exact form does those items again."""
    hd, T = 128, pos + n
    rows = -(-T // 64) * 64
    g = gen(n + pos)
    Q = torch.randn(n, nh, hd, device="cuda", generator=g).to(torch.bfloat16)
    c = cache_of(1, rows, nkv, hd, 64, "e4m3", seed=n)
    k, v = rows_of(n, (1, rows, nkv, hd), torch.float32, 0.3), rows_of(n + 1, (1, rows, nkv, hd), torch.float32, 0.3)
    if climb:
        k = 0.2 * k + torch.linspace(0, 12, rows, device="cuda")[:, None, None] * torch.sign(Q[n - 1, 0].float())
    attn.kv8_store(c, k, v, i32([0]))
    table = torch.tensor(plain.VALUES["e4m3"], device="cuda")
    k, v = ((table[t.long()] * torch.pow(2.0, s.double() - 127).repeat_interleave(64, 1)[..., None]) for t, s in ((c.k, c.k_scale), (c.v, c.v_scale)))
    spoil(c, [T])
    before = attn.ctx.launches
    got = attn.gqa_prefill_kv8(Q, c, pos)
    attn.ctx.sync()
    assert attn.ctx.launches - before == launches
    limits = pos + 1 + torch.arange(n, device="cuda")
    want, tol = plain.attend(Q.double(), k[0, :T], v[0, :T], limits, hd ** -0.5, BF16)
    assert bool(((got.double() - want).abs() <= tol).all()), float(((got.double() - want).abs() / tol).max())
    if climb:       # some row's scores outrun its first tile's by 2^64, which is what flags an item
        s = (Q[:, 0].double() @ k[0, :T, 0].T).masked_fill(torch.arange(T, device="cuda") >= limits[:, None], -torch.inf) * hd ** -0.5 / np.log(2)
        assert float((s.amax(1) - s[:, :64].amax(1)).max()) > 100


def test_prefill_of_heads_of_128_over_keys_that_leave_l2(attn):
    """Widened keys and values above 64 MB, items one by one: query tiles of one head after the other."""
    nh, nkv, hd, n, pos = 148, 4, 128, 128, 40000
    T = pos + n
    rows = -(-T // 64) * 64
    assert 4 * T * nkv * hd > 64 << 20
    c, k, v = filled(attn, 1, rows, nkv, hd, 64, "int8", seed=2)
    spoil(c, [T])
    Q = torch.randn(n, nh, hd, device="cuda", generator=gen(3)).to(torch.bfloat16)
    before = attn.ctx.launches
    got = attn.gqa_prefill_kv8(Q, c, pos)
    attn.ctx.sync()
    assert attn.ctx.launches - before == 3
    heads = [0, 36, 37, 74, 147]
    for h in heads:
        want, tol = plain.attend(Q[:, h:h + 1].double(), k[0, :T, h // 37:h // 37 + 1], v[0, :T, h // 37:h // 37 + 1],
                                 pos + 1 + torch.arange(n, device="cuda"), hd ** -0.5, BF16)
        assert bool(((got[:, h:h + 1].double() - want).abs() <= tol).all()), h


def test_a_growing_prompts_workspace_grows_by_doubling(attn):
    """A prompt in chunks from position 0 on, on the tensor cores: the context's workspace is taken anew a few times, not for every chunk, and ends
    at what the slot needs."""
    from cwick_b200.ops import Attn
    nh, nkv, hd, n, chunks = 16, 4, 256, 512, 40
    c, _, _ = filled(attn, 1, n * chunks, nkv, hd, 64, "e4m3", seed=3)
    Q = torch.randn(n, nh, hd, device="cuda", generator=gen(1)).to(torch.bfloat16)
    torch.cuda.synchronize()
    other = Attn(0)
    free = []
    for i in range(chunks):
        before = other.ctx.launches
        other.gqa_prefill_kv8(Q, c, i * n)
        other.ctx.sync()
        assert other.ctx.launches - before >= 3, "not on the tensor cores"
        free.append(torch.cuda.mem_get_info()[0])
    # the first of 4 MB, doublings to the slot's 84; and the records of chunks dealt out in shares, a buffer of one size
    assert len(set(free)) <= 7, free


# ---- together -------------------------------------------------------------------------------------------------------------------

def test_a_prompt_and_the_tokens_behind_it(attn):
    """A slot's prompt in two chunks (prep, prefill), then tokens one by one beside another slot (prep, decode): every output against the
    values that the cache holds by then; the same steps captured in a graph and replayed, positions on the device, give the same bytes."""
    from cwick_b200.ops import Kv8Cache
    nh, nkv, hd, block, rot, theta, eps = 16, 4, 256, 64, 64, 1e7, 1e-6
    g = gen(7)
    qn, kn = (0.1 * torch.randn(hd, device="cuda", generator=g) for _ in range(2))

    def inputs(B, n):
        return torch.randn(B, n, nh, 2 * hd, device="cuda", generator=g), *(torch.randn(B, n, nkv, hd, device="cuda", generator=g) for _ in range(2))
    prompt = [inputs(1, 100), inputs(1, 41)]
    steps = [inputs(2, 1) for _ in range(6)]
    table = torch.tensor(plain.VALUES["e4m3"], device="cuda")

    def values(c):
        return ((table[t.long()] * torch.pow(2.0, s.double() - 127).repeat_interleave(block, 1)[..., None]) for t, s in ((c.k, c.k_scale), (c.v, c.v_scale)))

    def prompt_into(c):
        pos = 0
        for qg, k, v in prompt:
            n = qg.shape[1]
            q = attn.gqa_qk_prep_kv8(c, qg, k, v, qn, kn, eps, rot, theta, i32([pos]))
            got = attn.gqa_prefill_kv8(q[0], c, pos)
            kk, vv = values(c)
            want, tol = plain.attend(q[0].double(), kk[0, :pos + n], vv[0, :pos + n], pos + 1 + torch.arange(n, device="cuda"), hd ** -0.5, BF16)
            assert bool(((got.double() - want).abs() <= tol).all())
            pos += n
        return pos
    c = Kv8Cache.empty(2, 256, nkv, hd, block)
    pos = prompt_into(c)
    at, lens = i32([pos, 0]), i32([pos + 1, 1])
    eager = []
    for qg, k, v in steps:
        q = attn.gqa_qk_prep_kv8(c, qg, k, v, qn, kn, eps, rot, theta, at)
        got = attn.gqa_decode_kv8(q, c, lens, max_kv_len=256)
        kk, vv = values(c)
        for b in range(2):
            m = int(lens[b])
            want, tol = plain.attend(q[b].double(), kk[b, :m], vv[b, :m], i32([m]), hd ** -0.5, F16)
            assert bool(((got[b][None].double() - want).abs() <= tol).all())
        eager.append(got)
        at += 1
        lens += 1
    # the same with one captured step
    d = Kv8Cache.empty(2, 256, nkv, hd, block)
    prompt_into(d)
    at, lens = i32([pos, 0]), i32([pos + 1, 1])
    qg, k, v = (torch.empty_like(t) for t in steps[0])
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    from cwick_b200.ops import Attn
    with torch.cuda.stream(side):
        other = Attn(0)
        q = other.gqa_qk_prep_kv8(Kv8Cache.empty(2, 256, nkv, hd, block), *steps[0], qn, kn, eps, rot, theta, at)     # (grows its buffers)
        other.gqa_decode_kv8(q, d, lens, max_kv_len=256)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = other.gqa_decode_kv8(other.gqa_qk_prep_kv8(d, qg, k, v, qn, kn, eps, rot, theta, at), d, lens, max_kv_len=256)
            at += 1
            lens += 1
        for x, want in zip(steps, eager):
            for t, u in zip((qg, k, v), x):
                t.copy_(u)
            graph.replay()
            side.synchronize()
            assert torch.equal(out, want)
    del graph
    for b, m in enumerate((pos + 6, 6)):
        assert torch.equal(c.k[b, :m], d.k[b, :m]) and torch.equal(c.v[b, :m], d.v[b, :m])
        assert torch.equal(c.k_scale[b, :-(-m // block)], d.k_scale[b, :-(-m // block)])


# ---- refusals -------------------------------------------------------------------------------------------------------------------

def test_refusals(attn):
    c = cache_of(2, 128, 2, 256, 64, "e4m3")
    k = rows_of(1, (2, 1, 2, 256), torch.bfloat16)
    q, pos, o = torch.zeros(2, 8, 256, dtype=torch.bfloat16, device="cuda"), i32([0, 0]), torch.zeros(2, 8, 256, dtype=torch.bfloat16, device="cuda")
    L, h, p = attn.lib, attn.ctx.h, lambda t: cl.vp(t.data_ptr())
    f = torch.zeros(2, 1, 8, 512, device="cuda")

    def status(**change):
        d = cl.Kv8(c.c.k, c.c.v, c.c.k_scale, c.c.v_scale, c.rows, c.slots, c.nkv, c.hd, c.block, 0)
        for name, x in change.items():
            setattr(d, name, x)
        a = C.addressof(d)
        got = {L.cwk_kv8_store(h, a, p(k), p(k), 0, p(pos), None, 2, 1), L.cwk_kv8_load(h, a, p(pos), None, 2, 1, p(k), p(k), 0),
               L.cwk_gqa_qk_prep_kv8(h, p(f), p(f), p(f), p(f), p(f), 1e-6, 64, 1e4, p(pos), None, 2, 1, 8, p(o), a),
               L.cwk_gqa_decode_kv8(h, p(q), a, p(pos), 64, 2, 1, 8, 1.0, p(o), 0), L.cwk_gqa_prefill_kv8(h, p(q), a, 0, 0, 2, 8, 1.0, p(o))}
        assert len(got) == 1
        return got.pop()
    assert status() == cl.OK
    for bad in (dict(hd=64), dict(block=16), dict(block=48), dict(type=2)):
        assert status(**bad) == cl.ERR_UNSUPPORTED, bad
    for bad in (dict(rows=100), dict(rows=0), dict(slots=0), dict(nkv=0), dict(k=None), dict(v_scale=None), dict(k=c.c.k + 8), dict(rows=2 ** 31)):
        assert status(**bad) == cl.ERR_ARGUMENT, bad
    a = c.address
    bad = [L.cwk_kv8_store(h, a, p(k), p(k), 0, p(pos), None, 3, 1), L.cwk_kv8_store(h, a, p(k), p(k), 0, p(pos), None, 2, 0),
           L.cwk_kv8_store(h, a, None, p(k), 0, p(pos), None, 2, 1), L.cwk_kv8_store(h, a, cl.vp(k.data_ptr() + 2), p(k), 0, p(pos), None, 2, 1),
           L.cwk_kv8_load(h, a, p(pos), None, 3, 1, p(k), p(k), 0), L.cwk_kv8_load(h, a, None, None, 2, 1, p(k), p(k), 0),
           L.cwk_gqa_qk_prep_kv8(h, p(f), p(f), p(f), p(f), p(f), 1e-6, 272, 1e4, p(pos), None, 2, 1, 8, p(o), a),
           L.cwk_gqa_qk_prep_kv8(h, p(f), p(f), p(f), p(f), p(f), 1e-6, 64, 0.0, p(pos), None, 2, 1, 8, p(o), a),
           L.cwk_gqa_decode_kv8(h, p(q), a, p(pos), 129, 2, 1, 8, 1.0, p(o), 0), L.cwk_gqa_decode_kv8(h, p(q), a, p(pos), 64, 2, 1, 7, 1.0, p(o), 0),
           L.cwk_gqa_decode_kv8(h, p(q), a, p(pos), 64, 3, 1, 8, 1.0, p(o), 0), L.cwk_gqa_decode_kv8(h, p(q), a, p(pos), 64, 2, 0, 8, 1.0, p(o), 0),
           L.cwk_gqa_prefill_kv8(h, p(q), a, 2, 0, 2, 8, 1.0, p(o)), L.cwk_gqa_prefill_kv8(h, p(q), a, 0, 127, 2, 8, 1.0, p(o)),
           L.cwk_gqa_prefill_kv8(h, p(q), a, 0, -1, 2, 8, 1.0, p(o)), L.cwk_gqa_prefill_kv8(h, p(q), a, -1, 0, 2, 8, 1.0, p(o))]
    assert bad == [cl.ERR_ARGUMENT] * len(bad)
    bad = [L.cwk_gqa_qk_prep_kv8(h, p(f), p(f), p(f), p(f), p(f), 1e-6, 24, 1e4, p(pos), None, 2, 1, 8, p(o), a),
           L.cwk_gqa_decode_kv8(h, p(q), a, p(pos), 64, 2, 1, 34, 1.0, p(o), 0)]
    assert bad == [cl.ERR_UNSUPPORTED] * len(bad)
    attn.ctx.sync()
