"""The 8-bit GQA cache without a GPU: the descriptor's layout, what is refused before any device is touched, the plain codec the GPU
tests compare with."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest
import torch

import kv8_plain as plain
from cwick_b200 import lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_the_descriptor_is_the_headers(tmp_path):
    src = tmp_path / "kv8.c"
    fields = [n for n, _ in lib.Kv8._fields_]
    src.write_text('#include <stdio.h>\n#include "cwk_attn.h"\nint main(void) { printf("%zu", sizeof(cwk_kv8));'
                   + "".join('printf(" %%zu", offsetof(cwk_kv8, %s));' % f for f in fields) + "return 0; }\n")
    subprocess.run([os.environ.get("CC", "gcc"), "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "kv8")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "kv8")], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [C.sizeof(lib.Kv8)] + [getattr(lib.Kv8, f).offset for f in fields]


def calls(L, d):
    a, x = None if d is None else C.addressof(d), 4096      # (no pointer is followed: there is no context)
    yield L.cwk_kv8_store(None, a, x, x, 0, x, None, 1, 1)
    yield L.cwk_kv8_load(None, a, x, None, 1, 1, x, x, 0)
    yield L.cwk_gqa_qk_prep_kv8(None, x, x, x, x, x, 1e-6, 64, 1e4, x, None, 1, 1, 8, x, a)
    yield L.cwk_gqa_decode_kv8(None, x, a, x, 64, 1, 1, 8, 1.0, x, 0)
    yield L.cwk_gqa_prefill_kv8(None, x, a, 0, 0, 1, 8, 1.0, x)


@pytest.mark.parametrize("change,want", [({}, lib.ERR_ARGUMENT), ({"hd": 64}, lib.ERR_UNSUPPORTED), ({"block": 16}, lib.ERR_UNSUPPORTED),
                                         ({"type": 7}, lib.ERR_UNSUPPORTED), ({"rows": 100}, lib.ERR_ARGUMENT), ({"k": None}, lib.ERR_ARGUMENT)])
def test_refusals_without_a_device(change, want):
    L = lib.load()
    d = lib.Kv8(4096, 4096, 4096, 4096, 128, 2, 2, 256, 64, lib.KV8_E4M3)
    for name, x in change.items():
        setattr(d, name, x)
    assert set(calls(L, d)) == {want}
    assert set(calls(L, None)) == {lib.ERR_ARGUMENT}


@pytest.mark.parametrize("name", ["cwk_kv8_store", "cwk_kv8_load", "cwk_gqa_qk_prep_kv8", "cwk_gqa_decode_kv8", "cwk_gqa_prefill_kv8"])
def test_a_decode_steps_calls_are_in_the_compiled_binding(name):
    L = lib.load()
    fn = lib.fast(L, name)
    assert type(fn).__name__ == "builtin_function_or_method"
    args = [0.0 if a in (C.c_float, C.c_double) else None if a is C.c_void_p else 1 for a in lib.SIGNATURES[name][1]]
    assert fn(*args) == lib.ERR_ARGUMENT == getattr(L, name)(*args)
    with pytest.raises(TypeError):
        fn(*args[:-1])


def test_the_plain_codec_is_torchs():
    x = torch.cat([torch.randn(20000) * 60, torch.linspace(-2 ** -5, 2 ** -5, 4001), torch.tensor([448.0, 464.0, -1e30, 0.0, -0.0, 2.0 ** -10, 1.5 * 2.0 ** -9])])
    want = x.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(plain.encode(x.double().numpy(), "e4m3", False), want)
    back = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(plain.VALUES["e4m3"], back, equal_nan=True)


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_the_plain_store_row_by_row_and_at_once(kind):
    """Within the roundings of codes that moved: none for E4M3's normal numbers, half a step of the final scale otherwise."""
    rng = np.random.default_rng(3)
    x = rng.standard_normal((1, 40, 2, 16)) * np.linspace(0.1, 9, 40)[None, :, None, None]
    one, all_ = (plain.Plain(np.zeros((1, 64, 2, 16), np.uint8), np.zeros((1, 2, 2), np.uint8), 32, kind, False) for _ in range(2))
    for r in range(40):
        one.store(x[:, r:r + 1], [r], [1])
    all_.store(x, [0], [40])
    assert np.array_equal(one.scale, all_.scale)
    unit = np.ldexp(1.0, one.scale.astype(int) - 127).repeat(32, 1)[..., None]
    assert np.all(np.abs(one.values() - all_.values()) <= (unit if kind == "int8" else unit * 2.0 ** -9))
    assert np.all(np.abs(all_.values()[:, :40] - x) <= (0.5 * unit[:, :40] if kind == "int8" else np.maximum(2.0 ** -4 * np.abs(x), 2.0 ** -10 * unit[:, :40])))


class Elsewhere:
    """Looks like a contiguous tensor of a GPU."""
    is_cuda = True

    def __init__(self, shape, dtype, device=0):
        self.shape, self.dtype, self.index = torch.Size(shape), dtype, device

    def get_device(self):
        return self.index

    def is_contiguous(self):
        return True

    def dim(self):
        return len(self.shape)

    def numel(self):
        return self.shape.numel()

    def data_ptr(self):
        return 4096


@pytest.mark.parametrize("what", ["kv8_store", "kv8_load", "gqa_qk_prep_kv8", "gqa_decode_kv8", "gqa_prefill_kv8"])
def test_tensors_of_another_gpu_are_refused(what, monkeypatch):
    """Every tensor of a call, one at a time on another GPU than the context's: refused before the address goes anywhere."""
    from types import SimpleNamespace

    from cwick_b200 import ops
    monkeypatch.setattr(torch, "empty_like", lambda t: t)
    B, n, nh, nkv, hd = 2, 3, 4, 2, 128
    f32, bf16, int32 = torch.float32, torch.bfloat16, torch.int32
    rows, row = (B, n, nkv, hd), ((B,), int32)
    cache = SimpleNamespace(nkv=nkv, hd=hd, device=0, address=4096)
    calls_made = []
    attn = object.__new__(ops.Attn)
    attn.device, attn.ctx = 0, SimpleNamespace(address=4096)
    setattr(attn, "_" + what, lambda *a: calls_made.append(a) or 0)
    tensors, call = {
        "kv8_store": ([(rows, bf16), (rows, bf16), row, row], lambda k, v, pos, count: attn.kv8_store(cache, k, v, pos, count)),
        "kv8_load": ([row, row, (rows, f32), (rows, f32)], lambda pos, count, k, v: attn.kv8_load(cache, pos, n, count, out=(k, v))),
        "gqa_qk_prep_kv8": ([((B, n, nh, 2 * hd), f32), (rows, f32), (rows, f32), ((hd,), f32), ((hd,), f32), row, row, ((B, n, nh, hd), bf16)],
                            lambda qg, k, v, qn, kn, pos, count, out: attn.gqa_qk_prep_kv8(cache, qg, k, v, qn, kn, 1e-6, 64, 1e4, pos, count, out)),
        "gqa_decode_kv8": ([((B, n, nh, hd), bf16), row, ((B, n, nh, hd), bf16)],
                           lambda q, lens, out: attn.gqa_decode_kv8(q, cache, lens, max_kv_len=64, out=out)),
        "gqa_prefill_kv8": ([((n, nh, hd), bf16)], lambda Q: attn.gqa_prefill_kv8(Q, cache, 0)),
    }[what]
    call(*(Elsewhere(*t) for t in tensors))
    assert len(calls_made) == 1
    for away in range(len(tensors)):
        for device in (1, -1):
            with pytest.raises(AssertionError):
                call(*(Elsewhere(*t, device if i == away else 0) for i, t in enumerate(tensors)))
    cache.device = 1
    with pytest.raises(AssertionError):
        call(*(Elsewhere(*t) for t in tensors))
    assert len(calls_made) == 1
