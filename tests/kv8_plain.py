"""The GQA cache held in 8 bits, written down plainly in 64 bits (numpy and torch on the CPU): what the tests of cwk_kv8_store, cwk_kv8_load,
cwk_gqa_qk_prep_kv8, cwk_gqa_decode_kv8 and cwk_gqa_prefill_kv8 compare with."""
import math

import numpy as np
import torch

LOW, HIGH, MOST = -100, {"e4m3": 119, "int8": 121}, {"e4m3": 448.0, "int8": 127.0}


def e4m3_value(b):
    sign, e, m = (-1.0 if b & 128 else 1.0), (b >> 3) & 15, b & 7
    return math.nan if (e, m) == (15, 7) else sign * (m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10))


VALUES = {"e4m3": np.array([e4m3_value(b) for b in range(256)]), "int8": np.arange(256, dtype=np.uint8).view(np.int8).astype(np.float64)}


def encode(y, kind, values_tensor):
    """float64 in units of the scale -> codes; a NaN becomes E4M3's NaN among keys, 0 among values (values_tensor) and in INT8."""
    y = np.asarray(y, np.float64)
    nan = np.isnan(y)
    y = np.clip(np.where(nan, 0.0, y), -MOST[kind], MOST[kind])
    if kind == "int8":
        return np.rint(y).astype(np.int8).view(np.uint8)
    a = np.abs(y)
    _, ex = np.frexp(np.maximum(a, 2.0 ** -6))                # a = f * 2^ex, f in [0.5, 1): eight steps from 2^(ex - 1) to 2^ex
    step = np.ldexp(1.0, ex - 4)
    a = np.rint(a / step) * step
    grid = VALUES["e4m3"][:127]                               # the magnitudes in order: code = place
    code = np.searchsorted(grid, a).astype(np.uint8)
    assert np.array_equal(grid[code], a)
    code = code | np.where(np.signbit(y), 128, 0).astype(np.uint8)
    return np.where(nan, 0 if values_tensor else 127, code).astype(np.uint8)


def exponent(x, kind):
    """Least e with every finite |x| <= MOST * 2^e, within the limits."""
    a = np.abs(x[np.isfinite(x)])
    top = a.max() if a.size else 0.0
    if top == 0:
        return LOW
    e = math.frexp(top / MOST[kind])[1] - 1                   # 2^e <= top / MOST (but for the quotient's rounding)
    while top > MOST[kind] * 2.0 ** e:
        e += 1
    while e > LOW and top <= MOST[kind] * 2.0 ** (e - 1):
        e -= 1
    return min(max(e, LOW), HIGH[kind])


class Plain:
    """K or V of all slots: codes uint8 [slots][rows][nkv][hd], scale uint8 [slots][rows / block][nkv], as numpy arrays."""

    def __init__(self, codes, scale, block, kind, values_tensor):
        self.codes, self.scale, self.block, self.kind, self.values_tensor = codes.copy(), scale.copy(), block, kind, values_tensor

    def store(self, x, pos, count):
        """x float64 [B][n][nkv][hd]."""
        for b in range(x.shape[0]):
            p, c = int(pos[b]), min(int(count[b]), x.shape[1])
            c = 0 if p < 0 else max(0, min(c, self.codes.shape[1] - p))
            for first in range(p // self.block * self.block, p + c, self.block):
                lo, hi = max(first, p), min(first + self.block, p + c)
                if lo >= hi:
                    continue
                for h in range(x.shape[2]):
                    new = x[b, lo - p:hi - p, h]
                    e = exponent(new, self.kind)
                    at = (b, first // self.block, h)
                    if lo > first:
                        was = min(max(int(self.scale[at]) - 127, LOW), HIGH[self.kind])
                        if was >= e:
                            e = was
                        else:
                            held = VALUES[self.kind][self.codes[b, first:lo, h]] * 2.0 ** (was - e)
                            self.codes[b, first:lo, h] = encode(held, self.kind, self.values_tensor)
                    self.scale[at] = e + 127
                    self.codes[b, lo:hi, h] = encode(new * 2.0 ** -e, self.kind, self.values_tensor)

    def values(self):
        return VALUES[self.kind][self.codes] * np.ldexp(1.0, self.scale.astype(np.int64) - 127).repeat(self.block, 1)[..., None]


def norm_rotate(x, w, eps, rot, theta, pos):
    """x float64 [n][H][hd] at positions pos [n]: RMS norm with (1 + w), rotate-half on the first rot values."""
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * (1.0 + w.astype(np.float64))
    if rot == 0:
        return y
    a = pos[:, None, None].astype(np.float64) * (theta ** (-2.0 * np.arange(rot // 2) / rot))
    lo, hi = y[..., :rot // 2], y[..., rot // 2:rot]
    return np.concatenate([lo * np.cos(a) - hi * np.sin(a), hi * np.cos(a) + lo * np.sin(a), y[..., rot:]], -1)


def attend(q, k, v, limits, scale, p_step):
    """q float64 [n][nh][hd], k, v float64 [T][nkv][hd], limits [n] -> (out, tolerance), both [n][nh][hd] (torch float64).

    The tolerance of an element is what the number formats allow, A = sum_j p_j |v_j|, S = scale * sum_d |q_d k_d| at its worst key:
      2^-8 |out|            the result's rounding to bf16
      p_step A              the probabilities' rounding (f16 2^-11, bf16 2^-8)
      2 (hd 2^-22 S + 2^-20) A   the scores' f32 sums (a term may be cut off, not rounded) and the exponential, in numerator and sum
      (2^-25 + 2^-25 S) sum_j |v_j| / l    probabilities below f16's normal range, queries below 2^-14 of their row's largest
    """
    n, nh, hd = q.shape
    T, nkv = k.shape[:2]
    out, tol = torch.zeros(n, nh, hd, dtype=torch.float64, device=q.device), torch.zeros(n, nh, hd, dtype=torch.float64, device=q.device)
    if T == 0:
        return out, tol
    seen = torch.arange(T, device=q.device)[None] < limits[:, None]
    some = (limits > 0)[:, None]
    for h in range(nh):
        kk, vv = k[:, h // (nh // nkv)], v[:, h // (nh // nkv)]
        vv = torch.where(seen.any(0)[:, None], vv, 0.0)
        s = torch.where(seen, q[:, h] @ kk.T * scale, -torch.inf)
        top = s.amax(-1, keepdim=True)
        e = torch.exp(s - torch.where(some, top, 0.0))
        l = e.sum(-1, keepdim=True)
        p = torch.where(some, e / torch.where(some, l, 1.0), 0.0)
        out[:, h] = p @ vv
        A = p @ vv.abs()
        S = torch.where(seen, q[:, h].abs() @ kk.abs().T * scale, 0.0).amax(-1, keepdim=True)
        flat = seen.double() @ vv.abs() / torch.where(some, l, 1.0)
        tol[:, h] = 2.0 ** -8 * out[:, h].abs() + (p_step + 2 * (hd * 2.0 ** -22 * S + 2.0 ** -20)) * A + 2.0 ** -25 * (1 + S) * flat
    return out, tol
