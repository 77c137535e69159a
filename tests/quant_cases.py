"""Caches held in 8 or 4 bits, in numpy: the buffer as aionhip_cache_quant_bytes describes it, and attention over it in 64 bits."""
import numpy as np

from aion_amd import backend as be

BITS = {be.Q8_0: 8, be.Q4_0: 4}
OFFSET = {be.Q8_0: 128, be.Q4_0: 8}


def padded(t_cap):
    return -(-t_cap // 64) * 64


def quantize(dtype, rows):
    """f32 rows [..., D] -> codes [..., D * bits / 8] as they are stored, scale bits [..., D / 32]. f32 arithmetic, every operation rounded on its own."""
    f32 = np.float32
    x = rows.reshape(rows.shape[:-1] + (-1, 32))
    top = np.abs(x).max(-1, keepdims=True)
    with np.errstate(divide="ignore", invalid="ignore", over="ignore"):
        full = np.where(top == 0, f32(1), top * (f32(1) / f32(127 if dtype == be.Q8_0 else 7)))
        held = full.astype(np.float16).astype(f32)
        if dtype == be.Q8_0:
            v = x * np.where((top == 0) | (held == 0), f32(0), f32(1) / held)
        else:
            v = x / full
    v = np.clip(np.copysign(np.floor(np.abs(v).astype(np.float64) + 0.5), v), -OFFSET[dtype], OFFSET[dtype] - 1)      # halves away from zero
    code = (v + OFFSET[dtype]).astype(np.uint8).reshape(rows.shape)
    if dtype == be.Q4_0:
        code = code[..., 0::2] | code[..., 1::2] << 4
    return code, full.astype(np.float16).view(np.uint16)[..., 0]


class QuantCache:
    """Host form of one cache: codes [B, H, Tp, D * bits / 8] and scales [B, H, D / 32, Tp] (f16 bits), views of one byte buffer."""

    def __init__(self, dtype, b, t_cap, h, d, fill=0):
        self.dtype, self.b, self.t_cap, self.h, self.d, self.tp = dtype, b, t_cap, h, d, padded(t_cap)
        n_codes = b * h * self.tp * d * BITS[dtype] // 8
        n_scales = b * h * self.tp * d // 32 * 2
        self.bytes = np.full(n_codes + n_scales, fill, np.uint8)
        self._views(n_codes)

    def _views(self, n_codes):
        self.codes = self.bytes[:n_codes].reshape(self.b, self.h, self.tp, -1)
        self.scales = self.bytes[n_codes:].view(np.uint16).reshape(self.b, self.h, self.d // 32, self.tp)

    def put(self, rows, b, row_index):
        """rows [S, H, D] f32, quantised, into rows row_index[i] of sequence b; a negative index: not written."""
        code, scale = quantize(self.dtype, np.ascontiguousarray(rows, np.float32))
        for i, r in enumerate(row_index):
            if r >= 0:
                self.codes[b, :, r] = code[i]
                self.scales[b, :, :, r] = scale[i]

    def values(self):
        """[B, Tp, H, D] in f64: every row of the buffer, whatever is in it."""
        code = self.codes
        if self.dtype == be.Q4_0:
            code = np.stack((code & 15, code >> 4), -1).reshape(self.b, self.h, self.tp, self.d)
        x = code.astype(np.float64) - OFFSET[self.dtype]
        with np.errstate(invalid="ignore"):
            x = x.reshape(self.b, self.h, self.tp, self.d // 32, 32) * self.scales.view(np.float16).astype(np.float64).transpose(0, 1, 3, 2)[..., None]
        return x.reshape(self.b, self.h, self.tp, self.d).transpose(0, 2, 1, 3)


def filled(rng, dtype, b, t_cap, h, d, sigma=1.0, fill=0xFF, rows=None):
    """A cache whose first `rows` rows (all) hold random numbers; what is behind them is `fill` (0xFF: scales that are NaN)."""
    c = QuantCache(dtype, b, t_cap, h, d, fill)
    n = t_cap if rows is None else rows
    spread = np.exp(0.4 * rng.standard_normal((h, d)))
    for i in range(b):
        c.put((rng.standard_normal((n, h, d)) * spread * sigma).astype(np.float32), i, range(n))
    return c


def window_bounds(window, pos, end):
    """AttentionWindow.keys for one position (graph/graph.zig:160-167)"""
    left, right, chunk = window
    pos = max(int(pos), 0)
    anchor = pos // chunk * chunk if chunk else pos
    span = chunk if chunk else 1
    lo = anchor - min(anchor, left)
    hi = end if right == be.UNBOUNDED else min(end, anchor + span + right)
    return lo, hi


class Bounds:
    """weight[B,L,Hq,Dv]: the sum of p |v| that an output element is an average over. reach[B,L,Hq]: the largest scale * sum |q k| that a score is made of.
    floor[B,L,Hq]: the keys times the largest p max|v| of one of them."""

    def __init__(self, weight, reach, floor):
        self.weight, self.reach, self.floor = weight, reach, floor


def attention_f64(q, k, v, scale, t_cap, window=be.CAUSAL, soft_cap=0.0, positions=None, kv_lengths=None, rolling=False):
    """q [B,L,Hq,D] and the rows k, v [B,T,Hkv,*] as the cache holds them, in 64 bits: (out, what its rounding errors are relative to)."""
    q = np.asarray(q, np.float64)
    bn, l, hq, _ = q.shape
    hkv, dv = k.shape[2], v.shape[3]
    out, near = np.zeros((bn, l, hq, dv)), Bounds(np.zeros((bn, l, hq, dv)), np.zeros((bn, l, hq)), np.zeros((bn, l, hq)))
    for b in range(bn):
        end = int(kv_lengths[b]) if kv_lengths is not None else t_cap
        end = max(end, 0) if rolling else max(0, min(end, t_cap))
        for i in range(l):
            lo, hi = window_bounds(window, positions[b][i] if positions is not None else i, end)
            if rolling:
                lo = max(lo, end - t_cap)
            if hi <= lo:
                continue
            rows = np.arange(lo, hi) % t_cap if rolling else np.arange(lo, hi)
            kb, vb = k[b, rows], v[b, rows]
            for h in range(hq):
                g = h // (hq // hkv)
                s = kb[:, g] @ q[b, i, h] * scale
                near.reach[b, i, h] = (np.abs(kb[:, g]) @ np.abs(q[b, i, h])).max() * abs(scale)
                if soft_cap > 0:
                    s = soft_cap * np.tanh(s / soft_cap)
                p = np.exp(s - s.max())
                p /= p.sum()
                out[b, i, h], near.weight[b, i, h] = p @ vb[:, g], p @ np.abs(vb[:, g])
                near.floor[b, i, h] = (hi - lo) * (p * np.abs(vb[:, g]).max(-1)).max()
    return out, near
