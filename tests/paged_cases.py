"""Caches in pages, in numpy: pools and tables as aionhip_paged_cache describes them, rows turned by their positions, attention and eviction in 64 bits."""
import math

import numpy as np

from aion_amd import backend as be
from quant_cases import window_bounds

EPS = {be.F32: 2.0 ** -24, be.F16: 2.0 ** -11, be.BF16: 2.0 ** -8}          # half a step, relative
TINY = {be.F32: 2.0 ** -150, be.F16: 2.0 ** -25, be.BF16: 2.0 ** -134}       # half a subnormal step


def to_bits(x, dtype):
    """f32 -> what is stored (nearest, ties to even)"""
    x = np.ascontiguousarray(x, np.float32)
    if dtype == be.F32:
        return x
    if dtype == be.F16:
        with np.errstate(over="ignore"):
            return x.astype(np.float16)
    u = x.view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def to_f64(bits, dtype):
    if dtype == be.BF16:
        return (np.asarray(bits, np.uint16).astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return np.asarray(bits).astype(np.float64)


def storage(dtype):
    return {be.F32: np.float32, be.F16: np.float16, be.BF16: np.uint16}[dtype]


class Pages:
    """Host form of a cache: pools `k`, `v` of stored elements and the table."""

    def __init__(self, rng, dtype, b, width, p, h, d, spare=3, pages=None, sigma=1.0):
        self.dtype, self.b, self.width, self.p, self.h, self.d = dtype, b, width, p, h, d
        self.pages = b * width + spare if pages is None else pages
        spread = np.exp(0.4 * rng.standard_normal((1, h, 1, d)))
        self.k, self.v = (to_bits((rng.standard_normal((self.pages, h, p, d)) * spread * sigma).astype(np.float32), dtype) for _ in range(2))
        self.table = rng.permutation(self.pages)[:b * width].reshape(b, width).astype(np.int32)

    @property
    def capacity(self):
        return self.width * self.p

    def page(self, b, t):
        """the page of step t, or -1"""
        if t < 0 or t >= self.capacity:
            return -1
        page = int(self.table[b, t // self.p])
        return page if 0 <= page < self.pages else -1

    def rows(self, which, b, steps):
        """[len(steps), H, D] in f64, and which of them are there"""
        pool, there = (self.k, self.v)[which], np.array([self.page(b, t) >= 0 for t in steps], bool)
        out = np.zeros((len(steps), self.h, self.d))
        for i, t in enumerate(steps):
            if there[i]:
                out[i] = to_f64(pool[self.page(b, t), :, t % self.p], self.dtype)
        return out, there

    def put(self, which, b, t, row):
        if self.page(b, t) >= 0:
            (self.k, self.v)[which][self.page(b, t), :, t % self.p] = to_bits(row, self.dtype)

    def upload(self, gpu):
        k, v, table = gpu.upload(self.k), gpu.upload(self.v), gpu.upload(self.table)
        return gpu.paged_cache(k, v, table, self.pages, self.b, self.width, self.p, self.h, self.d, self.dtype)

    def same(self, gpu, cache):
        return all(np.array_equal(gpu.download(buf, storage(self.dtype), want.shape).view(np.uint16), want.view(np.uint16))
                   for buf, want in ((cache.k_pages, self.k), (cache.v_pages, self.v)))


def free(cache, *more):
    for x in (cache.k_pages, cache.v_pages, cache.page_table) + more:
        x.free()


def frequencies(r):
    """radians a position of each pair, in 64 bits, from the f32 fields of an aionhip_rotary"""
    n, base, s = r.dims // 2, float(r.base), float(r.factor)
    f = base ** (-2.0 * np.arange(n) / r.dims) if n else np.zeros(0)
    if r.scaling == be.ROTARY_PLAIN:
        return f
    if r.scaling == be.ROTARY_LINEAR:
        return f / s
    if r.scaling == be.ROTARY_BANDS:
        kept = (r.original_length * f / (2 * math.pi) - r.low) / (r.high - r.low)
    else:
        at = [r.dims * math.log(r.original_length / (2 * math.pi * turns)) / (2 * math.log(base)) for turns in (r.high, r.low)]
        a, b = max(math.floor(at[0]), 0), min(math.ceil(at[1]), r.dims - 1)
        kept = 1 - (np.arange(n) - a) / max(b - a, 0.001)
    kept = np.clip(kept, 0, 1)
    return f * (kept + (1 - kept) / s)


def turned(x, positions, r):
    """x [B,T,H,D] f64, positions [B,T] -> (turned rows, what the rounding errors of each element are relative to)"""
    n = r.dims // 2
    y, near = x.copy(), np.abs(x) * 0
    lo, hi = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if r.interleaved else (slice(0, n), slice(n, 2 * n))
    angle = (positions.astype(np.float64)[..., None] * frequencies(r))[:, :, None]
    c, s, m = np.cos(angle), np.sin(angle), float(r.magnitude)
    y[..., lo], y[..., hi] = (x[..., lo] * c - x[..., hi] * s) * m, (x[..., lo] * s + x[..., hi] * c) * m
    near[..., lo] = near[..., hi] = (np.abs(x[..., lo]) + np.abs(x[..., hi])) * abs(m)
    return y, near


def turned_close(got, x, positions, r, dtype):
    """Sine and cosine are off by 3 * 2^-24 at most (their series' own roundings, 2e-9 of truncation and as much of the angle), by one rounding more for the magnitude; a product and
    a sum round once each: 6 * 2^-24 of |l| + |h|. At far positions numpy's own angle, position * f rounded to 2^-53 of itself, adds that. Then the result is rounded to its type."""
    want, near = turned(x, positions, r)
    n = r.dims // 2
    own = np.zeros(x.shape)
    if n:
        e = np.abs(positions.astype(np.float64))[:, :, None, None] * frequencies(r).max() * 2.0 ** -51
        own = near * e
    return np.abs(got - want) <= near * 6 * 2.0 ** -24 + own + EPS[dtype] * np.abs(want) * (1 + 2.0 ** -10) + TINY[dtype]


class Near:
    def __init__(self, out, weight, reach, keys):
        self.out, self.weight, self.reach, self.keys = out, weight, reach, keys

    def close(self, got):
        """A score is a sum of D products of a query in two or three halves (2^-21 of each lost at most) and a key, D * 2^-24 of the sum of their magnitudes at most, and is rounded three
        times more; what it is off by, twice (its own and the normalizer's), goes into a probability. Sums over the keys: 32 a product, then one after another, then
        segments: (keys / 32 + 64) roundings, in numerator and denominator; exp2 and the halves of a probability 2^-21 together."""
        d = got.shape[-1]
        bound = 2 * self.reach * (d + 16) * 2.0 ** -24 + 2 * (self.keys / 32 + 64) * 2.0 ** -24 + 2.0 ** -21
        return np.abs(got - self.out) <= self.weight * np.expm1(np.minimum(bound, 50))[..., None] + 1e-37

    def weights_close(self, got, want, rows):
        """The same of a probability, and a rounding for each row that adds to it."""
        bound = 2 * self.reach.max() * (self.out.shape[-1] + 16) * 2.0 ** -24 + 2 * (self.keys.max() / 32 + 64) * 2.0 ** -24 + 2.0 ** -21
        return np.abs(got - want) <= np.abs(want) * np.expm1(bound) + (rows + 1) * 2.0 ** -24 * np.abs(want) + 1e-37


def attention(q, pages, l, hq, scale, window=be.CAUSAL, soft_cap=0.0, positions=None, lengths=None):
    """q [B,L,Hq,D] f64 -> (Near, weights [B,H,capacity])"""
    b, h, d, cap = pages.b, pages.h, pages.d, pages.capacity
    out, weight, reach, keys = np.zeros((b, l, hq, d)), np.zeros((b, l, hq, d)), np.zeros((b, l, hq)), np.zeros((b, l, hq))
    drawn = np.zeros((b, h, cap))
    for i in range(b):
        end = cap if lengths is None else max(0, min(int(lengths[i]), cap))
        k, there = pages.rows(0, i, range(end))
        v, _ = pages.rows(1, i, range(end))
        for j in range(l):
            pos = end - l + j if positions is None else max(int(positions[i][j]), 0)
            if pos < 0:
                continue
            lo, hi = window_bounds(window, pos, end)
            at = np.array([t for t in range(lo, max(hi, lo)) if there[t]], int)
            if at.size == 0:
                continue
            for head in range(hq):
                g = head // (hq // h)
                s = k[at, g] @ q[i, j, head] * scale
                reach[i, j, head] = (np.abs(k[at, g]) @ np.abs(q[i, j, head])).max() * abs(scale)
                keys[i, j, head] = at.size
                if soft_cap > 0:
                    s = soft_cap * np.tanh(s / soft_cap)
                top = s.max()
                if top == -math.inf:
                    continue
                p = np.exp(s - top)
                p /= p.sum()
                out[i, j, head], weight[i, j, head] = p @ v[at, g], p @ np.abs(v[at, g])
                drawn[i, g, at] += p
    return Near(out, weight, reach, keys), drawn


def staying(w, n, limit, keep, first, recent):
    """the steps that one head keeps of n, by its weights"""
    if n <= limit:
        return np.arange(n)
    middle = np.arange(first, n - recent)
    x = w[middle].astype(np.float64) + 0.0
    order = np.lexsort((middle, -np.where(np.isnan(x), 0, x), ~np.isnan(x)))
    return np.concatenate((np.arange(first), np.sort(middle[order[:keep - first - recent]]), np.arange(n - recent, n))).astype(int)


def evict(pages, weights, lengths, limit, keep, first, recent, table_out=None):
    """Moves the rows of `pages` (in place, or to table_out's pages) -> (kept [B,H,limit], lengths, weights)"""
    b, h = pages.b, pages.h
    k, v = pages.k.copy(), pages.v.copy()
    cap = pages.capacity
    cap_out = cap if table_out is None else table_out.shape[1] * pages.p
    kept, out, new = np.full((b, h, limit), -1, np.int32), np.zeros((b, h, cap_out), np.float32), np.zeros(b, np.int32)
    for i in range(b):
        n = max(0, min(int(lengths[i]), cap))
        for g in range(h):
            rows = staying(weights[i, g], n, limit, keep, first, recent)
            new[i] = rows.size
            kept[i, g, :rows.size], out[i, g, :rows.size] = rows, weights[i, g, rows]
            if table_out is None and n <= limit:
                out[i, g] = weights[i, g]
                continue
            for to, t in enumerate(rows):
                source = pages.page(i, t)
                target = (pages.page(i, to) if table_out is None else int(table_out[i, to // pages.p]))
                if source < 0 or not 0 <= target < pages.pages:
                    continue
                pages.k[target, g, to % pages.p], pages.v[target, g, to % pages.p] = k[source, g, t % pages.p], v[source, g, t % pages.p]
    return kept, new, out
