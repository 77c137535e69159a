"""Attention over pages where a few keys hold nearly all of the probability and what counts are the others."""
import numpy as np
import pytest

from aion_amd import backend as be
from paged_cases import Near, Pages, to_bits, to_f64
from test_gpu_paged import attend

pytestmark = pytest.mark.gpu


def peaked(rng, dtype, n, hq, h, d, score, value):
    """One sequence of n keys, score(t) along the first column (the queries are 1 there and 0 elsewhere), values normal numbers times value(t) -> (pages, Near, drawn)"""
    p = 64
    pages = Pages(rng, dtype, 1, 1, p, h, d, pages=1)
    pages.width = -(-n // p)
    pages.pages = pages.width
    shape = (pages.pages, h, p, d)
    t = np.arange(pages.capacity)
    k = np.zeros((pages.pages, p), np.float32)
    k.reshape(-1)[:] = score(t)
    pages.k = to_bits(np.zeros(shape, np.float32), dtype)
    pages.k[..., 0] = to_bits(k, dtype)[:, None]
    v = (np.abs(rng.standard_normal(shape)) + 0.5).astype(np.float32) * np.asarray(value(t), np.float32).reshape(pages.pages, 1, p, 1)
    pages.v = to_bits(v, dtype)
    pages.table = np.arange(pages.pages, dtype=np.int32)[None]
    s = to_f64(pages.k[:, 0, :, 0], dtype).reshape(-1)[:n]
    e = np.exp(s - s.max())
    e /= e.sum()
    values = to_f64(pages.v, dtype).transpose(1, 0, 2, 3).reshape(h, -1, d)[:, :n]                  # [h, n, d]
    out = np.repeat(np.stack([e @ values[g] for g in range(h)]), hq // h, axis=0)[None, None]
    near = Near(out, np.abs(out), np.full((1, 1, hq), np.abs(s).max()), np.full((1, 1, hq), float(n)))      # (values of one sign: their sum is the sum of their magnitudes)
    drawn = np.zeros((1, h, pages.capacity))
    drawn[..., :n] = e * (hq // h)
    return pages, near, drawn


@pytest.mark.parametrize("dtype", [be.F16, be.BF16])
@pytest.mark.parametrize("hq, h, d", [(4, 2, 64), (8, 2, 128), (8, 1, 256), (2, 1, 72)])
@pytest.mark.parametrize("gap", [0.5, 18.0, 21.25, 22.0, 40.0, 61.0])
def test_one_dominant_key_whose_value_is_zero(gpu, dtype, hq, h, d, gap):
    """100001 equal keys `gap` nats below one whose value is nothing: the answer is theirs alone (a sink in front of a long text). Where the gap is 61, a key's share is 2^-88."""
    n = 100001 if d != 72 else 3001
    for sink in (0, n - 40):
        pages, near, drawn = peaked(np.random.default_rng(d), dtype, n, hq, h, d, lambda t: np.where(t == sink, gap, 0.0), lambda t: t != sink)
        for q_dtype in (be.F32, dtype):
            q = np.zeros((1, 1, hq, d), np.float32)
            q[..., 0] = 1.0
            got, weights = attend(gpu, pages, to_bits(q, q_dtype), q_dtype, 1.0, lengths=[n])
            assert near.close(got).all(), (sink, np.abs(got / near.out - 1).max())
            assert near.weights_close(weights, drawn, hq // h).all()


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("score", ["steps", "saw", "falling", "rising", "islands"])
def test_tiles_far_apart(gpu, d, score):
    """scores whose tiles lie up to 100 nats apart, back and forth; keys near the top have no value, so that those far below are the answer"""
    n = 5003
    shape = {"steps": lambda t: -16.0 * (t // 32 % 7), "saw": lambda t: -(t % 640) / 8.0, "falling": lambda t: -t / 50.0, "rising": lambda t: t / 50.0,
             "islands": lambda t: np.where(t % 97 == 5, 0.0, -30.0 - t % 3)}[score]
    top = max(shape(np.arange(n)))
    pages, near, drawn = peaked(np.random.default_rng(1), be.F16, n, 8, 2, d, shape, lambda t: shape(t) < top - 10.0)
    q = np.zeros((1, 1, 8, d), np.float32)
    q[..., 0] = 1.0
    got, weights = attend(gpu, pages, q, be.F32, 1.0, lengths=[n])
    # Where the top is in a tile of 32 keys with those far below it: a probability is a pair of f16 that ends at 2^-24, half a step of which is off, and its tile's largest is held as 2^6 at
    # least: 2^-31 of that a key.
    largest = np.pad(drawn[0, 0, :n] / 4, (0, -n % 32)).reshape(-1, 32).max(axis=1).repeat(32)[:n]
    off = np.repeat(np.stack([largest @ np.abs(to_f64(pages.v, be.F16).transpose(1, 0, 2, 3).reshape(2, -1, d)[g, :n]) for g in range(2)]), 4, axis=0)[None, None] * 2.0 ** -31
    assert near.close(near.out + np.maximum(np.abs(got - near.out) - off, 0.0)).all(), np.abs(got / near.out - 1).max()
    assert near.weights_close(weights, drawn, 4).all()


@pytest.mark.parametrize("hq, h, d", [(4, 2, 64), (8, 2, 128), (8, 1, 256), (2, 1, 72)])
@pytest.mark.parametrize("n", [1, 20, 3001])
@pytest.mark.parametrize("size", [100, 112, 120])
def test_values_past_the_range_of_f16(gpu, hq, h, d, n, size):
    """values of 2^size: their sum over the keys is far past f32's range before it is divided by that of the probabilities where a key counts for 2^15 or one"""
    if n > 1000 and size > 112:
        n = 200
    pages, near, drawn = peaked(np.random.default_rng(d), be.BF16, n, hq, h, d, lambda t: t % 5 * 0.5, lambda t: np.full(t.size, 2.0 ** size))
    q = np.zeros((1, 1, hq, d), np.float32)
    q[..., 0] = 1.0
    got, weights = attend(gpu, pages, q, be.F32, 1.0, lengths=[n])
    assert near.close(got).all() and near.weights_close(weights, drawn, hq // h).all()


@pytest.mark.parametrize("dtype", [be.F16, be.BF16])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_sums_keep_their_size_while_the_reference_moves(gpu, dtype, d):
    """Two keys of equal score and opposite values, at either end of a text whose tiles lie ten powers of two and more apart in turn: each wavefront's sums are brought to another reference up to a
    thousand times in between, and the answer is zero as long as that loses nothing. Each probability is off by 2^-23 (exp2) and 2^-22 (its halves) at most, and by 2^-23 in each of two meetings: 2^-20."""
    b, n = 1024, 131072 if d < 256 else 65536
    rng = np.random.default_rng(0)
    high, low = -16.5 + 3 * rng.random(n // 128), -23.5 - 8 * rng.random(n // 128)
    level = np.where(np.arange(n // 128) % 2 == 1, high, low)
    pages, _, _ = peaked(rng, dtype, n, 1, 1, d, lambda t: np.where((t == 0) | (t == n - 1), 0.0, level[t // 128]), lambda t: np.zeros(t.size))
    pages.v[0, 0, 0], pages.v[-1, 0, -1] = to_bits(np.array([1.0, -1.0], np.float32), dtype)
    pages.b, pages.table = b, np.repeat(pages.table, b, axis=0)
    q = np.zeros((b, 1, 1, d), np.float32)
    q[..., 0] = 1.0
    got, _ = attend(gpu, pages, q, be.F32, 1.0, lengths=[n] * b, weigh=False)
    launch = gpu.last_launch()
    assert launch["grid"][0] == 1 and n // 32 // (launch["block"][0] // 64) >= 256                     # (one segment)
    assert np.abs(got).max() <= 2.0 ** -20, np.abs(got).max()
