"""Caches in pages: rows turned, written, read back, attended to and evicted, through the C ABI, against numpy in 64 bits."""
import numpy as np
import pytest

from aion_amd import backend as be
from paged_cases import Pages, attention, evict, free, staying, storage, to_bits, to_f64, turned, turned_close

pytestmark = pytest.mark.gpu

TYPES = [be.F16, be.BF16]


def source(rng, shape, dtype):
    """what is uploaded, and its values"""
    x = to_bits((rng.standard_normal(shape) * np.exp(0.5 * rng.standard_normal(shape[-1]))).astype(np.float32), dtype)
    return x, to_f64(x, dtype)


# ---------------------------------------------------------------------------------------------------------------- append and read
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("b,s,width,p,h,d,starts,src", [
    (1, 1, 1, 16, 1, 8, [0], be.F32),
    (1, 1, 4, 64, 8, 128, [255], be.F32),
    (3, 5, 3, 16, 2, 64, [14, 0, 43], be.F16),
    (2, 130, 5, 32, 3, 72, [20, 3], be.BF16),
    (3, 9, 4, 16, 2, 256, [60, -4, 70], be.F32),                 # past the end, before the beginning, wholly outside
    (2, 64, 1, 1024, 2, 1024, [1000, 0], be.F16),
    (65, 1, 2, 16, 5, 40, [i % 33 for i in range(65)], be.F32),
    (2, 600, 40, 16, 1, 128, [3, 2147483647], be.F32),
])
def test_append_and_read(gpu, dtype, b, s, width, p, h, d, starts, src):
    rng = np.random.default_rng(b * 100 + s + d)
    pages = Pages(rng, dtype, b, width, p, h, d)
    if width > 2:
        pages.table[0, 1], pages.table[-1, 2] = -1, pages.pages          # no pages
    (kb, k), (vb, v) = (source(rng, (b, s, h, d), src) for _ in range(2))
    cache, at = pages.upload(gpu), gpu.upload(np.array(starts, np.int32))
    kd, vd = gpu.upload(kb), gpu.upload(vb)
    gpu.step_append_paged(cache, kd, vd, at, s, src_dtype=src)
    for i in range(b):
        for j in range(s):
            pages.put(0, i, starts[i] + j, k[i, j])
            pages.put(1, i, starts[i] + j, v[i, j])
    assert pages.same(gpu, cache)                                        # untouched rows as they were
    for out in (be.F32, be.F16, be.BF16):
        size = b * s * h * d * np.dtype(storage(out)).itemsize
        ko, vo = gpu.alloc(size), gpu.alloc(size)
        gpu.step_read_paged(cache, ko, vo, at, s, out_dtype=out)
        for which, buf in ((0, ko), (1, vo)):
            want = np.stack([pages.rows(which, i, range(starts[i], starts[i] + s))[0] for i in range(b)])
            assert np.array_equal(gpu.download(buf, storage(out), (b, s, h, d)), to_bits(want, out))
        ko.free(), vo.free()
    assert pages.same(gpu, cache)
    free(cache, at, kd, vd)


def test_a_page_of_two_sequences_is_read_by_both(gpu):
    rng = np.random.default_rng(5)
    pages = Pages(rng, be.F16, 3, 3, 16, 2, 64)
    pages.table[1, 0] = pages.table[2, 0] = pages.table[0, 0]
    cache, lengths = pages.upload(gpu), np.array([20, 33, 10], np.int32)
    q = rng.standard_normal((3, 1, 4, 64)).astype(np.float32)
    out, qd, ld = gpu.alloc(q.nbytes), gpu.upload(q), gpu.upload(lengths)
    gpu.step_attention_paged(out, qd, cache, 1, 4, 0.125, kv_lengths=ld)
    near, _ = attention(q.astype(np.float64), pages, 1, 4, 0.125, lengths=lengths)
    assert near.close(gpu.download(out, np.float32, q.shape)).all()
    free(cache, out, qd, ld)


# ---------------------------------------------------------------------------------------------------------------- turned by positions
TURNS = [
    dict(dims=64), dict(dims=64, interleaved=True, base=500000.0),
    dict(dims=48, scaling=be.ROTARY_LINEAR, factor=4.0), dict(dims=64, scaling=be.ROTARY_BANDS, base=500000.0, factor=8.0, original_length=8192.0, low=1.0, high=4.0),
    dict(dims=64, interleaved=True, scaling=be.ROTARY_RAMP, factor=16.0, original_length=4096.0, low=1.0, high=32.0, magnitude=1.25), dict(dims=0), dict(dims=2, magnitude=-0.5),
    dict(dims=6, interleaved=True, base=0.5), dict(dims=34, base=1.0), dict(dims=62, interleaved=True, base=10000.0, magnitude=0.0),
]


@pytest.mark.parametrize("dtype", [be.F32, be.F16, be.BF16])
@pytest.mark.parametrize("turn", range(len(TURNS)))
def test_rotary(gpu, dtype, turn):
    r = be.Rotary(**TURNS[turn])
    rng = np.random.default_rng(turn)
    for b, t, h, d, at in [(1, 1, 1, 64, 0), (2, 7, 5, 64, 1000000), (3, 1, 33, 66, -5), (1, 1100, 3, 64, 2147480000), (1, 5, 2, 512, 77), (2, 3, 2, 1024, 9), (2, 600, 9, 70, 131071)]:
        xb, x = source(rng, (b, t, h, d), dtype)
        positions = (at + np.arange(t)[None] + 13 * np.arange(b)[:, None]).astype(np.int32)
        xd, pd, out = gpu.upload(xb), gpu.upload(positions), gpu.alloc(xb.nbytes)
        gpu.step_rotary(out, xd, pd, b, t, h, d, r, dtype=dtype)
        bits = gpu.download(out, storage(dtype), x.shape)
        assert turned_close(to_f64(bits, dtype), x, positions, r, dtype).all(), (b, t, h, d)
        assert np.array_equal(bits[..., r.dims:], xb[..., r.dims:])
        gpu.step_rotary(xd, xd, pd, b, t, h, d, r, dtype=dtype)          # in place: the same bits
        assert np.array_equal(gpu.download(xd, storage(dtype), x.shape), bits)
        for buf in (xd, pd, out):
            buf.free()


def test_rotary_turns_what_is_not_finite_into_its_pair_alone(gpu):
    x = np.ones((1, 1, 1, 16), np.float32)
    x[..., 3], x[..., 9] = np.nan, np.inf
    for interleaved, hit in ((False, {3, 7, 9}), (True, {2, 3, 9})):
        buf, pos = gpu.upload(x), gpu.upload(np.array([3], np.int32))
        gpu.step_rotary(buf, buf, pos, 1, 1, 1, 16, be.Rotary(8, interleaved=interleaved))
        y = gpu.download(buf, np.float32, (16,))
        assert {i for i in range(16) if not np.isfinite(y[i])} == hit
        buf.free(), pos.free()


@pytest.mark.parametrize("dtype", [be.F32, be.F16, be.BF16])
@pytest.mark.parametrize("cache_dtype", TYPES)
@pytest.mark.parametrize("b,s,width,p,hq,h,d,turn", [(1, 1, 3, 16, 8, 1, 256, 0), (2, 1500, 50, 32, 4, 2, 64, 1), (64, 1, 2, 16, 8, 8, 64, 2), (1, 9, 1, 64, 32, 8, 128, 3), (3, 40, 4, 16, 3, 3, 72, 4)])
def test_rotary_append(gpu, dtype, cache_dtype, b, s, width, p, hq, h, d, turn):
    """q to the bits of the step alone; keys rounded once from the turned f32 value, values from what came in; the rest of the cache as it was"""
    r = be.Rotary(**TURNS[turn])
    rng = np.random.default_rng(d + s)
    pages = Pages(rng, cache_dtype, b, width, p, h, d)
    (qb, q), (kb, k), (vb, v) = source(rng, (b, s, hq, d), dtype), source(rng, (b, s, h, d), dtype), source(rng, (b, s, h, d), dtype)
    positions = (4000 + np.arange(s)[None] + 1000 * np.arange(b)[:, None]).astype(np.int32)
    starts = np.array([i % (width * p - s + 1) for i in range(b)], np.int32)
    cache = pages.upload(gpu)
    qd, kd, vd, pd, at = (gpu.upload(x) for x in (qb, kb, vb, positions, starts))
    alone, out = gpu.alloc(qb.nbytes), gpu.alloc(qb.nbytes)
    gpu.step_rotary(alone, qd, pd, b, s, hq, d, r, dtype=dtype)
    gpu.step_rotary_append_paged(cache, r, out, qd, kd, vd, pd, at, s, hq, dtype=dtype)
    assert np.array_equal(gpu.download(out, storage(dtype), q.shape), gpu.download(alone, storage(dtype), q.shape))
    got = gpu.download(cache.k_pages, storage(cache_dtype), pages.k.shape)
    rows = np.zeros((b, s, h, d), got.dtype)
    for i in range(b):
        for j in range(s):
            t = starts[i] + j
            rows[i, j] = got[pages.page(i, t), :, t % p]
            pages.k[pages.page(i, t), :, t % p] = rows[i, j]
            pages.put(1, i, t, v[i, j])
    assert turned_close(to_f64(rows, cache_dtype), k, positions, r, cache_dtype).all()
    assert pages.same(gpu, cache)
    gpu.step_rotary_append_paged(cache, r, qd, qd, kd, vd, pd, at, s, hq, dtype=dtype)          # q in place
    assert np.array_equal(gpu.download(qd, storage(dtype), q.shape), gpu.download(alone, storage(dtype), q.shape))
    free(cache, qd, kd, vd, pd, at, alone, out)


# ---------------------------------------------------------------------------------------------------------------- attention
def attend(gpu, pages, q, q_dtype, scale, lengths=None, positions=None, window=be.CAUSAL, soft_cap=0.0, weigh=True, before=None, cache=None):
    b, l, hq, d = q.shape
    own = cache is None
    cache = cache or pages.upload(gpu)
    qd, out = gpu.upload(q), gpu.upload(np.full((b, l, hq, d), np.nan, np.float32))
    ld = gpu.upload(np.asarray(lengths, np.int32)) if lengths is not None else None
    pd = gpu.upload(np.asarray(positions, np.int32)) if positions is not None else None
    w = gpu.upload(np.full((b, pages.h, pages.capacity), np.nan, np.float32)) if weigh else None
    bd = gpu.upload(before) if before is not None else None
    gpu.step_attention_paged(out, qd, cache, l, hq, scale, q_dtype=q_dtype, window=window, soft_cap=soft_cap, query_positions=pd, kv_lengths=ld, weights=w, weights_before=bd)
    got = gpu.download(out, np.float32, (b, l, hq, d))
    drawn = gpu.download(w, np.float32, (b, pages.h, pages.capacity)) if weigh else None
    for buf in (qd, out, ld, pd, w, bd):
        if buf is not None:
            buf.free()
    if own:
        free(cache)
    return got, drawn


def check(gpu, pages, q_bits, q, q_dtype, scale, **kw):
    near, drawn = attention(q, pages, q.shape[1], q.shape[2], scale, **{x: kw[x] for x in kw if x in ("window", "soft_cap", "positions", "lengths")})
    plain, _ = attend(gpu, pages, q_bits, q_dtype, scale, weigh=False, **kw)
    got, weights = attend(gpu, pages, q_bits, q_dtype, scale, **kw)
    assert near.close(plain).all(), np.nanmax(np.abs(plain - near.out))
    assert near.close(got).all(), np.nanmax(np.abs(got - near.out))
    assert near.weights_close(weights, drawn, q.shape[1] * q.shape[2] // pages.h).all(), np.nanmax(np.abs(weights - drawn))
    return got


SHAPES = [  # b, l, hq, h, d, width, p, lengths
    (1, 1, 8, 1, 256, 1, 16, [1]), (1, 1, 8, 1, 256, 40, 16, [531]), (2, 1, 32, 8, 128, 5, 64, [300, 17]), (3, 1, 16, 4, 64, 3, 128, [384, 0, 33]),
    (1, 1, 32, 32, 128, 2, 1024, [2048]), (4, 5, 4, 4, 128, 7, 32, [224, 5, 100, 3]), (2, 8, 8, 2, 256, 9, 32, [200, 288]), (1, 40, 16, 4, 64, 9, 16, [133]),
    (2, 1, 6, 3, 96, 9, 16, [131, 64]), (1, 3, 2, 1, 8, 3, 16, [48]), (1, 1, 2, 2, 1024, 5, 16, [70]), (1, 1, 1, 1, 64, 300, 16, [4800]), (70, 1, 8, 2, 64, 2, 32, list(range(70))),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("q_dtype", [be.F32, be.F16, be.BF16])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_attention(gpu, dtype, q_dtype, shape):
    b, l, hq, h, d, width, p, lengths = SHAPES[shape]
    rng = np.random.default_rng(shape)
    pages = Pages(rng, dtype, b, width, p, h, d)
    for i in range(b):
        pages.table[i, -(-lengths[i] // p):] = -1                        # nothing behind the last row's page
    bits, q = source(rng, (b, l, hq, d), q_dtype)
    check(gpu, pages, bits, q, q_dtype, d ** -0.5, lengths=lengths)


@pytest.mark.parametrize("d", [64, 128, 256, 80])
@pytest.mark.parametrize("window,soft_cap,positions", [
    ((63, 0, 0), 0.0, None), ((5, 0, 0), 30.0, None), ((be.UNBOUNDED, be.UNBOUNDED, 0), 0.0, None), ((0, 0, 0), 0.0, None), ((16, 3, 32), 5.0, None),
    (be.CAUSAL, 0.0, [[0, 5, 300], [-3, 100, 1000]]), ((20, 0, 0), 0.0, [[250, 7, 100], [900, 0, 60]]), ((0, 2, 16), 0.0, [[17, 40, 1], [3, 3, 3]]),
])
def test_attention_windows(gpu, d, window, soft_cap, positions):
    rng = np.random.default_rng(d)
    pages = Pages(rng, be.F16, 2, 17, 16, 2, d)
    bits, q = source(rng, (2, 3, 6, d), be.F32)
    check(gpu, pages, bits, q, be.F32, d ** -0.5, lengths=[272, 95], window=window, soft_cap=soft_cap, positions=positions)


def test_attention_takes_the_whole_capacity_without_lengths(gpu):
    rng = np.random.default_rng(0)
    pages = Pages(rng, be.BF16, 2, 5, 16, 2, 128)
    bits, q = source(rng, (2, 2, 4, 128), be.F32)
    check(gpu, pages, bits, q, be.F32, 0.1)
    check(gpu, pages, bits, q, be.F32, 0.1, lengths=[1000, -7])
    check(gpu, pages, bits, q, be.F32, -0.3, lengths=[79, 40])           # any scale
    check(gpu, pages, bits, q, be.F32, 0.0, lengths=[79, 40])


@pytest.mark.parametrize("d", [64, 128, 256, 40])
@pytest.mark.parametrize("dtype", TYPES)
def test_what_lies_behind_the_last_row_or_on_no_page_is_not_looked_at(gpu, d, dtype):
    rng = np.random.default_rng(d)
    pages = Pages(rng, dtype, 3, 6, 16, 2, d)
    lengths = [75, 33, 1]
    pages.table[0, 2], pages.table[1, 0] = -1, 1 << 30                   # a hole in the middle, one at the beginning
    odd = {be.F16: [0x7E00, 0x7C00, 0xFC00], be.BF16: [0x7FC0, 0x7F80, 0xFF80]}[dtype]
    seen = {(pages.page(i, t), t % 16) for i in range(3) for t in range(lengths[i])}
    for pool in (pages.k, pages.v):
        raw = pool.view(np.uint16)
        for page in range(pages.pages):
            for row in range(16):
                if (page, row) not in seen:
                    raw[page, :, row] = np.random.default_rng(page).choice(odd, raw[page, :, row].shape)
    bits, q = source(rng, (3, 2, 4, d), be.F32)
    check(gpu, pages, bits, q, be.F32, d ** -0.5, lengths=lengths)


@pytest.mark.parametrize("d", [64, 128, 256, 40])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
def test_a_value_that_is_not_finite_reaches_the_queries_that_see_it(gpu, d, dtype, value):
    """five queries at the end of 100 keys; the value of key 97 is odd in one column: queries 2, 3 and 4 see it there, the others nowhere"""
    rng = np.random.default_rng(d)
    pages = Pages(rng, dtype, 1, 7, 16, 1, d)
    bits, q = source(rng, (1, 5, 3, d), be.F32)
    near, drawn = attention(q, pages, 5, 3, d ** -0.5, lengths=[100])
    pages.v[pages.page(0, 97), 0, 97 % 16, 5] = to_bits(np.array([value], np.float32), dtype)[0]
    got, weights = attend(gpu, pages, bits, be.F32, d ** -0.5, lengths=[100])
    hit = np.zeros(got.shape, bool)
    hit[:, 2:, :, 5] = True
    assert not np.isfinite(got[hit]).any()
    assert np.array_equal(got[hit], np.full(hit.sum(), value, np.float32), equal_nan=True)
    near.out[hit] = got[hit] = 0.0
    assert near.close(got).all() and near.weights_close(weights, drawn, 15).all()
    # a key that is no number: the queries that see it have no answer
    pages.k[pages.page(0, 98), 0, 98 % 16, 1] = to_bits(np.array([np.nan], np.float32), dtype)[0]
    got, weights = attend(gpu, pages, bits, be.F32, d ** -0.5, lengths=[100])
    assert np.isnan(got[:, 3:]).all() and np.isfinite(got[:, :2]).all() and np.isnan(weights[0, 0, :99]).all() and not np.isnan(weights[0, 0, 100:]).any()


@pytest.mark.parametrize("d", [64, 128, 256, 40])
def test_scores_of_minus_infinity_and_queries_out_of_range(gpu, d):
    rng = np.random.default_rng(d)
    pages = Pages(rng, be.F16, 1, 6, 16, 1, d)
    pages.k[:] = np.abs(pages.k)
    pages.k[..., 0] = 1.0
    q = np.zeros((1, 3, 2, d), np.float32)
    q[0, 0, :, 0] = -np.inf                                              # every score minus infinity (the other products are zeros): zeros
    q[0, 1, :, 0] = np.inf                                               # plus infinity: no number
    q[0, 2] = rng.standard_normal((2, d))
    with np.errstate(invalid="ignore"):
        near, _ = attention(q[:, 2:].astype(np.float64), pages, 1, 2, 0.125, lengths=[90])
    got, _ = attend(gpu, pages, q, be.F32, 0.125, lengths=[90], positions=[[89, 89, 89]])
    assert (got[0, 0] == 0).all() and np.isnan(got[0, 1]).all() and near.close(got[:, 2:]).all()
    # queries far past f16's range, and far below it
    for size in (1e9, 1e-9, 1e30):
        x = (rng.standard_normal((1, 1, 2, d)) * size).astype(np.float32)
        near, _ = attention(x.astype(np.float64), pages, 1, 2, 1.0 / size, lengths=[90])
        got, _ = attend(gpu, pages, x, be.F32, 1.0 / size, lengths=[90])
        assert near.close(got).all()


def test_a_late_key_of_far_greater_score_and_scores_far_apart(gpu):
    """the reference moves up in steps; what lies 2^-100 below the largest vanishes, and nothing else does"""
    rng = np.random.default_rng(3)
    for d in (64, 128, 256, 40):
        pages = Pages(rng, be.F16, 1, 70, 16, 1, d)
        pages.k[:] = 0
        ramp = np.linspace(-40, 40, 1100)
        for t in range(1100):
            pages.k[pages.page(0, t), 0, t % 16, 0] = ramp[t]
        q = np.zeros((1, 1, 1, d), np.float32)
        for x in (1.0, -1.0, 0.2, 3.0):
            q[..., 0] = x
            near, drawn = attention(q.astype(np.float64), pages, 1, 1, 1.0, lengths=[1100])
            got, weights = attend(gpu, pages, q, be.F32, 1.0, lengths=[1100])
            assert near.close(got).all() and near.weights_close(weights, drawn, 1).all()


def test_weights_are_added_to_those_before(gpu):
    rng = np.random.default_rng(8)
    pages = Pages(rng, be.F16, 2, 5, 32, 2, 64)
    bits, q = source(rng, (2, 3, 8, 64), be.F32)
    before = rng.standard_normal((2, 2, 160)).astype(np.float32)
    near, drawn = attention(q, pages, 3, 8, 0.125, lengths=[150, 20])
    _, alone = attend(gpu, pages, bits, be.F32, 0.125, lengths=[150, 20])
    _, got = attend(gpu, pages, bits, be.F32, 0.125, lengths=[150, 20], before=before)
    assert np.array_equal(got, before + alone)
    cache, qd, out, w, ld = pages.upload(gpu), gpu.upload(bits), gpu.alloc(bits.nbytes), gpu.upload(before), gpu.upload(np.array([150, 20], np.int32))
    for i in range(3):                                                   # in place, step after step
        gpu.step_attention_paged(out, qd, cache, 3, 8, 0.125, kv_lengths=ld, weights=w, weights_before=w)
    want = before
    for i in range(3):
        want = want + alone
    assert np.array_equal(gpu.download(w, np.float32, before.shape), want)
    free(cache, qd, out, w, ld)


# ---------------------------------------------------------------------------------------------------------------- eviction
EVICTIONS = [  # dtype, b, width, p, h, d, lengths, limit, keep, first, recent
    (be.F16, 1, 4, 16, 1, 64, [64], 16, 16, 0, 0), (be.F16, 3, 9, 16, 2, 128, [144, 40, 100], 64, 50, 4, 10), (be.BF16, 2, 5, 32, 3, 72, [160, 0], 160, 8, 4, 4),
    (be.BF16, 2, 3, 64, 8, 256, [192, 191], 190, 190, 0, 190), (be.F16, 1, 2, 1024, 1, 8, [2000], 1500, 1, 0, 0), (be.F16, 2, 20, 16, 2, 1024, [300, 299], 299, 0, 0, 0),
    (be.F16, 1, 300, 16, 2, 64, [4711], 3000, 2900, 100, 700), (be.BF16, 5, 2, 16, 1, 128, [-1, 0, 1, 32, 99], 8, 8, 8, 0), (be.F16, 1, 5, 16, 1, 64, [80], 5000, 8, 0, 0),
    (be.F16, 1, 5, 16, 1, 64, [80], 0, 0, 0, 0),
]


def weigh(rng, shape, kind):
    w = np.exp(2 * rng.standard_normal(shape)).astype(np.float32)
    if kind == "ties":
        w = np.round(w).astype(np.float32)
        w[w == 0] = np.where(rng.integers(0, 2, (w == 0).sum()) == 0, np.float32(0.0), np.float32(-0.0))
    if kind == "odd":
        w = np.where(rng.random(shape) < 0.2, rng.choice(np.array([np.nan, -np.nan, np.inf, -np.inf, -1.0, 1e-42, -1e-42, 0.0, -0.0], np.float32), shape), w).astype(np.float32)
    if kind == "alike":
        w[:] = 0.25
    return w


@pytest.mark.parametrize("kind", ["plain", "ties", "odd", "alike"])
@pytest.mark.parametrize("case", range(len(EVICTIONS)))
@pytest.mark.parametrize("in_place", [True, False])
def test_evict(gpu, case, kind, in_place):
    dtype, b, width, p, h, d, lengths, limit, keep, first, recent = EVICTIONS[case]
    rng = np.random.default_rng(case)
    width_out = 0 if in_place else -(-limit // p) + case % 2 or 1
    pages = Pages(rng, dtype, b, width, p, h, d, spare=b * width_out + 2)
    if width > 4 and limit:
        pages.table[0, 1] = -1                                           # rows that are on no page stay behind
    rest = np.setdiff1d(np.arange(pages.pages), pages.table)
    table_out = None if in_place else rng.permutation(rest)[:b * width_out].reshape(b, width_out).astype(np.int32)
    weights, cap_out = weigh(rng, (b, h, width * p), kind), (width if in_place else width_out) * p
    cache, wd, ld = pages.upload(gpu), gpu.upload(weights), gpu.upload(np.array(lengths, np.int32))
    td = None if in_place else gpu.upload(table_out)
    wo, lo, kept = gpu.alloc(max(b * h * cap_out * 4, 4)), gpu.alloc(4 * b), gpu.alloc(max(b * h * limit * 4, 4))
    if in_place:
        gpu.copy(wo, wd, weights.nbytes)
    gpu.step_evict_paged(cache, wo if in_place else wd, ld, wo, lo, keep, limit=limit, first=first, recent=recent, table_out=td, width_out=width_out, kept=kept)
    want_kept, want_len, want_w = evict(pages, weights, lengths, limit, keep, first, recent, table_out)
    assert np.array_equal(gpu.download(kept, np.int32, (b, h, limit)), want_kept)
    assert np.array_equal(gpu.download(lo, np.int32, (b,)), want_len)
    assert np.array_equal(gpu.download(wo, np.float32, (b, h, cap_out)), want_w, equal_nan=True)
    assert pages.same(gpu, cache)
    if in_place:                                                         # what the library keeps the list in itself, lengths over themselves: nothing is over the limit any more
        assert not (want_len > limit).any()
        gpu.step_evict_paged(cache, wo, lo, wo, lo, keep, limit=limit, first=first, recent=recent)
        assert np.array_equal(gpu.download(lo, np.int32, (b,)), want_len) and pages.same(gpu, cache)
        assert np.array_equal(gpu.download(wo, np.float32, (b, h, cap_out)), want_w, equal_nan=True)
    else:
        assert np.array_equal(gpu.download(wd, np.float32, weights.shape), weights, equal_nan=True)
    free(cache, wd, ld, wo, lo, kept, *([] if in_place else [td]))


def test_evict_long(gpu):
    """past a workgroup's worth of everything: 70001 rows of one head"""
    rng = np.random.default_rng(0)
    pages = Pages(rng, be.F16, 1, 1100, 64, 1, 64, sigma=1.0)
    weights = weigh(rng, (1, 1, 70400), "ties")
    cache, wd, ld = pages.upload(gpu), gpu.upload(weights), gpu.upload(np.array([70001], np.int32))
    gpu.step_evict_paged(cache, wd, ld, wd, ld, 20011, first=3, recent=7000)
    _, want_len, want_w = evict(pages, weights, [70001], 20011, 20011, 3, 7000)
    assert np.array_equal(gpu.download(ld, np.int32, (1,)), want_len) and np.array_equal(gpu.download(wd, np.float32, weights.shape), want_w)
    assert pages.same(gpu, cache)
    free(cache, wd, ld)


def test_evict_in_place_a_part_of_the_heads_at_a_time(gpu):
    """rows that take more than the memory between holds at once: 20 heads of 4096 rows of 4 KiB"""
    rng = np.random.default_rng(2)
    pages = Pages(rng, be.F16, 2, 1, 16, 10, 1024)
    pages.p, pages.width, pages.pages = 64, 66, 133
    pages.k = np.arange(133 * 10 * 64 * 1024, dtype=np.uint32).astype(np.uint16).reshape(133, 10, 64, 1024)
    pages.k ^= np.arange(133 * 10 * 64, dtype=np.uint32).astype(np.uint16).reshape(133, 10, 64, 1)
    pages.v = pages.k[::-1].copy()
    pages.table = rng.permutation(133)[:132].reshape(2, 66).astype(np.int32)
    weights = weigh(rng, (2, 10, 66 * 64), "plain")
    cache, wd, ld = pages.upload(gpu), gpu.upload(weights), gpu.upload(np.array([4200, 4224], np.int32))
    gpu.step_evict_paged(cache, wd, ld, wd, ld, 4096, first=1, recent=100)
    _, want_len, want_w = evict(pages, weights, [4200, 4224], 4096, 4096, 1, 100)
    assert np.array_equal(gpu.download(ld, np.int32, (2,)), want_len) and np.array_equal(gpu.download(wd, np.float32, weights.shape), want_w)
    for buf, want in ((cache.k_pages, pages.k), (cache.v_pages, pages.v)):
        assert np.array_equal(gpu.download(buf, np.uint16, want.shape), want)
    free(cache, wd, ld)


# ---------------------------------------------------------------------------------------------------------------- together
def steps_together(gpu, record):
    """Tokens appended, attended to with weights kept, evicted in place every time a sequence passes its limit; against numpy at every step."""
    rng = np.random.default_rng(12)
    b, hq, h, d, p, width, limit, keep = 3, 8, 2, 64, 16, 4, 40, 24
    r = be.Rotary(32, base=500000.0, interleaved=True)
    pages = Pages(rng, be.F16, b, width, p, h, d)
    cache = pages.upload(gpu)
    lengths = np.array([37, 5, 39], np.int32)
    weights = np.abs(rng.standard_normal((b, h, width * p))).astype(np.float32)
    for i in range(b):
        weights[i, :, lengths[i]:] = 0
    positions = (lengths + 100000).astype(np.int32)
    one = gpu.upload(np.ones(b, np.int32))
    bufs = {"q": gpu.alloc(b * hq * d * 4), "k": gpu.alloc(b * h * d * 4), "v": gpu.alloc(b * h * d * 4), "out": gpu.alloc(b * hq * d * 4), "qr": gpu.alloc(b * hq * d * 4),
            "len": gpu.upload(lengths), "at": gpu.upload(lengths), "pos": gpu.upload(positions), "w": gpu.upload(weights)}

    def issue():
        gpu.step_rotary_append_paged(cache, r, bufs["qr"], bufs["q"], bufs["k"], bufs["v"], bufs["pos"], bufs["at"], 1, hq)
        gpu.step_add_i32(bufs["len"], bufs["len"], one, b)
        gpu.step_attention_paged(bufs["out"], bufs["qr"], cache, 1, hq, 0.125, kv_lengths=bufs["len"], weights=bufs["w"], weights_before=bufs["w"])
        gpu.step_evict_paged(cache, bufs["w"], bufs["len"], bufs["w"], bufs["len"], keep, limit=limit, first=2, recent=8)
        gpu.copy(bufs["at"], bufs["len"], 4 * b)
        gpu.step_add_i32(bufs["pos"], bufs["pos"], one, b)

    def reset():
        for name, x in (("len", lengths), ("at", lengths), ("pos", positions), ("w", weights)):
            gpu.write(bufs[name], x)
        gpu.write(cache.k_pages, start[0])
        gpu.write(cache.v_pages, start[1])

    start = pages.k.copy(), pages.v.copy()
    program = None
    if record:
        issue()                                                          # scratch memory and the table of turns
        gpu.sync()
        reset()
        program = gpu.record_program(issue)
    lens, pos, w = lengths.copy(), positions.copy(), weights.copy()
    cut = 0
    for step in range(30):
        rows = [rng.standard_normal((b, 1, n, d)).astype(np.float32) for n in (hq, h, h)]
        for name, x in zip("qkv", rows):
            gpu.write(bufs[name], x)
        if program is not None:
            gpu.program_execute(program)
        else:
            issue()
        q, _ = turned(rows[0].astype(np.float64), pos[:, None], r)
        k, _ = turned(rows[1].astype(np.float64), pos[:, None], r)
        got_q = gpu.download(bufs["qr"], np.float32, (b, 1, hq, d))
        assert turned_close(got_q, rows[0].astype(np.float64), pos[:, None], r, be.F32).all()
        before = pages.k.copy()
        for i in range(b):
            pages.put(0, i, lens[i], k[i, 0])
            pages.put(1, i, lens[i], rows[2][i, 0])
        lens += 1
        got_w = gpu.download(bufs["w"], np.float32, w.shape)
        near, drawn = attention(got_q.astype(np.float64), pages, 1, hq, 0.125, lengths=lens)
        got = gpu.download(bufs["out"], np.float32, (b, 1, hq, d))
        # (the host's keys may differ from the device's by an f16 step where the turned value lies beside a half: 2^-10 of a key's share of a score)
        assert np.abs(got - near.out).max() <= 2e-3
        # from here on with the device's own keys: the eviction is exact on its own weights
        after = np.array(lens)
        want_w = w + drawn
        full = lens > limit
        cut += full.sum()
        new = np.where(full, keep, lens)
        assert np.array_equal(gpu.download(bufs["len"], np.int32, (b,)), new)
        for i in range(b):
            if not full[i]:
                assert np.abs(got_w[i] - want_w[i]).max() <= 1e-3 * (1 + step)
                continue
            for g in range(h):
                stay = staying(want_w[i, g], after[i], limit, keep, 2, 8)
                assert np.abs(got_w[i, g, :keep] - want_w[i, g, stay]).max() <= 1e-3 * (1 + step)
                assert (got_w[i, g, keep:] == 0).all()
        pages.k = gpu.download(cache.k_pages, np.float16, before.shape)
        pages.v = gpu.download(cache.v_pages, np.float16, before.shape)
        lens, w, pos = new.astype(np.int32), got_w.copy(), pos + 1
    assert cut >= 4
    if program is not None:
        gpu.program_destroy(program)
    free(cache, one, *bufs.values())


def test_steps_together(gpu):
    steps_together(gpu, False)


def test_steps_together_recorded(gpu):
    steps_together(gpu, True)


def test_recorded_programs_give_the_bits_of_the_steps(gpu):
    """two programs of one context, replayed in turn with eager work between them"""
    rng = np.random.default_rng(4)
    made = []
    for b, l, hq, h, d, width, p, lengths in [(2, 1, 8, 2, 128, 20, 32, [600, 33]), (1, 5, 8, 1, 256, 60, 16, [950])]:
        pages = Pages(rng, be.F16, b, width, p, h, d)
        bits, _ = source(rng, (b, l, hq, d), be.F32)
        cache, qd, out, ld, w = pages.upload(gpu), gpu.upload(bits), gpu.alloc(bits.nbytes), gpu.upload(np.array(lengths, np.int32)), gpu.alloc(b * h * width * p * 4)

        def issue(cache=cache, qd=qd, out=out, ld=ld, w=w, l=l, hq=hq):
            gpu.step_attention_paged(out, qd, cache, l, hq, 0.1, kv_lengths=ld, weights=w)
        issue()
        want = gpu.download(out, np.float32, bits.shape), gpu.download(w, np.float32, (b, h, width * p))
        made.append((issue, out, w, want, cache, qd, ld))
    for m in made:
        m[0]()                                                           # the scratch memory is as large as both want it
    programs = [gpu.record_program(m[0]) for m in made]
    for _ in range(3):
        for prog, (issue, out, w, want, *_rest) in zip(programs, made):
            gpu.write(out, np.zeros_like(want[0]))
            gpu.program_execute(prog)
            assert np.array_equal(gpu.download(out, np.float32, want[0].shape), want[0]) and np.array_equal(gpu.download(w, np.float32, want[1].shape), want[1])
            issue()
            gpu.sync()
    for prog in programs:
        gpu.program_destroy(prog)
    for _, out, w, _, cache, qd, ld in made:
        free(cache, out, w, qd, ld)


@pytest.mark.parametrize("p", [16, 1024])
def test_pages_past_32_bits(gpu, p):
    """pools of 5 GiB: the pages of one sequence lie at their end"""
    rng = np.random.default_rng(p)
    h, d = 8, 128
    page = h * p * d * 2
    count = (5 << 30) // page
    small = Pages(rng, be.F16, 1, 2, p, h, d, pages=2)
    kd, vd = gpu.alloc(count * page), gpu.alloc(count * page)
    at = np.array([[count - 1, count - 2]], np.int32)
    for pool, buf in ((small.k, kd), (small.v, vd)):
        for i in range(2):
            gpu.write(buf, pool[small.table[0, i]], offset=int(at[0, i]) * page)
    table = gpu.upload(at)
    cache = gpu.paged_cache(kd, vd, table, count, 1, 2, p, h, d)
    q = rng.standard_normal((1, 1, 16, d)).astype(np.float32)
    n = 2 * p - 3
    qd, out, ld, w = gpu.upload(q), gpu.alloc(q.nbytes), gpu.upload(np.array([n], np.int32)), gpu.alloc(h * 2 * p * 4)
    gpu.step_attention_paged(out, qd, cache, 1, 16, 0.1, kv_lengths=ld, weights=w)
    near, drawn = attention(q.astype(np.float64), small, 1, 16, 0.1, lengths=[n])
    assert near.close(gpu.download(out, np.float32, q.shape)).all()
    row, first = rng.standard_normal((1, 1, h, d)).astype(np.float32), gpu.upload(np.array([n], np.int32))
    rd, back, back2 = gpu.upload(row), gpu.alloc(2 * row.nbytes), gpu.alloc(2 * row.nbytes)
    gpu.step_append_paged(cache, rd, rd, first, 1)
    gpu.step_read_paged(cache, back, back2, first, 2)
    got = gpu.download(back2, np.float32, (2, h, d))
    assert np.array_equal(got[0], row[0, 0].astype(np.float16).astype(np.float32))
    small.put(0, 0, n, row[0, 0]), small.put(1, 0, n, row[0, 0])
    drawn = gpu.download(w, np.float32, (1, h, 2 * p))
    evict(small, drawn, [n], p // 2 + 1, p // 2 + 1, 2, 3)
    gpu.step_evict_paged(cache, w, first, w, first, p // 2 + 1, first=2, recent=3)
    for i in range(2):
        for pool, buf in ((small.k, kd), (small.v, vd)):
            assert np.array_equal(gpu.download(buf, np.float16, (h, p, d), offset=int(at[0, i]) * page), pool[small.table[0, i]])
    free(cache, qd, out, ld, w, first, rd, back, back2)


def test_two_contexts(gpu):
    """another stream with scratch memory of its own: the same bits"""
    rng = np.random.default_rng(21)
    pages = Pages(rng, be.F16, 2, 30, 32, 2, 128)
    bits, _ = source(rng, (2, 1, 8, 128), be.F32)
    want, drawn = attend(gpu, pages, bits, be.F32, 0.1, lengths=[900, 411])
    other = be.HipBackend(0)
    try:
        got, weights = attend(other, pages, bits, be.F32, 0.1, lengths=[900, 411])
        assert np.array_equal(got, want) and np.array_equal(weights, drawn)
    finally:
        other.close()


def test_the_kernels_by_name(gpu):
    rng = np.random.default_rng(1)
    for d, name in ((64, "paged_attn"), (128, "paged_attn"), (256, "paged_attn"), (72, "paged_generic")):
        pages = Pages(rng, be.F16, 1, 2, 16, 1, d)
        bits, _ = source(rng, (1, 1, 2, d), be.F32)
        attend(gpu, pages, bits, be.F32, 0.1, lengths=[20])
        assert gpu.last_kernel() == name


# ---------------------------------------------------------------------------------------------------------------- the ends of the ranges
@pytest.mark.parametrize("d", [64, 72])
def test_weights_of_no_queries_are_those_before(gpu, d):
    rng = np.random.default_rng(12)
    pages = Pages(rng, be.F16, 2, 5, 32, 2, d)
    cache, q, out, ld = pages.upload(gpu), gpu.zeros(64), gpu.zeros(64), gpu.upload(np.array([150, 20], np.int32))
    before = rng.standard_normal((2, 2, 160)).astype(np.float32)
    bd, w = gpu.upload(before), gpu.upload(np.full(before.shape, np.nan, np.float32))
    for given, want in ((bd, before), (None, np.zeros_like(before))):
        gpu.step_attention_paged(out, q, cache, 0, 8, 0.125, kv_lengths=ld, weights=w, weights_before=given)
        assert np.array_equal(gpu.download(w, np.float32, before.shape), want)
    gpu.step_attention_paged(out, q, cache, 0, 8, 0.125, kv_lengths=ld, weights=bd, weights_before=bd)
    assert np.array_equal(gpu.download(bd, np.float32, before.shape), before)
    free(cache, q, out, ld, bd, w)


@pytest.mark.parametrize("hq, hkv, d", [(80, 1, 128), (33, 1, 64), (40, 2, 256)])
def test_more_query_heads_to_a_kv_head_than_a_tile_has_rows(gpu, hq, hkv, d):
    rng = np.random.default_rng(13)
    pages = Pages(rng, be.F16, 2, 9, 32, hkv, d)
    bits, q = source(rng, (2, 1, hq, d), be.F32)
    check(gpu, pages, bits, q, be.F32, d ** -0.5, lengths=[288, 65])


@pytest.mark.parametrize("keep", [7, 2 ** 31 - 65])
def test_a_limit_far_past_the_capacity_cuts_nothing_and_takes_no_memory_for_it(gpu, keep):
    rng = np.random.default_rng(14)
    pages = Pages(rng, be.F16, 2, 5, 16, 2, 64)
    weights = weigh(rng, (2, 2, 80), "plain")
    cache, wd, ld, lo = pages.upload(gpu), gpu.upload(weights), gpu.upload(np.array([80, 99], np.int32)), gpu.alloc(8)
    gpu.step_evict_paged(cache, wd, ld, wd, lo, keep, limit=2 ** 31 - 65, first=1, recent=2)
    assert np.array_equal(gpu.download(lo, np.int32, (2,)), [80, 80]) and np.array_equal(gpu.download(wd, np.float32, weights.shape), weights)
    assert pages.same(gpu, cache)
    free(cache, wd, ld, lo)


@pytest.mark.parametrize("hq, hkv, d, lengths", [(8, 1, 256, [3]), (8, 1, 256, [32]), (8, 1, 256, [33, 700]), (6, 2, 256, [1500, 0, 31]), (4, 4, 256, [2100]), (32, 8, 128, [31]), (32, 8, 128, [1001, 33]),
                                               (2, 1, 128, [5000, 1, 64])])
@pytest.mark.parametrize("l", [1, 3])
@pytest.mark.parametrize("dtype", TYPES)
def test_value_columns_in_shares(gpu, dtype, hq, hkv, d, lengths, l):
    """few workgroups: the columns are dealt out, the weights come from one share of them, and rows that end as no number are walked by each"""
    rng = np.random.default_rng(15)
    pages = Pages(rng, dtype, len(lengths), -(-max(lengths) // 32) + 1, 32, hkv, d)
    bits, q = source(rng, (len(lengths), l, hq, d), be.F32)
    check(gpu, pages, bits, q, be.F32, d ** -0.5, lengths=lengths)
    # an infinite value in one column of the last step but one, which the first of three queries does not see
    near, drawn = attention(q, pages, l, hq, d ** -0.5, lengths=lengths)
    pages.v[pages.page(0, lengths[0] - 2), hkv - 1, (lengths[0] - 2) % 32, d - 70] = to_bits(np.array([np.inf], np.float32), dtype)[0]
    got, weights = attend(gpu, pages, bits, be.F32, d ** -0.5, lengths=lengths)
    hit = np.zeros(got.shape, bool)
    hit[0, max(0, l - 2):, -(hq // hkv):, d - 70] = True
    assert (got[hit] == np.inf).all()
    near.out[hit] = got[hit] = 0.0
    assert near.close(got).all() and near.weights_close(weights, drawn, l * hq // hkv).all()


@pytest.mark.parametrize("d, hq, hkv, width", [(64, 4, 2, 64), (64, 4, 2, 65), (128, 8, 2, 64), (128, 8, 2, 65), (256, 8, 1, 128), (256, 8, 1, 129)])
@pytest.mark.parametrize("apart", [True, False])
def test_weights_within_the_launch_and_in_one_of_their_own(gpu, d, hq, hkv, width, apart):
    """capacities on either side of where a launch of its own adds them up; sequences without keys, entries that are no page, steps nobody sees keep what they had"""
    rng = np.random.default_rng(16)
    pages = Pages(rng, be.F16, 3, width, 32, hkv, d)
    pages.table[0, 3] = -1
    lengths = [width * 32, 0, 70]
    bits, q = source(rng, (3, 2, hq, d), be.F32)
    before = rng.standard_normal((3, hkv, width * 32)).astype(np.float32)
    near, drawn = attention(q, pages, 2, hq, d ** -0.5, lengths=lengths)
    cache, qd, out, ld = pages.upload(gpu), gpu.upload(bits), gpu.alloc(bits.nbytes), gpu.upload(np.array(lengths, np.int32))
    bd = gpu.upload(before)
    w = gpu.upload(np.full(before.shape, np.nan, np.float32)) if apart else bd
    want, size = before.astype(np.float64), np.abs(before).astype(np.float64)
    for _ in range(2):
        gpu.step_attention_paged(out, qd, cache, 2, hq, d ** -0.5, kv_lengths=ld, weights=w, weights_before=bd)
        got = gpu.download(w, np.float32, before.shape)
        want, size = (before + drawn, np.abs(before) + drawn) if apart else (want + drawn, size + drawn)
        assert near.close(gpu.download(out, np.float32, bits.shape)).all()
        # (a rounding for each addition to what was there, and what the weights themselves may be off by)
        bound = 2 * near.reach.max() * (d + 16) * 2.0 ** -24 + 2 * (near.keys.max() / 32 + 64) * 2.0 ** -24 + 2.0 ** -21
        assert (np.abs(got - want) <= 2 * drawn * (np.expm1(bound) + (2 * hq // hkv + 1) * 2.0 ** -24) + 2 * 2.0 ** -24 * size + 1e-37).all()
        assert np.array_equal(got[1], before[1]) and np.array_equal(got[2, :, 70:], before[2, :, 70:]) and np.array_equal(got[0, :, 96:128], before[0, :, 96:128])
    free(cache, qd, out, ld, *([bd, w] if apart else [bd]))


@pytest.mark.parametrize("b, l, hq, hkv, d, lengths", [(1, 5, 16, 2, 64, [700]), (3, 9, 8, 2, 128, [300, 0, 40]), (5, 3, 8, 1, 256, [9, 500, 64, 2, 333]), (1, 1, 8, 1, 256, [17000]), (2, 1, 4, 1, 128, [5000, 4097]),
                                                     (1, 40, 8, 1, 128, [2100])])
def test_workgroups_that_read_the_same_keys_side_by_side(gpu, b, l, hq, hkv, d, lengths):
    """row tiles and shares whose streams of keys are no multiple of eight, with and without weights"""
    rng = np.random.default_rng(17)
    pages = Pages(rng, be.F16, b, -(-max(lengths) // 64) + 1, 64, hkv, d)
    bits, q = source(rng, (b, l, hq, d), be.F32)
    check(gpu, pages, bits, q, be.F32, d ** -0.5, lengths=lengths)


@pytest.mark.parametrize("dtype", [be.F32] + TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d, dims, h", [(64, 62, 5), (64, 2, 3), (8, 6, 40), (72, 30, 7), (256, 150, 2), (1024, 1022, 1), (1024, 6, 3), (136, 134, 300)])
@pytest.mark.parametrize("rows", [7, 1030])
def test_rotary_of_heads_that_do_not_come_apart_evenly(gpu, dtype, interleaved, d, dims, h, rows):
    if rows > 7 and h * d > 8192:
        h = 9
    rng = np.random.default_rng(dims)
    r = be.Rotary(dims, base=10000.0, interleaved=interleaved, magnitude=1.25)
    bits, x = source(rng, (1, rows, h, d), dtype)
    positions = rng.integers(-5, 300000, (1, rows)).astype(np.int32)
    xd, pd = gpu.upload(bits), gpu.upload(positions)
    out = gpu.alloc(bits.nbytes)
    gpu.step_rotary(out, xd, pd, 1, rows, h, d, r, dtype=dtype)
    got = gpu.download(out, storage(dtype), bits.shape)
    assert turned_close(to_f64(got, dtype), x, positions, r, dtype).all()
    gpu.step_rotary(xd, xd, pd, 1, rows, h, d, r, dtype=dtype)
    assert np.array_equal(gpu.download(xd, storage(dtype), bits.shape).view(np.uint8), got.view(np.uint8))
    for buf in (xd, pd, out):
        buf.free()


@pytest.mark.parametrize("src", [be.F32] + TYPES)
@pytest.mark.parametrize("hq, h, d, dims, s", [(4, 2, 64, 62, 3), (7, 3, 72, 30, 1), (5, 5, 72, 0, 9), (8, 1, 256, 150, 1100), (32, 8, 128, 106, 2)])
def test_append_of_heads_that_do_not_come_apart_evenly(gpu, src, hq, h, d, dims, s):
    """q as the step alone has it, keys from the turned f32 values, values as they came; and the append without turning"""
    rng = np.random.default_rng(d + s)
    pages = Pages(rng, be.F16, 2, -(-s // 32) + 1, 32, h, d)
    r = be.Rotary(dims, base=500000.0)
    (qb, q), (kb, k), (vb, v) = source(rng, (2, s, hq, d), src), source(rng, (2, s, h, d), src), source(rng, (2, s, h, d), src)
    positions, start = rng.integers(0, 5000, (2, s)).astype(np.int32), np.array([5, 17], np.int32)
    cache, qd, kd, vd, pd, sd = pages.upload(gpu), gpu.upload(qb), gpu.upload(kb), gpu.upload(vb), gpu.upload(positions), gpu.upload(start)
    out, ko, vo = gpu.alloc(qb.nbytes), gpu.alloc(k.size * 4), gpu.alloc(k.size * 4)
    gpu.step_rotary_append_paged(cache, r, out, qd, kd, vd, pd, sd, s, hq, dtype=src)
    assert turned_close(to_f64(gpu.download(out, storage(src), qb.shape), src), q, positions, r, src).all()
    gpu.step_read_paged(cache, ko, vo, sd, s)
    assert turned_close(gpu.download(ko, np.float32, k.shape).astype(np.float64), k, positions, r, be.F16).all()
    plain = to_f64(to_bits(v.astype(np.float32), be.F16), be.F16)
    assert np.array_equal(gpu.download(vo, np.float32, v.shape), plain)
    gpu.step_append_paged(cache, vd, kd, sd, s, src_dtype=src)
    gpu.step_read_paged(cache, ko, vo, sd, s)
    assert np.array_equal(gpu.download(ko, np.float32, v.shape), plain)
    assert np.array_equal(gpu.download(vo, np.float32, k.shape), to_f64(to_bits(k.astype(np.float32), be.F16), be.F16))
    free(cache, qd, kd, vd, pd, sd, out, ko, vo)


@pytest.mark.parametrize("cut", [False, True])
def test_evict_where_steps_end_at_two_to_the_31(cut):
    """the largest capacity there is, all but two of its entries no page: rows move where both ends are on one"""
    gpu = be.HipBackend(0)                                               # (26 GB, and scratch memory that goes with the context)
    rng = np.random.default_rng(31)
    p, d = 1024, 8
    width = 0x7FFFFFC0 // p
    cap = width * p
    limit, first, recent = cap - 5000 if cut else cap, 3, 700
    keep = cap - 6000 if cut else cap
    pages = Pages(rng, be.F16, 1, 1, p, 1, d, pages=3)
    table, table_out = np.full(width, -1, np.int32), np.full(width, -1, np.int32)
    table[-1], table_out[-1 if not cut else -6] = 2, 1
    kd, vd, td, to = (gpu.upload(x) for x in (pages.k, pages.v, table, table_out))
    cache = gpu.paged_cache(kd, vd, td, 3, 1, width, p, 1, d)
    wd, wo, kept, ld, lo = gpu.zeros(cap * 4), gpu.alloc(cap * 4), gpu.alloc(limit * 4), gpu.upload(np.array([2 ** 31 - 1], np.int32)), gpu.alloc(4)
    tail = rng.random(20000).astype(np.float32)                          # the last rows have weights, all others none
    gpu.write(wd, tail, offset=(cap - 20000) * 4)
    gpu.step_evict_paged(cache, wd, ld, wo, lo, keep, limit=limit, first=first, recent=recent, table_out=to, width_out=width, kept=kept)
    assert gpu.download(lo, np.int32, (1,))[0] == keep
    # every weighed row stays, and of the others the oldest
    old = keep - 20000
    want = np.concatenate((np.arange(old - 9000, old), np.arange(cap - 20000, cap)))
    assert np.array_equal(gpu.download(kept, np.int32, (29000,), offset=(keep - 29000) * 4), want)
    assert np.array_equal(gpu.download(kept, np.int32, (9000,)), np.arange(9000)) and (gpu.download(kept, np.int32, (limit - keep,), offset=keep * 4) == -1).all()
    weights = gpu.download(wo, np.float32, (cap - keep + 29000,), offset=(keep - 29000) * 4)
    assert np.array_equal(weights, np.concatenate((np.zeros(9000, np.float32), tail, np.zeros(cap - keep, np.float32))))
    # the source's page holds the last 1024 steps; the target's one page of places
    page = width - (6 if cut else 1)
    for which, (pool, buf) in enumerate(((pages.k, kd), (pages.v, vd))):
        for to_step in range(page * p, min((page + 1) * p, keep)):
            t = cap - (keep - to_step)                                   # (a place among the weighed rows)
            if t // p == width - 1:
                pool[1, :, to_step % p] = pool[2, :, t % p]
        assert np.array_equal(gpu.download(buf, np.float16, pool.shape), pool), which
    for buf in (kd, vd, td, to, wd, wo, kept, ld, lo):
        buf.free()
    gpu.close()
