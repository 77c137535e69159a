"""Rows into caches held in 8 or 4 bits and out again, against the same arithmetic in numpy: the codes and scales bit for bit, the rows read back exactly
(a code times a scale is exact in f32 and is rounded once)."""
import numpy as np
import pytest

from aion_amd import backend as be
from quant_cases import QuantCache, filled
from test_gpu_attention import to_bf16

pytestmark = pytest.mark.gpu

FILL = 0xA5


def put(gpu, cache):
    return gpu.upload(cache.bytes)


def indices(at, s, t_cap, rolling):
    t = np.arange(at, at + s)
    return np.where(t < 0, -1, t % t_cap) if rolling else np.where((t < 0) | (t >= t_cap), -1, t)


def as_source(x, src):
    """what is uploaded, and the f32 values it stands for"""
    if src == be.F16:
        return x.astype(np.float16), x.astype(np.float16).astype(np.float32)
    if src == be.BF16:
        return to_bf16(x)
    return x, x


@pytest.mark.parametrize("dtype", [be.Q8_0, be.Q4_0])
@pytest.mark.parametrize("b,s,t_cap,h,d,starts,rolling,src", [
    (1, 1, 64, 1, 32, [0], False, be.F32),
    (1, 1, 1, 3, 64, [0], False, be.F32),
    (2, 1, 100, 8, 128, [99, 5], False, be.F32),
    (3, 7, 65, 2, 96, [0, 58, 30], False, be.F16),
    (2, 130, 200, 5, 64, [70, 3], False, be.BF16),
    (1, 300, 300, 2, 256, [0], False, be.F32),
    (3, 9, 50, 2, 160, [45, -4, 60], False, be.F32),           # past the end, before the beginning, wholly outside
    (3, 9, 50, 2, 128, [46, 1000003, -4], True, be.F32),       # rings: over the end, long after, before the beginning
    (2, 50, 50, 1, 64, [7, 2147483000], True, be.F16),         # the whole ring, and a step index near 2^31
])
def test_append(gpu, dtype, b, s, t_cap, h, d, starts, rolling, src):
    rng = np.random.default_rng(b * 1000 + s * 10 + d)
    rows = [(rng.standard_normal((b, s, h, d)) * np.exp(rng.standard_normal((b, s, h, 1)))).astype(np.float32) for _ in range(2)]
    rows[0][0, 0, 0, :32] = 0.0
    rows[1][-1, -1, -1, -32:] = 1e-9                              # a scale that f16 holds as zero
    want, bufs, srcs = [], [], []
    for x in rows:
        up, exact = as_source(x, src)
        c = QuantCache(dtype, b, t_cap, h, d, FILL)
        bufs.append(put(gpu, c))
        for i in range(b):
            c.put(exact[i], i, indices(starts[i], s, t_cap, rolling))
        want.append(c)
        srcs.append(gpu.upload(up))
    index = gpu.upload(np.array(starts, np.int32))
    shape = (b, s, t_cap, h, d)
    gpu.step_append_quant(dtype, bufs, srcs, index, shape, src_dtype=src, rolling=rolling)
    for buf, c in zip(bufs, want):
        assert np.array_equal(gpu.download(buf, np.uint8, c.bytes.shape), c.bytes)          # untouched bytes as they were
    alone = put(gpu, QuantCache(dtype, b, t_cap, h, d, FILL))
    gpu.step_append_quant(dtype, [alone], [srcs[1]], index, shape, src_dtype=src, rolling=rolling)
    assert np.array_equal(gpu.download(alone, np.uint8, want[1].bytes.shape), want[1].bytes)
    # the same rows back
    outs = [gpu.alloc(b * s * h * d * 4) for _ in range(2)]
    gpu.step_cache_read(dtype, outs, bufs, index, shape, rolling=rolling)
    for out, c in zip(outs, want):
        values = c.values()
        for i in range(b):
            at = indices(starts[i], s, t_cap, rolling)
            expect = np.where((at >= 0)[:, None, None], values[i, np.maximum(at, 0)], 0.0)
            assert np.array_equal(gpu.download(out, np.float32, (b, s, h, d))[i], expect.astype(np.float32))
    for x in bufs + srcs + outs + [index, alone]:
        x.free()


@pytest.mark.parametrize("dtype", [be.Q8_0, be.Q4_0])
@pytest.mark.parametrize("exponent", [-146, -126, -120, -30, -3, 0, 9, 100, 122])
def test_codes_beside_halves(gpu, dtype, exponent):
    """quotients at, just under and just over the halves between two codes, at scales from f32's smallest to its largest"""
    rng = np.random.default_rng(exponent + 200)
    s, h, d = 40, 2, 64
    levels = 127 if dtype == be.Q8_0 else 7
    top = np.ldexp(rng.uniform(1, 2, (1, s, h, d // 32, 1)), exponent).astype(np.float32)
    x = top * ((rng.integers(-levels, levels, (1, s, h, d // 32, 32)) + 0.5) / levels).astype(np.float32)
    for _ in range(2):
        x = np.where(rng.integers(0, 2, x.shape) == 0, x, np.nextafter(x, np.where(rng.integers(0, 2, x.shape) == 0, np.float32(-np.inf), np.float32(np.inf))))
    x[..., 7:8] = top
    x = np.clip(x, -top, top).astype(np.float32).reshape(1, s, h, d)
    want = QuantCache(dtype, 1, s, h, d, FILL)
    buf = put(gpu, want)
    with np.errstate(over="ignore"):
        want.put(x[0], 0, np.arange(s))
    gpu.step_append_quant(dtype, [buf], [gpu.upload(x)], gpu.upload(np.zeros(1, np.int32)), (1, s, s, h, d))
    assert np.array_equal(gpu.download(buf, np.uint8, want.bytes.shape), want.bytes)


@pytest.mark.parametrize("dtype", [be.Q8_0, be.Q4_0])
@pytest.mark.parametrize("s,h,d", [(1, 1, 2048), (5, 2, 2080), (3, 1, 4128), (11, 3, 1056), (9, 2, 672)])
def test_long_heads(gpu, dtype, s, h, d):
    """heads of more pieces than a workgroup has threads, and such as do not divide it"""
    rng = np.random.default_rng(d)
    x = rng.standard_normal((2, s, h, d)).astype(np.float32)
    want = QuantCache(dtype, 2, 80, h, d, FILL)
    buf = put(gpu, want)
    for i in range(2):
        want.put(x[i], i, np.arange(60 * i, 60 * i + s))
    index = gpu.upload(np.array([0, 60], np.int32))
    gpu.step_append_quant(dtype, [buf], [gpu.upload(x)], index, (2, s, 80, h, d))
    assert np.array_equal(gpu.download(buf, np.uint8, want.bytes.shape), want.bytes)
    out = gpu.alloc(x.nbytes)
    gpu.step_cache_read(dtype, [out], [buf], index, (2, s, 80, h, d))
    for i in range(2):
        assert np.array_equal(gpu.download(out, np.float32, x.shape)[i], want.values()[i, 60 * i:60 * i + s])


@pytest.mark.parametrize("offset", [1, 2, 3])
def test_rows_at_any_aligned_address(gpu, offset):
    rng = np.random.default_rng(offset)
    x = rng.standard_normal((1, 3, 2, 64)).astype(np.float32)
    for src, up in ((be.F32, x), (be.F16, x.astype(np.float16))):
        flat = np.concatenate([np.zeros(offset, up.dtype), up.ravel()])
        buf, cache, index, out = gpu.upload(flat), gpu.zeros(gpu.cache_quant_bytes(be.Q8_0, 1, 5, 2, 64)), gpu.upload(np.array([1], np.int32)), gpu.alloc(4 * (x.size + 4))
        gpu.step_append_quant(be.Q8_0, [cache], [buf.view(offset * up.itemsize)], index, (1, 3, 5, 2, 64), src_dtype=src)
        c = QuantCache(be.Q8_0, 1, 5, 2, 64)
        c.put(up.astype(np.float32)[0], 0, range(1, 4))
        assert np.array_equal(gpu.download(cache, np.uint8, c.bytes.shape), c.bytes)
        gpu.step_cache_read(be.Q8_0, [out.view(4 * offset)], [cache], index, (1, 3, 5, 2, 64))
        assert np.array_equal(gpu.download(out, np.float32, x.shape, offset=4 * offset)[0], c.values()[0, 1:4].astype(np.float32))
        for b in (buf, cache, index, out):
            b.free()


@pytest.mark.parametrize("dtype", [be.Q8_0, be.Q4_0])
@pytest.mark.parametrize("out_dtype", [be.F32, be.F16, be.BF16])
@pytest.mark.parametrize("b,s,t_cap,h,d,starts,rolling", [
    (1, 1, 1, 1, 32, [0], False), (2, 77, 130, 3, 64, [53, -9], False), (3, 64, 64, 2, 256, [0, 60, -64], False), (2, 33, 40, 4, 96, [77, -3], True)])
def test_read(gpu, dtype, out_dtype, b, s, t_cap, h, d, starts, rolling):
    rng = np.random.default_rng(s + d)
    c = filled(rng, dtype, b, t_cap, h, d)
    buf, index = put(gpu, c), gpu.upload(np.array(starts, np.int32))
    size = 4 if out_dtype == be.F32 else 2
    guard = 64
    out = gpu.upload(np.full(b * s * h * d * size + guard, FILL, np.uint8))
    gpu.step_cache_read(dtype, [out], [buf], index, (b, s, t_cap, h, d), out_dtype=out_dtype, rolling=rolling)
    raw = gpu.download(out, np.uint8, (b * s * h * d * size + guard,))
    assert (raw[-guard:] == FILL).all()
    values = c.values()
    want = np.zeros((b, s, h, d), np.float32)
    for i in range(b):
        at = indices(starts[i], s, t_cap, rolling)
        want[i] = np.where((at >= 0)[:, None, None], values[i, np.maximum(at, 0)], 0.0)
    got = raw[:-guard].view({be.F32: np.float32, be.F16: np.float16, be.BF16: np.uint16}[out_dtype]).reshape(want.shape)
    if out_dtype == be.BF16:
        keep = want != 0                                        # (a negative code times a scale of zero: the sign of the zero)
        assert np.array_equal(got[keep], to_bf16(want)[0][keep])
    else:
        assert np.array_equal(got, want.astype(got.dtype))
    for x in (buf, index, out):
        x.free()


@pytest.mark.parametrize("dtype", [be.Q8_0, be.Q4_0])
def test_what_is_not_finite_stays_in_its_block(gpu, dtype):
    rng = np.random.default_rng(1)
    x = rng.standard_normal((1, 4, 2, 64)).astype(np.float32)
    x[0, 0, 0, 3], x[0, 1, 1, 40], x[0, 2, 0, 63] = np.nan, np.inf, -np.inf
    src, index = gpu.upload(x), gpu.upload(np.array([0], np.int32))
    cache, out = gpu.zeros(gpu.cache_quant_bytes(dtype, 1, 4, 2, 64)), gpu.alloc(x.nbytes)
    gpu.step_append_quant(dtype, [cache], [src], index, (1, 4, 4, 2, 64))
    gpu.step_cache_read(dtype, [out], [cache], index, (1, 4, 4, 2, 64))
    got = gpu.download(out, np.float32, x.shape).reshape(1, 4, 2, 2, 32)
    gone = np.zeros((1, 4, 2, 2), bool)
    gone[0, 0, 0, 0] = gone[0, 1, 1, 1] = gone[0, 2, 0, 1] = True
    assert np.isnan(got[gone]).all()
    c = QuantCache(dtype, 1, 4, 2, 64)
    c.put(np.where(np.isfinite(x), x, 0)[0], 0, range(4))
    assert np.array_equal(got[~gone], c.values()[:, :4].reshape(got.shape)[~gone].astype(np.float32))
    for b in (src, index, cache, out):
        b.free()


@pytest.mark.parametrize("dtype", [be.Q8_0, be.Q4_0])
@pytest.mark.parametrize("b,s,t_cap,hq,hk,d,proportion,rolling", [
    (1, 1, 64, 8, 1, 256, 1.0, False), (2, 5, 40, 4, 2, 64, 0.5, False), (3, 3, 20, 3, 3, 96, 1.0, True), (1, 33, 64, 2, 1, 32, 0.3, False), (2, 1, 10, 4, 4, 128, 0.0, True)])
def test_rope_append(gpu, dtype, b, s, t_cap, hq, hk, d, proportion, rolling):
    """The bits of the separate steps."""
    rng = np.random.default_rng(s + d)
    q, k, v = (rng.standard_normal((b, s, h, d)).astype(np.float32) for h in (hq, hk, hk))
    starts = np.array([(t_cap - s) // (i + 1) + (3 * t_cap if rolling else 0) for i in range(b)], np.int32)
    pos = gpu.upload((starts[:, None] + np.arange(s)).astype(np.int32) % 4000)
    index = gpu.upload(starts)
    n = gpu.cache_quant_bytes(dtype, b, t_cap, hk, d)
    fill = np.full(n, FILL, np.uint8)
    ins = [gpu.upload(x) for x in (q, k, v)]
    outs = [gpu.alloc(x.nbytes) for x in (q, q, k)]
    caches = [gpu.upload(fill) for _ in range(4)]
    gpu.step_rope_append_quant(dtype, outs[0], *ins, *caches[:2], pos, index, b, s, t_cap, hq, hk, d, proportion=proportion, rolling=rolling)
    gpu.step_rope(outs[1], ins[0], pos, b, s, hq, d, proportion=proportion)
    gpu.step_rope(outs[2], ins[1], pos, b, s, hk, d, proportion=proportion)
    gpu.step_append_quant(dtype, caches[2:], [outs[2], ins[2]], index, (b, s, t_cap, hk, d), rolling=rolling)
    assert np.array_equal(gpu.download(outs[0], np.uint32, q.shape), gpu.download(outs[1], np.uint32, q.shape))
    for one, two in ((0, 2), (1, 3)):
        got = gpu.download(caches[one], np.uint8, (n,))
        assert np.array_equal(got, gpu.download(caches[two], np.uint8, (n,))) and not np.array_equal(got, fill)
    for x in ins + outs + caches + [pos, index]:
        x.free()


@pytest.mark.parametrize("dtype", [be.Q8_0, be.Q4_0])
def test_growth_by_its_two_parts(gpu, dtype):
    rng = np.random.default_rng(5)
    b, h, d, old, new = 2, 3, 64, 70, 200
    c = filled(rng, dtype, b, old, h, d, fill=0)
    grown = QuantCache(dtype, b, new, h, d)
    grown.codes[:, :, :c.tp], grown.scales[..., :c.tp] = c.codes, c.scales
    src, dst = put(gpu, c), gpu.alloc(grown.bytes.size)
    gpu.cache_grow(dst, src, b * h, c.codes[0, 0].size, grown.codes[0, 0].size)
    gpu.cache_grow(dst.view(grown.codes.size), src.view(c.codes.size), b * h * d // 32, c.tp * 2, grown.tp * 2)
    assert np.array_equal(gpu.download(dst, np.uint8, grown.bytes.shape), grown.bytes)
    src.free()
    dst.free()


def test_refusals(gpu):
    shape = (1, 2, 64, 2, 64)
    size = gpu.cache_quant_bytes(be.Q8_0, 1, 64, 2, 64)
    a, b, x, i = gpu.zeros(size + 16), gpu.zeros(size), gpu.zeros(4096), gpu.zeros(16)
    none = be.DeviceBuffer(gpu, 0, 0)

    def refused(status, f, *args, **kw):
        with pytest.raises(be.AionHipError) as e:
            f(*args, **kw)
        assert e.value.status == status, e.value

    bad, no = be.hip.INVALID_ARGUMENT, be.hip.UNSUPPORTED
    append, read = gpu.step_append_quant, gpu.step_cache_read
    for f, first in ((append, [a]), (read, [x])):
        second = [x] if f is append else [a]
        refused(bad, f, be.F16, first, second, i, shape)                        # not a block format
        refused(bad, f, be.Q8_0, [none], second, i, shape)
        refused(bad, f, be.Q8_0, first, [none], i, shape)
        refused(bad, f, be.Q8_0, first, second, none, shape)
        refused(bad, f, be.Q8_0, first, second, i, (1, 2, 64, 2, 48))           # whole blocks
        refused(bad, f, be.Q8_0, first, second, i, (1, 65, 64, 2, 64))          # more rows than the cache has
        refused(no, f, be.Q8_0, first, second, i, (1, 2, 64, 70000, 64))
        refused(no, f, be.Q8_0, first, second, i, (1, 2, 1 << 31, 2, 64))
        refused(bad, f, be.Q8_0, [a, b], [x], i, shape) if f is append else refused(bad, f, be.Q8_0, [x], [a, b], i, shape)
        refused(bad, f, be.Q8_0, [], second, i, shape)
    refused(bad, append, be.Q8_0, [a.view(8)], [x], i, shape)
    refused(bad, read, be.Q8_0, [x], [a.view(8)], i, shape)
    refused(bad, append, be.Q8_0, [a, a], [x, x], i, shape)
    refused(bad, append, be.Q8_0, [a, a.view(size - 16)], [x, x], i, shape)     # one in the other's end
    refused(bad, read, be.Q8_0, [x, x.view(1020)], [a, b], i, shape)
    refused(no, append, be.Q8_0, [a], [x], i, shape, src_dtype=be.I32)
    refused(no, read, be.Q8_0, [x], [a], i, shape, out_dtype=be.Q8_0)
    rope = gpu.step_rope_append_quant
    ok = (be.Q8_0, x.view(2048), x, x, x, a, b, i, i, 1, 2, 64, 2, 2, 64)
    refused(bad, rope, be.F32, *ok[1:])
    refused(bad, rope, *ok[:1], x, *ok[2:])                                     # in place
    refused(bad, rope, *ok[:1], x.view(1020), *ok[2:])                          # nearly
    refused(bad, rope, *ok[:6], a, *ok[7:])
    refused(bad, rope, *ok[:6], a.view(size - 16), *ok[7:])
    refused(bad, rope, *ok, proportion=1.5)
    refused(bad, rope, *ok, base=0.0)
    for e in (0, 1, 3, 4):                                                      # nothing to do is no error
        empty = list(shape)
        empty[e] = 0
        append(be.Q8_0, [a], [x], i, tuple(empty))
        read(be.Q8_0, [x], [a], i, tuple(empty))
    assert not gpu.download(a, np.uint8, (size,)).any() and not gpu.download(x, np.uint8, (4096,)).any()
    for buf in (a, b, x, i):
        buf.free()


def test_recorded_append_follows_the_index(gpu):
    """The write index is read on the device: a recorded append moves with it, replay by replay."""
    rng = np.random.default_rng(2)
    x = rng.standard_normal((1, 1, 2, 64)).astype(np.float32)
    c = QuantCache(be.Q4_0, 1, 20, 2, 64)
    cache, src, out = put(gpu, c), gpu.upload(x), gpu.alloc(x.nbytes)
    index = gpu.upload(np.array([0], np.int32))
    shape = (1, 1, 20, 2, 64)

    def issue():
        gpu.step_append_quant(be.Q4_0, [cache], [src], index, shape)
        gpu.step_cache_read(be.Q4_0, [out], [cache], index, shape)
    issue()
    prog = gpu.record_program(issue)
    for i in range(4):
        y = rng.standard_normal(x.shape).astype(np.float32)
        gpu.write(src, y)
        gpu.write(index, np.array([3 * i], np.int32))
        gpu.program_execute(prog)
        if i == 0:
            c.put(x[0], 0, [0])
        c.put(y[0], 0, [3 * i])
        assert np.array_equal(gpu.download(cache, np.uint8, c.bytes.shape), c.bytes)
        assert np.array_equal(gpu.download(out, np.float32, x.shape)[0, 0], c.values()[0, 3 * i].astype(np.float32))
    gpu.program_destroy(prog)
    for b in (cache, src, out, index):
        b.free()
