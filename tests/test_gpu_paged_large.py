"""Steps over pages in the forms that only large calls take: keys, values and rows past the caches, long walks of one wavefront, several row tiles behind windows."""
import numpy as np
import pytest

from aion_amd import backend as be
from paged_cases import Pages, attention, free, storage, to_bits, to_f64, turned_close
from test_gpu_paged import attend, check, source

pytestmark = pytest.mark.gpu


def instance(gpu):
    """the kernel of the last launch and its template arguments"""
    name = gpu.last_launch()["kernel"].replace("(anonymous namespace)::", "")
    return name[:name.index("<")].split()[-1], [x.strip() for x in name[name.index("<") + 1:name.index(">")].split(",")]


def wide(pages, width):
    """the same sequences in a cache of more entries, none of which is a page"""
    pages.table = np.concatenate((pages.table, np.full((pages.b, width - pages.width), -1, np.int32)), axis=1)
    pages.width = width
    return pages


# ---------------------------------------------------------------------------------------------------------------- attention
@pytest.mark.parametrize("dtype", [be.F16, be.BF16])
@pytest.mark.parametrize("q_dtype", [be.F32, be.F16, be.BF16])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_one_token_past_the_caches(gpu, dtype, q_dtype, d):
    """a capacity of 192 MiB and more decides, whatever the lengths are; wavefronts have up to three tiles"""
    rng = np.random.default_rng(d)
    b, h, hq, p = 2, 2, 6, 64
    lengths = [40003, 333]
    pages = Pages(rng, dtype, b, -(-lengths[0] // p), p, h, d)
    pages.table[1, 6:] = -1
    pages.table[0, 17] = -1
    wide(pages, (192 << 20) // (b * h * d * 4) // p)
    bits, q = source(rng, (b, 1, hq, d), q_dtype)
    check(gpu, pages, bits, q, q_dtype, d ** -0.5, lengths=lengths)
    attend(gpu, pages, bits, q_dtype, d ** -0.5, lengths=lengths, weigh=False)
    name, args = instance(gpu)
    parts = 1 if q_dtype == dtype else 2 if dtype == be.F16 else 3
    assert name == "paged_attn_kernel" and args == [str(dtype), str(d), str(parts), "false", "true", "1"]
    # one entry fewer: the same keys through the caches, to the same bits
    want, _ = attend(gpu, pages, bits, q_dtype, d ** -0.5, lengths=lengths)
    pages.table, pages.width = np.ascontiguousarray(pages.table[:, :-1]), pages.width - 1
    got, _ = attend(gpu, pages, bits, q_dtype, d ** -0.5, lengths=lengths, weigh=False)
    assert instance(gpu)[1][4] == "false" and np.array_equal(got, want)


@pytest.mark.parametrize("dtype, d, h", [(be.F16, 64, 16), (be.BF16, 128, 16), (be.F16, 256, 8)])
@pytest.mark.parametrize("l", [1, 2])
def test_walks_of_more_than_32_tiles(gpu, dtype, d, h, l):
    """64 sequences over the same pages: few segments, so that a wavefront fetches its page numbers more than once"""
    rng = np.random.default_rng(d)
    b, p, n = 64, 16, 9011 if d < 256 else 17011
    pages = Pages(rng, dtype, 1, -(-n // p), p, h, d)
    pages.b, pages.table = 3, np.repeat(pages.table, 3, axis=0)
    lengths = [n, n - 5000, 37]
    bits, q = source(rng, (1, l, h, d), be.F32)
    near, drawn = attention(np.repeat(q, 3, axis=0), pages, l, h, d ** -0.5, lengths=lengths)
    which = [0] * 61 + [1, 2, 0]
    pages.b, pages.table = b, np.repeat(pages.table[:1], b, axis=0)
    got, weights = attend(gpu, pages, np.repeat(bits, b, axis=0), be.F32, d ** -0.5, lengths=[lengths[i] for i in which])
    for i in range(b):
        assert np.array_equal(got[i], got[which.index(which[i])]) and np.array_equal(weights[i], weights[which.index(which[i])]), i
    first = [which.index(i) for i in range(3)]
    assert near.close(got[first]).all() and near.weights_close(weights[first], drawn, l).all()
    attend(gpu, pages, np.repeat(bits, b, axis=0), be.F32, d ** -0.5, lengths=[lengths[i] for i in which], weigh=False)
    launch = gpu.last_launch()
    segments = launch["grid"][0] // (1 if launch["grid"][1] > 1 else b * h)
    assert instance(gpu)[1][4] == ("true" if l == 1 else "false") and -(-n // 32) > 32 * segments * launch["block"][0] // 64


@pytest.mark.parametrize("d, hq, h", [(64, 6, 2), (128, 6, 2), (256, 8, 1), (80, 6, 2)])
@pytest.mark.parametrize("window, soft_cap, given", [
    ((700, 0, 0), 0.0, False), ((33, 0, 0), 0.0, False), ((0, 0, 0), 20.0, False), ((be.UNBOUNDED, be.UNBOUNDED, 0), 0.0, False), ((100, 9, 256), 0.0, False),
    (be.CAUSAL, 0.0, True), ((200, 0, 0), 0.0, True), ((90, 50, 128), 5.0, True),
])
def test_row_tiles_behind_windows(gpu, d, hq, h, window, soft_cap, given):
    """twenty queries, four row tiles and more of a KV head: each has a first key and segments of its own"""
    rng = np.random.default_rng(d + window[1])
    b, l = 2, 20
    lengths = [1900, 811]
    pages = Pages(rng, be.F16, b, 60, 32, h, d)
    pages.table[0, 50] = -1
    bits, q = source(rng, (b, l, hq, d), be.F32)
    positions = None
    if given:                                                                    # in no order, some before the first key, some past the last
        positions = rng.integers(-20, 2000, (b, l)).astype(np.int32)
    check(gpu, pages, bits, q, be.F32, d ** -0.5, lengths=lengths, window=window, soft_cap=soft_cap, positions=positions)


# ---------------------------------------------------------------------------------------------------------------- rows
ROWS = [  # heads of q, of keys and values (0: rotary alone), d, dims, tokens
    (32, 0, 128, 128, 8200), (32, 0, 128, 96, 8200), (32, 0, 128, 126, 8200), (20, 8, 128, 128, 7400), (20, 8, 128, 62, 7400), (32, 4, 1024, 1024, 1000), (32, 4, 1024, 1022, 1000),
]


@pytest.mark.parametrize("dtype, cache_dtype", [(be.F16, be.F16), (be.F16, be.BF16), (be.BF16, be.BF16), (be.BF16, be.F16), (be.F32, be.F16), (be.F32, be.BF16)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("hq, h, d, dims, tokens", ROWS)
def test_rows_past_the_caches(gpu, dtype, cache_dtype, interleaved, hq, h, d, dims, tokens):
    """128 MiB and more, read and written: the bits of the same rows in two calls through the caches, and a few rows in 64 bits"""
    if not h and cache_dtype != be.F16:
        return
    rng = np.random.default_rng(dims)
    if dtype == be.F32:
        tokens //= 2
    half, r, size = tokens // 2, be.Rotary(dims, base=500000.0, interleaved=interleaved, magnitude=1.25), np.dtype(storage(dtype)).itemsize
    assert tokens * (hq + 2 * h) * d * 2 * size >= 128 << 20 > (tokens - half) * (hq + 2 * h) * d * 2 * size
    draw = lambda n: to_bits(rng.standard_normal((1, tokens, n, d), np.float32), dtype)  # noqa: E731
    positions = rng.integers(0, 200000, (1, tokens)).astype(np.int32)
    qb, pd = draw(hq), gpu.upload(positions)
    qd, out, twice = gpu.upload(qb), gpu.alloc(qb.nbytes), gpu.alloc(qb.nbytes)
    parts = [(0, half), (half, tokens - half)]
    if not h:
        gpu.step_rotary(out, qd, pd, 1, tokens, hq, d, r, dtype=dtype)
        name, args = instance(gpu)
        for at, n in parts:
            gpu.step_rotary(twice.view(at * hq * d * size), qd.view(at * hq * d * size), pd.view(at * 4), 1, n, hq, d, r, dtype=dtype)
    else:
        kb, vb = draw(h), draw(h)
        kd, vd = gpu.upload(kb), gpu.upload(vb)
        pages = Pages(rng, cache_dtype, 1, -(-tokens // 128), 128, h, d)
        a, b = pages.upload(gpu), pages.upload(gpu)
        zero = gpu.upload(np.zeros(1, np.int32))
        gpu.step_rotary_append_paged(a, r, out, qd, kd, vd, pd, zero, tokens, hq, dtype=dtype)
        name, args = instance(gpu)
        for at, n in parts:
            to, row = gpu.upload(np.array([at], np.int32)), at * d * size
            gpu.step_rotary_append_paged(b, r, twice.view(row * hq), qd.view(row * hq), kd.view(row * h), vd.view(row * h), pd.view(at * 4), to, n, hq, dtype=dtype)
            gpu.sync()
            to.free()
        for x, y in ((a.k_pages, b.k_pages), (a.v_pages, b.v_pages)):
            assert np.array_equal(gpu.download(x, np.uint16), gpu.download(y, np.uint16))
        # keys and values of a few rows
        ko, vo = gpu.alloc(tokens * h * d * 4), gpu.alloc(tokens * h * d * 4)
        gpu.step_read_paged(a, ko, vo, zero, tokens)
        some = rng.integers(0, tokens, 40)
        k = gpu.download(ko, np.float32, kb.shape)[:, some].astype(np.float64)
        assert turned_close(k, to_f64(kb[:, some], dtype), positions[:, some], r, cache_dtype).all()
        assert np.array_equal(gpu.download(vo, np.float32, vb.shape)[:, some], to_f64(to_bits(to_f64(vb[:, some], dtype).astype(np.float32), cache_dtype), cache_dtype))
        free(a, kd, vd, zero, ko, vo)
        free(b)
    # (f32 rows past the caches come in pieces always; heads that do not come apart evenly through LDS else)
    each = 4 if dtype == be.F32 else 8
    whole = (dims % (2 * each) if interleaved else dims // 2 % each) == 0 and (d - dims) % (2 * each) == 0
    assert name == ("rotary_kernel" if whole or dtype == be.F32 else "rotary_rows_kernel") and args[-1] == "true"
    got = gpu.download(out, storage(dtype), qb.shape)
    assert np.array_equal(got.view(np.uint8), gpu.download(twice, storage(dtype), qb.shape).view(np.uint8))
    some = rng.integers(0, tokens, 40)
    assert turned_close(to_f64(got[:, some], dtype), to_f64(qb[:, some], dtype), positions[:, some], r, dtype).all()
    for buf in (qd, pd, out, twice):
        buf.free()
