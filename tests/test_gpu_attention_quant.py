"""Attention over caches held in 8 or 4 bits, against 64-bit attention over the numbers that the cache holds (codes times scales, exact in 64 bits).

The bound of an output element is relative to the sum of p |v| it is an average over, and adds up what the step may round:
  scores         the query as two f16 parts (2^-21 of a product, the products exact), f32 sums of at most 32 products and 32 blocks on
                 the way, scales and factors: less than 2^-18 of scale * sum |q k|. A score that is off by e changes the average by at most 2 e
                 of it (numerator and normalizer).
  exponentials   an argument a is rounded to 2^-24 a, and e^-a a stays below 0.37; the exponential itself 2^-22; together less than 2^-20
  products       probabilities as two half-precision parts, 2^-18 (bf16: 2^-9 * 2^-9), in prompts the values too, and the product of the two small
                 parts left out, 2^-16; f32 sums of at most 5000 / 64 tiles of 64 products, 2^-24 * 144 < 2^-16
so 2^-14 of the sum in all, and 2^-17 times scale * sum |q k| of it. A soft cap adds the error of a tanh, 2^-21 of the cap. And what a key adds may be
small beside the row's largest p |v| without that one showing in the column (its code there is zero): probabilities are held to an absolute 2^-25 where the
largest product of a probability and a scale is at least 2^9, so to 2^-34 of it, a code is at most 127 / 126 of the largest one of its block (q8_0; q4_0 8 / 7) and there
are as many errors as keys: less than 2^-33 of keys * max p max|v|. (An exponential below 2^-126 of the row's largest vanishes, which is less.)
"""
import math

import numpy as np
import pytest

from aion_amd import backend as be
from quant_cases import QuantCache, attention_f64, filled
from test_gpu_attention import to_bf16

pytestmark = pytest.mark.gpu


def as_queries(x, dtype):
    if dtype == be.F16:
        return x.astype(np.float16), x.astype(np.float16).astype(np.float64)
    if dtype == be.BF16:
        bits, values = to_bf16(x)
        return bits, values.astype(np.float64)
    return x, x.astype(np.float64)


def step(gpu, q, kc, vc, t_cap, scale, q_dtype=be.F32, window=be.CAUSAL, soft_cap=0.0, positions=None, kv_lengths=None, rolling=False):
    bn, l, hq, dk = q.shape
    guard = 64
    out = gpu.upload(np.full(bn * l * hq * vc.d + guard, -7.5, np.float32))
    bufs = [gpu.upload(q), gpu.upload(kc.bytes), gpu.upload(vc.bytes)]
    pos = gpu.upload(np.ascontiguousarray(positions, np.int32)) if positions is not None else None
    lens = gpu.upload(np.ascontiguousarray(kv_lengths, np.int32)) if kv_lengths is not None else None
    gpu.step_attention(out, *bufs, (bn, l, t_cap, hq, kc.h, dk, vc.d), scale, q_dtype=q_dtype, kv_dtype=kc.dtype, window=window, soft_cap=soft_cap,
                       query_positions=pos, kv_lengths=lens, rolling=rolling)
    got = gpu.download(out, np.float32, (bn * l * hq * vc.d + guard,))
    assert (got[-guard:] == -7.5).all()
    for b in bufs + [out] + [x for x in (pos, lens) if x is not None]:
        b.free()
    return got[:-guard].reshape(bn, l, hq, vc.d)


def bound_of(near, soft_cap=0.0):
    return near.weight * (2.0 ** -14 + 2.0 ** -17 * near.reach[..., None] + 2.0 ** -20 * soft_cap) + 2.0 ** -33 * near.floor[..., None]


def check(gpu, q, kc, vc, t_cap, scale, q_dtype=be.F32, **options):
    up, exact = as_queries(q, q_dtype)
    want, near = attention_f64(exact, kc.values(), vc.values(), scale, t_cap, **options)
    got = step(gpu, up, kc, vc, t_cap, scale, q_dtype, **options)
    bound = bound_of(near, options.get("soft_cap", 0.0))
    err = np.abs(got - want)
    worst = float((err / np.maximum(bound, 1e-300))[bound > 0].max(initial=0.0))
    print("  %s max error / bound %.3f   relative error %.1e" % (gpu.last_kernel(), worst, float(np.linalg.norm(err) / max(np.linalg.norm(want), 1e-30))), flush=True)
    inside = bool(np.isfinite(got).all() and (err <= bound).all())
    assert inside, worst
    return got


def case(seed, dtype, bn, l, t_cap, hq, hk, d, dv=None, sigma=1.0, rows=None):
    rng = np.random.default_rng(seed)
    q = rng.standard_normal((bn, l, hq, d)).astype(np.float32)
    return q, filled(rng, dtype, bn, t_cap, hk, d, sigma, rows=rows), filled(rng, dtype, bn, t_cap, hk, dv or d, 1.0, rows=rows)


BOTH = pytest.mark.parametrize("dtype", [be.Q8_0, be.Q4_0])
HEADS = [(8, 1, 256), (32, 8, 128), (16, 4, 64), (4, 4, 128), (3, 1, 64), (10, 1, 256), (40, 2, 128)]


@BOTH
@pytest.mark.parametrize("hq,hk,d", HEADS)
@pytest.mark.parametrize("t", [1, 31, 64, 65, 500])
def test_one_token(gpu, dtype, hq, hk, d, t):
    q, kc, vc = case(t + d, dtype, 1, 1, t, hq, hk, d)
    check(gpu, q, kc, vc, t, 1 / math.sqrt(d), positions=[[t - 1]], kv_lengths=[t])


@BOTH
@pytest.mark.parametrize("q_dtype", [be.F32, be.F16, be.BF16])
@pytest.mark.parametrize("hq,hk,d", [(8, 1, 256), (32, 8, 128), (16, 4, 64)])
def test_ragged_batch_with_an_idle_sequence(gpu, dtype, q_dtype, hq, hk, d):
    """Lengths from none to past the capacity (clipped to it); rows behind a sequence's end hold NaN scales."""
    t_cap = 333
    lengths = [333, 0, 1, 64, 200, 5000]
    q, kc, vc = case(d, dtype, len(lengths), 1, t_cap, hq, hk, d)
    for c in (kc, vc):
        for i, n in enumerate(lengths):
            c.scales[i, :, :, n:] = 0x7E00
    got = check(gpu, q, kc, vc, t_cap, 1 / math.sqrt(d), q_dtype, positions=[[max(n - 1, 0)] for n in lengths], kv_lengths=lengths)
    assert not got[1].any()


@BOTH
@pytest.mark.parametrize("hq,hk,d", [(8, 2, 256), (32, 8, 128), (6, 2, 64)])
@pytest.mark.parametrize("l,t", [(2, 70), (5, 301), (9, 64), (17, 400), (40, 130), (130, 130), (200, 777)])
def test_several_queries(gpu, dtype, hq, hk, d, l, t):
    q, kc, vc = case(l + t + d, dtype, 2, l, t, hq, hk, d)
    pos = np.stack([np.arange(t - l, t), np.arange(0, l)])
    check(gpu, q, kc, vc, t, 1 / math.sqrt(d), positions=pos, kv_lengths=[t, l])


@BOTH
@pytest.mark.parametrize("l,t", [(1, 600), (7, 600), (150, 600)])
@pytest.mark.parametrize("window", [be.FULL, (63, 0, 0), (0, 0, 0), (100, 20, 0), (be.UNBOUNDED, 5, 0), (0, 0, 64), (64, 0, 50)])
def test_windows(gpu, dtype, l, t, window):
    q, kc, vc = case(l, dtype, 2, l, t, 8, 2, 128)
    pos = np.stack([np.arange(t - l, t), np.arange(100, 100 + l)])
    check(gpu, q, kc, vc, t, 0.1, window=window, positions=pos, kv_lengths=[t, t - 37])


@BOTH
@pytest.mark.parametrize("l", [1, 6, 140])
def test_rows_that_see_nothing_beside_rows_that_do(gpu, dtype, l):
    """Positions far behind a short sequence and a small window: an empty interval gives zeros, also beside rows of the same tile."""
    q, kc, vc = case(l, dtype, 2, l, 200, 8, 2, 64)
    pos = np.stack([np.where(np.arange(l) % 2 == 0, 150, 500), np.full(l, 90)])
    got = check(gpu, q, kc, vc, 200, 0.125, window=(40, 0, 0), positions=pos, kv_lengths=[200, 30])
    assert not got[1].any() and (l == 1 or not got[0, 1].any()) and got[0, 0].any()


@BOTH
@pytest.mark.parametrize("hq,hk,d", [(8, 1, 256), (16, 4, 64), (32, 8, 128)])
@pytest.mark.parametrize("t_cap,window", [(1, be.CAUSAL), (63, be.CAUSAL), (64, (30, 0, 0)), (150, be.CAUSAL), (150, (99, 0, 0)), (700, (511, 0, 0)), (700, be.CAUSAL)])
def test_rings(gpu, dtype, hq, hk, d, t_cap, window):
    lengths = [t_cap // 2 + 1, t_cap, t_cap + 1, 3 * t_cap + 7, 1000 * t_cap + t_cap // 3, 0]
    q, kc, vc = case(d + t_cap, dtype, len(lengths), 1, t_cap, hq, hk, d)
    for c in (kc, vc):
        c.scales[0, :, :, lengths[0]:] = 0x7E00
    check(gpu, q, kc, vc, t_cap, 1 / math.sqrt(d), window=window, positions=[[max(n - 1, 0)] for n in lengths], kv_lengths=lengths, rolling=True)


@BOTH
@pytest.mark.parametrize("l", [4, 150])
def test_rings_and_several_queries(gpu, dtype, l):
    t_cap = 260
    q, kc, vc = case(l, dtype, 2, l, t_cap, 8, 2, 128)
    lengths = [1000, l + 10]
    pos = np.stack([np.arange(n - l, n) for n in lengths])
    check(gpu, q, kc, vc, t_cap, 0.1, window=(99, 0, 0), positions=pos, kv_lengths=lengths, rolling=True)


@BOTH
@pytest.mark.parametrize("l,d", [(1, 128), (1, 96), (5, 64), (150, 128), (90, 256), (4, 96)])
def test_rings_as_far_as_an_index_goes(gpu, dtype, l, d):
    q, kc, vc = case(77 + l, dtype, 2, l, 170, 4, 2, d)
    lengths = [2147483647, 2147483647 - 40]
    check(gpu, q, kc, vc, 170, 0.1, window=(120, 0, 0), positions=[list(range(n - l, n)) for n in lengths], kv_lengths=lengths, rolling=True)


@BOTH
@pytest.mark.parametrize("l", [1, 5, 140])
@pytest.mark.parametrize("soft_cap,scale", [(30.0, 0.2), (5.0, 1.0), (0.0, -0.1), (0.0, 0.0)])
def test_soft_cap_and_odd_scales(gpu, dtype, l, soft_cap, scale):
    q, kc, vc = case(l, dtype, 1, l, 300, 8, 2, 64)
    check(gpu, q, kc, vc, 300, scale, soft_cap=soft_cap, positions=[np.arange(300 - l, 300)], kv_lengths=[300])


@BOTH
@pytest.mark.parametrize("l", [1, 140])
@pytest.mark.parametrize("hq,hk,d,dv", [(4, 2, 32, 32), (2, 1, 96, 160), (2, 2, 64, 128), (1, 1, 512, 32)])
def test_other_head_sizes(gpu, dtype, l, hq, hk, d, dv):
    q, kc, vc = case(d, dtype, 2, l, 150, hq, hk, d, dv)
    check(gpu, q, kc, vc, 150, 1 / math.sqrt(d), positions=[np.arange(150 - l, 150)] * 2, kv_lengths=[150, 149])


@BOTH
@pytest.mark.parametrize("l", [1, 150])
def test_no_index_operands(gpu, dtype, l):
    q, kc, vc = case(l, dtype, 2, l, 200, 8, 2, 128)
    check(gpu, q, kc, vc, 200, 0.1)
    check(gpu, q, kc, vc, 200, 0.1, window=be.FULL)


@BOTH
@pytest.mark.parametrize("l", [1, 150])
@pytest.mark.parametrize("q_size,k_size,v_size", [(1e4, 1e-4, 1.0), (1e-6, 1e4, 1e-4), (1.0, 1.0, 3e4), (300.0, 1.0, 1.0), (1e30, 1e-4, 1.0)])
def test_magnitudes(gpu, dtype, l, q_size, k_size, v_size):
    """Queries, keys and values far from one: nothing may leave a half-precision range on the way, and small scales keep their relative accuracy."""
    rng = np.random.default_rng(4)
    q, kc, vc = case(l, dtype, 1, l, 300, 8, 2, 64)
    for c, size in ((kc, k_size), (vc, v_size)):
        x = rng.standard_normal((300, 2, 64)).astype(np.float32) * np.float32(size)
        c.put(x, 0, range(300))
    scale = 0.125 if q_size == 300.0 else 0.3 / (q_size * k_size)
    check(gpu, (q * np.float32(q_size)).astype(np.float32), kc, vc, 300, scale, positions=[np.arange(300 - l, 300)], kv_lengths=[300])


@BOTH
@pytest.mark.parametrize("l", [1, 6])
def test_values_of_very_different_size_along_the_cache(gpu, dtype, l):
    """The scales of the values rise and fall by 2^15 along the cache: the sums follow."""
    rng = np.random.default_rng(6)
    q, kc, vc = case(l, dtype, 1, l, 1500, 8, 2, 128)
    size = np.exp2(rng.integers(-10, 6, 1500)).astype(np.float32)
    size[:64], size[700:800] = 2.0 ** -12, 2.0 ** 12
    vc.put(rng.standard_normal((1500, 2, 128)).astype(np.float32) * size[:, None, None], 0, range(1500))
    check(gpu, q, kc, vc, 1500, 0.1, positions=[np.arange(1500 - l, 1500)], kv_lengths=[1500])


@BOTH
@pytest.mark.parametrize("fill", [0x7B, 0xFB, 0x7C])
@pytest.mark.parametrize("l,d", [(1, 128), (5, 64), (150, 128), (90, 256), (300, 64)])
def test_large_scales_of_rows_nobody_sees(gpu, dtype, l, d, fill):
    """Behind the last row, and before a window, lie scales near f16's largest, of either sign, or NaN."""
    rng = np.random.default_rng(fill + l)
    t, rows = 700, 470
    q = rng.standard_normal((2, l, 4, d)).astype(np.float32)
    kc, vc = (filled(rng, dtype, 2, t, 2, d, 1.0, fill=fill, rows=rows) for _ in range(2))
    small = rng.standard_normal((rows, 2, d)).astype(np.float32) * np.float32(1e-3)
    for b in range(2):
        vc.put(small, b, range(rows))
    first = rows - l - 60
    for c in (kc, vc):
        c.scales[:, :, :, :first] = fill * 257
    pos = [np.arange(rows - l, rows)] * 2
    check(gpu, q, kc, vc, t, 0.1, positions=pos, kv_lengths=[rows, rows], window=(59, 0, 0))


@BOTH
@pytest.mark.parametrize("l", [1, 150])
def test_columns_of_very_different_size(gpu, dtype, l):
    """The blocks of the values lie 2^30 apart; each column is as exact as its own size asks for."""
    rng = np.random.default_rng(l)
    q, kc, vc = case(l, dtype, 1, l, 333, 4, 2, 128)
    size = np.repeat(np.float32([2.0 ** 12, 2.0 ** -16, 1.0, 2.0 ** -18]), 32)
    vc.put(rng.standard_normal((333, 2, 128)).astype(np.float32) * size, 0, range(333))
    check(gpu, q, kc, vc, 333, 0.1, positions=[np.arange(333 - l, 333)], kv_lengths=[333])


@BOTH
@pytest.mark.parametrize("l", [1, 5, 150])
def test_what_is_not_finite_stays_where_it_is_seen(gpu, dtype, l):
    """A NaN key or value is seen by the rows whose interval holds it, and by nobody else; of a value only its block's columns."""
    t = 260
    q, kc, vc = case(l, dtype, 1, l, t, 4, 2, 64)
    pos = 100 + np.arange(l) % 30
    pos[-1] = 250
    check(gpu, q, kc, vc, t, 0.125, positions=[pos], kv_lengths=[t], window=(20, 0, 0))
    want, bounds = attention_f64(q, kc.values(), vc.values(), 0.125, t, positions=[pos], kv_lengths=[t], window=(20, 0, 0))
    kc.scales[0, 0, 1, 240] = 0x7E00
    vc.scales[0, 1, 0, 245] = 0x7C00                             # an infinity
    got = step(gpu, q, kc, vc, t, 0.125, positions=[pos], kv_lengths=[t], window=(20, 0, 0))
    sees = [p for p in range(l) if pos[p] - 20 <= 240 <= pos[p]]
    assert sees == [l - 1]
    assert np.isnan(got[0, -1, :2]).all()
    assert not np.isfinite(got[0, -1, 2:, :32]).any()
    near = np.abs(got - want) <= bound_of(bounds)
    assert near[0, :-1].all() and near[0, -1, 2:, 32:].all()
    empty = step(gpu, q, kc, vc, t, 0.125, positions=[np.full(l, 100)], kv_lengths=[50], window=(20, 0, 0))
    assert not empty.any()


@BOTH
@pytest.mark.parametrize("bn,l,hq,hk,d,t", [(1, 1, 8, 1, 256, 5000), (1, 1, 32, 8, 128, 4100), (3, 1, 16, 4, 64, 3000), (1, 40, 8, 2, 128, 4000), (1, 200, 8, 1, 256, 3000)])
def test_long_caches_are_divided(gpu, dtype, bn, l, hq, hk, d, t):
    q, kc, vc = case(t, dtype, bn, l, t, hq, hk, d)
    lengths = [t - 700 * i for i in range(bn)]
    check(gpu, q, kc, vc, t, 1 / math.sqrt(d), positions=[np.arange(n - l, n) for n in lengths], kv_lengths=lengths)


def test_refusals(gpu):
    buf, x, out = gpu.zeros(1 << 20), gpu.zeros(1 << 16), gpu.zeros(1 << 16)
    none = be.DeviceBuffer(gpu, 0, 0)

    def refused(status, shape, k=buf, v=buf, **kw):
        with pytest.raises(be.AionHipError) as e:
            gpu.step_attention(out, x, k, v, shape, 0.1, **{"kv_dtype": be.Q8_0, **kw})
        assert e.value.status == status, e.value

    bad, no = be.hip.INVALID_ARGUMENT, be.hip.UNSUPPORTED
    refused(bad, (1, 1, 64, 2, 1, 48, 64))
    refused(bad, (1, 1, 64, 2, 1, 64, 40))
    refused(no, (1, 1, 64, 2, 1, 2048, 64))
    refused(bad, (1, 1, 64, 3, 2, 64, 64))
    refused(bad, (1, 1, 64, 2, 1, 64, 64), k=buf.view(8))
    refused(bad, (1, 1, 64, 2, 1, 64, 64), v=none)
    refused(no, (1, 1, 64, 2, 1, 64, 64), kv_dtype=be.I32)
    refused(no, (1, 1, 64, 2, 1, 64, 64), q_dtype=be.Q8_0)
    gpu.step_attention(out, x, buf, buf, (1, 0, 64, 2, 1, 64, 64), 0.1, kv_dtype=be.Q8_0)
    gpu.write(out, np.full(128, 3.0, np.float32))
    gpu.step_attention(out, x, buf, buf, (1, 1, 0, 2, 1, 64, 64), 0.1, kv_dtype=be.Q4_0)        # no keys at all: zeros
    assert not gpu.download(out, np.float32, (128,)).any()
    w = gpu.upload_weight(be.Q8_0, be.ROWS_NK, 32, 128, be.quantize_blocks(be.Q8_0, np.zeros((32, 128), np.float32), 1))
    assert gpu.step_attention_matmul(w, x, buf, buf, (1, 1, 64, 2, 1, 64, 64), 0.1, out, kv_dtype=be.Q8_0) is False
    w.free()
    for b in (buf, x, out):
        b.free()


@BOTH
def test_a_decode_recorded_and_replayed(gpu, dtype):
    """Append and attention of one token as a program: token by token, each replay against 64 bits, with eager work between the replays."""
    rng = np.random.default_rng(8)
    b, t_cap, hq, hk, d = 2, 200, 8, 2, 128
    kc, vc = (filled(rng, dtype, b, t_cap, hk, d, rows=100) for _ in range(2))
    bufs = [gpu.upload(c.bytes) for c in (kc, vc)]
    rows = [gpu.alloc(b * hk * d * 4) for _ in range(2)]
    q, out = gpu.alloc(b * hq * d * 4), gpu.alloc(b * hq * d * 4)
    index, lens, pos = (gpu.upload(np.zeros(b, np.int32)) for _ in range(3))

    def issue():
        gpu.step_append_quant(dtype, bufs, rows, index, (b, 1, t_cap, hk, d))
        gpu.step_attention(out, q, *bufs, (b, 1, t_cap, hq, hk, d, d), 0.1, kv_dtype=dtype, query_positions=pos, kv_lengths=lens)

    prog = None
    for i in range(6):
        at = np.array([100 + i, 30 + i], np.int32)
        new = [rng.standard_normal((b, 1, hk, d)).astype(np.float32) for _ in range(2)]
        qv = rng.standard_normal((b, 1, hq, d)).astype(np.float32)
        for buf, x in zip(rows + [q, index, lens, pos], new + [qv, at, at + 1, at]):
            gpu.write(buf, x)
        for c, x in zip((kc, vc), new):
            for j in range(b):
                c.put(x[j], j, [at[j]])
        if prog is None:
            issue()
            prog = gpu.record_program(issue)
        gpu.program_execute(prog)
        got = gpu.download(out, np.float32, (b, 1, hq, d))
        want, near = attention_f64(qv, kc.values(), vc.values(), 0.1, t_cap, positions=at[:, None], kv_lengths=at + 1)
        inside = bool((np.abs(got - want) <= bound_of(near)).all())
        assert inside, i
        issue()
        assert np.array_equal(gpu.download(out, np.float32, (b, 1, hq, d)), got)
    gpu.program_destroy(prog)
    for x in bufs + rows + [q, out, index, lens, pos]:
        x.free()


@BOTH
def test_two_programs_of_one_context(gpu, dtype):
    """A chunk of a prompt and a token as programs that share the context's work buffers, replayed in turn: appended rows, attention, rows read back."""
    rng = np.random.default_rng(9)
    t_cap, hq, hk, d = 1500, 8, 2, 128
    kc, vc = (filled(rng, dtype, 1, t_cap, hk, d, rows=900) for _ in range(2))
    bufs = [gpu.upload(c.bytes) for c in (kc, vc)]
    index, lens = (gpu.upload(np.zeros(1, np.int32)) for _ in range(2))
    calls = {}
    for s in (150, 1):
        rows, back = [[gpu.alloc(s * hk * d * 4) for _ in range(2)] for _ in range(2)]
        q, out, pos = gpu.alloc(s * hq * d * 4), gpu.alloc(s * hq * d * 4), gpu.alloc(s * 4)

        def issue(s=s, rows=rows, back=back, q=q, out=out, pos=pos):
            gpu.step_append_quant(dtype, bufs, rows, index, (1, s, t_cap, hk, d))
            gpu.step_attention(out, q, *bufs, (1, s, t_cap, hq, hk, d, d), 0.1, kv_dtype=dtype, query_positions=pos, kv_lengths=lens)
            gpu.step_cache_read(dtype, back, bufs, index, (1, s, t_cap, hk, d))
        calls[s] = (issue, rows, back, q, out, pos)
        issue()
    for c, buf in zip((kc, vc), bufs):
        gpu.write(buf, c.bytes)
    progs = {s: gpu.record_program(calls[s][0]) for s in calls}
    at = 900
    for s in (150, 1, 1, 150, 1):
        _, rows, back, q, out, pos = calls[s]
        new = [rng.standard_normal((1, s, hk, d)).astype(np.float32) for _ in range(2)]
        qv = rng.standard_normal((1, s, hq, d)).astype(np.float32)
        steps = np.arange(at, at + s, dtype=np.int32)
        for buf, x in zip(rows + [q, index, lens, pos], new + [qv, steps[:1], steps[-1:] + 1, steps]):
            gpu.write(buf, x)
        for c, x in zip((kc, vc), new):
            c.put(x[0], 0, steps)
        gpu.program_execute(progs[s])
        got = gpu.download(out, np.float32, qv.shape)
        want, near = attention_f64(qv, kc.values(), vc.values(), 0.1, t_cap, positions=[steps], kv_lengths=[at + s])
        inside = bool((np.abs(got - want) <= bound_of(near)).all())
        assert inside, (at, s)
        for c, buf, o in zip((kc, vc), bufs, back):
            assert np.array_equal(gpu.download(buf, np.uint8, c.bytes.shape), c.bytes)
            assert np.array_equal(gpu.download(o, np.float32, (s, hk, d)), c.values()[0, steps].astype(np.float32))
        at += s
    for p in progs.values():
        gpu.program_destroy(p)
    for x in bufs + [index, lens] + [y for _, rows, back, q, out, pos in calls.values() for y in rows + back + [q, out, pos]]:
        x.free()


@BOTH
@pytest.mark.parametrize("l,t,hq,hk,d", [(1, 4000, 8, 1, 256), (300, 1000, 16, 8, 128), (1100, 2200, 16, 4, 64), (40, 600, 4, 4, 96)])
def test_recorded_without_having_run(dtype, l, t, hq, hk, d):
    fresh = be.HipBackend(0)
    q, kc, vc = case(3, dtype, 1, l, t, hq, hk, d)
    bufs = [fresh.upload(x) for x in (q, kc.bytes, vc.bytes)]
    pos, lens, out = fresh.upload(np.arange(t - l, t, dtype=np.int32)), fresh.upload(np.array([t], np.int32)), fresh.zeros(q.nbytes)

    def issue():
        fresh.step_attention(out, *bufs, (1, l, t, hq, hk, d, d), 0.1, kv_dtype=dtype, query_positions=pos, kv_lengths=lens)

    prog = fresh.record_program(issue)
    want, near = attention_f64(q, kc.values(), vc.values(), 0.1, t, positions=[np.arange(t - l, t)], kv_lengths=[t])
    for _ in range(3):
        fresh.write(out, np.full(q.shape, np.nan, np.float32))
        fresh.program_execute(prog)
        got = fresh.download(out, np.float32, q.shape)
        inside = bool((np.abs(got - want) <= bound_of(near)).all())
        assert inside
    issue()
    assert np.array_equal(fresh.download(out, np.float32, q.shape), got)
    fresh.program_destroy(prog)
    fresh.close()


@BOTH
@pytest.mark.parametrize("d", [256, 128, 96])
def test_offsets_beyond_32_bits(gpu, dtype, d):
    """The last rows of caches of more than 4 GiB of codes: appended, read back, attended to; against the same rows in a small cache."""
    rng = np.random.default_rng(d)
    hq, hk, s, tail = 4, 2, 260, 300
    t_cap = (1 << 32) // (d if dtype == be.Q8_0 else d // 2) // hk + 40000
    size = gpu.cache_quant_bytes(dtype, 1, t_cap, hk, d)
    bufs = [gpu.alloc(size) for _ in range(2)]
    new = [rng.standard_normal((1, s, hk, d)).astype(np.float32) for _ in range(2)]
    small = [QuantCache(dtype, 1, tail, hk, d) for _ in range(2)]
    for c, x in zip(small, new):
        c.put(x[0], 0, np.arange(tail - s, tail))
    rows = [gpu.upload(x) for x in new]
    index = gpu.upload(np.array([t_cap - s], np.int32))
    gpu.step_append_quant(dtype, bufs, rows, index, (1, s, t_cap, hk, d))
    backs = [gpu.alloc(x.nbytes) for x in new]
    gpu.step_cache_read(dtype, backs, bufs, index, (1, s, t_cap, hk, d))
    for o, c in zip(backs, small):
        assert np.array_equal(gpu.download(o, np.float32, (s, hk, d)), c.values()[0, tail - s:tail].astype(np.float32))
    for l in (1, 9, 150):
        q = rng.standard_normal((1, l, hq, d)).astype(np.float32)
        pos = np.arange(tail - l, tail)
        want, near = attention_f64(q, small[0].values(), small[1].values(), 0.1, tail, window=(100, 0, 0), positions=[pos], kv_lengths=[tail])
        up, out = gpu.upload(q), gpu.alloc(q.nbytes)
        at, length = gpu.upload((pos + t_cap - tail).astype(np.int32)), gpu.upload(np.array([t_cap], np.int32))
        gpu.step_attention(out, up, *bufs, (1, l, t_cap, hq, hk, d, d), 0.1, kv_dtype=dtype, window=(100, 0, 0), query_positions=at, kv_lengths=length)
        inside = bool((np.abs(gpu.download(out, np.float32, q.shape) - want) <= bound_of(near)).all())
        assert inside, l
        for x in (up, out, at, length):
            x.free()
    for x in bufs + rows + backs + [index]:
        x.free()
