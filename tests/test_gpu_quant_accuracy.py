"""Attention over caches held in 8 or 4 bits: what the header promises - about 1e-6 of the result for numbers of ordinary size - and the forms that the other tests of
it leave out: half-precision queries of more than one token, and values that rise and fall along a cache of many query rows."""
import numpy as np
import pytest

from aion_amd import backend as be
from quant_cases import attention_f64, filled
from test_gpu_attention_quant import BOTH, as_queries, bound_of, case, step

pytestmark = pytest.mark.gpu

# The norm of the error over the norm of the result. What is rounded: a probability and (many rows) a value as the sum of two half-precision numbers, both truncated,
# 2^-20 of it at most and a quarter of that on average, the smallest product of two such pairs left out, as much again, and f32 sums; all of them far below 2^-20
# of the norm where they do not point the same way. Two bf16 in their place give 3e-6.
PROMISED = 1e-6


def relative(got, want):
    return float(np.linalg.norm(got - want) / np.linalg.norm(want))


@BOTH
@pytest.mark.parametrize("q_dtype", [be.F32, be.F16, be.BF16])
@pytest.mark.parametrize("l,hq,hk,d", [(5, 16, 4, 64), (5, 8, 2, 128), (5, 8, 1, 256), (40, 4, 2, 64), (40, 4, 1, 128), (40, 2, 2, 256), (150, 8, 4, 64), (150, 4, 2, 128),
                                       (150, 2, 1, 256), (1100, 2, 1, 64), (1100, 2, 2, 128), (1100, 1, 1, 256), (5, 4, 2, 96), (150, 2, 1, 96)])
def test_several_queries_of_every_type(gpu, dtype, q_dtype, l, hq, hk, d):
    """Positions as a chunk has them: the last `l` of t tokens."""
    t = l + 333
    q, kc, vc = case(l + d, dtype, 1, l, t, hq, hk, d)
    up, exact = as_queries(q, q_dtype)
    options = {"positions": [np.arange(t - l, t)], "kv_lengths": [t]}
    want, near = attention_f64(exact, kc.values(), vc.values(), d ** -0.5, t, **options)
    got = step(gpu, up, kc, vc, t, d ** -0.5, q_dtype, **options)
    print("  %s relative error %.1e" % (gpu.last_kernel(), relative(got, want)), flush=True)
    inside = bool((np.abs(got - want) <= bound_of(near)).all())
    assert inside and relative(got, want) <= PROMISED


@BOTH
@pytest.mark.parametrize("l,d", [(1, 64), (1, 128), (1, 256), (6, 128), (30, 64), (30, 128), (30, 256), (200, 64), (200, 128), (200, 256)])
def test_the_promised_accuracy(gpu, dtype, l, d):
    t = 1500
    q, kc, vc = case(l, dtype, 1, l, t, 8, 2, d)
    options = {"positions": [np.arange(t - l, t)], "kv_lengths": [t]}
    want, _ = attention_f64(q, kc.values(), vc.values(), d ** -0.5, t, **options)
    got = step(gpu, q, kc, vc, t, d ** -0.5, **options)
    print("  %s relative error %.1e" % (gpu.last_kernel(), relative(got, want)), flush=True)
    assert relative(got, want) <= PROMISED


@BOTH
@pytest.mark.parametrize("l", [1, 150])
@pytest.mark.parametrize("soft_cap", [5.0, 50.0])
def test_the_promised_accuracy_under_a_soft_cap(gpu, dtype, l, soft_cap):
    """A capped score is off by up to 2^-22 of the cap, and the probability it makes by as much of itself."""
    t = 1500
    q, kc, vc = case(l, dtype, 1, l, t, 8, 2, 128)
    options = {"positions": [np.arange(t - l, t)], "kv_lengths": [t], "soft_cap": soft_cap}
    want, _ = attention_f64(q, kc.values(), vc.values(), 128 ** -0.5, t, **options)
    assert relative(step(gpu, q, kc, vc, t, 128 ** -0.5, **options), want) <= PROMISED + 2.0 ** -22 * soft_cap


@BOTH
@pytest.mark.parametrize("l,d,window", [(150, 128, be.CAUSAL), (300, 128, be.CAUSAL), (300, 64, (40, 0, 0)), (300, 128, (40, 0, 0)), (300, 256, (40, 0, 0)), (600, 128, (7, 0, 0))])
def test_values_of_very_different_size_along_many_rows(gpu, dtype, l, d, window):
    """Behind a window some rows see small values only, beside rows of the same workgroup that see large ones: what they get is held to 2^-40 of the largest value that
    any of up to 256 neighbouring rows sees in the same 32 columns, for each key that they see."""
    rng = np.random.default_rng(l + d)
    t, hq, hk = 1500, 4, 2
    q, kc, vc = case(l, dtype, 1, l, t, hq, hk, d)
    size = np.exp2(rng.integers(-12, 5, t)).astype(np.float32)
    size[t - l:t - l + 100] = 2.0 ** -12                                        # (whole windows of small values)
    size[t - 60:t - 50] = 2.0 ** 8
    vc.put(rng.standard_normal((t, hk, d)).astype(np.float32) * size[:, None, None], 0, range(t))
    options = {"positions": [np.arange(t - l, t)], "kv_lengths": [t], "window": window}
    want, near = attention_f64(q, kc.values(), vc.values(), d ** -0.5, t, **options)
    got = step(gpu, q, kc, vc, t, d ** -0.5, **options)
    keys = min(t, window[0] + 1) if window != be.CAUSAL else t
    held = 2.0 ** -40 * keys * np.abs(vc.values()[:, :t]).max()
    inside = bool((np.abs(got - want) <= bound_of(near) + held).all())
    assert inside and np.isfinite(got).all()


@BOTH
@pytest.mark.parametrize("hq,hk,d", [(8, 1, 256), (32, 8, 128), (16, 4, 64)])
@pytest.mark.parametrize("t,most", [(200, 40), (900, 6)])
def test_a_sequences_bits_do_not_depend_on_its_batch(gpu, dtype, hq, hk, d, t, most):
    """As long as the key segments that a capacity asks for, one to 256 keys (128 at head size 256), fit two to a CU."""
    segments = -(-t // (128 if d == 256 else 256))
    most = min(most, 512 // (segments * hk))
    q, kc, vc = case(t, dtype, most, 1, t, hq, hk, d)
    lengths = [t - 7 * i for i in range(most)]
    options = lambda n: {"positions": [[x - 1] for x in lengths[:n]], "kv_lengths": lengths[:n]}  # noqa: E731
    whole = step(gpu, q, kc, vc, t, d ** -0.5, **options(most))
    for n in (1, 2, most // 2):
        part_k, part_v = (filled(np.random.default_rng(0), dtype, n, t, hk, d) for _ in range(2))
        for part, c in ((part_k, kc), (part_v, vc)):
            part.codes[:], part.scales[:] = c.codes[:n], c.scales[:n]
        assert np.array_equal(step(gpu, q[:n], part_k, part_v, t, d ** -0.5, **options(n)), whole[:n])
