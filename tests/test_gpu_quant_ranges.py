"""Attention over caches held in 8 or 4 bits at the ends of its ranges: keys that outweigh all others and have no values, against 64 bits.

The bounds are those of test_gpu_attention_quant.py and what a probability is held to when the largest of its row meets a value of zero. Few rows: the product of a
probability and a scale is the sum of two half-precision numbers, truncated at 2^-24 or relative to its size, where the row's largest probability is at most 2^80; a code
is at most 128: keys * 2^-97 of an output. Many rows: probabilities alone are truncated at 2^-24, the row's largest being at least 2^7: keys * 2^-31 * max|v|.
"""
import numpy as np
import pytest

from aion_amd import backend as be
from quant_cases import attention_f64, filled
from test_gpu_attention_quant import BOTH, bound_of, step

pytestmark = pytest.mark.gpu


def peaked(rng, dtype, t, hk, d, gap, keys):
    """Keys whose scores against queries near one are near zero, `gap` at the places in `keys` (softmax scale d^-1/2)."""
    c = filled(rng, dtype, 1, t, hk, d, 0.02)
    c.put(np.full((len(keys), hk, d), gap / np.sqrt(d), np.float32), 0, keys)
    return c


def queries(rng, l, hq, d):
    return (1 + 0.01 * rng.standard_normal((1, l, hq, d))).astype(np.float32)


@BOTH
@pytest.mark.parametrize("d", [64, 96, 128, 256])
@pytest.mark.parametrize("l,t,best,second", [
    (1, 60, 5, None), (1, 60, 40, 41), (1, 500, 3, 270), (1, 500, 3, 80), (1, 4100, 100, 4000), (3, 500, 5, None), (3, 500, 5, 330), (5, 60, 7, 8), (5, 500, 3, 270),
    (5, 4100, 4000, 90), (40, 500, 3, 400), (150, 500, 3, 400)])
def test_the_best_key_has_no_values(gpu, dtype, d, l, t, best, second):
    """Its scales are zero in one block or in all, the other keys' scores lie `gap` below; `second` is as strong and has values: in the same tile, in a later one
    of the same wavefront, in another wavefront, in another segment."""
    rng = np.random.default_rng(t + l + d)
    hq, hk = 4, 2
    q = queries(rng, l, hq, d)
    vc = filled(rng, dtype, 1, t, hk, d)
    for empty in (slice(0, 1), slice(None)):
        vc.scales[0, :, empty, best] = 0
        values = vc.values()
        lost = t * 2.0 ** -97
        if l * hq // hk > (64 if d == 256 else 128) and d != 96:
            lost += t * 2.0 ** -31 * np.abs(values[:, :t]).max()
        for gap in (20, 60, 70, 75, 80, 88, 92, 97, 110, 150, 200):
            kc = peaked(rng, dtype, t, hk, d, gap, [best] if second is None else [best, second])
            got = step(gpu, q, kc, vc, t, d ** -0.5, window=be.FULL)
            want, near = attention_f64(q, kc.values(), values, d ** -0.5, t, window=be.FULL)
            inside = bool((np.abs(got - want) <= bound_of(near) + lost).all())
            assert inside, (gap, gpu.last_kernel(), float(np.abs(got - want).max()), bool(np.isfinite(got).all()))


@BOTH
@pytest.mark.parametrize("size", [1.0, 300.0, 1e4])
@pytest.mark.parametrize("what", [0x7C00, 0x7E00])
@pytest.mark.parametrize("l,d", [(1, 64), (1, 128), (1, 256), (3, 128), (3, 256), (6, 64), (7, 128), (30, 128), (30, 256), (150, 128), (150, 256), (5, 96)])
def test_a_block_that_is_not_finite_leaves_the_others_their_range(gpu, dtype, l, d, what, size):
    """A value that every row sees has no finite scale in one block, at the first key or at a later one; the other blocks' scales are below and above one."""
    rng = np.random.default_rng(l + d)
    t, hq, hk, blocks = 400, 4, 2, d // 32
    q = rng.standard_normal((1, l, hq, d)).astype(np.float32)
    kc, vc = filled(rng, dtype, 1, t, hk, d), filled(rng, dtype, 1, t, hk, d, size)
    want, near = attention_f64(q, kc.values(), vc.values(), 0.1, t, window=be.FULL)
    assert np.isfinite(want).all()                                # (scales that f16 holds)
    for key in (0, 130):
        for block in (0, blocks - 1):
            held = vc.scales[0, :, block, key].copy()
            vc.scales[0, :, block, key] = what
            got = step(gpu, q, kc, vc, t, 0.1, window=be.FULL).reshape(1, l, hq, blocks, 32)
            vc.scales[0, :, block, key] = held
            others = [j for j in range(blocks) if j != block]
            gone = not np.isfinite(got[..., block, :]).any()
            near_enough = (np.abs(got.reshape(want.shape) - want) <= bound_of(near)).reshape(got.shape)[..., others, :].all()
            assert gone and near_enough, (key, block, gone, gpu.last_kernel())
