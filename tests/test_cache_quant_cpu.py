"""Caches held in 8 or 4 bits: what needs no GPU - the size of a cache, and the tests' own host form of it."""
import numpy as np
import pytest

from aion_amd import backend as be
from aion_amd import hip
from quant_cases import QuantCache, padded


def size(*a):
    return hip.load_library().aionhip_cache_quant_bytes(*a)


@pytest.mark.parametrize("dtype", [be.Q8_0, be.Q4_0])
@pytest.mark.parametrize("b,t,h,d", [(1, 1, 1, 32), (3, 64, 2, 64), (2, 65, 5, 96), (1, 4095, 8, 128), (64, 131072, 8, 256)])
def test_size(dtype, b, t, h, d):
    per = d * (8 if dtype == be.Q8_0 else 4) // 8 + d // 32 * 2
    assert size(dtype, b, t, h, d) == b * h * padded(t) * per
    if b * t < 10000:
        assert QuantCache(dtype, b, t, h, d).bytes.size == size(dtype, b, t, h, d)


def test_sizes_out_of_range():
    assert size(be.F16, 1, 64, 1, 64) == 0 and size(be.Q8_0, 1, 64, 1, 48) == 0
    for i in range(1, 5):
        shape = [1, 64, 1, 64]
        shape[i - 1] = 0
        assert size(be.Q4_0, *shape) == 0
    assert size(be.Q8_0, 1, 1 << 31, 1, 64) == 0 and size(be.Q8_0, 1, 64, 65536, 64) == 0 and size(be.Q8_0, 1, 64, 1, 65536) == 0
    assert size(be.Q8_0, 1 << 62, 64, 1, 64) == 0 and size(be.Q8_0, 1 << 40, 1 << 30, 60000, 65504) == 0
    # past 32 bits
    assert size(be.Q4_0, 1, 0x7FFFFFC0, 8, 128) == 0x7FFFFFC0 * 8 * 72


@pytest.mark.parametrize("dtype", [be.Q8_0, be.Q4_0])
def test_host_form_against_the_oracles_blocks(orc, dtype):
    """The block quantizers' codes and scales, but where a product by 1 / 7 (1 / 127) and a quotient round to different f16 scales."""
    rng = np.random.default_rng(3)
    x = rng.standard_normal((700, 3, 64)).astype(np.float32)
    x[5, 1, :32] = 0.0
    c = QuantCache(dtype, 1, 700, 3, 64)
    c.put(x, 0, range(700))
    got = c.values()[0, :700]
    want = orc.dequantize(dtype, orc.quantize(dtype, x.reshape(-1, 32), 1), (700 * 3 * 2, 32), 1).reshape(700, 3, 64).astype(np.float64)
    # one f16 step of the scale (2^-10 at most), which moves an 8-bit code by less than an eighth, so by one at most; 4-bit codes go by the unrounded scale
    other = (got != want).reshape(700, 3, 2, 32).any(-1)
    top = np.abs(x.reshape(700, 3, 2, 32)).max(-1)
    assert other.mean() < 1e-2 and (np.abs(got - want).reshape(700, 3, 2, 32).max(-1) <= top * (1.0 / 127 + 2.0 ** -10)).all()
    half_step = 0.5 / (127 if dtype == be.Q8_0 else 7) + 2.0 ** -10                # of the block's maximum; the scale is an f16
    assert (np.abs(x - got).reshape(700, 3, 2, 32).max(-1) <= top * half_step).all()
