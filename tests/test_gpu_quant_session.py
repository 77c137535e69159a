"""Which steps of a session's list a tensor marked as a quantized cache may be an operand of: the mark stands for a layout of its own, of as many bytes as aion's
blocks where the capacity is a multiple of 64."""
import numpy as np
import pytest

from aion_amd import backend as be
from aion_amd import session as ss

pytestmark = pytest.mark.gpu


def refused(gpu, steps):
    sess = ss.Session(gpu)
    with pytest.raises(be.AionHipError) as e:
        sess.execute(steps)
    assert e.value.status == be.hip.INVALID_ARGUMENT, e.value
    sess.close()


@pytest.mark.parametrize("dtype", [be.Q8_0, be.Q4_0])
def test_a_copy_keeps_the_layout(gpu, dtype):
    shape = (2, 64, 2, 64)
    n = gpu.cache_quant_bytes(dtype, *shape)
    assert n == 2 * 64 * 2 * 64 // 32 * (34 if dtype == be.Q8_0 else 18)
    data = np.random.default_rng(0).integers(0, 256, n).astype(np.uint8)
    src, dst = gpu.upload(data), gpu.zeros(n)

    def copy(a, a_cache, b, b_cache):
        p = ss.Steps()
        p.copy(ss.tensor(src, dtype, a, quant_cache=a_cache), ss.tensor(dst, dtype, b, quant_cache=b_cache))
        return p

    refused(gpu, copy(shape, True, shape, False))
    refused(gpu, copy(shape, False, shape, True))
    for other in ((1, 128, 2, 64), (2, 64, 1, 128), (2, 64, 4, 32), (1, 64, 4, 64)):        # as many bytes, in another order
        assert gpu.cache_quant_bytes(dtype, *other) == n
        refused(gpu, copy(shape, True, other, True))
    assert not gpu.download(dst, np.uint8, (n,)).any()
    sess = ss.Session(gpu)
    for cache in (True, False):
        sess.execute(copy(shape, cache, shape, cache))
        assert np.array_equal(gpu.download(dst, np.uint8, (n,)), data)
        gpu.write(dst, np.zeros(n, np.uint8))
    sess.close()
    src.free()
    dst.free()


def test_no_other_step_takes_a_cache(gpu):
    buf, out, ids = gpu.zeros(1 << 16), gpu.zeros(1 << 16), gpu.zeros(256)
    mark = lambda dtype, *shape: ss.tensor(buf, dtype, shape, quant_cache=True)  # noqa: E731
    f32, i32 = (lambda *s: ss.tensor(out, be.F32, s)), (lambda *s: ss.tensor(ids, be.I32, s))
    lists = []
    for add in (lambda p: p.matmul(f32(1, 64), mark(be.Q4_0, 64, 32), f32(1, 32)),                       # a weight
                lambda p: p.gather_rows(mark(be.Q8_0, 64, 64), i32(1, 1), f32(1, 1, 64)),               # a table
                lambda p: p.rope1d(mark(be.F32, 1, 1, 2, 64), i32(1, 1), f32(1, 1, 2, 64)),             # queries
                lambda p: p.copy(mark(be.F16, 1, 64, 2, 64), mark(be.F16, 1, 64, 2, 64)),               # no block type
                lambda p: p.copy(mark(be.Q8_0, 64, 64), mark(be.Q8_0, 64, 64)),                         # not four axes
                lambda p: p.sequence_append(ss.tensor(out, be.F16, (1, 64, 2, 64)), mark(be.Q8_0, 1, 1, 2, 64), i32(1)),
                lambda p: p.attention(mark(be.Q8_0, 1, 1, 2, 64), ss.tensor(buf, be.F16, (1, 64, 2, 64)), ss.tensor(buf, be.F16, (1, 64, 2, 64)), f32(1, 1, 2, 64), 0.1),
                lambda p: p.attention(f32(1, 1, 2, 64), mark(be.F16, 1, 64, 2, 64), mark(be.F16, 1, 64, 2, 64), f32(1, 1, 2, 64), 0.1)):
        p = ss.Steps()
        add(p)
        lists.append(p)
    for p in lists:
        refused(gpu, p)
    for b in (buf, out, ids):
        b.free()
