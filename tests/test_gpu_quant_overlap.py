"""Rows that lie in a cache which the same call writes or reads are refused, before anything is launched."""
import numpy as np
import pytest

from aion_amd import backend as be

pytestmark = pytest.mark.gpu


def test_rows_in_a_cache(gpu):
    b, s, t, h, d = 1, 2, 64, 2, 64
    shape, rows = (b, s, t, h, d), b * s * h * d * 4
    n = gpu.cache_quant_bytes(be.Q8_0, b, t, h, d)
    arena, x, i = gpu.zeros(2 * n + 8 * rows), gpu.zeros(8 * rows), gpu.zeros(64)
    kc, vc, behind = arena.view(0), arena.view(n), arena.view(2 * n)                # two caches, and what follows them
    last = arena.view(2 * n - 16)                                                    # the end of the second
    q_out, q, k, v = (x.view(j * rows) for j in range(4))

    def refused(f, *args, **kw):
        with pytest.raises(be.AionHipError) as e:
            f(*args, **kw)
        assert e.value.status == be.hip.INVALID_ARGUMENT, e.value

    for bad in (kc, last):
        refused(gpu.step_append_quant, be.Q8_0, [kc, vc], [bad, x], i, shape)
        refused(gpu.step_append_quant, be.Q8_0, [kc, vc], [x, bad], i, shape)
        refused(gpu.step_cache_read, be.Q8_0, [bad, x], [kc, vc], i, shape)
        refused(gpu.step_cache_read, be.Q8_0, [x, bad], [kc, vc], i, shape)
        for place in range(4):
            ops = [q_out, q, k, v]
            ops[place] = bad
            refused(gpu.step_rope_append_quant, be.Q8_0, *ops, kc, vc, i, i, b, s, t, h, h, d)
        refused(gpu.step_attention, bad, q, kc, vc, (b, s, t, h, h, d, d), 0.1, kv_dtype=be.Q8_0)
    refused(gpu.step_append_quant, be.Q8_0, [vc], [last], i, shape)
    assert not gpu.download(arena, np.uint8, (2 * n + 8 * rows,)).any() and not gpu.download(x, np.uint8, (8 * rows,)).any()
    # right behind them is no overlap
    gpu.step_append_quant(be.Q8_0, [kc, vc], [behind, x], i, shape)
    gpu.step_cache_read(be.Q8_0, [behind, x], [kc, vc], i, shape)
    gpu.step_rope_append_quant(be.Q8_0, behind, q, k, v, kc, vc, i, i, b, s, t, h, h, d)
    gpu.step_attention(behind, q, kc, vc, (b, s, t, h, h, d, d), 0.1, kv_dtype=be.Q8_0)
    gpu.sync()
    for buf in (arena, x, i):
        buf.free()
