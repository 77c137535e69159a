"""The decoder over caches in pages: recorded and eager steps, turning, eviction while it decodes."""
import numpy as np
import pytest

from aion_amd import backend as be
from aion_amd.decoder import Decoder, DecoderConfig, SessionDecoder, SyntheticWeights
from paged_cases import turned_close

SHAPE = dict(layers=2, hidden=256, heads=4, kv_heads=2, head_dim=64, ffn=512, vocab=1024)


def both(gpu, cfg, other=None, seed=7):
    w = SyntheticWeights(cfg, seed)
    return Decoder(gpu, cfg, w), Decoder(gpu, other or cfg, w)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [be.F16, be.BF16])
@pytest.mark.parametrize("rotary", [None, be.Rotary(48, base=500000.0, interleaved=True, scaling=be.ROTARY_BANDS, factor=8.0, original_length=64.0, low=1.0, high=4.0)])
def test_recorded_steps_are_the_eager_ones(gpu, dtype, rotary):
    cfg = DecoderConfig(max_seq=150, page_rows=16, cache_dtype=dtype, rotary=rotary, **SHAPE)
    a, b = both(gpu, cfg)
    try:
        prompt = np.random.default_rng(4).integers(0, cfg.vocab, 90).astype(np.int32)
        ta, tb = a.prefill(prompt), b.prefill(prompt)
        assert ta == tb and np.array_equal(a.logits_host(), b.logits_host()) and np.isfinite(a.logits_host()).all()
        a.begin_decode(ta)
        for step in range(6):
            ta, tb = a.decode_step(), b.decode_step_eager(tb)
            assert np.array_equal(a.logits_host(), b.logits_host()), step
            assert ta == tb, step
        # the first block's keys, from the embedding alone: norm and projection as separate steps, turned in 64 bits
        n, g = prompt.size, gpu
        x, k = g.alloc(n * cfg.hidden * 4), g.alloc(n * cfg.kv_dim * 4)
        ids, zero = g.upload(prompt), g.upload(np.zeros(1, np.int32))
        g.step_gather_rows(be.F32, x, a.embed, ids, n, cfg.hidden, cfg.vocab)
        g.step_rmsnorm_matmul([a.w["l0.wk"]], x, a.gamma, n, [k], cfg.eps)
        rows = g.download(k, np.float32, (1, n, cfg.kv_heads, cfg.head_dim)).astype(np.float64)
        ko, vo = g.alloc(n * cfg.kv_dim * 4), g.alloc(n * cfg.kv_dim * 4)
        g.step_read_paged(a.caches[0], ko, vo, zero, n)
        got = g.download(ko, np.float32, rows.shape).astype(np.float64)
        assert turned_close(got, rows, np.arange(n)[None], a.rotary, dtype).all()
        for buf in (x, k, ids, zero, ko, vo):
            buf.free()
    finally:
        a.close()
        b.close()


@pytest.mark.gpu
def test_pages_and_linear_caches_agree(gpu):
    """The same keys and values but for the angles' f32 roundings (2^-24 of a position's radians) and the queries' in linear attention (off here: the precise mode). What is left is
    int8 codes of activations that lie beside a half, one step of 127 to a block of 32: held to a tenth of the logits' spread, where a wrong row moves them by all of it."""
    linear = DecoderConfig(max_seq=150, **SHAPE)
    a, b = both(gpu, linear, DecoderConfig(max_seq=150, page_rows=32, **SHAPE))
    gpu.set_attention_precise(True)
    try:
        prompt = np.random.default_rng(5).integers(0, linear.vocab, 77).astype(np.int32)
        a.prefill(prompt)
        b.prefill(prompt)
        x, y = a.logits_host(), b.logits_host()
        assert np.abs(x - y).max() <= 0.1 * x.std()
    finally:
        gpu.set_attention_precise(False)
        a.close()
        b.close()


@pytest.mark.gpu
def test_eviction_that_never_comes_changes_nothing(gpu):
    plain = DecoderConfig(max_seq=150, page_rows=16, **SHAPE)
    a, b = both(gpu, plain, DecoderConfig(max_seq=150, page_rows=16, evict_keep=40, **SHAPE))
    try:
        prompt = np.random.default_rng(6).integers(0, plain.vocab, 70).astype(np.int32)
        ta, tb = a.prefill(prompt), b.prefill(prompt)
        a.begin_decode(ta)
        b.begin_decode(tb)
        assert np.array_equal(a.decode_run(20), b.decode_run(20)) and np.array_equal(a.logits_host(), b.logits_host())
        total = sum(gpu.download(w, np.float32).sum() for w in b.drawn)
        # (every head of every query that was asked draws one in all: the prompt's last 64, then 20)
        assert abs(total - plain.layers * plain.heads * (64 + 20)) <= 1e-2
    finally:
        a.close()
        b.close()


@pytest.mark.gpu
def test_a_text_longer_than_the_caches(gpu):
    cfg = DecoderConfig(max_seq=64, page_rows=16, evict_keep=32, evict_limit=48, evict_recent=12, **SHAPE)
    a, b = both(gpu, cfg)
    try:
        rng = np.random.default_rng(9)
        first, second = rng.integers(0, cfg.vocab, 60).astype(np.int32), rng.integers(0, cfg.vocab, 10).astype(np.int32)
        for d in (a, b):
            d.prefill(first)
            assert d.rows == 32 and d.pos == 60
        ta, tb = a.prefill(second), b.prefill(second)
        assert ta == tb and a.rows == 42
        a.begin_decode(ta)
        tokens = a.decode_run(100)
        for step in range(100):
            tb = b.decode_step_eager(tb)
            assert tokens[step] == tb, step
        assert np.array_equal(a.logits_host(), b.logits_host()) and np.isfinite(a.logits_host()).all()
        assert a.pos == 170 and a.rows == b.rows and cfg.evict_keep <= a.rows <= 48
        state = a._buffers(1)
        assert gpu.download(state["write_index"], np.int32)[0] == a.rows and gpu.download(state["kv_len"], np.int32)[0] == a.rows + 1
        # a new text begins as the first did
        before = tokens
        for d in (a, b):
            d.reset()
            d.prefill(first)
        a.begin_decode(a.prefill(second))
        assert np.array_equal(a.decode_run(100), before)
        with pytest.raises(ValueError):
            b.prefill(np.zeros(40, np.int32))
    finally:
        a.close()
        b.close()


def test_configurations_that_are_none():
    cfg = lambda **kw: DecoderConfig(max_seq=64, **SHAPE, **kw)  # noqa: E731
    with pytest.raises(ValueError):
        cfg(page_rows=16, cache_dtype=be.Q4_0).cache_bytes(None)
    with pytest.raises(ValueError):
        cfg(evict_keep=8).eviction()
    with pytest.raises(ValueError):
        cfg(page_rows=16, evict_keep=8, evict_limit=64).eviction()
    with pytest.raises(ValueError):
        cfg(page_rows=16, evict_keep=40, evict_limit=32).eviction()
    with pytest.raises(ValueError):
        SessionDecoder(None, cfg(page_rows=16), None)
    assert cfg(page_rows=16, evict_keep=8).eviction() == (8, 63, 4, 2) and cfg(page_rows=16, evict_keep=3).eviction() == (3, 63, 3, 0) and cfg().eviction() is None
