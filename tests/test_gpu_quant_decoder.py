"""Caches held in 8 or 4 bits where a program meets them: as tensors of a session's step list, and in the decoders."""
import numpy as np
import pytest

from aion_amd import backend as be
from aion_amd import session as ss
from aion_amd.decoder import Decoder, DecoderConfig, SessionDecoder, SyntheticWeights
from quant_cases import QuantCache

pytestmark = pytest.mark.gpu

BOTH = pytest.mark.parametrize("dtype", [be.Q8_0, be.Q4_0])


class Layer:
    """The cache side and the attention of a block as step records, on buffers of its own."""

    B, T, HQ, HK, D = 2, 70, 4, 2, 64

    def __init__(self, gpu, dtype, s, rolling=False, flagged=True, order=(0, 1, 2, 3), scratch_v=False):
        rng = np.random.default_rng(7)
        b, t, hq, hk, d = self.B, self.T, self.HQ, self.HK, self.D
        self.gpu, self.shape = gpu, (b, s, hq, d)
        up = lambda *sh: gpu.upload(rng.standard_normal(sh).astype(np.float32))  # noqa: E731
        start = np.array([5, 40], np.int32) + (3 * t if rolling else 0)
        self.bufs = {"q": up(b, s, hq, d), "k": up(b, s, hk, d), "v": up(b, s, hk, d), "qr": gpu.zeros(b * s * hq * d * 4), "kr": gpu.zeros(b * s * hk * d * 4),
                     "out": gpu.zeros(b * s * hq * d * 4), "pos": gpu.upload((start[:, None] + np.arange(s)).astype(np.int32)), "end": gpu.upload(start),
                     "len": gpu.upload(start + s)}
        self.cache_bytes = gpu.cache_quant_bytes(dtype, b, t, hk, d)
        fill = QuantCache(dtype, b, t, hk, d)                                   # the rows before the new ones: any codes, small scales
        fill.codes[:] = rng.integers(17, 239, fill.codes.shape)
        fill.scales[:] = rng.random(fill.scales.shape).astype(np.float16).view(np.uint16)
        for name in ("kc", "vc"):
            self.bufs[name] = gpu.upload(fill.bytes)
        f = lambda nm, *sh, **kw: ss.tensor(self.bufs[nm], be.F32, sh, **kw)  # noqa: E731
        cache = lambda nm: ss.tensor(self.bufs[nm], dtype, (b, t, hk, d), rolling=rolling, quant_cache=flagged)  # noqa: E731
        i32 = lambda nm, *sh: ss.tensor(self.bufs[nm], be.I32, sh)  # noqa: E731
        kr = f("kr", b, s, hk, d, workspace=True)
        p = self.steps = ss.Steps()
        parts = [lambda: p.rope1d(f("q", b, s, hq, d), i32("pos", b, s), f("qr", b, s, hq, d)), lambda: p.rope1d(f("k", b, s, hk, d), i32("pos", b, s), kr),
                 lambda: p.sequence_append(cache("kc"), kr, i32("end", b)), lambda: p.sequence_append(cache("vc"), f("v", b, s, hk, d), i32("end", b))]
        for j in order:
            parts[j]()
        p.attention(f("qr", b, s, hq, d), cache("kc"), cache("vc"), f("out", b, s, hq, d), 0.125, query_positions=i32("pos", b, s), kv_lengths=i32("len", b))

    def results(self):
        g = self.gpu
        return [g.download(self.bufs["out"], np.float32, self.shape), g.download(self.bufs["qr"], np.float32, self.shape)] + \
               [g.download(self.bufs[n], np.uint8, (self.cache_bytes,)) for n in ("kc", "vc")]

    def free(self):
        for b in self.bufs.values():
            b.free()


@BOTH
@pytest.mark.parametrize("s,rolling", [(1, False), (1, True), (6, False), (20, True)])
@pytest.mark.parametrize("order", [(0, 1, 2, 3), (1, 2, 3, 0), (1, 0, 3, 2), (0, 1, 3, 2)])
def test_a_session_folds_the_cache_side_to_the_same_bits(gpu, dtype, s, rolling, order):
    sess, got = ss.Session(gpu), []
    for fusion in (0, ss.FUSE_SIBLINGS | ss.FUSE_WORKSPACE):
        layer = Layer(gpu, dtype, s, rolling, order=order)
        sess.set_fusion(fusion)
        sess.execute(layer.steps)
        got.append((layer.results(), sess.stats()[0]))
        layer.free()
    assert got[0][1] == 5 and got[1][1] == 2
    for x, y in zip(got[0][0], got[1][0]):
        assert np.array_equal(x, y)
    assert np.isfinite(got[0][0][0]).all() and got[0][0][0].any()
    sess.close()


@BOTH
def test_a_session_does_not_fold_what_is_read_again(gpu, dtype):
    """The rotated keys are an output of the list when something reads them later: the four steps run as they are."""
    layer = Layer(gpu, dtype, 3)
    b, s, hk, d = layer.B, 3, layer.HK, layer.D
    kr = ss.tensor(layer.bufs["kr"], be.F32, (b, s, hk, d), workspace=True)
    layer.bufs["copy"] = gpu.zeros(b * s * hk * d * 4)
    layer.steps.copy(kr, ss.tensor(layer.bufs["copy"], be.F32, (b, s, hk, d)))
    sess = ss.Session(gpu)
    sess.execute(layer.steps)
    assert sess.stats()[0] == 6 and gpu.download(layer.bufs["copy"], np.float32, (b * s * hk * d,)).any()
    sess.close()
    layer.free()


def test_a_session_refuses_block_tensors_that_are_no_caches(gpu):
    sess, layer = ss.Session(gpu), Layer(gpu, be.Q8_0, 2, flagged=False)
    with pytest.raises(be.AionHipError) as e:
        sess.execute(layer.steps)
    assert e.value.status in (be.hip.UNSUPPORTED, be.hip.INVALID_ARGUMENT)
    assert not layer.results()[1].any()                                          # nothing of the list has run
    layer.free()
    p, buf = ss.Steps(), gpu.zeros(1 << 16)
    cache = ss.tensor(buf, be.Q4_0, (1, 8, 1, 48), quant_cache=True)
    p.sequence_append(cache, ss.tensor(buf, be.F32, (1, 1, 1, 48)), ss.tensor(buf, be.I32, (1,)))
    with pytest.raises(be.AionHipError) as e:
        sess.execute(p)
    assert e.value.status == be.hip.INVALID_ARGUMENT
    buf.free()
    sess.close()


@BOTH
def test_a_cache_is_copied_whole(gpu, dtype):
    n = gpu.cache_quant_bytes(dtype, 2, 70, 3, 64)
    data = np.random.default_rng(0).integers(0, 256, n).astype(np.uint8)
    src, dst, p, sess = gpu.upload(data), gpu.zeros(n), ss.Steps(), ss.Session(gpu)
    p.copy(*(ss.tensor(x, dtype, (2, 70, 3, 64), quant_cache=True) for x in (src, dst)))
    sess.execute(p)
    assert np.array_equal(gpu.download(dst, np.uint8, (n,)), data)
    sess.close()
    src.free()
    dst.free()


SHAPE = dict(layers=2, hidden=256, heads=4, kv_heads=2, head_dim=64, ffn=512, vocab=1024, max_seq=150)


@BOTH
def test_decoders_over_quantized_caches(gpu, dtype):
    """The hand-routed decoder and the session over the same step list: the same logits to the bit, prompt and replayed steps; the keys of the first block
    are what the separate steps quantise."""
    cfg = DecoderConfig(cache_dtype=dtype, **SHAPE)
    w = SyntheticWeights(cfg, 7)
    a, b = Decoder(gpu, cfg, w, one_launch=True), SessionDecoder(gpu, cfg, w)
    try:
        assert a.stack is None
        prompt = np.random.default_rng(4).integers(0, cfg.vocab, 90).astype(np.int32)
        ta, tb = a.prefill(prompt), b.prefill(prompt)
        assert np.array_equal(a.logits_host(), b.logits_host()) and ta == tb and np.isfinite(a.logits_host()).all()
        a.begin_decode(ta)
        b.begin_decode(tb)
        for step in range(6):
            ta, tb = a.decode_step(), b.decode_step()
            assert np.array_equal(a.logits_host(), b.logits_host()), step
            assert ta == tb, step
        # the first block's keys, from the embedding alone: norm, projection, rotation, quantization as separate steps
        n, g = prompt.size, gpu
        x, k, kr = g.alloc(n * cfg.hidden * 4), g.alloc(n * cfg.kv_dim * 4), g.alloc(n * cfg.kv_dim * 4)
        ids, pos, zero = g.upload(prompt), g.upload(np.arange(n, dtype=np.int32)), g.upload(np.zeros(1, np.int32))
        g.step_gather_rows(be.F32, x, a.embed, ids, n, cfg.hidden, cfg.vocab)
        g.step_rmsnorm_matmul([a.w["l0.wk"]], x, a.gamma, n, [k], cfg.eps)
        g.step_rope(kr, k, pos, 1, n, cfg.kv_heads, cfg.head_dim, base=cfg.rope_base)
        want = QuantCache(dtype, 1, cfg.max_seq, cfg.kv_heads, cfg.head_dim)
        want.put(g.download(kr, np.float32, (n, cfg.kv_heads, cfg.head_dim)), 0, range(n))
        out = g.alloc(n * cfg.kv_dim * 4)
        g.step_cache_read(dtype, [out], [a.kc[0]], zero, (1, n, cfg.max_seq, cfg.kv_heads, cfg.head_dim))
        assert np.array_equal(g.download(out, np.float32, (n, cfg.kv_heads, cfg.head_dim)), want.values()[0, :n].astype(np.float32))
        for buf in (x, k, kr, ids, pos, zero, out):
            buf.free()
    finally:
        a.close()
        b.close()


def test_a_cache_type_that_is_none(gpu):
    with pytest.raises(ValueError):
        DecoderConfig(cache_dtype=be.F32, **SHAPE).cache_bytes(gpu)
