"""Where a decoder writes its rows after `pos` has been set: with a stand-in for the backend that keeps what is written, and on the GPU against a decoder that has seen nothing else."""
import numpy as np
import pytest

from aion_amd import backend as be
from aion_amd.decoder import Decoder, DecoderConfig, SessionDecoder, SyntheticWeights

SHAPE = dict(layers=2, hidden=256, heads=4, kv_heads=2, head_dim=64, ffn=512, vocab=1024)
KINDS = {"linear": {}, "q8": dict(cache_dtype=be.Q8_0), "pages": dict(page_rows=16), "evicting": dict(page_rows=16, evict_keep=16, evict_limit=36)}


class Buffer:
    def __init__(self, nbytes):
        self.nbytes, self.value, self.handle = nbytes, None, 0

    def view(self, offset):
        return self


class Backend:
    """Takes every step, runs none: buffers keep what the host wrote, step_advance_state counts."""

    def alloc(self, nbytes):
        return Buffer(nbytes)

    zeros = alloc

    def upload(self, x):
        b = Buffer(np.asarray(x).nbytes)
        b.value = np.array(x)
        return b

    def upload_weight(self, *a):
        return Buffer(0)

    def cache_quant_bytes(self, *a):
        return 64

    def paged_cache(self, *a):
        return be.PagedCache(*a)

    def write(self, buf, x):
        buf.value = np.array(x)

    def copy(self, dst, src, nbytes):
        dst.value = np.array(src.value)

    def download(self, buf, dtype, shape=None, offset=0):
        return np.zeros(shape, dtype) if buf.value is None else buf.value[offset // 4:offset // 4 + shape[0]].copy()

    def step_argmax(self, token, logits, rows, columns):
        token.value = np.array([0 if token.value is None else int(token.value[0]) + 1], np.int32)

    def step_advance_state(self, dst, src, n, counters, log, log_index, log_capacity):
        at = int(log_index.value[0])
        if at < log_capacity:
            if log.value is None:
                log.value = np.full(log.nbytes // 4, -1, np.int32)
            log.value[at] = src.value[0]
        for c in counters:
            c.value = c.value + 1

    def step_evict_paged(self, cache, w, lengths, wo, lengths_out, keep, limit, first, recent):
        lengths_out.value = np.minimum(lengths.value, keep) if lengths.value[0] > limit else np.array(lengths.value)

    def record_program(self, issue):
        return issue

    def program_execute(self, program):
        program()

    def program_is_current(self, program):
        return True

    def step_attention_matmul(self, *a, **kw):
        return True

    def __getattr__(self, name):
        return lambda *a, **kw: None


def state(d, s):
    b = d._buffers(s)
    return int(b["positions"].value[0]), int(b["write_index"].value[0]), int(b["kv_len"].value[0])


class Blank(SyntheticWeights):
    def blocks(self, name):
        return np.zeros(0, np.uint8)


def blank(kind):
    cfg = DecoderConfig(max_seq=40, **KINDS[kind], **SHAPE)
    return Decoder(Backend(), cfg, Blank(cfg, 1))


@pytest.mark.parametrize("kind", ["linear", "q8", "pages"])
def test_rows_go_where_pos_says(kind):
    d = blank(kind)
    for _ in range(4):                                       # as many prompts as there are, each from the beginning
        d.pos = 0
        d.prefill(np.zeros(16, np.int32))
        assert state(d, 16) == (0, 0, 16) and (d.pos, d.rows) == (16, 16)
    for _ in range(4):
        d.pos = 16
        d.begin_decode(3)
        assert state(d, 1) == (16, 16, 17)
        d.decode_run(12)
        assert state(d, 1) == (28, 28, 29) and d.rows == 28
    d.pos = 20
    d.prefill(np.zeros(7, np.int32))
    assert state(d, 7) == (20, 20, 27)
    with pytest.raises(ValueError):
        d.prefill(np.zeros(14, np.int32))


def test_under_eviction_a_text_goes_on_or_begins_anew():
    d = blank("evicting")
    for again in range(2):
        d.prefill(np.zeros(20, np.int32))
        for pos in (19, 21, 1):
            with pytest.raises(ValueError):
                d.pos = pos
        d.pos = 20
        d.prefill(np.zeros(17, np.int32))
        assert state(d, 17) == (20, 20, 37) and (d.pos, d.rows, d.gone) == (37, 16, 21)
        d.begin_decode(3)
        assert state(d, 1) == (37, 16, 17)
        d.decode_run(20)
        assert state(d, 1) == (57, 36, 37) and d.rows == 36
        d.decode_step()                                      # the 37th row passes the limit
        assert state(d, 1) == (58, 16, 17) and (d.pos, d.rows) == (58, 16)
        with pytest.raises(ValueError):
            d.pos = 57
        for w in d.drawn:
            w.value = None
        d.pos = 0                                            # as reset()
        assert d.rows == 0 and all((w.value == 0).all() for w in d.drawn)


@pytest.mark.parametrize("kind, runs", [("linear", [5, 0, 18]), ("evicting", [3, 0, 40, 41, 200, 66000, 7])])
def test_a_run_returns_its_tokens_however_long_the_text_is(kind, runs):
    """the stand-in's tokens are numbered; under eviction the text passes the caches and any log of it"""
    d = blank(kind)
    d.prefill(np.zeros(16, np.int32))
    d.begin_decode(3)
    d.decode_step(read_token=False)                          # (not a run's)
    at = int(d.token.value[0])
    for n in runs:
        assert np.array_equal(d.decode_run(n), at + 1 + np.arange(n))
        at += n
    assert d.pos == 17 + sum(runs)
    if kind == "linear":
        with pytest.raises(ValueError):
            d.decode_run(1)


@pytest.mark.parametrize("kind, s, more", [("linear", 100, set()), ("linear", 1, set()), ("q8", 100, set()), ("pages", 64, set()), ("pages", 65, {"row_positions"}), ("evicting", 1, {"kept_len"}),
                                           ("evicting", 65, {"kept_len", "row_positions", "tail"})])
def test_only_caches_in_pages_cost_what_they_need(kind, s, more):
    assert set(blank(kind)._buffers(s)) & {"kept_len", "row_positions", "tail"} == more


def test_no_newest_rows_need_stay():
    cfg = lambda **kw: DecoderConfig(max_seq=64, page_rows=16, evict_keep=16, **SHAPE, **kw).eviction()  # noqa: E731
    assert cfg(evict_recent=0) == (16, 63, 4, 0) and cfg(evict_recent=0, evict_first=0) == (16, 63, 0, 0)
    assert cfg() == cfg(evict_recent=None) == (16, 63, 4, 4) and cfg(evict_recent=40) == (16, 63, 4, 12)


def test_what_only_caches_in_pages_have_is_refused_elsewhere():
    for options in (dict(rotary=be.Rotary(32)), dict(evict_keep=16), dict(cache_dtype=be.Q8_0, rotary=be.Rotary(64))):
        cfg = DecoderConfig(max_seq=64, **options, **SHAPE)
        with pytest.raises(ValueError):
            Decoder(Backend(), cfg, Blank(cfg, 1))
        with pytest.raises(ValueError):
            SessionDecoder(Backend(), cfg, Blank(cfg, 1))
    cfg = DecoderConfig(max_seq=64, page_rows=16, rotary=be.Rotary(32), **SHAPE)
    assert Decoder(Backend(), cfg, Blank(cfg, 1)).rotary is cfg.rotary


@pytest.mark.gpu
@pytest.mark.parametrize("kind, one_launch", [("linear", False), ("linear", True), ("q8", False), ("pages", False)])
def test_a_text_taken_back_is_the_text_of_a_fresh_decoder(gpu, kind, one_launch):
    cfg = DecoderConfig(max_seq=150, **KINDS[kind], **SHAPE)
    weights = SyntheticWeights(cfg, 3)
    rng = np.random.default_rng(1)
    first, second = (rng.integers(0, cfg.vocab, 70).astype(np.int32) for _ in range(2))
    d = Decoder(gpu, cfg, weights, one_launch=one_launch)
    fresh, other = (Decoder(gpu, cfg, weights, one_launch=one_launch) for _ in range(2))
    try:
        d.begin_decode(d.prefill(first))
        d.decode_run(30)
        d.pos = 0
        a, b = d.prefill(second), fresh.prefill(second)
        assert a == b and np.array_equal(d.logits_host(), fresh.logits_host())
        d.begin_decode(a)
        fresh.begin_decode(b)
        want = fresh.decode_run(30)
        assert np.array_equal(d.decode_run(30), want) and np.array_equal(d.logits_host(), fresh.logits_host())
        for _ in range(3):                                   # the same run again and again
            d.pos = second.size
            d.begin_decode(a)
            assert np.array_equal(d.decode_run(30), want) and np.array_equal(d.logits_host(), fresh.logits_host())
        d.pos = 40                                           # the rest of the prompt once more, in front of another end of the text
        other.prefill(second)                                # (of 40 tokens alone the prompt's own sums would be split otherwise)
        other.pos = 40
        assert d.prefill(first[:25]) == other.prefill(first[:25]) and np.array_equal(d.logits_host(), other.logits_host())
    finally:
        d.close()
        fresh.close()
        other.close()


@pytest.mark.gpu
def test_a_run_longer_than_the_log(gpu):
    cfg = DecoderConfig(max_seq=40, **KINDS["evicting"], **SHAPE)
    weights = SyntheticWeights(cfg, 3)
    prompt = np.random.default_rng(2).integers(0, cfg.vocab, 33).astype(np.int32)
    a, b = (Decoder(gpu, cfg, weights) for _ in range(2))
    try:
        a.begin_decode(a.prefill(prompt))
        b.begin_decode(b.prefill(prompt))
        want = [b.decode_step() for _ in range(170)]
        assert list(a.decode_run(130)) + list(a.decode_run(40)) == want
    finally:
        a.close()
        b.close()
