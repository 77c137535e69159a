"""Steps over caches in pages: what the host refuses, before anything is launched."""
import numpy as np
import pytest

from aion_amd import backend as be
from aion_amd import hip

B, W, P, H, D, HQ, S = 2, 3, 16, 2, 64, 4, 2
PAGES = 8
BIG = 1 << 20          # every operand of the refused calls has a place of its own, this far from the next


def cache(at, **change):
    fields = dict(k_pages=at(0), v_pages=at(1), page_table=at(2), pages=PAGES, batch=B, table_width=W, page_rows=P, h_kv=H, d=D, dtype=be.F16)
    fields.update(change)
    return hip.PagedCache(*(fields[n] for n, _ in hip.PagedCache._fields_))


BAD_CACHES = [
    (dict(k_pages=0), hip.INVALID_ARGUMENT), (dict(v_pages=0), hip.INVALID_ARGUMENT), (dict(page_table=0), hip.INVALID_ARGUMENT), (dict(dtype=be.F32), hip.UNSUPPORTED),
    (dict(dtype=be.Q8_0), hip.UNSUPPORTED), (dict(page_rows=0), hip.INVALID_ARGUMENT), (dict(page_rows=8), hip.INVALID_ARGUMENT), (dict(page_rows=48), hip.INVALID_ARGUMENT),
    (dict(page_rows=2048), hip.INVALID_ARGUMENT), (dict(pages=0), hip.INVALID_ARGUMENT), (dict(table_width=0), hip.INVALID_ARGUMENT), (dict(h_kv=0), hip.INVALID_ARGUMENT),
    (dict(d=0), hip.INVALID_ARGUMENT), (dict(d=60), hip.INVALID_ARGUMENT), (dict(d=1032), hip.UNSUPPORTED), (dict(h_kv=1 << 16), hip.UNSUPPORTED), (dict(batch=1 << 16), hip.UNSUPPORTED),
    (dict(pages=1 << 31), hip.UNSUPPORTED), (dict(table_width=1 << 27), hip.UNSUPPORTED), (dict(h_kv=4096, page_rows=1024, d=1024), hip.UNSUPPORTED),
    (dict(k_pages=lambda at: at(0) + 2), hip.INVALID_ARGUMENT), (dict(v_pages=lambda at: at(0) + 4096), hip.INVALID_ARGUMENT), (dict(page_table=lambda at: at(2) + 2), hip.INVALID_ARGUMENT),
]


def made(at, change):
    return cache(at, **{k: v(at) if callable(v) else v for k, v in change.items()})


def rotary(**change):
    fields = dict(dims=D, base=10000.0, scaling=be.ROTARY_RAMP, factor=8.0, original_length=4096.0, low=1.0, high=32.0)
    fields.update(change)
    return be.Rotary(**fields)


BAD_ROTARY = [dict(dims=63), dict(dims=D + 2), dict(base=0.0), dict(base=-1.0), dict(base=float("inf")), dict(base=float("nan")), dict(magnitude=float("nan")), dict(magnitude=float("inf")),
              dict(scaling=4), dict(scaling=-1), dict(factor=0.0), dict(factor=float("nan")), dict(original_length=0.0), dict(low=0.0), dict(low=32.0), dict(high=float("inf")), dict(base=1.0),
              dict(scaling=be.ROTARY_LINEAR, factor=-2.0), dict(scaling=be.ROTARY_BANDS, low=4.0, high=1.0)]


def refusals(lib, ctx, at):
    """[(what, status that came, status that should)] of every refused call; `at(i)`: the i-th operand's place"""
    ref, out = hip.C.byref, []
    INV, UNS = hip.INVALID_ARGUMENT, hip.UNSUPPORTED
    good = cache(at)
    pool = PAGES * H * P * D * 2

    def say(what, got, want):
        out.append((what, got, want))

    def append(c, k=at(3), v=at(4), src=be.F32, index=at(5), s=S):
        return lib.aionhip_step_append_paged(ctx, ref(c) if c is not None else None, k, v, src, index, s)

    def rappend(c, r, qo=at(6), q=at(7), k=at(3), v=at(4), dtype=be.F32, pos=at(8), index=at(5), s=S, hq=HQ):
        return lib.aionhip_step_rotary_append_paged(ctx, ref(c) if c is not None else None, ref(r) if r is not None else None, qo, q, k, v, dtype, pos, index, s, hq)

    def read(c, k=at(3), v=at(4), dtype=be.F32, first=at(5), s=S):
        return lib.aionhip_step_read_paged(ctx, ref(c) if c is not None else None, k, v, dtype, first, s)

    def attend(c, before=0, weights=0, cap=W * P, **change):
        f = dict(out=at(6), q=at(7), k=0, v=0, query_positions=0, kv_lengths=at(5), batch=B, l_q=S, t_kv=cap, h_q=HQ, h_kv=H, d_k=D, d_v=D, q_dtype=be.F32, kv_dtype=be.F16,
                 scale=0.1, attn_logits_soft_cap=0.0, window_left=be.UNBOUNDED, window_right=0, window_chunk=0, rolling=0)
        f.update(change)
        p = hip.Attention(*(f[n] for n, _ in hip.Attention._fields_))
        return lib.aionhip_step_attention_paged(ctx, ref(p), ref(c) if c is not None else None, before, weights)

    def evict(c, **change):
        f = dict(weights=at(9), kv_lengths=at(5), weights_out=at(10), lengths_out=at(11), table_out=at(12), kept=at(13), width_out=3, limit=40, keep=30, first=2, recent=4)
        f.update(change)
        return lib.aionhip_step_evict_paged(ctx, ref(c) if c is not None else None, ref(hip.Eviction(*(f[n] for n, _ in hip.Eviction._fields_))))

    for what, call in (("append", append), ("rotary_append", lambda c: rappend(c, rotary())), ("read", read), ("attention", attend), ("evict", evict)):
        say((what, "no cache"), call(None), INV)
        for change, want in BAD_CACHES:
            say((what, str(change)), call(made(at, change)), want)
    for name in ("k", "v", "index"):
        say(("append", name), append(good, **{name: 0}), INV)
    say(("append", "type"), append(good, src=be.Q8_0), UNS)
    say(("append", "rows"), append(good, s=W * P + 1), INV)
    say(("append", "in a pool"), append(good, k=at(1) + pool - 16), INV)
    say(("append", "in the table"), append(good, v=at(2)), INV)
    say(("append", "index in a pool"), append(good, index=at(0) + 8), INV)
    say(("rotary_append", "positions in a pool"), rappend(good, rotary(), pos=at(1) + 8), INV)
    say(("rotary_append", "q over positions"), rappend(good, rotary(), qo=at(8)), INV)
    say(("rotary_append", "q over the index"), rappend(good, rotary(), qo=at(5)), INV)
    say(("read", "over the index"), read(good, v=at(5)), INV)
    say(("attention", "over the lengths"), attend(good, out=at(5)), INV)
    say(("attention", "over the positions"), attend(good, weights=at(9), query_positions=at(9) + 8), INV)
    for change in BAD_ROTARY:
        say(("rotary_append", str(change)), rappend(good, rotary(**change)), INV)
        say(("rotary", str(change)), lib.aionhip_step_rotary(ctx, at(6), at(7), at(8), be.F32, B, S, HQ, D, ref(rotary(**change))), INV)
    say(("rotary_append", "none"), rappend(good, None), INV)
    for name in ("qo", "q", "k", "v", "pos", "index"):
        say(("rotary_append", name), rappend(good, rotary(), **{name: 0}), INV)
    say(("rotary_append", "type"), rappend(good, rotary(), dtype=be.I32), UNS)
    say(("rotary_append", "heads"), rappend(good, rotary(), hq=1 << 16), UNS)
    say(("rotary_append", "rows"), rappend(good, rotary(), s=W * P + 1), INV)
    say(("rotary_append", "q beside itself"), rappend(good, rotary(), qo=at(7) + 16), INV)
    say(("rotary_append", "q over k"), rappend(good, rotary(), qo=at(3)), INV)
    say(("rotary_append", "q in a pool"), rappend(good, rotary(), qo=at(0)), INV)
    say(("rotary", "none"), lib.aionhip_step_rotary(ctx, at(6), at(7), at(8), be.F32, B, S, HQ, D, None), INV)
    for i in range(3):
        ops = [at(6), at(7), at(8)]
        ops[i] = 0
        say(("rotary", "null", i), lib.aionhip_step_rotary(ctx, *ops, be.F32, B, S, HQ, D, ref(rotary())), INV)
    say(("rotary", "type"), lib.aionhip_step_rotary(ctx, at(6), at(7), at(8), be.Q4_0, B, S, HQ, D, ref(rotary())), UNS)
    say(("rotary", "head"), lib.aionhip_step_rotary(ctx, at(6), at(7), at(8), be.F32, B, S, HQ, 1026, ref(rotary())), UNS)
    say(("rotary", "rows"), lib.aionhip_step_rotary(ctx, at(6), at(7), at(8), be.F32, 1 << 20, 1 << 20, HQ, D, ref(rotary())), UNS)
    say(("rotary", "beside itself"), lib.aionhip_step_rotary(ctx, at(6) + 4, at(6), at(8), be.F32, B, S, HQ, D, ref(rotary())), INV)
    say(("rotary", "over the positions"), lib.aionhip_step_rotary(ctx, at(6), at(7), at(6), be.F32, B, S, HQ, D, ref(rotary())), INV)
    for name in ("k", "v", "first"):
        say(("read", name), read(good, **{name: 0}), INV)
    say(("read", "type"), read(good, dtype=hip.I8), UNS)
    say(("read", "rows"), read(good, s=W * P + 1), INV)
    say(("read", "one place"), read(good, k=at(4) + 32), INV)
    say(("read", "into a pool"), read(good, k=at(0) + 64), INV)
    for change in (dict(out=0), dict(q=0), dict(k=at(0)), dict(v=at(1)), dict(rolling=1), dict(batch=1), dict(cap=W * P - 1), dict(h_kv=1), dict(d_k=32), dict(d_v=128), dict(kv_dtype=be.BF16),
                   dict(h_q=3), dict(h_q=0), dict(before=at(9)), dict(out=at(7)), dict(out=at(1)), dict(weights=at(0)), dict(weights=at(6)), dict(weights=at(9), before=at(9) + 64),
                   dict(weights=at(9), q=at(9))):
        say(("attention", str(change)), attend(good, **change), INV)
    say(("attention", "type"), attend(good, q_dtype=be.Q8_0), UNS)
    say(("attention", "heads"), attend(good, h_q=1 << 17), UNS)
    say(("attention", "queries"), attend(good, l_q=1 << 30), UNS)
    wide = cache(at, table_width=1 << 20, page_table=1 << 47)
    far = [1 << 46, 1 << 47, 1 << 48]
    say(("rotary", "rows of one launch"), lib.aionhip_step_rotary(ctx, far[0], far[1], far[2], be.F32, 1, 1 << 27, 1, D, ref(rotary())), UNS)
    say(("append", "rows of one launch"), append(cache(at, table_width=1 << 26, batch=4, page_table=far[0]), k=far[1], v=far[2], s=1 << 26), UNS)
    say(("read", "rows of one launch"), read(cache(at, table_width=1 << 26, batch=4, page_table=far[0]), k=far[1], v=far[2], s=1 << 28), UNS)
    say(("attention", "queries of one launch"), attend(cache(at, d=72), out=far[0], q=far[1], l_q=1 << 24, d_k=72, d_v=72), UNS)
    say(("attention", "scores"), attend(wide, weights=1 << 50, l_q=64, cap=P << 20), UNS)
    for change in (dict(weights=0), dict(kv_lengths=0), dict(weights_out=0), dict(lengths_out=0), dict(keep=41), dict(first=27), dict(recent=29), dict(limit=1 << 31), dict(width_out=2),
                   dict(table_out=0), dict(table_out=at(2)), dict(weights_out=at(9)), dict(weights_out=at(9) + 16), dict(lengths_out=at(10)), dict(kept=at(9)), dict(kept=at(10) + 4),
                   dict(kept=at(5)), dict(kept=at(11)), dict(kept=at(0)), dict(weights_out=at(1)), dict(table_out=at(13)), dict(table_out=at(0)), dict(lengths_out=at(5) + 4),
                   dict(weights=at(11)), dict(kv_lengths=at(10)), dict(table_out=0, width_out=0, weights_out=at(9) + 4), dict(lengths_out=at(2)), dict(weights=at(1)), dict(table_out=at(10)),
                   dict(table_out=at(11)), dict(recent=2 ** 64 - 1), dict(first=2 ** 64 - 1)):
        say(("evict", str(change)), evict(good, **change), INV)
    return out


@pytest.mark.gpu
def test_refusals(gpu):
    room = gpu.zeros(16 * BIG)
    for what, got, want in refusals(gpu._lib, gpu._ctx, lambda i: room.handle + i * BIG):
        assert got == want, what
        assert gpu._lib.aionhip_last_error(gpu._ctx)
    gpu.sync()
    assert not gpu.download(room, np.uint8).any()
    # what is nothing to do is no error
    at = lambda i: room.handle + i * BIG  # noqa: E731
    lib, ctx, ref = gpu._lib, gpu._ctx, hip.C.byref
    empty = cache(at, batch=0)
    assert lib.aionhip_step_append_paged(ctx, ref(empty), at(3), at(4), be.F32, at(5), 1) == hip.OK
    assert lib.aionhip_step_append_paged(ctx, ref(cache(at)), at(3), at(4), be.F32, at(5), 0) == hip.OK
    assert lib.aionhip_step_read_paged(ctx, ref(cache(at)), at(3), at(4), be.F32, at(5), 0) == hip.OK
    assert lib.aionhip_step_rotary(ctx, at(6), at(7), at(8), be.F32, 0, 1, HQ, D, ref(rotary())) == hip.OK
    assert lib.aionhip_step_evict_paged(ctx, ref(empty), ref(hip.Eviction(at(9), at(5), at(10), at(11), at(12), at(13), 3, 40, 30, 2, 4))) == hip.OK
    gpu.sync()
    room.free()


def test_null_contexts():
    lib, ref = hip.load_library(), hip.C.byref
    c = cache(lambda i: (i + 1) * BIG)
    assert lib.aionhip_step_rotary(None, 1, 1, 1, be.F32, 1, 1, 1, 8, ref(be.Rotary(8))) == hip.INVALID_ARGUMENT
    assert lib.aionhip_step_append_paged(None, ref(c), 1, 1, be.F32, 1, 1) == hip.INVALID_ARGUMENT
    assert lib.aionhip_step_rotary_append_paged(None, ref(c), ref(be.Rotary(8)), 1, 1, 1, 1, be.F32, 1, 1, 1, 1) == hip.INVALID_ARGUMENT
    assert lib.aionhip_step_read_paged(None, ref(c), 1, 1, be.F32, 1, 1) == hip.INVALID_ARGUMENT
    assert lib.aionhip_step_attention_paged(None, ref(hip.Attention()), ref(c), 0, 0) == hip.INVALID_ARGUMENT
    assert lib.aionhip_step_evict_paged(None, ref(c), ref(hip.Eviction())) == hip.INVALID_ARGUMENT
