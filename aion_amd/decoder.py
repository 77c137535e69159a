"""Synthetic decoder-only transformer assembled from the backend's steps.

The step sequence is the one aion's graph compiler emits for a decoder (pattern of
src/bench/models.zig:433-536, trimmed to a plain pre-norm block): Gather -> per layer
[RMSNorm -> MatMul q,k,v -> RoPE1D(q,k) -> Cast f16 + SequenceAppend(k,v) -> Attention ->
MatMul o -> add -> RMSNorm -> MatMul gate,up -> gate(gelu) -> MatMul down -> add] ->
RMSNorm -> MatMul lm_head -> ArgMax. With `cache_dtype` Q8_0 or Q4_0 the keys and values are quantised as they are appended
(SequenceAppend takes the f32 rows, no Cast) and attention reads the codes. With `page_rows` the caches are pools of pages under one
page table; q and k turn as `rotary` says, and with `evict_keep` a sequence that passes `evict_limit` rows keeps that many of them: the first, the newest, and the ones
whose keys have drawn the most attention, decided on the device at every step. The text may then be longer than the caches, though no prompt may (it is refused whole, before
anything is evicted for it). What keys draw is counted from the queries of every decode step and of a prompt's last 64 tokens, so that a text handed over in
several prompts counts more queries, and may keep other rows, than in one. q4_0 weights are [K,N] quant_axis 0 MatMul operands (the
only q4 layout aion has), q8_0 weights are [N,K] quant_axis 1 MatMulNT operands.

Prefill runs the steps eagerly; the single-token decode step is recorded once into a program
(HIP graph) and replayed per token. Token id, position, cache write index and kv length stay in
device buffers: the argmax of one replay is the gather index of the next.
With `one_launch=True` (and a shape that qualifies) all blocks of a decode step run as ONE launch
(aionhip_step_decoder_stack); the step is then gather, that launch, the logits GEMV, the argmax and the
state advance. It gives the same bits as the recorded program; it is not the default because on MI355X it
measures 0.93 ms per token of the 26-layer decoder against 0.86 ms for the program replay.
"""
import math
from dataclasses import dataclass

import numpy as np

from . import backend as be


@dataclass
class DecoderConfig:
    layers: int = 26
    hidden: int = 2048
    heads: int = 8
    kv_heads: int = 1
    head_dim: int = 256
    ffn: int = 8192
    vocab: int = 262144
    max_seq: int = 256
    eps: float = 1e-6
    rope_base: float = 10000.0
    wdtype: int = be.Q4_0
    cache_dtype: int = be.F16        # F16, or Q8_0 / Q4_0: keys and values held in 8 or 4 bits (head_dim a multiple of 32); in pages F16 or BF16
    page_rows: int = 0               # 0: linear caches; else caches in pages of that many rows (a power of two, 16 to 1024)
    rotary: object = None            # caches in pages: how q and k turn (backend.Rotary); None: the whole head, in halves, by rope_base
    evict_keep: int = 0              # caches in pages: rows that a sequence keeps when it passes evict_limit; 0: no eviction
    evict_limit: int = 0             # 0: max_seq - 1
    evict_first: int = 4             # of those, the oldest and the newest that stay in any case
    evict_recent: int = None         # None: a quarter of evict_keep

    @property
    def q_dim(self):
        return self.heads * self.head_dim

    @property
    def kv_dim(self):
        return self.kv_heads * self.head_dim

    @property
    def quant_cache(self):
        return self.cache_dtype in be.BLOCK_BYTES

    @property
    def pages(self):
        return -(-self.max_seq // self.page_rows)

    def eviction(self):
        """(keep, limit, first, recent), or None"""
        if not self.evict_keep:
            return None
        if not self.page_rows:
            raise ValueError("evict_keep: eviction is from caches in pages (page_rows)")
        limit = self.evict_limit or self.max_seq - 1
        first = min(self.evict_first, self.evict_keep)
        recent = min(self.evict_keep // 4 if self.evict_recent is None else self.evict_recent, self.evict_keep - first)
        if not self.evict_keep <= limit < self.max_seq:
            raise ValueError("evict_keep %d <= evict_limit %d < max_seq %d must hold" % (self.evict_keep, limit, self.max_seq))
        return self.evict_keep, limit, first, recent

    def turning(self):
        """How q and k turn on caches in pages."""
        if self.rotary is not None and not self.page_rows:
            raise ValueError("rotary: linear caches turn the whole head by rope_base (page_rows)")
        return self.rotary or be.Rotary(self.head_dim, base=self.rope_base)

    def cache_bytes(self, gpu):
        """Bytes of one layer's cache of keys (or values)."""
        if self.page_rows:
            if self.cache_dtype not in (be.F16, be.BF16):
                raise ValueError("cache_dtype: caches in pages are F16 or BF16")
            return self.pages * self.page_rows * self.kv_dim * 2
        if self.quant_cache:
            return gpu.cache_quant_bytes(self.cache_dtype, 1, self.max_seq, self.kv_heads, self.head_dim)
        if self.cache_dtype != be.F16:
            raise ValueError("cache_dtype: F16, Q8_0 or Q4_0")
        return self.max_seq * self.kv_dim * 2


def weight_shapes(cfg):
    """name -> (n, k) of every quantized matmul weight (C[.., n] = A[.., k] @ W)."""
    shapes = {}
    for l in range(cfg.layers):
        shapes["l%d.wq" % l] = (cfg.q_dim, cfg.hidden)
        shapes["l%d.wk" % l] = (cfg.kv_dim, cfg.hidden)
        shapes["l%d.wv" % l] = (cfg.kv_dim, cfg.hidden)
        shapes["l%d.wo" % l] = (cfg.hidden, cfg.q_dim)
        shapes["l%d.wgate" % l] = (cfg.ffn, cfg.hidden)
        shapes["l%d.wup" % l] = (cfg.ffn, cfg.hidden)
        shapes["l%d.wdown" % l] = (cfg.hidden, cfg.ffn)
    shapes["lm_head"] = (cfg.vocab, cfg.hidden)
    return shapes


class SyntheticWeights:
    """Seeded ~N(0,0.02) weights through the aion quantizers. A 2^22-sample normal pool is read at a
    per-tensor offset and tiled, which keeps a 2-billion-parameter model's set-up to seconds; the
    per-block statistics are those of N(0,0.02)."""

    def __init__(self, cfg, seed=0):
        self.cfg = cfg
        rng = np.random.default_rng(seed)
        self.pool = (rng.standard_normal(1 << 22) * 0.02).astype(np.float32)
        self.seed = seed

    def _values(self, name, count):
        off = (hash_name(name) * 2654435761 + self.seed) % (self.pool.size - 1)
        reps = -(-(count + off) // self.pool.size)
        return np.tile(self.pool, reps)[off:off + count]

    def blocks(self, name):
        n, k = weight_shapes(self.cfg)[name]
        v = self._values(name, n * k)
        if self.cfg.wdtype == be.Q8_0:
            return be.quantize_blocks(be.Q8_0, v.reshape(n, k), 1)       # [N,K] axis 1
        return be.quantize_blocks(be.Q4_0, v.reshape(k, n), 0)           # [K,N] axis 0

    def embed(self):
        return self._values("embed", self.cfg.vocab * self.cfg.hidden).reshape(self.cfg.vocab, self.cfg.hidden).copy()


def hash_name(name):
    h = 2166136261
    for ch in name.encode():
        h = ((h ^ ch) * 16777619) & 0xFFFFFFFF
    return h


PROMPT_ROWS = 64        # caches in pages: longer prompts attend to keys and values read back in order; of them that many last queries say what the keys draw


class Decoder:
    def __init__(self, gpu, cfg, weights, on_weight=None, one_launch=False):
        """on_weight(name, host_array) is called for every tensor (the tests feed the oracle with it)."""
        self.gpu, self.cfg = gpu, cfg
        self.eviction, self.rotary = cfg.eviction(), cfg.turning()
        self.stack = None
        layout = be.ROWS_NK if cfg.wdtype == be.Q8_0 else be.KMAJOR_KN
        self.w = {}
        for name, (n, k) in weight_shapes(cfg).items():
            blocks = weights.blocks(name)
            self.w[name] = gpu.upload_weight(cfg.wdtype, layout, n, k, blocks)
            if on_weight:
                on_weight(name, blocks)
        emb = weights.embed()
        self.embed = gpu.upload(emb)
        if on_weight:
            on_weight("embed", emb)
        ones = np.ones(cfg.hidden, np.float32)
        self.gamma = gpu.upload(ones)          # every RMSNorm uses gamma = 1 (config 5)
        if on_weight:
            for l in range(cfg.layers):
                on_weight("l%d.norm1" % l, ones)
                on_weight("l%d.norm2" % l, ones)
            on_weight("norm_f", ones)
        kv_bytes = cfg.cache_bytes(gpu)
        self.kc = [gpu.zeros(kv_bytes) for _ in range(cfg.layers)]
        self.vc = [gpu.zeros(kv_bytes) for _ in range(cfg.layers)]
        self.page_table, self.caches, self.drawn, self.linear = None, [], [], None
        if cfg.page_rows:
            self.page_table = gpu.upload(np.arange(cfg.pages, dtype=np.int32))
            self.caches = [gpu.paged_cache(k, v, self.page_table, cfg.pages, 1, cfg.pages, cfg.page_rows, cfg.kv_heads, cfg.head_dim, cfg.cache_dtype)
                           for k, v in zip(self.kc, self.vc)]
        if self.eviction:
            self.drawn = [gpu.zeros(cfg.kv_heads * self.caches[0].capacity * 4) for _ in range(cfg.layers)]      # what each key has drawn
        self.one = gpu.upload(np.ones(1, np.int32))
        self.logits = gpu.alloc(cfg.vocab * 4)
        self.token = gpu.alloc(4)
        self.history = gpu.alloc(cfg.max_seq * 4)        # the tokens that a run of decode steps has produced, the first at 0
        self.logged = gpu.upload(np.zeros(1, np.int32))  # how many
        self.state = {}        # S -> activation buffers
        self.program = self.cut_program = None
        self._pos = self.gone = 0                        # tokens of the text; of their rows, how many eviction has taken
        if one_launch and not cfg.quant_cache and not cfg.page_rows:               # (the one-launch form reads linear f16 caches)
            layers = [{"wq": self.w["l%d.wq" % l], "wk": self.w["l%d.wk" % l], "wv": self.w["l%d.wv" % l], "wo": self.w["l%d.wo" % l],
                       "w_gate": self.w["l%d.wgate" % l], "w_up": self.w["l%d.wup" % l], "w_down": self.w["l%d.wdown" % l],
                       "norm1_gamma": self.gamma, "norm2_gamma": self.gamma, "k_cache": self.kc[l], "v_cache": self.vc[l]}
                      for l in range(cfg.layers)]
            try:
                self.stack = gpu.decoder_stack_create(layers, cfg.hidden, cfg.heads, cfg.kv_heads, cfg.head_dim, cfg.ffn, cfg.max_seq,
                                                      cfg.eps, cfg.eps, 1.0 / math.sqrt(cfg.head_dim), rope_base=cfg.rope_base)
            except be.AionHipError as e:
                if e.status != be.hip.UNSUPPORTED:
                    raise                                  # a shape outside the one-launch form's limits: separate steps

    def _buffers(self, s):
        if s in self.state:
            return self.state[s]
        c, g = self.cfg, self.gpu
        f = 4 * s
        b = {
            "ids": g.alloc(4 * s), "positions": g.alloc(4 * s), "write_index": g.alloc(4), "kv_len": g.alloc(4),
            "x": g.alloc(f * c.hidden), "h": g.alloc(f * c.hidden), "o": g.alloc(f * c.hidden),
            "q": g.alloc(f * c.q_dim), "qr": g.alloc(f * c.q_dim), "att": g.alloc(f * c.q_dim),
            "k": g.alloc(f * c.kv_dim), "kr": g.alloc(f * c.kv_dim), "v": g.alloc(f * c.kv_dim),
            "gate": g.alloc(f * c.ffn), "up": g.alloc(f * c.ffn), "act": g.alloc(f * c.ffn),
            "hl": g.alloc(4 * c.hidden),
        }
        if c.page_rows and s > PROMPT_ROWS:
            b["row_positions"] = g.alloc(4 * s)
        if self.eviction:
            b["kept_len"] = g.alloc(4)
            if s > PROMPT_ROWS:
                b["tail"] = g.alloc(4 * PROMPT_ROWS * c.q_dim)
        self.state[s] = b
        return b

    def _forward(self, s, b, cut=None):
        """Launches every step of one forward pass over `s` tokens (eagerly, or into an open recording). cut: with the eviction behind each block (None: where it is due)."""
        c, g = self.cfg, self.gpu
        g.step_gather_rows(be.F32, b["x"], self.embed, b["ids"], s, c.hidden, c.vocab)
        scale = 1.0 / math.sqrt(c.head_dim)
        for l in range(c.layers if not (s == 1 and self.stack is not None) else 0):
            p = "l%d." % l
            if c.page_rows:
                self._paged_block(l, s, b, scale, self._due(s) if cut is None else cut)
            elif c.quant_cache:
                # RMSNorm -> MatMul q, k, v (one call), RoPE1D(q), RoPE1D(k) -> quantized append of k and v (one launch)
                g.step_rmsnorm_matmul([self.w[p + "wq"], self.w[p + "wk"], self.w[p + "wv"]], b["x"], self.gamma, s,
                                      [b["q"], b["k"], b["v"]], c.eps)
                g.step_rope_append_quant(c.cache_dtype, b["qr"], b["q"], b["k"], b["v"], self.kc[l], self.vc[l], b["positions"], b["write_index"],
                                         1, s, c.max_seq, c.heads, c.kv_heads, c.head_dim, base=c.rope_base)
            elif s == 1 and c.hidden <= 8192 and c.head_dim % 8 == 0:
                # one new token: RMSNorm -> MatMul q, k, v -> RoPE1D(q), RoPE1D(k) -> f16 -> append, one launch
                g.step_rmsnorm_qkv_rope_append(self.w[p + "wq"], self.w[p + "wk"], self.w[p + "wv"], b["x"], self.gamma, c.eps,
                                               b["qr"], self.kc[l], self.vc[l], b["positions"], b["write_index"],
                                               c.max_seq, c.heads, c.kv_heads, c.head_dim, base=c.rope_base)
            # many tokens: the same, two launches, where the exact GEMM runs the projections
            elif not g.step_rmsnorm_qkv_rope_append_rows(self.w[p + "wq"], self.w[p + "wk"], self.w[p + "wv"], b["x"], self.gamma, c.eps, b["qr"],
                                                         self.kc[l], self.vc[l], b["positions"], b["write_index"], 1, s, c.max_seq, c.heads,
                                                         c.kv_heads, c.head_dim, base=c.rope_base):
                # RMSNorm -> MatMul q, k, v (one call: the norm is not materialised)
                g.step_rmsnorm_matmul([self.w[p + "wq"], self.w[p + "wk"], self.w[p + "wv"]], b["x"], self.gamma, s,
                                      [b["q"], b["k"], b["v"]], c.eps)
                # RoPE1D(q), RoPE1D(k) -> f16 -> append, v -> f16 -> append
                g.step_rope_append(b["qr"], b["q"], b["k"], b["v"], self.kc[l], self.vc[l], b["positions"], b["write_index"],
                                   1, s, c.max_seq, c.heads, c.kv_heads, c.head_dim, base=c.rope_base)
            # attention, then MatMul o with beta = 1: x = x + att @ Wo (the residual add rides on the matmul's beta); a prompt's attention leaves
            # its rows as the exact GEMM reads them
            shape = (1, s, c.max_seq, c.heads, c.kv_heads, c.head_dim, c.head_dim)
            options = {"q_dtype": be.F32, "kv_dtype": c.cache_dtype, "window": be.CAUSAL, "query_positions": b["positions"], "kv_lengths": b["kv_len"]}
            if c.page_rows:
                g.step_matmul(self.w[p + "wo"], b["att"], s, b["x"], beta=1.0)
            elif s == 1 or c.quant_cache or not g.step_attention_matmul(self.w[p + "wo"], b["qr"], self.kc[l], self.vc[l], shape, scale, b["x"], beta=1.0, **options):
                g.step_attention(b["att"], b["qr"], self.kc[l], self.vc[l], shape, scale, **options)
                g.step_matmul(self.w[p + "wo"], b["att"], s, b["x"], beta=1.0)
            if s == 1 and c.hidden <= 8192 and c.ffn % 32 == 0:
                # one row: RMSNorm -> MatMul gate, up -> gate(gelu) -> MatMul down (beta = 1), two launches
                g.step_rmsnorm_geglu_matmul(self.w[p + "wgate"], self.w[p + "wup"], self.w[p + "wdown"], b["x"], self.gamma, c.eps,
                                            b["x"], beta=1.0)
            # many rows: the same, three launches, where the exact GEMM runs all three matmuls
            elif not g.step_rmsnorm_geglu_matmul_rows(self.w[p + "wgate"], self.w[p + "wup"], self.w[p + "wdown"], b["x"], self.gamma, s, c.eps,
                                                      b["x"], beta=1.0):
                g.step_rmsnorm_matmul([self.w[p + "wgate"], self.w[p + "wup"]], b["x"], self.gamma, s, [b["gate"], b["up"]], c.eps)
                # gate(gelu) -> MatMul down, beta = 1
                g.step_gate_matmul(self.w[p + "wdown"], b["gate"], b["up"], s, b["x"], beta=1.0)
        if s == 1 and self.stack is not None:
            g.step_decoder_stack(self.stack, b["x"], b["x"], b["positions"], b["write_index"], b["kv_len"])
        last = b["x"].view((s - 1) * c.hidden * 4)
        g.step_rmsnorm_matmul([self.w["lm_head"]], last, self.gamma, 1, [self.logits], c.eps)
        g.step_argmax(self.token, self.logits, 1, c.vocab)

    def _paged_block(self, l, s, b, scale, cut):
        """The input side and the attention of one block over caches in pages, and with `cut` the eviction; b["kept_len"]: the rows that stay."""
        c, g, p, cache = self.cfg, self.gpu, "l%d." % l, self.caches[l]
        g.step_rmsnorm_matmul([self.w[p + "wq"], self.w[p + "wk"], self.w[p + "wv"]], b["x"], self.gamma, s, [b["q"], b["k"], b["v"]], c.eps)
        g.step_rotary_append_paged(cache, self.rotary, b["qr"], b["q"], b["k"], b["v"], b["positions"], b["write_index"], s, c.heads)
        asked = min(s, PROMPT_ROWS)
        if asked < s:
            # a prompt: its keys and values in order, for the kernel that shares them among many rows
            n = self.rows + s
            if self.linear is None:
                self.linear = [g.alloc(c.cache_bytes(g)) for _ in range(2)] + [g.upload(np.zeros(1, np.int32))]
            g.step_read_paged(cache, self.linear[0], self.linear[1], self.linear[2], n, out_dtype=c.cache_dtype)
            g.step_attention(b["att"], b["qr"], self.linear[0], self.linear[1], (1, s, n, c.heads, c.kv_heads, c.head_dim, c.head_dim), scale, kv_dtype=c.cache_dtype,
                             query_positions=b["row_positions"])
        elif not self.eviction:
            g.step_attention_paged(b["att"], b["qr"], cache, s, c.heads, scale, kv_lengths=b["kv_len"])
        if not self.eviction:
            return
        # (of a prompt the last queries alone say what the keys draw; their rows are there already)
        out = b["att"] if asked == s else b["tail"]
        g.step_attention_paged(out, b["qr"].view((s - asked) * c.q_dim * 4), cache, asked, c.heads, scale, kv_lengths=b["kv_len"], weights=self.drawn[l], weights_before=self.drawn[l])
        if not cut:
            return
        keep, limit, first, recent = self.eviction
        g.step_evict_paged(cache, self.drawn[l], b["kv_len"], self.drawn[l], b["kept_len"], keep, limit=limit, first=first, recent=recent)

    def _due(self, s):
        """Whether s tokens more take the caches past their limit: how many rows there are is known here, which ones stay is not."""
        return bool(self.eviction) and self.rows + s > self.eviction[1]

    @property
    def pos(self):
        """Tokens of the text so far. May be set: the text goes on from there, over what was behind. Under eviction only to 0, which is reset(): which rows a shorter text would still have,
        and what its keys had drawn, is not kept."""
        return self._pos

    @pos.setter
    def pos(self, pos):
        if self.eviction and pos != self._pos:
            if pos:
                raise ValueError("pos %d: under eviction a text goes on from its end (%d) or begins anew (0)" % (pos, self._pos))
            self.reset()
        self._pos = pos

    @property
    def rows(self):
        """Rows of the caches: fewer than the text has tokens, once rows have been evicted."""
        return self._pos - self.gone

    def _advanced(self, s):
        """The text and the caches are s tokens further."""
        due = self._due(s)
        self._pos += s
        if due:
            self.gone = self._pos - self.eviction[0]

    def reset(self):
        self._pos = self.gone = 0
        for w in self.drawn:
            self.gpu.write(w, np.zeros(w.nbytes // 4, np.float32))

    def prefill(self, tokens):
        """Runs the prompt (positions pos .. pos+len-1); returns the greedy next token."""
        t = np.ascontiguousarray(tokens, np.int32)
        s = t.size
        if self.rows + s > self.cfg.max_seq:
            raise ValueError("prompt exceeds the cache capacity")
        b = self._buffers(s)
        g = self.gpu
        g.write(b["ids"], t)
        g.write(b["positions"], np.arange(self.pos, self.pos + s, dtype=np.int32))
        if "row_positions" in b:
            g.write(b["row_positions"], np.arange(self.rows, self.rows + s, dtype=np.int32))
        g.write(b["write_index"], np.array([self.rows], np.int32))
        g.write(b["kv_len"], np.array([self.rows + s], np.int32))
        self._forward(s, b)
        self._advanced(s)
        return int(g.download(self.token, np.int32, (1,))[0])

    def logits_host(self):
        return self.gpu.download(self.logits, np.float32, (self.cfg.vocab,))

    def begin_decode(self, first_token):
        """Prepares the single-token state and records the decode program (one warm-up step runs
        eagerly first so that every scratch buffer has its final size; it is then rolled back)."""
        g = self.gpu
        b = self._buffers(1)
        self._set_decode_state(b, first_token, self.pos)
        if self.program is not None and not (g.program_is_current(self.program) and (self.cut_program is None or g.program_is_current(self.cut_program))):
            # a longer prompt since the recording made the context replace a work buffer the program's launches address
            self._drop_programs()
        if self.stack is not None:
            self._decode_buffers = b                 # one launch per step already: nothing to record
            return
        if self.program is None:
            if self.eviction:                        # (of no keys: nothing draws weight, and no row is evicted)
                g.write(b["kv_len"], np.zeros(1, np.int32))
            self._forward(1, b, cut=bool(self.eviction))     # eager warm-up at the current position
            g.sync()
            self._set_decode_state(b, first_token, self.pos)

            def issue(cut):
                self._forward(1, b, cut)
                if cut:                              # the next row goes behind those that stay
                    g.copy(b["write_index"], b["kept_len"], 4)
                    g.copy(b["kv_len"], b["kept_len"], 4)
                # advance the device-resident loop state: next id = argmax, positions/write index/kv length += 1; the token
                # is also logged behind those before it, so that a run of steps needs no read-back per step
                g.step_advance_state(b["ids"], self.token, 1, [b["positions"], b["kv_len"], self.logged] + ([] if cut else [b["write_index"]]),
                                     log=self.history, log_index=self.logged, log_capacity=self.cfg.max_seq)
            self.program = g.record_program(lambda: issue(False))
            if self.eviction:                        # the step that takes the caches past their limit is a program of its own
                self.cut_program = g.record_program(lambda: issue(True))

    def _drop_programs(self):
        for p in (self.program, self.cut_program):
            if p is not None:
                self.gpu.program_destroy(p)
        self.program = self.cut_program = None

    def _set_decode_state(self, b, token, pos):
        g, rows = self.gpu, pos - self.gone
        g.write(b["ids"], np.array([token], np.int32))
        g.write(b["positions"], np.array([pos], np.int32))
        g.write(b["write_index"], np.array([rows], np.int32))
        g.write(b["kv_len"], np.array([rows + 1], np.int32))

    def _step_on_device(self):
        """One decode step whose loop state stays on the device: the recorded program, or with the one-launch stack the five
        launches themselves."""
        if self.stack is None:
            self.gpu.program_execute(self.cut_program if self._due(1) else self.program)
            return
        b, g = self._decode_buffers, self.gpu
        self._forward(1, b)
        g.step_advance_state(b["ids"], self.token, 1, [b["positions"], b["write_index"], b["kv_len"], self.logged],
                             log=self.history, log_index=self.logged, log_capacity=self.cfg.max_seq)

    def decode_step(self, read_token=True):
        """One decode step on the device-resident state; returns the token it produced (a 4-byte read-back)."""
        if not self.eviction and self.pos + 1 > self.cfg.max_seq:
            raise ValueError("cache capacity exhausted")
        self._step_on_device()
        self._advanced(1)
        if read_token:
            return int(self.gpu.download(self.token, np.int32, (1,))[0])
        return None

    def decode_run(self, n):
        """Replays the decode program n times back to back (nothing is read back in between: the loop state and the token
        log live on the device; under eviction, where the text may outgrow the log, the log is read whenever it is full) and returns the n tokens."""
        if not self.eviction and self.pos + n > self.cfg.max_seq:
            raise ValueError("cache capacity exhausted")
        tokens = np.zeros(n, np.int32)
        for start in range(0, n, self.cfg.max_seq):
            run = min(n - start, self.cfg.max_seq)
            self.gpu.write(self.logged, np.zeros(1, np.int32))
            for _ in range(run):
                self._step_on_device()
                self._advanced(1)
            tokens[start:start + run] = self.gpu.download(self.history, np.int32, (run,))
        if self.stack is not None:
            self.gpu.decoder_stack_status(self.stack)      # raises if a launch gave up waiting (its tokens would be invalid)
        return tokens

    def decode_step_eager(self, token):
        """The same step without a program (used by tests to check the replayed graph)."""
        b = self._buffers(1)
        self._set_decode_state(b, token, self.pos)
        self._forward(1, b)
        self._advanced(1)
        return int(self.gpu.download(self.token, np.int32, (1,))[0])

    def close(self):
        self._drop_programs()
        if self.stack is not None:
            self.gpu.decoder_stack_destroy(self.stack)
            self.stack = None
        for w in self.w.values():
            w.free()
        for lst in (self.kc, self.vc):
            for t in lst:
                t.free()
        for bufs in self.state.values():
            for t in bufs.values():
                t.free()
        for t in [self.embed, self.gamma, self.one, self.logits, self.token, self.history, self.logged] + self.drawn + ([self.page_table] if self.page_table else []) + (self.linear or []):
            t.free()


class SessionDecoder:
    """The same decoder the way a compiled aion program reaches a backend: one record per step of the sequence in this
    module's header, nothing pre-fused, handed to the library's session executor (aionhip_session_execute), which folds
    what it may. Parameters are device tensors in aion's packed form; the session re-lays them at first use. The residual
    adds accumulate in place (x = x + o), the activations between the block's input and its output are workspace tensors.
    Gives the tokens of `Decoder` over the same weights."""

    def __init__(self, gpu, cfg, weights, fusion=None):
        from . import session as ss
        if cfg.page_rows or cfg.rotary is not None or cfg.evict_keep:
            raise ValueError("page_rows, rotary, evict_keep: aion's step list has no caches in pages")
        self.ss, self.gpu, self.cfg = ss, gpu, cfg
        self.sess = ss.Session(gpu)
        if fusion is not None:
            self.sess.set_fusion(fusion)
        self.nt = cfg.wdtype == be.Q8_0
        self.w = {name: gpu.upload(weights.blocks(name)) for name in weight_shapes(cfg)}
        self.embed = gpu.upload(weights.embed())
        self.gamma = gpu.upload(np.ones(cfg.hidden, np.float32))
        kv_bytes = cfg.cache_bytes(gpu)
        self.kc = [gpu.zeros(kv_bytes) for _ in range(cfg.layers)]
        self.vc = [gpu.zeros(kv_bytes) for _ in range(cfg.layers)]
        self.one = gpu.upload(np.ones(1, np.int32))
        self.logits = gpu.alloc(cfg.vocab * 4)
        self.token = gpu.alloc(4)
        self.state = {}
        self.program = None
        self.pos = 0

    def _weight(self, name):
        n, k = weight_shapes(self.cfg)[name]
        return self.ss.tensor(self.w[name], self.cfg.wdtype, (n, k) if self.nt else (k, n))

    def _program(self, s, advance=False):
        """-> (buffers, step records) of one forward pass over `s` tokens; advance: the loop state moves on the device
        behind it (the produced token becomes the next input, the three counters go up by one)."""
        key = (s, advance)
        if key in self.state:
            return self.state[key]
        c, g, ss = self.cfg, self.gpu, self.ss
        f4 = 4 * s
        b = self.state[(s, not advance)][0] if (s, not advance) in self.state else {
            "ids": g.alloc(4 * s), "positions": g.alloc(4 * s), "write_index": g.alloc(4), "kv_len": g.alloc(4),
            "x": g.alloc(f4 * c.hidden), "h": g.alloc(f4 * c.hidden), "o": g.alloc(f4 * c.hidden), "q": g.alloc(f4 * c.q_dim),
            "qr": g.alloc(f4 * c.q_dim), "att": g.alloc(f4 * c.q_dim), "k": g.alloc(f4 * c.kv_dim), "kr": g.alloc(f4 * c.kv_dim),
            "v": g.alloc(f4 * c.kv_dim), "k16": g.alloc(2 * s * c.kv_dim), "v16": g.alloc(2 * s * c.kv_dim), "gate": g.alloc(f4 * c.ffn),
            "up": g.alloc(f4 * c.ffn), "act": g.alloc(f4 * c.ffn), "hl": g.alloc(4 * c.hidden)}
        work = lambda nm, *shape: ss.tensor(b[nm], be.F32, shape, workspace=True)  # noqa: E731
        x = ss.tensor(b["x"], be.F32, (1, s, c.hidden))
        gamma = ss.tensor(self.gamma, be.F32, (c.hidden,))
        pos, widx, kvl = (ss.tensor(b[nm], be.I32, shape) for nm, shape in (("positions", (1, s)), ("write_index", (1,)), ("kv_len", (1,))))
        mm = (lambda p, a, w, out, **kw: p.matmul_nt(a, w, out, **kw)) if self.nt else (lambda p, a, w, out, **kw: p.matmul(a, w, out, **kw))
        p = ss.Steps()
        p.gather_rows(ss.tensor(self.embed, be.F32, (c.vocab, c.hidden)), ss.tensor(b["ids"], be.I32, (1, s)), x)
        for l in range(c.layers):
            n = "l%d." % l
            kc = ss.tensor(self.kc[l], c.cache_dtype, (1, c.max_seq, c.kv_heads, c.head_dim), quant_cache=c.quant_cache)
            vc = ss.tensor(self.vc[l], c.cache_dtype, (1, c.max_seq, c.kv_heads, c.head_dim), quant_cache=c.quant_cache)
            p.rmsnorm(x, gamma, None, work("h", 1, s, c.hidden), c.eps)
            mm(p, work("h", 1, s, c.hidden), self._weight(n + "wq"), work("q", 1, s, c.q_dim))
            mm(p, work("h", 1, s, c.hidden), self._weight(n + "wk"), work("k", 1, s, c.kv_dim))
            mm(p, work("h", 1, s, c.hidden), self._weight(n + "wv"), work("v", 1, s, c.kv_dim))
            p.rope1d(work("q", 1, s, c.heads, c.head_dim), pos, work("qr", 1, s, c.heads, c.head_dim), base_frequency=c.rope_base)
            p.rope1d(work("k", 1, s, c.kv_heads, c.head_dim), pos, work("kr", 1, s, c.kv_heads, c.head_dim), base_frequency=c.rope_base)
            if c.quant_cache:
                p.sequence_append(kc, work("kr", 1, s, c.kv_heads, c.head_dim), widx)
                p.sequence_append(vc, work("v", 1, s, c.kv_heads, c.head_dim), widx)
            else:
                k16 = ss.tensor(b["k16"], be.F16, (1, s, c.kv_heads, c.head_dim), workspace=True)
                v16 = ss.tensor(b["v16"], be.F16, (1, s, c.kv_heads, c.head_dim), workspace=True)
                p.cast(work("kr", 1, s, c.kv_heads, c.head_dim), k16)
                p.sequence_append(kc, k16, widx)
                p.cast(work("v", 1, s, c.kv_heads, c.head_dim), v16)
                p.sequence_append(vc, v16, widx)
            p.attention(work("qr", 1, s, c.heads, c.head_dim), kc, vc, work("att", 1, s, c.heads, c.head_dim), 1.0 / math.sqrt(c.head_dim),
                        query_positions=pos, kv_lengths=kvl)
            mm(p, work("att", 1, s, c.q_dim), self._weight(n + "wo"), work("o", 1, s, c.hidden))
            p.elemwise_binary(ss.ADD, x, work("o", 1, s, c.hidden), x)
            p.rmsnorm(x, gamma, None, work("h", 1, s, c.hidden), c.eps)
            mm(p, work("h", 1, s, c.hidden), self._weight(n + "wgate"), work("gate", 1, s, c.ffn))
            mm(p, work("h", 1, s, c.hidden), self._weight(n + "wup"), work("up", 1, s, c.ffn))
            p.elemwise_binary(ss.GATE, work("gate", 1, s, c.ffn), work("up", 1, s, c.ffn), work("act", 1, s, c.ffn), act=ss.GELU)
            mm(p, work("act", 1, s, c.ffn), self._weight(n + "wdown"), work("o", 1, s, c.hidden))
            p.elemwise_binary(ss.ADD, x, work("o", 1, s, c.hidden), x)
        last = ss.tensor(b["x"], be.F32, (1, c.hidden), offset=(s - 1) * c.hidden * 4)
        p.rmsnorm(last, gamma, None, work("hl", 1, c.hidden), c.eps)
        mm(p, work("hl", 1, c.hidden), self._weight("lm_head"), ss.tensor(self.logits, be.F32, (1, c.vocab)))
        p.argmax(ss.tensor(self.logits, be.F32, (1, c.vocab)), ss.tensor(self.token, be.I32, (1,)), axis=1)
        if advance:
            one = ss.tensor(self.one, be.I32, (1,))
            p.copy(ss.tensor(self.token, be.I32, (1,)), ss.tensor(b["ids"], be.I32, (1,)))
            for t in (pos, widx, kvl):
                p.elemwise_binary(ss.ADD, t, one, t)
        self.state[key] = (b, p, p.array())
        return self.state[key]

    def _set_state(self, b, tokens, pos):
        g, t = self.gpu, np.ascontiguousarray(tokens, np.int32)
        g.write(b["ids"], t)
        g.write(b["positions"], np.arange(pos, pos + t.size, dtype=np.int32))
        g.write(b["write_index"], np.array([pos], np.int32))
        g.write(b["kv_len"], np.array([pos + t.size], np.int32))

    def prefill(self, tokens):
        s = len(tokens)
        if self.pos + s > self.cfg.max_seq:
            raise ValueError("prompt exceeds the cache capacity")
        b, _, arr = self._program(s)
        self._set_state(b, tokens, self.pos)
        self.sess.execute(arr)
        self.pos += s
        return int(self.gpu.download(self.token, np.int32, (1,))[0])

    def logits_host(self):
        return self.gpu.download(self.logits, np.float32, (self.cfg.vocab,))

    def begin_decode(self, first_token):
        """One eager step at the current position (weights, scratch), rolled back, then the list recorded as a program."""
        g = self.gpu
        b, _, arr = self._program(1, advance=True)
        if self.program is not None and not g.program_is_current(self.program):
            g.program_destroy(self.program)
            self.program = None
        if self.program is None:
            self._set_state(b, [first_token], self.pos)
            self.sess.execute(arr)
            g.sync()
            self.calls_per_step = self.sess.stats()[0]
            self.program = g.record_program(lambda: self.sess.execute(arr))
        self._set_state(b, [first_token], self.pos)

    def decode_step(self, read_token=True):
        if self.pos + 1 > self.cfg.max_seq:
            raise ValueError("cache capacity exhausted")
        self.gpu.program_execute(self.program)
        self.pos += 1
        return int(self.gpu.download(self.token, np.int32, (1,))[0]) if read_token else None

    def close(self):
        if self.program is not None:
            self.gpu.program_destroy(self.program)
            self.program = None
        self.sess.close()
        for buf in list(self.w.values()) + [self.embed, self.gamma, self.one, self.logits, self.token] + self.kc + self.vc:
            buf.free()
        seen = set()
        for b, _, _ in self.state.values():
            for buf in b.values():
                if id(buf) not in seen:
                    seen.add(id(buf))
                    buf.free()
        self.state = {}
