"""Key/value caches held in 8 or 4 bits: what their operators compute, in plain torch, and the framework's own calls for it.

  append     new rows of a layer's keys and values are quantised into their caches and read back (`step_append_quant`, `step_cache_read`)
  read       a span of cached rows as numbers (`step_cache_read`): to hand a prefix to another cache, or to code that takes f16 rows
  attention  one attention step over such caches (`step_attention`)

A cache of T rows for B sequences, H heads of D elements (D a multiple of 32) is one buffer. It holds the codes first, [B, H, Tp, D * bits / 8] bytes
with Tp = T rounded up to 64, then one f16 scale to every 32 elements of a row, [B, H, D / 32, Tp]. A code is stored with 128 (8 bits)
or 8 (4 bits, the even element in the low half of the byte) added, an element is code * scale.

`listed()` holds one case per kind of use, `draw()` samples the ranges they stand for.
"""
import math

import torch

own = False

BITS = {"q8": 8, "q4": 4}
FLOAT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HEADS = [(8, 1, 256), (8, 2, 256), (32, 8, 128), (32, 32, 128), (16, 4, 64)]


def listed():
    return [
        # one new token of one sequence: what a decode step adds to a layer's cache, the smallest call
        {"name": "append_q4_1x1", "family": "append", "cache": "q4", "batch": 1, "rows": 1, "capacity": 2048, "kv_heads": 8, "head": 128, "source": "f32", "rolling": False},
        # a token each for many sequences, each at its own place of a ring
        {"name": "append_q8_48x1_ring", "family": "append", "cache": "q8", "batch": 48, "rows": 1, "capacity": 1500, "kv_heads": 2, "head": 256, "source": "f32", "rolling": True},
        # a long prompt's rows at once
        {"name": "append_q4_1x8000", "family": "append", "cache": "q4", "batch": 1, "rows": 8000, "capacity": 8192, "kv_heads": 8, "head": 128, "source": "f32", "rolling": False},
        # a short prefix out of a cache, as f32 rows
        {"name": "read_q8_2x77", "family": "read", "cache": "q8", "batch": 2, "rows": 77, "capacity": 4096, "kv_heads": 4, "head": 64, "result": "f32", "rolling": False},
        # whole sequences as f16 rows
        {"name": "read_q4_4x16000", "family": "read", "cache": "q4", "batch": 4, "rows": 16000, "capacity": 16384, "kv_heads": 8, "head": 128, "result": "f16", "rolling": False},
        # one token over a short cache: latency
        {"name": "decode_q4_1x531", "family": "attention", "cache": "q4", "batch": 1, "queries": 1, "keys": 531, "heads": 8, "kv_heads": 1, "head": 256,
         "query": "f32", "window": 0, "rolling": False, "idle": False},
        # one token over a very long cache
        {"name": "decode_q8_1x131072", "family": "attention", "cache": "q8", "batch": 1, "queries": 1, "keys": 131072, "heads": 32, "kv_heads": 8, "head": 128,
         "query": "f32", "window": 0, "rolling": False, "idle": False},
        # a serving batch at ragged lengths, one slot of it idle
        {"name": "decode_q4_32x16384", "family": "attention", "cache": "q4", "batch": 32, "queries": 1, "keys": 16384, "heads": 32, "kv_heads": 8, "head": 128,
         "query": "f32", "window": 0, "rolling": False, "idle": True},
        # a layer with a sliding window over rings
        {"name": "decode_q8_16x1100_ring", "family": "attention", "cache": "q8", "batch": 16, "queries": 1, "keys": 1100, "heads": 16, "kv_heads": 4, "head": 64,
         "query": "f16", "window": 1023, "rolling": True, "idle": False},
        # the few tokens of a draft that are checked together, every query head with keys of its own
        {"name": "verify_q4_4x5x3001", "family": "attention", "cache": "q4", "batch": 4, "queries": 5, "keys": 3001, "heads": 32, "kv_heads": 32, "head": 128,
         "query": "bf16", "window": 0, "rolling": False, "idle": False},
        # a prompt over its own keys
        {"name": "prompt_q8_1x4096", "family": "attention", "cache": "q8", "batch": 1, "queries": 4096, "keys": 4096, "heads": 32, "kv_heads": 8, "head": 128,
         "query": "f32", "window": 0, "rolling": False, "idle": False},
        # a later piece of two prompts over what the cache holds of them
        {"name": "chunk_q4_2x500x9000", "family": "attention", "cache": "q4", "batch": 2, "queries": 500, "keys": 9000, "heads": 8, "kv_heads": 2, "head": 256,
         "query": "f32", "window": 0, "rolling": False, "idle": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw(rng):
    heads, kv_heads, head = rng.choice(HEADS)
    family = rng.choice(["append", "read", "attention", "attention", "attention"])
    case = {"family": family, "cache": rng.choice(["q8", "q4"]), "kv_heads": kv_heads, "head": head}
    if family != "attention":
        batch = _log(rng, 1, 64)
        rows = 1 if family == "append" and rng.random() < 0.4 else _log(rng, 1, 16384)
        case.update(batch=batch, rows=rows, capacity=rows + _log(rng, 1, 4096), rolling=rng.random() < 0.3)
        case.update({"source": rng.choice(["f32", "f32", "f16"])} if family == "append" else {"result": rng.choice(["f32", "f16", "bf16"])})
        return case
    u = rng.random()
    if u < 0.6:
        batch, queries, keys = _log(rng, 1, 64), 1, _log(rng, 1, 131072)
    elif u < 0.7:
        batch, queries, keys = _log(rng, 1, 16), rng.randint(2, 8), _log(rng, 16, 32768)
    elif u < 0.85:
        queries = _log(rng, 9, 4096)
        batch, keys = rng.choice([1, 1, 2, 4]), queries
    else:
        queries = _log(rng, 9, 1024)
        batch, keys = rng.choice([1, 1, 2, 4]), queries + _log(rng, 64, 16384)
    case.update(batch=batch, queries=queries, keys=keys, heads=heads, query=rng.choice(["f32", "f32", "f16", "bf16"]),
                window=0 if rng.random() < 0.7 else _log(rng, 64, 4096), rolling=queries == 1 and keys >= 64 and rng.random() < 0.25,
                idle=batch > 1 and queries == 1 and rng.random() < 0.3)
    return case


def draw(rng):
    most = {}
    for c in listed():
        most[_kind(c)] = max(most.get(_kind(c), 0.0), _cost(c))
    while True:
        case = _draw(rng)
        if _cost(case) <= most[_kind(case)]:
            return case


def _kind(case):
    return case["family"] + (" of many queries" if case.get("queries", 1) > 8 else "")


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 4e12, w["flops"] / 2e14)


# ---------------------------------------------------------------------------------------------------------- what a pass needs
def _row_bytes(case):
    """One row of one head in a cache: codes and scales."""
    return case["head"] * BITS[case["cache"]] // 8 + case["head"] // 32 * 2


def _lengths(case):
    """Keys of each sequence: a prompt fills its cache, sequences that are decoded together are at different lengths, and past the capacity of a ring."""
    t, b = case["keys"], case["batch"]
    if case["queries"] > 8:
        return [t] * b
    lengths = [max(min(t, case["queries"]), t - i * t // (2 * b)) for i in range(b)]
    if case["rolling"]:
        lengths = [n + (i % 4) * 797 for i, n in enumerate(lengths)]
    if case["idle"]:
        lengths[b // 2] = 0
    return lengths


def _spans(case):
    """Per sequence the (first, last + 1) visible key of each of its queries."""
    spans = []
    for length in _lengths(case):
        oldest = max(0, length - case["keys"]) if case["rolling"] else 0
        w = case["window"]
        spans.append([(max(oldest, 0 if w == 0 else p - w), p + 1) for p in range(length - case["queries"], length) if p >= 0])
    return spans


def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2}
    row = _row_bytes(case) * case["kv_heads"]
    if case["family"] != "attention":
        values = case["batch"] * case["rows"] * case["kv_heads"] * case["head"]
        if case["family"] == "read":
            return {"bytes": case["batch"] * case["rows"] * row + values * size[case["result"]], "flops": values}
        # keys and values: the new rows are read, their quantised form is written, and read again for the f32 rows that go out
        return {"bytes": 2 * (values * size[case["source"]] + 2 * case["batch"] * case["rows"] * row + values * 4), "flops": 2 * 6 * values}
    pairs = keys = 0
    for spans in _spans(case):
        if spans:
            pairs += sum(hi - lo for lo, hi in spans)
            keys += spans[-1][1] - spans[0][0]
    rows = case["batch"] * case["queries"] * case["heads"] * case["head"]
    return {"bytes": rows * (size[case["query"]] + 4) + 2 * keys * row, "flops": 4 * pairs * case["heads"] * case["head"]}


# ------------------------------------------------------------------------------------------------------- what a program has in hand
def _pad(rows):
    return (rows + 63) // 64 * 64


class _Cache:
    """A cache's buffer and its two parts as tensors."""

    def __init__(self, case, capacity):
        self.kind, self.batch, self.capacity, self.heads, self.head = case["cache"], case["batch"], capacity, case["kv_heads"], case["head"]
        tp = _pad(capacity)
        n_codes = self.batch * self.heads * tp * self.head * BITS[self.kind] // 8
        n_scales = self.batch * self.heads * tp * self.head // 32 * 2
        self.buffer = torch.zeros(n_codes + n_scales, dtype=torch.uint8, device="cuda")
        self.codes = self.buffer[:n_codes].view(self.batch, self.heads, tp, -1)
        self.scales = self.buffer[n_codes:].view(torch.float16).view(self.batch, self.heads, self.head // 32, tp)


def _quantise(x, kind):
    """Rows [..., D] in f32 as what is stored: codes [..., D * bits / 8] of uint8 and scales [..., D / 32] of f16. A block's scale is its largest
    magnitude over 127 or 7; 8-bit codes go by the scale as stored, 4-bit codes by the scale before it is rounded; halves are rounded away from zero."""
    blocks = x.unflatten(-1, (-1, 32))
    top = blocks.abs().amax(-1, keepdim=True)
    if kind == "q8":
        scale = torch.where(top == 0, torch.ones_like(top), top / 127).half()
        held = scale.float()
        by = torch.where((top == 0) | (held == 0), torch.zeros_like(held), 1 / held)
        lowest, most, off = -128, 127, 128
        v = blocks * by
    else:
        full = torch.where(top == 0, torch.ones_like(top), top / 7)
        scale = full.half()
        lowest, most, off = -8, 7, 8
        v = blocks / full
    a = v.abs().add_(0.5)
    a = torch.where(v.abs() == 0.49999997, torch.zeros_like(a), a.floor_())        # (its sum with a half is rounded up to one)
    codes = (torch.copysign(a, v).clamp_(lowest, most) + off).to(torch.uint8).flatten(-2)
    if kind == "q4":
        codes = codes[..., 0::2] | codes[..., 1::2] << 4
    return codes, scale.squeeze(-1)


def _values(codes, scales, kind):
    """What codes [..., D * bits / 8] and scales [..., D / 32] stand for, in f32."""
    if kind == "q4":
        codes = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
        x = codes.float().sub_(8.0)
    else:
        x = codes.float().sub_(128.0)
    return (x.unflatten(-1, (-1, 32)) * scales.float().unsqueeze(-1)).flatten(-2)


def _rows(generator, shape, head):
    """Rows as projections give them: a spread and an offset to each channel, a few channels far out."""
    spread = torch.exp(0.4 * torch.randn(head, generator=generator, device="cuda"))
    spread[torch.randint(head, (max(1, head // 64),), generator=generator, device="cuda")] *= 4.0
    offset = 0.5 * torch.randn(head, generator=generator, device="cuda")
    return torch.randn(*shape, head, generator=generator, device="cuda").mul_(spread).add_(offset)


def _filled(case, capacity, generator):
    """A cache every row of which has been written, a few sequences at a time."""
    cache = _Cache(case, capacity)
    step = max(1, (1 << 27) // (capacity * cache.heads * cache.head))
    for b in range(0, cache.batch, step):
        n = min(step, cache.batch - b)
        codes, scales = _quantise(_rows(generator, (n, cache.heads, capacity), cache.head), cache.kind)
        cache.codes[b:b + n, :, :capacity] = codes
        cache.scales[b:b + n, :, :, :capacity] = scales.transpose(2, 3)
    return cache


def _starts(case):
    """Where each sequence's rows begin: anywhere in a cache with room for them, past the capacity of a ring."""
    room = case["capacity"] - case["rows"]
    return [(i * 37) % (room + 1) + (case["capacity"] * (1 + i % 3) if case["rolling"] else 0) for i in range(case["batch"])]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    state = {"case": case}
    b, h, d = case["batch"], case["kv_heads"], case["head"]
    if case["family"] == "append":
        state["caches"] = [_Cache(case, case["capacity"]) for _ in range(2)]
        state["rows"] = [_rows(g, (b, case["rows"], h), d).to(FLOAT[case["source"]]) for _ in range(2)]
        state["index"] = torch.tensor(_starts(case), dtype=torch.int32, device="cuda")
        state["out"] = [torch.empty((b, case["rows"], h, d), device="cuda") for _ in range(2)]
    elif case["family"] == "read":
        state["caches"] = [_filled(case, case["capacity"], g)]
        state["index"] = torch.tensor(_starts(case), dtype=torch.int32, device="cuda")
        state["out"] = [torch.empty((b, case["rows"], h, d), dtype=FLOAT[case["result"]], device="cuda")]
    else:
        state["caches"] = [_filled(case, case["keys"], g) for _ in range(2)]
        state["q"] = torch.randn((b, case["queries"], case["heads"], d), generator=g, device="cuda").to(FLOAT[case["query"]])
        state["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")
        first = (state["lengths"] - case["queries"]).clamp_(min=0)
        state["positions"] = (first[:, None] + torch.arange(case["queries"], dtype=torch.int32, device="cuda")).contiguous()
        state["out"] = [torch.empty((b, case["queries"], case["heads"], d), device="cuda")]
    return state


# ------------------------------------------------------------------------------------------------------------------- the plain forms
def _places(case, index):
    """(sequence, row) index tensors of a span of rows, [B, 1] and [B, S]."""
    at = index.long()[:, None] + torch.arange(case["rows"], device=index.device)
    return torch.arange(case["batch"], device=index.device)[:, None], at % case["capacity"] if case["rolling"] else at


def _plain_append(state):
    case = state["case"]
    seq, at = _places(case, state["index"])
    out = []
    for cache, rows in zip(state["caches"], state["rows"]):
        codes, scales = _quantise(rows.float(), case["cache"])
        cache.codes.transpose(1, 2)[seq, at] = codes
        cache.scales.permute(0, 3, 1, 2)[seq, at] = scales
        out.append(_values(cache.codes.transpose(1, 2)[seq, at], cache.scales.permute(0, 3, 1, 2)[seq, at], case["cache"]))
    return out


def _plain_read(state):
    case, cache = state["case"], state["caches"][0]
    seq, at = _places(case, state["index"])
    return [_values(cache.codes.transpose(1, 2)[seq, at], cache.scales.permute(0, 3, 1, 2)[seq, at], case["cache"]).to(FLOAT[case["result"]])]


def _plain_attention(state):
    case = state["case"]
    b, l, t, hq, hk, d = (case[x] for x in ("batch", "queries", "keys", "heads", "kv_heads", "head"))
    k, v = (_values(c.codes[:, :, :t], c.scales[..., :t].transpose(2, 3), case["cache"]) for c in state["caches"])           # [B, Hk, T, D]
    q = state["q"].float().view(b, l, hk, hq // hk, d).permute(0, 2, 3, 1, 4).reshape(b, hk, -1, d)
    scores = torch.matmul(q, k.transpose(2, 3)).mul_(1.0 / math.sqrt(d)).view(b, hk, hq // hk, l, t)
    end, key = state["lengths"].long()[:, None, None], torch.arange(t, device=q.device)
    if case["rolling"]:                                      # the newest step that lies in each row
        key = end - 1 - (end - 1 - key) % t
    pos = state["positions"].long()[..., None]
    seen = (key >= 0) & (key < end) & (key <= pos)
    if case["window"]:
        seen = seen & (key >= pos - case["window"])
    seen = seen[:, None, None]
    scores = scores.masked_fill_(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(b, hk, -1, t), v).view(b, hk, -1, l, d) / torch.where(total == 0, torch.ones_like(total), total)
    return [out.permute(0, 3, 1, 2, 4).reshape(b, l, hq, d)]


# ------------------------------------------------------------------------------------------------------------------- the framework
_gpu = None


def _context():
    """One context for the whole program, as a serving process keeps it."""
    global _gpu
    if _gpu is None:
        from aion_amd import backend
        _gpu = backend.HipBackend(0)
    return _gpu


def _buffer(gpu, tensor):
    """A torch tensor's memory as an operand of the steps (the tensor keeps owning it)."""
    from aion_amd import backend
    return backend.DeviceBuffer(gpu, tensor.data_ptr(), tensor.numel() * tensor.element_size())


def _own(state):
    from aion_amd import backend as be
    gpu, case = _context(), state["case"]
    if "operands" not in state:                              # a program makes these once, with its buffers
        state["operands"] = {
            "caches": [_buffer(gpu, c.buffer) for c in state["caches"]], "out": [_buffer(gpu, x) for x in state["out"]],
            "rows": [_buffer(gpu, x) for x in state.get("rows", [])],
            **{name: _buffer(gpu, state[name]) for name in ("q", "lengths", "positions", "index") if name in state}}
    at = state["operands"]
    kind = {"q8": be.Q8_0, "q4": be.Q4_0}[case["cache"]]
    dtype = {"f32": be.F32, "f16": be.F16, "bf16": be.BF16}
    if case["family"] == "attention":
        b, l, t, hq, hk, d = (case[x] for x in ("batch", "queries", "keys", "heads", "kv_heads", "head"))
        gpu.step_attention(at["out"][0], at["q"], *at["caches"], (b, l, t, hq, hk, d, d), 1.0 / math.sqrt(d), q_dtype=dtype[case["query"]], kv_dtype=kind,
                           window=(case["window"], 0, 0) if case["window"] else be.CAUSAL, query_positions=at["positions"], kv_lengths=at["lengths"],
                           rolling=case["rolling"])
        return state["out"]
    shape = (case["batch"], case["rows"], case["capacity"], case["kv_heads"], case["head"])
    if case["family"] == "append":
        gpu.step_append_quant(kind, at["caches"], at["rows"], at["index"], shape, src_dtype=dtype[case["source"]], rolling=case["rolling"])
        gpu.step_cache_read(kind, at["out"], at["caches"], at["index"], shape, rolling=case["rolling"])
    else:
        gpu.step_cache_read(kind, at["out"], at["caches"], at["index"], shape, out_dtype=dtype[case["result"]], rolling=case["rolling"])
    return state["out"]


def run(state):
    if own:
        return _own(state)
    return {"append": _plain_append, "read": _plain_read, "attention": _plain_attention}[state["case"]["family"]](state)


# -------------------------------------------------------------------------------------------------------------- in 64 bits, row by row
def _stored(cache, b, h, rows):
    """Elements of the given rows of one head, from the two parts of the buffer, in f64."""
    byte = cache.codes[b, h, rows].to(torch.int64)
    if cache.kind == "q4":
        code = torch.zeros(byte.shape[0], cache.head, dtype=torch.float64, device=byte.device)
        code[:, 0::2], code[:, 1::2] = (byte % 16 - 8).double(), (torch.div(byte, 16, rounding_mode="floor") - 8).double()
    else:
        code = (byte - 128).double()
    return code * cache.scales[b, h][:, rows].double().repeat_interleave(32, 0).t()


def exact(case, seed):
    state = prepare(case, seed)
    if case["family"] == "append":
        out = []
        for x in state["rows"]:
            x = x.double().reshape(-1, 32)
            top = x.abs().max(1, keepdim=True).values
            steps = 127.0 if case["cache"] == "q8" else 7.0
            scale = top / steps
            held = scale.half().double()
            code = x / (held if case["cache"] == "q8" else scale)
            code = torch.where(code < 0, torch.ceil(code - 0.5), torch.floor(code + 0.5)).clamp(-128 if case["cache"] == "q8" else -8, steps)
            out.append(torch.where(held > 0, code * held, torch.zeros_like(code)).nan_to_num(0.0).view(state["out"][0].shape))
        return out
    if case["family"] == "read":
        cache, out = state["caches"][0], torch.empty(state["out"][0].shape, dtype=torch.float64, device="cuda")
        for b, start in enumerate(_starts(case)):
            rows = torch.tensor([(start + i) % case["capacity"] if case["rolling"] else start + i for i in range(case["rows"])], device="cuda")
            for h in range(case["kv_heads"]):
                out[b, :, h] = _stored(cache, b, h, rows)
        return [out]
    groups, out = case["heads"] // case["kv_heads"], torch.zeros(state["out"][0].shape, dtype=torch.float64, device="cuda")
    if work(case)["flops"] > 4e12:
        return None
    for b, spans in enumerate(_spans(case)):
        if not spans:
            continue
        first, last = min(lo for lo, _ in spans), max(hi for _, hi in spans)
        step = torch.arange(first, last, device="cuda")
        lo, hi = (torch.tensor([s[i] for s in spans], device="cuda") for i in (0, 1))
        hidden = (step < lo[:, None]) | (step >= hi[:, None])
        for h in range(case["kv_heads"]):
            rows = step % case["keys"] if case["rolling"] else step
            k, v = (_stored(c, b, h, rows) for c in state["caches"])
            for head in range(h * groups, (h + 1) * groups):
                s = state["q"][b, :, head].double() @ k.t().contiguous() / math.sqrt(case["head"])
                out[b, :, head] = torch.softmax(s.masked_fill(hidden, -math.inf), 1) @ v
    return [out]
