"""Key/value caches in pages: what their operators compute, in plain torch, and the framework's own calls for it.

  append     a step's queries and keys turned by their positions, keys and values written to the pages of their sequences (`step_rotary_append_paged`)
  rotary     rows turned by their positions and nothing else (`step_rotary`)
  attention  one attention step over the pages of each sequence (`step_attention_paged`), with what the step adds to the weight that each key has drawn
  evict      the rows of each sequence that have drawn the most weight, and the newest, moved to pages of their own (`step_evict_paged`)

A cache is two pools of pages, [pages, H, P, D] each for keys and values, and a table [B, W] of page numbers: step t of sequence b is row t % P of page
table[b, t // P]. An entry that is no page (-1) stands where a sequence has none.

`listed()` holds one case per kind of use, `draw()` samples the ranges they stand for.
"""
import math

import numpy as np
import torch

own = False

FLOAT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
HEADS = [(8, 1, 256), (8, 2, 256), (32, 8, 128), (32, 32, 128), (16, 4, 64)]
PAGES = [16, 32, 64, 128, 256]


def listed():
    return [
        # one new token of one sequence: what a decode step does in front of attention, the smallest call
        {"name": "append_1x1", "family": "append", "batch": 1, "rows": 1, "start": 700, "heads": 32, "kv_heads": 8, "head": 128, "dims": 128, "pairs": "halves",
         "scaling": "none", "source": "f32", "cache": "f16", "page": 64},
        # a token each for many sequences far into their texts, a quarter of each head turned, neighbours paired
        {"name": "append_64x1_far", "family": "append", "batch": 64, "rows": 1, "start": 900001, "heads": 8, "kv_heads": 2, "head": 256, "dims": 64, "pairs": "neighbours",
         "scaling": "linear", "source": "bf16", "cache": "bf16", "page": 16},
        # a long prompt's rows at once
        {"name": "append_1x8000", "family": "append", "batch": 1, "rows": 8000, "start": 0, "heads": 32, "kv_heads": 8, "head": 128, "dims": 128, "pairs": "halves",
         "scaling": "ramp", "source": "f32", "cache": "f16", "page": 64},
        # a short prompt's queries alone
        {"name": "rotary_2x77", "family": "rotary", "batch": 2, "rows": 77, "start": 5000, "heads": 16, "head": 64, "dims": 64, "pairs": "neighbours", "scaling": "none", "source": "f16"},
        # the queries of a long text
        {"name": "rotary_2x9000", "family": "rotary", "batch": 2, "rows": 9000, "start": 131072, "heads": 32, "head": 128, "dims": 96, "pairs": "halves", "scaling": "bands",
         "source": "f32"},
        # one token over a short cache in small pages: latency
        {"name": "token_1x531", "family": "attention", "batch": 1, "queries": 1, "keys": 531, "heads": 8, "kv_heads": 1, "head": 256, "query": "f32", "cache": "f16", "page": 16,
         "window": 0, "idle": False, "weigh": False},
        # one token over a very long cache
        {"name": "token_1x131072", "family": "attention", "batch": 1, "queries": 1, "keys": 131072, "heads": 32, "kv_heads": 8, "head": 128, "query": "f32", "cache": "f16", "page": 256,
         "window": 0, "idle": False, "weigh": False},
        # a serving batch at ragged lengths, one slot of it idle
        {"name": "token_32x16384", "family": "attention", "batch": 32, "queries": 1, "keys": 16384, "heads": 32, "kv_heads": 8, "head": 128, "query": "bf16", "cache": "bf16", "page": 64,
         "window": 0, "idle": True, "weigh": False},
        # a few sequences whose keys' weights are kept for the next eviction
        {"name": "token_8x9001_weighed", "family": "attention", "batch": 8, "queries": 1, "keys": 9001, "heads": 16, "kv_heads": 4, "head": 64, "query": "f32", "cache": "f16", "page": 32,
         "window": 0, "idle": False, "weigh": True},
        # the few tokens of a draft that are checked together, every query head with keys of its own
        {"name": "verify_4x5x3001", "family": "attention", "batch": 4, "queries": 5, "keys": 3001, "heads": 32, "kv_heads": 32, "head": 128, "query": "f16", "cache": "f16", "page": 128,
         "window": 0, "idle": False, "weigh": False},
        # sequences of a batch that have reached their limit, some of them not yet
        {"name": "evict_8x1280", "family": "evict", "batch": 8, "rows": 1280, "keep": 1024, "first": 4, "recent": 128, "kv_heads": 2, "head": 256, "cache": "f16", "page": 32, "ragged": True},
        # long prompts cut to what they go on with
        {"name": "evict_4x32768", "family": "evict", "batch": 4, "rows": 32768, "keep": 8192, "first": 16, "recent": 1024, "kv_heads": 8, "head": 128, "cache": "bf16", "page": 64,
         "ragged": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw(rng):
    heads, kv_heads, head = rng.choice(HEADS)
    family = rng.choice(["append", "append", "rotary", "attention", "attention", "attention", "attention", "evict", "evict"])
    case = {"family": family, "batch": _log(rng, 1, 64), "head": head}
    if family in ("append", "rotary"):
        case.update(rows=1 if rng.random() < 0.4 else _log(rng, 1, 9000), start=_log(rng, 1, 2000000) - 1, heads=heads, dims=head if rng.random() < 0.6 else 2 * rng.randint(8, head // 2),
                    pairs=rng.choice(["halves", "neighbours"]), scaling=rng.choice(["none", "linear", "bands", "ramp"]), source=rng.choice(["f32", "f32", "f16", "bf16"]))
        if family == "append":
            case.update(kv_heads=kv_heads, cache=rng.choice(["f16", "bf16"]), page=rng.choice(PAGES))
        return case
    case.update(kv_heads=kv_heads, cache=rng.choice(["f16", "bf16"]), page=rng.choice(PAGES))
    if family == "evict":
        keep = _log(rng, 48, 8192)
        recent = rng.randint(0, keep // 4)
        case.update(rows=min(65536, keep + _log(rng, 1, 24 * keep)), keep=keep, first=rng.choice([0, 4, rng.randint(0, keep // 8)]), recent=recent, ragged=rng.random() < 0.5)
        return case
    queries = 1 if rng.random() < 0.75 else rng.randint(2, 16)
    case.update(queries=queries, keys=max(queries, _log(rng, 1, 131072)), heads=heads, query=rng.choice(["f32", "f32", "f16", "bf16"]),
                window=0 if rng.random() < 0.75 else _log(rng, 16, 4096), idle=case["batch"] > 1 and rng.random() < 0.3, weigh=rng.random() < 0.3)
    return case


def draw(rng):
    most = {}
    for c in listed():
        most[c["family"]] = max(most.get(c["family"], 0.0), _cost(c))
    while True:
        case = _draw(rng)
        if _cost(case) <= most[case["family"]]:
            return case


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 4e12, w["flops"] / 2e14)


# ---------------------------------------------------------------------------------------------------------- what a pass needs
def _lengths(case):
    """Keys of each sequence: sequences that are decoded together are at different lengths."""
    b = case["batch"]
    if case["family"] == "evict":
        n, keep = case["rows"], case["keep"]
        return [n - (i * (n - keep // 2) // b if case["ragged"] else 0) for i in range(b)]
    t = case["keys"]
    lengths = [max(min(t, case["queries"]), t - i * t // (2 * b)) for i in range(b)]
    if case["idle"]:
        lengths[b // 2] = 0
    return lengths


def _spans(case):
    """Per sequence the (first, last + 1) visible key of each of its queries."""
    spans = []
    for length in _lengths(case):
        w = case["window"]
        spans.append([(0 if w == 0 else max(0, p - w), p + 1) for p in range(length - case["queries"], length) if p >= 0])
    return spans


def _up(n, to):
    return -(-n // to)


def work(case):
    b, d = case["batch"], case["head"]
    if case["family"] in ("append", "rotary"):
        rows, size = b * case["rows"], SIZE[case["source"]]
        turned = rows * (case["heads"] + case.get("kv_heads", 0)) * case["dims"]
        values = 2 * rows * case.get("kv_heads", 0) * d
        return {"bytes": 2 * rows * case["heads"] * d * size + values * (size + 2), "flops": 3 * turned}
    if case["family"] == "evict":
        h = case["kv_heads"]
        kept = sum(case["keep"] if n > case["keep"] else n for n in _lengths(case))
        return {"bytes": 4 * h * (sum(_lengths(case)) + b * _up(case["keep"], case["page"]) * case["page"] + b * case["keep"]) + 8 * h * kept * d, "flops": 0}
    pairs = keys = 0
    for spans in _spans(case):
        if spans:
            pairs += sum(hi - lo for lo, hi in spans)
            keys += spans[-1][1] - spans[0][0]
    rows = b * case["queries"] * case["heads"] * d
    weighed = 8 * b * case["kv_heads"] * _width(case) * case["page"] if case["weigh"] else 0
    return {"bytes": rows * (SIZE[case["query"]] + 4) + 4 * keys * case["kv_heads"] * d + weighed, "flops": 4 * pairs * case["heads"] * d}


# ------------------------------------------------------------------------------------------------------- what a program has in hand
def _width(case):
    """Entries of a sequence in the table."""
    return _up(case["keys"] if case["family"] == "attention" else case["rows"], case["page"]) + 1


def _rows(generator, shape, head):
    """Rows as projections give them: a spread and an offset to each channel, a few channels far out."""
    spread = torch.exp(0.4 * torch.randn(head, generator=generator, device="cuda"))
    spread[torch.randint(head, (max(1, head // 64),), generator=generator, device="cuda")] *= 4.0
    offset = 0.5 * torch.randn(head, generator=generator, device="cuda")
    return torch.randn(*shape, head, generator=generator, device="cuda").mul_(spread).add_(offset)


def _pool(case, pages, generator):
    """A pool every row of which has been written, a few pages at a time."""
    pool = torch.empty((pages, case["kv_heads"], case["page"], case["head"]), dtype=FLOAT[case["cache"]], device="cuda")
    step = max(1, (1 << 27) // pool[0].numel())
    for i in range(0, pages, step):
        pool[i:i + step] = _rows(generator, pool[i:i + step].shape[:-1], case["head"])
    return pool


def _table(counts, width, order):
    """Pages in no order to sequences that have `counts` of them, -1 behind."""
    table, at = torch.full((len(counts), width), -1, dtype=torch.int32), 0
    for i, n in enumerate(counts):
        table[i, :n] = order[at:at + n]
        at += n
    return table.cuda()


def _frequencies(case):
    """Radians a position for each pair of a head, in 64 bits. `linear`: positions are divided by 8. `bands`: what turns fewer than 1 time in 8192
    positions is slowed by 8, what turns more than 4 times is not, between them by how often. `ramp`: the same between pair numbers at which 1 and 32 turns lie."""
    n = case["dims"] // 2
    f = 500000.0 ** (-torch.arange(n, dtype=torch.float64, device="cuda") * 2 / case["dims"])
    if case["scaling"] == "none":
        return f
    if case["scaling"] == "linear":
        return f / 8
    if case["scaling"] == "bands":
        kept = ((8192 * f / (2 * math.pi) - 1) / (4 - 1)).clamp(0, 1)
    else:
        first, last = (case["dims"] * math.log(8192 / (turns * 2 * math.pi)) / (2 * math.log(500000.0)) for turns in (32, 1))
        first, last = max(math.floor(first), 0), min(math.ceil(last), case["dims"] - 1)
        kept = 1 - ((torch.arange(n, dtype=torch.float64, device="cuda") - first) / max(last - first, 1e-3)).clamp(0, 1)
    return f * kept + f / 8 * (1 - kept)


def _magnitude(case):
    return 1.25 if case["scaling"] == "ramp" else 1.0


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    on_cpu = torch.Generator().manual_seed(seed)
    state = {"case": case}
    b, d = case["batch"], case["head"]
    if case["family"] in ("append", "rotary"):
        starts = torch.tensor([case["start"] + i * 37 for i in range(b)], dtype=torch.int32, device="cuda")
        state["positions"] = (starts[:, None] + torch.arange(case["rows"], dtype=torch.int32, device="cuda")).contiguous()
        state["q"] = _rows(g, (b, case["rows"], case["heads"]), d).to(FLOAT[case["source"]])
        state["q_out"] = torch.empty_like(state["q"])
        if case["family"] == "append":
            width, p = _width(case), case["page"]
            state["k"], state["v"] = (_rows(g, (b, case["rows"], case["kv_heads"]), d).to(FLOAT[case["source"]]) for _ in range(2))
            state["index"] = torch.tensor([i % (p + 1) for i in range(b)], dtype=torch.int32, device="cuda")     # in a page of a sequence that has begun in it
            state["k_pages"], state["v_pages"] = (_pool(case, b * width, g) for _ in range(2))
            state["table"] = _table([width] * b, width, torch.randperm(b * width, generator=on_cpu).int())
        return state
    lengths = _lengths(case)
    counts, width = [_up(n, case["page"]) for n in lengths], _width(case)
    fresh = b * _up(case["keep"], case["page"]) if case["family"] == "evict" else 0
    pages = max(sum(counts), 1)
    state["k_pages"], state["v_pages"] = (_pool(case, pages + fresh, g) for _ in range(2))
    state["table"] = _table(counts, width, torch.randperm(pages, generator=on_cpu).int())
    state["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    weights = torch.exp(2.0 * torch.randn((b, case["kv_heads"], width * case["page"]), generator=g, device="cuda"))
    if case["family"] == "attention":
        state["q"] = torch.randn((b, case["queries"], case["heads"], d), generator=g, device="cuda").to(FLOAT[case["query"]])
        state["out"] = torch.empty((b, case["queries"], case["heads"], d), device="cuda")
        if case["weigh"]:
            state["weights"] = weights
            state["weights_out"] = torch.empty_like(weights)
        return state
    # weights as sums of probabilities are: many alike, some zero
    state["weights"] = torch.where(weights < 0.2, torch.zeros_like(weights), (weights * 64).round_() / 64)
    keep_width = _up(case["keep"], case["page"])
    state["table_out"] = _table([keep_width] * b, keep_width, torch.randperm(fresh, generator=on_cpu).int() + pages)
    state["weights_out"] = torch.empty((b, case["kv_heads"], keep_width * case["page"]), device="cuda")
    state["lengths_out"] = torch.empty_like(state["lengths"])
    state["kept"] = torch.empty((b, case["kv_heads"], case["keep"]), dtype=torch.int32, device="cuda")
    state["pages"] = pages
    return state


# ------------------------------------------------------------------------------------------------------------------- the plain forms
def _turned(x, positions, case):
    """Rows [B, S, H, D] in f32, turned: the angles in 64 bits."""
    n = case["dims"] // 2
    angle = positions.double()[..., None] * _frequencies(case)
    c, s = (f(angle).float().unsqueeze(2) * _magnitude(case) for f in (torch.cos, torch.sin))
    x = x.float()
    y = x.clone()
    if case["pairs"] == "halves":
        low, high = x[..., :n], x[..., n:2 * n]
        y[..., :n], y[..., n:2 * n] = low * c - high * s, low * s + high * c
    else:
        low, high = x[..., 0:2 * n:2], x[..., 1:2 * n:2]
        y[..., 0:2 * n:2], y[..., 1:2 * n:2] = low * c - high * s, low * s + high * c
    return y


def _plain_rotary(state):
    return [_turned(state["q"], state["positions"], state["case"]).to(state["q"].dtype)]


def _plain_append(state):
    case = state["case"]
    step = state["index"].long()[:, None] + torch.arange(case["rows"], device="cuda")
    page = torch.gather(state["table"].long(), 1, step // case["page"])
    q = _turned(state["q"], state["positions"], case).to(state["q"].dtype)
    state["k_pages"][page, :, step % case["page"]] = _turned(state["k"], state["positions"], case).to(FLOAT[case["cache"]])
    state["v_pages"][page, :, step % case["page"]] = state["v"].to(FLOAT[case["cache"]])
    return [q, state["k_pages"], state["v_pages"]]


def _gathered(pool, table, page):
    """Every row of each sequence, [B, H, W * P, D] in f32."""
    x = pool[table.long().clamp(min=0)]
    return x.transpose(1, 2).flatten(2, 3).float()


def _plain_attention(state):
    case = state["case"]
    b, l, hq, hk, d = (case[x] for x in ("batch", "queries", "heads", "kv_heads", "head"))
    k, v = (_gathered(state[x], state["table"], case["page"]) for x in ("k_pages", "v_pages"))
    t = k.shape[2]
    q = state["q"].float().view(b, l, hk, hq // hk, d).permute(0, 2, 3, 1, 4).reshape(b, hk, -1, d)
    scores = torch.matmul(q, k.transpose(2, 3)).mul_(1.0 / math.sqrt(d)).view(b, hk, hq // hk, l, t)
    key = torch.arange(t, device="cuda")
    pos = state["lengths"].long()[:, None, None] - l + torch.arange(l, device="cuda")[:, None]
    seen = key <= pos
    if case["window"]:
        seen = seen & (key >= pos - case["window"])
    seen = seen[:, None, None]
    scores = scores.masked_fill_(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)))
    total = p.sum(-1, keepdim=True)
    total = torch.where(total == 0, torch.ones_like(total), total)
    out = torch.matmul(p.view(b, hk, -1, t), v).view(b, hk, -1, l, d) / total
    result = [out.permute(0, 3, 1, 2, 4).reshape(b, l, hq, d)]
    if case["weigh"]:
        result.append(state["weights"] + (p / total).sum((2, 3)))
    return result


def _plain_evict(state):
    case = state["case"]
    b, h, p, keep = case["batch"], case["kv_heads"], case["page"], case["keep"]
    n = state["lengths"].long()[:, None, None]
    slot = torch.arange(state["weights"].shape[2], device="cuda")
    rank = state["weights"].masked_fill((slot < case["first"]) | (slot >= n - case["recent"]), math.inf).masked_fill(slot >= n, -math.inf)
    best = torch.sort(rank, dim=2, descending=True, stable=True).indices[..., :keep]
    count = torch.minimum(n, torch.full_like(n, keep))
    row = torch.arange(keep, device="cuda")
    best = torch.sort(best.masked_fill(row >= count, slot.numel()), dim=2).values
    live = row < count
    kept = torch.where(live, best, torch.full_like(best, -1))
    at = kept.clamp(min=0)
    seq, head = torch.arange(b, device="cuda")[:, None, None], torch.arange(h, device="cuda")[None, :, None]
    source = state["table"].long().clamp(min=0)[seq, at // p]
    target = state["table_out"].long()[seq, (row // p).expand_as(at)]
    for name in ("k_pages", "v_pages"):
        rows = state[name][source, head, at % p]
        old = state[name][target, head, row % p]
        state[name][target, head, (row % p).expand_as(at)] = torch.where(live[..., None], rows, old)
    weights = torch.zeros_like(state["weights_out"])
    weights[..., :keep] = torch.where(live, torch.gather(state["weights"], 2, at), torch.zeros((), device="cuda"))
    return [kept.int(), count.flatten().int(), weights, state["k_pages"][state["pages"]:], state["v_pages"][state["pages"]:]]


# ------------------------------------------------------------------------------------------------------------------- the framework
_gpu = None


def _context():
    """One context for the whole program, as a serving process keeps it."""
    global _gpu
    if _gpu is None:
        from aion_amd import backend
        _gpu = backend.HipBackend(0)
    return _gpu


def _operands(gpu, state):
    """Torch tensors' memory as operands of the steps (the tensors keep owning it), the cache and the turning: a program makes these once, with its buffers."""
    from aion_amd import backend as be
    case = state["case"]
    dtype = {"f32": be.F32, "f16": be.F16, "bf16": be.BF16}
    at = {name: be.DeviceBuffer(gpu, x.data_ptr(), x.numel() * x.element_size()) for name, x in state.items() if torch.is_tensor(x)}
    if "table" in state:
        at["cache"] = gpu.paged_cache(at["k_pages"], at["v_pages"], at["table"], state["k_pages"].shape[0], case["batch"], state["table"].shape[1], case["page"], case["kv_heads"],
                                      case["head"], dtype[case["cache"]])
    if "dims" in case:
        scaling = {"none": be.ROTARY_PLAIN, "linear": be.ROTARY_LINEAR, "bands": be.ROTARY_BANDS, "ramp": be.ROTARY_RAMP}[case["scaling"]]
        low, high = (1.0, 4.0) if case["scaling"] == "bands" else (1.0, 32.0)
        at["rotary"] = be.Rotary(case["dims"], base=500000.0, interleaved=case["pairs"] == "neighbours", scaling=scaling, factor=8.0, original_length=8192.0, low=low, high=high,
                                 magnitude=_magnitude(case))
    at["source"], at["query"] = dtype[case.get("source", "f32")], dtype[case.get("query", "f32")]
    return at


def _own(state):
    gpu, case = _context(), state["case"]
    if "operands" not in state:
        state["operands"] = _operands(gpu, state)
    at = state["operands"]
    if case["family"] == "rotary":
        gpu.step_rotary(at["q_out"], at["q"], at["positions"], case["batch"], case["rows"], case["heads"], case["head"], at["rotary"], dtype=at["source"])
        return [state["q_out"]]
    if case["family"] == "append":
        gpu.step_rotary_append_paged(at["cache"], at["rotary"], at["q_out"], at["q"], at["k"], at["v"], at["positions"], at["index"], case["rows"], case["heads"], dtype=at["source"])
        return [state["q_out"], state["k_pages"], state["v_pages"]]
    if case["family"] == "attention":
        from aion_amd import backend as be
        gpu.step_attention_paged(at["out"], at["q"], at["cache"], case["queries"], case["heads"], 1.0 / math.sqrt(case["head"]), q_dtype=at["query"],
                                 window=(case["window"], 0, 0) if case["window"] else be.CAUSAL, kv_lengths=at["lengths"], weights=at.get("weights_out"),
                                 weights_before=at.get("weights"))
        return [state["out"]] + ([state["weights_out"]] if case["weigh"] else [])
    gpu.step_evict_paged(at["cache"], at["weights"], at["lengths"], at["weights_out"], at["lengths_out"], case["keep"], first=case["first"], recent=case["recent"],
                         table_out=at["table_out"], width_out=state["table_out"].shape[1], kept=at["kept"])
    return [state["kept"], state["lengths_out"], state["weights_out"], state["k_pages"][state["pages"]:], state["v_pages"][state["pages"]:]]


def run(state):
    if own:
        return _own(state)
    return {"append": _plain_append, "rotary": _plain_rotary, "attention": _plain_attention, "evict": _plain_evict}[state["case"]["family"]](state)


# -------------------------------------------------------------------------------------------------------------- in 64 bits, row by row
def _exact_turn(x, positions, case):
    """Each pair as a complex number, times one of length `magnitude` at its position's angle."""
    x, n = x.double().clone(), case["dims"] // 2
    turn = torch.polar(torch.full((1,), _magnitude(case), dtype=torch.float64, device="cuda"), torch.remainder(positions.double()[:, :, None, None] * _frequencies(case), 2 * math.pi))
    low, high = (slice(0, n), slice(n, 2 * n)) if case["pairs"] == "halves" else (slice(0, 2 * n, 2), slice(1, 2 * n, 2))
    y = torch.complex(x[..., low].contiguous(), x[..., high].contiguous()) * turn
    x[..., low], x[..., high] = y.real, y.imag
    return x


def _exact_append(state):
    case, out = state["case"], [_exact_turn(state["q"], state["positions"], state["case"])]
    for pool, rows in ((state["k_pages"], _exact_turn(state["k"], state["positions"], case)), (state["v_pages"], state["v"].double())):
        pool = pool.double()
        for b in range(case["batch"]):
            first, at = int(state["index"][b]), 0
            while at < case["rows"]:                        # a page's run at a time
                page, row = int(state["table"][b, (first + at) // case["page"]]), (first + at) % case["page"]
                n = min(case["page"] - row, case["rows"] - at)
                pool[page, :, row:row + n] = rows[b, at:at + n].transpose(0, 1)
                at += n
        out.append(pool)
    return out


def _exact_attention(state):
    case = state["case"]
    if work(case)["flops"] > 4e12:
        return None
    groups, out = case["heads"] // case["kv_heads"], torch.zeros(state["out"].shape, dtype=torch.float64, device="cuda")
    weights = state["weights"].double() if case["weigh"] else None
    for b, spans in enumerate(_spans(case)):
        if not spans:
            continue
        last, skip = spans[-1][1], case["queries"] - len(spans)
        pages = state["table"][b, :_up(last, case["page"])].long()
        step = torch.arange(last, device="cuda")
        lo, hi = (torch.tensor([s[i] for s in spans], device="cuda") for i in (0, 1))
        hidden = (step < lo[:, None]) | (step >= hi[:, None])
        for h in range(case["kv_heads"]):
            k, v = (state[x][pages, h].reshape(-1, case["head"])[:last].double() for x in ("k_pages", "v_pages"))
            for head in range(h * groups, (h + 1) * groups):
                s = state["q"][b, skip:, head].double() @ k.t().contiguous() / math.sqrt(case["head"])
                p = torch.softmax(s.masked_fill(hidden, -math.inf), 1)
                out[b, skip:, head] = p @ v
                if weights is not None:
                    weights[b, h, :last] += p.sum(0)
    return [out] + ([weights] if case["weigh"] else [])


def _exact_evict(state):
    case, p = state["case"], state["case"]["page"]
    table, table_out = state["table"].cpu().numpy(), state["table_out"].cpu().numpy()
    w = state["weights"].cpu().numpy().astype(np.float64)
    k, v = (state[x].double() for x in ("k_pages", "v_pages"))
    kept = np.full(state["kept"].shape, -1, np.int32)
    weights = np.zeros(state["weights_out"].shape)
    lengths = [min(n, case["keep"]) for n in _lengths(case)]
    for b, n in enumerate(_lengths(case)):
        for h in range(case["kv_heads"]):
            rows = np.arange(n)
            if n > case["keep"]:
                middle = np.arange(case["first"], n - case["recent"])
                order = np.lexsort((middle, -w[b, h, middle]))
                middle = np.sort(middle[order[:case["keep"] - case["first"] - case["recent"]]])
                rows = np.concatenate((np.arange(case["first"]), middle, np.arange(n - case["recent"], n)))
            kept[b, h, :rows.size], weights[b, h, :rows.size] = rows, w[b, h, rows]
            to = np.arange(rows.size)
            source, source_row, target, target_row = (torch.from_numpy(x.astype(np.int64)).cuda() for x in (table[b, rows // p], rows % p, table_out[b, to // p], to % p))
            for pool in (k, v):
                pool[target, h, target_row] = pool[source, h, source_row]
    return [torch.from_numpy(kept), torch.tensor(lengths, dtype=torch.int32), torch.from_numpy(weights), k[state["pages"]:], v[state["pages"]:]]


def exact(case, seed):
    state = prepare(case, seed)
    if case["family"] == "rotary":
        return [_exact_turn(state["q"], state["positions"], case)]
    return {"append": _exact_append, "attention": _exact_attention, "evict": _exact_evict}[case["family"]](state)
