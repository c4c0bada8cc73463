"""Measured cases of the operators around the paged 4-bit key/value cache.

Four operators, as one decode step of a batch of conversations uses them:

- ``tables``: the block table, the slot of every new token and the lengths of a batch, built on the GPU from
  how many tokens each conversation keeps and how many it brings;
- ``store``: keys and values quantised to 4 bits (groups of 64 along the head dimension, one float16 scale and
  low per group), written to the slots, and read back as the values they stand for;
- ``attend``: the new tokens stored, then causal attention of their queries over the whole 4-bit cache;
- ``choose``: penalties for repeated tokens, biases and a grammar mask on the logits, and the best token.

``run`` computes them in elementary torch operations, or (``own``) through the calls of this package. ``exact``
computes the same from the definitions in 64 bits.
"""

import math
import os
import random
import sys

import torch

own = False

PAGE = 64   # tokens of a page
GROUP = 64  # elements that share a scale and a low

GEOMETRY = {  # query heads, key/value heads, head dimension
    "1b": (32, 8, 64),
    "3b": (24, 8, 128),
}
VOCAB = 128256


def _package():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "dimmer-kv_b200")
    if path not in sys.path:
        sys.path.insert(0, path)


# ----------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # One conversation takes its next token: the smallest call, all latency.
        dict(name="tables-token", op="tables", n_seq=1, low=327, high=327, new=1, ragged=False),
        # 64 prompts of 4K to 16K tokens arrive at once: about 640 thousand slots.
        dict(name="tables-prompts", op="tables", n_seq=64, low=0, high=0, new=16384, ragged=True),
        # One decoded token of 16 conversations.
        dict(name="store-token", op="store", geometry="1b", dtype="float16", n_seq=16, new=1, ragged=False),
        # The prompts of 16 conversations, ragged up to 4095 tokens.
        dict(name="store-prompts", op="store", geometry="3b", dtype="bfloat16", n_seq=16, new=4095, ragged=True),
        # One short conversation, one token.
        dict(name="attend-1b-1x1536", op="attend", geometry="1b", dtype="bfloat16", n_seq=1, low=1536, high=1536,
             new=1, ragged=False),
        # One long conversation, one token: all of the GPU on one row of heads.
        dict(name="attend-3b-1x131072", op="attend", geometry="3b", dtype="bfloat16", n_seq=1, low=131072,
             high=131072, new=1, ragged=False),
        # A decode step of the batch that this repository's benchmark serves: 64 conversations, 4K to 16K tokens.
        dict(name="attend-3b-64x16384", op="attend", geometry="3b", dtype="bfloat16", n_seq=64, low=4096,
             high=16384, new=1, ragged=False),
        # Short drafts of up to five tokens over odd lengths, some conversations just begun.
        dict(name="attend-1b-drafts", op="attend", geometry="1b", dtype="float16", n_seq=9, low=0, high=8191,
             new=5, ragged=True),
        # A question of 64 tokens over one context of 32K.
        dict(name="attend-3b-question", op="attend", geometry="3b", dtype="bfloat16", n_seq=1, low=32768,
             high=32768, new=64, ragged=False),
        # Prompt chunks of 512 tokens over contexts of up to 8K.
        dict(name="attend-3b-chunk", op="attend", geometry="3b", dtype="float16", n_seq=4, low=2047, high=8191,
             new=512, ragged=False),
        # The next token of one conversation.
        dict(name="choose-1", op="choose", n_seq=1, vocab=VOCAB, dtype="bfloat16", history=1536, n_bias=0,
             grammar=False),
        # The next tokens of 64 conversations with long histories, biases and a grammar each.
        dict(name="choose-64", op="choose", n_seq=64, vocab=VOCAB, dtype="bfloat16", history=4096, n_bias=64,
             grammar=True),
    ]


def _between(rng, low, high):
    """A whole number of [low, high], spread over its logarithm."""
    return min(high, max(low, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    op = rng.choice(["tables", "store", "attend", "attend", "choose"])
    if op == "tables":
        high = _between(rng, 1, 16384)
        return dict(op=op, n_seq=_between(rng, 1, 64), low=rng.randint(0, high), high=high,
                    new=_between(rng, 1, 16384), ragged=rng.random() < 0.7)
    if op == "choose":
        return dict(op=op, n_seq=_between(rng, 1, 64), vocab=_between(rng, 1000, VOCAB),
                    dtype=rng.choice(["bfloat16", "float16", "float32"]), history=_between(rng, 1, 16384),
                    n_bias=rng.choice([0, _between(rng, 1, 300)]), grammar=rng.random() < 0.5)
    geometry = rng.choice(["1b", "3b"])
    dtype = rng.choice(["bfloat16", "float16"])
    n_seq = _between(rng, 1, 64)
    if op == "store":
        new = _between(rng, 1, max(1, 65000 // n_seq))
        return dict(op=op, geometry=geometry, dtype=dtype, n_seq=n_seq, new=new, ragged=rng.random() < 0.6)
    new = rng.choice([1, 1, rng.randint(2, 8), _between(rng, 9, 512)])
    high = _between(rng, 1, 131072)
    # Bounded by the listed batch step's cache bytes and by the listed chunk's products.
    n_seq = max(1, min(n_seq, 640000 // (high + new), 12 * 10 ** 6 // (new * (high + new))))
    high = min(high, max(1, 12 * 10 ** 6 // new - new))
    return dict(op=op, geometry=geometry, dtype=dtype, n_seq=n_seq, low=rng.randint(0, high), high=high, new=new,
                ragged=rng.random() < 0.5)


def _lengths(case):
    """(tokens held, new tokens) of every conversation: part of the case, not of the seed."""
    rng = random.Random(case["n_seq"] * 7919 + case["new"] * 31 + case.get("high", 0))
    n, low, high, new = case["n_seq"], case.get("low", 0), case.get("high", 0), case["new"]
    held = [high if n == 1 else rng.randint(low, high) for _ in range(n)]
    fresh = [new] * n
    if case["ragged"] and n > 1:
        # A quarter of the full count or more, the first conversation with all of it; in short drafts some
        # conversations bring nothing.
        fresh = [new] + [rng.randint(0 if new <= 8 else max(1, new // 4), new) for _ in range(n - 1)]
    return held, fresh


def _round_up(x, m):
    return (x + m - 1) // m * m


def work(case):
    n = case["n_seq"]
    if case["op"] == "choose":
        size = 4 if case["dtype"] == "float32" else 2
        words = (case["vocab"] + 31) // 32 if case["grammar"] else 0
        b = n * (case["vocab"] * (size + 4) + case["history"] * 4 + case["n_bias"] * 8 + words * 4 + 24)
        return {"bytes": b, "flops": n * case["vocab"]}
    held, fresh = _lengths(case)
    if case["op"] == "tables":
        pages = [_round_up(h + f, PAGE) // PAGE for h, f in zip(held, fresh)]
        cols = _round_up(max(h + f for h, f in zip(held, fresh)), PAGE) // PAGE
        # keep, lengths and counts in; lengths and starts out; the block table's rows; one slot a token
        return {"bytes": n * 4 * 5 + sum(pages) * 4 + n * cols * 4 + n * case["new"] * 4,
                "flops": n * case["new"]}
    q_heads, kv_heads, dim = GEOMETRY[case["geometry"]]
    cell = kv_heads * (dim // 2 + dim // GROUP * 4)  # bytes of one token's keys (or values) in 4 bits
    if case["op"] == "store":
        tokens = sum(fresh)
        return {"bytes": 2 * (tokens * kv_heads * dim * 2 + 2 * tokens * cell + n * case["new"] * kv_heads * dim * 2),
                "flops": 2 * tokens * kv_heads * dim * 6}
    total = sum(h + f for h, f in zip(held, fresh))
    new = sum(fresh)
    seen = sum(f * h + f * (f + 1) // 2 for h, f in zip(held, fresh))  # (query, key) pairs of a head
    io = new * q_heads * dim * 2 + n * case["new"] * q_heads * dim * 2 + 2 * new * kv_heads * dim * 2
    return {"bytes": 2 * total * cell + io, "flops": 4 * seen * q_heads * dim}


# ----------------------------------------------------------------------------------------------- inputs
def _generator(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed((seed * 1000003 + case["n_seq"] * 101 + case.get("new", 0) * 7 + case.get("high", 0)) % (1 << 62))
    return g


def _dtype(case):
    return getattr(torch, case["dtype"])


def _rows(g, n, heads, tokens, dim, dtype, kind):
    """[n, heads, tokens, dim] as the model's projections leave it: a transposed view of [n, tokens, heads, dim].
    Keys have a mean of their own in every channel and a few wide channels; values are centred."""
    x = torch.randn(n, tokens, heads, dim, generator=g, device="cuda", dtype=torch.float32)
    if kind == "key":
        c = torch.arange(dim, device="cuda", dtype=torch.float32)
        x = x * (0.6 + 2.0 * (c % 29 == 3)) + torch.sin(c * 1.7) * 1.5
    elif kind == "value":
        x = x * 0.5
    return x.to(dtype).transpose(1, 2)


def _history(g, case):
    """Token ids with repeats, as text has them: small ids far more often than large ones."""
    u = torch.rand(case["n_seq"], case["history"], generator=g, device="cuda")
    return (u.pow(3) * (case["vocab"] - 1)).to(torch.int32)


def _inputs(case, seed):
    """Everything random of a case, made in one order from the seed (``prepare`` and ``exact`` share it)."""
    g = _generator(case, seed)
    n = case["n_seq"]
    if case["op"] == "tables":
        held, fresh = _lengths(case)
        # The free pages lie in an order of their own, as after hours of serving.
        pages = _pool(case)
        return dict(held=torch.tensor(held, dtype=torch.int32, device="cuda"),
                    new=torch.tensor(fresh, dtype=torch.int32, device="cuda"),
                    free=torch.randperm(pages, generator=g, device="cuda").to(torch.int32))
    if case["op"] == "choose":
        v = case["vocab"]
        logits = (torch.randn(n, v, generator=g, device="cuda") * 3).to(_dtype(case))
        history = _history(g, case)
        half = max(1, case["history"] // 2)
        lengths = torch.randint(half, case["history"] + 1, (n,), generator=g, device="cuda", dtype=torch.int32)
        prompts = torch.div(lengths, 2, rounding_mode="floor").to(torch.int32)
        pen = lambda lo, hi: torch.rand(n, generator=g, device="cuda") * (hi - lo) + lo
        out = dict(logits=logits, history=history, lengths=lengths, prompts=prompts, repetition=pen(1.0, 1.4),
                   frequency=pen(0.0, 0.5), presence=pen(0.0, 0.6), bias_ids=None, bias_values=None, allowed=None)
        if case["n_bias"]:
            k = min(case["n_bias"], v)
            first = torch.randint(0, v, (n, 1), generator=g, device="cuda")
            out["bias_ids"] = ((first + torch.arange(k, device="cuda") * max(1, v // k)) % v).to(torch.int32)
            out["bias_values"] = torch.randn(n, k, generator=g, device="cuda") * 4
        if case["grammar"]:
            words = (v + 31) // 32
            out["allowed"] = torch.randint(-2 ** 31, 2 ** 31, (n, words), generator=g, device="cuda",
                                           dtype=torch.int64).to(torch.int32)
        return out
    q_heads, kv_heads, dim = GEOMETRY[case["geometry"]]
    dtype = _dtype(case)
    held, fresh = _lengths(case)
    out = dict(held=held, fresh=fresh,
               key=_rows(g, n, kv_heads, case["new"], dim, dtype, "key"),
               value=_rows(g, n, kv_heads, case["new"], dim, dtype, "value"))
    if case["op"] == "attend":
        out["query"] = _rows(g, n, q_heads, case["new"], dim, dtype, "query")
        out["scaling"] = dim ** -0.5
    out["generator"] = g  # the context's chunks follow
    return out


def _context(case, inputs):
    """The held tokens in chunks: (first token, counts per conversation, keys, values)."""
    n = case["n_seq"]
    _, kv_heads, dim = GEOMETRY[case["geometry"]]
    step = max(64, 65536 // n)
    for first in range(0, max(inputs["held"]), step):
        counts = [min(step, max(0, h - first)) for h in inputs["held"]]
        size = max(counts)
        yield (first, counts, _rows(inputs["generator"], n, kv_heads, size, dim, _dtype(case), "key"),
               _rows(inputs["generator"], n, kv_heads, size, dim, _dtype(case), "value"))


def _pool(case):
    """Pages of the pool: what the conversations need, and some to spare."""
    held, fresh = _lengths(case)
    return sum(_round_up(h + f, PAGE) // PAGE for h, f in zip(held, fresh)) + case["n_seq"] + 3


def _capacity(case):
    held, fresh = _lengths(case)
    return _round_up(max(h + f for h, f in zip(held, fresh)), PAGE)


# ----------------------------------------------------------------------------------------------- prepare
def prepare(case, seed):
    inputs = _inputs(case, seed)
    state = dict(case=case, **{k: v for k, v in inputs.items() if k != "generator"})
    n = case["n_seq"]
    if own:
        _package()
    if case["op"] == "tables":
        if own:
            from dimmerkv.paging import PageTable

            table = PageTable(n, _pool(case), _capacity(case), device="cuda", free=inputs["free"])
            table.plan(inputs["held"], max(1, case["high"]))
            state["table"] = table
        else:
            cols = _capacity(case) // PAGE
            held = inputs["held"].long()
            taken = (held + PAGE - 1) // PAGE
            rank = (taken.cumsum(0) - taken)[:, None] + torch.arange(cols, device="cuda")
            mine = torch.arange(cols, device="cuda") < taken[:, None]
            top = inputs["free"].flip(0)
            state["blocks"] = torch.where(mine, top[rank.clamp_max(top.numel() - 1)], -1).to(torch.int32)
            state["n_free"] = inputs["free"].numel() - int(taken.sum())
    elif case["op"] == "choose":
        if own:
            from dimmerkv.logits import LogitRules

            rules = LogitRules(n, case["vocab"], device="cuda", capacity=case["history"] + 1,
                               repetition=inputs["repetition"], frequency=inputs["frequency"],
                               presence=inputs["presence"], bias_ids=inputs["bias_ids"],
                               bias_values=inputs["bias_values"])
            rules.load(inputs["history"], inputs["lengths"], inputs["prompts"])
            state["rules"] = rules
    else:
        q_heads, kv_heads, dim = GEOMETRY[case["geometry"]]
        counts = torch.tensor(inputs["fresh"], dtype=torch.int32, device="cuda")
        if own:
            from dimmerkv.q4 import Q4Batch

            batch = Q4Batch(n, layers=1, kv_heads=kv_heads, q_heads=q_heads, head_dim=dim, max_tokens=_capacity(case),
                            n_pages=_pool(case), device="cuda", dtype=_dtype(case))
            for _, part, keys, values in _context(case, inputs):
                batch.plan(torch.tensor(part, dtype=torch.int32, device="cuda"), keys.shape[2])
                batch.append(0, keys, values)
            batch.plan(counts, case["new"])
            state["batch"] = batch
        elif case["op"] == "attend":
            cap = _capacity(case)
            cache = {k: dict(codes=torch.zeros(n, kv_heads, cap, dim // 2, dtype=torch.uint8, device="cuda"),
                             scale=torch.zeros(n, kv_heads, cap, dim // GROUP, dtype=torch.float16, device="cuda"),
                             low=torch.zeros(n, kv_heads, cap, dim // GROUP, dtype=torch.float16, device="cuda"))
                     for k in ("key", "value")}
            for first, part, keys, values in _context(case, inputs):
                for kind, x in (("key", keys), ("value", values)):
                    for s, c in enumerate(part):
                        if c:
                            _plain_write(cache[kind], s, first, x[s, :, :c])
            state["cache"] = cache
        state["counts"] = counts
    return state


# ----------------------------------------------------------------------------------------------- plain form
def _plain_quantise(x):
    """[..., dim] -> codes (whole numbers 0..15), scale and low (float16, one per group). The codes are taken in
    64 bits: a value next to a border between two of them must not cross it by a rounding."""
    g = x.float().unflatten(-1, (-1, GROUP))
    low = g.amin(-1).half()
    scale = ((g.amax(-1) - low.float()) / 15).half()
    step = scale.double()[..., None]
    q = (g.double() - low.double()[..., None]) / torch.where(step > 0, step, 1.0)
    q = torch.where(step > 0, q.round().clamp(0, 15), 0.0)
    return q.to(torch.uint8).flatten(-2), scale, low


def _plain_value(codes, scale, low):
    g = codes.float().unflatten(-1, (-1, GROUP))
    return (g * scale.float()[..., None] + low.float()[..., None]).flatten(-2)


def _plain_write(cache, s, first, x):
    codes, scale, low = _plain_quantise(x)
    end = first + x.shape[-2]
    cache["codes"][s, :, first:end] = codes[..., ::2] | (codes[..., 1::2] << 4)
    cache["scale"][s, :, first:end] = scale
    cache["low"][s, :, first:end] = low


def _plain_read(cache, s, end):
    packed = cache["codes"][s, :, :end]
    codes = torch.stack([packed & 15, packed >> 4], dim=-1).flatten(-2)
    return _plain_value(codes, cache["scale"][s, :, :end], cache["low"][s, :, :end])


def _plain_tables(state):
    case = state["case"]
    held, new, blocks = state["held"].long(), state["new"].long(), state["blocks"]
    cols = blocks.shape[1]
    have, need = (held + PAGE - 1) // PAGE, (held + new + PAGE - 1) // PAGE
    take = need - have
    rank = (take.cumsum(0) - take)[:, None] + torch.arange(cols, device="cuda") - have[:, None]
    col = torch.arange(cols, device="cuda")
    mine = (col >= have[:, None]) & (col < need[:, None])
    page = state["free"][(state["n_free"] - 1 - rank).clamp(0, state["free"].numel() - 1)]
    blocks = torch.where(mine, page, blocks)
    i = torch.arange(case["new"], device="cuda")
    at = held[:, None] + i
    page = blocks.gather(1, (at // PAGE).clamp_max(cols - 1)).long()
    slots = torch.where(i < new[:, None], page * PAGE + at % PAGE, -1).to(torch.int32)
    return slots, blocks, (held + new).to(torch.int32), state["held"]


def _plain_store(state):
    keep = (torch.arange(state["key"].shape[2], device="cuda") < state["counts"][:, None])[:, None, :, None]
    out = []
    for x in (state["key"], state["value"]):
        out.append(torch.where(keep, _plain_value(*_plain_quantise(x)), 0.0).to(x.dtype))
    return tuple(out)


def _plain_attend(state):
    query = state["query"]
    n, q_heads, q_len, dim = query.shape
    kv_heads = state["key"].shape[1]
    out = torch.zeros(n, q_len, q_heads, dim, dtype=query.dtype, device="cuda")
    for s in range(n):
        held, new = state["held"][s], state["fresh"][s]
        if new == 0:
            continue
        for kind in ("key", "value"):
            _plain_write(state["cache"][kind], s, held, state[kind][s, :, :new])
        keys = _plain_read(state["cache"]["key"], s, held + new)
        values = _plain_read(state["cache"]["value"], s, held + new)
        q = query[s, :, :new].float().unflatten(0, (kv_heads, -1))  # [kv, group, new, dim]
        hidden = torch.arange(held + new, device="cuda") > held + torch.arange(new, device="cuda")[:, None]
        for h in range(kv_heads):
            scores = torch.matmul(q[h], keys[h].T) * state["scaling"]
            scores = scores.masked_fill(hidden, -math.inf)
            p = torch.exp(scores - scores.amax(-1, keepdim=True))
            o = torch.matmul(p, values[h]) / p.sum(-1, keepdim=True)  # [group, new, dim]
            group = q.shape[1]
            out[s, :new, h * group:(h + 1) * group] = o.transpose(0, 1).to(out.dtype)
    return out


def _plain_choose(state):
    x = state["logits"].float()
    n, v = x.shape
    at = torch.arange(state["history"].shape[1], device="cuda")
    real = at < state["lengths"][:, None]
    made = real & (at >= state["prompts"][:, None])
    ids = state["history"].long()
    seen = torch.zeros(n, v, device="cuda").scatter_add_(1, ids, real.float()) > 0
    count = torch.zeros(n, v, device="cuda").scatter_add_(1, ids, made.float())
    r = state["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
    x = x - state["frequency"][:, None] * count
    x = torch.where(count > 0, x - state["presence"][:, None], x)
    if state["bias_ids"] is not None:
        x = x.scatter_add(1, state["bias_ids"].long(), state["bias_values"])
    if state["allowed"] is not None:
        bit = torch.arange(v, device="cuda")
        word = state["allowed"][:, bit // 32]
        x = torch.where((word >> (bit % 32)) & 1 != 0, x, -math.inf)
    best = x.amax(-1, keepdim=True)
    first = torch.where(x == best, torch.arange(v, device="cuda"), v).amin(-1)
    return x, torch.where(best[:, 0] == -math.inf, -1, first)


# ----------------------------------------------------------------------------------------------- run
def run(state):
    op = state["case"]["op"]
    if not own:
        return {"tables": _plain_tables, "store": _plain_store, "attend": _plain_attend,
                "choose": _plain_choose}[op](state)
    if op == "tables":
        # The conversations go back to what they keep, then the new tokens get their slots.
        table = state["table"]
        table.trim(state["held"])
        slots = table.plan(state["new"], state["case"]["new"])
        return slots, table.blocks, table.lengths, table.starts
    if op == "store":
        state["batch"].append(0, state["key"], state["value"])
        return state["batch"].read(0)
    if op == "attend":
        return state["batch"].attend_layer(0, state["query"], state["key"], state["value"], state["scaling"])
    return state["rules"].apply(state["logits"], state["allowed"])


# ----------------------------------------------------------------------------------------------- exact
def _exact_cells(x):
    """The values that 4 bits hold for x, in 64 bits."""
    x64 = x.double()
    parts = []
    for first in range(0, x.shape[-1], GROUP):
        g = x64[..., first:first + GROUP]
        low = g.min(-1, keepdim=True).values.half().double()
        scale = ((g.max(-1, keepdim=True).values - low) / 15).float().half().double()
        k = torch.where(scale > 0, torch.round((g - low) / scale.clamp_min(1e-30)), torch.zeros_like(g))
        parts.append(low + scale * k.clamp(0, 15))
    return torch.cat(parts, -1)


def exact(case, seed):
    if case["op"] == "tables":
        return None
    inputs = _inputs(case, seed)
    n = case["n_seq"]
    if case["op"] == "choose":
        rows = []
        for s in range(n):
            x = inputs["logits"][s].double()
            length, prompt = int(inputs["lengths"][s]), int(inputs["prompts"][s])
            ids = inputs["history"][s, :length].long()
            total = torch.bincount(ids, minlength=case["vocab"])
            made = torch.bincount(ids[prompt:], minlength=case["vocab"]).double()
            r = inputs["repetition"][s].double()
            x = torch.where((total > 0) & (x > 0), x / r, torch.where(total > 0, x * r, x))
            x = x - inputs["frequency"][s].double() * made - inputs["presence"][s].double() * (made > 0)
            if inputs["bias_ids"] is not None:
                x.index_add_(0, inputs["bias_ids"][s].long(), inputs["bias_values"][s].double())
            if inputs["allowed"] is not None:
                bits = torch.arange(32, device="cuda")
                ok = ((inputs["allowed"][s][:, None] >> bits) & 1).bool().flatten()[:case["vocab"]]
                x[~ok] = -math.inf
            rows.append(x)
        return torch.stack(rows), None
    if case["op"] == "store":
        out = []
        for x in (inputs["key"], inputs["value"]):
            y = torch.zeros(x.shape, dtype=torch.float64, device="cuda")
            for s, c in enumerate(inputs["fresh"]):
                y[s, :, :c] = _exact_cells(x[s, :, :c])
            out.append(y)
        return tuple(out)
    held, fresh = inputs["held"], inputs["fresh"]
    q_heads, kv_heads, dim = GEOMETRY[case["geometry"]]
    share = q_heads // kv_heads
    keys = [[] for _ in range(n)]
    values = [[] for _ in range(n)]
    for _, counts, k, v in _context(case, inputs):
        for s, c in enumerate(counts):
            if c:
                keys[s].append(k[s, :, :c])
                values[s].append(v[s, :, :c])
    out = torch.zeros(n, case["new"], q_heads, dim, dtype=torch.float64, device="cuda")
    for s in range(n):
        c = fresh[s]
        if not c:
            continue
        k = _exact_cells(torch.cat(keys[s] + [inputs["key"][s, :, :c]], 1))
        v = _exact_cells(torch.cat(values[s] + [inputs["value"][s, :, :c]], 1))
        last = held[s] + torch.arange(c, device="cuda")
        sees = torch.arange(held[s] + c, device="cuda")[None] <= last[:, None]
        for h in range(q_heads):
            z = inputs["query"][s, h, :c].double() @ k[h // share].transpose(0, 1) * inputs["scaling"]
            z = z.masked_fill(~sees, -math.inf)
            out[s, :c, h] = torch.softmax(z, -1) @ v[h // share]
    return out
