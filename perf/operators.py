"""Bounded- and shared-cache attention operators: what is measured, on which inputs, and what the results are.

Five operators around the KV cache of a serving engine (cache rows [token][kv_head][head_dim], fp16 or bf16):

  sink_decode   decode / few-token attention over the first `sink` tokens and a sliding window (optionally a ring cache)
  sink_prefill  the same visibility for a prompt chunk
  prefix        decode / few-token attention of sessions that share a long prefix, the prefix read once per group
  accumulate    decode / few-token attention that also adds every key's attention weight to a per-row statistic
  evict         eviction from a cache by that statistic: the rows to keep are chosen per KV head and compacted

`own` selects what run() does: False, the plain form in elementary torch operations; True, the framework's calls.
"""
import math
import random

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


# ------------------------------------------------------------------ cases

def listed():
    return [
        # one chat session of the dense 2B-shaped model deep into an endless stream: latency of one token
        {"name": "sink decode, 1 session", "op": "sink_decode", "dtype": "fp16", "hq": 8, "hkv": 2, "hd": 256, "n": 1, "rows": 1,
         "sink": 4, "window": 1020, "ring": 1024, "lo": 200_000, "hi": 400_000},
        # the 35B-A3B-shaped decode batch with ragged contexts, a 4096-token window over plain (unwrapped) caches
        {"name": "sink decode, 32 sessions", "op": "sink_decode", "dtype": "bf16", "hq": 16, "hkv": 2, "hd": 256, "n": 32, "rows": 1,
         "sink": 4, "window": 4096, "ring": 0, "lo": 1024, "hi": 32768},
        # a chunk of a long prompt written into a ring cache
        {"name": "sink prefill, chunk of 1000", "op": "sink_prefill", "dtype": "fp16", "hq": 16, "hkv": 2, "hd": 256, "start": 7001,
         "tokens": 1000, "sink": 4, "window": 1024, "ring": 2048},
        # a whole prompt of the prefill configuration, sixteen sinks, a window of a quarter of it
        {"name": "sink prefill, 8192 tokens", "op": "sink_prefill", "dtype": "bf16", "hq": 16, "hkv": 2, "hd": 256, "start": 0,
         "tokens": 8192, "sink": 16, "window": 2048, "ring": 0},
        # four continuations of one system prompt, just begun
        {"name": "prefix, 4 sessions", "op": "prefix", "dtype": "fp16", "hq": 8, "hkv": 2, "hd": 256, "groups": 1, "per": 4, "rows": 1,
         "prefix_lo": 2000, "prefix_hi": 2000, "lo": 1, "hi": 128},
        # a served batch behind one long shared document
        {"name": "prefix, 64 sessions", "op": "prefix", "dtype": "fp16", "hq": 16, "hkv": 2, "hd": 256, "groups": 1, "per": 64, "rows": 1,
         "prefix_lo": 32768, "prefix_hi": 32768, "lo": 1, "hi": 1024},
        # speculative verify (4 draft rows, 125B-A6B-shaped heads) of four tenants with a prompt each
        {"name": "prefix verify, 4 x 4 sessions", "op": "prefix", "dtype": "bf16", "hq": 32, "hkv": 2, "hd": 256, "groups": 4, "per": 4,
         "rows": 4, "prefix_lo": 6000, "prefix_hi": 16384, "lo": 4, "hi": 700},
        # statistics of one session at the dense configuration's context
        {"name": "accumulate, 1 session", "op": "accumulate", "dtype": "fp16", "hq": 8, "hkv": 2, "hd": 256, "n": 1, "rows": 1,
         "lo": 4096, "hi": 4096},
        # statistics of the whole ragged decode batch
        {"name": "accumulate, 32 sessions", "op": "accumulate", "dtype": "bf16", "hq": 16, "hkv": 2, "hd": 256, "n": 32, "rows": 1,
         "lo": 1024, "hi": 32768},
        # one session at its budget: one token in, one out, every step
        {"name": "evict one row", "op": "evict", "dtype": "fp16", "hkv": 2, "hd": 256, "n": 1, "lo": 2049, "hi": 2049, "budget": 2048,
         "sink": 4, "recent": 256, "in_place": True},
        # a batch that evicts a block of rows every couple of hundred steps
        {"name": "evict a block, 32 sessions", "op": "evict", "dtype": "bf16", "hkv": 2, "hd": 256, "n": 32, "lo": 3900, "hi": 4352,
         "budget": 4096, "sink": 4, "recent": 512, "in_place": True},
        # a long prompt's cache reduced into a session's small one
        {"name": "evict a prompt of 131071", "op": "evict", "dtype": "fp16", "hkv": 2, "hd": 256, "n": 1, "lo": 131071, "hi": 131071,
         "budget": 8192, "sink": 4, "recent": 1024, "in_place": False},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["sink_decode", "sink_prefill", "prefix", "accumulate", "evict"])
    dtype = rng.choice(["fp16", "bf16"])
    hq, hkv = rng.choice([(8, 2), (16, 2), (24, 2), (32, 2), (8, 1), (16, 4), (8, 8)])
    hd = rng.choice([64, 128, 256, 256])
    wide = max(1, hkv * hd // 512)                                              # rows wider than 2 x 256: fewer sessions
    if op == "sink_decode":
        n = _log_int(rng, 1, 48 // wide)
        rows = rng.choice([1, 1, 1, 2, 4])
        window = _log_int(rng, 16, 4096)
        ring = rng.choice([0, window + rows - 1 + rng.randrange(0, 300)])
        hi = _log_int(rng, 64, 16384) if ring == 0 else _log_int(rng, 64, 1_000_000)
        return {"op": op, "dtype": dtype, "hq": hq, "hkv": hkv, "hd": hd, "n": n, "rows": rows, "sink": rng.choice([0, 1, 4, 4, 16, 100]),
                "window": window, "ring": ring, "lo": max(rows, hi // 16), "hi": max(rows, hi)}
    if op == "sink_prefill":
        # head_dim 256: the head size of every full-attention configuration here
        tokens = _log_int(rng, 1, 4096)
        window = _log_int(rng, 64, 4096)
        ring = rng.choice([0, (window + tokens + 62) // 64 * 64 + 64 * rng.randrange(0, 4)])
        return {"op": op, "dtype": dtype, "hq": rng.choice([8, 16]), "hkv": 2, "hd": 256, "start": rng.choice([0, _log_int(rng, 1, 12000)]),
                "tokens": tokens, "sink": rng.choice([0, 1, 4, 4, 16, 200]), "window": window, "ring": ring}
    if op == "prefix":
        groups = rng.choice([1, 1, 2, 3])
        rows = rng.choice([1, 1, 2, 4])
        prefix = _log_int(rng, 32, 16384)
        suffix = _log_int(rng, 4, 1024)
        return {"op": op, "dtype": dtype, "hq": hq, "hkv": hkv, "hd": hd, "groups": groups,
                "per": _log_int(rng, 1, 48 // groups // max(1, rows // 2)), "rows": rows, "prefix_lo": max(1, prefix // 3),
                "prefix_hi": prefix, "lo": rows, "hi": max(rows, suffix)}
    if op == "accumulate":
        n = _log_int(rng, 1, 32 // wide)
        hi = _log_int(rng, 8, 16384)
        return {"op": op, "dtype": dtype, "hq": hq, "hkv": hkv, "hd": hd, "n": n,
                "rows": rng.choice([1, 1, 2, 4]), "lo": max(4, hi // 16), "hi": max(4, hi)}
    n = _log_int(rng, 1, 32 // wide)
    hi = _log_int(rng, 40, 131072 // n // wide)
    budget = max(8, int(hi * rng.uniform(0.1, 0.95)))
    sink = rng.choice([0, 1, 4])
    return {"op": op, "dtype": dtype, "hkv": hkv, "hd": hd, "n": n, "lo": max(4, hi // 2), "hi": hi,
            "budget": budget, "sink": sink, "recent": rng.randrange(0, budget - sink + 1), "in_place": rng.random() < 0.5}


# ------------------------------------------------------------------ inputs

def _lens(rng, n, lo, hi):
    got = [rng.randint(lo, hi) for _ in range(n)]
    got[rng.randrange(n)] = hi
    return got


def prepare(case, seed):
    """The caches, queries and statistics a serving process holds before the call."""
    rng = random.Random(seed * 7919 + 17)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt, op = DTYPES[case["dtype"]], case["op"]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=dt)

    s = dict(case)
    hkv, hd = case["hkv"], case["hd"]
    if op == "sink_decode":
        n, w, hq = case["n"], case["rows"], case["hq"]
        s["lens"] = _lens(rng, n, case["lo"], case["hi"])
        cap = case["sink"] + case["ring"] if case["ring"] else max(s["lens"])
        s["q"], s["k"], s["v"] = normal(n, w, hq, hd), normal(n, cap, hkv, hd), normal(n, cap, hkv, hd)
        s["out"] = torch.empty_like(s["q"])
    elif op == "sink_prefill":
        t, hq = case["tokens"], case["hq"]
        valid = case["start"] + t
        cap = case["sink"] + case["ring"] if case["ring"] else valid
        s["valid"] = valid
        s["q"], s["k"], s["v"] = normal(t, hq, hd), normal(cap, hkv, hd), normal(cap, hkv, hd)
        s["out"] = torch.empty_like(s["q"])
    elif op == "prefix":
        g, per, w, hq = case["groups"], case["per"], case["rows"], case["hq"]
        s["prefix_lens"] = _lens(rng, g, case["prefix_lo"], case["prefix_hi"])
        s["lens"] = _lens(rng, g * per, case["lo"], case["hi"])
        s["pk"], s["pv"] = normal(g, max(s["prefix_lens"]), hkv, hd), normal(g, max(s["prefix_lens"]), hkv, hd)
        s["q"], s["k"], s["v"] = normal(g * per, w, hq, hd), normal(g * per, max(s["lens"]), hkv, hd), normal(g * per, max(s["lens"]), hkv, hd)
        s["out"] = torch.empty_like(s["q"])
        s["prefix_lens_d"] = torch.tensor(s["prefix_lens"], device="cuda")
    elif op == "accumulate":
        n, w, hq = case["n"], case["rows"], case["hq"]
        s["lens"] = _lens(rng, n, case["lo"], case["hi"])
        cap = max(s["lens"])
        s["q"], s["k"], s["v"] = normal(n, w, hq, hd), normal(n, cap, hkv, hd), normal(n, cap, hkv, hd)
        s["out"] = torch.empty_like(s["q"])
        s["weights"] = torch.rand(n, hkv, cap, generator=gen, device="cuda").square_().mul_(2.0)
        s["positions"] = torch.arange(cap, device="cuda", dtype=torch.int32).expand(n, hkv, cap).contiguous()
        s["ends"] = [x + 5 for x in s["lens"]]          # some rows were evicted earlier: rows and positions differ
    else:
        n, budget = case["n"], case["budget"]
        s["lens"] = _lens(rng, n, case["lo"], case["hi"])
        cap = max(s["lens"])
        s["k"], s["v"] = normal(n, cap, hkv, hd), normal(n, cap, hkv, hd)
        # accumulated softmax weights are heavy-tailed; the newest rows have collected little and tie at zero
        s["weights"] = torch.randn(n, hkv, cap, generator=gen, device="cuda").mul_(2.0).exp_()
        s["weights"][:, :, cap - cap // 16:] = 0.0
        # an earlier eviction left the rows in a scrambled order of positions, another one per head
        perm = torch.rand(n, hkv, cap, generator=gen, device="cuda").argsort(-1)
        s["positions"] = perm.to(torch.int32)
        s["ends"] = [cap] * n
        s["kept"] = [min(x, budget) for x in s["lens"]]
        s["weights_out"] = torch.zeros(n, hkv, budget, device="cuda")
        s["positions_out"] = torch.zeros(n, hkv, budget, device="cuda", dtype=torch.int32)
        room = min(budget, cap)
        s["k_out"] = s["k"][:, :room] if case["in_place"] else torch.zeros(n, room, hkv, hd, device="cuda", dtype=dt)
        s["v_out"] = s["v"][:, :room] if case["in_place"] else torch.zeros(n, room, hkv, hd, device="cuda", dtype=dt)
        s["ends_d"] = torch.tensor(s["ends"], device="cuda")
    if "lens" in s:
        s["lens_d"] = torch.tensor(s["lens"], device="cuda")
    torch.cuda.synchronize()
    return s


# ------------------------------------------------------------------ the framework's calls

_runtime = None


def _framework():
    """The context and the operators a program creates once."""
    global _runtime
    if _runtime is None:
        import tinytitan_b200 as tt
        context = tt.Context(torch.cuda.current_device())
        _runtime = (tt, context, tt.Attention(context), tt.PrefillAttention(context))
    return _runtime


def _run_own(s):
    tt, context, attention, prefill = _framework()
    op, hd, hkv = s["op"], s["hd"], s["hkv"]
    if op == "sink_decode":
        sessions = tt.SessionTable.over_cache(s["q"], s["out"], s["k"], s["v"], s["lens"])
        attention.encode_sink_window(sessions, hd, s["hq"], hkv, s["sink"], s["window"], ring_capacity=s["ring"])
        return s["out"]
    if op == "sink_prefill":
        params = tt.PrefillAttentionParams(s["start"], s["tokens"], hd, s["hq"], hkv, s["valid"], s["window"], hkv * hd, s["hq"] * hd,
                                           s["hq"] * hd, 1.0 / math.sqrt(hd))
        prefill.encode_sink_window(s["q"], s["k"], s["v"], s["out"], params, s["sink"], kv_ring_capacity=s["ring"])
        return s["out"]
    if op == "prefix":
        groups = tt.PrefixTable.over_cache(s["pk"], s["pv"], s["prefix_lens"], s["per"])
        sessions = tt.SessionTable.over_cache(s["q"], s["out"], s["k"], s["v"], s["lens"])
        attention.encode_shared_prefix(groups, sessions, hd, s["hq"], hkv)
        return s["out"]
    if op == "accumulate":
        sessions = tt.SessionTable.over_cache(s["q"], s["out"], s["k"], s["v"], s["lens"])
        attention.encode_accumulate(sessions, s["weights"], hd, s["hq"], hkv, positions=s["positions"], fresh_rows=s["rows"],
                                    end_positions=s["ends"])
        return s["out"], s["weights"], s["positions"]
    tt.evict_kv_rows(context, s["k"], s["v"], s["weights"], s["lens"], s["budget"], sink_tokens=s["sink"], recent_tokens=s["recent"],
                     positions=s["positions"], end_positions=s["ends"], k_out=s["k_out"], v_out=s["v_out"],
                     weights_out=s["weights_out"], positions_out=s["positions_out"])
    return s["k_out"], s["v_out"], s["weights_out"], s["positions_out"]


# ------------------------------------------------------------------ the plain form

def _softmax_sums(scores, visible):
    """exp(scores - max) over the visible entries, their sum (zero where nothing is visible), and the maximum."""
    scores = scores.masked_fill(~visible, -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    e = torch.exp(scores - top)
    return e, e.sum(-1, keepdim=True), top


def _normalised(x, total):
    return torch.where(total > 0, x / total, torch.zeros_like(x))


def _plain_sink_decode(s):
    n, w, hq, hkv, hd = s["n"], s["rows"], s["hq"], s["hkv"], s["hd"]
    sink, window, ring = s["sink"], s["window"], s["ring"]
    lens = s["lens_d"][:, None]
    # candidate keys of a session: the sinks, then the union of its rows' windows behind them
    c = torch.arange(sink + window + w - 1, device="cuda")[None]
    first = (lens - (w - 1) - window).clamp(min=sink)
    key = torch.where(c < sink, c, first + c - sink)                            # [n, C]
    row = torch.where(key < sink, key, sink + (key - sink) % ring) if ring else key
    row = row.clamp(max=s["k"].shape[1] - 1)
    which = torch.arange(n, device="cuda")[:, None]
    k, v = s["k"][which, row].float(), s["v"][which, row].float()               # [n, C, hkv, hd]
    end = lens - (w - 1) + torch.arange(w, device="cuda")[None]                 # [n, w]: keys below it are causal
    visible = (key[:, None] < end[..., None]) & ((key[:, None] < sink) | (key[:, None] >= end[..., None] - window))
    q = s["q"].float().reshape(n, w, hkv, hq // hkv, hd)
    scores = torch.einsum("nwhgd,nchd->nwhgc", q, k) / math.sqrt(hd)
    e, total, _ = _softmax_sums(scores, visible[:, :, None, None])
    out = _normalised(torch.einsum("nwhgc,nchd->nwhgd", e, v), total)
    return out.reshape(n, w, hq, hd).to(s["q"].dtype)


def _plain_sink_prefill(s):
    t, hq, hkv, hd, sink, ring = s["tokens"], s["hq"], s["hkv"], s["hd"], s["sink"], s["ring"]
    low = max(0, s["start"] + 1 - s["window"]) if ring else 0                   # a ring has only the rows that are still needed
    key = torch.cat([torch.arange(min(sink, low), device="cuda"), torch.arange(low, s["valid"], device="cuda")])
    row = torch.where(key < sink, key, sink + (key - sink) % ring) if ring else key
    k, v = s["k"][row].float(), s["v"][row].float()
    at = s["start"] + torch.arange(t, device="cuda")[:, None]
    visible = (key[None] <= at) & ((key[None] < sink) | (key[None] > at - s["window"]))
    q = s["q"].float().reshape(t, hkv, hq // hkv, hd)
    scores = torch.einsum("thgd,chd->hgtc", q, k) / math.sqrt(hd)
    e, total, _ = _softmax_sums(scores, visible)
    out = _normalised(torch.einsum("hgtc,chd->hgtd", e, v), total)
    return out.permute(2, 0, 1, 3).reshape(t, hq, hd).to(s["q"].dtype)


def _plain_prefix(s):
    g, per, w, hq, hkv, hd = s["groups"], s["per"], s["rows"], s["hq"], s["hkv"], s["hd"]
    n = g * per
    q = s["q"].float().reshape(n, w, hkv, hq // hkv, hd)
    shared = torch.einsum("gnwhed,gchd->gnwhec", q.reshape(g, per, w, hkv, -1, hd), s["pk"].float()) / math.sqrt(hd)
    seen = torch.arange(shared.shape[-1], device="cuda")[None] < s["prefix_lens_d"][:, None]
    e, total, top = _softmax_sums(shared, seen[:, None, None, None, None])
    acc = torch.einsum("gnwhec,gchd->gnwhed", e, s["pv"].float()).reshape(n, w, hkv, -1, hd)
    total, top = total.reshape(n, w, hkv, -1, 1), top.reshape(n, w, hkv, -1, 1)
    tail = torch.einsum("nwhed,nchd->nwhec", q, s["k"].float()) / math.sqrt(hd)
    end = s["lens_d"][:, None] - (w - 1) + torch.arange(w, device="cuda")[None]
    seen = torch.arange(tail.shape[-1], device="cuda") < end[..., None]
    e2, total2, top2 = _softmax_sums(tail, seen[:, :, None, None])
    acc2 = torch.einsum("nwhec,nchd->nwhed", e2, s["v"].float())
    best = torch.maximum(top, top2)
    a, b = torch.exp(top - best), torch.exp(top2 - best)
    return _normalised(acc * a + acc2 * b, total * a + total2 * b).reshape(n, w, hq, hd).to(s["q"].dtype)


def _plain_accumulate(s):
    n, w, hq, hkv, hd = s["n"], s["rows"], s["hq"], s["hkv"], s["hd"]
    q = s["q"].float().reshape(n, w, hkv, hq // hkv, hd)
    key = torch.arange(s["k"].shape[1], device="cuda")
    scores = torch.einsum("nwhgd,nchd->nwhgc", q, s["k"].float()) / math.sqrt(hd)
    end = s["lens_d"][:, None] - (w - 1) + torch.arange(w, device="cuda")[None]
    e, total, _ = _softmax_sums(scores, (key < end[..., None])[:, :, None, None])
    p = _normalised(e, total)
    out = torch.einsum("nwhgc,nchd->nwhgd", p, s["v"].float()).reshape(n, w, hq, hd).to(s["q"].dtype)
    lens = s["lens_d"][:, None, None]
    fresh = (key >= lens - w) & (key < lens)
    weights = torch.where(fresh, torch.zeros_like(s["weights"]), s["weights"]) + p.sum((1, 3))
    s["weights"].copy_(torch.where(key < lens, weights, s["weights"]))
    position = (lens + 5 - (lens - key)).to(torch.int32)
    s["positions"].copy_(torch.where(fresh, position, s["positions"]))
    return out, s["weights"], s["positions"]


def _plain_evict(s):
    n, hkv, hd, budget = s["n"], s["hkv"], s["hd"], s["budget"]
    cap = s["k"].shape[1]
    row = torch.arange(cap, device="cuda")
    lens, ends = s["lens_d"][:, None, None], s["ends_d"][:, None, None]
    protected = (s["positions"] < s["sink"]) | (s["positions"] >= ends - s["recent"])
    rank = torch.where(protected, torch.full_like(s["weights"], math.inf), s["weights"])
    rank = torch.where(row < lens, rank, torch.full_like(rank, -math.inf))
    order = rank.sort(dim=-1, descending=True, stable=True).indices
    keep = torch.zeros(n, hkv, cap, dtype=torch.bool, device="cuda")
    keep.scatter_(-1, order[..., :budget], True)
    keep &= row < lens
    # kept rows stay where they are; the rows given up below `budget` are filled, in order, by the kept rows above it
    room = min(budget, cap)
    hole = ~keep[..., :room]
    fill = (~(keep & (row >= budget))).to(torch.uint8).sort(dim=-1, stable=True).indices
    src = torch.where(hole, fill.gather(-1, (hole.cumsum(-1) - 1).clamp(min=0)), row[:room])
    live = row[:room] < lens.clamp(max=budget)
    src = torch.where(live, src, row[:room])
    which, head = torch.arange(n, device="cuda")[:, None, None], torch.arange(hkv, device="cuda")[None, :, None]
    mask = live.transpose(1, 2)[..., None]
    k, v = s["k"][which, src, head].transpose(1, 2), s["v"][which, src, head].transpose(1, 2)
    s["k_out"].copy_(torch.where(mask, k, s["k_out"]))
    s["v_out"].copy_(torch.where(mask, v, s["v_out"]))
    s["weights_out"][..., :room] = torch.where(live, s["weights"].gather(-1, src), s["weights_out"][..., :room])
    s["positions_out"][..., :room] = torch.where(live, s["positions"].gather(-1, src), s["positions_out"][..., :room])
    return s["k_out"], s["v_out"], s["weights_out"], s["positions_out"]


def run(s):
    if own:
        return _run_own(s)
    op = s["op"]
    if op == "sink_decode":
        return _plain_sink_decode(s)
    if op == "sink_prefill":
        return _plain_sink_prefill(s)
    if op == "prefix":
        return _plain_prefix(s)
    if op == "accumulate":
        return _plain_accumulate(s)
    return _plain_evict(s)


# ------------------------------------------------------------------ what a pass cannot do without

def _mean(lo, hi):
    return (lo + hi) / 2


def work(case):
    op, hkv, hd = case["op"], case["hkv"], case["hd"]
    row = 2 * hkv * hd * 2                                                      # one token's K and V
    if op == "sink_decode":
        keys = case["n"] * min(_mean(case["lo"], case["hi"]), case["sink"] + case["window"] + case["rows"] - 1)
        io = 2 * case["n"] * case["rows"] * case["hq"] * hd * 2
        return {"bytes": keys * row + io, "flops": 4 * keys * case["rows"] * case["hq"] * hd}
    if op == "sink_prefill":
        at = [min(p + 1, case["window"] + min(case["sink"], max(0, p + 1 - case["window"])))
              for p in range(case["start"], case["start"] + case["tokens"])]
        keys = min(case["start"] + case["tokens"], case["sink"] + case["window"] + case["tokens"] - 1)
        return {"bytes": keys * row + 2 * case["tokens"] * case["hq"] * hd * 2, "flops": 4 * sum(at) * case["hq"] * hd}
    if op == "prefix":
        prefix, tail = case["groups"] * _mean(case["prefix_lo"], case["prefix_hi"]), case["groups"] * case["per"] * _mean(case["lo"], case["hi"])
        io = 2 * case["groups"] * case["per"] * case["rows"] * case["hq"] * hd * 2
        return {"bytes": (prefix + tail) * row + io, "flops": 4 * (prefix * case["per"] + tail) * case["rows"] * case["hq"] * hd}
    if op == "accumulate":
        keys = case["n"] * _mean(case["lo"], case["hi"])
        io = 2 * case["n"] * case["rows"] * case["hq"] * hd * 2
        return {"bytes": keys * (row + 2 * 4 * hkv) + io, "flops": 4 * keys * case["rows"] * case["hq"] * hd}
    rows = case["n"] * _mean(case["lo"], case["hi"])
    kept = case["n"] * min(case["budget"], _mean(case["lo"], case["hi"]))
    # in place, a row kept below `budget` does not move: on average a share 1 - budget / rows of them is filled from above
    moved = kept * (1 - kept / rows) if case["in_place"] else kept
    return {"bytes": rows * hkv * 8 + kept * hkv * 8 + 2 * moved * row, "flops": rows * hkv}


# ------------------------------------------------------------------ the definition, in 64 bits

def _attend(q, k, v):
    """q [hq, hd], k and v [keys, hkv, hd] of the visible keys only, in 64 bits: (output [hq, hd], weights [hq, keys])."""
    hq, hd = q.shape
    hkv = k.shape[1]
    if k.shape[0] == 0:
        return torch.zeros_like(q), q.new_zeros(hq, 0)
    group = hq // hkv
    kh, vh = k.repeat_interleave(group, 1).transpose(0, 1), v.repeat_interleave(group, 1).transpose(0, 1)
    p = torch.softmax((kh @ q[:, :, None]).squeeze(-1) * hd ** -0.5, -1)
    return (p[:, None] @ vh).squeeze(1), p


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "sink_decode":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        for i, length in enumerate(s["lens"]):
            for r in range(case["rows"]):
                end = length - (case["rows"] - 1) + r
                keys = sorted(set(range(min(case["sink"], end))) | set(range(max(0, end - case["window"]), end)))
                rows = [x if x < case["sink"] or not case["ring"] else case["sink"] + (x - case["sink"]) % case["ring"] for x in keys]
                rows = torch.tensor(rows, dtype=torch.long, device="cuda")
                out[i, r] = _attend(s["q"][i, r].double(), s["k"][i, rows].double(), s["v"][i, rows].double())[0]
        return out
    if op == "sink_prefill":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        group = case["hq"] // case["hkv"]
        for t0 in range(0, case["tokens"], 256):
            t1 = min(case["tokens"], t0 + 256)
            low = max(0, case["start"] + t0 + 1 - case["window"])
            keys = list(range(min(case["sink"], low))) + list(range(low, case["start"] + t1))
            rows = [x if x < case["sink"] or not case["ring"] else case["sink"] + (x - case["sink"]) % case["ring"] for x in keys]
            keys, rows = torch.tensor(keys, device="cuda"), torch.tensor(rows, device="cuda")
            at = torch.arange(case["start"] + t0, case["start"] + t1, device="cuda")[:, None]
            hidden = (keys[None] > at) | ((keys[None] <= at - case["window"]) & (keys[None] >= case["sink"]))
            for h in range(case["hq"]):
                k, v = s["k"][rows, h // group].double(), s["v"][rows, h // group].double()
                x = (s["q"][t0:t1, h].double() @ k.T * case["hd"] ** -0.5).masked_fill(hidden, -math.inf)
                out[t0:t1, h] = torch.softmax(x, -1) @ v
        return out
    if op == "prefix":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        for i, length in enumerate(s["lens"]):
            g = i // case["per"]
            pk, pv = s["pk"][g, :s["prefix_lens"][g]].double(), s["pv"][g, :s["prefix_lens"][g]].double()
            for r in range(case["rows"]):
                end = max(0, length - (case["rows"] - 1) + r)
                k, v = torch.cat([pk, s["k"][i, :end].double()]), torch.cat([pv, s["v"][i, :end].double()])
                out[i, r] = _attend(s["q"][i, r].double(), k, v)[0]
        return out
    if op == "accumulate":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        weights, positions = s["weights"].double(), s["positions"].clone()
        group = case["hq"] // case["hkv"]
        for i, length in enumerate(s["lens"]):
            begin = max(0, length - case["rows"])
            weights[i, :, begin:length] = 0.0
            positions[i, :, begin:length] = torch.arange(s["ends"][i] - (length - begin), s["ends"][i], device="cuda", dtype=torch.int32)
            for r in range(case["rows"]):
                end = max(0, length - (case["rows"] - 1) + r)
                out[i, r], p = _attend(s["q"][i, r].double(), s["k"][i, :end].double(), s["v"][i, :end].double())
                weights[i, :, :end] += p.reshape(case["hkv"], group, end).sum(1)
        return out, weights, positions
    k_out, v_out = s["k_out"].double(), s["v_out"].double()
    weights_out, positions_out = s["weights_out"].double(), s["positions_out"].clone()
    for i, length in enumerate(s["lens"]):
        for h in range(case["hkv"]):
            w, p = s["weights"][i, h, :length].tolist(), s["positions"][i, h, :length].tolist()
            safe = [x < case["sink"] or x >= s["ends"][i] - case["recent"] for x in p]
            best = sorted(range(length), key=lambda j: (not safe[j], -w[j] if not safe[j] else 0.0, j))[:case["budget"]]
            kept = set(best)
            fills = iter(sorted(j for j in kept if j >= case["budget"]))
            src = torch.tensor([j if j in kept else next(fills) for j in range(len(best))], dtype=torch.long, device="cuda")
            k_out[i, :len(best), h], v_out[i, :len(best), h] = s["k"][i, src, h].double(), s["v"][i, src, h].double()
            weights_out[i, h, :len(best)], positions_out[i, h, :len(best)] = s["weights"][i, h, src].double(), s["positions"][i, h, src]
    return k_out, v_out, weights_out, positions_out
