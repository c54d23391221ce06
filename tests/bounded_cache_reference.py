"""Plain 64-bit references of the bounded- and shared-cache operators, and the error their 16-bit arithmetic may have."""
import torch


def attend(q, k, v):
    """q [hq, hd]; k, v [keys, hkv, hd] of the visible keys: output [hq, hd], weights [hq, keys], error bound [hq, hd].

    The kernels round each weight p to the 16-bit type (relative error d = eps / 2, and for fp16 2^-25 absolute below its
    normal range, relative to the row's largest weight, 1) and divide by the sum of the rounded weights, so that
    |o' - o| <= sum_i |p'_i - p_i| |v_i - o| / sum p', and round the output (d |o|). 32-bit arithmetic in between: scores
    of size <= 64 before a scale of 1/16, sums of 16 products rounded 16 times at 2^-23, exponentials and sums: under
    2e-5 of the same sum."""
    hq, hd = q.shape
    dtype, q, k, v = q.dtype, q.double(), k.double(), v.double()
    if k.shape[0] == 0:
        zero = torch.zeros(hq, hd, dtype=torch.float64)
        return zero, torch.zeros(hq, 0, dtype=torch.float64), zero
    g = hq // k.shape[1]
    kh, vh = k.repeat_interleave(g, 1).transpose(0, 1), v.repeat_interleave(g, 1).transpose(0, 1)      # [hq, keys, hd]
    s = torch.einsum("hkd,hd->hk", kh, q) * hd ** -0.5
    p = torch.softmax(s, -1)
    o = torch.einsum("hk,hkd->hd", p, vh)
    dev = (vh - o[:, None]).abs()
    half = torch.finfo(dtype).eps / 2
    spread = torch.einsum("hk,hkd->hd", p, dev)
    tiny = 2.0 ** -25 * dev.sum(1) * p.amax(-1, keepdim=True) if dtype == torch.float16 else 0.0
    bound = half * o.abs() + 1.01 * half * spread + tiny + 2e-5 * (spread + o.abs()) + (2.0 ** -25 if dtype == torch.float16 else 0.0)
    return o, p, bound


def sink_keys(end, sink, window):
    """The keys below `end` a row with a window and sinks sees."""
    lo = max(0, end - window) if window else 0
    return sorted(set(range(min(sink, end))) | set(range(lo, end)))


def ring_row(key, sink, ring):
    return key if key < sink or not ring else sink + (key - sink) % ring


def evict(weights, positions, rows, budget, sink, recent, end):
    """One head: source row of every kept row after the eviction, as the definition says it."""
    if rows <= budget:
        return list(range(rows))
    import math
    safe = [p < sink or p >= end - recent for p in positions[:rows]]

    def rank(j):
        w = weights[j]
        return (not safe[j], 0.0 if safe[j] else (math.inf if math.isnan(w) else -w), 0 if safe[j] else int(math.isnan(w)), j)
    kept = set(sorted(range(rows), key=rank)[:budget])
    fills = iter(sorted(j for j in kept if j >= budget))
    return [j if j in kept else next(fills) for j in range(budget)]
