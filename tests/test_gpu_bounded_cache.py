"""Attention over a bounded or shared KV cache (sinks + window, shared prefix, accumulated weights, eviction) on the GPU,
against plain 64-bit references."""
import numpy as np
import pytest
import torch

import tinytitan_b200 as tt
from bounded_cache_reference import attend, evict, ring_row, sink_keys
from gpu_util import context

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16
NAN = float("nan")


def normal(seed, *shape, dtype=F16):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def check(got, want, bound):
    got = got.double().cpu()
    assert torch.isfinite(got).all()
    worst = ((got - want).abs() - bound).max().item()
    assert worst <= 0, f"off by {worst} more than the bound"


def done():
    torch.cuda.synchronize()
    assert context().poll_status() == 0


# ------------------------------------------------------------------ sinks and a window, decode

def run_sink_decode(hd, hq, hkv, dtype, rows, lens, sink, window, ring, pad=0, seed=0, attention=None):
    """Every cache row that no query row may see holds NaN; rows are `pad` elements apart. Returns nothing: checks."""
    n = len(lens)
    cap = sink + ring if ring else max(lens) + 3
    q = normal(seed, n, rows, hq, hd, dtype=dtype)
    k = torch.full((n, cap, hkv * hd + pad), NAN, dtype=dtype)
    v = torch.full((n, cap, hkv * hd + pad), NAN, dtype=dtype)
    keys = [normal(seed + 10 + i, 2, max(1, lens[i]), hkv, hd, dtype=dtype) for i in range(n)]
    for i, length in enumerate(lens):
        seen = set()
        for r in range(rows):
            seen |= set(sink_keys(length - (rows - 1 - r), sink, window))
        for j in sorted(seen):
            at = ring_row(j, sink, ring)
            k[i, at, :hkv * hd], v[i, at, :hkv * hd] = keys[i][0, j].flatten(), keys[i][1, j].flatten()
    qd, kd, vd = q.cuda(), k.cuda(), v.cuda()
    out = torch.full((n, rows, hq * hd + pad), NAN, dtype=dtype, device="cuda")
    sessions = [tt.DecodeSession(qd[i], out[i], kd[i], vd[i], lens[i], rows) for i in range(n)]
    a = attention or tt.Attention(context())
    a.encode_sink_window(sessions, hd, hq, hkv, sink, window, ring_capacity=ring, kv_token_stride_elements=hkv * hd + pad,
                         out_row_stride_elements=hq * hd + pad)
    done()
    assert torch.isnan(out[..., hq * hd:].float()).all() or pad == 0
    for i, length in enumerate(lens):
        for r in range(rows):
            vis = torch.tensor(sink_keys(length - (rows - 1 - r), sink, window), dtype=torch.long)
            want, _, bound = attend(q[i, r], keys[i][0, vis], keys[i][1, vis])
            check(out[i, r, :hq * hd].reshape(hq, hd), want, bound)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd,hq,hkv", [(64, 8, 8), (128, 8, 1), (256, 8, 2), (256, 16, 2), (256, 24, 2), (128, 16, 4), (64, 9, 3)])
def test_sink_decode_shapes(hd, hq, hkv, dtype):
    run_sink_decode(hd, hq, hkv, dtype, 1, [1, 5, 300, 77], 4, 65, 0, seed=hd + hq)


@pytest.mark.parametrize("sink", [0, 1, 4, 100])
@pytest.mark.parametrize("window", [0, 1, 16, 130])
def test_sink_decode_lengths(sink, window):
    # lengths 0 and 1, shorter than the sinks, one below, at and above sink + window, several splits
    lens = sorted({0, 1, 3, 4, 5, sink, sink + window, max(1, sink + window) - 1, sink + window + 1, 517})
    run_sink_decode(256, 8, 2, F16, 1, lens, sink, window, 0, seed=window)


@pytest.mark.parametrize("rows", [2, 3, 8])
@pytest.mark.parametrize("sink,window,ring", [(4, 33, 0), (0, 16, 0), (4, 33, 40), (1, 100, 107), (20, 5, 64)])
def test_sink_decode_few_tokens(rows, sink, window, ring):
    lens = [rows - 1, rows, sink + rows, window + sink + rows - 1, 400]
    run_sink_decode(256, 16, 2, F16, rows, lens, sink, window, ring, seed=rows)
    run_sink_decode(128, 8, 8, BF16, rows, lens, sink, window, ring, seed=rows)


@pytest.mark.parametrize("pad", [8, 24])
def test_sink_decode_ring_of_an_endless_session(pad):
    # positions far beyond the ring, a ring that is exactly the window and one that is not a multiple of anything
    run_sink_decode(256, 8, 2, F16, 1, [1000, 1001, 1063, 64, 67, 70], 4, 63, 63, pad=pad)
    run_sink_decode(256, 8, 2, BF16, 1, [999, 1999], 3, 50, 71, pad=pad)


def test_sink_decode_many_sessions_uses_the_uploaded_tables():
    r = np.random.default_rng(5)
    lens = [int(x) for x in r.integers(0, 200, size=90)]
    run_sink_decode(64, 4, 2, F16, 1, lens, 2, 40, 0)
    run_sink_decode(128, 4, 2, BF16, 2, [max(1, x) for x in lens], 2, 40, 45)


def test_sink_decode_window_covering_everything_is_plain_decode():
    # too many keys for clusters of parts: the same keys in the same order through the same arithmetic, bit for bit
    n, hq, hkv, hd = 3, 16, 2, 256
    q, k, v = (normal(i, *s).cuda() for i, s in enumerate([(n, 1, hq, hd), (n, 1700, hkv, hd), (n, 1700, hkv, hd)]))
    a = tt.Attention(context())
    outs = [torch.empty_like(q) for _ in range(2)]
    t = [tt.SessionTable.over_cache(q, o, k, v, [1700, 256, 3]) for o in outs]
    a.encode_sink_window(t[0], hd, hq, hkv, 0, 1700)
    a.encode_batched([tt.DecodeSession(q[i], outs[1][i], k[i], v[i], s) for i, s in enumerate([1700, 256, 3])], hd, hq, hkv)
    done()
    assert torch.equal(outs[0], outs[1])


@pytest.mark.parametrize("longest", [1, 16, 17, 33, 65, 129, 257, 1000, 1024])       # clusters of 1 .. 16 CTAs, down to parts without keys
@pytest.mark.parametrize("hd,hq,hkv,rows", [(64, 8, 2, 1), (128, 5, 5, 1), (256, 8, 2, 1), (256, 16, 2, 3), (128, 24, 3, 2), (64, 40, 1, 1)])
def test_sink_decode_clusters(hd, hq, hkv, rows, longest):
    least = rows - 1
    lens = [max(least, x) for x in (longest, least, longest // 3, min(longest, 20))]
    run_sink_decode(hd, hq, hkv, F16 if longest % 2 else BF16, rows, lens, 2, max(1, longest - 2), 0)
    run_sink_decode(hd, hq, hkv, BF16, rows, [x * 5 for x in lens], 3, max(1, longest - 3), longest + 40)


@pytest.mark.parametrize("hd,hq,hkv,n,rows,longest", [(64, 8, 8, 64, 1, 300), (256, 8, 2, 64, 1, 270), (128, 4, 1, 64, 1, 1100), (64, 16, 2, 64, 4, 300)])
def test_sink_decode_clusters_that_fill_the_machine(hd, hq, hkv, n, rows, longest):
    run_sink_decode(hd, hq, hkv, F16, rows, [longest + i % 7 for i in range(n)], 1, longest + 3, 0)


@pytest.mark.parametrize("hd,hq,hkv,rows", [(64, 40, 2, 1), (128, 16, 2, 4), (256, 16, 2, 3), (256, 32, 2, 9), (128, 9, 3, 64), (256, 24, 1, 6)])
@pytest.mark.parametrize("sink,window", [(0, 130), (4, 700), (70, 64), (200, 1), (3, 0)])
def test_sink_decode_draft_rows(hd, hq, hkv, rows, sink, window):
    # items of 64, 128 and 256 packed rows and several of them, halves of sinks and window, rows without keys
    lens = [max(rows - 1, x) for x in (900, 0, 131, 64, sink, sink + window, sink + window + 1, 1500)]
    run_sink_decode(hd, hq, hkv, F16, rows, lens, sink, window, 0, pad=8)
    if window:
        run_sink_decode(hd, hq, hkv, BF16, rows, lens[1:5], sink, window, 1000)          # a ring that has not wrapped
        run_sink_decode(hd, hq, hkv, BF16, rows, lens, sink, window, window + rows + 60)    # ... and one that has


@pytest.mark.parametrize("sessions", [40, 41, 90])
def test_sink_decode_draft_rows_of_many_sessions(sessions):
    lens = [5 + (41 * i) % 300 for i in range(sessions)]
    run_sink_decode(256, 16, 2, F16, 3, lens, 4, 100, 0)
    run_sink_decode(64, 20, 1, BF16, 2, lens, 0, 64, 0)


def test_sink_decode_refusals():
    n, hq, hkv, hd = 1, 8, 2, 256
    q, k, v = (torch.zeros(*s, dtype=F16, device="cuda") for s in [(n, 2, hq, hd), (n, 64, hkv, hd), (n, 64, hkv, hd)])
    out = torch.empty_like(q)
    a = tt.Attention(context())

    def call(sessions=None, sink=4, window=16, ring=0, **kw):
        a.encode_sink_window(sessions or [tt.DecodeSession(q, out, k, v, 40, 2)], hd, hq, hkv, sink, window, ring_capacity=ring, **kw)
    call()
    for bad in (dict(ring=16), dict(window=0, ring=32), dict(sink=2 ** 31), dict(sessions=[tt.DecodeSession(q, out, k, v, 40, 2, kv_start=1)]),
                dict(sessions=[tt.DecodeSession(q, out, k, v, 0, 2)]), dict(sessions=[tt.DecodeSession(q, out, k, v, 40, 0)]),
                dict(sessions=[tt.DecodeSession(q, out, k, v, 2 ** 31, 1)]), dict(kv_token_stride_elements=256)):
        with pytest.raises(tt.InvalidArgument):
            call(**bad)
    for bad in (dict(kv_token_stride_elements=516), dict(sessions=[tt.DecodeSession(q, out, k, v, 40, 1, k_offset=2)])):
        with pytest.raises(tt.UnsupportedShape):
            call(**bad)
    call(sessions=[tt.DecodeSession(q, out, k, v, 20, 2)], ring=16)      # nothing has wrapped yet: any ring will do
    done()


# ------------------------------------------------------------------ sinks and a window, prefill

def run_sink_prefill(tokens, start, sink, window, ring, dtype=F16, hd=256, hq=4, hkv=2, pad=0, path="tcgen05", extra=0):
    valid = start + tokens + extra
    cap = sink + ring if ring else valid
    keys = normal(7, 2, valid, hkv, hd, dtype=dtype)
    k = torch.full((cap + 2, hkv * hd + pad), 0.0 if ring else NAN, dtype=dtype)
    v = torch.full((cap + 2, hkv * hd + pad), 0.0 if ring else NAN, dtype=dtype)
    k[cap:], v[cap:] = NAN, NAN                               # rows behind the last one
    lo = max(0, start + 1 - window) if window else 0
    for j in list(range(min(sink, valid))) + list(range(max(lo, sink), valid)):       # what was evicted is NaN (0 in a ring)
        at = ring_row(j, sink, ring)
        k[at, :hkv * hd], v[at, :hkv * hd] = keys[0, j].flatten(), keys[1, j].flatten()
    q = normal(8, tokens, hq * hd + pad, dtype=dtype)
    out = torch.full((tokens + 1, hq * hd + pad), NAN, dtype=dtype, device="cuda")
    qd, kd, vd = q.cuda(), k.cuda(), v.cuda()
    p = tt.PrefillAttentionParams(start, tokens, hd, hq, hkv, valid, window, hkv * hd + pad, hq * hd + pad, hq * hd + pad, hd ** -0.5)
    prefill = tt.PrefillAttention(context())
    assert prefill.sink_window_path(qd, kd, vd, out, p, ring) == path
    prefill.encode_sink_window(qd, kd, vd, out, p, sink, kv_ring_capacity=ring)
    done()
    assert torch.isnan(out[tokens:].float()).all() and (pad == 0 or torch.isnan(out[:, hq * hd:].float()).all())
    rows = range(tokens) if tokens <= 40 else sorted({0, 1, 7, 8, 31, 32, 33, 63, 64, 127, 128, 129, tokens // 2, tokens - 2, tokens - 1} & set(range(tokens)))
    for t in rows:
        vis = torch.tensor(sink_keys(start + t + 1, sink, window), dtype=torch.long)
        want, _, bound = attend(q[t, :hq * hd].reshape(hq, hd), keys[0, vis], keys[1, vis])
        check(out[t, :hq * hd].reshape(hq, hd), want, bound)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("tokens,start,sink,window", [
    (1, 0, 4, 8), (1, 1000, 4, 64), (33, 0, 4, 8), (129, 5, 0, 1), (300, 0, 4, 64), (300, 700, 4, 64), (257, 1000, 130, 100),
    (200, 400, 1, 300), (128, 128, 128, 128), (200, 0, 500, 16), (64, 100, 16, 0), (300, 900, 200, 129)])
def test_sink_prefill(tokens, start, sink, window, dtype):
    run_sink_prefill(tokens, start, sink, window, 0, dtype)


@pytest.mark.parametrize("tokens,start,sink,window,ring", [
    (1, 1000, 4, 64, 64), (100, 0, 4, 64, 192), (100, 60, 4, 64, 192), (100, 700, 4, 64, 192), (300, 1000, 4, 200, 512),
    (129, 5000, 0, 128, 256), (65, 777, 200, 64, 128), (300, 100, 7, 600, 960)])
def test_sink_prefill_ring(tokens, start, sink, window, ring):
    run_sink_prefill(tokens, start, sink, window, ring)
    run_sink_prefill(tokens, start, sink, window, ring, BF16, pad=8)


@pytest.mark.parametrize("hq,hkv", [(2, 2), (6, 2), (8, 2), (16, 2), (12, 1), (16, 1), (24, 1), (32, 1), (64, 1)])     # 1 .. 32 heads of an item's rows
@pytest.mark.parametrize("tokens,start,sink,window,ring", [(70, 300, 20, 100, 0), (100, 0, 70, 30, 0), (70, 300, 130, 64, 256)])
def test_sink_prefill_head_groups(tokens, start, sink, window, ring, hq, hkv):
    run_sink_prefill(tokens, start, sink, window, ring, hq=hq, hkv=hkv)


@pytest.mark.parametrize("tokens,start,sink,window,ring,hd,pad", [
    (20, 0, 4, 8, 0, 64, 0), (20, 50, 4, 8, 0, 128, 3), (9, 30, 0, 1, 0, 256, 1), (20, 50, 4, 8, 27, 256, 0), (17, 300, 3, 20, 37, 32, 0)])
def test_sink_prefill_generic_kernel(tokens, start, sink, window, ring, hd, pad):
    run_sink_prefill(tokens, start, sink, window, ring, hd=hd, pad=pad, path="generic")


def test_sink_prefill_rows_behind_the_chunk():
    # rows of tokens that are already in the cache but later than the chunk stay invisible
    run_sink_prefill(50, 100, 4, 40, 0, extra=30)
    run_sink_prefill(50, 100, 4, 40, 128, extra=30)


def test_sink_prefill_refusals():
    x = torch.zeros(300, 512, dtype=F16, device="cuda")
    prefill = tt.PrefillAttention(context())

    def call(ring=0, window=64, start=0, tokens=100, valid=100, sink=4, **kw):
        p = tt.PrefillAttentionParams(start, tokens, 256, 2, 2, valid, window, 512, 512, 512, 0.0625, **kw)
        prefill.encode_sink_window(x, x, x, torch.empty_like(x), p, sink, kv_ring_capacity=ring)
    call()
    call(ring=100)                          # not wrapped
    for bad in (dict(ring=64), dict(start=100, valid=200, ring=128), dict(start=100, valid=200, ring=192, window=0), dict(valid=99), dict(sink=2 ** 31)):
        with pytest.raises(tt.InvalidArgument):
            call(**bad)
    with pytest.raises(tt.UnsupportedShape):
        call(kv_bits=8, kv_token_stride_bytes=544, kv_value_bytes=512)
    done()


# ------------------------------------------------------------------ shared prefixes

def run_prefix(hd, hq, hkv, dtype, prefix_lens, per, rows, lens, pad=0, seed=0, ctx=None):
    """per[g] sessions with rows[i] query rows each; rows behind a prefix's or a session's last one hold NaN."""
    width, n, g = hkv * hd + pad, len(lens), len(prefix_lens)
    pk, pv = normal(seed, g, max(prefix_lens) + 2, hkv * hd, dtype=dtype), normal(seed + 1, g, max(prefix_lens) + 2, hkv * hd, dtype=dtype)
    k, v = normal(seed + 2, n, max(lens) + 2, hkv * hd, dtype=dtype), normal(seed + 3, n, max(lens) + 2, hkv * hd, dtype=dtype)
    q = normal(seed + 4, n, max(rows), hq * hd, dtype=dtype)

    def spread(x, used):
        wide = torch.full(x.shape[:2] + (width,), NAN, dtype=dtype)
        for i, m in enumerate(used):
            wide[i, :m, :hkv * hd] = x[i, :m]
        return wide.cuda()
    pkd, pvd, kd, vd, qd = spread(pk, prefix_lens), spread(pv, prefix_lens), spread(k, lens), spread(v, lens), q.cuda()
    out = torch.full((n, max(rows), hq * hd + pad), NAN, dtype=dtype, device="cuda")
    ctx = ctx or context()
    groups = [tt.PrefixGroup(pkd[i], pvd[i], prefix_lens[i], per[i]) for i in range(g)]
    sessions = [tt.DecodeSession(qd[i], out[i], kd[i], vd[i], lens[i], rows[i]) for i in range(n)]
    tt.Attention(ctx).encode_shared_prefix(groups, sessions, hd, hq, hkv, kv_token_stride_elements=width,
                                           out_row_stride_elements=hq * hd + pad)
    torch.cuda.synchronize()
    assert ctx.poll_status() == 0
    owner = [x for x, m in enumerate(per) for _ in range(m)]
    for i in range(n):
        p = prefix_lens[owner[i]]
        assert torch.isnan(out[i, rows[i]:].float()).all()                  # rows the session does not have
        for r in range(rows[i]):
            end = lens[i] - (rows[i] - 1 - r)
            kk = torch.cat([pk[owner[i], :p], k[i, :end]]).reshape(-1, hkv, hd)
            vv = torch.cat([pv[owner[i], :p], v[i, :end]]).reshape(-1, hkv, hd)
            want, _, bound = attend(q[i, r].reshape(hq, hd), kk, vv)
            check(out[i, r, :hq * hd].reshape(hq, hd), want, bound)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd,hq,hkv", [(64, 8, 8), (128, 8, 1), (256, 8, 2), (256, 16, 2), (128, 32, 2), (64, 9, 3), (256, 3, 3)])
def test_prefix_shapes(hd, hq, hkv, dtype):
    run_prefix(hd, hq, hkv, dtype, [300], [3], [1] * 3, [1, 40, 17], seed=hd + hq)


@pytest.mark.parametrize("prefix", [1, 2, 127, 128, 129, 1000])
@pytest.mark.parametrize("hd", [64, 256])
def test_prefix_lengths(prefix, hd):
    run_prefix(hd, 8, 2, F16, [prefix], [2], [1, 1], [0, 3], pad=8)


@pytest.mark.parametrize("sessions", [1, 8, 9, 16, 17, 33])
def test_prefix_row_tiles(sessions):
    # 8 packed rows a session: below, at and above 64 and 128 rows, several row tiles
    run_prefix(256, 16, 2, F16, [400], [sessions], [1] * sessions, [(7 * i) % 50 for i in range(sessions)])


def test_prefix_groups_and_ragged_rows():
    rows = [1, 4, 2, 1, 3, 1, 8]
    lens = [0, 3, 1, 5, 300, 64, 20]
    run_prefix(256, 16, 2, BF16, [0, 513, 7], [2, 4, 1], rows, lens)
    run_prefix(128, 8, 8, F16, [100, 0, 257], [1, 2, 4], rows, lens, pad=16)
    run_prefix(64, 32, 2, F16, [3, 129, 2], [3, 3, 1], rows, lens)


@pytest.mark.parametrize("sessions", [1, 5, 16, 17, 20])                # their own rows as items of the prefix pass
@pytest.mark.parametrize("hd,hq,hkv", [(64, 8, 2), (128, 4, 1), (256, 8, 2)])
def test_prefix_long_suffixes(hd, hq, hkv, sessions):
    # query rows whose last keys lie on both sides of a tile's edge, a last part that only the last rows see, rows without keys
    rows = ([4, 64, 9, 1, 33] * 4)[:sessions]
    lens = ([129, 63, 515, 1000, 256, 130, 127, 8, 0, 161, 385, 700, 10, 128, 32, 3, 65, 12, 260, 40])[:sessions]
    run_prefix(hd, hq, hkv, BF16, [5], [sessions], rows, lens, pad=8)
    run_prefix(hd, hq, hkv, F16, [0] * (sessions > 1) + [130], [1] * (sessions > 1) + [sessions - (sessions > 1)], rows, lens)


@pytest.mark.parametrize("hd,hq,hkv,rows,sessions", [
    (256, 16, 2, 1, 17), (256, 16, 2, 1, 64), (256, 16, 2, 3, 40),           # a pass of their own; a pair's items
    (128, 16, 2, 1, 32), (128, 16, 2, 1, 33), (64, 8, 8, 1, 32), (128, 16, 1, 2, 64), (64, 18, 2, 2, 50)])
def test_prefix_many_sessions(hd, hq, hkv, rows, sessions):
    lens = [rows - 1 + (37 * i) % 290 for i in range(sessions)]
    run_prefix(hd, hq, hkv, F16, [260, 0, 131], [sessions - 3, 1, 2], [rows] * sessions, lens, pad=8)
    run_prefix(hd, hq, hkv, BF16, [140], [sessions], [1 + i % rows for i in range(sessions)], lens)


def test_prefix_large_tables():
    n = 70
    run_prefix(128, 4, 2, F16, [200], [n], [1] * n, [i % 9 for i in range(n)])
    run_prefix(64, 4, 2, BF16, [10 * i for i in range(10)], [3] * 10, [1 + i % 2 for i in range(30)], [1 + i % 9 for i in range(30)])


def test_prefix_peaked_rows_and_late_maxima():
    # the largest score of a row comes late and is far above the others: the running maximum is raised and O rescaled
    hd, hq, hkv, n, p = 256, 8, 2, 3, 600
    pk, pv = normal(1, 1, p, hkv, hd), normal(2, 1, p, hkv, hd)
    k, v = normal(3, n, 4, hkv, hd), normal(4, n, 4, hkv, hd)
    q = normal(5, n, 1, hq, hd)
    for j, f in ((100, 1.0), (300, 2.0), (599, 3.0)):
        pk[0, j] = (q[0, 0].reshape(hkv, -1, hd)[:, 0].float() * f).half()
    out = torch.empty_like(q).cuda()
    d = [x.cuda() for x in (pk, pv, k, v, q)]
    tt.Attention(context()).encode_shared_prefix(tt.PrefixTable.over_cache(d[0], d[1], p, n),
                                                 tt.SessionTable.over_cache(d[4], out, d[2], d[3], 4), hd, hq, hkv)
    done()
    for i in range(n):
        want, _, bound = attend(q[i, 0], torch.cat([pk[0], k[i]]), torch.cat([pv[0], v[i]]))
        check(out[i, 0], want, bound)


def test_prefix_refusals():
    hd, hq, hkv, n = 256, 8, 2, 3
    q = torch.zeros(n, 1, hq, hd, dtype=F16, device="cuda")
    k = torch.zeros(n, 16, hkv, hd, dtype=F16, device="cuda")
    out, a = torch.empty_like(q), tt.Attention(context())
    ok = [tt.DecodeSession(q[i], out[i], k[i], k[i], 5) for i in range(n)]

    def call(groups=None, sessions=ok, **kw):
        a.encode_shared_prefix(groups or [tt.PrefixGroup(k, k, 16, n)], sessions, hd, hq, hkv, **kw)
    call()
    for bad in (dict(groups=[tt.PrefixGroup(k, k, 16, 2)]), dict(groups=[tt.PrefixGroup(k, k, 16, 3), tt.PrefixGroup(k, k, 16, 0)]),
                dict(groups=[tt.PrefixGroup(0, k, 16, 3)]), dict(groups=[tt.PrefixGroup(k, k, 2 ** 31, 3)]),
                dict(sessions=ok[:2] + [tt.DecodeSession(q[2], out[2], k[2], k[2], 5, kv_start=1)]),
                dict(sessions=ok[:2] + [tt.DecodeSession(q[2], out[2], k[2], k[2], 5, q_rows=65)]),
                dict(sessions=ok[:2] + [tt.DecodeSession(q[2], out[2], k[2], k[2], 0, q_rows=2)]), dict(kv_token_stride_elements=256)):
        with pytest.raises(tt.InvalidArgument):
            call(**bad)
    for bad in (dict(groups=[tt.PrefixGroup(k, k, 16, 3, k_offset=2)]), dict(scale=-1.0)):
        with pytest.raises(tt.UnsupportedShape):
            call(**bad)
    small = tt.Context(0, workspace_bytes=1 << 14)
    with pytest.raises(tt.TinyTitanError):
        tt.Attention(small).encode_shared_prefix([tt.PrefixGroup(k, k, 16, n)], ok, hd, hq, hkv)
    small.close()
    done()


# ------------------------------------------------------------------ accumulated weights

def run_accumulate(hd, hq, hkv, dtype, rows, lens, fresh, cap=None, seed=0, ctx=None):
    n, cap = len(lens), cap or max(lens) + 5
    q = normal(seed, n, max(rows), hq, hd, dtype=dtype)
    k, v = normal(seed + 1, n, cap, hkv, hd, dtype=dtype), normal(seed + 2, n, cap, hkv, hd, dtype=dtype)
    for i, m in enumerate(lens):
        k[i, m:], v[i, m:] = NAN, NAN
    start = torch.rand(n, hkv, cap, generator=torch.Generator().manual_seed(seed + 3))
    for i, m in enumerate(lens):
        start[i, :, m - fresh[i]:m] = NAN                    # whatever stood in a fresh row is gone
    weights, positions = start.cuda(), torch.full((n, hkv, cap), -7, dtype=torch.int32, device="cuda")
    d = [x.cuda() for x in (q, k, v)]
    out = torch.full((n, max(rows), hq, hd), NAN, dtype=dtype, device="cuda")
    sessions = [tt.DecodeSession(d[0][i], out[i], d[1][i], d[2][i], lens[i], rows[i]) for i in range(n)]
    ctx = ctx or context()
    tt.Attention(ctx).encode_accumulate(sessions, weights, hd, hq, hkv, positions=positions, fresh_rows=fresh,
                                        end_positions=[m + 100 for m in lens])
    torch.cuda.synchronize()
    assert ctx.poll_status() == 0
    got = weights.cpu()
    for i, m in enumerate(lens):
        want = start[i].double().clone()
        want[:, m - fresh[i]:m] = 0.0
        added = torch.zeros_like(want)
        for r in range(rows[i]):
            end = m - (rows[i] - 1 - r)
            o, p, bound = attend(q[i, r], k[i, :end], v[i, :end])
            check(out[i, r], o, bound)
            added[:, :end] += p.reshape(hkv, hq // hkv, end).sum(1)
        want += added
        # 32-bit scores, exponentials and normaliser: 2e-5 of what was added (see attend); sums of up to 1 + rows * group
        # terms rounded at 2^-24 of their size each
        bound = 2e-5 * added + (1 + rows[i] * hq // hkv) * 2.0 ** -24 * want
        assert ((got[i, :, :m].double() - want[:, :m]).abs() <= bound[:, :m]).all(), ((got[i, :, :m] - want[:, :m]).abs() - bound[:, :m]).max()
        assert torch.equal(got[i, :, m:], start[i, :, m:])                                  # behind the session: untouched
        pos = positions[i].cpu()
        assert (pos[:, :m - fresh[i]] == -7).all() and (pos[:, m:] == -7).all()
        assert (pos[:, m - fresh[i]:m] == torch.arange(m + 100 - fresh[i], m + 100, dtype=torch.int32)).all()
    return out, weights


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd,hq,hkv", [(64, 8, 8), (128, 8, 1), (256, 8, 2), (256, 16, 2), (256, 24, 2), (128, 16, 4), (64, 9, 3)])
def test_accumulate_shapes(hd, hq, hkv, dtype):
    lens = [1, 2, 16, 300, 1025]
    run_accumulate(hd, hq, hkv, dtype, [1] * 5, lens, [1, 0, 5, 300, 1], seed=hd + hq)


@pytest.mark.parametrize("rows", [[2, 3, 4], [1, 8, 5], [16, 1, 64]])
def test_accumulate_few_tokens_and_prompt_tails(rows):
    lens = [max(70, r) for r in rows]
    lens[1] = rows[1]                       # a prompt of nothing but its queries
    run_accumulate(256, 8, 2, F16, rows, lens, rows, seed=3)
    run_accumulate(128, 32, 2, BF16, rows, lens, [0, rows[1], 10], seed=4)


def test_accumulate_lengths_zero_and_no_rows_visible():
    run_accumulate(256, 8, 2, F16, [1, 2, 3], [0, 1, 2], [0, 1, 2], cap=8)


def test_accumulate_many_sessions():
    lens = [1 + (37 * i) % 90 for i in range(130)]
    run_accumulate(64, 4, 2, F16, [1] * 130, lens, [1] * 130)


def test_accumulate_in_a_small_workspace():
    # the batch, then single sessions, then the rows of one session are taken in several passes
    ctx = tt.Context(0, workspace_bytes=3 << 20)
    run_accumulate(256, 16, 2, F16, [1, 1, 2, 9, 40, 1], [900, 50, 2000, 700, 1500, 333], [1, 1, 2, 9, 40, 333], ctx=ctx)
    tiny = tt.Context(0, workspace_bytes=1 << 16)
    q, k = torch.zeros(1, 1, 8, 256, dtype=F16, device="cuda"), torch.zeros(1, 5000, 2, 256, dtype=F16, device="cuda")
    weights = torch.zeros(1, 2, 5000, device="cuda")
    with pytest.raises(tt.TinyTitanError):
        tt.Attention(tiny).encode_accumulate(tt.SessionTable.over_cache(q, torch.empty_like(q), k, k, 5000), weights, 256, 8, 2)
    ctx.close(), tiny.close()


def test_accumulate_is_deterministic_and_its_output_is_that_of_decode():
    n, hq, hkv, hd, s = 4, 16, 2, 256, 3000
    q, k, v = (normal(i, *x).cuda() for i, x in enumerate([(n, 1, hq, hd), (n, s, hkv, hd), (n, s, hkv, hd)]))
    a = tt.Attention(context())
    outs, stats = [torch.empty_like(q) for _ in range(3)], [torch.zeros(n, hkv, s, device="cuda") for _ in range(2)]
    lens = [3000, 2000, 77, 1]
    for o, w in zip(outs, stats):
        a.encode_accumulate(tt.SessionTable.over_cache(q, o, k, v, lens), w, hd, hq, hkv)
    a.encode_batched([tt.DecodeSession(q[i], outs[2][i], k[i], v[i], m) for i, m in enumerate(lens)], hd, hq, hkv)
    done()
    assert torch.equal(stats[0], stats[1]) and torch.equal(outs[0], outs[1])
    # the same partials merged in another order: 32-bit sums of a few dozen terms, then one rounding (half a step each)
    a, b = outs[0].double(), outs[2].double()
    assert ((a - b).abs() <= 2 * 2.0 ** -11 * b.abs() + 1e-6).all()
    # every row of the softmax weighs one: the statistic of a KV head grows by its number of query heads
    total = stats[0].double().sum(-1)
    assert ((total - hq // hkv).abs() <= 2e-5 * hq // hkv + 1e-4).all()


def test_accumulate_refusals():
    hd, hq, hkv = 256, 8, 2
    q, k = torch.zeros(1, 1, hq, hd, dtype=F16, device="cuda"), torch.zeros(1, 40, hkv, hd, dtype=F16, device="cuda")
    out, a = torch.empty_like(q), tt.Attention(context())
    w, pos = torch.zeros(1, hkv, 40, device="cuda"), torch.zeros(1, hkv, 40, dtype=torch.int32, device="cuda")
    t = tt.SessionTable.over_cache(q, out, k, k, 40)
    for bad in (dict(weights=w[:, :1]), dict(weights=w.double()), dict(weights=w[:, :, :39]), dict(weights=w.cpu()), dict(positions=pos.long()),
                dict(positions=pos[:, :, :39]), dict(fresh_rows=41), dict(sessions=[tt.DecodeSession(q, out, k, k, 40, 1, kv_start=2)]),
                dict(sessions=[tt.DecodeSession(q, out, k, k, 40, 65)]), dict(fresh_rows=[1, 2])):
        with pytest.raises(tt.InvalidArgument):
            a.encode_accumulate(bad.pop("sessions", t), bad.pop("weights", w), hd, hq, hkv, **{"positions": pos, **bad})
    with pytest.raises(tt.UnsupportedShape):
        a.encode_accumulate(t, w, hd, hq, hkv, scale=0.0)
    done()
    assert (w == 0).all()


# ------------------------------------------------------------------ eviction

def run_evict(lens, budget, sink, recent, hkv=2, hd=256, dtype=F16, in_place=True, keep_positions=True, seed=0, mix=False, cap=None,
              stats_in_place=False, pad=0):
    n, cap = len(lens), cap or max(lens) + 3
    g = torch.Generator().manual_seed(seed)
    k = torch.randn(n, cap, hkv * hd + pad, generator=g).to(dtype)[:, :, :hkv * hd].unflatten(2, (hkv, hd))
    v = torch.randn(n, cap, hkv * hd + pad, generator=g).to(dtype)[:, :, :hkv * hd].unflatten(2, (hkv, hd))
    w = torch.randn(n, hkv, cap, generator=g).exp()
    w[torch.rand(n, hkv, cap, generator=g) < 0.3] = 0.5                       # ties
    if mix:
        for x in (0.0, -0.0, -1.0, float("inf"), float("-inf"), NAN):
            w[torch.rand(n, hkv, cap, generator=g) < 0.05] = x
    pos = torch.rand(n, hkv, cap, generator=g).argsort(-1).to(torch.int32)
    ends = [cap] * n
    if not keep_positions:
        pos, ends = torch.arange(cap, dtype=torch.int32).expand(n, hkv, cap), list(lens)
    kd = torch.empty(n, cap, hkv * hd + pad, dtype=dtype, device="cuda")[:, :, :hkv * hd].unflatten(2, (hkv, hd)).copy_(k)
    vd = torch.empty(n, cap, hkv * hd + pad, dtype=dtype, device="cuda")[:, :, :hkv * hd].unflatten(2, (hkv, hd)).copy_(v)
    wd, pd = w.cuda(), pos.cuda().contiguous()
    room = min(budget, max(lens)) + 1
    outs = dict(k_out=torch.full((n, room, hkv, hd), 9.0, dtype=dtype, device="cuda"),
                v_out=torch.full((n, room, hkv, hd), 9.0, dtype=dtype, device="cuda"))
    stats = dict(weights_out=torch.full((n, hkv, room), 9.0, device="cuda"),
                 positions_out=torch.full((n, hkv, room), 9, dtype=torch.int32, device="cuda"))
    tt.evict_kv_rows(context(), kd, vd, wd, lens, budget, sink, recent, positions=pd if keep_positions else None, end_positions=ends,
                     **({} if in_place else outs), **({} if stats_in_place else stats))
    done()
    got_k, got_v = (kd, vd) if in_place else (outs["k_out"], outs["v_out"])
    got_w, got_p = (wd, pd) if stats_in_place else (stats["weights_out"], stats["positions_out"])
    got_k, got_v, got_w, got_p = got_k.cpu(), got_v.cpu(), got_w.cpu(), got_p.cpu()
    for i, m in enumerate(lens):
        for h in range(hkv):
            src = torch.tensor(evict(w[i, h].tolist(), pos[i, h].tolist(), m, budget, sink, recent, ends[i]), dtype=torch.long)
            b = len(src)
            assert torch.equal(got_p[i, h, :b], pos[i, h, src]), (i, h)
            assert torch.equal(got_w[i, h, :b].view(torch.int32), w[i, h, src].view(torch.int32))
            assert torch.equal(got_k[i, :b, h], k[i, src, h]) and torch.equal(got_v[i, :b, h], v[i, src, h])
        b = min(m, budget)
        # behind the kept rows nothing is written
        for got, was in ((got_k[i, b:], k[i, b:] if in_place else 9.0), (got_v[i, b:], v[i, b:] if in_place else 9.0)):
            assert (got == was).all()
        if stats_in_place:
            assert torch.equal(got_w[i, :, b:].view(torch.int32), w[i, :, b:].view(torch.int32)) and torch.equal(got_p[i, :, b:], pos[i, :, b:])
        else:
            assert (got_w[i, :, b:] == 9).all() and (got_p[i, :, b:] == 9).all()


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("lens,budget,sink,recent", [
    ([9], 8, 0, 0), ([1, 2, 3, 0], 1, 0, 1), ([100, 37, 64, 5], 37, 4, 9), ([513, 512, 511, 700], 512, 4, 256), ([2049], 2048, 4, 256),
    ([5000, 4097, 4096, 1], 777, 0, 0), ([300], 290, 100, 190), ([1000, 20], 5000, 4, 4)])
def test_evict(lens, budget, sink, recent, in_place):
    run_evict(lens, budget, sink, recent, in_place=in_place)


@pytest.mark.parametrize("hkv,hd,dtype", [(1, 64, F16), (8, 64, BF16), (3, 128, F16), (4, 256, BF16)])
def test_evict_layouts(hkv, hd, dtype):
    run_evict([200, 130, 64], 100, 2, 10, hkv, hd, dtype, in_place=False, pad=8)
    run_evict([200, 130, 64], 100, 2, 10, hkv, hd, dtype, in_place=True, stats_in_place=True, pad=24)


def test_evict_special_weights_and_ties():
    run_evict([700, 650], 200, 3, 50, mix=True, in_place=False)
    run_evict([700, 650], 649, 0, 0, mix=True)
    # nothing but ties: the lower rows stay
    n, hkv, hd, cap = 1, 2, 64, 300
    k = torch.arange(cap, dtype=F16, device="cuda")[None, :, None, None].expand(n, cap, hkv, hd).contiguous()
    w, p = torch.ones(n, hkv, cap, device="cuda"), torch.zeros(n, hkv, cap, dtype=torch.int32, device="cuda")
    tt.evict_kv_rows(context(), k, k.clone(), w, cap, 100, positions_out=p)
    done()
    assert (p[..., :100] == torch.arange(100, device="cuda", dtype=torch.int32)).all() and (k[0, :100, 0, 0] == torch.arange(100, device="cuda")).all()


@pytest.mark.parametrize("close", [1, 2, 5, 255, 256, 257, 600])        # rows whose weights share their leading bits: compared or counted
@pytest.mark.parametrize("values", ["different", "two", "zero"])
def test_evict_threshold_among_close_weights(close, values):
    rows, hkv, hd = 1500, 1, 64
    g = torch.Generator().manual_seed(close)
    apart = torch.cat([torch.linspace(2.0, 900.0, 500), torch.linspace(-3.0, -900.0, rows - 500 - close)])
    near = {"different": 1.0 + 0.2 * torch.rand(close, generator=g), "two": 1.0 + 0.125 * (torch.rand(close, generator=g) < 0.5).float(),
            "zero": torch.zeros(close)}[values]
    w = torch.cat([apart, near])[torch.randperm(rows, generator=g)]
    for kept in sorted({1, (close + 1) // 2, close}):
        budget = 500 + kept                                  # the threshold is the kept-th largest of the close ones
        k = torch.arange(rows, dtype=torch.float32)[None, :, None, None].expand(1, rows, hkv, hd).to(BF16).cuda().contiguous()
        p = torch.zeros(1, hkv, rows, dtype=torch.int32, device="cuda")
        tt.evict_kv_rows(context(), k, k.clone(), w[None, None].cuda(), rows, budget, positions_out=p)
        done()
        assert p[0, 0, :budget].tolist() == evict(w.tolist(), list(range(rows)), rows, budget, 0, 0, rows)


def test_evict_positions_default_to_the_rows():
    run_evict([400, 90], 80, 4, 20, keep_positions=False, in_place=False)
    run_evict([400, 90], 80, 4, 20, keep_positions=False)


def test_evict_clusters_and_long_caches():
    run_evict([40000, 30000], 5000, 4, 1000, hkv=1, hd=64, in_place=False)                    # several CTAs a head
    run_evict([450001], 300000, 4, 1000, hkv=1, hd=64, in_place=False)                        # more keys than a cluster holds
    run_evict([450001, 1000], 700, 4, 10, hkv=1, hd=64, in_place=False, keep_positions=False)
    run_evict([100 + 7 * i for i in range(70)], 150, 1, 9, hkv=2, hd=64)                      # more sessions than one launch takes


@pytest.mark.parametrize("sessions", [1, 16, 32, 40])                   # clusters of 8, 4, 2 and 1 beyond 10000 rows
def test_evict_around_one_cta(sessions):
    lens = [10000 + 7 * i for i in range(sessions)]
    run_evict(lens, 9990, 4, 100, hkv=1, hd=64)
    run_evict(lens, 300, 0, 0, hkv=1, hd=64, in_place=False, mix=True)


@pytest.mark.parametrize("sessions,given_up", [(15, 256), (15, 257), (16, 512), (16, 513), (32, 1024), (32, 1025)])
def test_evict_moves_by_the_selecting_cta(sessions, given_up):
    # the most rows one launch moves, and one more
    lens = [2500 - (i % 3) * 400 for i in range(sessions)]
    run_evict(lens, 2500 - given_up, 3, 50, hkv=2, hd=64)
    run_evict(lens, 2500 - given_up, 0, 0, hkv=2, hd=128, dtype=BF16, mix=True)


def test_evict_refusals():
    k, v = torch.zeros(2, 64, 2, 64, dtype=F16, device="cuda"), torch.zeros(2, 64, 2, 64, dtype=F16, device="cuda")
    w, pos = torch.zeros(2, 2, 64, device="cuda"), torch.zeros(2, 2, 64, dtype=torch.int32, device="cuda")

    def call(rows=64, budget=32, weights=w, **kw):
        tt.evict_kv_rows(context(), kw.pop("k", k), kw.pop("v", v), weights, rows, budget, **kw)
    call()
    half = k[:, :40]
    for bad in (dict(rows=65), dict(budget=0), dict(sink_tokens=20, recent_tokens=13), dict(weights=w[:, :, :60]), dict(weights=w.double()),
                dict(positions=pos.long()), dict(k=k.float()), dict(v=v[:1]), dict(k_out=half[:, :31], v_out=half[:, :31]),
                dict(k_out=k[:, 1:]), dict(weights_out=w[:, :, :31]), dict(weights_out=w[:, :, 1:]), dict(positions=pos, positions_out=pos[:, :, 2:]),
                dict(k=k.cpu(), v=v.cpu())):
        with pytest.raises(tt.InvalidArgument):
            call(**bad)
    with pytest.raises(tt.UnsupportedShape):
        call(k=k[..., :32].contiguous(), v=v[..., :32].contiguous())
    done()


# ------------------------------------------------------------------ together, streams, graphs

def test_session_with_a_bounded_cache():
    """A prompt, then decode steps over a cache of `budget` rows per head: statistics from the prompt's last rows, an
    eviction in place, then every step appends a row, accumulates, evicts one row. The cache is followed in 64 bits."""
    hd, hq, hkv, budget, prompt, tail, steps, sink, recent = 64, 8, 2, 96, 300, 16, 20, 4, 16
    g = hq // hkv
    k, v = normal(1, prompt + steps, hkv, hd), normal(2, prompt + steps, hkv, hd)
    q = normal(3, prompt + steps, hq, hd)
    kd = torch.zeros(1, prompt + 1, hkv, hd, dtype=F16, device="cuda")
    vd = torch.zeros_like(kd)
    kd[0, :prompt], vd[0, :prompt] = k[:prompt].cuda(), v[:prompt].cuda()
    w = torch.full((1, hkv, prompt + 1), NAN, device="cuda")
    pos = torch.full((1, hkv, prompt + 1), -1, dtype=torch.int32, device="cuda")
    a, ctx = tt.Attention(context()), context()
    qd = q.cuda()
    out = torch.empty(1, tail, hq, hd, dtype=F16, device="cuda")
    a.encode_accumulate(tt.SessionTable.over_cache(qd[None, prompt - tail:prompt], out, kd, vd, prompt), w, hd, hq, hkv, positions=pos,
                        fresh_rows=prompt, end_positions=prompt)
    held = [list(range(prompt)) for _ in range(hkv)]              # token in every cache row, per head
    stat = [torch.zeros(prompt, dtype=torch.float64) for _ in range(hkv)]
    for r in range(tail):
        t = prompt - tail + r
        want, p, bound = attend(q[t], k[:t + 1], v[:t + 1])
        check(out[0, r], want, bound)
        for h in range(hkv):
            stat[h][:t + 1] += p[h * g:(h + 1) * g].sum(0)
    rows = prompt
    for step in range(steps + 1):
        if step:
            t = prompt + step - 1
            kd[0, rows], vd[0, rows] = k[t].cuda(), v[t].cuda()
            rows += 1
            one = torch.empty(1, 1, hq, hd, dtype=F16, device="cuda")
            a.encode_accumulate(tt.SessionTable.over_cache(qd[None, t:t + 1], one, kd, vd, rows), w, hd, hq, hkv, positions=pos,
                                fresh_rows=1, end_positions=t + 1)
            for h in range(hkv):
                held[h].append(t)
                want, p, bound = attend(q[t, h * g:(h + 1) * g], k[held[h], h:h + 1], v[held[h], h:h + 1])
                check(one[0, 0, h * g:(h + 1) * g], want, bound)
                stat[h] = torch.cat([stat[h], torch.zeros(1, dtype=torch.float64)]) + p.sum(0)
        done()
        end = prompt + step
        for h in range(hkv):
            assert pos[0, h, :rows].tolist() == held[h]
            # each call adds its own rounding (2e-5 of what it adds, see attend), and the sums one of 2^-24 per term
            assert ((w[0, h, :rows].cpu().double() - stat[h]).abs() <= 2e-5 * stat[h] + 2.0 ** -24 * (tail + steps) * g * stat[h]).all()
        before = w.cpu()
        tt.evict_kv_rows(ctx, kd, vd, w, rows, budget, sink, recent, positions=pos, end_positions=end)
        done()
        for h in range(hkv):
            src = evict(before[0, h].tolist(), held[h], rows, budget, sink, recent, end)
            held[h], stat[h] = [held[h][s] for s in src], stat[h][src]
            assert torch.equal(kd[0, :budget, h].cpu(), k[held[h], h])
        rows = budget


def test_prompt_and_decode_in_one_ring():
    """A prompt in chunks and then tokens one by one through one ring cache of sinks and a window."""
    hd, hq, hkv, sink, window, ring, total = 256, 8, 2, 4, 100, 256, 700
    k, v, q = normal(1, total, hkv, hd), normal(2, total, hkv, hd), normal(3, total, hq, hd)
    kd, vd = (torch.zeros(1, sink + ring, hkv, hd, dtype=F16, device="cuda") for _ in range(2))
    qd, out = q.cuda(), torch.empty(total, hq, hd, dtype=F16, device="cuda")
    a, prefill = tt.Attention(context()), tt.PrefillAttention(context())

    def write(lo, hi):
        at = torch.tensor([ring_row(j, sink, ring) for j in range(lo, hi)], device="cuda")
        kd[0, at], vd[0, at] = k[lo:hi].cuda(), v[lo:hi].cuda()
    done_to = 0
    for chunk in (1, 150, 157, 100, 157):
        write(done_to, done_to + chunk)
        p = tt.PrefillAttentionParams(done_to, chunk, hd, hq, hkv, done_to + chunk, window, hkv * hd, hq * hd, hq * hd, hd ** -0.5)
        prefill.encode_sink_window(qd[done_to:], kd, vd, out[done_to:], p, sink, kv_ring_capacity=ring)
        done_to += chunk
    while done_to < total:
        rows = min(3, total - done_to)
        write(done_to, done_to + rows)
        done_to += rows
        a.encode_sink_window(tt.SessionTable.over_cache(qd[None, done_to - rows:done_to], out[None, done_to - rows:done_to], kd, vd, done_to),
                             hd, hq, hkv, sink, window, ring_capacity=ring)
    done()
    for t in sorted(set(range(0, total, 41)) | {1, 150, 151, 564, 565, 566, 699}):
        vis = torch.tensor(sink_keys(t + 1, sink, window))
        want, _, bound = attend(q[t], k[vis], v[vis])
        check(out[t], want, bound)


def _calls(n=3):
    """One of each decode-side call, its outputs, and a function that clears them."""
    hd, hq, hkv, s = 256, 16, 2, 400
    q, k, v = (normal(i, *x).cuda() for i, x in enumerate([(n, 1, hq, hd), (n, s, hkv, hd), (n, s, hkv, hd)]))
    pk, pv = normal(5, 1, 300, hkv, hd).cuda(), normal(6, 1, 300, hkv, hd).cuda()
    outs = [torch.zeros_like(q) for _ in range(3)]
    w, wo = torch.zeros(n, hkv, s, device="cuda"), torch.zeros(n, hkv, 100, device="cuda")
    po = torch.zeros(n, hkv, 100, dtype=torch.int32, device="cuda")
    ko, vo = torch.zeros(n, 100, hkv, hd, dtype=F16, device="cuda"), torch.zeros(n, 100, hkv, hd, dtype=F16, device="cuda")

    def run(ctx):
        a = tt.Attention(ctx)
        a.encode_sink_window(tt.SessionTable.over_cache(q, outs[0], k, v, [s, 50, 7][:n]), hd, hq, hkv, 4, 64)
        a.encode_shared_prefix(tt.PrefixTable.over_cache(pk, pv, 300, n), tt.SessionTable.over_cache(q, outs[1], k, v, [s, 50, 7][:n]), hd, hq, hkv)
        a.encode_accumulate(tt.SessionTable.over_cache(q, outs[2], k, v, s), w, hd, hq, hkv, fresh_rows=s)
        tt.evict_kv_rows(ctx, k, v, w, s, 100, 4, 20, k_out=ko, v_out=vo, weights_out=wo, positions_out=po)
    return run, outs + [w, wo, po, ko, vo]


def test_streams_and_graphs_give_the_same_results():
    ctx = tt.Context(0)
    run, results = _calls()
    run(ctx)
    torch.cuda.synchronize()
    want = [x.clone() for x in results]

    def cleared():
        for x in results:
            x.zero_()
        torch.cuda.synchronize()
    cleared()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        run(ctx)
    side.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(results, want))
    cleared()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        run(ctx)
    cleared()
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(results, want))
    # another call between two replays does not disturb the graph's own arguments
    tt.Attention(ctx).encode_batched([tt.DecodeSession(results[0][0], torch.empty_like(results[0][0]), results[6][0], results[7][0], 100)], 256, 16, 2)
    cleared()
    graph.replay()
    torch.cuda.synchronize()
    assert ctx.poll_status() == 0
    assert all(torch.equal(x, y) for x, y in zip(results, want))
    del graph
    ctx.close()


def test_first_calls_inside_a_capture():
    # nothing of these calls ran before in this context: what they ask the driver once must not disturb the capture
    ctx = tt.Context(0)
    run, results = _calls()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        run(ctx)
    graph.replay()
    torch.cuda.synchronize()
    assert ctx.poll_status() == 0
    got = [x.clone() for x in results]
    for x in results:
        x.zero_()
    run(ctx)
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(results, got))
    del graph
    ctx.close()


def test_two_contexts_at_once():
    contexts = [tt.Context(0) for _ in range(2)]
    calls = [_calls(), _calls(2)]
    want = []
    for ctx, (run, results) in zip(contexts, calls):
        run(ctx)
        torch.cuda.synchronize()
        want.append([x.clone() for x in results])
        for x in results:
            x.zero_()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(20):
        for ctx, (run, _results), stream in zip(contexts, calls, streams):
            with torch.cuda.stream(stream):
                _results[3].zero_()                       # the statistic starts anew
                run(ctx)
    torch.cuda.synchronize()
    for ctx, (_run, results), expected in zip(contexts, calls, want):
        assert ctx.poll_status() == 0
        assert all(torch.equal(x, y) for x, y in zip(results, expected))
        ctx.close()


def test_calls_that_upload_tables_refuse_a_capture():
    hd, hq, hkv, n = 64, 4, 2, 65
    q, k = torch.zeros(n, 1, hq, hd, dtype=F16, device="cuda"), torch.zeros(n, 8, hkv, hd, dtype=F16, device="cuda")
    out, a = torch.zeros_like(q), tt.Attention(context())
    t = tt.SessionTable.over_cache(q, out, k, k, 5)
    few = tt.SessionTable.over_cache(q[:9], out[:9], k[:9], k[:9], 5)
    w = torch.zeros(n, hkv, 8, device="cuda")
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        with pytest.raises(tt.UnsupportedShape):
            a.encode_sink_window(t, hd, hq, hkv, 1, 4)
        with pytest.raises(tt.UnsupportedShape):
            a.encode_shared_prefix(tt.PrefixTable.over_cache(k[:1], k[:1], 4, n), t, hd, hq, hkv)
        with pytest.raises(tt.UnsupportedShape):
            a.encode_shared_prefix(tt.PrefixTable.over_cache(k[:9], k[:9], 4, 1), few, hd, hq, hkv)
        a.encode_accumulate(t, w, hd, hq, hkv)
        tt.evict_kv_rows(context(), k, k.clone(), w, 8, 4)
    graph.replay()
    done()
    assert torch.allclose(w[:, :, :5].sum(-1), torch.tensor(2.0, device="cuda"), atol=1e-4) and (w[:, :, 5:] == 0).all()
    del graph
