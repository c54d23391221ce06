"""Calls at the edges of the bounded- and shared-cache operators on the GPU, against plain 64-bit references."""
import pytest
import torch

import tinytitan_b200 as tt
from bounded_cache_reference import attend, sink_keys
from gpu_util import context
from test_gpu_bounded_cache import BF16, F16, NAN, check, normal, run_accumulate, run_evict, run_prefix, run_sink_decode

pytestmark = pytest.mark.gpu


# Draft rows over a plain sliding window (no sinks) whose keys fill an odd number of 64-key halves: the spare half of the last
# tile belongs to no row, and the cache's first row, long behind the window, holds NaN like every row that nobody sees.
@pytest.mark.parametrize("hd,hq,hkv,sessions", [(256, 16, 2, 3), (128, 16, 2, 40), (64, 32, 1, 40), (128, 64, 1, 3)])
@pytest.mark.parametrize("window,ring", [(130, 0), (520, 0), (1024, 0), (130, 1100), (520, 1100)])
def test_draft_rows_behind_a_window_without_sinks(hd, hq, hkv, sessions, window, ring):
    rows = 4                                                     # window + 3 keys: 3, 9 and 17 halves
    lens = [window + 777 + i % 5 for i in range(sessions)]       # in the ring: wrapped (1800 of 1100) or not yet, the window in one piece
    if ring:
        lens = [1800 + i % 5 for i in range(sessions)]
        assert all((n - window - 3) % ring + window + 3 <= ring for n in lens)
    run_sink_decode(hd, hq, hkv, F16 if window == 520 else BF16, rows, lens, 0, window, ring)


@pytest.mark.parametrize("max_sessions", [1, 3])
def test_accumulate_takes_more_sessions_than_its_context_has_places(max_sessions):
    ctx = tt.Context(0, max_sessions=max_sessions)
    lens = [5 + 9 * i for i in range(10)]
    run_accumulate(64, 8, 2, F16, [1 + i % 3 for i in range(10)], lens, [1 + i % 3 for i in range(10)], ctx=ctx)
    run_accumulate(256, 16, 2, BF16, [1] * 70, [1 + i for i in range(70)], [0] * 70, ctx=ctx)
    ctx.close()


def test_accumulate_refused_calls_add_nothing():
    """A call that takes several passes is refused before the first of them, whichever session is at fault."""
    hd, hq, hkv, n, cap = 64, 8, 2, 70, 40
    q, k, w = torch.zeros(n, 1, hq, hd, dtype=F16, device="cuda"), torch.ones(n, cap, hkv, hd, dtype=F16, device="cuda"), torch.zeros(n, hkv, cap, device="cuda")
    out = torch.full_like(q, 7.0)
    a = tt.Attention(tt.Context(0))
    good = [tt.DecodeSession(q[i], out[i], k[i], k[i], 30) for i in range(n)]
    last = n - 1
    for error, bad in ((tt.InvalidArgument, tt.DecodeSession(q[last], out[last], None, k[last], 30)),
                       (tt.InvalidArgument, tt.DecodeSession(q[last], None, k[last], k[last], 30)),
                       (tt.UnsupportedShape, tt.DecodeSession(q[last], out[last], k[last], k[last], 30, v_offset=2)),
                       (tt.UnsupportedShape, tt.DecodeSession(q[last], out[last], k[last], k[last], 30, q_offset=8))):
        with pytest.raises(error):
            a.encode_accumulate(good[:last] + [bad], w, hd, hq, hkv, fresh_rows=1)
    torch.cuda.synchronize()
    assert (w == 0).all() and (out == 7).all()
    # the last session's scores, then its partials, do not fit the workspace
    for length, rows, room in ((5000, 1, 1 << 17), (4, 64, 1 << 17)):
        small = tt.Context(0, workspace_bytes=room)
        lens = [30] * 3 + [length]
        qs, ks = torch.zeros(4, rows, hq, hd, dtype=F16, device="cuda"), torch.zeros(4, max(lens), hkv, hd, dtype=F16, device="cuda")
        ws, outs = torch.zeros(4, hkv, max(lens), device="cuda"), torch.full((4, rows, hq, hd), 7.0, dtype=F16, device="cuda")
        sessions = [tt.DecodeSession(qs[i], outs[i], ks[i], ks[i], max(lens[i], rows - 1), rows if i == 3 else 1) for i in range(4)]
        with pytest.raises(tt.TinyTitanError):
            tt.Attention(small).encode_accumulate(sessions, ws, hd, hq, hkv)
        torch.cuda.synchronize()
        assert (ws == 0).all() and (outs == 7).all()
        small.close()


def test_accumulate_cut_by_rows_with_a_narrowly_padded_output():
    # an output row stride that keeps rows 8-byte aligned: passes behind the first start at such rows
    hd, hq, hkv, rows, m, pad = 64, 32, 2, 3, 2000, 4            # one row a pass
    ctx = tt.Context(0, workspace_bytes=900_000)
    q, k, v = normal(1, rows, hq, hd), normal(2, m, hkv, hd), normal(3, m, hkv, hd)
    out, w = torch.full((rows, hq * hd + pad), NAN, dtype=F16, device="cuda"), torch.zeros(1, hkv, m, device="cuda")
    d = [x.cuda() for x in (q, k, v)]
    tt.Attention(ctx).encode_accumulate([tt.DecodeSession(d[0], out, d[1], d[2], m, rows)], w, hd, hq, hkv, out_row_stride_elements=hq * hd + pad)
    torch.cuda.synchronize()
    added = torch.zeros(hkv, m, dtype=torch.float64)
    for r in range(rows):
        end = m - (rows - 1 - r)
        o, p, bound = attend(q[r], k[:end], v[:end])
        check(out[r, :hq * hd].reshape(hq, hd), o, bound)
        added[:, :end] += p.reshape(hkv, hq // hkv, end).sum(1)
    # 32-bit scores, exponentials and normaliser (2e-5, see attend), and one rounding of 2^-24 per added weight
    assert ((w[0].cpu().double() - added).abs() <= (2e-5 + (1 + rows * hq // hkv) * 2.0 ** -24) * added).all()
    ctx.close()


def test_evict_refused_calls_move_nothing():
    """A call whose last session's row map does not fit the workspace is refused before any session gives up a row."""
    ctx = tt.Context(0, workspace_bytes=6000)                    # 1500 map entries: a session of 1001 rows needs 1001, one of 2000 rows 2000
    n, cap, budget = 3, 2000, 1000
    k = normal(1, n, cap, 1, 64).cuda()
    v, w = k.clone(), torch.rand(n, 1, cap, generator=torch.Generator().manual_seed(2)).cuda()
    before = [x.clone() for x in (k, v, w)]
    with pytest.raises(tt.TinyTitanError):
        tt.evict_kv_rows(ctx, k, v, w, [1001, 1001, 2000], budget)
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip((k, v, w), before))
    tt.evict_kv_rows(ctx, k, v, w, [1001, 1001, 1400], budget)   # each fits alone: one launch a session
    torch.cuda.synchronize()
    assert not any(torch.equal(w[i], before[2][i]) for i in range(n))
    ctx.close()


@pytest.mark.parametrize("rows", [1, 4])
def test_plain_decode_over_session_tables(rows):
    # the rows that an eviction leaves, by plain decode: a table gives what a list of sessions does
    n, hq, hkv, hd, cap = 5, 16, 2, 256, 300
    q, k, v = (normal(i, *x).cuda() for i, x in enumerate([(n, rows, hq, hd), (n, cap, hkv, hd), (n, cap, hkv, hd)]))
    w, lens, a = torch.rand(n, hkv, cap, generator=torch.Generator().manual_seed(3)).cuda(), [300, 150, 64, 99, 7], tt.Attention(context())
    tt.evict_kv_rows(context(), k, v, w, lens, 64)
    left = [min(x, 64) for x in lens]
    outs = [torch.zeros_like(q) for _ in range(3)]
    a.encode_batched([tt.DecodeSession(q[i], outs[0][i], k[i], v[i], left[i], rows) for i in range(n)], hd, hq, hkv)
    a.encode_batched(tt.SessionTable.over_cache(q, outs[1], k, v, left), hd, hq, hkv)
    a.encode_prepared(a.prepare_batch(tt.SessionTable.over_cache(q, outs[2], k, v, left), hd, hq, hkv))
    torch.cuda.synchronize()
    assert context().poll_status() == 0
    assert outs[0].any() and torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


@pytest.mark.parametrize("in_place", [True, False])
def test_evict_more_keys_than_a_cluster_holds(in_place):
    # 16 CTAs hold 800,000 selection keys; beyond, every round reads the statistic and the positions again
    run_evict([810_003, 800_000], 500_000, 4, 1000, hkv=1, hd=64, in_place=in_place)
    run_evict([810_003], 900, 0, 0, hkv=1, hd=64, in_place=in_place, mix=True, keep_positions=False)


# Tables of 24 and of 72 groups travel in the parameters: prefixes and sessions on both sides, draft rows of 12 and 36 sessions.
@pytest.mark.parametrize("sessions", [16, 17, 32])
def test_prefix_tables_on_both_sides_of_their_sizes(sessions):
    per = [sessions // 8 + (i < sessions % 8) for i in range(8)]
    run_prefix(128, 16, 2, F16, [130 + 9 * i for i in range(8)], per, [1] * sessions, [(11 * i) % 140 for i in range(sessions)])
    run_prefix(256, 16, 2, BF16, [7 + 40 * i for i in range(8)], per, [3] * sessions, [2 + (13 * i) % 90 for i in range(sessions)])


@pytest.mark.parametrize("sessions", [12, 13, 36, 37])
def test_draft_rows_on_both_sides_of_the_table_sizes(sessions):
    run_sink_decode(128, 16, 2, F16, 4, [700 + 31 * (i % 9) for i in range(sessions)], 4, 400, 0)
    run_sink_decode(256, 16, 2, BF16, 3, [900 + 31 * (i % 9) for i in range(sessions)], 3, 300, 333)


# Own rows in a pass of their own whose streams leave the machine four places each, two, or one, and heads of all sizes.
@pytest.mark.parametrize("hd,hq,hkv,n", [(256, 8, 4, 33), (256, 8, 4, 64), (256, 8, 8, 64), (128, 8, 8, 40), (128, 3, 3, 40), (64, 8, 8, 64), (64, 3, 1, 64)])
def test_prefix_streams_of_own_rows(hd, hq, hkv, n):
    run_prefix(hd, hq, hkv, F16, [140], [n], [1] * n, [[3, 900, 64, 65, 400][i % 5] + i for i in range(n)])


# ------------------------------------------------------------------ caches of more than 4 GiB (rows of 1 KB)

LONG = 4_300_000


@pytest.fixture(scope="module")
def long_cache():
    cache = [torch.empty(LONG, 2, 256, dtype=F16, device="cuda") for _ in range(2)]
    yield cache
    cache.clear()
    torch.cuda.empty_cache()


@pytest.mark.parametrize("rows", [1, 4])
@pytest.mark.parametrize("hq", [8, 16])
def test_sink_decode_beyond_four_gigabytes(long_cache, hq, rows):
    hd, hkv, sink, window = 256, 2, 5, 700
    k, v = normal(1, window + rows, hkv, hd), normal(2, window + rows, hkv, hd)
    ks, vs, q = normal(3, sink, hkv, hd), normal(4, sink, hkv, hd), normal(5, rows, hq, hd)
    first = LONG - window - rows
    for cache, near, far in ((long_cache[0], ks, k), (long_cache[1], vs, v)):
        cache[:sink], cache[first:] = near.cuda(), far.cuda()
        cache[sink:first:1009] = NAN
    out = torch.empty(1, rows, hq, hd, dtype=F16, device="cuda")
    t = tt.SessionTable.over_cache(q.cuda()[None], out, long_cache[0][None], long_cache[1][None], LONG)
    tt.Attention(context()).encode_sink_window(t, hd, hq, hkv, sink, window)
    torch.cuda.synchronize()
    assert context().poll_status() == 0
    for r in range(rows):
        at = torch.tensor([j - first for j in sink_keys(LONG - (rows - 1 - r), sink, window) if j >= sink])
        o, _, bound = attend(q[r], torch.cat([ks, k[at]]), torch.cat([vs, v[at]]))
        check(out[0, r], o, bound)


def test_sink_prefill_beyond_four_gigabytes(long_cache):
    hd, hq, hkv, sink, window, tokens = 256, 8, 2, 70, 300, 50
    start = LONG - tokens
    first = start + 1 - window
    k, v = normal(1, LONG - first, hkv, hd), normal(2, LONG - first, hkv, hd)
    ks, vs, q = normal(3, sink, hkv, hd), normal(4, sink, hkv, hd), normal(5, tokens, hq, hd)
    for cache, near, far in ((long_cache[0], ks, k), (long_cache[1], vs, v)):
        cache[:sink], cache[first:] = near.cuda(), far.cuda()
    out = torch.empty(tokens, hq, hd, dtype=F16, device="cuda")
    p = tt.PrefillAttentionParams(start, tokens, hd, hq, hkv, LONG, window, hkv * hd, hq * hd, hq * hd, hd ** -0.5)
    tt.PrefillAttention(context()).encode_sink_window(q.cuda(), long_cache[0], long_cache[1], out, p, sink)
    torch.cuda.synchronize()
    assert context().poll_status() == 0
    for t in (0, 1, 31, 32, 49):
        at = torch.tensor([j - first for j in sink_keys(start + t + 1, sink, window) if j >= sink])
        o, _, bound = attend(q[t], torch.cat([ks, k[at]]), torch.cat([vs, v[at]]))
        check(out[t], o, bound)


def test_prefix_and_accumulate_beyond_four_gigabytes(long_cache):
    # all keys but a few near the end score far below them: the few weigh everything, the others nothing
    hd, hq, hkv = 256, 8, 2
    few = torch.tensor([LONG - 1, LONG - 2, LONG - 130, LONG - 5000])
    q, kf, vf = normal(5, hq, hd), normal(6, len(few), hkv, hd), normal(7, len(few), hkv, hd)
    q[:, 0], kf[:, :, 0] = 16.0, 16.0                                # a score of 16 against one of -160 * 16 / 16
    for cache in long_cache:
        cache.zero_()
    long_cache[0][:, :, 0] = -160.0
    long_cache[0][few.cuda()], long_cache[1][few.cuda()] = kf.cuda(), vf.cuda()
    out = torch.empty(2, 1, 1, hq, hd, dtype=F16, device="cuda")
    ctx = tt.Context(0, workspace_bytes=1 << 30)                     # the scores of so many keys
    a, qd, w = tt.Attention(ctx), q.cuda()[None, None], torch.zeros(1, hkv, LONG, device="cuda")
    k, v = long_cache[0][None], long_cache[1][None]
    a.encode_shared_prefix(tt.PrefixTable.over_cache(k, v, LONG, 1), tt.SessionTable.over_cache(qd, out[0], k, v, 0), hd, hq, hkv)
    a.encode_accumulate(tt.SessionTable.over_cache(qd, out[1], k, v, LONG), w, hd, hq, hkv)
    torch.cuda.synchronize()
    assert ctx.poll_status() == 0
    o, p, bound = attend(q, kf, vf)
    added = p.reshape(hkv, hq // hkv, -1).sum(1)
    assert (p > 0).all()
    for x in out:
        check(x[0, 0], o, bound)
    # 32-bit scores, exponentials and normaliser (2e-5, see attend); exp(-160) is below every 32-bit number that counts
    assert ((w[0].cpu()[:, few].double() - added).abs() <= 2e-5 * added + 1e-30).all()
    w[0][:, few.cuda()] = 0
    assert (w < 1e-30).all()
    ctx.close()


def test_evict_beyond_four_gigabytes(long_cache):
    given_up, budget = 100_000, LONG - 100_000
    row = torch.arange(LONG, device="cuda")
    for cache, shift in zip(long_cache, (0, 1)):
        for h in range(2):
            for digit in range(3):                                   # rows by their digits to the base 256
                cache[:, h, digit] = ((row + shift + h >> 8 * digit) & 255).half()
    w = torch.rand(1, 2, LONG, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    before, p = w.clone(), torch.zeros(1, 2, LONG, dtype=torch.int32, device="cuda")
    ctx = tt.Context(0)
    tt.evict_kv_rows(ctx, long_cache[0][None], long_cache[1][None], w, LONG, budget, positions_out=p)
    torch.cuda.synchronize()
    assert ctx.poll_status() == 0
    for h in range(2):
        order = before[0, h].sort(descending=True, stable=True).indices[:budget]
        keep = torch.zeros(LONG, dtype=torch.bool, device="cuda")
        keep[order] = True
        src, fills = row[:budget].clone(), row[keep & (row >= budget)]
        src[~keep[:budget]] = fills
        assert len(fills) and torch.equal(p[0, h, :budget].long(), src) and torch.equal(w[0, h, :budget], before[0, h, src])
        for cache, shift in zip(long_cache, (0, 1)):
            held = sum(cache[:budget, h, digit].long() << 8 * digit for digit in range(3))
            assert torch.equal(held, src + shift + h)
    ctx.close()


# ------------------------------------------------------------------ layouts

@pytest.mark.parametrize("layout", ["interleaved", "token-major"])
@pytest.mark.parametrize("rows", [1, 4])
def test_layouts_give_the_same_bits(layout, rows):
    """K beside V in every row, or the sessions' rows side by side: what the contiguous cache gives, bit for bit."""
    n, cap, hq, hkv, hd = 4, 300, 16, 2, 256
    q, k, v, w0 = normal(1, n, rows, hq, hd).cuda(), normal(2, n, cap, hkv, hd).cuda(), normal(3, n, cap, hkv, hd).cuda(), torch.rand(n, hkv, cap, generator=torch.Generator().manual_seed(4)).cuda()
    lens, a = [300, 77, 200, rows], tt.Attention(context())

    def lay(x, y):
        if layout == "interleaved":
            both = torch.stack([x, y], dim=2)
            return both[:, :, 0], both[:, :, 1]
        return tuple(t.transpose(0, 1).contiguous().transpose(0, 1) for t in (x, y))
    got = []
    for kk, vv in ((k.clone(), v.clone()), lay(k, v)):
        outs, w = [torch.zeros_like(q) for _ in range(4)], w0.clone()
        table = [tt.SessionTable.over_cache(q, o, kk, vv, lens) for o in outs]
        a.encode_sink_window(table[0], hd, hq, hkv, 4, 100)
        a.encode_shared_prefix(tt.PrefixTable.over_cache(kk[1:2], vv[1:2], 250, n), table[1], hd, hq, hkv)
        a.encode_accumulate(table[2], w, hd, hq, hkv, fresh_rows=rows)
        a.encode_batched(table[3], hd, hq, hkv)
        tt.evict_kv_rows(context(), kk, vv, w, lens, 90, 2, 10)
        torch.cuda.synchronize()
        assert context().poll_status() == 0
        got.append(outs + [w, kk.contiguous(), vv.contiguous()])
    assert all(x.any() and torch.equal(x, y) for x, y in zip(*got))


def test_sessions_that_read_one_slot():
    # the branches of one search: several sessions over one slot, each with queries and a length of its own
    n, cap, hq, hkv, hd, slots, lens = 5, 200, 8, 2, 128, [1, 1, 0, 1, 0], [200, 150, 33, 150, 200]
    q, k, v, a = normal(1, n, 1, hq, hd), normal(2, 2, cap, hkv, hd), normal(3, 2, cap, hkv, hd), tt.Attention(context())
    d = [x.cuda() for x in (q, k, v)]
    out, w = [torch.zeros_like(d[0]) for _ in range(2)], torch.zeros(n, hkv, cap, device="cuda")
    a.encode_sink_window(tt.SessionTable.over_cache(d[0], out[0], d[1], d[2], lens, slots=slots), hd, hq, hkv, 3, 60)
    a.encode_accumulate(tt.SessionTable.over_cache(d[0], out[1], d[1], d[2], lens, slots=slots), w, hd, hq, hkv)
    torch.cuda.synchronize()
    for i in range(n):
        at = torch.tensor(sink_keys(lens[i], 3, 60))
        o, _, bound = attend(q[i, 0], k[slots[i], at], v[slots[i], at])
        check(out[0][i, 0], o, bound)
        o, p, bound = attend(q[i, 0], k[slots[i], :lens[i]], v[slots[i], :lens[i]])
        check(out[1][i, 0], o, bound)
        added = p.reshape(hkv, hq // hkv, -1).sum(1)             # 32-bit scores to normaliser 2e-5 (see attend), four sums of 2^-24
        assert ((w[i, :, :lens[i]].cpu().double() - added).abs() <= (2e-5 + 5 * 2.0 ** -24) * added).all()
