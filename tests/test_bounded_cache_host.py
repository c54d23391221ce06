"""Host side of the bounded- and shared-cache operators: key sets, split plans, session tables, refusals. No GPU."""
import ctypes as C
import random

import numpy as np
import pytest
import torch

import tinytitan_b200 as tt
from bounded_cache_reference import evict, sink_keys
from tinytitan_b200 import _lib as L


def _sink(seq_len, q_rows, sink, window):
    start, keys = C.c_uint32(0), C.c_uint32(0)
    rc = L.lib().tt_attn_sink_keys(seq_len, q_rows, sink, window, C.byref(start), C.byref(keys))
    return rc, start.value, keys.value


@pytest.mark.parametrize("q_rows", [1, 2, 5])
@pytest.mark.parametrize("sink", [0, 1, 4, 9, 40])
@pytest.mark.parametrize("window", [0, 1, 3, 8, 100])
def test_sink_keys_are_the_union_of_the_rows(q_rows, sink, window):
    for seq_len in range(q_rows - 1, 40):
        rc, start, count = _sink(seq_len, q_rows, sink, window)
        assert rc == 0
        union = set()
        for r in range(q_rows):
            union |= set(sink_keys(seq_len - (q_rows - 1 - r), sink, window))
        # what the kernel reads: the sinks, then every key from `start` on
        reads = set(range(min(sink, seq_len))) | set(range(start, seq_len))
        assert count == len(reads) and start >= sink
        assert union <= reads
        # a sink that only a later row may see is read; nothing else is read in vain
        assert all(j < sink for j in reads - union)


def test_sink_keys_refusals():
    assert _sink(3, 5, 4, 8)[0] == L.TT_ERR_INVALID_ARG
    assert _sink(3, 0, 4, 8)[0] == L.TT_ERR_INVALID_ARG
    assert _sink(2 ** 31, 1, 4, 8)[0] == L.TT_ERR_INVALID_ARG
    rc, start, keys = _sink(2 ** 31 - 1, 1, 4, 1000)
    assert rc == 0 and start == 2 ** 31 - 1001 and keys == 1004


def _prefix_plan(lens, rows, hd=256, hq=16, hkv=2, sms=148, ws=128 << 20):
    n = len(lens)
    per, items = C.c_uint32(0), C.c_uint32(0)
    rc = L.lib().tt_attn_plan_prefix_splits((C.c_uint32 * n)(*lens), (C.c_uint32 * n)(*rows), n, hd, hq, hkv, sms, ws,
                                            C.byref(per), C.byref(items))
    return rc, per.value, items.value


def test_prefix_plan():
    # one long prefix, 64 sessions x 8 heads = 512 packed rows: two items of 256 rows (a pair of SMs each) x 2 KV heads = 4
    # streams, cut so that one wave fills the 74 pairs
    rc, per, items = _prefix_plan([32768], [64])
    assert rc == 0 and per % 128 == 0 and items == 4 * -(-32768 // per) and 50 <= items <= 74
    # 128 packed rows fit one SM: 2 streams over 148 of them; at head_dim 128 512 rows are four items of 128
    rc, per, items = _prefix_plan([32768], [16])
    assert rc == 0 and items == 2 * -(-32768 // per) and 100 <= items <= 148
    rc, per, items = _prefix_plan([32768], [64], hd=128)
    assert rc == 0 and items == 8 * -(-32768 // per) and 100 <= items <= 148
    # a short prefix of a few sessions: one tile per item
    rc, per, items = _prefix_plan([2000], [4], hq=8)
    assert rc == 0 and per == 128 and items == 2 * 16
    # a group without a prefix has no items
    rc, per, items = _prefix_plan([0, 500], [1, 1])
    assert rc == 0 and items == 2 * -(-500 // per)
    rc, per, items = _prefix_plan([0], [3])
    assert rc == 0 and items == 0
    # partials that do not fit are split less, and refused when one part per prefix is too much
    rc, per, items = _prefix_plan([32768], [64], ws=4 << 20)
    assert rc == 0 and -(-32768 // per) * 64 * 16 * 258 * 4 <= 4 << 20
    assert _prefix_plan([32768], [64], ws=1 << 10)[0] == L.TT_ERR_OOM
    assert _prefix_plan([32768], [64], hq=15)[0] == L.TT_ERR_INVALID_ARG


def test_eviction_reference_keeps_the_budget():
    r = random.Random(3)
    for _ in range(50):
        rows = r.randint(1, 60)
        budget = r.randint(1, 60)
        w = [r.choice([0.0, 1.0, r.random(), float("nan"), float("inf")]) for _ in range(rows)]
        pos = list(range(rows))
        r.shuffle(pos)
        sink = r.randint(0, min(3, budget))
        recent = r.randint(0, budget - sink)
        src = evict(w, pos, rows, budget, sink, recent, rows)
        assert len(src) == min(rows, budget) == len(set(src))
        assert all(s == j or s >= budget for j, s in enumerate(src))
        if rows > budget:
            assert {j for j in range(rows) if pos[j] < sink or pos[j] >= rows - recent} <= set(src)


class _Context:
    """What the wrappers need of a context before they reach the library."""
    handle, device = None, 0

    def check(self, status):
        raise AssertionError("the library was called")

    check_device = tt.Context.check_device
    stream = tt.Context.stream


def test_session_table_addresses():
    q = torch.zeros(3, 2, 8, 64, dtype=torch.float16)
    out = torch.zeros(3, 2, 8, 64, dtype=torch.float16)
    k = torch.zeros(5, 20, 2, 64, dtype=torch.float16)
    v = torch.zeros(5, 20, 2, 64, dtype=torch.float16)
    t = tt.SessionTable.over_cache(q, out, k, v, [4, 20, 7], slots=[4, 0, 2])
    assert list(t.records["k"]) == [k[4].data_ptr(), k[0].data_ptr(), k[2].data_ptr()]
    assert list(t.records["q"]) == [q[i].data_ptr() for i in range(3)]
    assert list(t.records["seq_len"]) == [4, 20, 7] and set(t.records["q_rows"]) == {2}
    assert (t.kv_stride, t.q_stride, t.out_stride, t.io_dtype) == (128, 512, 512, tt.TT_F16)
    assert t.records.itemsize == C.sizeof(L.AttnSession)
    # a list of sessions gives the same block
    same = tt.SessionTable.of([tt.DecodeSession(q[i], out[i], k[s], v[s], n, 2) for i, (s, n) in enumerate([(4, 4), (0, 20), (2, 7)])])
    assert np.array_equal(same.records, t.records)
    # a cache whose rows are wider than its heads
    wide = torch.zeros(5, 20, 3, 64, dtype=torch.float16)[:, :, :2]
    assert tt.SessionTable.over_cache(q, out, wide, wide, 3).kv_stride == 192
    assert tt.PrefixTable.record.itemsize == C.sizeof(L.AttnPrefix)
    p = tt.PrefixTable.over_cache(k, v, [3, 0, 20, 1, 5], 2)
    assert list(p.records["v"]) == [v[i].data_ptr() for i in range(5)] and list(p.records["prefix_len"]) == [3, 0, 20, 1, 5]


@pytest.mark.parametrize("n", [0, 1, 2, 6, 7, 65])
@pytest.mark.parametrize("kind", [list, tuple, np.array, lambda x: list(np.array(x, dtype=np.int32)), torch.tensor])
def test_session_table_sizes(n, kind):
    q, k = torch.zeros(n, 3, 4, 64, dtype=torch.bfloat16), torch.zeros(n + 2, 9, 2, 64, dtype=torch.bfloat16)
    lens, slots = [i % 10 for i in range(n)], [n + 1 - i for i in range(n)]
    for t, where in ((tt.SessionTable.over_cache(q, q, k, k, kind(lens)), range(n)),
                     (tt.SessionTable.over_cache(q, q, k, k, kind(lens), slots=kind(slots)), slots)):
        assert len(t) == len(t.records) == n and t.longest == max(lens, default=0)
        for i, r in enumerate(t.records):
            assert r.tolist() == (q[i].data_ptr(), q[i].data_ptr(), k[where[i]].data_ptr(), k[where[i]].data_ptr(), lens[i], 3, 0, 0)
    p = tt.PrefixTable.over_cache(k[:n], k[:n], kind(lens), kind([1 + i for i in range(n)]))
    assert len(p) == n and [r.tolist() for r in p.records] == [(k[i].data_ptr(), k[i].data_ptr(), lens[i], 1 + i) for i in range(n)]


def test_wrappers_refuse_before_the_library():
    h = torch.float16
    q, out = torch.zeros(3, 1, 8, 64, dtype=h), torch.zeros(3, 1, 8, 64, dtype=h)
    k, v = torch.zeros(3, 20, 2, 64, dtype=h), torch.zeros(3, 20, 2, 64, dtype=h)
    over = tt.SessionTable.over_cache
    with pytest.raises(tt.InvalidArgument):
        over(q, out, k.bfloat16(), v, 4)
    with pytest.raises(tt.InvalidArgument):
        over(q.float(), out.float(), k.float(), v.float(), 4)
    with pytest.raises(tt.InvalidArgument):
        over(q, out, k[:2], v[:2], 4)
    with pytest.raises(tt.InvalidArgument):
        over(q, out, k, v, 4, slots=[0, 1, 3])
    with pytest.raises(tt.InvalidArgument):
        over(q, out, k.transpose(2, 3), v.transpose(2, 3), 4)
    with pytest.raises(tt.InvalidArgument):
        over(q, out, k, v, [4, -1, 4])
    with pytest.raises(tt.InvalidArgument):
        over(q, out[:, :, :4], k, v, 4)
    attention = tt.Attention(_Context())
    # tensors that are not on the context's device
    with pytest.raises(tt.InvalidArgument):
        attention.encode_sink_window(over(q, out, k, v, 4), 64, 8, 2, 4, 8)
    on_gpu = over(q, out, k, v, 21)
    on_gpu.device = None
    with pytest.raises(tt.InvalidArgument):
        attention.encode_sink_window(on_gpu, 64, 8, 2, 4, 8)                      # longer than its slot
    with pytest.raises(tt.InvalidArgument):
        attention.encode_sink_window(on_gpu, 64, 8, 2, 4, 8, ring_capacity=17)    # sinks + ring do not fit the slot
    with pytest.raises(tt.InvalidArgument):
        tt.PrefixTable.over_cache(k, v, 21, 1)
    with pytest.raises(tt.InvalidArgument):
        tt.evict_kv_rows(_Context(), k, v, torch.zeros(3, 2, 20), 20, 8)          # CPU tensors
    # the blocks of 64-bit words the wrappers build are the C structures
    assert C.sizeof(L.KVEvictSession) == 9 * 8 and C.sizeof(L.AttnWeightRows) == 3 * 8
    assert [getattr(L.KVEvictSession, n).offset for n in ("k_out", "weights", "positions_out", "rows", "end_position")] == [16, 32, 56, 64, 68]
    assert [getattr(L.AttnWeightRows, n).offset for n in ("positions", "fresh_rows", "end_position")] == [8, 16, 20]
