"""What the wrappers over bounded and shared caches refuse before they reach the library. No GPU."""
import pytest
import torch

import tinytitan_b200 as tt

H, B = torch.float16, torch.bfloat16


class LibraryCalled(Exception):
    pass


class HostContext:
    """A context whose device is the host's, so that every check but the library's own is passed on the way to it."""
    handle, device = None, -1

    def check(self, status):
        raise LibraryCalled

    check_device = tt.Context.check_device
    stream = tt.Context.stream


def attention():
    return tt.Attention(HostContext())


def cache(n=3, rows=20, hkv=2, hd=64, dtype=H, pad=0):
    """[n, rows, hkv, hd], rows `pad` heads wider than that."""
    return torch.zeros(n, rows, hkv + pad, hd, dtype=dtype)[:, :, :hkv]


def queries(n=3, rows=1, hq=8, hd=64, dtype=H):
    return torch.zeros(n, rows, hq, hd, dtype=dtype)


def sessions(k=None, q=None, lens=4):
    k, q = cache() if k is None else k, queries() if q is None else q
    return tt.SessionTable.over_cache(q, q, k, k, lens)


def refused(call, *args, **kw):
    with pytest.raises(tt.InvalidArgument):
        call(*args, command_buffer=0, **kw)


def reaches_the_library(call, *args, **kw):
    with pytest.raises(LibraryCalled):
        call(*args, command_buffer=0, **kw)


def test_prefix_tables_must_match_their_sessions():
    shared = attention().encode_shared_prefix
    prefix = tt.PrefixTable.over_cache(cache(1), cache(1), 7, 3)
    reaches_the_library(shared, prefix, sessions(), 64, 8, 2)
    wide = tt.PrefixTable.over_cache(cache(1, pad=1), cache(1, pad=1), 7, 3)
    refused(shared, wide, sessions(), 64, 8, 2)                                          # rows of another stride
    refused(shared, prefix, sessions(cache(pad=1)), 64, 8, 2)
    reaches_the_library(shared, wide, sessions(cache(pad=1)), 64, 8, 2)
    refused(shared, prefix, sessions(cache(dtype=B), queries(dtype=B)), 64, 8, 2)        # of another type
    refused(shared, tt.PrefixTable.over_cache(cache(1, hkv=1), cache(1, hkv=1), 7, 3), sessions(), 64, 8, 2)    # other heads
    refused(shared, tt.PrefixTable.over_cache(cache(1, hkv=1, hd=128), cache(1, hkv=1, hd=128), 7, 3), sessions(), 64, 8, 2)
    # lists of sessions have the strides and the type that the call says
    q, k = queries(), cache()
    each = [tt.DecodeSession(q[i], q[i], k[i], k[i], 4) for i in range(3)]
    reaches_the_library(shared, prefix, each, 64, 8, 2)
    reaches_the_library(shared, wide, each, 64, 8, 2, kv_token_stride_elements=192)
    refused(shared, wide, each, 64, 8, 2)
    refused(shared, prefix, each, 64, 8, 2, kv_token_stride_elements=192)
    refused(shared, prefix, each, 64, 8, 2, io_dtype=tt.TT_BF16)
    # one row has no stride
    reaches_the_library(shared, tt.PrefixTable.over_cache(cache(1, 1, pad=1), cache(1, 1, pad=1), 1, 3), sessions(), 64, 8, 2)


def test_session_tables_must_match_their_call():
    weights = torch.zeros(3, 2, 20)
    for call, tail in ((attention().encode_sink_window, (4, 8)), (attention().encode_accumulate, None)):
        def args(t, hd=64, hq=8, hkv=2):
            return (t, hd, hq, hkv) + tail if tail else (t, weights if hkv == 2 else torch.zeros(3, hkv, 20), hd, hq, hkv)
        reaches_the_library(call, *args(sessions()))
        wide = sessions(cache(pad=2), torch.zeros(3, 1, 12, 64, dtype=H)[:, :, :8])      # room for the heads that are not there
        reaches_the_library(call, *args(wide))
        refused(call, *args(wide, hkv=4))
        refused(call, *args(wide, hq=12))
        refused(call, *args(sessions(), hq=4))
        refused(call, *args(sessions(), hd=32))
        refused(call, *args(sessions(), hd=128, hq=4, hkv=1))
        # what the tensors say is not to be contradicted, but may be said again
        two = sessions(cache(pad=1), queries(rows=2))
        reaches_the_library(call, *args(two), kv_token_stride_elements=192, q_row_stride_elements=512, out_row_stride_elements=512, io_dtype=tt.TT_F16)
        for bad in (dict(kv_token_stride_elements=128), dict(q_row_stride_elements=520), dict(out_row_stride_elements=1024), dict(io_dtype=tt.TT_BF16)):
            refused(call, *args(two), **bad)


def test_one_row_has_no_stride():
    call = attention().encode_sink_window
    one = torch.zeros(3, 5, 8, 64, dtype=H)[:, 2:3]
    reaches_the_library(call, sessions(q=one), 64, 8, 2, 4, 8, q_row_stride_elements=1024, out_row_stride_elements=520)
    single = sessions(cache(rows=1), lens=1)
    wide = tt.PrefixTable.over_cache(cache(1, pad=1), cache(1, pad=1), 7, 3)
    reaches_the_library(attention().encode_shared_prefix, wide, single, 64, 8, 2)


def test_expanded_tensors():
    """Tensors that show one row, head or session several times: read where the layout can say so, else refused, never written."""
    over = tt.SessionTable.over_cache
    q, k = queries(rows=2), cache()
    one_row = cache(rows=1).expand(3, 20, 2, 64)                # one row shown twenty times
    with pytest.raises(tt.InvalidArgument):
        over(q, q, one_row, one_row, 4)
    with pytest.raises(tt.InvalidArgument):
        tt.PrefixTable.over_cache(one_row, one_row, 4, 1)
    with pytest.raises(tt.InvalidArgument):
        over(queries(rows=1).expand(3, 2, 8, 64), q, k, k, 4)
    with pytest.raises(tt.InvalidArgument):
        over(q, queries(rows=1).expand(3, 2, 8, 64), k, k, 4)
    with pytest.raises(tt.InvalidArgument):
        over(q, queries(1, 2).expand(3, 2, 8, 64), k, k, 4)     # outputs of all sessions in one place
    shared = cache(1).expand(3, 20, 2, 64)                      # one cache read by all sessions
    over(queries(1, 2).expand(3, 2, 8, 64), q, shared, shared, 4)
    tt.PrefixTable.over_cache(shared, shared, 4, 1)
    accumulate, w = attention().encode_accumulate, torch.zeros(3, 2, 20)
    reaches_the_library(accumulate, over(q, q, k, k, 4), w, 64, 8, 2, positions=w.int())
    for bad in (w[:1].expand(3, 2, 20), w[:, :1].expand(3, 2, 20)):
        refused(accumulate, over(q, q, k, k, 4), bad, 64, 8, 2)
        refused(accumulate, over(q, q, k, k, 4), w, 64, 8, 2, positions=bad.int()[:1].expand(3, 2, 20))
    single = torch.zeros(1, 2, 20)
    reaches_the_library(accumulate, over(q[:1], q[:1], k[:1], k[:1], 4), single.expand(1, 2, 20), 64, 8, 2)


def test_expanded_tensors_in_evictions():
    k, w = cache(), torch.zeros(3, 2, 20)
    p = w.int()
    outs = dict(k_out=cache(rows=8), v_out=cache(rows=8), weights_out=torch.zeros(3, 2, 8), positions_out=torch.zeros(3, 2, 8, dtype=torch.int32))

    def evict(k=k, w=w, **kw):
        tt.evict_kv_rows(HostContext(), k, k, w, 20, 8, command_buffer=kw.pop("command_buffer"), **kw)
    reaches_the_library(evict)
    reaches_the_library(evict, positions=p, **outs)
    shared, flat = cache(1).expand(3, 20, 2, 64), cache(rows=1).expand(3, 20, 2, 64)
    refused(evict, k=shared)                                                            # in place, all sessions in one
    refused(evict, k=flat)
    refused(evict, k=flat, **outs)
    reaches_the_library(evict, k=shared, w=w[:1].expand(3, 2, 20), positions=p[:1].expand(3, 2, 20), **outs)
    refused(evict, w=w[:1].expand(3, 2, 20))
    refused(evict, w=w[:, :1].expand(3, 2, 20))
    refused(evict, positions=p[:1].expand(3, 2, 20))
    for name in outs:
        t = outs[name]
        refused(evict, positions=p, **{**outs, name: t[:1].expand_as(t)})
    for name in ("weights_out", "positions_out"):
        refused(evict, positions=p, **{name: outs[name][:, :1].expand_as(outs[name])})
    for name in ("k_out", "v_out"):
        refused(evict, **{name: cache(rows=1).expand(3, 8, 2, 64)})


@pytest.mark.parametrize("bad", [-1, 2 ** 32, 2 ** 32 + 64, -2 ** 32 + 64, 1.5, None, "4"])
def test_counts_that_32_bits_do_not_hold(bad):
    k, q, w = cache(), queries(), torch.zeros(3, 2, 20)
    sink = attention().encode_sink_window
    refused(sink, sessions(), 64, 8, 2, bad, 8)
    refused(sink, sessions(), 64, 8, 2, 4, bad)
    refused(sink, sessions(), 64, 8, 2, 4, 8, ring_capacity=bad)
    for i in range(3):
        refused(tt.evict_kv_rows, HostContext(), k, k, w, 20, *[bad if i == x else 2 + 4 * (x == 0) for x in range(3)])
    p = tt.PrefillAttentionParams(0, 3, 64, 8, 2, 3, 8, 128, 512, 512, 0.125)
    prefill = tt.PrefillAttention(HostContext()).encode_sink_window
    reaches_the_library(prefill, q, k, k, q, p, 4)
    refused(prefill, q, k, k, q, p, bad)
    refused(prefill, q, k, k, q, p, 4, kv_ring_capacity=bad)


def test_counts_of_other_integer_types():
    import numpy as np
    reaches_the_library(attention().encode_sink_window, sessions(), 64, 8, 2, np.int64(4), torch.tensor(8), ring_capacity=np.uint32(16))
    reaches_the_library(tt.evict_kv_rows, HostContext(), cache(), cache(), torch.zeros(3, 2, 20), 20, np.int32(8), np.int64(1), True)


class ElsewhereTensor:
    """What a list of sessions looks at in a tensor, on a device of its own."""
    dtype = H

    def __init__(self, device):
        self.get_device = lambda: device

    def data_ptr(self):
        return 1 << 20


def test_lists_over_tensors_of_another_device():
    a, here, there = attention(), ElsewhereTensor(-1), ElsewhereTensor(1)

    def session(**kw):
        return tt.DecodeSession(**{**dict(q=here, out=here, k=here, v=here, seq_len=4), **kw})
    reaches_the_library(a.encode_sink_window, [session()], 64, 8, 2, 4, 8)
    reaches_the_library(a.encode_sink_window, [session(q=1 << 20, out=1 << 20, k=1 << 20, v=1 << 20)], 64, 8, 2, 4, 8)       # addresses
    weights = torch.zeros(2, 2, 20)
    prefix = [tt.PrefixGroup(here, here, 7, 2)]
    reaches_the_library(a.encode_shared_prefix, prefix, [session()] * 2, 64, 8, 2)
    for name in ("q", "out", "k", "v"):
        some = [session(), session(**{name: there})]
        refused(a.encode_sink_window, some, 64, 8, 2, 4, 8)
        refused(a.encode_accumulate, some, weights, 64, 8, 2)
        refused(a.encode_shared_prefix, prefix, some, 64, 8, 2)
    refused(a.encode_shared_prefix, [tt.PrefixGroup(there, here, 7, 1), tt.PrefixGroup(here, here, 7, 1)], [session()] * 2, 64, 8, 2)
    refused(a.encode_shared_prefix, [tt.PrefixGroup(here, there, 7, 2)], [session()] * 2, 64, 8, 2)


def test_lists_with_lengths_that_32_bits_do_not_hold():
    a, k = attention(), cache()
    for bad in (-1, 2 ** 32, None):
        refused(a.encode_sink_window, [tt.DecodeSession(k, k, k, k, bad)], 64, 8, 2, 4, 8)
        refused(a.encode_sink_window, [tt.DecodeSession(k, k, k, k, 4, q_rows=bad)], 64, 8, 2, 4, 8)
        refused(a.encode_shared_prefix, [tt.PrefixGroup(k, k, bad, 1)], [tt.DecodeSession(k, k, k, k, 4)], 64, 8, 2)


def test_plain_decode_takes_session_tables():
    a = attention()
    reaches_the_library(a.encode_batched, sessions(), 64, 8, 2)
    refused(a.encode_batched, sessions(), 64, 8, 4)
    refused(a.encode_batched, sessions(lens=21), 64, 8, 2)
    words, n, p = a.prepare_batch(sessions(cache(pad=1), queries(rows=2), lens=[4, 5, 6]), 64, 8, 2)
    assert n == 3 and [s.seq_len for s in words] == [4, 5, 6] and {s.q_rows for s in words} == {2}
    assert (p.kv_token_stride_elements, p.q_row_stride_elements, p.io_dtype) == (192, 512, tt.TT_F16)
    assert a.prepare_batch(sessions(torch.zeros(0, 20, 2, 64, dtype=H), queries(0)), 64, 8, 2)[1] == 0


def test_evictions_into_one_buffer_are_refused():
    k, v, w, one = cache(), cache(), torch.zeros(3, 2, 20), cache(rows=8)

    def evict(k, v, **kw):
        tt.evict_kv_rows(HostContext(), k, v, w, 20, 8, **kw)
    refused(evict, k, v, k_out=one, v_out=one)
    refused(evict, k, v, k_out=v)
    refused(evict, k, v, v_out=k)
    reaches_the_library(evict, k, k)                             # keys that are the values too
    reaches_the_library(evict, k, k, k_out=one, v_out=one)
    reaches_the_library(evict, k, v, k_out=k, v_out=v)
    reaches_the_library(evict, k, v, k_out=one)
