"""Host-side mirror of the reference's attention operator classes over the C ABI.

The classes keep the names, argument meaning and error behaviour of the Swift operators they
stand in for, so call sites and tests read like the reference's:

  Attention         sources/TinyTitan/Kernels/Attention/Attention.swift:270-470
  PrefillAttention  sources/TinyTitan/Kernels/Attention/PrefillAttention.swift:5-55, :165-258
  GDN               sources/TinyTitan/Kernels/GDN/GDN.swift:318-396

A "buffer" is a torch CUDA tensor or an integer device address; `*_offset` arguments are byte
offsets as in the reference. `command_buffer` is the CUDA stream handle (default: torch's
current stream); every encode* call enqueues and returns.
"""
from __future__ import annotations

import ctypes as C
import math
import operator
from array import array
from dataclasses import dataclass
from typing import Optional, Sequence

import numpy as np

from . import _lib as L


def _addr(buf, offset: int = 0) -> int:
    if buf is None:
        return 0
    base = buf.data_ptr() if hasattr(buf, "data_ptr") else int(buf)
    return base + int(offset)


def _stream(command_buffer) -> int:
    if command_buffer is not None:
        return int(getattr(command_buffer, "cuda_stream", command_buffer))
    import torch
    return int(torch.cuda.current_stream().cuda_stream)


def _dtype_of(buf, default=L.TT_F16) -> int:
    dt = getattr(buf, "dtype", None)
    if dt is None:
        return default
    import torch
    if dt == torch.bfloat16:
        return L.TT_BF16
    return L.TT_F16


class Context:
    """One per device and per runner: device scratch allocated once, not re-entrant."""

    def __init__(self, device: int = 0, workspace_bytes: int = 0, max_sessions: int = 0):
        err = C.c_int(0)
        opts = L.ContextOptions(workspace_bytes, max_sessions, 0)
        self.handle = L.lib().tt_context_create(device, C.byref(opts), C.byref(err))
        if not self.handle:
            L.check(err.value or L.TT_ERR_CUDA)
            raise L.TinyTitanError(L.TT_ERR_CUDA, "tt_context_create failed")
        self.device = device

    def close(self):
        if getattr(self, "handle", None):
            L.lib().tt_context_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def check(self, status: int):
        L.check(status, self.handle)

    def poll_status(self, command_buffer=None) -> int:
        flags = C.c_uint32(0)
        self.check(L.lib().tt_ctx_poll_status(self.handle, _stream(command_buffer), C.byref(flags)))
        return flags.value

    def synchronize(self, command_buffer=None):
        self.check(L.lib().tt_stream_synchronize(self.handle, _stream(command_buffer)))

    PROFILE_DECODE_PARTIAL = 1
    PROFILE_GDN_STEP = 2
    PROFILE_EXCHANGE = 4

    def profile_enable(self, enabled=True):
        """`enabled`: False/0 off, True/1 the split-KV pass-1 kernel, or a mask of PROFILE_*."""
        self.check(L.lib().tt_ctx_profile_enable(self.handle, int(enabled)))

    def profile_collect(self):
        """Durations (ms), in launch order, of the profiled launches recorded since the last collect."""
        buf = (C.c_float * 256)()
        n = C.c_uint32(0)
        self.check(L.lib().tt_ctx_profile_collect(self.handle, buf, 256, C.byref(n)))
        return [buf[i] for i in range(n.value)]

    def set_exchange_poll_limit(self, polls: int):
        """Polls (~0.25 us each) the exchange kernels wait for peers before giving up; 0 = default."""
        self.check(L.lib().tt_ctx_set_exchange_poll_limit(self.handle, polls))

    def stream(self, command_buffer=None) -> int:
        """The stream handle of a call: `command_buffer`, else torch's current stream of THIS context's device."""
        if command_buffer is not None:
            return int(getattr(command_buffer, "cuda_stream", command_buffer))
        raw = self.__dict__.get("_raw_stream")      # the handle without a Stream object: 0.2 us instead of 1.4
        if raw is not None:
            return raw(self.device)
        import torch
        now = torch.cuda.current_stream(self.device).cuda_stream
        self._raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
        return now

    def check_device(self, *holders):
        """Refuses tensors (or tables over tensors) that are not on this context's device. Raw addresses pass."""
        for t in holders:
            get = getattr(t, "get_device", None)            # CUDA index, -1 on the host
            if get is not None and get() not in (self.device, None):
                _refuse(f"a buffer is on device {get()}, the context on cuda:{self.device}")

    @property
    def launch_count(self) -> int:
        return int(L.lib().tt_ctx_launch_count(self.handle))


@dataclass
class KVFormat:
    bits: int = 16
    stride: int = 0
    value_bytes: int = 0
    group_size: int = 64


@dataclass
class AttentionSplitGeometry:
    effective_length: int
    num_chunks: int
    chunk_length: int
    partial_threadgroups: int
    use_swa_grouped_partial: bool


@dataclass
class DecodeSession:
    """One row group of a batched / few-token decode step (tt_attn_session)."""
    q: object
    out: object
    k: object
    v: object
    seq_len: int
    q_rows: int = 1
    kv_start: int = 0
    q_offset: int = 0
    out_offset: int = 0
    k_offset: int = 0
    v_offset: int = 0


@dataclass
class PrefixGroup:
    """The shared prefix of the next `n_sessions` sessions of a call (tt_attn_prefix)."""
    k: object
    v: object
    prefix_len: int
    n_sessions: int
    k_offset: int = 0
    v_offset: int = 0


def _refuse(message: str):
    raise L.InvalidArgument(L.TT_ERR_INVALID_ARG, message)


def _device_of(buffers):
    """The device of those that are tensors (None: all are addresses)."""
    found = {t.get_device() for t in buffers if hasattr(t, "get_device")}
    if len(found) > 1:
        _refuse(f"the buffers of a call are on devices {sorted(found)}")
    return found.pop() if found else None


def _pair(what: str, a, b):
    """Of two [batch, rows, heads, head_dim] tensors of one shape, type and device with tight rows: the shape and their
    strides."""
    shape, s, t = a.shape, a.stride(), b.stride()
    if b.shape != shape or len(shape) != 4 or s[3] != 1 or t[3] != 1 or s[2] != shape[3] or t[2] != shape[3]:
        _refuse(f"{what} must be [batch, rows, heads, head_dim] of one shape with tight rows")
    if shape[1] > 1 and (s[1] < shape[2] * shape[3] or t[1] < shape[2] * shape[3]):
        _refuse(f"the rows of {what} overlap")
    if b.dtype is not a.dtype or a.get_device() != b.get_device():
        _refuse(f"{what} must share one dtype and one device")
    return shape, s, t


def _check_apart(what: str, n: int, *steps):
    """Refuses results of n sessions that lie in one place (an expanded tensor)."""
    if n > 1 and 0 in steps:
        _refuse(f"the sessions share {what}")


def _half_dtype(what: str, dtype) -> int:
    name = str(dtype)
    if name == "torch.float16":
        return L.TT_F16
    if name != "torch.bfloat16":
        _refuse(f"{what} must be fp16 or bf16, not {name}")
    return L.TT_BF16


def _counts(name: str, values, n: int) -> array:
    """n numbers in 0..2^32-1 from a sequence, or from one int for all."""
    try:
        if isinstance(values, int):
            found = array("I", (values,)) * n
        else:
            found = array("I", values if isinstance(values, list) else [int(x) for x in values])
    except (OverflowError, TypeError):
        found = None
    if found is None or len(found) != n:
        _refuse(f"{name} must be {n} numbers in 0..2^32-1")
    return found


def _count(name: str, value) -> int:
    """A number in 0..2^32-1, which is what ctypes would make of any other without a word."""
    if type(value) is int and 0 <= value <= 0xffffffff:
        return value
    try:
        found = operator.index(value)
    except TypeError:
        found = -1
    if not 0 <= found <= 0xffffffff:
        _refuse(f"{name} must be in 0..2^32-1, not {value!r}")
    return found


def _block(n: int, places, lows: array, highs, spare=0, indices=None) -> array:
    """n records of 64-bit words as the C structures lay them out: for every (address, step) of `places` address + i * step (or
    + indices[i] * step), one word of two 32-bit numbers (`highs`: an array too, or one int), `spare` zero words."""
    one = isinstance(highs, int)
    if n <= 3 or indices is not None:   # up to three records Python is as fast as the call below
        flat, rest = [], [0] * spare
        for i in range(n):
            if indices is None:
                flat += [address + i * step for address, step in places]
            else:                       # per place, None for i itself
                flat += [p[0] + int(i if which is None else which[i]) * p[1] for p, which in zip(places, indices)]
            flat.append(lows[i] | (highs if one else highs[i]) << 32)
            flat += rest
        return array("Q", flat)
    width = len(places)
    block = array("Q", bytes(8 * n * (width + 1 + spare)))
    at = array("Q", [p[0] for p in places] + [p[1] for p in places])
    L.lib().tt_table_fill(block.buffer_info()[0], n, width, spare, at.buffer_info()[0], lows.buffer_info()[0],
                          None if one else highs.buffer_info()[0], highs if one else 0)
    return block


def _pointer(words: array) -> int:
    return words.buffer_info()[0]


class SessionTable:
    """The sessions of a batched decode call as one block of tt_attn_session, built from whole tensors.

    Call sites whose sessions live in the slots of one cache build the block without a Python object per
    session; it is accepted wherever a list of DecodeSession is. The tensors must outlive the call."""

    record = np.dtype([("q", "u8"), ("out", "u8"), ("k", "u8"), ("v", "u8"), ("seq_len", "u4"), ("q_rows", "u4"),
                       ("kv_start", "u4"), ("reserved", "u4")])

    def __init__(self, words, longest=0, kv_stride=None, q_stride=None, out_stride=None, io_dtype=None, capacity=None, device=None,
                 heads=None):
        self.words, self.longest, self.kv_stride, self.q_stride, self.out_stride = words, longest, kv_stride, q_stride, out_stride
        self.io_dtype, self.capacity, self.device = io_dtype, capacity, device
        self.heads = heads              # over whole tensors: (head_dim, n_q_heads, n_kv_heads)

    def __len__(self):
        return len(self.words) // 6

    def get_device(self):
        return self.device

    @property
    def records(self):
        return np.frombuffer(self.words, dtype=self.record)

    @property
    def pointer(self) -> int:
        return self.words.buffer_info()[0]

    @classmethod
    def over_cache(cls, q, out, k, v, seq_lens, slots=None) -> "SessionTable":
        """q, out: [n, q_rows, n_q_heads, head_dim]; k, v: [slots, capacity, n_kv_heads, head_dim], session i in
        slot i or slots[i]; seq_lens[i] keys are visible to the last of its rows."""
        q_shape, q_strides, out_strides = _pair("q and out", q, out)
        k_shape, k_strides, v_strides = _pair("k and v", k, v)
        device, io_dtype = k.get_device(), _half_dtype("q, out, k and v", q.dtype)
        if k.dtype is not q.dtype or q.get_device() != device or v_strides[1] != k_strides[1]:
            _refuse("q and k must share one dtype and one device, and v be laid out like k")
        n, q_rows = q_shape[0], q_shape[1]
        _check_apart("out", n, out_strides[0])
        if slots is None:
            if k_shape[0] < n:
                _refuse(f"{n} sessions, but the cache has {k_shape[0]} slots")
        elif len(slots) != n or (n and not (0 <= min(slots) and max(slots) < k_shape[0])):
            _refuse(f"slots must name {n} of the cache's {k_shape[0]} slots")
        lens = _counts("seq_lens", seq_lens, n)
        places = ((q.data_ptr(), 2 * q_strides[0]), (out.data_ptr(), 2 * out_strides[0]),
                  (k.data_ptr(), 2 * k_strides[0]), (v.data_ptr(), 2 * v_strides[0]))
        words = _block(n, places, lens, q_rows, 1, None if slots is None else (None, None, slots, slots))
        if q_shape[3] != k_shape[3]:
            _refuse(f"q has heads of {q_shape[3]}, k of {k_shape[3]}")
        kv_stride = k_strides[1] if k_shape[1] > 1 else None                       # one row has no stride
        q_stride, out_stride = (q_strides[1], out_strides[1]) if q_rows > 1 else (None, None)
        return cls(words, max(lens, default=0), kv_stride, q_stride, out_stride, io_dtype, k_shape[1], device,
                   (k_shape[3], q_shape[2], k_shape[2]))

    @classmethod
    def of(cls, sessions) -> "SessionTable":
        if isinstance(sessions, cls):
            return sessions
        words = array("Q", bytes(48 * len(sessions)))
        r = np.frombuffer(words, dtype=cls.record)
        for i, s in enumerate(sessions):
            r[i] = (_addr(s.q, s.q_offset), _addr(s.out, s.out_offset), _addr(s.k, s.k_offset), _addr(s.v, s.v_offset),
                    _count("seq_len", s.seq_len), _count("q_rows", s.q_rows), _count("kv_start", s.kv_start), 0)
        return cls(words, max((s.seq_len for s in sessions), default=0),
                   io_dtype=_dtype_of(sessions[0].q) if len(sessions) else None,
                   device=_device_of(t for s in sessions for t in (s.q, s.out, s.k, s.v)))

    def params(self, attention, head_dim, num_q_heads, num_kv_heads, kv_token_stride_elements, q_row_stride_elements,
               out_row_stride_elements, scale, io_dtype) -> "L.AttnBatchParams":
        tight_q = num_q_heads * head_dim
        dtype = io_dtype if io_dtype is not None else self.io_dtype
        if self.heads is not None:      # the call may repeat what the tensors say, not contradict it
            if self.heads != (head_dim, num_q_heads, num_kv_heads):
                _refuse("the tensors have heads of %d, %d of q, %d of k; " % self.heads + f"the call {head_dim}, {num_q_heads}, {num_kv_heads}")
            if dtype != self.io_dtype:
                _refuse("io_dtype is not the type of the tensors")
            for name, given, known in (("kv_token", kv_token_stride_elements, self.kv_stride), ("q_row", q_row_stride_elements, self.q_stride),
                                       ("out_row", out_row_stride_elements, self.out_stride)):
                if given and known and given != known:
                    _refuse(f"{name}_stride_elements {given}, but the tensors' rows are {known} apart")
        return L.AttnBatchParams(head_dim, num_q_heads, num_kv_heads,
                                 kv_token_stride_elements or self.kv_stride or num_kv_heads * head_dim,
                                 q_row_stride_elements or self.q_stride or tight_q,
                                 out_row_stride_elements or self.out_stride or tight_q,
                                 attention.default_scale(head_dim) if scale is None else scale,
                                 dtype if dtype is not None else L.TT_F16)

    def check_capacity(self, rows=None):
        """Refuses sessions that reach past their slot; `rows`: the rows a ring cache has."""
        need = self.longest if rows is None else min(self.longest, rows)
        if self.capacity is not None and need > self.capacity:
            _refuse(f"a session needs {need} rows, its slot has {self.capacity}")


class PrefixTable:
    """The groups of a shared-prefix call as one block of tt_attn_prefix."""

    record = np.dtype([("k", "u8"), ("v", "u8"), ("prefix_len", "u4"), ("n_sessions", "u4")])

    def __init__(self, words, device=None, kv_stride=None, io_dtype=None, heads=None):
        self.words, self.device = words, device
        self.kv_stride, self.io_dtype, self.heads = kv_stride, io_dtype, heads      # heads: (n_kv_heads, head_dim)

    def __len__(self):
        return len(self.words) // 3

    def get_device(self):
        return self.device

    @property
    def records(self):
        return np.frombuffer(self.words, dtype=self.record)

    @property
    def pointer(self) -> int:
        return self.words.buffer_info()[0]

    @classmethod
    def over_cache(cls, k, v, prefix_lens, n_sessions) -> "PrefixTable":
        """k, v: [groups, capacity, n_kv_heads, head_dim]; n_sessions: per group, or one number for all."""
        shape, k_strides, v_strides = _pair("k and v", k, v)
        io_dtype = _half_dtype("k and v", k.dtype)
        if v_strides[1] != k_strides[1]:
            _refuse("v must be laid out like k")
        g = shape[0]
        lens, counts = _counts("prefix_lens", prefix_lens, g), _counts("n_sessions", n_sessions, g)
        if max(lens, default=0) > shape[1]:
            _refuse(f"a prefix is longer than the {shape[1]} rows of its slot")
        words = _block(g, ((k.data_ptr(), 2 * k_strides[0]), (v.data_ptr(), 2 * v_strides[0])), lens, counts)
        return cls(words, k.get_device(), k_strides[1] if shape[1] > 1 else None, io_dtype, (shape[2], shape[3]))

    def check_rows(self, p: "L.AttnBatchParams"):
        """Refuses a call that would read the prefixes' rows by another stride, type or number of heads than they have."""
        if self.heads is None:
            return
        if self.kv_stride not in (None, p.kv_token_stride_elements):
            _refuse(f"the prefixes' rows are {self.kv_stride} elements apart, the sessions' {p.kv_token_stride_elements}")
        if self.io_dtype != p.io_dtype:
            _refuse("the prefixes and the sessions must share one dtype")
        if self.heads != (p.n_kv_heads, p.head_dim):
            _refuse(f"the prefixes have {self.heads[0]} heads of {self.heads[1]}, the call {p.n_kv_heads} of {p.head_dim}")

    @classmethod
    def of(cls, groups) -> "PrefixTable":
        if isinstance(groups, cls):
            return groups
        words = array("Q", bytes(24 * len(groups)))
        r = np.frombuffer(words, dtype=cls.record)
        for i, g in enumerate(groups):
            r[i] = (_addr(g.k, g.k_offset), _addr(g.v, g.v_offset), _count("prefix_len", g.prefix_len), _count("n_sessions", g.n_sessions))
        return cls(words, _device_of(t for g in groups for t in (g.k, g.v)))


class Attention:
    max_q_heads = 96
    max_head_dim = 512

    def __init__(self, context: Context):
        self.context = context

    @staticmethod
    def default_scale(head_dim: int) -> float:
        return 1.0 / math.sqrt(head_dim)

    @staticmethod
    def split_geometry(num_q_heads: int, num_kv_heads: int, seq_len: int, kv_start: int,
                       prefer_gqa_swa: bool) -> AttentionSplitGeometry:
        g = L.SplitGeometry()
        L.lib().tt_attn_reference_split_geometry(num_q_heads, num_kv_heads, seq_len, kv_start,
                                                 int(prefer_gqa_swa), C.byref(g))
        return AttentionSplitGeometry(g.effective_length, g.num_chunks, g.chunk_length,
                                      g.partial_threadgroups, bool(g.use_swa_grouped_partial))

    def _encode(self, command_buffer, q, q_offset, k, k_offset, v, v_offset, out, out_offset, head_dim,
                num_q_heads, num_kv_heads, seq_len, kv_start, scale, kv_format, keep_mask, ring_capacity):
        if num_kv_heads <= 0 or num_q_heads % num_kv_heads != 0:
            raise L.InvalidArgument(L.TT_ERR_INVALID_ARG, "numQHeads must be a multiple of numKVHeads for GQA")
        if head_dim > self.max_head_dim:
            raise L.InvalidArgument(L.TT_ERR_INVALID_ARG, "head_dim must be <= 512")
        fmt = None
        if kv_format is not None:
            fmt = L.KVFormat(kv_format.bits, kv_format.stride, kv_format.value_bytes, kv_format.group_size)
        sc = self.default_scale(head_dim) if scale is None else scale
        self.context.check(L.lib().tt_attn_decode(
            self.context.handle, _stream(command_buffer), _addr(q, q_offset), _addr(k, k_offset),
            _addr(v, v_offset), _addr(out, out_offset), head_dim, num_q_heads, num_kv_heads, seq_len, kv_start,
            sc, C.byref(fmt) if fmt is not None else None, _addr(keep_mask), ring_capacity))

    def encode_full(self, q, k, v, out, head_dim, num_q_heads, num_kv_heads, seq_len, scale=None,
                    kv_format: Optional[KVFormat] = None, keep_mask=None, command_buffer=None, q_offset=0,
                    k_offset=0, v_offset=0, out_offset=0):
        """Attention.encodeFull (Attention.swift:270-307)."""
        if seq_len <= 0:
            raise L.InvalidArgument(L.TT_ERR_INVALID_ARG, "full attention requires at least one KV position")
        self._encode(command_buffer, q, q_offset, k, k_offset, v, v_offset, out, out_offset, head_dim, num_q_heads,
                     num_kv_heads, seq_len, 0, scale, kv_format, keep_mask, 0)

    def encode_window(self, q, k, v, out, head_dim, num_q_heads, num_kv_heads, sel_rows, sel_count, scale=None,
                      kv_format: Optional[KVFormat] = None, command_buffer=None):
        """encodeFull(windowSelection:): attention over sel_count keys, key s at row sel_rows[s]."""
        fmt = None
        if kv_format is not None:
            fmt = L.KVFormat(kv_format.bits, kv_format.stride, kv_format.value_bytes, kv_format.group_size)
        self.context.check(L.lib().tt_attn_decode_window(
            self.context.handle, _stream(command_buffer), _addr(q), _addr(k), _addr(v), _addr(out), head_dim,
            num_q_heads, num_kv_heads, sel_count, self.default_scale(head_dim) if scale is None else scale,
            C.byref(fmt) if fmt is not None else None, _addr(sel_rows)))

    def encode_swa(self, q, k, v, out, head_dim, num_q_heads, num_kv_heads, seq_len, window, scale=None,
                   ring_capacity=0, kv_format: Optional[KVFormat] = None, command_buffer=None, q_offset=0,
                   k_offset=0, v_offset=0, out_offset=0):
        """Attention.encodeSWA (Attention.swift:233-266): keys [max(0, seqLen-window), seqLen)."""
        kv_start = seq_len - window if seq_len > window else 0
        self._encode(command_buffer, q, q_offset, k, k_offset, v, v_offset, out, out_offset, head_dim, num_q_heads,
                     num_kv_heads, seq_len, kv_start, scale, kv_format, None, ring_capacity)

    def encode_batched(self, sessions: Sequence[DecodeSession], head_dim, num_q_heads, num_kv_heads,
                       kv_token_stride_elements=None, q_row_stride_elements=None, out_row_stride_elements=None,
                       scale=None, io_dtype=None, command_buffer=None):
        """All rows of a batched decode / verify step in one launch pair (tt_attn_decode_batched)."""
        if isinstance(sessions, SessionTable):
            batch = self.prepare_batch(sessions, head_dim, num_q_heads, num_kv_heads, kv_token_stride_elements, q_row_stride_elements,
                                       out_row_stride_elements, scale, io_dtype)
            self.encode_prepared(batch, self.context.stream(command_buffer))
            return
        n = len(sessions)
        arr = (L.AttnSession * max(n, 1))()
        for i, s in enumerate(sessions):
            arr[i] = L.AttnSession(_addr(s.q, s.q_offset), _addr(s.out, s.out_offset), _addr(s.k, s.k_offset),
                                   _addr(s.v, s.v_offset), s.seq_len, s.q_rows, s.kv_start, 0)
        tight_q = num_q_heads * head_dim
        p = L.AttnBatchParams(head_dim, num_q_heads, num_kv_heads,
                              kv_token_stride_elements or num_kv_heads * head_dim,
                              q_row_stride_elements or tight_q, out_row_stride_elements or tight_q,
                              self.default_scale(head_dim) if scale is None else scale,
                              io_dtype if io_dtype is not None else (_dtype_of(sessions[0].q) if n else L.TT_F16))
        self.context.check(L.lib().tt_attn_decode_batched(self.context.handle, _stream(command_buffer), arr, n,
                                                          C.byref(p)))

    def prepare_batch(self, sessions: Sequence[DecodeSession], head_dim, num_q_heads, num_kv_heads,
                      kv_token_stride_elements=None, q_row_stride_elements=None, out_row_stride_elements=None,
                      scale=None, io_dtype=None):
        """The argument block of encode_batched built once, for a step that is replayed with the
        same buffers (the reference re-encodes the same bindings every token as well)."""
        if isinstance(sessions, SessionTable):
            t = self._table(sessions)
            t.check_capacity()
            p = t.params(self, head_dim, num_q_heads, num_kv_heads, kv_token_stride_elements, q_row_stride_elements,
                         out_row_stride_elements, scale, io_dtype)
            return ((L.AttnSession * max(len(t), 1)).from_buffer_copy(t.words if len(t) else bytes(C.sizeof(L.AttnSession))), len(t), p)
        n = len(sessions)
        arr = (L.AttnSession * max(n, 1))()
        for i, s in enumerate(sessions):
            arr[i] = L.AttnSession(_addr(s.q, s.q_offset), _addr(s.out, s.out_offset), _addr(s.k, s.k_offset),
                                   _addr(s.v, s.v_offset), s.seq_len, s.q_rows, s.kv_start, 0)
        tight_q = num_q_heads * head_dim
        p = L.AttnBatchParams(head_dim, num_q_heads, num_kv_heads,
                              kv_token_stride_elements or num_kv_heads * head_dim,
                              q_row_stride_elements or tight_q, out_row_stride_elements or tight_q,
                              self.default_scale(head_dim) if scale is None else scale,
                              io_dtype if io_dtype is not None else (_dtype_of(sessions[0].q) if n else L.TT_F16))
        return (arr, n, p)

    def encode_prepared(self, batch, command_buffer=None):
        arr, n, p = batch
        self.context.check(L.lib().tt_attn_decode_batched(self.context.handle, _stream(command_buffer), arr, n,
                                                          C.byref(p)))

    def _table(self, sessions) -> SessionTable:
        table = SessionTable.of(sessions)
        self.context.check_device(table)
        return table

    def encode_sink_window(self, sessions, head_dim, num_q_heads, num_kv_heads, sink_tokens, window, ring_capacity=0,
                           kv_token_stride_elements=None, q_row_stride_elements=None, out_row_stride_elements=None,
                           scale=None, io_dtype=None, command_buffer=None):
        """Decode / few-token attention over the first `sink_tokens` keys and the last `window` ones
        (tt_attn_decode_sink_window). `sessions`: DecodeSession list or SessionTable; with `ring_capacity` R a
        session's cache has sink_tokens + R rows and key j >= sink_tokens is row sink_tokens + (j - sink_tokens) % R."""
        t = self._table(sessions)
        sink_tokens, window, ring_capacity = _count("sink_tokens", sink_tokens), _count("window", window), _count("ring_capacity", ring_capacity)
        t.check_capacity(sink_tokens + ring_capacity if ring_capacity else None)
        p = t.params(self, head_dim, num_q_heads, num_kv_heads, kv_token_stride_elements, q_row_stride_elements,
                     out_row_stride_elements, scale, io_dtype)
        self.context.check(L.lib().tt_attn_decode_sink_window(
            self.context.handle, self.context.stream(command_buffer), t.pointer, len(t), C.byref(p), sink_tokens, window,
            ring_capacity))

    def encode_shared_prefix(self, groups, sessions, head_dim, num_q_heads, num_kv_heads, kv_token_stride_elements=None,
                             q_row_stride_elements=None, out_row_stride_elements=None, scale=None, io_dtype=None,
                             command_buffer=None):
        """Decode / few-token attention of sessions that continue shared prefixes (tt_attn_decode_shared_prefix).
        `groups`: PrefixGroup list or PrefixTable, each owning the next n_sessions of `sessions`, whose k, v and
        seq_len describe the rows behind the prefix. Prefix and session rows have one row stride."""
        t, g = self._table(sessions), PrefixTable.of(groups)
        self.context.check_device(g)
        t.check_capacity()
        if t.heads is not None and t.kv_stride is None:
            kv_token_stride_elements = kv_token_stride_elements or g.kv_stride
        p = t.params(self, head_dim, num_q_heads, num_kv_heads, kv_token_stride_elements, q_row_stride_elements,
                     out_row_stride_elements, scale, io_dtype)
        g.check_rows(p)
        self.context.check(L.lib().tt_attn_decode_shared_prefix(
            self.context.handle, self.context.stream(command_buffer), g.pointer, len(g), t.pointer, len(t), C.byref(p)))

    def encode_accumulate(self, sessions, weights, head_dim, num_q_heads, num_kv_heads, positions=None, fresh_rows=0,
                          end_positions=None, kv_token_stride_elements=None, q_row_stride_elements=None,
                          out_row_stride_elements=None, scale=None, io_dtype=None, command_buffer=None):
        """Decode / few-token attention that adds every key's attention weight to `weights`
        (tt_attn_decode_accumulate). weights: fp32 [n, n_kv_heads, rows]; positions: int32 like it, or None;
        fresh_rows, end_positions: one per session or one for all (end_positions default: the sessions' seq_len)."""
        t = self._table(sessions)
        t.check_capacity()
        n = len(t)
        head_stride, at = _statistic("weights", weights, "torch.float32", n, num_kv_heads, self.context)
        at_positions = (0, 0)
        if positions is not None:
            stride, at_positions = _statistic("positions", positions, "torch.int32", n, num_kv_heads, self.context)
            if stride != head_stride or positions.shape != weights.shape:
                _refuse("positions must be laid out like weights")
        if t.longest > weights.shape[2]:
            _refuse(f"a session is longer than a weight row of {weights.shape[2]}")
        ends = array("I", t.records["seq_len"].tolist()) if end_positions is None else _counts("end_positions", end_positions, n)
        words = _block(n, (at, at_positions), _counts("fresh_rows", fresh_rows, n), ends)      # tt_attn_weight_rows
        p = t.params(self, head_dim, num_q_heads, num_kv_heads, kv_token_stride_elements, q_row_stride_elements,
                     out_row_stride_elements, scale, io_dtype)
        self.context.check(L.lib().tt_attn_decode_accumulate(
            self.context.handle, self.context.stream(command_buffer), t.pointer, _pointer(words), n,
            C.byref(p), head_stride))

    def encode_pre(self, q_packed, q_out, gate_out, k_rows, q_norm_weight, k_norm_weight, head_dim, num_q_heads,
                   num_kv_heads, rotary_dim, theta, eps, position, rows=1, k_row_stride_elements=None,
                   command_buffer=None):
        """Split [query; gate], per-head q/k RMS norm, NeoX partial RoPE (encodeGatedFullPostProjection)."""
        self.context.check(L.lib().tt_attn_pre(
            self.context.handle, _stream(command_buffer), _addr(q_packed), _addr(q_out), _addr(gate_out), _addr(k_rows),
            _addr(q_norm_weight), _addr(k_norm_weight), head_dim, num_q_heads, num_kv_heads, rotary_dim, theta, eps,
            position, rows, k_row_stride_elements or num_kv_heads * head_dim))

    def encode_gate_mul(self, out, gate, count, command_buffer=None):
        """out *= sigmoid(gate): the full-attention output gate."""
        self.context.check(L.lib().tt_attn_gate_mul(self.context.handle, _stream(command_buffer), _addr(out),
                                                    _addr(gate), count))

    def encode_partial(self, q, k, v, head_dim, num_q_heads, num_kv_heads, seq_len, kv_start, m_out, d_out, o_out,
                       scale=None, kv_token_stride_elements=0, io_dtype=None, command_buffer=None):
        """Pass 1 alone: one unnormalised (m, d, o) triple per q head for this device's keys."""
        self.context.check(L.lib().tt_attn_decode_partial(
            self.context.handle, _stream(command_buffer), _addr(q), _addr(k), _addr(v), head_dim, num_q_heads,
            num_kv_heads, seq_len, kv_start, self.default_scale(head_dim) if scale is None else scale,
            kv_token_stride_elements, io_dtype if io_dtype is not None else _dtype_of(q), _addr(m_out), _addr(d_out),
            _addr(o_out)))

    def encode_combine(self, m, d, o, n_parts, num_q_heads, head_dim, out, io_dtype=None, command_buffer=None):
        """Pass 2 alone: log-sum-exp merge of n_parts triples."""
        self.context.check(L.lib().tt_attn_combine(
            self.context.handle, _stream(command_buffer), _addr(m), _addr(d), _addr(o), n_parts, num_q_heads,
            head_dim, _addr(out), io_dtype if io_dtype is not None else _dtype_of(out)))

    def encode_exchange_combine(self, m, d, o, exchange, num_q_heads, head_dim, out, io_dtype=None, command_buffer=None):
        """Cross-GPU merge in one kernel: this rank's triple goes to every rank's exchange buffer over
        peer memory, the kernel waits (bounded) for the others' and merges. `exchange` is a PeerExchange."""
        self.context.check(L.lib().tt_attn_exchange_combine(
            self.context.handle, _stream(command_buffer), _addr(m), _addr(d), _addr(o), exchange.pointer_array,
            exchange.rank, exchange.world, num_q_heads, head_dim, exchange.next_epoch(), _addr(out),
            io_dtype if io_dtype is not None else _dtype_of(out)))


    def encode_decode_exchange(self, q, k, v, head_dim, num_q_heads, num_kv_heads, seq_len, kv_start, exchange, out,
                               scale=None, kv_token_stride_elements=0, io_dtype=None, command_buffer=None):
        """One step of a session split over GPUs in two launches: pass 1 over this GPU's rows, then the
        local merge fused with the peer exchange and the cross-GPU merge."""
        x = L.AttnExchange(exchange.pointer_array, exchange.rank, exchange.world, exchange.next_epoch(), 0, _addr(out))
        self.context.check(L.lib().tt_attn_decode_exchange(
            self.context.handle, _stream(command_buffer), _addr(q), _addr(k), _addr(v), head_dim, num_q_heads,
            num_kv_heads, seq_len, kv_start, scale if scale is not None else head_dim ** -0.5,
            kv_token_stride_elements, io_dtype if io_dtype is not None else _dtype_of(q), C.byref(x)))


class PeerExchange:
    """One exchange buffer per rank, mapped into every rank of the group (one process per GPU, one node).

    `gather_handles(handle_bytes) -> list of every rank's handle bytes` is the host channel; with
    torch.distributed it is an all_gather_object."""

    def __init__(self, context: Context, rank: int, world: int, num_q_heads: int, head_dim: int, gather_handles):
        self.context, self.rank, self.world = context, rank, world
        self.bytes = L.lib().tt_attn_exchange_bytes(world, num_q_heads, head_dim)
        mine = C.c_void_p()
        handle = C.create_string_buffer(64)
        context.check(L.lib().tt_peer_buffer_create(context.handle, self.bytes, C.byref(mine), handle))
        self.local = mine.value
        handles = gather_handles(handle.raw)
        self.opened = []
        ptrs = []
        for r in range(world):
            if r == rank:
                ptrs.append(self.local)
                continue
            p = C.c_void_p()
            context.check(L.lib().tt_peer_buffer_open(context.handle, handles[r], C.byref(p)))
            self.opened.append(p.value)
            ptrs.append(p.value)
        self.pointer_array = (C.c_void_p * world)(*ptrs)
        self.epoch = 0

    def next_epoch(self) -> int:
        self.epoch += 1
        return self.epoch

    def close(self):
        """Unmap the peers' buffers and free this rank's (every rank must have stopped using them)."""
        for p in self.opened:
            L.lib().tt_peer_buffer_close(self.context.handle, p)
        self.opened = []
        if self.local:
            L.lib().tt_peer_buffer_destroy(self.context.handle, self.local)
            self.local = None


def quantize_kv_rows(context: Context, source, destination, element_count: int, bits: int, tokens: int,
                     source_stride_elements=None, destination_stride_bytes=None, values_bytes=None, group_size=64,
                     command_buffer=None, source_offset=0, destination_offset=0):
    """kv_cache_quantize_affine: fp16 rows -> the cache's packed row format (codes, scales, biases)."""
    packed = (element_count * bits + 7) // 8
    vb = values_bytes if values_bytes is not None else (packed + 1) & ~1
    groups = (element_count + group_size - 1) // group_size
    context.check(L.lib().tt_kv_quantize_affine(
        context.handle, _stream(command_buffer), _addr(source, source_offset), _addr(destination, destination_offset),
        source_stride_elements or element_count, destination_stride_bytes or vb + groups * 4, vb, element_count, bits,
        group_size, tokens))


def _statistic(name: str, t, dtype: str, n: int, num_kv_heads: int, context: Context, written: bool = True):
    """A [sessions, n_kv_heads, rows] tensor of one 32-bit number per cache row: elements between its heads, and
    (address, bytes between sessions)."""
    shape, stride = t.shape, t.stride()
    if str(t.dtype) != dtype or len(shape) != 3 or shape[0] < n or shape[1] != num_kv_heads or (shape[2] > 1 and stride[2] != 1):
        _refuse(f"{name} must be {dtype} [{n}, {num_kv_heads}, rows], rows contiguous")
    if num_kv_heads > 1 and stride[1] < shape[2]:
        _refuse(f"the heads of {name} overlap")
    if written:
        _check_apart(name, n, stride[0])
    if t.get_device() != context.device:
        context.check_device(t)
    return stride[1] if num_kv_heads > 1 else shape[2], (t.data_ptr(), 4 * stride[0])


_nowhere = (0, 0)


def evict_kv_rows(context: Context, k, v, weights, rows, budget: int, sink_tokens=0, recent_tokens=0, positions=None,
                  end_positions=None, k_out=None, v_out=None, weights_out=None, positions_out=None, command_buffer=None):
    """Keeps `budget` rows per KV head of every session's cache and compacts them (tt_kv_evict).

    k, v: [n, capacity, n_kv_heads, head_dim], the first rows[i] of slot i in use; weights: fp32 [n, n_kv_heads, *];
    positions: int32 like weights, None = row j holds position j; end_positions: position of the next token (default:
    rows). *_out: None for in place, or tensors of the same kind with room for min(rows, budget) rows. Afterwards
    session i has min(rows[i], budget) rows per head."""
    budget, sink_tokens, recent_tokens = _count("budget", budget), _count("sink_tokens", sink_tokens), _count("recent_tokens", recent_tokens)
    shape, k_strides, v_strides = _pair("k and v", k, v)
    _half_dtype("k and v", k.dtype)
    context.check_device(k)
    in_stride = k_strides[1]
    if v_strides[1] != in_stride:
        _refuse("v must be laid out like k")
    n, capacity, num_kv_heads, head_dim = shape
    used = _counts("rows", rows, n)
    most = max(used, default=0)
    kept = min(most, budget)
    if most > capacity:
        _refuse(f"a session has more rows than the {capacity} of its slot")
    # destinations of K and V
    if k_out is None:
        _check_apart("k", n, k_strides[0])
    if v_out is None:
        _check_apart("v", n, v_strides[0])
    out_stride, at_k, at_v = in_stride, _nowhere, _nowhere
    if k_out is not None or v_out is not None:
        a, b = (v_out if k_out is None else k_out), (k_out if v_out is None else v_out)
        room, a_strides, b_strides = _pair("k_out and v_out", a, b)
        out_stride = a_strides[1]
        if (a.dtype is not k.dtype or a.get_device() != k.get_device() or room[0] < n or room[1] < kept or room[2] != num_kv_heads or
                room[3] != head_dim or b_strides[1] != out_stride):
            _refuse(f"k_out and v_out must hold the kept rows of {n} sessions, in the layout of k and v")
        _check_apart("k_out or v_out", n, a_strides[0], b_strides[0])
        if k_out is not None:
            at_k = (k_out.data_ptr(), 2 * a_strides[0])
        if v_out is not None:
            at_v = (v_out.data_ptr(), 2 * b_strides[0])
    to_k, to_v = k if k_out is None else k_out, v if v_out is None else v_out
    if kept and to_k.data_ptr() == to_v.data_ptr() and k.data_ptr() != v.data_ptr():
        _refuse("K and V would go to one place")
    # the statistic and the positions, then where they go
    stat, at_w = _statistic("weights", weights, "torch.float32", n, num_kv_heads, context, weights_out is None)
    at_p, at_wo, at_po, stat_out = _nowhere, _nowhere, _nowhere, None
    if positions is not None:
        stride, at_p = _statistic("positions", positions, "torch.int32", n, num_kv_heads, context, positions_out is None)
        if stride != stat or positions.shape[2] < most:
            _refuse(f"positions must be laid out like weights and hold {most} rows")
    if weights.shape[2] < most:
        _refuse(f"weights must hold {most} rows")
    if weights_out is not None:
        stat_out, at_wo = _statistic("weights_out", weights_out, "torch.float32", n, num_kv_heads, context)
        if weights_out.shape[2] < kept:
            _refuse(f"weights_out must hold {kept} rows")
    if positions_out is not None:
        stride, at_po = _statistic("positions_out", positions_out, "torch.int32", n, num_kv_heads, context)
        if positions_out.shape[2] < kept or stat_out not in (None, stride):
            _refuse(f"positions_out must hold {kept} rows and be laid out like weights_out")
        stat_out = stride
    ends = used if end_positions is None else _counts("end_positions", end_positions, n)
    words = _block(n, ((k.data_ptr(), 2 * k_strides[0]), (v.data_ptr(), 2 * v_strides[0]), at_k, at_v, at_w, at_wo, at_p, at_po), used, ends)  # tt_kv_evict_session
    p = L.KVEvictParams(head_dim, num_kv_heads, budget, sink_tokens, recent_tokens, in_stride, out_stride, stat, stat_out or stat, 0)
    context.check(L.lib().tt_kv_evict(context.handle, context.stream(command_buffer), _pointer(words), n, C.byref(p)))


@dataclass
class PrefillAttentionParams:
    """PrefillAttentionParams (PrefillAttention.swift:5-55), same fields and defaults."""
    start_position: int
    query_count: int
    head_dim: int
    num_q_heads: int
    num_kv_heads: int
    kv_valid_count: int
    sliding_window: int
    kv_token_stride_elements: int
    q_token_stride_elements: int
    o_token_stride_elements: int
    scale: float
    kv_bits: int = 16
    kv_token_stride_bytes: int = 0
    kv_value_bytes: int = 0
    kv_group_size: int = 64

    def to_c(self) -> "L.PrefillParams":
        return L.PrefillParams(self.start_position, self.query_count, self.head_dim, self.num_q_heads,
                               self.num_kv_heads, self.kv_valid_count, self.sliding_window,
                               self.kv_token_stride_elements, self.q_token_stride_elements,
                               self.o_token_stride_elements, self.scale, self.kv_bits,
                               self.kv_token_stride_bytes, self.kv_value_bytes, self.kv_group_size)


class PrefillAttention:
    def __init__(self, context: Context):
        self.context = context

    def encode_causal(self, q, k, v, out, params: PrefillAttentionParams, kv_ring_capacity=0, io_dtype=None,
                      command_buffer=None, q_offset=0, k_offset=0, v_offset=0, out_offset=0, keep_mask=None,
                      keep_stride=0, keep_indices=None, keep_index_stride=0, keep_counts=None, keep_rows=None):
        """PrefillAttention.encodeCausal (PrefillAttention.swift:165-258); the keep* arguments are its
        per-query key selection (mask, compact index list with counts, window rows)."""
        cp = params.to_c()
        if keep_mask is not None or keep_indices is not None or keep_counts is not None or keep_rows is not None:
            self.context.check(L.lib().tt_attn_prefill_causal_selected(
                self.context.handle, _stream(command_buffer), _addr(q, q_offset), _addr(k, k_offset),
                _addr(v, v_offset), _addr(out, out_offset), C.byref(cp), kv_ring_capacity,
                io_dtype if io_dtype is not None else _dtype_of(q), _addr(keep_mask) or None, keep_stride,
                _addr(keep_indices) or None, keep_index_stride, _addr(keep_counts) or None, _addr(keep_rows) or None))
            return
        self.context.check(L.lib().tt_attn_prefill_causal(
            self.context.handle, _stream(command_buffer), _addr(q, q_offset), _addr(k, k_offset),
            _addr(v, v_offset), _addr(out, out_offset), C.byref(cp), kv_ring_capacity,
            io_dtype if io_dtype is not None else _dtype_of(q)))

    def encode_sink_window(self, q, k, v, out, params: PrefillAttentionParams, sink_tokens, kv_ring_capacity=0,
                           io_dtype=None, command_buffer=None, q_offset=0, k_offset=0, v_offset=0, out_offset=0):
        """Causal prefill over the first `sink_tokens` keys and a sliding window of params.sliding_window
        (tt_attn_prefill_sink_window); a ring lies behind the sinks' rows as in Attention.encode_sink_window."""
        self.context.check_device(q, k, v, out)
        sink_tokens, kv_ring_capacity = _count("sink_tokens", sink_tokens), _count("kv_ring_capacity", kv_ring_capacity)
        self.context.check(L.lib().tt_attn_prefill_sink_window(
            self.context.handle, self.context.stream(command_buffer), _addr(q, q_offset), _addr(k, k_offset),
            _addr(v, v_offset), _addr(out, out_offset), C.byref(params.to_c()), sink_tokens, kv_ring_capacity,
            io_dtype if io_dtype is not None else _dtype_of(q)))

    @staticmethod
    def sink_window_path(q, k, v, out, params: PrefillAttentionParams, kv_ring_capacity=0) -> str:
        path = L.lib().tt_attn_prefill_sink_path(_addr(q), _addr(k), _addr(v), _addr(out), C.byref(params.to_c()),
                                                 kv_ring_capacity)
        return "tcgen05" if path == 1 else "generic"

    @staticmethod
    def selected_path(q, k, v, out, params: PrefillAttentionParams, kv_ring_capacity=0, q_offset=0, k_offset=0,
                      v_offset=0, out_offset=0) -> str:
        cp = params.to_c()
        path = L.lib().tt_attn_prefill_path(_addr(q, q_offset), _addr(k, k_offset), _addr(v, v_offset),
                                            _addr(out, out_offset), C.byref(cp), kv_ring_capacity)
        return "tcgen05" if path == 1 else "generic"


@dataclass(frozen=True)
class SparseIndexerConfig:
    """SparseIndexerConfig of the reference's ArchConfig (ModelTypes.swift:129-133)."""
    num_heads: int = 4
    head_dim: int = 128
    budget: int = 2048
    compress_ratio: int = 4


class QSAIndexer:
    """Device side of QSAIndexer (sources/TinyTitan/Kernels/Attention/QSAIndexer.swift): pooled-key cache
    maintenance, block scores and the key selection. The caller owns the buffers (raw keys, pooled
    blocks, scores, selection), like the Swift class; projections are the caller's GEMVs."""

    def __init__(self, context: Context, config: SparseIndexerConfig, rope_theta: float = 1e7, eps: float = 1e-6,
                 budget: Optional[int] = None):
        self.context, self.config = context, config
        self.heads, self.head_dim, self.compress_ratio = config.num_heads, config.head_dim, config.compress_ratio
        self.budget = config.budget if budget is None else budget
        self.rope_theta, self.eps = rope_theta, eps

    @property
    def selection_width(self) -> int:
        """Cells a query keeps: the budget plus the tail block's extra members."""
        return self.budget + self.compress_ratio - 1

    def encode_pool(self, raw_keys, pooled, first_block, block_count, visible_keys, key_norm_weight=None,
                    command_buffer=None):
        """encodePoolPrefill / the repool of encodeAppendKey: pool + norm + rotation of a block range."""
        self.context.check(L.lib().tt_qsa_pool_blocks(
            self.context.handle, _stream(command_buffer), _addr(raw_keys), _addr(pooled), self.head_dim, first_block,
            block_count, self.compress_ratio, visible_keys, _addr(key_norm_weight) or None, self.eps, self.rope_theta))

    def encode_pool_prefill(self, raw_keys, pooled, start_position, tokens, key_norm_weight, command_buffer=None):
        first = start_position // self.compress_ratio
        last = (start_position + tokens - 1) // self.compress_ratio
        self.encode_pool(raw_keys, pooled, first, last - first + 1, start_position + tokens, key_norm_weight, command_buffer)

    def encode_append_key(self, raw_keys, pooled, position, key_norm_weight, command_buffer=None):
        """Repool the block token `position` joined (its raw key is already in the cache)."""
        self.encode_pool(raw_keys, pooled, position // self.compress_ratio, 1, position + 1, key_norm_weight, command_buffer)

    def encode_query(self, query, rows, position, query_norm_weight, command_buffer=None):
        self.context.check(L.lib().tt_qsa_query_norm_rope(
            self.context.handle, _stream(command_buffer), _addr(query), self.head_dim, self.heads, rows, position,
            _addr(query_norm_weight), self.eps, self.rope_theta))

    def encode_scores(self, query, pooled, scores, blocks, rows=1, score_stride=None, command_buffer=None):
        """encodeScores (rows = 1) / encodeScoresPrefill after the query's norm and rotation."""
        self.context.check(L.lib().tt_qsa_block_scores(
            self.context.handle, _stream(command_buffer), _addr(query), _addr(pooled), _addr(scores), self.head_dim,
            self.heads, blocks, rows, score_stride or blocks))

    def encode_select_keys(self, scores, score_stride, start_position, rows, keep=None, keep_stride=0, indices=None,
                           index_stride=0, counts=None, command_buffer=None):
        """encodeSelectKeys / selectKeysCompact (rows = 1) and selectKeysPrefill, mask and compact list at once."""
        self.context.check(L.lib().tt_qsa_select_keys(
            self.context.handle, _stream(command_buffer), _addr(scores), score_stride, start_position, rows,
            self.compress_ratio, self.selection_width, _addr(keep) or None, keep_stride, _addr(indices) or None,
            index_stride, _addr(counts) or None))


@dataclass(frozen=True)
class LinearAttentionConfig:
    """LinearAttentionConfig (sources/TinyTitanCore/Format/ModelTypes+Configs.swift:147-188)."""
    num_k_heads: int
    num_v_heads: int
    key_head_dim: int
    value_head_dim: int
    conv_kernel_size: int = 4

    @property
    def qkv_dim(self) -> int:
        return 2 * self.num_k_heads * self.key_head_dim + self.num_v_heads * self.value_head_dim

    @property
    def value_dim(self) -> int:
        return self.num_v_heads * self.value_head_dim


@dataclass
class GDNSession:
    conv_out: object
    a_proj: object
    b_proj: object
    state: object
    y: object
    checkpoint_state: object = None
    conv_out_offset: int = 0
    a_proj_offset: int = 0
    b_proj_offset: int = 0
    state_offset: int = 0
    y_offset: int = 0
    checkpoint_state_offset: int = 0


class GDN:
    def __init__(self, context: Context, config: LinearAttentionConfig, a_log_preexp=False, v_tiled=False,
                 readout_scale=1.0, gates_f32=False):
        self.context = context
        self.config = config
        flags = (L.TT_GDN_A_LOG_PREEXP if a_log_preexp else 0) | (L.TT_GDN_V_TILED if v_tiled else 0) | \
                (L.TT_GDN_GATES_F32 if gates_f32 else 0)
        self.shape = L.GdnShape(config.num_k_heads, config.num_v_heads, config.key_head_dim,
                                config.value_head_dim, flags, readout_scale)

    # ---- the elementwise kernels around the delta rule (GDN.swift:185-313, :399-427) ----
    def encode_conv_decode(self, tail, qkv, conv_weight, out, command_buffer=None, tail_offset=0, qkv_offset=0,
                           conv_weight_offset=0, out_offset=0):
        """GDN.encodeConvDecode: conv + SiLU of one row, the tail shifted in place."""
        self.context.check(L.lib().tt_gdn_conv_mix(
            self.context.handle, _stream(command_buffer), _addr(tail, tail_offset), _addr(qkv, qkv_offset),
            _addr(conv_weight, conv_weight_offset), _addr(out, out_offset), self.config.qkv_dim,
            self.config.conv_kernel_size, 1, 1))

    def encode_decode_prologue(self, sessions, conv_weight, command_buffer=None):
        """encodeConvDecode + encodeQKNorm for a batch of sessions in one launch; `sessions` is a sequence of
        (tail, qkv, conv_out) buffers (tensors or device addresses)."""
        n = len(sessions)
        arr = (L.GdnPreSession * max(n, 1))()
        for i, (tail, qkv, conv_out) in enumerate(sessions):
            arr[i] = L.GdnPreSession(_addr(tail), _addr(qkv), _addr(conv_out))
        self.context.check(L.lib().tt_gdn_decode_pre(
            self.context.handle, _stream(command_buffer), arr, n, _addr(conv_weight), self.config.num_k_heads,
            self.config.key_head_dim, self.config.qkv_dim, self.config.conv_kernel_size))

    def encode_prefill_prologue(self, tail, qkv_rows, conv_weight, conv_out, rows, checkpoint_tail=None, update_tail=True,
                                command_buffer=None):
        """encodeConvPrefill + encodeConvTailCheckpoint + encodeConvTailUpdate + encodeQKNorm over a chunk of rows in
        one launch (bit-identical to the four separate calls)."""
        self.context.check(L.lib().tt_gdn_prefill_pre(
            self.context.handle, _stream(command_buffer), _addr(tail), _addr(qkv_rows), _addr(conv_weight),
            _addr(conv_out), _addr(checkpoint_tail) if checkpoint_tail is not None else None, self.config.num_k_heads,
            self.config.key_head_dim, self.config.qkv_dim, self.config.conv_kernel_size, rows, int(update_tail)))

    def encode_conv_prefill(self, tail, qkv_rows, conv_weight, out, rows, command_buffer=None, tail_offset=0,
                            qkv_rows_offset=0, conv_weight_offset=0, out_offset=0):
        """GDN.encodeConvPrefill: conv over [tail | chunk rows]; the tail is read-only here."""
        self.context.check(L.lib().tt_gdn_conv_mix(
            self.context.handle, _stream(command_buffer), _addr(tail, tail_offset), _addr(qkv_rows, qkv_rows_offset),
            _addr(conv_weight, conv_weight_offset), _addr(out, out_offset), self.config.qkv_dim,
            self.config.conv_kernel_size, rows, 0))

    def encode_conv_tail_update(self, tail, qkv_rows, rows, command_buffer=None, tail_offset=0, qkv_rows_offset=0):
        """GDN.encodeConvTailUpdate: tail := last (kernel-1) raw rows of [tail | chunk]."""
        self.context.check(L.lib().tt_gdn_conv_tail_update(
            self.context.handle, _stream(command_buffer), _addr(tail, tail_offset), _addr(qkv_rows, qkv_rows_offset),
            self.config.qkv_dim, self.config.conv_kernel_size, rows))

    def encode_conv_tail_checkpoint(self, tail, qkv, checkpoint, command_buffer=None, tail_offset=0, qkv_offset=0,
                                    checkpoint_offset=0):
        """GDN.encodeConvTailCheckpoint: the tail as it stands after row 0 alone."""
        self.context.check(L.lib().tt_gdn_conv_tail_checkpoint(
            self.context.handle, _stream(command_buffer), _addr(tail, tail_offset), _addr(qkv, qkv_offset),
            _addr(checkpoint, checkpoint_offset), self.config.qkv_dim, self.config.conv_kernel_size))

    def encode_qk_norm(self, conv_out, rows=1, row_stride=None, command_buffer=None, conv_out_offset=0):
        """GDN.encodeQKNorm: per-head RMS norm of the q and k slices, delta-rule scales folded in."""
        self.context.check(L.lib().tt_gdn_qk_norm(
            self.context.handle, _stream(command_buffer), _addr(conv_out, conv_out_offset), self.config.num_k_heads,
            self.config.key_head_dim, row_stride or self.config.qkv_dim, rows))

    def encode_gated_norm(self, y, z, norm_weight, out, rows=1, sigmoid_gate=False, command_buffer=None, y_offset=0,
                          z_offset=0, norm_weight_offset=0, out_offset=0):
        """GDN.encodeGatedNorm: rmsnorm(y) * weight * silu(z) (or sigmoid(z)) per value head."""
        self.context.check(L.lib().tt_gdn_gated_norm(
            self.context.handle, _stream(command_buffer), _addr(y, y_offset), _addr(z, z_offset),
            _addr(norm_weight, norm_weight_offset), _addr(out, out_offset), self.config.num_v_heads,
            self.config.value_head_dim, rows, int(sigmoid_gate)))

    def encode_delta_step_decode(self, conv_out, a_proj, b_proj, a_log, dt_bias, state, y, command_buffer=None,
                                 conv_out_offset=0, a_proj_offset=0, b_proj_offset=0, a_log_offset=0,
                                 dt_bias_offset=0, state_offset=0, y_offset=0):
        """GDN.encodeDeltaStepDecode (GDN.swift:318-347)."""
        self.encode_delta_step_prefill(conv_out, a_proj, b_proj, a_log, dt_bias, state, y, rows=1,
                                       command_buffer=command_buffer, conv_out_offset=conv_out_offset,
                                       a_proj_offset=a_proj_offset, b_proj_offset=b_proj_offset,
                                       a_log_offset=a_log_offset, dt_bias_offset=dt_bias_offset,
                                       state_offset=state_offset, y_offset=y_offset)

    def encode_delta_step_prefill(self, conv_out, a_proj, b_proj, a_log, dt_bias, state, y, rows,
                                  checkpoint_state=None, row_stride=None, command_buffer=None, conv_out_offset=0,
                                  a_proj_offset=0, b_proj_offset=0, a_log_offset=0, dt_bias_offset=0,
                                  state_offset=0, checkpoint_state_offset=0, y_offset=0):
        """GDN.encodeDeltaStepPrefill (GDN.swift:351-396): rows applied in order, exact arithmetic."""
        self.context.check(L.lib().tt_gdn_step(
            self.context.handle, _stream(command_buffer), _addr(conv_out, conv_out_offset),
            _addr(a_proj, a_proj_offset), _addr(b_proj, b_proj_offset), _addr(a_log, a_log_offset),
            _addr(dt_bias, dt_bias_offset), _addr(state, state_offset), _addr(y, y_offset), C.byref(self.shape),
            rows, row_stride or self.config.qkv_dim,
            _addr(checkpoint_state, checkpoint_state_offset) if checkpoint_state is not None else None))

    def encode_delta_step_batched(self, sessions: Sequence[GDNSession], a_log, dt_bias, rows=1, row_stride=None,
                                  command_buffer=None):
        n = len(sessions)
        arr = (L.GdnSession * max(n, 1))()
        for i, s in enumerate(sessions):
            arr[i] = L.GdnSession(_addr(s.conv_out, s.conv_out_offset), _addr(s.a_proj, s.a_proj_offset),
                                  _addr(s.b_proj, s.b_proj_offset), _addr(s.state, s.state_offset),
                                  _addr(s.y, s.y_offset),
                                  _addr(s.checkpoint_state, s.checkpoint_state_offset)
                                  if s.checkpoint_state is not None else None)
        self.context.check(L.lib().tt_gdn_step_batched(
            self.context.handle, _stream(command_buffer), arr, n, _addr(a_log), _addr(dt_bias),
            C.byref(self.shape), rows, row_stride or self.config.qkv_dim))

    def prepare_batch(self, sessions: Sequence[GDNSession]):
        n = len(sessions)
        arr = (L.GdnSession * max(n, 1))()
        for i, s in enumerate(sessions):
            arr[i] = L.GdnSession(_addr(s.conv_out, s.conv_out_offset), _addr(s.a_proj, s.a_proj_offset),
                                  _addr(s.b_proj, s.b_proj_offset), _addr(s.state, s.state_offset),
                                  _addr(s.y, s.y_offset),
                                  _addr(s.checkpoint_state, s.checkpoint_state_offset)
                                  if s.checkpoint_state is not None else None)
        return (arr, n)

    def encode_prepared(self, batch, a_log, dt_bias, rows=1, row_stride=None, command_buffer=None):
        arr, n = batch
        self.context.check(L.lib().tt_gdn_step_batched(
            self.context.handle, _stream(command_buffer), arr, n, _addr(a_log), _addr(dt_bias),
            C.byref(self.shape), rows, row_stride or self.config.qkv_dim))

    def encode_delta_scan_chunked(self, conv_out, a_proj, b_proj, a_log, dt_bias, state, y, rows, chunk=64,
                                  row_stride=None, command_buffer=None, state_offset=0):
        """Chunk-parallel form of encode_delta_step_prefill (tt_gdn_scan_chunked)."""
        self.context.check(L.lib().tt_gdn_scan_chunked(
            self.context.handle, _stream(command_buffer), _addr(conv_out), _addr(a_proj), _addr(b_proj),
            _addr(a_log), _addr(dt_bias), _addr(state, state_offset), _addr(y), C.byref(self.shape), rows,
            row_stride or self.config.qkv_dim, chunk))
