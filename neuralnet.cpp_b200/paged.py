"""The paged key-value cache and its operators over the C-ABI: appending, attention of one new token per sequence,
eviction by accumulated attention, and the adjustment of logits before sampling.

The operators become methods of Engine, like those of engine.py.  Unlike those they follow torch's current stream: where the
engine launches on another one, each call waits for the work enqueued so far and the current stream waits for the call.
"""
from __future__ import annotations

import ctypes as C

import torch

from ._lib import NnbError, check, lib
from .engine import BF16, F32, Engine

_DTYPES = {torch.float32: F32, torch.bfloat16: BF16}


class _Cache(C.Structure):
    _fields_ = [("d_k", C.c_void_p), ("d_v", C.c_void_p), ("d_weight", C.c_void_p), ("dtype", C.c_int32), ("n_pages", C.c_int32),
                ("page_size", C.c_int32), ("n_head_kv", C.c_int32), ("dk", C.c_int32)]


class _Seqs(C.Structure):
    _fields_ = [("d_table", C.c_void_p), ("d_len", C.c_void_p), ("n_seq", C.c_int32), ("max_pages", C.c_int32), ("table_stride", C.c_size_t)]


class _Tokens(C.Structure):
    _fields_ = [("d_q", C.c_void_p), ("d_k", C.c_void_p), ("d_v", C.c_void_p), ("d_q_out", C.c_void_p), ("q_stride", C.c_size_t),
                ("k_stride", C.c_size_t), ("v_stride", C.c_size_t), ("q_out_stride", C.c_size_t), ("dtype", C.c_int32), ("n_head", C.c_int32),
                ("n_rows", C.c_size_t), ("d_row_start", C.c_void_p), ("d_pos", C.c_void_p), ("d_rope_cos", C.c_void_p), ("d_rope_sin", C.c_void_p),
                ("rope_ctx", C.c_int32)]


class _Logits(C.Structure):
    _fields_ = [("d_history", C.c_void_p), ("history_stride", C.c_size_t), ("max_history", C.c_size_t), ("d_history_len", C.c_void_p),
                ("d_prompt_len", C.c_void_p), ("repeat_window", C.c_int32), ("d_repeat", C.c_void_p), ("d_presence", C.c_void_p),
                ("d_frequency", C.c_void_p), ("d_bias", C.c_void_p), ("bias_stride", C.c_size_t), ("d_allowed", C.c_void_p),
                ("allowed_stride", C.c_size_t)]


def _need(cond, text):
    if not cond:
        raise NnbError(text)


class PagedCache:
    """One layer's pool of pages: k and v (n_pages, n_head_kv, page_size, pitch) f32 or bf16 with pitch = dk rounded up to 8,
    and weight (n_pages, n_head_kv, page_size) f32 (the attention each position has received), or None."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, dk: int | None = None, weight: torch.Tensor | None = None):
        _need(k.dim() == 4 and k.shape == v.shape and k.dtype == v.dtype and k.dtype in _DTYPES,
              "keys and values are (n_pages, n_head_kv, page_size, pitch) tensors of one shape and type, f32 or bf16")
        dk = k.shape[3] if dk is None else int(dk)
        if k.shape[3] != (dk + 7) // 8 * 8:
            raise NnbError(f"a head size of {dk} needs rows of {(dk + 7) // 8 * 8} features, not {k.shape[3]}")
        _need(weight is None or (weight.shape == k.shape[:3] and weight.dtype == torch.float32), "weights are (n_pages, n_head_kv, page_size) f32")
        _need(k.is_cuda and k.is_contiguous() and v.is_contiguous() and v.device == k.device
              and (weight is None or (weight.is_contiguous() and weight.device == k.device)), "the cache consists of contiguous CUDA tensors of one device")
        self.k, self.v, self.weight, self.dk = k, v, weight, dk
        self.n_pages, self.n_head_kv, self.page_size, self.pitch = k.shape
        self._c = _Cache(k.data_ptr(), v.data_ptr(), weight.data_ptr() if weight is not None else None, _DTYPES[k.dtype], self.n_pages,
                         self.page_size, self.n_head_kv, dk)

    @classmethod
    def empty(cls, n_pages: int, n_head_kv: int, page_size: int, dk: int, dtype=torch.bfloat16, device="cuda", track_weight=False):
        """A zeroed pool."""
        shape = (n_pages, n_head_kv, page_size, (dk + 7) // 8 * 8)
        k, v = torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device)
        return cls(k, v, dk, torch.zeros(shape[:3], device=device) if track_weight else None)

    def row(self, table_row, head: int, pos: int) -> int:
        """Index of a position's row in k.view(-1, pitch), v and weight.view(-1), from its sequence's page ids; -1: it has no page."""
        ids = (C.c_int32 * len(table_row))(*[int(x) for x in table_row])
        return int(lib().nnb_paged_row(C.byref(self._c), ids, len(table_row), head, pos))


def _call(eng, fn, *args):
    """fn(engine, *args), ordered with torch's current stream where the engine launches on another one."""
    ptr = eng._lib.nnb_engine_stream(eng._h) or 0
    if ptr == torch._C._cuda_getCurrentRawStream(eng.device.index):
        check(fn(eng._h, *args))
        return
    cur = torch.cuda.current_stream(eng.device)
    own = torch.cuda.ExternalStream(ptr, device=eng.device) if ptr else torch.cuda.default_stream(eng.device)
    own.wait_stream(cur)
    try:
        check(fn(eng._h, *args))
    finally:
        cur.wait_stream(own)


# The checks below run on every call: one condition each, and messages only once it fails.
def _wrong(eng, name, t, dtype, shape):
    if t.device != eng.device:
        return NnbError(f"{name} is on {t.device}, the engine on {eng.device}")
    if t.dtype != dtype:
        return NnbError(f"{name} is {t.dtype}, not {dtype}")
    if shape is not None and t.shape != shape:
        return NnbError(f"{name} has shape {tuple(t.shape)}, not {tuple(shape)}")
    return NnbError(f"{name} is not contiguous")


def _flat(eng, name, t, dtype, shape):
    if t.dtype is dtype and t.shape == shape and t.is_contiguous() and t.device == eng.device:
        return t.data_ptr()
    raise _wrong(eng, name, t, dtype, shape)


def _matrix(eng, name, t, dtype):
    """(rows, cols) with contiguous rows"""
    if t.dim() == 2 and t.dtype is dtype and t.device == eng.device and (t.stride(1) == 1 or t.numel() == 0):
        return t.shape
    raise _wrong(eng, name, t, dtype, None) if t.dtype != dtype or t.device != eng.device else NnbError(f"{name} is a matrix with contiguous rows")


def _rows(eng, name, t, heads, dk, dtype):
    """(rows, heads, dk) with contiguous rows, any distance apart; returns the distance in elements."""
    shape = t.shape
    if len(shape) == 3 and shape[1] == heads and shape[2] == dk and t.dtype is dtype and t.device == eng.device:
        row, head, one = t.stride()
        if (one == 1 and (head == dk or heads == 1) and row >= 0) or t.numel() == 0:
            return row
        raise NnbError(f"the rows of {name} are not contiguous")
    raise _wrong(eng, name, t, dtype, (shape[0] if len(shape) else 0, heads, dk))


def _seqs(eng, cache, table, lengths):
    if cache.k.device != eng.device:
        raise NnbError(f"the cache is on {cache.k.device}, the engine on {eng.device}")
    n, cols = _matrix(eng, "table", table, torch.int32)
    return _Seqs(table.data_ptr(), _flat(eng, "lengths", lengths, torch.int32, (n,)), n, cols, table.stride(0) if n > 1 else cols)


def _heads(name, t):
    """the heads of a (rows, heads, dk) tensor, f32 or bf16"""
    if t.dim() != 3 or t.dtype not in _DTYPES:
        raise NnbError(f"{name} is a (rows, heads, dk) tensor, f32 or bf16")
    return t.shape[1]


def paged_append(self, cache, table, lengths, k, v, q=None, row_start=None, rope=None, positions=None, q_out=None, lengths_out=None):
    """New tokens into the cache: k, v (rows, n_head_kv, dk), q (rows, n_head, dk), rotated by rope = (cos, sin) at their
    positions (default: their place in the cache).  row_start (n_seq + 1): the rows of each sequence; None: one row per
    sequence, idle where its position is negative.  Returns (rotated q or None, new lengths); lengths_out may be lengths."""
    s = _seqs(self, cache, table, lengths)
    _heads("k", k)
    rows, n, io, dk = k.shape[0], s.n_seq, k.dtype, cache.dk
    ks, vs = _rows(self, "k", k, cache.n_head_kv, dk, io), _rows(self, "v", v, cache.n_head_kv, dk, io)
    if v.shape[0] != rows or (q is not None and q.shape[0] != rows):
        raise NnbError("q, k and v differ in rows")
    qs = q_ptr = out_ptr = out_stride = heads = start = pos = cos_ptr = sin_ptr = ctx = 0
    if q is not None:
        heads = _heads("q", q)
        qs, q_ptr = _rows(self, "q", q, heads, dk, io), q.data_ptr()
        if q_out is None:
            q_out, out_stride = torch.empty_like(q, memory_format=torch.contiguous_format), heads * dk
        else:
            out_stride = _rows(self, "q_out", q_out, heads, dk, io)
            if q_out.shape[0] != rows:
                raise NnbError("q_out and q differ in rows")
        out_ptr = q_out.data_ptr()
    else:
        q_out = None
    if row_start is not None:
        start = _flat(self, "row_start", row_start, torch.int32, (n + 1,))
    if positions is not None:
        pos = _flat(self, "positions", positions, torch.int32, (rows,))
    if rope is not None:
        cos, sin = rope
        ctx = cos.shape[0]
        cos_ptr, sin_ptr = _flat(self, "cos", cos, torch.float32, (ctx, dk // 2)), _flat(self, "sin", sin, torch.float32, (ctx, dk // 2))
    if lengths_out is None:
        lengths_out = torch.empty_like(lengths)
        len_ptr = lengths_out.data_ptr()
    else:
        len_ptr = _flat(self, "lengths_out", lengths_out, torch.int32, (n,))
    t = _Tokens(q_ptr, k.data_ptr(), v.data_ptr(), out_ptr, qs, ks, vs, out_stride, _DTYPES[io], heads, rows, start, pos, cos_ptr, sin_ptr, ctx)
    _call(self, self._lib.nnb_paged_append, C.byref(cache._c), C.byref(s), C.byref(t), len_ptr)
    return q_out, lengths_out


def paged_attention_decode(self, cache, table, lengths, q, scale=0.0, accumulate=False, out=None, lse=None):
    """Attention of one new token per sequence, q (n_seq, n_head, dk), over the `lengths` cached positions.  Returns
    (out (n_seq, n_head, dk) of q's type, lse (n_seq, n_head) f32); accumulate adds the attention weights to cache.weight."""
    s = _seqs(self, cache, table, lengths)
    n, heads, io = s.n_seq, _heads("q", q), q.dtype
    stride = _rows(self, "q", q, heads, cache.dk, io)
    if q.shape[0] != n:
        raise NnbError(f"{q.shape[0]} queries for {n} sequences")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    else:
        _flat(self, "out", out, io, q.shape)
    if lse is None:
        lse = torch.empty((n, heads), device=self.device, dtype=torch.float32)
    else:
        _flat(self, "lse", lse, torch.float32, (n, heads))
    accumulate, c, s = int(accumulate), C.byref(cache._c), C.byref(s)
    size = self._lib.nnb_paged_attention_workspace(self._h, c, s, heads, accumulate)
    ws = torch.empty(size, device=self.device, dtype=torch.uint8)
    _call(self, self._lib.nnb_paged_attention_decode, c, s, q.data_ptr(), _DTYPES[io], stride, heads, scale, out.data_ptr(), lse.data_ptr(), accumulate,
          ws.data_ptr(), size)
    return out, lse


def paged_evict(self, cache, table, lengths, dst, dst_table, budget, sinks=0, recent=0, lengths_out=None):
    """Copies, per KV head, the first `sinks`, the last `recent` and the heaviest other positions of every sequence, `budget`
    in all, into the pages of dst_table in the pool dst.  Returns the new lengths."""
    s = _seqs(self, cache, table, lengths)
    d = _seqs(self, dst, dst_table, lengths)
    if lengths_out is None:
        lengths_out = torch.empty_like(lengths)
    n_out = _flat(self, "lengths_out", lengths_out, torch.int32, (s.n_seq,))
    _need(budget >= 0 and sinks >= 0 and recent >= 0, "budget, sinks and recent are not negative")
    size = self._lib.nnb_paged_evict_workspace(self._h, C.byref(cache._c), C.byref(s), budget)
    ws = torch.empty(size, device=self.device, dtype=torch.uint8)
    _call(self, self._lib.nnb_paged_evict, C.byref(cache._c), C.byref(s), budget, sinks, recent, C.byref(dst._c), d.d_table, d.max_pages, d.table_stride,
          n_out, ws.data_ptr(), size)
    return lengths_out


def adjust_logits(self, logits, history=None, history_len=None, prompt_len=None, repeat_window=0, repeat_penalty=None, presence_penalty=None,
                  frequency_penalty=None, bias=None, allowed=None, out=None):
    """logits (n_seq, vocab) f32 or bf16 with a bias, penalties for the ids of history (n_seq, max_history) and a mask of
    allowed ids (one bit each, (n_seq, ceil(vocab / 32)) int32), in this order.  Penalties are (n_seq) f32, bias and allowed
    one row for all or one per sequence; out may be logits.  Returns out."""
    io = logits.dtype
    if io not in _DTYPES:
        raise NnbError("logits are f32 or bf16")
    n, vocab = _matrix(self, "logits", logits, io)
    if out is None:
        out = torch.empty_like(logits, memory_format=torch.contiguous_format)
    elif _matrix(self, "out", out, io) != logits.shape:
        raise NnbError(f"out has shape {tuple(out.shape)}, not {tuple(logits.shape)}")
    c = _Logits()
    c.repeat_window = repeat_window
    if history is None:
        _need(repeat_penalty is None and presence_penalty is None and frequency_penalty is None, "penalties need a history")
    else:
        rows, width = _matrix(self, "history", history, torch.int32)
        _need(rows == n and history_len is not None, "history has a row and a length for every sequence")
        f32, one = torch.float32, (n,)
        lens = _flat(self, "history_len", history_len, torch.int32, one)
        prompt = _flat(self, "prompt_len", prompt_len, torch.int32, one) if prompt_len is not None else 0
        rep = _flat(self, "repeat_penalty", repeat_penalty, f32, one) if repeat_penalty is not None else 0
        pres = _flat(self, "presence_penalty", presence_penalty, f32, one) if presence_penalty is not None else 0
        freq = _flat(self, "frequency_penalty", frequency_penalty, f32, one) if frequency_penalty is not None else 0
        if rows * width:  # with an empty one there is nothing to penalise
            c.d_history, c.history_stride, c.max_history, c.d_history_len = history.data_ptr(), history.stride(0), width, lens
            c.d_prompt_len, c.d_repeat, c.d_presence, c.d_frequency = prompt, rep, pres, freq
    for name, t, dtype, width in (("bias", bias, torch.float32, vocab), ("allowed", allowed, torch.int32, (vocab + 31) // 32)):
        if t is not None:
            if t.dtype != dtype or t.device != self.device:
                raise _wrong(self, name, t, dtype, None)
            if tuple(t.shape) not in ((width,), (n, width)) or t.stride(-1) != 1:
                raise NnbError(f"{name} is ({width}) or ({n}, {width}) with contiguous rows")
            setattr(c, "d_" + name, t.data_ptr())
            setattr(c, name + "_stride", t.stride(0) if t.dim() == 2 else 0)
    _call(self, self._lib.nnb_adjust_logits, logits.data_ptr(), _DTYPES[logits.dtype], n, vocab, logits.stride(0), C.byref(c), out.data_ptr(), out.stride(0))
    return out


for _f in (paged_append, paged_attention_decode, paged_evict, adjust_logits):
    setattr(Engine, _f.__name__, _f)
