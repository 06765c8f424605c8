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
        for t in (k, v) if weight is None else (k, v, weight):
            _need(t.is_cuda and t.is_contiguous() and t.device == k.device, "the cache consists of contiguous CUDA tensors of one device")
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


# The checks below run on every call: messages are only put together when one fails.
def _on(eng, name, t, dtype, shape=None):
    if t.device != eng.device:
        raise NnbError(f"{name} is on {t.device}, the engine on {eng.device}")
    if t.dtype != dtype:
        raise NnbError(f"{name} is {t.dtype}, not {dtype}")
    if shape is not None and t.shape != shape:
        raise NnbError(f"{name} has shape {tuple(t.shape)}, not {shape}")
    return t


def _flat(eng, name, t, dtype, shape):
    if not _on(eng, name, t, dtype, shape).is_contiguous():
        raise NnbError(f"{name} is not contiguous")
    return t.data_ptr()


def _rows(eng, name, t, heads=None, dk=None):
    """(rows, heads, dk) with contiguous rows, any distance apart; returns the distance in elements."""
    if t.device != eng.device:
        raise NnbError(f"{name} is on {t.device}, the engine on {eng.device}")
    shape = t.shape
    if len(shape) != 3 or t.dtype not in _DTYPES:
        raise NnbError(f"{name} is a (rows, heads, dk) tensor, f32 or bf16")
    if (heads is not None and shape[1] != heads) or (dk is not None and shape[2] != dk):
        raise NnbError(f"{name} has shape {tuple(shape)}")
    row, head, one = t.stride()
    if (one != 1 or (shape[1] != 1 and head != shape[2]) or row < 0) and t.numel():
        raise NnbError(f"the rows of {name} are not contiguous")
    return row


def _seqs(eng, cache, table, lengths):
    if cache.k.device != eng.device:
        raise NnbError(f"the cache is on {cache.k.device}, the engine on {eng.device}")
    if _on(eng, "table", table, torch.int32).dim() != 2 or (table.stride(1) != 1 and table.numel()):
        raise NnbError("table is (n_seq, max_pages) with contiguous rows")
    n, cols = table.shape
    return _Seqs(table.data_ptr(), _flat(eng, "lengths", lengths, torch.int32, (n,)), n, cols, table.stride(0) if n > 1 else cols)


def paged_append(self, cache, table, lengths, k, v, q=None, row_start=None, rope=None, positions=None, q_out=None, lengths_out=None):
    """New tokens into the cache: k, v (rows, n_head_kv, dk), q (rows, n_head, dk), rotated by rope = (cos, sin) at their
    positions (default: their place in the cache).  row_start (n_seq + 1): the rows of each sequence; None: one row per
    sequence, idle where its position is negative.  Returns (rotated q or None, new lengths); lengths_out may be lengths."""
    s = _seqs(self, cache, table, lengths)
    rows, n = k.shape[0], s.n_seq
    ks, vs = _rows(self, "k", k, cache.n_head_kv, cache.dk), _rows(self, "v", v, cache.n_head_kv, cache.dk)
    if v.shape[0] != rows or v.dtype != k.dtype:
        raise NnbError("k and v differ in rows or type")
    t = _Tokens(None, k.data_ptr(), v.data_ptr(), None, 0, ks, vs, 0, _DTYPES[k.dtype], 0, rows, None, None, None, None, 0)
    if q is not None:
        t.q_stride = _rows(self, "q", q, None, cache.dk)
        if q.shape[0] != rows or q.dtype != k.dtype:
            raise NnbError("q and k differ in rows or type")
        if q_out is None:
            q_out, t.q_out_stride = q.new_empty(q.shape), q.shape[1] * q.shape[2]
        else:
            t.q_out_stride = _rows(self, "q_out", q_out)
            if q_out.shape != q.shape or q_out.dtype != q.dtype:
                raise NnbError("q_out and q differ in shape or type")
        t.n_head, t.d_q, t.d_q_out = q.shape[1], q.data_ptr(), q_out.data_ptr()
    else:
        q_out = None
    if row_start is not None:
        t.d_row_start = _flat(self, "row_start", row_start, torch.int32, (n + 1,))
    if positions is not None:
        t.d_pos = _flat(self, "positions", positions, torch.int32, (rows,))
    if rope is not None:
        cos, sin = rope
        t.d_rope_cos = _flat(self, "cos", cos, torch.float32, (cos.shape[0], cache.dk // 2))
        t.d_rope_sin, t.rope_ctx = _flat(self, "sin", sin, torch.float32, tuple(cos.shape)), cos.shape[0]
    if lengths_out is None:
        lengths_out = torch.empty_like(lengths)
    out = _flat(self, "lengths_out", lengths_out, torch.int32, (n,))
    _call(self, self._lib.nnb_paged_append, C.byref(cache._c), C.byref(s), C.byref(t), out)
    return q_out, lengths_out


def paged_attention_decode(self, cache, table, lengths, q, scale=0.0, accumulate=False, out=None, lse=None):
    """Attention of one new token per sequence, q (n_seq, n_head, dk), over the `lengths` cached positions.  Returns
    (out (n_seq, n_head, dk) of q's type, lse (n_seq, n_head) f32); accumulate adds the attention weights to cache.weight."""
    s = _seqs(self, cache, table, lengths)
    stride = _rows(self, "q", q, None, cache.dk)
    n, heads = s.n_seq, q.shape[1]
    if q.shape[0] != n:
        raise NnbError(f"{q.shape[0]} queries for {n} sequences")
    if out is None:
        out = q.new_empty(q.shape)
    else:
        _flat(self, "out", out, q.dtype, q.shape)
    if lse is None:
        lse = q.new_empty((n, heads), dtype=torch.float32)
    else:
        _flat(self, "lse", lse, torch.float32, (n, heads))
    accumulate, d_out, d_lse = int(accumulate), out.data_ptr(), lse.data_ptr()
    size = self._lib.nnb_paged_attention_workspace(self._h, C.byref(cache._c), C.byref(s), heads, accumulate)
    ws = q.new_empty(size, dtype=torch.uint8)
    _call(self, self._lib.nnb_paged_attention_decode, C.byref(cache._c), C.byref(s), q.data_ptr(), _DTYPES[q.dtype], stride, heads, scale, d_out, d_lse,
          accumulate, ws.data_ptr(), size)
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
    ws = lengths.new_empty(size, dtype=torch.uint8)
    _call(self, self._lib.nnb_paged_evict, C.byref(cache._c), C.byref(s), budget, sinks, recent, C.byref(dst._c), d.d_table, d.max_pages, d.table_stride,
          n_out, ws.data_ptr(), size)
    return lengths_out


def adjust_logits(self, logits, history=None, history_len=None, prompt_len=None, repeat_window=0, repeat_penalty=None, presence_penalty=None,
                  frequency_penalty=None, bias=None, allowed=None, out=None):
    """logits (n_seq, vocab) f32 or bf16 with a bias, penalties for the ids of history (n_seq, max_history) and a mask of
    allowed ids (one bit each, (n_seq, ceil(vocab / 32)) int32), in this order.  Penalties are (n_seq) f32, bias and allowed
    one row for all or one per sequence; out may be logits.  Returns out."""
    _need(logits.dim() == 2 and logits.dtype in _DTYPES and logits.device == self.device, "logits is an (n_seq, vocab) tensor on the engine's device, f32 or bf16")
    n, vocab = logits.shape
    if out is None:
        out = logits.new_empty((n, vocab))
    else:
        _on(self, "out", out, logits.dtype, (n, vocab))
    _need(n == 0 or (logits.stride(1) == 1 and out.stride(1) == 1), "rows of the logits are not contiguous")
    c = _Logits()
    c.repeat_window = repeat_window
    penalties = (("d_repeat", "repeat_penalty", repeat_penalty), ("d_presence", "presence_penalty", presence_penalty),
                 ("d_frequency", "frequency_penalty", frequency_penalty))
    if history is None:
        _need(all(t is None for _, _, t in penalties), "penalties need a history")
    else:
        _need(_on(self, "history", history, torch.int32).dim() == 2 and history.shape[0] == n and (history.numel() == 0 or history.stride(1) == 1),
              "history is (n_seq, max_history) with contiguous rows")
        _need(history_len is not None, "history needs history_len")
        given = [(field, _flat(self, name, t, torch.float32, (n,))) for field, name, t in penalties if t is not None]
        lens = _flat(self, "history_len", history_len, torch.int32, (n,))
        prompt = _flat(self, "prompt_len", prompt_len, torch.int32, (n,)) if prompt_len is not None else None
        if history.numel():  # with an empty one there is nothing to penalise
            c.d_history, c.history_stride, c.max_history = history.data_ptr(), history.stride(0), history.shape[1]
            c.d_history_len, c.d_prompt_len = lens, prompt
            for field, ptr in given:
                setattr(c, field, ptr)
    for name, t, dtype, width in (("bias", bias, torch.float32, vocab), ("allowed", allowed, torch.int32, (vocab + 31) // 32)):
        if t is not None:
            _on(self, name, t, dtype)
            if tuple(t.shape) not in ((width,), (n, width)) or t.stride(-1) != 1:
                raise NnbError(f"{name} is ({width}) or ({n}, {width}) with contiguous rows")
            setattr(c, "d_" + name, t.data_ptr())
            setattr(c, name + "_stride", t.stride(0) if t.dim() == 2 else 0)
    _call(self, self._lib.nnb_adjust_logits, logits.data_ptr(), _DTYPES[logits.dtype], n, vocab, logits.stride(0), C.byref(c), out.data_ptr(), out.stride(0))
    return out


for _f in (paged_append, paged_attention_decode, paged_evict, adjust_logits):
    setattr(Engine, _f.__name__, _f)
