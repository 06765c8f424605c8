"""The paged-cache operators without a GPU: the place of a position in the pool, and the refusal of every bad argument
(checked before anything reaches a device, so the pointers here are only numbers)."""
import ctypes as C

import pytest

FAKE = 4096  # an aligned address that is never followed


def _structs(pkg):
    from neuralnet_cpp_b200 import paged

    return paged


def _cache(pkg, **kw):
    p = _structs(pkg)
    f = dict(d_k=FAKE, d_v=FAKE, d_weight=FAKE, dtype=1, n_pages=7, page_size=16, n_head_kv=2, dk=100)
    f.update(kw)
    return p._Cache(**f)


def _seqs(pkg, **kw):
    p = _structs(pkg)
    f = dict(d_table=FAKE, d_len=FAKE, n_seq=3, max_pages=4, table_stride=4)
    f.update(kw)
    return p._Seqs(**f)


def _tokens(pkg, **kw):
    p = _structs(pkg)
    f = dict(d_q=FAKE, d_k=FAKE, d_v=FAKE, d_q_out=FAKE, q_stride=400, k_stride=200, v_stride=200, q_out_stride=400, dtype=0, n_head=4, n_rows=3,
             d_row_start=None, d_pos=None, d_rope_cos=FAKE, d_rope_sin=FAKE, rope_ctx=64)
    f.update(kw)
    return p._Tokens(**f)


def test_pitch_and_row(pkg):
    lib = pkg.lib()
    assert [lib.nnb_paged_pitch(d) for d in (2, 8, 64, 100, 128, 250)] == [8, 8, 64, 104, 128, 256]
    c = _cache(pkg)
    ids = (C.c_int32 * 4)(6, 0, -1, 7)
    row = lambda head, pos, n=4: lib.nnb_paged_row(C.byref(c), ids, n, head, pos)  # noqa: E731
    assert row(0, 0) == 6 * 2 * 16 and row(1, 15) == (6 * 2 + 1) * 16 + 15 and row(1, 16) == 16 and row(0, 31) == 15
    assert row(0, 32) == -1 and row(0, 48) == -1  # page ids -1 and 7 are not in the pool of 7
    assert row(0, 64) == -1 and row(0, 16, 1) == -1 and row(2, 0) == -1 and row(-1, 0) == -1 and row(0, -1) == -1
    big = _cache(pkg, n_pages=2**31 - 1, page_size=1024, n_head_kv=64)
    far = (C.c_int32 * 1)(2**31 - 2)
    assert lib.nnb_paged_row(C.byref(big), far, 1, 63, 1023) == ((2**31 - 2) * 64 + 63) * 1024 + 1023


BAD_CACHE = [(dict(d_k=None), "no keys"), (dict(d_v=None), "no keys"), (dict(dtype=2), "dtype"), (dict(n_pages=0), "no pages"),
             (dict(page_size=0), "no pages"), (dict(n_head_kv=0), "no pages"), (dict(n_head_kv=-1), "no pages"), (dict(dk=0), "head size"),
             (dict(dk=65), "head size"), (dict(dk=258), "head size"), (dict(d_k=FAKE + 8), "16-byte"), (dict(d_v=FAKE + 2), "16-byte"),
             (dict(n_pages=2**20, page_size=2**10, n_head_kv=4), "2^31")]
BAD_SEQS = [(dict(n_seq=-1), "number of sequences"), (dict(max_pages=0), "number of sequences"), (dict(d_table=None), "NULL"), (dict(d_len=None), "NULL"),
            (dict(table_stride=3), "overlap"), (dict(max_pages=2**27, table_stride=2**27), "2^30")]


def _refused(pkg, status, text):
    msg = pkg.lib().nnb_last_error().decode()
    assert status == -1 and text in msg, (status, msg, text)


@pytest.mark.parametrize("bad,text", BAD_CACHE)
def test_bad_caches_are_refused(pkg, bad, text):
    lib, c, s = pkg.lib(), _cache(pkg, **bad), _seqs(pkg)
    _refused(pkg, lib.nnb_paged_append(None, C.byref(c), C.byref(s), C.byref(_tokens(pkg)), FAKE), text)
    _refused(pkg, lib.nnb_paged_attention_decode(None, C.byref(c), C.byref(s), FAKE, 0, 400, 4, 0.0, FAKE, FAKE, 0, FAKE, 1 << 20), text)
    ok = _cache(pkg)
    for a, b in ((c, ok), (ok, c)):
        _refused(pkg, lib.nnb_paged_evict(None, C.byref(a), C.byref(s), 8, 1, 1, C.byref(b), FAKE, 4, 4, FAKE, FAKE, 1 << 20), text)
    assert lib.nnb_paged_evict_workspace(None, C.byref(c), C.byref(s), 8) == 0
    assert lib.nnb_paged_attention_workspace(None, C.byref(c), C.byref(s), 4, 0) == 0


@pytest.mark.parametrize("bad,text", BAD_SEQS)
def test_bad_sequences_are_refused(pkg, bad, text):
    lib, c, s = pkg.lib(), _cache(pkg), _seqs(pkg, **bad)
    _refused(pkg, lib.nnb_paged_append(None, C.byref(c), C.byref(s), C.byref(_tokens(pkg)), FAKE), text)
    _refused(pkg, lib.nnb_paged_attention_decode(None, C.byref(c), C.byref(s), FAKE, 0, 400, 4, 0.0, FAKE, FAKE, 0, FAKE, 1 << 20), text)
    _refused(pkg, lib.nnb_paged_evict(None, C.byref(c), C.byref(s), 8, 1, 1, C.byref(c), FAKE, 4, 4, FAKE, FAKE, 1 << 20), text)


@pytest.mark.parametrize("bad,text", [
    (dict(dtype=3), "dtype"), (dict(n_rows=4), "row_start"), (dict(d_k=None), "NULL"), (dict(d_v=None), "NULL"), (dict(n_head=0), "go together"),
    (dict(d_q=None), "go together"), (dict(d_q_out=None), "go together"), (dict(k_stride=199), "overlap"), (dict(v_stride=10), "overlap"),
    (dict(q_stride=399), "overlap"), (dict(q_out_stride=0), "overlap"), (dict(q_stride=500), "one stride"), (dict(d_k=FAKE + 2), "misaligned"),
    (dict(d_rope_sin=None), "tables go together"), (dict(rope_ctx=0), "empty rope"), (dict(n_rows=2**31, d_row_start=FAKE), "2^30"), (dict(), "engine is NULL")])
def test_bad_tokens_are_refused(pkg, bad, text):
    lib = pkg.lib()
    _refused(pkg, lib.nnb_paged_append(None, C.byref(_cache(pkg)), C.byref(_seqs(pkg)), C.byref(_tokens(pkg, **bad)), FAKE), text)


@pytest.mark.parametrize("kw,text", [
    (dict(dtype=5), "dtype"), (dict(n_head=3), "share"), (dict(n_head=0), "share"), (dict(q=None), "NULL"), (dict(out=None), "NULL"),
    (dict(q_stride=399), "overlap"), (dict(q=FAKE + 1), "misaligned"), (dict(out=FAKE + 2), "misaligned"), (dict(scale=float("nan")), "scale"),
    (dict(scale=float("inf")), "scale"), (dict(accumulate=1, weight=None), "no weights"), (dict(n_head=2**31), "2^31"), (dict(), "engine is NULL")])
def test_bad_decode_calls_are_refused(pkg, kw, text):
    f = dict(dtype=0, n_head=4, q=FAKE, out=FAKE, q_stride=400, scale=0.0, accumulate=0, weight=FAKE)
    f.update(kw)
    st = pkg.lib().nnb_paged_attention_decode(None, C.byref(_cache(pkg, d_weight=f["weight"])), C.byref(_seqs(pkg)), f["q"], f["dtype"], f["q_stride"],
                                              f["n_head"], f["scale"], f["out"], FAKE, f["accumulate"], FAKE, 1 << 20)
    _refused(pkg, st, text)


@pytest.mark.parametrize("kw,text", [
    (dict(budget=0), "budget"), (dict(sinks=9), "budget"), (dict(recent=8), "budget"), (dict(sinks=2**64 - 1, recent=2), "budget"),
    (dict(budget=2**31), "budget"), (dict(table=None), "NULL"), (dict(len_out=None), "NULL"), (dict(stride=3), "overlap"), (dict(pages=0), "overlap"),
    (dict(budget=33, pages=2), "fewer than 33"), (dict(budget=1000, pages=3), "fewer than 64"), (dict(len_out="len"), "own array"),
    (dict(src=dict(d_weight=None)), "weights"), (dict(dst=dict(d_weight=None)), "weights"), (dict(dst=dict(dtype=0)), "differ"),
    (dict(dst=dict(n_head_kv=4)), "differ"), (dict(dst=dict(dk=102)), "differ"), (dict(), "engine is NULL")])
def test_bad_evictions_are_refused(pkg, kw, text):
    f = dict(budget=8, sinks=1, recent=2, table=FAKE, pages=4, stride=4, len_out=FAKE * 2, src={}, dst={})
    f.update(kw)
    st = pkg.lib().nnb_paged_evict(None, C.byref(_cache(pkg, **f["src"])), C.byref(_seqs(pkg)), f["budget"], f["sinks"], f["recent"],
                                   C.byref(_cache(pkg, **f["dst"])), f["table"], f["pages"], f["stride"], FAKE if f["len_out"] == "len" else f["len_out"],
                                   FAKE, 1 << 20)
    _refused(pkg, st, text)


@pytest.mark.parametrize("kw,text", [
    (dict(logits=None), "NULL"), (dict(out=None), "NULL"), (dict(cfg=None), "NULL"), (dict(dtype=2), "dtype"), (dict(vocab=0), "bad shape"),
    (dict(vocab=2**31, stride=2**31), "bad shape"), (dict(n=2**31), "bad shape"), (dict(stride=99), "overlap"), (dict(out_stride=99), "overlap"),
    (dict(out_stride=200, out=FAKE), "one stride"), (dict(logits=FAKE + 1), "misaligned"), (dict(c=dict(d_history_len=None)), "go together"),
    (dict(c=dict(d_history=None, d_history_len=None)), "need a history"), (dict(c=dict(max_history=11)), "history overlap"),
    (dict(c=dict(repeat_window=-1)), "window"), (dict(c=dict(bias_stride=99)), "bias overlap"), (dict(c=dict(allowed_stride=3)), "mask overlap"),
    (dict(), "engine is NULL")])
def test_bad_logit_calls_are_refused(pkg, kw, text):
    f = dict(logits=FAKE, out=2 * FAKE, dtype=0, n=3, vocab=100, stride=100, out_stride=100, c={}, cfg=1)
    f.update(kw)
    c = dict(d_history=FAKE, history_stride=10, max_history=10, d_history_len=FAKE, d_prompt_len=FAKE, repeat_window=0, d_repeat=FAKE, d_presence=FAKE,
             d_frequency=FAKE, d_bias=FAKE, bias_stride=0, d_allowed=FAKE, allowed_stride=4)
    c.update(f["c"])
    cfg = _structs(pkg)._Logits(**c)
    st = pkg.lib().nnb_adjust_logits(None, f["logits"], f["dtype"], f["n"], f["vocab"], f["stride"], C.byref(cfg) if f["cfg"] else None, f["out"],
                                     f["out_stride"])
    _refused(pkg, st, text)


def test_null_structs_are_refused(pkg):
    lib, c, s = pkg.lib(), _cache(pkg), _seqs(pkg)
    assert lib.nnb_paged_append(None, None, C.byref(s), C.byref(_tokens(pkg)), FAKE) == -1
    assert lib.nnb_paged_append(None, C.byref(c), None, C.byref(_tokens(pkg)), FAKE) == -1
    assert lib.nnb_paged_append(None, C.byref(c), C.byref(s), None, FAKE) == -1
    assert lib.nnb_paged_row(None, (C.c_int32 * 1)(0), 1, 0, 0) == -1 and lib.nnb_paged_row(C.byref(c), None, 1, 0, 0) == -1


def test_pools_of_another_shape_are_refused(pkg):
    import torch

    k = torch.zeros(3, 2, 4, 104)
    for args in ((k, k, 96), (k, k[:2], 100), (k, k.bfloat16(), 100), (k[0], k[0], 100), (k.double(), k.double(), 100), (k, k, 100, torch.zeros(3, 2, 5)),
                 (k, k, 100, torch.zeros(3, 2, 4).double()), (k, k, 100)):  # the last: not on a GPU
        with pytest.raises(pkg.NnbError):
            pkg.PagedCache(*args)
