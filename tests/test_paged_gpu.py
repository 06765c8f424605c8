"""The paged-cache operators on the GPU against their definitions in 64 bits (plain loops over sequences and heads).

Tolerances are first-order rounding bounds of the operators' own arithmetic: u = 2^-24 for every f32 step, half a step of the
output's type for the rounding at the end.  Selections (eviction) and copies have to be exact."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
F32, BF16 = torch.float32, torch.bfloat16


def _pool(pkg, eng, lens, hk, page, dk, dtype, seed=0, room=0, track=False, spare=2, extra_cols=1):
    """A pool whose every unused place holds NaN, with the sequences' pages scattered over it; unused table entries are out of
    the pool, so reading one would be reported."""
    rng = np.random.default_rng(seed)
    used = [(n + room + page - 1) // page for n in lens]
    n_pages = sum(used) + spare
    ids = rng.permutation(n_pages)
    cols = max(max(used, default=0), 1) + extra_cols
    table = np.full((len(lens), cols), 2**30, np.int32)
    at = 0
    for i, u in enumerate(used):
        table[i, :u] = ids[at:at + u]
        at += u
    pitch = (dk + 7) // 8 * 8
    g = torch.Generator(device="cpu").manual_seed(seed)
    k, v = torch.full((n_pages, hk, page, pitch), float("nan")), torch.full((n_pages, hk, page, pitch), float("nan"))
    w = torch.full((n_pages, hk, page), float("nan"))
    for i, n in enumerate(lens):
        for t in range(0, n, page):
            m, p = min(page, n - t), int(table[i, t // page])
            k[p, :, :m] = 0
            v[p, :, :m] = 0
            k[p, :, :m, :dk] = torch.randn((hk, m, dk), generator=g)
            v[p, :, :m, :dk] = torch.randn((hk, m, dk), generator=g)
            w[p, :, :m] = torch.rand((hk, m), generator=g)
    dev = eng.device
    cache = pkg.PagedCache(k.to(dtype).to(dev), v.to(dtype).to(dev), dk, w.to(dev) if track else None)
    return cache, torch.from_numpy(table).to(dev), torch.tensor(lens, dtype=torch.int32, device=dev)


def _read(cache, table, seq, n):
    """k, v (heads, n, dk) in f64 and the weights of one sequence, on the CPU."""
    pos = torch.arange(n)
    pages, at = table[seq].cpu().long()[pos // cache.page_size], pos % cache.page_size
    k, v = cache.k.cpu()[pages, :, at, :cache.dk].double().transpose(0, 1), cache.v.cpu()[pages, :, at, :cache.dk].double().transpose(0, 1)
    return k, v, None if cache.weight is None else cache.weight.cpu()[pages, :, at].double().t()


def _check_decode(cache, table, lens, q, out, lse, scale=None, w_before=None):
    """Bounds: a score is a dot product of dk terms, off by (dk + 4) u sum |q k| scale + its own rounding; p = exp(x - m) is off
    by twice that (numerator and sum) plus a few u of exp; the sums over n positions by n u; all relative to sum p |v|.
    With bf16 queries on a bf16 cache p enters the product with V as two bf16 pieces: the leading 8 bits cut off leave less than
    2^-7 p, whose rounding to 8 bits is off by at most half a step, 2^-8 of it: 2^-15 p in all."""
    hk, dk, heads = cache.n_head_kv, cache.dk, q.shape[1]
    g = heads // hk
    scale = dk ** -0.5 if scale is None else scale
    half, cut = HALF[out.dtype], 2.0 ** -15 if q.dtype == cache.k.dtype == BF16 else 0.0
    out, lse, q = out.cpu().double(), lse.cpu().double(), q.cpu().double()
    for i, n in enumerate(lens):
        if n == 0:
            assert bool((out[i] == 0).all()) and bool((lse[i] == -np.inf).all())
            continue
        k, v, w = _read(cache, table, i, n)
        qq = q[i].view(hk, g, dk)
        x = torch.einsum("hgd,htd->hgt", qq, k) * scale
        delta = ((dk + 4) * U * abs(scale) * torch.einsum("hgd,htd->hgt", qq.abs(), k.abs())).amax(-1, keepdim=True) + 4 * U * x.abs().amax(-1, keepdim=True) + 8 * U
        p = torch.softmax(x, -1)
        want = torch.einsum("hgt,htd->hgd", p, v)
        tol = (2 * delta + (n + 16) * U + cut) * torch.einsum("hgt,htd->hgd", p, v.abs())
        got = out[i].view(hk, g, dk)
        assert bool(((got - want).abs() <= tol + half * (want.abs() + tol) + 1e-38).all()), (i, n, ((got - want).abs() - tol).max())
        z = torch.logsumexp(x, -1)
        assert bool(((lse[i].view(hk, g) - z).abs() <= delta[..., 0] + (n + 16) * U + 4 * U * z.abs()).all()), (i, n)
        if w_before is not None:
            add = p.sum(1)
            wt = w_before[i] + add
            bound = (p * (2 * delta + (n + 16 + g) * U)).sum(1) + 2 * U * wt
            assert bool(((w - wt).abs() <= bound).all()), (i, n, (w - wt).abs().max())


def _decode(pkg, eng, lens, heads, hk, page, dk, cache_dtype, io, seed=0, scale=None, track=False, spread=1.5):
    cache, table, lengths = _pool(pkg, eng, lens, hk, page, dk, cache_dtype, seed, track=track)
    g = torch.Generator(device="cpu").manual_seed(seed + 1)
    q = (torch.randn((len(lens), heads, dk), generator=g) * spread).to(io).to(eng.device)
    before = [_read(cache, table, i, n)[2] for i, n in enumerate(lens)] if track else None
    out, lse = eng.paged_attention_decode(cache, table, lengths, q, scale=scale or 0.0, accumulate=track)
    eng.check_device_errors()
    _check_decode(cache, table, lens, q, out, lse, scale, before)
    return cache, table, lengths, q, out, lse


EDGE = [0, 1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 129, 200]


@pytest.mark.parametrize("io", [F32, BF16])
@pytest.mark.parametrize("cache_dtype", [F32, BF16])
@pytest.mark.parametrize("heads,hk,page,dk", [(4, 4, 16, 64), (20, 5, 16, 128), (8, 2, 3, 100), (2, 1, 1, 128), (7, 1, 64, 80), (32, 2, 48, 64),
                                              (3, 3, 7, 2), (16, 1, 32, 256), (24, 2, 16, 34), (40, 1, 8, 128), (6, 2, 256, 200)])
def test_decode_matches_the_definition(pkg, eng, heads, hk, page, dk, cache_dtype, io):
    _decode(pkg, eng, EDGE, heads, hk, page, dk, cache_dtype, io, seed=heads + dk)


@pytest.mark.parametrize("cache_dtype,io", [(BF16, F32), (BF16, BF16), (F32, F32)])
@pytest.mark.parametrize("lens,heads,hk,page,dk", [([5000], 4, 1, 16, 128), ([3001, 0, 17], 8, 8, 64, 64), ([12345, 999], 20, 5, 48, 128),
                                                   ([4096, 4097], 2, 2, 32, 100), ([700] * 40, 4, 4, 16, 64)])
def test_decode_of_long_contexts_is_split_and_joined(pkg, eng, lens, heads, hk, page, dk, cache_dtype, io):
    _decode(pkg, eng, lens, heads, hk, page, dk, cache_dtype, io, seed=len(lens))


@pytest.mark.parametrize("cache_dtype,io", [(BF16, F32), (BF16, BF16), (F32, F32)])
@pytest.mark.parametrize("heads,hk,page,dk", [(3, 1, 3, 8), (8, 1, 16, 2), (8, 4, 16, 16), (4, 2, 8, 72), (5, 5, 16, 136)])
def test_decode_of_more_sequences_than_workers(pkg, eng, heads, hk, page, dk, cache_dtype, io):
    """Several short sequences per worker, empty ones among them, and narrow rows (a tile smaller than a result)."""
    rng = np.random.default_rng(dk)
    lens = [int(x) for x in rng.integers(0, 40, 700) * (rng.random(700) > 0.1)]
    _decode(pkg, eng, lens, heads, hk, page, dk, cache_dtype, io, seed=dk)


@pytest.mark.parametrize("cache_dtype,io", [(BF16, F32), (BF16, BF16), (F32, BF16), (F32, F32)])
@pytest.mark.parametrize("heads,hk,page,dk,lens", [(4, 4, 16, 64, EDGE), (20, 5, 5, 128, [3000, 1, 0, 64, 65]), (32, 2, 64, 100, [500, 700]),
                                                   (8, 1, 16, 128, [6001])])
def test_decode_accumulates_the_attention_weights(pkg, eng, heads, hk, page, dk, lens, cache_dtype, io):
    cache, table, lengths, q, _, _ = _decode(pkg, eng, lens, heads, hk, page, dk, cache_dtype, io, seed=3, track=True)
    # what no sequence owns is as it was (NaN in every unused place)
    total = sum(lens) * hk
    assert int((~torch.isnan(cache.weight)).sum()) == total
    seen = [_read(cache, table, i, n)[2] for i, n in enumerate(lens)]
    out, lse = eng.paged_attention_decode(cache, table, lengths, q, accumulate=True)  # and once more on top
    _check_decode(cache, table, lens, q, out, lse, None, seen)


def test_decode_scale_and_peaked_scores(pkg, eng):
    """Another scale, a negative one, and scores far apart (one position takes all the weight)."""
    for scale in (1.0, -0.3, 1e-3):
        _decode(pkg, eng, [1, 64, 300], 8, 2, 16, 64, BF16, F32, seed=4, scale=scale)
    _decode(pkg, eng, [1, 64, 300], 8, 2, 16, 128, BF16, F32, seed=5, spread=100.0)
    _decode(pkg, eng, [1, 64, 300], 8, 2, 16, 128, F32, BF16, seed=5, spread=100.0)


@pytest.mark.parametrize("cache_dtype,io", [(BF16, F32), (BF16, BF16), (F32, F32)])
def test_decode_takes_strided_and_oddly_aligned_queries(pkg, eng, cache_dtype, io):
    lens, heads, hk, dk = [5, 100, 0, 33], 8, 2, 100
    cache, table, lengths = _pool(pkg, eng, lens, hk, 16, dk, cache_dtype)
    q = torch.randn((4, heads, dk), device=eng.device).to(io)
    want = eng.paged_attention_decode(cache, table, lengths, q)
    wide = torch.randn((4, heads + 2 * hk, dk), device=eng.device).to(io)
    wide[:, :heads] = q
    odd = torch.zeros(4 * (heads * dk + 3) + 1, device=eng.device, dtype=io)[1:].view(4, heads * dk + 3)[:, :heads * dk].unflatten(1, (heads, dk))
    odd.copy_(q)
    for view in (wide[:, :heads], odd):
        got = eng.paged_attention_decode(cache, table, lengths, view)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    tall = torch.full((4, table.shape[1] + 5), -7, dtype=torch.int32, device=eng.device)
    tall[:, :table.shape[1]] = table
    got = eng.paged_attention_decode(cache, tall[:, :table.shape[1]], lengths, q)  # a table with longer rows
    assert torch.equal(got[0], want[0])


def test_decode_is_the_same_every_time_and_ignores_batch_neighbours(pkg, eng):
    """Run-to-run identical; a sequence alone and in a batch agree within the bounds (they may be split differently)."""
    cache, table, lengths, q, out, lse = _decode(pkg, eng, [900, 3, 2500, 64], 20, 5, 16, 128, BF16, F32, seed=8)
    for _ in range(3):
        o, z = eng.paged_attention_decode(cache, table, lengths, q)
        assert torch.equal(o, out) and torch.equal(z, lse)
    o, z = eng.paged_attention_decode(cache, table[2:3], lengths[2:3], q[2:3])
    _check_decode(cache, table[2:3], [2500], q[2:3], o, z)


@pytest.mark.parametrize("cache_dtype", [F32, BF16])
@pytest.mark.parametrize("lens", [[90, 0, 33], [3000, 5, 70]])
def test_decode_through_the_c_interface_without_lse(pkg, eng, lens, cache_dtype):
    """d_lse NULL with accumulated weights; a workspace full of NaN, exactly as large as asked for; one byte less is refused."""
    import ctypes as C

    lib = pkg.lib()
    cache, table, lengths = _pool(pkg, eng, lens, 2, 16, 64, cache_dtype, track=True)
    w0 = cache.weight.clone()
    q = torch.randn((3, 8, 64), device=eng.device)
    want, _ = eng.paged_attention_decode(cache, table, lengths, q, accumulate=True)
    w1 = cache.weight.clone()
    cache.weight.copy_(w0)
    from neuralnet_cpp_b200 import paged

    s = paged._Seqs(table.data_ptr(), lengths.data_ptr(), 3, table.shape[1], table.stride(0))
    size = lib.nnb_paged_attention_workspace(eng.handle, C.byref(cache._c), C.byref(s), 8, 1)
    ws = torch.full((size // 4 + 64,), float("nan"), device=eng.device)
    out = torch.empty_like(q)
    call = lambda n: lib.nnb_paged_attention_decode(eng.handle, C.byref(cache._c), C.byref(s), q.data_ptr(), 0, 512, 8, 0.0, out.data_ptr(), None, 1,  # noqa: E731
                                                    ws.data_ptr(), n)
    assert call(size - 1) == -1 and b"too small" in lib.nnb_last_error()
    assert call(size) == 0
    eng.check_device_errors()
    assert torch.equal(out, want) and torch.equal(cache.weight.nan_to_num(9.0), w1.nan_to_num(9.0))
    assert bool(ws[size // 4:].isnan().all())  # nothing behind the workspace was touched


def test_sequences_may_share_pages(pkg, eng):
    """The completions of one prompt: their tables begin with the same pages."""
    cache, table, lengths, q, out, _ = _decode(pkg, eng, [256, 300, 280], 8, 2, 16, 64, BF16, F32, seed=9)
    shared = table.clone()
    shared[1:, :8] = table[0, :8]
    o, z = eng.paged_attention_decode(cache, shared, lengths, q)
    eng.check_device_errors()
    _check_decode(cache, shared, [256, 300, 280], q, o, z)


@pytest.mark.parametrize("cache_dtype", [F32, BF16])
def test_bad_pages_and_lengths_are_skipped_and_reported(pkg, eng, cache_dtype):
    lens = [40, 70, 33]
    cache, table, lengths = _pool(pkg, eng, lens, 2, 16, 64, cache_dtype, track=True, extra_cols=0)
    q = torch.randn((3, 4, 64), device=eng.device)
    good = eng.paged_attention_decode(cache, table, lengths, q)[0]
    bad = table.clone()
    bad[0, 1], bad[1, 4] = -1, cache.n_pages
    w0 = cache.weight.clone()
    out, lse = eng.paged_attention_decode(cache, bad, lengths, q, accumulate=True)
    with pytest.raises(pkg.NnbError, match="page id"):
        eng.check_device_errors()
    eng.check_device_errors()  # reported once
    assert torch.equal(out[2], good[2])
    # sequence 0 without positions 16..31: as a cache of the other 24
    short = torch.stack([table[0, [0, 2, 2, 2, 2]]] * 1)
    want, z = eng.paged_attention_decode(cache, short, torch.tensor([24], dtype=torch.int32, device=eng.device), q[:1])
    assert torch.allclose(out[:1], want, rtol=1e-5, atol=1e-6) and torch.allclose(lse[:1], z, rtol=1e-6)
    gone = w0.isnan()
    assert torch.equal(cache.weight.isnan(), gone)
    # lengths outside the table count as its ends
    eng.paged_attention_decode(cache, table, torch.tensor([40, -5, 33], dtype=torch.int32, device=eng.device), q)
    with pytest.raises(pkg.NnbError, match="length"):
        eng.check_device_errors()
    cache2, table2, _ = _pool(pkg, eng, [80, 80], 2, 16, 64, cache_dtype, extra_cols=0)
    a = eng.paged_attention_decode(cache2, table2, torch.tensor([2**31 - 1, 80], dtype=torch.int32, device=eng.device), q[:2])[0]
    with pytest.raises(pkg.NnbError, match="length"):
        eng.check_device_errors()
    b = eng.paged_attention_decode(cache2, table2, torch.tensor([80, 80], dtype=torch.int32, device=eng.device), q[:2])[0]
    assert torch.equal(a, b)
    eng.check_device_errors()


def test_row_of_a_position(pkg, eng):
    cache, table, lengths = _pool(pkg, eng, [40, 7], 3, 16, 100, BF16, track=True)
    k, v, w = _read(cache, table, 0, 40)
    rows = cache.k.view(-1, cache.pitch).cpu()
    for head, pos in ((0, 0), (2, 15), (1, 16), (2, 39)):
        r = cache.row(table[0].tolist(), head, pos)
        assert torch.equal(rows[r, :100].double(), k[head, pos]) and cache.weight.view(-1)[r].item() == w[head, pos].item()
    assert cache.row(table[0].tolist(), 0, 16 * table.shape[1]) == -1 and cache.row(table[1].tolist(), 0, 16) == -1


def test_offsets_beyond_32_bits(pkg, eng):
    """A pool of more than 2^31 elements per tensor; the sequences' pages lie at its end."""
    hk, page, dk = 8, 64, 128
    n_pages = 2**31 // (hk * page * dk) + 40
    k = torch.empty((n_pages, hk, page, dk), device=eng.device, dtype=BF16)
    v = torch.empty_like(k)
    w = torch.zeros((n_pages, hk, page), device=eng.device)
    k[-40:].normal_()
    v[-40:].normal_()
    cache = pkg.PagedCache(k, v, dk, w)
    lens = [1000, 70]
    table = torch.arange(n_pages - 34, n_pages, device=eng.device, dtype=torch.int32).view(2, 17)
    lengths = torch.tensor(lens, dtype=torch.int32, device=eng.device)
    tail = pkg.PagedCache(k[-40:].clone(), v[-40:].clone(), dk, w[-40:].clone())
    q = torch.randn((2, 32, dk), device=eng.device)
    new = torch.randn((2, hk, dk), device=eng.device)
    for c, t in ((cache, table), (tail, table - (n_pages - 40))):
        n = eng.paged_append(c, t, lengths, new, new)[1]
        c.out = eng.paged_attention_decode(c, t, n, q, accumulate=True)
    assert torch.equal(cache.out[0], tail.out[0]) and torch.equal(cache.out[1], tail.out[1])
    assert torch.equal(cache.k[-40:], tail.k) and torch.equal(cache.weight[-40:], tail.weight)
    dst = pkg.PagedCache.empty(4, hk, page, dk, device=eng.device, track_weight=True)
    dst2 = pkg.PagedCache.empty(4, hk, page, dk, device=eng.device, track_weight=True)
    dt = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device=eng.device)
    eng.paged_evict(cache, table, n, dst, dt, budget=100, sinks=4, recent=20)
    eng.paged_evict(tail, table - (n_pages - 40), n, dst2, dt, budget=100, sinks=4, recent=20)
    eng.check_device_errors()
    assert torch.equal(dst.k, dst2.k) and torch.equal(dst.v, dst2.v) and torch.equal(dst.weight, dst2.weight)


# ------------------------------------------------------------------------------------------------ append
def _tables(eng, dk, ctx):
    cos, sin = torch.empty((ctx, dk // 2), device=eng.device), torch.empty((ctx, dk // 2), device=eng.device)
    ang = torch.arange(ctx, dtype=torch.float64)[:, None] * 10000.0 ** (-2.0 * torch.arange(dk // 2, dtype=torch.float64) / dk)
    cos.copy_(ang.cos())
    sin.copy_(ang.sin())
    return cos, sin


def _turned(x, cos, sin):
    """(rows, heads, dk) in f64, and the bound on the error before the last rounding: two products and a sum in f32."""
    a, b = x.cpu().double().chunk(2, -1)
    c, s = cos.cpu().double()[:, None], sin.cpu().double()[:, None]
    y = torch.cat([a * c - b * s, b * c + a * s], -1)
    size = torch.cat([(a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()], -1)
    return y, 3 * U * size


def _near(got, want, slack):
    half = HALF[got.dtype]
    return bool(((got.cpu().double() - want).abs() <= slack + half * (want.abs() + slack)).all())


@pytest.mark.parametrize("io", [F32, BF16])
@pytest.mark.parametrize("cache_dtype", [F32, BF16])
@pytest.mark.parametrize("heads,hk,page,dk", [(16, 4, 16, 64), (20, 5, 7, 128), (4, 4, 1, 100), (1, 1, 3, 2), (2, 1, 16, 250), (3, 3, 64, 256)])
def test_append_one_token_each(pkg, eng, heads, hk, page, dk, cache_dtype, io):
    lens = [0, 1, 2, 15, 16, 17, 6, 7]
    cache, table, lengths = _pool(pkg, eng, lens, hk, page, dk, cache_dtype, room=1, track=True)
    k0, v0, w0 = cache.k.clone(), cache.v.clone(), cache.weight.clone()
    n = len(lens)
    qkv = torch.randn((n, heads + 2 * hk, dk), device=eng.device).to(io)
    q, k, v = qkv.split([heads, hk, hk], 1)
    cos, sin = _tables(eng, dk, 32)
    got_q, new = eng.paged_append(cache, table, lengths, k, v, q=q, rope=(cos, sin))
    eng.check_device_errors()
    assert new.tolist() == [t + 1 for t in lens] and lengths.tolist() == lens
    at = lengths.long()
    want, slack = _turned(q, cos[at], sin[at])
    assert _near(got_q, want, slack)
    want, slack = _turned(k, cos[at], sin[at])
    hit = torch.zeros_like(w0, dtype=torch.bool)
    for i, t in enumerate(lens):
        p, s = int(table[i, t // page]), t % page
        hit[p, :, s] = True
        assert _near(cache.k[p, :, s, :dk], want[i], slack[i])
        assert torch.equal(cache.v[p, :, s, :dk], v[i].to(cache_dtype))
        assert not cache.k[p, :, s, dk:].any() and not cache.v[p, :, s, dk:].any() and not cache.weight[p, :, s].any()
    # everything else is as it was, bit for bit
    kind = torch.int32 if cache_dtype == F32 else torch.int16
    for now, was in ((cache.k, k0), (cache.v, v0)):
        assert torch.equal(now.view(kind)[~hit], was.view(kind)[~hit])
    assert torch.equal(cache.weight.view(torch.int32)[~hit], w0.view(torch.int32)[~hit])


@pytest.mark.parametrize("io,cache_dtype", [(F32, BF16), (BF16, BF16), (F32, F32), (BF16, F32)])
@pytest.mark.parametrize("new", [[3, 0, 40, 1], [0, 0, 0, 0], [1, 1, 1, 1], [70, 5, 0, 0], [0] * 40 + [5] + [0] * 30 + [2, 1, 0]])
def test_append_ragged_prompts(pkg, eng, new, io, cache_dtype):
    heads, hk, page, dk = 4, 2, 16, 64
    lens = [(5 * i) % 23 for i in range(len(new))]
    cache, table, lengths = _pool(pkg, eng, lens, hk, page, dk, cache_dtype, room=max(new), track=True)
    start = np.concatenate([[2], 2 + np.cumsum(new)])  # two rows before the first sequence and three behind the last belong to nobody
    rows = int(start[-1]) + 3
    q, k, v = (torch.randn((rows, h, dk), device=eng.device).to(io) for h in (heads, hk, hk))
    cos, sin = _tables(eng, dk, 128)
    q_out = torch.full_like(q, 7.0)
    seq = np.repeat(np.arange(len(new)), new)
    pos = torch.from_numpy(np.concatenate([np.arange(n) + 3 * i % 11 for i, n in enumerate(new)] or [np.zeros(0)]).astype(np.int64))
    positions = torch.full((rows,), -9, dtype=torch.int32, device=eng.device)
    positions[2:rows - 3] = pos.int().to(eng.device)
    out = lengths.clone()
    got_q, n = eng.paged_append(cache, table, out, k, v, q=q, row_start=torch.from_numpy(start).int().to(eng.device), rope=(cos, sin), positions=positions,
                                q_out=q_out, lengths_out=out)
    eng.check_device_errors()
    assert n.data_ptr() == out.data_ptr() and n.tolist() == [a + b for a, b in zip(lens, new)]
    assert bool((got_q[:2] == 7).all()) and bool((got_q[rows - 3:] == 7).all())
    want, slack = _turned(q[2:rows - 3], cos.cpu()[pos], sin.cpu()[pos])
    assert _near(got_q[2:rows - 3], want, slack)
    want, slack = _turned(k[2:rows - 3], cos.cpu()[pos], sin.cpu()[pos])
    kc, vc = cache.k.cpu(), cache.v.cpu()
    for r, i in enumerate(seq):
        t = lens[i] + r + 2 - int(start[i])
        p, s = int(table[i, t // page]), t % page
        assert _near(kc[p, :, s], want[r], slack[r])
        assert torch.equal(vc[p, :, s], v[r + 2].to(cache_dtype).cpu())


@pytest.mark.parametrize("heads,hk,dk,n,io", [(64, 8, 256, 5, F32), (128, 1, 128, 700, F32), (8, 2, 100, 2500, BF16), (7, 1, 34, 3000, F32), (2, 1, 50, 900, BF16)])
def test_append_many_and_wide_tokens(pkg, eng, heads, hk, dk, n, io):
    """Rows too wide for shared memory, odd head sizes, and enough tokens for several per CTA (the last CTA partly filled)."""
    lens = [(7 * i) % 13 for i in range(n)]
    cache, table, lengths = _pool(pkg, eng, lens, hk, 16, dk, BF16, room=1)
    qkv = torch.randn((n, heads + 2 * hk, dk), device=eng.device).to(io)
    q, k, v = qkv.split([heads, hk, hk], 1)
    cos, sin = _tables(eng, dk, 16)
    got_q, new = eng.paged_append(cache, table, lengths, k, v, q=q, rope=(cos, sin))
    eng.check_device_errors()
    at = lengths.long()
    assert torch.equal(new, lengths + 1)
    want, slack = _turned(q, cos[at], sin[at])
    assert _near(got_q, want, slack)
    want, slack = _turned(k, cos[at], sin[at])
    rows = torch.arange(n, device=eng.device)
    page = table[rows, at // 16].long()
    assert _near(cache.k[page, :, at % 16, :dk], want, slack)
    assert torch.equal(cache.v[page, :, at % 16, :dk], v.to(BF16))
    assert not cache.k[page, :, at % 16, dk:].any() and not cache.v[page, :, at % 16, dk:].any()


def test_append_without_queries_rotation_or_alignment(pkg, eng):
    lens, hk, dk = [3, 9], 2, 64
    for io, cache_dtype in ((F32, F32), (BF16, BF16)):
        cache, table, lengths = _pool(pkg, eng, lens, hk, 4, dk, cache_dtype, room=1)
        odd = torch.randn(2 * (2 * hk * dk + 1) + 1, device=eng.device).to(io)[1:].view(2, 2 * hk * dk + 1)
        k, v = odd[:, :hk * dk].unflatten(1, (hk, dk)), odd[:, hk * dk:2 * hk * dk].unflatten(1, (hk, dk))
        q, n = eng.paged_append(cache, table, lengths, k, v, lengths_out=lengths)
        assert q is None and n is lengths and lengths.tolist() == [4, 10]
        for i, t in enumerate(lens):
            p, s = int(table[i, t // 4]), t % 4
            assert torch.equal(cache.k[p, :, s], k[i]) and torch.equal(cache.v[p, :, s], v[i])
        eng.check_device_errors()


def test_append_in_place_queries_idle_sequences_and_no_room(pkg, eng):
    lens, hk, dk, heads = [4, 8, 7, 2], 1, 64, 2
    cache, table, lengths = _pool(pkg, eng, lens, hk, 4, dk, BF16, room=0, extra_cols=0, spare=3)  # two pages per sequence: [1] is full
    table[0, 1] = cache.n_pages  # [0]'s next token falls on a page outside the pool
    k0 = cache.k.clone()
    cos, sin = _tables(eng, dk, 16)
    q = torch.randn((4, heads, dk), device=eng.device)
    q0 = q.clone()
    k, v = torch.randn((2, 4, hk, dk), device=eng.device)
    pos = torch.tensor([5, 6, -1, 15], dtype=torch.int32, device=eng.device)
    got, n = eng.paged_append(cache, table, lengths, k, v, q=q, rope=(cos, sin), positions=pos, q_out=q)
    with pytest.raises(pkg.NnbError, match="page id.*behind the end"):
        eng.check_device_errors()
    assert got.data_ptr() == q.data_ptr() and n.tolist() == [5, 8, 7, 3]
    assert torch.equal(q[:3], q0[:3])  # no place, no room, idle: not written
    want, slack = _turned(q0[3:], cos[15:16], sin[15:16])
    assert _near(q[3:], want, slack)
    changed = (cache.k.view(torch.int16) != k0.view(torch.int16)).any(-1).nonzero()
    assert changed.tolist() == [[int(table[3, 0]), 0, 2]]
    pos = torch.tensor([16, 0, 0, -2], dtype=torch.int32, device=eng.device)  # behind the tables; a negative one with row_start
    eng.paged_append(cache, table, torch.tensor([0, 0, 0, 0], dtype=torch.int32, device=eng.device), k, v, rope=(cos, sin), positions=pos,
                     row_start=torch.arange(5, dtype=torch.int32, device=eng.device))
    with pytest.raises(pkg.NnbError, match="position"):
        eng.check_device_errors()
    eng.check_device_errors()


# ------------------------------------------------------------------------------------------------ eviction
def _kept(w, n, budget, sinks, recent):
    """The definition: w (n) weights; positions in order."""
    if n <= budget:
        return np.arange(n)
    mid = np.arange(sinks, n - recent)
    score = np.where(np.isnan(w[mid]), -np.inf, w[mid].astype(np.float64))
    nan_last = np.lexsort((mid, np.isnan(w[mid]), -score))
    return np.sort(np.concatenate([np.arange(sinks), mid[nan_last[:budget - sinks - recent]], np.arange(n - recent, n)]))


@pytest.mark.parametrize("cache_dtype", [F32, BF16])
@pytest.mark.parametrize("lens,hk,page,dk,budget,sinks,recent,dst_page", [
    ([0, 1, 63, 64, 65, 200, 1500], 2, 16, 64, 64, 4, 16, 16), ([2500, 100], 3, 7, 100, 1024, 0, 0, 48), ([300, 33], 1, 16, 2, 32, 0, 32, 5),
    ([300, 33], 2, 16, 128, 32, 32, 0, 32), ([300], 2, 64, 64, 1, 0, 0, 1), ([300, 299], 2, 16, 64, 299, 150, 149, 16), ([9000], 2, 64, 128, 3000, 4, 500, 64),
    ([50, 60], 1, 16, 256, 5000, 10, 10, 16)])
@pytest.mark.parametrize("kind", ["random", "ties", "odd"])
def test_evict_keeps_the_heaviest(pkg, eng, lens, hk, page, dk, budget, sinks, recent, dst_page, cache_dtype, kind):
    cache, table, lengths = _pool(pkg, eng, lens, hk, page, dk, cache_dtype, seed=7, track=True)
    live = ~cache.weight.isnan()
    if kind == "ties":  # few distinct values, zeros of both signs among them
        cache.weight.copy_(torch.where(live, (cache.weight * 4).floor() / 4 * torch.where(cache.weight > 0.1, 1.0, -1.0), cache.weight))
    elif kind == "odd":  # negative, huge, tiny, infinite and NaN weights
        x = (cache.weight - 0.5) * 1e30
        x = torch.where(cache.weight > 0.9, torch.full_like(x, float("inf")), torch.where(cache.weight < 0.1, torch.full_like(x, float("-inf")), x))
        x = torch.where((cache.weight > 0.4) & (cache.weight < 0.5), (cache.weight - 0.45) * 1e-38, x)
        x = torch.where((cache.weight > 0.2) & (cache.weight < 0.25), torch.full_like(x, float("nan")), x)
        cache.weight.copy_(torch.where(live, x, cache.weight))
    src = [t.clone() for t in (cache.k, cache.v, cache.weight)]
    cols = (min(budget, max(lens) + page) + dst_page - 1) // dst_page + 1
    ids = torch.randperm(cols * len(lens) + 1, generator=torch.Generator().manual_seed(1))
    dst_table = ids[:cols * len(lens)].view(len(lens), cols).int().to(eng.device)
    shape = (len(ids), hk, dst_page, cache.pitch)
    dst = pkg.PagedCache(torch.full(shape, 3.0, device=eng.device, dtype=cache_dtype), torch.full(shape, 3.0, device=eng.device, dtype=cache_dtype), dk,
                         torch.full(shape[:3], 3.0, device=eng.device))
    n = eng.paged_evict(cache, table, lengths, dst, dst_table, budget=budget, sinks=sinks, recent=recent)
    eng.check_device_errors()
    assert n.tolist() == [min(t, budget) for t in lens]
    for now, was in zip((cache.k, cache.v, cache.weight), src):  # the source is only read
        assert torch.equal(now.view(torch.uint8), was.view(torch.uint8))
    written = torch.zeros(shape[:3], dtype=torch.bool)
    for i, t in enumerate(lens):
        pages = table[i].cpu().long()
        for h in range(hk):
            pos = np.arange(t)
            w = src[2].cpu()[pages[pos // page], h, pos % page].numpy()
            keep = _kept(w, t, budget, sinks, recent)
            sp, sa = pages[keep // page], torch.from_numpy(keep % page)
            r = np.arange(len(keep))
            dp, da = dst_table[i].cpu().long()[r // dst_page], torch.from_numpy(r % dst_page)
            written[dp, h, da] = True
            for now, was in ((dst.k, src[0]), (dst.v, src[1]), (dst.weight, src[2])):
                a, b = now.cpu()[dp, h, da], was.cpu()[sp, h, sa]
                assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), (i, h)
    rest = ~written
    assert bool((dst.k.cpu()[rest] == 3).all()) and bool((dst.v.cpu()[rest] == 3).all()) and bool((dst.weight.cpu()[rest] == 3).all())


def test_evict_within_one_pool_and_bad_pages(pkg, eng):
    """Source and destination pages in the same pool; a bad source page counts as zero, a bad destination page is not written."""
    lens = [40, 25]
    cache, table, lengths = _pool(pkg, eng, lens, 2, 8, 64, BF16, track=True, spare=6)
    free = [p for p in range(cache.n_pages) if p not in table.cpu().numpy()]
    dst_table = torch.tensor([free[:2], free[2:4]], dtype=torch.int32, device=eng.device)
    for t in (cache.k, cache.v, cache.weight):
        t[torch.tensor(free, device=eng.device)] = 0
    k0 = cache.k.clone()
    n = eng.paged_evict(cache, table, lengths, cache, dst_table, budget=16, recent=8)
    eng.check_device_errors()
    assert n.tolist() == [16, 16] and bool((cache.k[torch.tensor(free[:4], device=eng.device)] != 0).any())
    assert torch.equal(cache.k[table[0, 4].long(), :, 0:8].view(torch.int16)[:, :8], k0[table[0, 4].long(), :, 0:8].view(torch.int16)[:, :8])
    bad = table.clone()
    bad[0, 4] = -3  # the recent page
    eng.paged_evict(cache, bad, lengths, cache, dst_table, budget=16, recent=8)
    with pytest.raises(pkg.NnbError, match="page id"):
        eng.check_device_errors()
    assert bool((cache.k[free[1]] == 0).all())
    before = cache.k.clone()
    worse = dst_table.clone()
    worse[0, 0] = cache.n_pages
    eng.paged_evict(cache, table, lengths, cache, worse, budget=16, recent=8)
    with pytest.raises(pkg.NnbError, match="page id"):
        eng.check_device_errors()
    assert torch.equal(cache.k[free[0]], before[free[0]]) and bool((cache.k[free[1]] != 0).any())


# ------------------------------------------------------------------------------------------------ logits
def _adjusted(x, hist, n, prompt, window, rep, pres, freq, bias, words):
    """The definition for one sequence in f64, and a bound on the error before the last rounding: u per operation."""
    y = x.astype(np.float64)
    tol = np.zeros_like(y)
    if bias is not None:
        y = y + bias
        tol += U * np.abs(y)
    ids = hist[:n]
    ok = (ids >= 0) & (ids < len(y))
    recent = np.unique(ids[max(0, n - window) if window > 0 else 0:][ok[max(0, n - window) if window > 0 else 0:]])
    if rep is not None and rep > 0 and rep != 1:
        f = np.where(y[recent] > 0, 1 / np.float64(rep), np.float64(rep))
        y[recent] *= f
        tol[recent] = tol[recent] * f + U * np.abs(y[recent])
    toks, counts = np.unique(ids[prompt:][ok[prompt:]], return_counts=True)
    if pres is not None or freq is not None:
        fr, pr = np.float64(freq or 0), np.float64(pres or 0)
        y[toks] -= fr * counts + pr
        tol[toks] += 3 * U * (np.abs(fr) * counts + np.abs(pr)) + U * np.abs(y[toks])
    if words is not None:
        bits = np.unpackbits(words.view(np.uint8), bitorder="little")[:len(y)]
        y[bits == 0] = -np.inf
    return y, tol


def _check_logits(eng, x, out, kw, window=0):
    x, got = x.float().cpu().numpy(), out.cpu()
    num = {k: v.cpu().numpy() for k, v in kw.items() if v is not None}
    for s in range(x.shape[0]):
        hist = num.get("history")
        cap = hist.shape[1] if hist is not None else 0
        n = int(np.clip(num["history_len"][s], 0, cap)) if hist is not None else 0
        one = {k: float(num[k][s]) if k in num else None for k in ("repeat_penalty", "presence_penalty", "frequency_penalty")}
        row = lambda k: None if k not in num else num[k] if num[k].ndim == 1 else num[k][s]  # noqa: E731
        y, tol = _adjusted(x[s], hist[s] if hist is not None else np.zeros(0, np.int32), n, int(max(num["prompt_len"][s], 0)) if "prompt_len" in num else 0, window,
                           one["repeat_penalty"], one["presence_penalty"], one["frequency_penalty"], row("bias"), row("allowed"))
        g = got[s].double().numpy()
        inf = np.isinf(y)
        assert np.array_equal(g[inf], y[inf]) and not np.isinf(g[~inf]).any()
        err = np.abs(g[~inf] - y[~inf])
        bound = tol[~inf] + HALF[out.dtype] * (np.abs(y[~inf]) + tol[~inf])
        assert (err <= bound).all(), (s, (err - bound).max())


def _logit_case(eng, n, v, hist, io, seed=0):
    g = torch.Generator(device=eng.device).manual_seed(seed)
    rng = np.random.default_rng(seed)
    x = (torch.randn((n, v), generator=g, device=eng.device) * 3).to(io)
    ids = rng.integers(-1, min(v, 50) + 1, (n, hist)).astype(np.int32)
    ids[:, ::5] = rng.integers(0, v, ids[:, ::5].shape)
    lens = rng.integers(0, hist + 1, n).astype(np.int32)
    lens[:2] = [hist + 3, -1][:min(n, 2)]
    dev = lambda a: torch.from_numpy(a).to(eng.device)  # noqa: E731
    return x, dict(history=dev(ids), history_len=dev(lens), prompt_len=dev((np.maximum(lens, 0) // 3).astype(np.int32)),
                   repeat_penalty=dev(rng.choice([0.0, 1.0, 1.3, 0.7, -1.0], n).astype(np.float32)), presence_penalty=dev(rng.normal(size=n).astype(np.float32)),
                   frequency_penalty=dev(rng.normal(size=n).astype(np.float32)), bias=dev(rng.normal(size=v).astype(np.float32)),
                   allowed=dev(rng.integers(-2**31, 2**31, (n, (v + 31) // 32)).astype(np.int32)))


@pytest.mark.parametrize("io", [F32, BF16])
@pytest.mark.parametrize("n,v,hist", [(1, 1, 3), (3, 31, 40), (2, 4096, 10), (5, 4097, 300), (9, 32002, 2000), (3, 128256, 5000), (40, 777, 64), (300, 1000, 33)])
def test_adjust_logits_matches_the_definition(pkg, eng, n, v, hist, io):
    x, kw = _logit_case(eng, n, v, hist, io, seed=v)
    x0 = x.clone()
    for window in (0, 7, 10**9):
        _check_logits(eng, x, eng.adjust_logits(x, repeat_window=window, **kw), kw, window)
    assert torch.equal(x, x0)
    for drop in (["bias", "allowed"], ["history", "history_len", "prompt_len", "repeat_penalty", "presence_penalty", "frequency_penalty"], ["prompt_len"],
                 ["repeat_penalty", "bias"], ["presence_penalty", "frequency_penalty", "allowed"], ["frequency_penalty"]):
        some = {k: (None if k in drop else t) for k, t in kw.items()}
        _check_logits(eng, x, eng.adjust_logits(x, **some), some)
    some = {k: (None if k in ("bias", "allowed") else t) for k, t in kw.items()}
    want = eng.adjust_logits(x, **some)
    y = x.clone()
    assert eng.adjust_logits(y, out=y, **some).data_ptr() == y.data_ptr() and torch.equal(y, want)  # in place, penalties only
    y = x.clone()
    assert torch.equal(eng.adjust_logits(y, out=y, **kw), eng.adjust_logits(x, **kw))


@pytest.mark.parametrize("io", [F32, BF16])
def test_adjust_logits_strides_shared_rows_and_odd_values(pkg, eng, io):
    n, v = 4, 1003
    x, kw = _logit_case(eng, n, v, 50, io)
    wide = torch.zeros((n, v + 13), device=eng.device, dtype=io)
    wide[:, 5:5 + v] = x
    out = torch.full((n, v + 9), 7.0, device=eng.device, dtype=io)
    got = eng.adjust_logits(wide[:, 5:5 + v], out=out[:, 2:2 + v], **kw)
    want = eng.adjust_logits(x, **kw)
    assert torch.equal(got, want) and bool((out[:, :2] == 7).all()) and bool((out[:, 2 + v:] == 7).all())
    assert torch.equal(eng.adjust_logits(wide[:, 5:5 + v], out=wide[:, 5:5 + v], **kw), want)  # in place in a wider matrix
    rows = dict(kw, bias=torch.randn((n, v), device=eng.device), allowed=kw["allowed"][0].contiguous())
    _check_logits(eng, x, eng.adjust_logits(x, **rows), rows)
    # an infinite or NaN logit in a masked place is -inf, an infinite one elsewhere stays
    y = x.clone()
    y[:, ::3] = float("nan")
    y[:, 1::3] = float("-inf")
    none = torch.zeros_like(kw["allowed"])
    assert bool((eng.adjust_logits(y, **dict(kw, allowed=none)) == float("-inf")).all())  # a row whose mask leaves nothing
    got = eng.adjust_logits(y, **dict(kw, allowed=torch.full_like(none, -1)))
    assert bool((got[:, 1::3] == float("-inf")).all()) and bool(got[:, ::3].isnan().all()) and not got[:, 2::3].isnan().any()


# ------------------------------------------------------------------------------------------------ as they are used
def test_refusals_of_the_python_entry_points(pkg, eng):
    cache, table, lengths = _pool(pkg, eng, [5, 6], 2, 4, 64, BF16, track=False)
    q, k = torch.zeros((2, 4, 64), device=eng.device), torch.zeros((2, 2, 64), device=eng.device)
    bad = [lambda: eng.paged_attention_decode(cache, table, lengths, q, accumulate=True), lambda: eng.paged_attention_decode(cache, table, lengths, q[:1]),
           lambda: eng.paged_attention_decode(cache, table, lengths, q[..., :32]), lambda: eng.paged_attention_decode(cache, table, lengths, q[:, :3]),
           lambda: eng.paged_attention_decode(cache, table, lengths.long(), q), lambda: eng.paged_attention_decode(cache, table.cpu(), lengths, q),
           lambda: eng.paged_attention_decode(cache, table, lengths, q.half()), lambda: eng.paged_attention_decode(cache, table.t(), lengths, q),
           lambda: eng.paged_attention_decode(cache, table, lengths, q.transpose(1, 2)), lambda: eng.paged_append(cache, table, lengths, k, k[:1]),
           lambda: eng.paged_append(cache, table, lengths, k[:1], k[:1]), lambda: eng.paged_append(cache, table, lengths, k, k.bfloat16()),
           lambda: eng.paged_append(cache, table, lengths, q, q), lambda: eng.paged_append(cache, table, lengths, k, k, q=q[:1]),
           lambda: eng.paged_append(cache, table, lengths, k, k, rope=(k, k)), lambda: eng.paged_append(cache, table, lengths, k, k, positions=lengths[:1]),
           lambda: eng.paged_evict(cache, table, lengths, cache, table, budget=4), lambda: eng.adjust_logits(q), lambda: eng.adjust_logits(q[0], bias=q[0, :, 0]),
           lambda: eng.adjust_logits(q[0], repeat_penalty=q[0, :, 0].contiguous()), lambda: eng.adjust_logits(q[0], history=table), lambda: eng.adjust_logits(q[0].half())]
    for call in bad:
        with pytest.raises(pkg.NnbError):
            call()
    none = torch.empty((0, 3), dtype=torch.int32, device=eng.device)
    assert eng.paged_attention_decode(cache, none, lengths[:0], q[:0])[0].shape == (0, 4, 64)  # an empty batch is no error
    assert eng.paged_append(cache, none, lengths[:0], k[:0], k[:0], q=q[:0])[1].shape == (0,)
    assert eng.adjust_logits(q[0][:0]).shape == (0, 64)
    eng.check_device_errors()


class _Model:
    """The serving loop in f64: a list of rows per (sequence, KV head), everything by definition."""

    def __init__(self, n, hk, dk, cos, sin):
        self.rows = [[[] for _ in range(hk)] for _ in range(n)]
        self.hk, self.dk, self.cos, self.sin = hk, dk, cos.cpu().double(), sin.cpu().double()

    def turn(self, x, p):
        a, b = x.chunk(2, -1)
        return torch.cat([a * self.cos[p] - b * self.sin[p], b * self.cos[p] + a * self.sin[p]], -1)

    def step(self, i, q, k, v, pos, kind):
        for h in range(self.hk):
            self.rows[i][h].append([self.turn(k[h], pos).to(kind).double(), v[h].to(kind).double(), 0.0])
        g = q.shape[0] // self.hk
        out = torch.zeros_like(q)
        for h in range(self.hk):
            kk, vv = torch.stack([r[0] for r in self.rows[i][h]]), torch.stack([r[1] for r in self.rows[i][h]])
            p = torch.softmax(self.turn(q[h * g:(h + 1) * g], pos) @ kk.t() * self.dk ** -0.5, -1)
            out[h * g:(h + 1) * g] = p @ vv
            for r, w in zip(self.rows[i][h], p.sum(0).tolist()):
                r[2] += w
        return out


@pytest.mark.parametrize("cache_dtype", [F32, BF16])
def test_a_serving_loop(pkg, eng, cache_dtype):
    """Prompts enter, tokens are decoded with their weights accumulated, the caches are cut down and decoding goes on with the
    true rotary positions; the logits of each step are adjusted by the tokens so far."""
    n, heads, hk, dk, page, budget = 3, 8, 2, 64, 4, 12
    cos, sin = _tables(eng, dk, 64)
    rng = torch.Generator().manual_seed(0)
    normal = lambda *s: torch.randn(s, generator=rng)  # noqa: E731
    cache = pkg.PagedCache.empty(40, hk, page, dk, dtype=cache_dtype, device=eng.device, track_weight=True)
    free = list(range(40))
    table = torch.tensor([[free.pop() for _ in range(6)] for _ in range(n)], dtype=torch.int32, device=eng.device)
    lengths = torch.zeros(n, dtype=torch.int32, device=eng.device)
    model = _Model(n, hk, dk, cos, sin)
    prompts = [5, 1, 9]
    k, v, q = normal(sum(prompts), hk, dk), normal(sum(prompts), hk, dk), normal(sum(prompts), heads, dk)
    start = torch.tensor([0, 5, 6, 15], dtype=torch.int32, device=eng.device)
    dev = eng.device
    eng.paged_append(cache, table, lengths, k.to(dev), v.to(dev), row_start=start, rope=(cos, sin), lengths_out=lengths)
    r = 0
    for i, m in enumerate(prompts):
        for t in range(m):
            for h in range(hk):
                model.rows[i][h].append([model.turn(k[r, h].double(), t).to(cache_dtype).double(), v[r, h].to(cache_dtype).double(), 0.0])
            r += 1
    pos = torch.tensor(prompts, dtype=torch.int32, device=dev)
    history = torch.zeros((n, 64), dtype=torch.int32, device=dev)
    penalty = torch.tensor([1.2, 1.5, 2.0], device=dev)
    # the f64 model rounds its keys from f64, the engine from f32: a key may fall to the other side, one step of the type away
    step = 2 * HALF[cache_dtype] if cache_dtype == BF16 else 1e-5
    for s in range(12):
        q, k, v = normal(n, heads, dk), normal(n, hk, dk), normal(n, hk, dk)
        if s == 5:  # back to the budget
            new_table = torch.tensor([[free.pop() for _ in range(4)] for _ in range(n)], dtype=torch.int32, device=dev)
            lengths = eng.paged_evict(cache, table, lengths, cache, new_table, budget=budget, sinks=1, recent=3)
            free += table.flatten().tolist()
            table = torch.cat([new_table, torch.tensor([[free.pop(0) for _ in range(2)] for _ in range(n)], dtype=torch.int32, device=dev)], 1)
            for i in range(n):
                for h in range(hk):
                    rows = model.rows[i][h]
                    keep = _kept(np.array([x[2] for x in rows]), len(rows), budget, 1, 3)
                    model.rows[i][h] = [rows[j] for j in keep]
        qd, _ = eng.paged_append(cache, table, lengths, k.to(dev), v.to(dev), q=q.to(dev), rope=(cos, sin), positions=pos, lengths_out=lengths)
        out, _ = eng.paged_attention_decode(cache, table, lengths, qd, accumulate=True)
        eng.check_device_errors()
        logits = out.reshape(n, -1)
        for i in range(n):
            want = model.step(i, q[i].double(), k[i].double(), v[i].double(), int(pos[i]), cache_dtype)
            # one step of a key changes a score by at most step * |q||k| / sqrt(dk) (rarely, in few features); values exactly rounded
            assert (out[i].cpu().double() - want).abs().max() <= 8 * step * max(1.0, want.abs().max().item()), (s, i)
        assert lengths.tolist() == [len(model.rows[i][0]) for i in range(n)]
        length = torch.full((n,), s, dtype=torch.int32, device=dev)
        before = logits.clone()
        after = eng.adjust_logits(logits, history=history, history_len=length, repeat_penalty=penalty)
        kw = dict(history=history, history_len=length, repeat_penalty=penalty)
        _check_logits(eng, before, after, kw)
        history[:, s] = after.argmax(-1).int()
        pos += 1


@pytest.mark.parametrize("cols", [1, 150])  # a short table (a cluster per item) and a long one (workers and a joining launch)
def test_captured_steps_follow_lengths_and_tables(pkg, eng, cols):
    """append, decode (weights accumulated), evict and adjust_logits captured once on a side stream, replayed with other lengths,
    tables and inputs; two graphs captured from the same calls do not disturb each other."""
    n, heads, hk, dk, page = 4, 8, 2, 128, 16
    lens = [40, 3, 0, 700]
    cos, sin = _tables(eng, dk, 1024)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())

    def state(seed):
        cache, table, lengths = _pool(pkg, eng, lens, hk, page, dk, BF16, seed=seed, room=64, track=True, extra_cols=cols)
        q, k, v = (torch.randn((n, h, dk), device=eng.device) for h in (heads, hk, hk))
        dst = pkg.PagedCache.empty(8, hk, page, dk, device=eng.device, track_weight=True)
        dt = torch.arange(8, dtype=torch.int32, device=eng.device).view(4, 2)
        return dict(cache=cache, table=table, lengths=lengths, q=q, k=k, v=v, dst=dst, dt=dt)

    def step(e, s):
        qd, new = e.paged_append(s["cache"], s["table"], s["lengths"], s["k"], s["v"], q=s["q"], rope=(cos, sin))
        out, lse = e.paged_attention_decode(s["cache"], s["table"], new, qd, accumulate=True)
        left = e.paged_evict(s["cache"], s["table"], new, s["dst"], s["dt"], budget=32, sinks=2, recent=8)
        y = e.adjust_logits(out.reshape(n, -1), history=s["table"], history_len=new, repeat_penalty=torch.full((n,), 1.5, device=eng.device))
        return dict(q=qd, new=new, out=out, lse=lse, left=left, y=y)

    states, twins = [state(1), state(2)], [state(1), state(2)]
    with torch.cuda.stream(side):
        e2 = pkg.Engine(0)
        for s in (state(3),):
            step(e2, s)  # loads the kernels before capture
        side.synchronize()
        graphs, outs = [], []
        for s in states:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                outs.append(step(e2, s))
            graphs.append(g)
    torch.cuda.synchronize()
    for a, b in zip(states, twins):  # capturing ran nothing; the twins get the same inputs
        for m in ("q", "k", "v"):
            b[m].copy_(a[m])
    for turn in range(3):
        if turn:
            for a, b in zip(states, twins):
                for s in (a, b):
                    # shorter sequences, then the same ones in another order (every position read holds a number)
                    s["lengths"].copy_(torch.tensor([30, 3, 0, 64] if turn == 1 else [64, 30, 3, 0], dtype=torch.int32))
                    s["table"].copy_(s["table"] if turn == 1 else s["table"].roll(1, 0))
                    s["q"].mul_(0.5)
        other = torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.stream(other):
            graphs[1].replay()  # at the same time as the other graph
        with torch.cuda.stream(side):
            graphs[0].replay()
        torch.cuda.synchronize()
        for s, t, o in zip(states, twins, outs):
            want = step(eng, t)
            torch.cuda.synchronize()
            for m in want:
                assert torch.equal(o[m], want[m]), (turn, m)
            assert torch.equal(s["cache"].weight.nan_to_num(7.0), t["cache"].weight.nan_to_num(7.0))
            assert torch.equal(s["dst"].k, t["dst"].k)
    e2.close()


def test_calls_follow_torchs_current_stream(pkg, eng):
    """The engine launches on the default stream; a caller inside another stream's context gets its results in order."""
    cache, table, lengths = _pool(pkg, eng, [600, 30], 2, 16, 64, BF16)
    side = torch.cuda.Stream()
    big = torch.randn((4096, 4096), device=eng.device)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        x = big
        for _ in range(4):
            x = (x @ big).clamp(-1, 1)
        q = x.flatten()[:2 * 4 * 64].view(2, 4, 64).clone()
        out, lse = eng.paged_attention_decode(cache, table, lengths, q)
        y = eng.adjust_logits(out.view(2, -1), bias=out.view(2, -1)[0].contiguous())
        got = [t.clone() for t in (q, out, lse, y)]
    side.synchronize()
    q, out, lse, y = got
    _check_decode(cache, table, [600, 30], q, out, lse)
    assert torch.equal(y, out.view(2, -1) + out.view(2, -1)[0])


def test_an_engine_on_its_own_stream_is_ordered_with_torchs(pkg):
    """The engine launches on its own stream: inputs made and outputs read on torch's current stream still come in order."""
    e = pkg.Engine(0, use_torch_stream=False)
    e.set_stream(None)
    dev = e.device
    big = torch.randn((4096, 4096), device=dev)
    cache, table, lengths = _pool(pkg, e, [600, 30], 2, 16, 64, BF16)
    want = None
    for _ in range(5):
        x = big
        for _ in range(4):
            x = (x @ big).clamp(-1, 1)  # some milliseconds of work before the queries exist
        q = x.flatten()[:2 * 4 * 64].view(2, 4, 64).clone()
        out, lse = e.paged_attention_decode(cache, table, lengths, q)
        got = out.clone()
        del out, lse
        torch.empty((2, 4, 64), device=dev).fill_(9.0)  # reuses freed memory at once
        torch.cuda.synchronize()
        want = got if want is None else want
        assert torch.equal(got, want)
    out, lse = e.paged_attention_decode(cache, table, lengths, q)
    _check_decode(cache, table, [600, 30], q, out, lse)
    e.close()
