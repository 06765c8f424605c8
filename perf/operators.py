"""The paged-cache serving operators, as they are measured: appending to a paged key-value cache, attention of one
new token per sequence over it (with the accumulation of attention weights), eviction by those weights, and the
adjustment of logits before sampling.

`own` selects the side: False computes each operator from elementary torch operations, True through this
framework's Engine.  Both sides take what `prepare` makes.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
ITEM = {"f32": 4, "bf16": 2}


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one decode step of the 1B policy (16 heads of 128): 128 sequences, one new token each
        dict(name="append_step", op="append", n_seq=128, n_head=16, n_kv=16, dk=128, page=16, lo=128, hi=640, new_lo=1, new_hi=1,
             io="f32", cache="bf16"),
        # eight ragged prompts entering a grouped-query cache (20 heads on 5 key / value heads of 128)
        dict(name="append_prompts", op="append", n_seq=8, n_head=20, n_kv=5, dk=128, page=64, lo=0, hi=0, new_lo=100, new_hi=2000,
             io="bf16", cache="bf16"),
        # the smallest call: a single user, a short context, latency counts
        dict(name="decode_single", op="decode", n_seq=1, n_head=20, n_kv=5, dk=128, page=16, lo=700, hi=700, io="f32", cache="bf16",
             track=False),
        # a decode step of the 1B policy: multi-head attention, short ragged contexts, one slot idle
        dict(name="decode_batch", op="decode", n_seq=128, n_head=16, n_kv=16, dk=128, page=16, lo=0, hi=640, io="f32", cache="bf16",
             track=False),
        # the 3B decode shape: 32 heads of 100, a head size that is no power of two
        dict(name="decode_heads100", op="decode", n_seq=32, n_head=32, n_kv=32, dk=100, page=32, lo=256, hi=2048, io="f32",
             cache="bf16", track=False),
        # few users with long documents: the cache's length is the only parallelism
        dict(name="decode_long", op="decode", n_seq=3, n_head=20, n_kv=5, dk=128, page=64, lo=9000, hi=65536, io="bf16", cache="bf16",
             track=False),
        # the largest call: a full serving batch, grouped queries, bf16 in and out
        dict(name="decode_large", op="decode", n_seq=64, n_head=32, n_kv=8, dk=128, page=64, lo=1000, hi=8192, io="bf16", cache="bf16",
             track=False),
        # an f32 cache (the GPT-2-small heads) whose attention weights are accumulated for eviction
        dict(name="decode_tracked", op="decode", n_seq=16, n_head=12, n_kv=12, dk=64, page=16, lo=300, hi=4096, io="f32", cache="f32",
             track=True),
        # caches of a batch brought back to 1024 tokens
        dict(name="evict_batch", op="evict", n_seq=32, n_kv=5, dk=128, page=16, lo=900, hi=2048, budget=1024, sinks=4, recent=256,
             cache="bf16"),
        # two long contexts cut to an eighth
        dict(name="evict_long", op="evict", n_seq=2, n_kv=8, dk=128, page=64, lo=50001, hi=65536, budget=8192, sinks=16, recent=1024,
             cache="bf16"),
        # a serving batch with the 128256-token vocabulary, all adjustments on
        dict(name="logits_batch", op="logits", n_seq=128, vocab=128256, hist=2048, io="f32", window=0, bias=True, mask=True),
        # a few users, 32000 tokens, penalties only
        dict(name="logits_small", op="logits", n_seq=4, vocab=32000, hist=640, io="bf16", window=128, bias=False, mask=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "decode", "decode", "evict", "logits"])
    page = rng.choice([8, 16, 32, 64, 48])
    n_kv, group = rng.choice([(1, 8), (5, 4), (8, 4), (8, 1), (12, 1), (16, 1), (32, 1), (4, 7), (2, 16)])
    dk = rng.choice([64, 100, 128, 80])
    if op == "append":
        cache = rng.choice(["bf16", "bf16", "f32"])
        io = rng.choice(["f32", "bf16"])
        if rng.random() < 0.5:
            n = _log(rng, 1, 512)
            return dict(op=op, n_seq=n, n_head=n_kv * group, n_kv=n_kv, dk=dk, page=page, lo=0, hi=_log(rng, 16, 1024), new_lo=1, new_hi=1,
                        io=io, cache=cache)
        n = _log(rng, 1, 16)
        return dict(op=op, n_seq=n, n_head=n_kv * group, n_kv=n_kv, dk=dk, page=page, lo=0, hi=_log(rng, 1, 300), new_lo=1,
                    new_hi=_log(rng, 2, 2000), io=io, cache=cache)
    if op == "decode":
        cache = rng.choice(["bf16", "bf16", "bf16", "f32"])
        n = _log(rng, 1, 256)
        # at most a quarter of the largest listed case's cache
        most = int(64 * 8192 * 8 * 128 / 4 / (n * n_kv * dk * (2 if cache == "f32" else 1)))
        hi = _log(rng, 33, max(40, min(65536, most)))
        lo = rng.choice([0, 1, hi // 2, hi])
        return dict(op=op, n_seq=n, n_head=n_kv * group, n_kv=n_kv, dk=dk, page=page, lo=lo, hi=hi, io=rng.choice(["f32", "bf16"]),
                    cache=cache, track=rng.random() < 0.3)
    if op == "evict":
        n = _log(rng, 1, 64)
        hi = _log(rng, 64, max(65, min(32768, int(2 * 65536 * 8 * 128 / (n * n_kv * dk)))))
        budget = max(8, int(hi * rng.uniform(0.1, 0.9)))
        sinks = rng.choice([0, 1, 4])
        return dict(op=op, n_seq=n, n_kv=n_kv, dk=dk, page=page, lo=hi // 2, hi=hi, budget=budget, sinks=sinks,
                    recent=rng.choice([0, 1, max(0, budget // 4 - sinks), budget - sinks]), cache=rng.choice(["bf16", "bf16", "f32"]))
    return dict(op="logits", n_seq=_log(rng, 1, 128), vocab=rng.choice([32000, 32002, 128256, 10000, 50257]), hist=_log(rng, 1, 4096),
                io=rng.choice(["f32", "bf16"]), window=rng.choice([0, 64]), bias=rng.random() < 0.5, mask=rng.random() < 0.5)


# ------------------------------------------------------------------------------------------------ inputs
def _spread(lo, hi, n):
    """n lengths from lo to hi, evenly spread: which sequence has which goes by the seed, their sum does not."""
    return [int(round(lo + (hi - lo) * (i / (n - 1) if n > 1 else 1.0))) for i in range(n)]


def _pitch(dk):
    return (dk + 7) // 8 * 8


def _tables(host, lengths, page, max_pages, first=0):
    """Page ids of each sequence, scattered over the pool; entries behind a sequence's last page are -1."""
    used = [(t + page - 1) // page for t in lengths]
    ids = host.permutation(sum(used)) + first
    table = np.full((len(lengths), max_pages), -1, np.int32)
    at = 0
    for i, u in enumerate(used):
        table[i, :u] = ids[at:at + u]
        at += u
    return table, max(1, sum(used)) + first


def prepare(case, seed):
    c, dev = dict(case), torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(int(seed))
    host = np.random.RandomState(int(seed) % (2**31))
    s = {"case": c}

    def normal(shape, kind, scale=1.0):
        return (torch.randn(shape, generator=gen, device=dev) * scale).to(DTYPES[kind])

    def ints(a):
        return torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(dev)

    if c["op"] == "logits":
        n, v = c["n_seq"], c["vocab"]
        s["logits"] = normal((n, v), c["io"], 3.0)
        hist = np.minimum(host.zipf(1.3, (n, c["hist"])), v) - 1  # natural text repeats few tokens often
        lens = np.array(_spread(max(1, c["hist"] // 2), c["hist"], n))[host.permutation(n)]
        s["history"], s["history_len"] = ints(hist), ints(lens)
        s["prompt_len"] = ints(lens // 3)
        for name, lo, hi in (("repeat_penalty", 1.0, 1.5), ("presence_penalty", 0.0, 1.0), ("frequency_penalty", 0.0, 0.5)):
            s[name] = torch.from_numpy(host.uniform(lo, hi, n).astype(np.float32)).to(dev)
        s["bias"] = normal((v,), "f32") if c["bias"] else None
        # one bit per token, 1 = allowed; each row has a grammar of its own
        s["allowed"] = torch.randint(-2**31, 2**31, (n, (v + 31) // 32), generator=gen, device=dev).to(torch.int32) if c["mask"] else None
        return s

    n, hk, dk, page, pitch = c["n_seq"], c["n_kv"], c["dk"], c["page"], _pitch(c["dk"])
    order = host.permutation(n)
    lens = np.array(_spread(c["lo"], c["hi"], n))[order]
    if c["op"] == "append":
        new = np.array(_spread(c["new_lo"], c["new_hi"], n))[host.permutation(n)]
        total = lens + new
    else:
        new, total = None, lens
    max_pages = max(1, (int(total.max()) + page - 1) // page)
    table, n_pages = _tables(host, [int(t) for t in total], page, max_pages)
    s["table"], s["lengths"] = ints(table), ints(lens)
    s["k"] = normal((n_pages, hk, page, pitch), c["cache"])
    s["v"] = normal((n_pages, hk, page, pitch), c["cache"])
    if pitch > dk:
        s["k"][..., dk:] = 0
        s["v"][..., dk:] = 0
    if c["op"] == "append":
        rows = int(new.sum())
        s["row_start"] = None if c["new_hi"] == 1 else ints(np.concatenate([[0], np.cumsum(new)]))
        # the projections of the new tokens come as one matrix, as a fused q|k|v product leaves them
        qkv = normal((rows, c["n_head"] + 2 * hk, dk), c["io"])
        s["q_new"], s["k_new"], s["v_new"] = qkv.split([c["n_head"], hk, hk], dim=1)
        ctx = int(total.max())
        ang = torch.arange(ctx, device=dev, dtype=torch.float64)[:, None] * (10000.0 ** (-2.0 * torch.arange(dk // 2, device=dev, dtype=torch.float64) / dk))
        s["cos"], s["sin"] = ang.cos().float(), ang.sin().float()
    elif c["op"] == "decode":
        s["q"] = normal((n, c["n_head"], dk), c["io"], 1.5)
        s["weight"] = torch.rand((n_pages, hk, page), generator=gen, device=dev) if c["track"] else None
    else:
        # accumulated weights fall off steeply, and what was never attended to has exactly none
        w = torch.randn((n_pages, hk, page), generator=gen, device=dev).mul_(2.0).exp_()
        s["weight"] = torch.where(w < 0.2, torch.zeros_like(w), w)
        dst, dst_pages = _tables(host, [c["budget"]] * n, page, (c["budget"] + page - 1) // page)
        s["dst_table"] = ints(dst)
        s["dst_k"], s["dst_v"] = torch.zeros((dst_pages, hk, page, pitch), device=dev, dtype=DTYPES[c["cache"]]), torch.zeros(
            (dst_pages, hk, page, pitch), device=dev, dtype=DTYPES[c["cache"]])
        s["dst_weight"] = torch.zeros((dst_pages, hk, page), device=dev)
    return s


# ------------------------------------------------------------------------------------------------ the two sides
_ENGINE = []


def _engine():
    if not _ENGINE:
        from __graft_entry__ import load_package

        pkg = load_package()
        _ENGINE.append((pkg, pkg.Engine(0)))
    return _ENGINE[0]


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    return {"append": _plain_append, "decode": _plain_decode, "evict": _plain_evict, "logits": _plain_logits}[op](state)


def _own(s):
    c = s["case"]
    pkg, eng = _engine()
    if c["op"] == "append":
        cache = pkg.PagedCache(s["k"], s["v"], c["dk"])
        q, lengths = eng.paged_append(cache, s["table"], s["lengths"], s["k_new"], s["v_new"], q=s["q_new"], row_start=s["row_start"],
                                      rope=(s["cos"], s["sin"]))
        return {"q": q, "k": s["k"], "v": s["v"], "lengths": lengths}
    if c["op"] == "decode":
        weight = s["weight"].clone() if c["track"] else None  # the call adds to it in place
        cache = pkg.PagedCache(s["k"], s["v"], c["dk"], weight)
        out, lse = eng.paged_attention_decode(cache, s["table"], s["lengths"], s["q"], accumulate=c["track"])
        return {"out": out, "lse": lse, "weight": weight} if c["track"] else {"out": out, "lse": lse}
    if c["op"] == "evict":
        src = pkg.PagedCache(s["k"], s["v"], c["dk"], s["weight"])
        dst = pkg.PagedCache(s["dst_k"], s["dst_v"], c["dk"], s["dst_weight"])
        lengths = eng.paged_evict(src, s["table"], s["lengths"], dst, s["dst_table"], budget=c["budget"], sinks=c["sinks"], recent=c["recent"])
        return {"k": s["dst_k"], "v": s["dst_v"], "weight": s["dst_weight"], "lengths": lengths}
    return eng.adjust_logits(s["logits"], history=s["history"], history_len=s["history_len"], prompt_len=s["prompt_len"],
                             repeat_window=c["window"], repeat_penalty=s["repeat_penalty"], presence_penalty=s["presence_penalty"],
                             frequency_penalty=s["frequency_penalty"], bias=s["bias"], allowed=s["allowed"])


def _rotate(x, cos, sin):
    """Pairs (j, j + dk/2) of each head turned by the angle of the row's position."""
    a, b = x.float().chunk(2, dim=-1)
    cos, sin = cos[:, None], sin[:, None]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)


def _plain_append(s):
    c = s["case"]
    rows, lens, dev = s["k_new"].shape[0], s["lengths"].long(), s["k"].device
    row = torch.arange(rows, device=dev)
    if s["row_start"] is None:
        seq, index = row, torch.zeros_like(row)
        count = torch.ones_like(lens)
    else:
        start = s["row_start"].long()
        seq = torch.searchsorted(start, row, right=True) - 1
        index = row - start[seq]
        count = start[1:] - start[:-1]
    slot = lens[seq] + index
    cos, sin = s["cos"][slot], s["sin"][slot]
    page, at = s["table"][seq, slot // c["page"]].long(), slot % c["page"]
    dk = c["dk"]
    s["k"][page, :, at, :dk] = _rotate(s["k_new"], cos, sin).to(s["k"].dtype)
    s["v"][page, :, at, :dk] = s["v_new"].to(s["v"].dtype)
    return {"q": _rotate(s["q_new"], cos, sin).to(s["q_new"].dtype), "k": s["k"], "v": s["v"], "lengths": (lens + count).int()}


def _plain_decode(s):
    c = s["case"]
    n, hk, dk = c["n_seq"], c["n_kv"], c["dk"]
    group = c["n_head"] // hk
    table = s["table"].long().clamp(min=0)
    cap = table.shape[1] * c["page"]
    live = torch.arange(cap, device=table.device)[None] < s["lengths"][:, None]
    keys = s["k"][table][..., :dk].float().permute(0, 2, 1, 3, 4).reshape(n, hk, cap, dk)
    q = s["q"].float().view(n, hk, group, dk) / math.sqrt(dk)
    x = torch.matmul(q, keys.transpose(-1, -2)).masked_fill(~live[:, None, None], -math.inf)
    del keys
    top = x.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = torch.exp(x - top)
    total = p.sum(-1, keepdim=True)
    p = torch.where(total > 0, p / total, torch.zeros_like(p))
    values = s["v"][table][..., :dk].float().permute(0, 2, 1, 3, 4).reshape(n, hk, cap, dk)
    values = torch.where(live[:, None, :, None], values, torch.zeros_like(values))
    out = torch.matmul(p, values).view(n, c["n_head"], dk).to(s["q"].dtype)
    lse = (top + torch.log(total)).view(n, c["n_head"])
    if not c["track"]:
        return {"out": out, "lse": lse}
    seen = p.sum(2).view(n, hk, table.shape[1], c["page"]).permute(0, 2, 1, 3)
    weight = s["weight"].clone()
    weight.index_add_(0, table.reshape(-1), seen.reshape(-1, hk, c["page"]))
    return {"out": out, "lse": lse, "weight": weight}


def _plain_evict(s):
    c = s["case"]
    n, hk, page, budget = c["n_seq"], c["n_kv"], c["page"], c["budget"]
    dev = s["k"].device
    table = s["table"].long().clamp(min=0)
    cap = table.shape[1] * page
    lens = s["lengths"].long()[:, None]
    at = torch.arange(cap, device=dev)[None]
    weight = s["weight"][table].permute(0, 2, 1, 3).reshape(n, hk, cap)
    pinned = (at < c["sinks"]) | (at >= lens - c["recent"])
    rank = torch.where(pinned[:, None], torch.full_like(weight, math.inf), weight)
    rank = torch.where((at < lens)[:, None], rank, torch.full_like(weight, -math.inf))
    take = min(budget, cap)
    kept = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :take].sort(-1).values
    left = lens.clamp(max=budget)
    # a sequence below the budget keeps its first `left` positions; what sorting put behind them is not written
    live = torch.arange(take, device=dev)[None, None] < left[:, None]
    src_page = torch.gather(table[:, None].expand(n, hk, -1), 2, kept // page)
    head = torch.arange(hk, device=dev)[None, :, None]
    slot = torch.arange(take, device=dev)
    dst_page = s["dst_table"].long()[:, slot // page][:, None].expand(n, hk, take)
    dst_at = (slot % page)[None, None].expand(n, hk, take)
    for name in ("k", "v", "weight"):
        new = s[name][src_page, head, kept % page]
        old = s["dst_" + name][dst_page, head, dst_at]
        s["dst_" + name][dst_page, head, dst_at] = torch.where(live[..., None] if new.dim() == 4 else live, new, old)
    return {"k": s["dst_k"], "v": s["dst_v"], "weight": s["dst_weight"], "lengths": left[:, 0].int()}


def _plain_logits(s):
    c = s["case"]
    n, v = c["n_seq"], c["vocab"]
    x = s["logits"].float()
    if s["bias"] is not None:
        x = x + s["bias"]
    at = torch.arange(c["hist"], device=x.device)[None]
    end = s["history_len"][:, None]
    ids = s["history"].long()
    first = end - c["window"] if c["window"] > 0 else torch.zeros_like(end)
    seen = torch.zeros((n, v), device=x.device).scatter_add_(1, ids, ((at < end) & (at >= first)).float())
    count = torch.zeros((n, v), device=x.device).scatter_add_(1, ids, ((at < end) & (at >= s["prompt_len"][:, None])).float())
    r = s["repeat_penalty"][:, None]
    x = torch.where(seen > 0, torch.where(x > 0, x / r, x * r), x)
    x = x - (s["frequency_penalty"][:, None] * count + s["presence_penalty"][:, None] * (count > 0))
    if s["allowed"] is not None:
        bits = (s["allowed"][..., None] >> torch.arange(32, device=x.device, dtype=torch.int32)) & 1
        x = x.masked_fill(bits.view(n, -1)[:, :v] == 0, -math.inf)
    return x.to(s["logits"].dtype)


# ------------------------------------------------------------------------------------------------ what a pass needs
def work(case):
    c = case
    if c["op"] == "logits":
        n, v = c["n_seq"], c["vocab"]
        hist = sum(_spread(max(1, c["hist"] // 2), c["hist"], n))
        b = 2 * n * v * ITEM[c["io"]] + 4 * hist + (4 * v if c["bias"] else 0) + (n * v / 8 if c["mask"] else 0)
        return {"bytes": b, "flops": 3.0 * n * v}
    row = c["n_kv"] * c["dk"]
    tokens = sum(_spread(c["lo"], c["hi"], c["n_seq"]))
    if c["op"] == "append":
        new = sum(_spread(c["new_lo"], c["new_hi"], c["n_seq"]))
        q = 2 * c["n_head"] * c["dk"] * ITEM[c["io"]]
        return {"bytes": new * (q + 2 * row * (ITEM[c["io"]] + ITEM[c["cache"]])), "flops": 3.0 * new * (c["n_head"] * c["dk"] + row)}
    if c["op"] == "decode":
        b = 2 * tokens * row * ITEM[c["cache"]] + 2 * c["n_seq"] * c["n_head"] * c["dk"] * ITEM[c["io"]]
        return {"bytes": b + (8 * tokens * c["n_kv"] if c["track"] else 0), "flops": 4.0 * tokens * c["n_head"] * c["dk"]}
    kept = sum(min(t, c["budget"]) for t in _spread(c["lo"], c["hi"], c["n_seq"]))
    return {"bytes": 4 * tokens * c["n_kv"] + kept * (4 * row * ITEM[c["cache"]] + 4 * c["n_kv"]), "flops": float(tokens * c["n_kv"])}


# ------------------------------------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    s, c = prepare(case, seed), dict(case)
    if c["op"] == "append":
        q, k, v = s["q_new"].double().clone(), s["k"].double(), s["v"].double()
        lens, half = s["lengths"].tolist(), c["dk"] // 2
        starts = list(range(c["n_seq"] + 1)) if s["row_start"] is None else s["row_start"].tolist()
        cos, sin, table = s["cos"].double(), s["sin"].double(), s["table"].tolist()

        def turned(x, p):
            return torch.cat([x[..., :half] * cos[p][:, None] - x[..., half:] * sin[p][:, None],
                              x[..., half:] * cos[p][:, None] + x[..., :half] * sin[p][:, None]], -1)

        for i in range(c["n_seq"]):
            r0, r1 = starts[i], starts[i + 1]
            p = torch.arange(lens[i], lens[i] + r1 - r0, device=q.device)
            q[r0:r1] = turned(s["q_new"][r0:r1].double(), p)
            pages, at = torch.tensor([table[i][int(t) // c["page"]] for t in p.tolist()], device=q.device), p % c["page"]
            k[pages, :, at, :c["dk"]] = turned(s["k_new"][r0:r1].double(), p)
            v[pages, :, at, :c["dk"]] = s["v_new"][r0:r1].double()
        return {"q": q, "k": k, "v": v, "lengths": None}
    if c["op"] == "decode":
        n, hk, dk = c["n_seq"], c["n_kv"], c["dk"]
        g = c["n_head"] // hk
        out, lse = torch.zeros((n, c["n_head"], dk), dtype=torch.float64, device=s["q"].device), torch.full(
            (n, c["n_head"]), -math.inf, dtype=torch.float64, device=s["q"].device)
        weight = s["weight"].double() if c["track"] else None
        for i, t in enumerate(s["lengths"].tolist()):
            if t == 0:
                continue
            pos = torch.arange(t, device=out.device)
            pages, at = s["table"][i].long()[pos // c["page"]], pos % c["page"]
            kk, vv = s["k"][pages, :, at, :dk].double(), s["v"][pages, :, at, :dk].double()
            x = torch.einsum("hgd,thd->hgt", s["q"][i].double().view(hk, g, dk), kk) * dk ** -0.5
            lse[i] = torch.logsumexp(x, -1).view(-1)
            p = torch.softmax(x, -1)
            out[i] = torch.einsum("hgt,thd->hgd", p, vv).reshape(c["n_head"], dk)
            if c["track"]:
                weight[pages, :, at] += p.sum(1).t()
        return {"out": out, "lse": lse, "weight": weight} if c["track"] else {"out": out, "lse": lse}
    if c["op"] == "evict":
        k, v, w = s["dst_k"].double(), s["dst_v"].double(), s["dst_weight"].double()
        table, dst, weights = s["table"].cpu().numpy(), s["dst_table"].cpu().numpy(), s["weight"].cpu().numpy()
        heads = torch.arange(c["n_kv"], device=k.device)[:, None]
        for i, t in enumerate(s["lengths"].tolist()):
            pos = np.arange(t)
            chosen = []
            for h in range(c["n_kv"]):
                if t <= c["budget"]:
                    chosen.append(pos)
                    continue
                middle = np.arange(c["sinks"], t - c["recent"])
                score = weights[table[i][middle // c["page"]], h, middle % c["page"]]
                best = middle[np.argsort(-score.astype(np.float64), kind="stable")[:c["budget"] - c["sinks"] - c["recent"]]]
                chosen.append(np.sort(np.concatenate([pos[:c["sinks"]], best, pos[t - c["recent"]:] if c["recent"] else pos[:0]])))
            chosen = np.stack(chosen)
            slot = np.arange(chosen.shape[1])
            sp, sa = torch.from_numpy(table[i][chosen // c["page"]]).long().to(k.device), torch.from_numpy(chosen % c["page"]).to(k.device)
            dp, da = torch.from_numpy(dst[i][slot // c["page"]]).long().to(k.device)[None], torch.from_numpy(slot % c["page"]).to(k.device)[None]
            k[dp, heads, da], v[dp, heads, da], w[dp, heads, da] = (s[m][sp, heads, sa].double() for m in ("k", "v", "weight"))
        return {"k": k, "v": v, "weight": w, "lengths": None}
    x = s["logits"].double().cpu().numpy()
    if s["bias"] is not None:
        x = x + s["bias"].double().cpu().numpy()
    hist, hl, pl = s["history"].cpu().numpy(), s["history_len"].tolist(), s["prompt_len"].tolist()
    rep, pres, freq = (s[m].double().cpu().numpy() for m in ("repeat_penalty", "presence_penalty", "frequency_penalty"))
    words = None if s["allowed"] is None else s["allowed"].cpu().numpy().view(np.uint8)
    for i in range(c["n_seq"]):
        recent = np.unique(hist[i, max(0, hl[i] - c["window"]) if c["window"] > 0 else 0:hl[i]])
        y = x[i, recent]
        x[i, recent] = np.where(y > 0, y / rep[i], y * rep[i])
        ids, counts = np.unique(hist[i, pl[i]:hl[i]], return_counts=True)
        x[i, ids] -= freq[i] * counts + pres[i]
        if words is not None:
            x[i, np.unpackbits(words[i], bitorder="little")[:c["vocab"]] == 0] = -np.inf
    return x
