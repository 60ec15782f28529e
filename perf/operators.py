"""Operators around a paged key/value cache: the inputs they are timed on, their plain forms and their definition in 64 bits.

Four calls of a decoder layer that serves its linears from this package:

* ``rope``  - ``ops.qkv_rope_cache_cuda``: norms of queries and keys for each head and the position rotation, keys and values
  written to their cache slots, all from the output of the fused qkv linear;
* ``attn``  - ``ops.paged_attention_cuda``: attention of each sequence's newest tokens (one, or a chunk) over its pages;
* ``sums``  - ``ops.cache_weight_sums_cuda``: the attention weight each cache slot has received from the newest tokens;
* ``evict`` - ``ops.cache_evict_cuda``: the slots with the most weight, moved in order to the start of a smaller cache.

A case is a dict of plain values.  ``listed()`` gives the standing ones, ``draw(rng)`` one more of the same ranges,
``prepare`` what a serving program holds before the call, ``run`` one call, ``work`` what it cannot do without, ``exact`` its
result in 64 bits.  The sequences of a case have lengths that follow from the case alone: ``_news`` and ``_lens``.
"""

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6
ROPE_THETA = 500000.0


# ---------------------------------------------------------------------------------------------------------------- cases

def _case(name, kind, dtype, heads, kv_heads, dim, page, seqs, new, max_len, ragged, **more):
    return {"name": name, "kind": kind, "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page,
            "seqs": seqs, "new": new, "max_len": max_len, "ragged": ragged, **more}


def listed():
    return [
        # one decode step of a batch of 32 on the 8B head layout, pairs next to each other, no norms: latency counts
        _case("rope_decode_32", "rope", "fp16", 32, 8, 128, 64, 32, 1, 1024, False, norm=False, interleaved=True),
        # chunks of five prompts, odd lengths, with norms of queries and keys, after an eviction (positions ahead of slots)
        _case("rope_chunks_ragged", "rope", "bf16", 32, 8, 128, 16, 5, 611, 1500, True, norm=True, interleaved=False),
        # a long prompt on the 70B head layout: memory traffic counts
        _case("rope_prompt_16384", "rope", "fp16", 64, 8, 128, 128, 2, 8192, 8192, False, norm=True, interleaved=False),
        # one user with a long history, one token: few rows, so the history is split over the whole card
        _case("attn_decode_1", "attn", "fp16", 32, 8, 128, 64, 1, 1, 8191, False),
        # the decode batch of the decoder stack, histories of every length
        _case("attn_decode_32", "attn", "fp16", 32, 8, 128, 64, 32, 1, 4096, True),
        # eight long histories on the 70B head layout
        _case("attn_decode_8_long", "attn", "bf16", 64, 8, 128, 128, 8, 1, 32768, True),
        # chunks of three prompts over what is cached of them already, pages smaller than any tile
        _case("attn_chunks_ragged", "attn", "bf16", 32, 8, 128, 16, 3, 500, 7001, True),
        # a whole prompt of 8192 tokens: tensor cores count
        _case("attn_prompt_8192", "attn", "fp16", 32, 8, 128, 64, 1, 8192, 8192, False),
        # the weight of a decode step, added up for a later eviction
        _case("sums_decode_32", "sums", "fp16", 32, 8, 128, 64, 32, 1, 4096, True),
        # the weight of the last 64 tokens of four prompts
        _case("sums_window_64", "sums", "bf16", 32, 8, 128, 16, 4, 64, 8000, True),
        # a few short histories cut to a quarter
        _case("evict_4", "evict", "bf16", 32, 8, 128, 16, 4, 1, 2000, True, budget=500, sink=4, recent=32),
        # a batch of histories cut to a quarter: memory traffic counts
        _case("evict_32", "evict", "fp16", 32, 8, 128, 64, 32, 1, 8192, True, budget=2048, sink=4, recent=256),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(["rope", "attn", "attn", "sums", "evict"])
    heads, kv_heads = rng.choice([(32, 8), (32, 8), (64, 8), (16, 16), (20, 4), (8, 1), (28, 4)])
    dim = rng.choice([128, 128, 64])
    dtype, page = rng.choice(["fp16", "bf16"]), rng.choice([16, 32, 48, 64, 128])
    ragged = rng.random() < 0.8
    more = {}
    if kind == "rope":
        seqs, new = _log_int(rng, 1, 64), rng.choice([1, _log_int(rng, 2, 2048)])
        max_len = new + _log_int(rng, 1, 1024)
        more = {"norm": rng.random() < 0.6, "interleaved": rng.random() < 0.5}
    elif kind == "evict":
        seqs, new, max_len = _log_int(rng, 1, 32), 1, _log_int(rng, 64, 8192)
        sink, recent = rng.randint(0, 8), rng.randint(0, max_len // 16)
        more = {"budget": max(1, sink + recent, int(max_len * rng.uniform(0.1, 0.9))), "sink": sink, "recent": recent}
    else:
        seqs, new = _log_int(rng, 1, 64), rng.choice([1, 1, rng.randint(2, 8), _log_int(rng, 9, 2048)])
        max_len = new + _log_int(rng, 1, 16384)
        if kind == "sums":
            new = min(new, 128)
    c = _case("", kind, dtype, heads, kv_heads, dim, page, seqs, new, max_len, ragged, **more)
    del c["name"]
    # no more than the largest listed case: slots held, heads times pairs, tokens
    while (c["seqs"] * c["max_len"] * kv_heads * dim > 8 * 32768 * 8 * 128 or c["seqs"] * c["new"] > 16384
           or c["seqs"] * c["new"] * (c["max_len"] - c["new"] // 2) * heads > 32 * 8192 * 4096):
        if c["seqs"] > 1:
            c["seqs"] -= 1
        else:
            c["new"], c["max_len"] = (c["new"] + 1) // 2, (c["max_len"] + 1) // 2
    return c


def _news(case):
    """New tokens of each sequence."""
    n, new = case["seqs"], case["new"]
    if not case["ragged"] or new == 1:
        return [new] * n
    return [new if b == 0 else new * ((5 * b + 3) % n) // n for b in range(n)]


def _lens(case):
    """Cache slots of each sequence in use, the new tokens' among them."""
    n, top = case["seqs"], case["max_len"]
    if not case["ragged"]:
        return [top] * n
    return [top if b == 0 else q + (top - q) * ((7 * b + 2) % (n + 1)) // (n + 1) for b, q in enumerate(_news(case))]


# --------------------------------------------------------------------------------------------------------------- inputs

def _inputs(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev).manual_seed(seed)
    dt, H, G, D, page = DTYPES[case["dtype"]], case["heads"], case["kv_heads"], case["dim"], case["page"]
    news, lens = _news(case), _lens(case)
    n, T = case["seqs"], sum(news)

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device=dev).to(dt)

    def pool(slots):
        """Pages for n sequences of up to `slots` slots, handed out in no order, and three that nobody has."""
        cols = (slots + page - 1) // page
        table = torch.randperm(n * cols + 3, generator=gen, device=dev)[:n * cols].reshape(n, cols).to(torch.int32)
        return (n * cols + 3, G, page, D), table

    shape, table = pool(case["max_len"])
    s = {"case": case, "news": news, "lens": lens, "table": table, "k_pages": randn(*shape), "v_pages": randn(*shape),
         "lengths": torch.tensor(lens, dtype=torch.int32, device=dev),
         "cu": torch.tensor([sum(news[:b]) for b in range(n + 1)], dtype=torch.int32, device=dev)}
    if case["kind"] == "rope":
        s["qkv"] = randn(T, (H + 2 * G) * D)
        off = torch.arange(n, dtype=torch.int32, device=dev) * 17 if case["ragged"] else None
        s["offsets"] = off
        pos = torch.arange(case["max_len"] + 17 * n, dtype=torch.float64, device=dev)
        ang = pos[:, None] * ROPE_THETA ** (-torch.arange(0, D, 2, dtype=torch.float64, device=dev) / D)
        s["cos"], s["sin"] = ang.cos().float(), ang.sin().float()
        s["q_norm"] = s["k_norm"] = None
        if case["norm"]:
            s["q_norm"], s["k_norm"] = ((1 + 0.2 * torch.randn(D, generator=gen, device=dev)).to(dt) for _ in range(2))
    elif case["kind"] in ("attn", "sums"):
        # normed heads: queries and keys of unit variance, queries sharper than that so that the weights are uneven
        s["q"] = (2 * torch.randn(T, H, D, generator=gen, device=dev)).to(dt)
    if case["kind"] == "sums":
        s["lse"] = _attention(s, torch.float32, values=False)
    if case["kind"] == "evict":
        # accumulated weight: heavy-tailed, the older half partly never looked at (equal scores)
        w = torch.randn(n, G, table.shape[1] * page, generator=gen, device=dev)
        s["sums"] = torch.where(w < -0.5, torch.zeros_like(w), torch.exp(3 * w))
        ishape, s["into_table"] = pool(case["budget"])
        s["into_k"], s["into_v"] = (torch.zeros(ishape, dtype=dt, device=dev) for _ in range(2))
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        # a program keeps the handles of its caches from step to step
        from zip_kernel_b200 import ops
        s["kv"] = ops.PagedKV(s["k_pages"], s["v_pages"], s["table"])
        if case["kind"] == "evict":
            s["into"] = ops.PagedKV(s["into_k"], s["into_v"], s["into_table"])
    return s


# ---------------------------------------------------------------------------------------------------------- plain forms

def _slots(table, slots, page):
    """Page and place in it of cache slots `slots` of one sequence."""
    return table[slots // page].long(), slots % page


def _gather(pages, table, n):
    """(kv heads, n, dim): the first n slots of one sequence."""
    page = pages.shape[2]
    got = pages[table[:(n + page - 1) // page].long()]
    return got.transpose(0, 1).reshape(pages.shape[1], -1, pages.shape[3])[:, :n]


def _heads_scores(s, b, r0, r1, ft):
    """Scores (kv heads, group, rows, slots) of new tokens r0 .. r1 - 1 of sequence b, minus infinity where hidden."""
    c = s["case"]
    G, D = c["kv_heads"], c["dim"]
    nq, n, t0 = s["news"][b], s["lens"][b], sum(s["news"][:b])
    q = s["q"][t0 + r0:t0 + r1].to(ft).reshape(r1 - r0, G, c["heads"] // G, D).permute(1, 2, 0, 3)
    k = _gather(s["k_pages"], s["table"][b], n).to(ft)
    sc = (q.reshape(G, -1, D) @ k.transpose(1, 2)).reshape(G, -1, r1 - r0, n) * D ** -0.5
    slot = torch.arange(n, device=q.device)
    row = torch.arange(r0, r1, device=q.device) + (n - nq)
    return sc.masked_fill(slot[None, :] > row[:, None], float("-inf"))


def _attention(s, ft, values=True):
    """(output, natural logarithm of the sum of exponentials), or the latter alone."""
    c = s["case"]
    G, D, T = c["kv_heads"], c["dim"], int(s["q"].shape[0])
    out = torch.zeros(T, c["heads"], D, dtype=ft, device=s["q"].device) if values else None
    lse = torch.full((T, c["heads"]), float("-inf"), dtype=ft, device=s["q"].device)
    t0 = 0
    for b, nq in enumerate(s["news"]):
        for r0 in range(0, nq, 512):
            r1 = min(nq, r0 + 512)
            sc = _heads_scores(s, b, r0, r1, ft)
            m = sc.amax(-1, keepdim=True)
            p = torch.exp(sc - m)
            total = p.sum(-1, keepdim=True)
            lse[t0 + r0:t0 + r1] = (m + total.log()).squeeze(-1).permute(2, 0, 1).reshape(r1 - r0, -1)
            if values:
                v = _gather(s["v_pages"], s["table"][b], s["lens"][b]).to(ft)
                o = ((p / total).reshape(G, -1, p.shape[-1]) @ v).reshape(G, -1, r1 - r0, D)
                out[t0 + r0:t0 + r1] = o.permute(2, 0, 1, 3).reshape(r1 - r0, -1, D)
        t0 += nq
    return (out, lse) if values else lse


def _plain_rope(s):
    c = s["case"]
    H, G, D, dt = c["heads"], c["kv_heads"], c["dim"], s["qkv"].dtype
    T, dev = int(s["qkv"].shape[0]), s["qkv"].device
    x = s["qkv"].float().reshape(T, H + 2 * G, D)
    seq = torch.repeat_interleave(torch.arange(c["seqs"], device=dev), s["cu"][1:] - s["cu"][:-1], output_size=T)
    slot = s["lengths"][seq] - s["cu"][seq + 1] + torch.arange(T, device=dev)
    pos = slot if s["offsets"] is None else slot + s["offsets"][seq]
    y = x[:, :H + G]
    if c["norm"]:
        w = torch.cat((s["q_norm"].float().expand(H, D), s["k_norm"].float().expand(G, D)))
        y = y * torch.rsqrt(y.pow(2).mean(-1, keepdim=True) + EPS) * w
    cos, sin = s["cos"][pos.long()][:, None], s["sin"][pos.long()][:, None]
    if c["interleaved"]:
        a, b = y[..., ::2], y[..., 1::2]
        y = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = y[..., :D // 2], y[..., D // 2:]
        y = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    y = y.to(dt)
    pg = s["table"][seq, slot.long() // c["page"]].long()
    s["k_pages"][pg, :, slot.long() % c["page"]] = y[:, H:]
    s["v_pages"][pg, :, slot.long() % c["page"]] = x[:, H + G:].to(dt)
    return {"q": y[:, :H].contiguous(), "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _weight_sums(s, ft):
    c = s["case"]
    sums = torch.zeros(c["seqs"], c["kv_heads"], s["table"].shape[1] * c["page"], dtype=ft, device=s["q"].device)
    t0 = 0
    for b, nq in enumerate(s["news"]):
        if nq:
            sc = _heads_scores(s, b, 0, nq, ft)
            lse = s["lse"][t0:t0 + nq].to(ft).reshape(nq, c["kv_heads"], -1).permute(1, 2, 0)
            sums[b, :, :s["lens"][b]] = torch.exp(sc - lse[..., None]).sum((1, 2))
        t0 += nq
    return sums


def _plain_evict(s):
    c = s["case"]
    B, G, page, budget = c["seqs"], c["kv_heads"], c["page"], c["budget"]
    dev, n = s["sums"].device, s["sums"].shape[2]
    slot = torch.arange(n, device=dev)
    length = s["lengths"].long()[:, None, None]
    score = s["sums"].masked_fill((slot < c["sink"]) | (slot >= length - c["recent"]), float("inf"))
    score = score.masked_fill(slot >= length, float("-inf"))
    kept = score.sort(dim=-1, descending=True, stable=True).indices[..., :budget]          # equal scores: the lowest slot first
    kept = kept.masked_fill(kept >= length, n).sort(-1).values                         # in order, what does not exist at the end
    if kept.shape[2] < budget:
        kept = torch.nn.functional.pad(kept, (0, budget - kept.shape[2]), value=n)
    live, new_len = kept < n, torch.minimum(s["lengths"], torch.full_like(s["lengths"], budget))
    new_sums = torch.zeros(B, G, s["into_table"].shape[1] * page, device=dev)
    new_sums[..., :budget] = torch.where(live, s["sums"].gather(2, kept.clamp(max=n - 1)), torch.zeros((), device=dev))
    b, g, j = live.nonzero(as_tuple=True)
    src = kept[b, g, j]
    at, to = s["table"][b, src // page].long(), s["into_table"][b, j // page].long()
    s["into_k"][to, g, j % page] = s["k_pages"][at, g, src % page]
    s["into_v"][to, g, j % page] = s["v_pages"][at, g, src % page]
    return {"kept": kept.masked_fill(~live, -1).to(torch.int32), "lengths": new_len, "sums": new_sums,
            "k_pages": s["into_k"], "v_pages": s["into_v"]}


def run(s):
    c = s["case"]
    if not own:
        if c["kind"] == "rope":
            return _plain_rope(s)
        if c["kind"] == "attn":
            return {"out": _attention(s, torch.float32)[0].to(s["q"].dtype)}
        return {"sums": _weight_sums(s, torch.float32)} if c["kind"] == "sums" else _plain_evict(s)
    from zip_kernel_b200 import ops
    if c["kind"] == "rope":
        q = ops.qkv_rope_cache_cuda(s["qkv"], s["kv"], s["cu"], s["lengths"], s["cos"], s["sin"], q_norm=s["q_norm"],
                                    k_norm=s["k_norm"], eps=EPS, interleaved=c["interleaved"], offsets=s["offsets"])
        return {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    if c["kind"] == "attn":
        return {"out": ops.paged_attention_cuda(s["q"], s["kv"], s["cu"], s["lengths"], max_q_len=c["new"])}
    if c["kind"] == "sums":
        return {"sums": ops.cache_weight_sums_cuda(s["q"], s["kv"], s["cu"], s["lengths"], s["lse"], max_q_len=c["new"])}
    kept, lengths, sums = ops.cache_evict_cuda(s["kv"], s["lengths"], s["sums"], c["budget"], n_sink=c["sink"],
                                               n_recent=c["recent"], into=s["into"])
    return {"kept": kept, "lengths": lengths, "sums": sums, "k_pages": s["into_k"], "v_pages": s["into_v"]}


# ----------------------------------------------------------------------------------------------------------------- work

def work(case):
    """Every input read once, every output written once; a multiply-add is two operations."""
    H, G, D = case["heads"], case["kv_heads"], case["dim"]
    news, lens = _news(case), _lens(case)
    T, row = sum(news), 2 * D
    table = sum(4 * ((n + case["page"] - 1) // case["page"]) for n in lens) + 8 * len(lens)
    pairs = sum(q * n - q * (q - 1) / 2 for q, n in zip(news, lens))
    slots = sum(n for q, n in zip(news, lens) if q)
    if case["kind"] == "rope":
        # 4 * D: a position's cosines and sines, once for all heads
        return {"bytes": 2 * T * (H + 2 * G) * row + 4 * T * D + table, "flops": T * (H + G) * D * (7 if case["norm"] else 3)}
    if case["kind"] == "attn":
        return {"bytes": 2 * T * H * row + 2 * slots * G * row + table, "flops": 4 * pairs * H * D}
    if case["kind"] == "sums":
        return {"bytes": T * H * (row + 4) + slots * G * (row + 4) + table, "flops": 2 * pairs * H * D}
    moved = sum(min(n, case["budget"]) for n in lens)
    return {"bytes": G * (4 * moved * row + 4 * sum(lens) + 8 * moved) + 2 * table, "flops": G * sum(lens)}


# ---------------------------------------------------------------------------------------------------------------- exact

def exact(case, seed):
    """The definitions, one sequence and one head after the other, in 64 bits."""
    s = _inputs(case, seed)
    H, G, D, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    per, t0 = H // G, 0
    if case["kind"] == "evict":
        return _exact_evict(s)
    if case["kind"] == "rope":
        out = {"q": torch.zeros(sum(s["news"]), H, D, dtype=torch.float64, device=s["qkv"].device),
               "k_pages": s["k_pages"].double(), "v_pages": s["v_pages"].double()}
        for b, (nq, n) in enumerate(zip(s["news"], s["lens"])):
            slots = torch.arange(n - nq, n, device=s["qkv"].device)
            pos = slots + (17 * b if case["ragged"] else 0)
            c, sn = s["cos"][pos].double(), s["sin"][pos].double()
            pg, at = _slots(s["table"][b], slots, page)
            for h in range(H + 2 * G):
                x = s["qkv"][t0:t0 + nq, h * D:(h + 1) * D].double()
                if h >= H + G:
                    out["v_pages"][pg, h - H - G, at] = x
                    continue
                if case["norm"]:
                    x = x / torch.sqrt((x * x).sum(1, keepdim=True) / D + EPS) * (s["q_norm"] if h < H else s["k_norm"]).double()
                first = slice(0, D, 2) if case["interleaved"] else slice(0, D // 2)
                second = slice(1, D, 2) if case["interleaved"] else slice(D // 2, D)
                y = torch.empty_like(x)
                y[:, first] = x[:, first] * c - x[:, second] * sn
                y[:, second] = x[:, first] * sn + x[:, second] * c
                if h < H:
                    out["q"][t0:t0 + nq, h] = y
                else:
                    out["k_pages"][pg, h - H, at] = y
            t0 += nq
        return out
    res = (torch.zeros_like(s["q"], dtype=torch.float64) if case["kind"] == "attn"
           else torch.zeros(case["seqs"], G, s["table"].shape[1] * page, dtype=torch.float64, device=s["q"].device))
    for b, (nq, n) in enumerate(zip(s["news"], s["lens"])):
        pg, at = _slots(s["table"][b], torch.arange(n, device=s["q"].device), page)
        for g in range(G if nq else 0):
            k = s["k_pages"][pg, g, at].double()
            v = s["v_pages"][pg, g, at].double()
            for h in range(g * per, (g + 1) * per):
                for r0 in range(0, nq, 2048):
                    q = s["q"][t0 + r0:min(t0 + nq, t0 + r0 + 2048), h].double()
                    r1 = r0 + q.shape[0]
                    x = q @ k.T / float(D) ** 0.5
                    seen = torch.ones(r1 - r0, n, dtype=torch.bool, device=q.device).tril(n - nq + r0)
                    if case["kind"] == "attn":
                        e = torch.where(seen, torch.exp(x - torch.where(seen, x, -torch.inf).max(1, keepdim=True).values), 0.0)
                        res[t0 + r0:t0 + r1, h] = e @ v / e.sum(1, keepdim=True)
                    else:
                        w = torch.exp(x - s["lse"][t0 + r0:t0 + r1, h, None].double())
                        res[b, g, :n] += torch.where(seen, w, 0.0).sum(0)
        t0 += nq
    return {"out": res} if case["kind"] == "attn" else {"sums": res}


def _exact_evict(s):
    c = s["case"]
    B, G, budget, page = c["seqs"], c["kv_heads"], c["budget"], c["page"]
    dev = s["sums"].device
    kept = torch.full((B, G, budget), -1, dtype=torch.int32, device=dev)
    sums = torch.zeros(B, G, s["into_table"].shape[1] * page, dtype=torch.float64, device=dev)
    k_pages, v_pages = s["into_k"].double(), s["into_v"].double()
    for b, n in enumerate(s["lens"]):
        m = min(n, budget)
        to_pg, to_at = _slots(s["into_table"][b], torch.arange(m, device=dev), page)
        for g in range(G):
            key = s["sums"][b, g, :n].double().cpu().tolist()
            free = range(min(c["sink"], n), max(min(c["sink"], n), n - c["recent"]))
            must = n - len(free)
            best = sorted(free, key=lambda i: (-key[i], i))[:max(0, m - must)]
            keep = range(n) if n <= budget else sorted(set(range(n)) - set(free) | set(best))
            idx = torch.tensor(list(keep), device=dev)
            kept[b, g, :m] = idx.to(torch.int32)
            sums[b, g, :m] = s["sums"][b, g, idx].double()
            pg, at = _slots(s["table"][b], idx, page)
            k_pages[to_pg, g, to_at] = s["k_pages"][pg, g, at].double()
            v_pages[to_pg, g, to_at] = s["v_pages"][pg, g, at].double()
    return {"kept": kept, "lengths": s["lengths"].clamp(max=budget), "sums": sums, "k_pages": k_pages, "v_pages": v_pages}
