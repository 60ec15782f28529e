"""Plain 64-bit forms of the operators on a paged cache, and the inputs of their tests."""

import torch

DT = {"fp16": torch.float16, "bf16": torch.bfloat16}


class Case:
    """Sequences with given new tokens and cache lengths, pages handed out in random order, NaN in every slot that no
    sequence has in use (and in the spare pages)."""

    def __init__(self, news, lens, heads, kv_heads, dim=128, page=16, dtype="fp16", seed=0, max_pages=None, tail=0, nhd=False,
                 q_scale=1.0):
        g = torch.Generator().manual_seed(seed)
        self.news, self.lens, self.heads, self.kv_heads, self.dim, self.page = news, lens, heads, kv_heads, dim, page
        self.dt, self.n = DT[dtype], len(news)
        cols = max_pages or max(1, max((x + page - 1) // page for x in lens))
        self.cols = cols
        n_pages = self.n * cols + 2
        self.table = torch.randperm(n_pages, generator=g)[:self.n * cols].reshape(self.n, cols).to(torch.int32)
        self.k = torch.full((n_pages, kv_heads, page, dim), float("nan"), dtype=self.dt)
        self.v = self.k.clone()
        for b, n in enumerate(lens):
            for j in range(n):
                p, i = int(self.table[b, j // page]), j % page
                self.k[p, :, i] = torch.randn(kv_heads, dim, generator=g).to(self.dt)
                self.v[p, :, i] = torch.randn(kv_heads, dim, generator=g).to(self.dt)
        self.T = sum(news) + tail                       # tail: tokens behind the last sequence
        self.cu = torch.tensor([sum(news[:b]) for b in range(self.n + 1)], dtype=torch.int32)
        self.lengths = torch.tensor(lens, dtype=torch.int32)
        self.q = (q_scale * torch.randn(self.T, heads, dim, generator=g)).to(self.dt)
        self.qkv = torch.randn(self.T, (heads + 2 * kv_heads) * dim, generator=g).to(self.dt)
        self.nhd = nhd

    def pages(self, t, device="cuda"):
        """On the GPU, as stored (page, head, slot) or transposed from (page, slot, head)."""
        t = t.to(device)
        return t.transpose(1, 2).contiguous().transpose(1, 2) if self.nhd else t

    def kv(self, k=None, v=None, table=None):
        from zip_kernel_b200 import ops
        return ops.PagedKV(self.pages(self.k) if k is None else k, self.pages(self.v) if v is None else v,
                           (self.table if table is None else table).cuda())

    def rows(self, t, b, g, n=None):
        """The first n slots of sequence b, head g, in 64 bits."""
        n = self.lens[b] if n is None else n
        j = torch.arange(n)
        return t[self.table[b, j // self.page].long(), g, j % self.page].double()


def attention_ref(c, scale=None):
    """out, lse, and per (token, head) the weighted mean of |v| and the largest sum of |q k| over a visible slot."""
    scale = c.dim ** -0.5 if scale is None else scale
    out = torch.zeros(c.T, c.heads, c.dim, dtype=torch.float64)
    lse = torch.full((c.T, c.heads), float("-inf"), dtype=torch.float64)
    amp, mag = torch.zeros(c.T, c.heads, c.dim, dtype=torch.float64), torch.zeros(c.T, c.heads, dtype=torch.float64)
    per = c.heads // c.kv_heads
    for b in range(c.n):
        t0, nq, n = int(c.cu[b]), c.news[b], c.lens[b]
        if nq == 0 or n == 0:
            continue
        for h in range(c.heads):
            k, v = c.rows(c.k, b, h // per), c.rows(c.v, b, h // per)
            q = c.q[t0:t0 + nq, h].double()
            s = q @ k.T * scale
            seen = torch.arange(n)[None, :] <= (torch.arange(nq) + n - nq)[:, None]
            s = s.masked_fill(~seen, float("-inf"))
            l = torch.logsumexp(s, 1)
            w = torch.where(seen, torch.exp(s - l[:, None].clamp(min=-1e300)), torch.zeros((), dtype=torch.float64))
            out[t0:t0 + nq, h], lse[t0:t0 + nq, h], amp[t0:t0 + nq, h] = w @ v, l, w @ v.abs()
            mag[t0:t0 + nq, h] = (q.abs() @ k.abs().T * scale).amax(1)
    return out, lse, amp, mag


def score_error(c, mag):
    """Bound on a score's error in fp32 accumulation: every product and addition off by a step of 2^-23 at most (the
    tensor cores' additions truncate) of the sum of magnitudes."""
    return (c.dim + 8) * 2.0 ** -23 * mag


def attention_tolerance(c, ref, amp, mag):
    """Half a step of the output, half a step of a 16-bit weight, the scores' errors on both sides of the quotient, the
    sum's additions; and weights below the 16-bit type's normal range, off by 2^-25 of a weight of one each."""
    u = torch.finfo(c.dt).eps / 2
    n = max(c.lens + [1])
    rel = u + 2 * score_error(c, mag) + (n + 16) * 2.0 ** -24
    vmax = max([float(c.rows(c.v, b, g).abs().max()) for b in range(c.n) for g in range(c.kv_heads) if c.lens[b]] + [0.0])
    return u * ref.abs() + rel[..., None] * (amp + ref.abs()) + n * 2.0 ** -25 * vmax + 2.0 ** -24


def lse_tolerance(c, lse, mag):
    n = max(c.lens + [1])
    return score_error(c, mag) + (n + 16) * 2.0 ** -24 + 2.0 ** -21 * (1 + lse.abs().nan_to_num(0, 0, 0))


def sums_ref(c, lse, scale=None):
    """sums (B, kv heads, slots) and the bound on their relative error."""
    scale = c.dim ** -0.5 if scale is None else scale
    res = torch.zeros(c.n, c.kv_heads, c.cols * c.page, dtype=torch.float64)
    rel = 0.0
    per = c.heads // c.kv_heads
    for b in range(c.n):
        t0, nq, n = int(c.cu[b]), c.news[b], c.lens[b]
        if nq == 0 or n == 0:
            continue
        for h in range(c.heads):
            k, q = c.rows(c.k, b, h // per), c.q[t0:t0 + nq, h].double()
            l = lse[t0:t0 + nq, h].double()
            s = q @ k.T * scale
            seen = (torch.arange(n)[None, :] <= (torch.arange(nq) + n - nq)[:, None]) & torch.isfinite(l)[:, None]
            res[b, h // per, :n] += torch.where(seen, torch.exp(s - l.nan_to_num(0, 0, 0)[:, None]), torch.zeros((), dtype=torch.float64)).sum(0)
            mag = float((q.abs() @ k.abs().T * scale).max())
            big = float(l.abs().nan_to_num(0, 0, 0).max())
            # the score, its product with log2 e, the logarithm taken off, the exponential, and the additions
            rel = max(rel, 2 * (c.dim + 8) * 2.0 ** -23 * mag + 2.0 ** -21 * (1 + mag + big) + nq * per * 2.0 ** -24)
    return res, rel


def rope_ref(c, cos, sin, q_norm=None, k_norm=None, eps=1e-6, interleaved=False, offsets=None):
    """(q, k pages, v pages, bound of the fp32 error) with untouched slots as they were."""
    H, G, D, half = c.heads, c.kv_heads, c.dim, cos.shape[1]
    q, k, v = torch.full((c.T, H, D), float("nan"), dtype=torch.float64), c.k.double(), c.v.double()
    err = 0.0
    for b in range(c.n):
        for i in range(c.news[b]):
            t, slot = int(c.cu[b]) + i, c.lens[b] - c.news[b] + i
            pos = slot + (int(offsets[b]) if offsets is not None else 0)
            p, at = int(c.table[b, slot // c.page]), slot % c.page
            x = c.qkv[t].double().reshape(H + 2 * G, D)
            y = x.clone()
            for rows, w in ((slice(0, H), q_norm), (slice(H, H + G), k_norm)):
                if w is not None:
                    y[rows] = x[rows] / torch.sqrt((x[rows] ** 2).mean(1, keepdim=True) + eps) * w.double()
            r = slice(0, H + G)
            first = slice(0, 2 * half, 2) if interleaved else slice(0, half)
            second = slice(1, 2 * half, 2) if interleaved else slice(half, 2 * half)
            a, bb = y[r, first].clone(), y[r, second].clone()
            cs, sn = cos[pos].double(), sin[pos].double()
            y[r, first], y[r, second] = a * cs - bb * sn, bb * cs + a * sn
            err = max(err, float(y[r].abs().max()) * 2 * 32 * 2.0 ** -24)
            q[t], k[p, :, at], v[p, :, at] = y[:H], y[H:H + G], x[H + G:]
    return q, k, v, err


def evict_ref(c, sums, budget, sink, recent):
    """kept (B, kv heads, budget), new lengths, new sums by slot (B, kv heads, budget)."""
    kept = torch.full((c.n, c.kv_heads, budget), -1, dtype=torch.int32)
    new = torch.zeros(c.n, c.kv_heads, budget)
    for b, n in enumerate(c.lens):
        for g in range(c.kv_heads):
            s = [float(x) for x in sums[b, g, :n]]
            key = [(0, 0.0) if x != x else (1, x) for x in s]                  # NaN is the least, below minus infinity
            if n <= budget:
                keep = list(range(n))
            else:
                free = list(range(sink, n - recent))
                top = sorted(free, key=lambda j: (-key[j][0], -key[j][1], j))[:budget - sink - recent]
                keep = sorted(set(range(n)) - set(free) | set(top))
            kept[b, g, :len(keep)] = torch.tensor(keep, dtype=torch.int32)
            new[b, g, :len(keep)] = sums[b, g, keep]
    return kept, c.lengths.clamp(max=budget), new


def assert_within(got, ref, tol, what=""):
    got, ref = got.detach().cpu().double(), ref.double()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    err = (got - ref).abs()
    bad = ~(err <= tol)                                    # (a NaN is bad)
    same = (got == ref) | (torch.isnan(got) & torch.isnan(ref))
    bad &= ~same
    if bad.any():
        i = tuple(int(x) for x in bad.nonzero()[0])
        t = tol[i] if torch.is_tensor(tol) and tol.dim() else float(tol)
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} outside; first at {i}: {float(got[i])!r} for {float(ref[i])!r}, "
                             f"tolerance {float(t):.3g}; largest error {float(err.nan_to_num(1e30).max()):.3g}")
