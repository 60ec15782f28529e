"""The paged-cache operators as a serving loop uses them: one after the other over growing and shortened histories, captured
and replayed, on other streams, with metadata that cannot be true, and beyond 32-bit offsets."""

import pytest
import torch

from tests import paged_helpers as R

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def device_error():
    from zip_kernel_b200 import _lib
    return _lib.device_error(DEV)


@pytest.fixture(autouse=True)
def start_without_error():
    device_error()
    yield


class View(R.Case):
    """A Case over what a cache holds now: references are taken from the rounded keys and values themselves."""

    def __init__(self, kv, news, lens, q):
        self.news, self.lens, self.heads, self.kv_heads, self.dim, self.page = news, lens, q.shape[1], kv.n_kv_heads, kv.head_dim, kv.page_size
        self.dt, self.n, self.cols = kv.dtype, len(news), kv.max_pages
        self.table, self.k, self.v, self.q, self.T = kv.block_table.cpu(), kv.k_pages.cpu(), kv.v_pages.cpu(), q.cpu(), q.shape[0]
        self.cu = torch.tensor([sum(news[:b]) for b in range(self.n + 1)], dtype=torch.int32)
        self.lengths = torch.tensor(lens, dtype=torch.int32)


def tables(n, half):
    ang = torch.arange(n, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(half, dtype=torch.float64) / half)
    return ang.cos().float(), ang.sin().float()


@pytest.mark.parametrize("dtype,dim,heads,kv_heads", [("fp16", 128, 8, 2), ("bf16", 64, 6, 3)])
def test_prompt_chunks_decode_eviction_decode(dtype, dim, heads, kv_heads):
    """Two chunks of a prompt, decode steps, an eviction, decode steps: every operator of every step against 64 bits."""
    from zip_kernel_b200 import ops
    from zip_kernel_b200.paged_cache import PagedKVCache
    B, dt = 3, R.DT[dtype]
    cache = PagedKVCache(1, B, 200, kv_heads, dim, page_size=16, dtype=dt, device=DEV, track_weights=True)
    kv = cache.layer(0)
    cos, sin = tables(256, dim // 2)
    g = torch.Generator().manual_seed(0)
    u = torch.finfo(dt).eps / 2
    total = torch.zeros(B, kv_heads, cache.max_slots, dtype=torch.float64)
    slack = torch.zeros_like(total)
    seen = 0

    def step(n, interleaved):
        nonlocal seen, total, slack
        cu = cache.advance(n)
        qkv = torch.randn(B * n, (heads + 2 * kv_heads) * dim, generator=g).to(dt)
        before_k, before_v = kv.k_pages.cpu(), kv.v_pages.cpu()
        q = ops.qkv_rope_cache_cuda(qkv.to(DEV), kv, cu, cache.lengths, cos.to(DEV), sin.to(DEV), interleaved=interleaved, offsets=cache.offsets)
        lens = cache.lengths.tolist()
        c = View(kv, [n] * B, lens, q)
        c.qkv, c.k, c.v = qkv, before_k, before_v
        qr, kr, vr, err = R.rope_ref(c, cos, sin, interleaved=interleaved, offsets=cache.offsets.cpu())
        assert int(cache.offsets[0]) + lens[0] == seen + n
        R.assert_within(q, qr, u * qr.abs() + err + 2.0 ** -24, "queries")
        R.assert_within(kv.k_pages, kr, u * kr.abs() + err + 2.0 ** -24, "keys")
        R.assert_within(kv.v_pages, vr, 0.0, "values")
        out, lse = ops.paged_attention_cuda(q, kv, cu, cache.lengths, max_q_len=n, return_lse=True)
        c = View(kv, [n] * B, lens, q)
        ref, ref_lse, amp, mag = R.attention_ref(c)
        R.assert_within(out, ref, R.attention_tolerance(c, ref, amp, mag), "attention")
        R.assert_within(lse, ref_lse, R.lse_tolerance(c, ref_lse, mag), "lse")
        cache.add_weights(0, q, lse, cu, n)
        add, rel = R.sums_ref(c, lse.cpu())
        total += add
        slack += rel * add + 2.0 ** -23 * total
        R.assert_within(cache.sums[0], total, slack, "sums")
        seen += n

    step(37, True)
    step(70, True)
    step(1, True)
    step(2, True)
    sums = cache.sums[0].cpu()
    c = View(kv, [0] * B, cache.lengths.tolist(), torch.zeros(0, heads, dim, dtype=dt))
    kept, new_len, new_sums = R.evict_ref(c, sums, 50, 4, 10)
    got = cache.evict(50, n_sink=4, n_recent=10)
    assert torch.equal(got[0].cpu(), kept) and cache.lengths.tolist() == [50] * B and cache.offsets.tolist() == [60] * B
    assert torch.equal(cache.sums[0, ..., :50].cpu(), new_sums) and not cache.sums[0, ..., 50:].any()
    for b in range(B):
        for h in range(kv_heads):
            j = torch.arange(50)
            old = kept[b, h].long()
            for now, was in ((kv.k_pages.cpu(), c.k), (kv.v_pages.cpu(), c.v)):
                assert torch.equal(now[c.table[b, j // 16].long(), h, j % 16], was[c.table[b, old // 16].long(), h, old % 16])
    total, slack = cache.sums[0].cpu().double(), torch.zeros_like(total)
    step(1, True)
    step(5, True)
    assert device_error() == 0


def test_eviction_of_all_layers_equals_one_by_one():
    from zip_kernel_b200 import ops
    from zip_kernel_b200.paged_cache import PagedKVCache
    cache = PagedKVCache(3, 2, 300, 2, 64, page_size=32, dtype=torch.bfloat16, device=DEV, track_weights=True)
    g = torch.Generator(device=DEV).manual_seed(1)
    cache.k_pages.normal_(generator=g)
    cache.v_pages.normal_(generator=g)
    cache.sums.uniform_(generator=g)
    cache.lengths.copy_(torch.tensor([260, 90], dtype=torch.int32))
    k, v, sums = cache.k_pages.clone(), cache.v_pages.clone(), cache.sums.clone()
    kept = cache.evict(128, n_sink=2, n_recent=20)
    for i in range(3):
        kv = ops.PagedKV(k[i], v[i], cache.block_table)
        one = ops.cache_evict_cuda(kv, torch.tensor([260, 90], dtype=torch.int32, device=DEV), sums[i], 128, n_sink=2, n_recent=20)
        assert torch.equal(one[0], kept[i]) and torch.equal(one[1], cache.lengths) and torch.equal(one[2], cache.sums[i])
    assert torch.equal(k, cache.k_pages) and torch.equal(v, cache.v_pages)
    assert cache.lengths.tolist() == [128, 90] and cache.offsets.tolist() == [132, 0]


def decode_once(cache, qkv, cos, sin, out):
    from zip_kernel_b200 import ops
    kv, cu = cache.layer(0), cache.advance(1)
    q = ops.qkv_rope_cache_cuda(qkv, kv, cu, cache.lengths, cos, sin, offsets=cache.offsets)
    o, lse = ops.paged_attention_cuda(q, kv, cu, cache.lengths, max_q_len=1, return_lse=True)
    cache.add_weights(0, q, lse, cu, 1)
    out.copy_(o)


def filled(seed, lens, max_slots=700):
    from zip_kernel_b200.paged_cache import PagedKVCache
    cache = PagedKVCache(1, len(lens), max_slots, 2, 128, page_size=16, device=DEV, track_weights=True)
    g = torch.Generator(device=DEV).manual_seed(seed)
    cache.k_pages.normal_(generator=g)
    cache.v_pages.normal_(generator=g)
    cache.lengths.copy_(torch.tensor(lens, dtype=torch.int32))
    return cache, torch.randn(len(lens), 12 * 128, generator=g, device=DEV).half()


def test_captured_steps_replay_like_eager_ones_and_graphs_run_side_by_side():
    """Two graphs with scratch of their own, replayed on two streams at once, against eager steps: the same bits."""
    from zip_kernel_b200 import _lib
    cos, sin = (t.to(DEV) for t in tables(1024, 64))
    lens = [[600, 1, 333], [512, 64, 9]]
    want = []
    for i in range(2):
        cache, qkv = filled(i, lens[i])
        out, outs = torch.empty(3, 8, 128, dtype=torch.float16, device=DEV), []
        for _ in range(4):
            decode_once(cache, qkv, cos, sin, out)
            outs.append(out.clone())
        want.append((torch.stack(outs), cache.k_pages.clone(), cache.sums.clone()))
    jobs = []
    for i in range(2):
        cache, qkv = filled(i, lens[i])
        out, hold, stream, graph = torch.empty(3, 8, 128, dtype=torch.float16, device=DEV), _lib.WorkspaceHolder(), torch.cuda.Stream(), torch.cuda.CUDAGraph()
        stream.wait_stream(torch.cuda.current_stream())
        with _lib.use_workspace(hold), torch.cuda.stream(stream):
            decode_once(cache, qkv, cos, sin, out)
            fresh, _ = filled(i, lens[i])
            for a, b in ((cache.k_pages, fresh.k_pages), (cache.v_pages, fresh.v_pages), (cache.lengths, fresh.lengths), (cache.sums, fresh.sums)):
                a.copy_(b)
            stream.synchronize()
            with torch.cuda.graph(graph, stream=stream):
                decode_once(cache, qkv, cos, sin, out)
        jobs.append((cache, out, hold, stream, graph, [], qkv))        # (a graph keeps no tensor alive)
    torch.cuda.synchronize()
    for _ in range(4):
        for cache, out, hold, stream, graph, outs, _ in jobs:
            with torch.cuda.stream(stream):
                graph.replay()
                outs.append(out.clone())
    torch.cuda.synchronize()
    for (cache, _, _, _, _, outs, _), (o, k, s) in zip(jobs, want):
        assert torch.equal(torch.stack(outs), o) and torch.equal(cache.k_pages, k) and torch.equal(cache.sums, s)
    assert device_error() == 0


def test_prompt_attention_captured_and_on_another_stream():
    from zip_kernel_b200 import _lib, ops
    c = R.Case([300, 2, 40], [700, 90, 40], 8, 2, 128, 16, "fp16", seed=11)
    q, kv, cu, n = c.q.to(DEV), c.kv(), c.cu.to(DEV), c.lengths.to(DEV)
    want = ops.paged_attention_cuda(q, kv, cu, n)
    side, hold, graph = torch.cuda.Stream(), _lib.WorkspaceHolder(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with _lib.use_workspace(hold), torch.cuda.stream(side):
        assert torch.equal(ops.paged_attention_cuda(q, kv, cu, n), want)
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            out = ops.paged_attention_cuda(q, kv, cu, n)
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    with pytest.raises(RuntimeError, match="workspace"):
        with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=torch.cuda.Stream()):
            n.add_(0)
            ops.paged_attention_cuda(q, kv, cu, n)
    torch.cuda.synchronize()


BAD = {
    "page number beyond the pages": (dict(), lambda c: c.table.__setitem__((1, 1), 10 ** 6)),
    "negative page number": (dict(), lambda c: c.table.__setitem__((1, 0), -7)),
    "length beyond the table": (dict(), lambda c: c.lengths.__setitem__(1, 10 ** 9)),
    "negative length": (dict(), lambda c: c.lengths.__setitem__(1, -5)),
    "offsets that fall": (dict(), lambda c: c.cu.__setitem__(2, 0)),
    "offsets beyond the tokens": (dict(), lambda c: c.cu.__setitem__(2, 10 ** 6)),
}


@pytest.mark.parametrize("name", list(BAD))
@pytest.mark.parametrize("news", [[1, 1], [3, 40]])
def test_metadata_that_cannot_be_true_sets_the_error_word(name, news):
    """Nothing is read or written out of range, sequence 0 (before the bad one) is right, and the next call is clean."""
    from zip_kernel_b200 import ops
    def case():
        return R.Case(news, [50, 60], 8, 2, 128, 16, "fp16", seed=12, max_pages=6)
    good, c = case(), case()
    BAD[name][1](c)
    cos, sin = (t.to(DEV) for t in tables(128, 64))
    want = ops.paged_attention_cuda(good.q.to(DEV), good.kv(), good.cu.to(DEV), good.lengths.to(DEV))
    assert device_error() == 0
    # values must be finite up to the length the kernels see
    c.k, c.v = c.k.nan_to_num(0.0), c.v.nan_to_num(0.0)
    q, kv, cu, n = c.q.to(DEV), c.kv(), c.cu.to(DEV), c.lengths.to(DEV)
    out, lse = ops.paged_attention_cuda(q, kv, cu, n, return_lse=True)
    assert device_error() != 0
    if "offsets" not in name:
        assert torch.equal(out[:news[0]], want[:news[0]])
    ops.cache_weight_sums_cuda(q, kv, cu, n, lse)
    assert device_error() != 0
    ops.qkv_rope_cache_cuda(c.qkv.to(DEV), kv, cu, n, cos, sin)
    assert device_error() != 0 or "page" in name               # (one new token lies on a page that is not the bad one)
    if "offsets" not in name:
        sums = torch.rand(2, 2, kv.max_slots, device=DEV)
        ops.cache_evict_cuda(kv, n, sums, 20)
        word = device_error()
        assert word != 0 or "page" in name                     # (seen where a kept slot is on that page)
    got = ops.paged_attention_cuda(good.q.to(DEV), good.kv(), good.cu.to(DEV), good.lengths.to(DEV))
    assert torch.equal(got, want) and device_error() == 0


def test_too_long_a_chunk_and_position_set_the_error_word():
    from zip_kernel_b200 import ops
    c = R.Case([2, 9], [50, 60], 8, 2, 128, 16, "fp16", seed=13)
    q, kv, cu, n = c.q.to(DEV), c.kv(), c.cu.to(DEV), c.lengths.to(DEV)
    ops.paged_attention_cuda(q, kv, cu, n, max_q_len=1)
    assert device_error() != 0
    ops.paged_attention_cuda(q, kv, cu, n, max_q_len=8)
    assert device_error() != 0
    ops.cache_weight_sums_cuda(q, kv, cu, n, torch.zeros(11, 8, device=DEV), max_q_len=8)
    assert device_error() != 0
    cos, sin = (t.to(DEV) for t in tables(55, 64))
    ops.qkv_rope_cache_cuda(c.qkv.to(DEV), kv, cu, n, cos, sin)
    assert device_error() != 0
    ops.paged_attention_cuda(q, kv, cu, n, max_q_len=9)
    assert device_error() == 0


def test_refused_arguments():
    from zip_kernel_b200 import ops
    c = R.Case([1, 3], [50, 60], 8, 2, 128, 16, "fp16", seed=14)
    kv, cu, n, q = c.kv(), c.cu.to(DEV), c.lengths.to(DEV), c.q.to(DEV)
    k, v, table = kv.k_pages, kv.v_pages, kv.block_table
    for bad in (lambda: ops.PagedKV(k.float(), v, table), lambda: ops.PagedKV(k, v[:1], table), lambda: ops.PagedKV(k, v, table.long()),
                lambda: ops.PagedKV(k[..., :96], v[..., :96], table), lambda: ops.PagedKV(k[:, :, :8], v[:, :, :8], table),
                lambda: ops.PagedKV(k.expand(2, -1, -1, -1, -1)[0][..., ::2], v[..., ::2], table), lambda: ops.PagedKV(k, v, table.cpu()),
                lambda: ops.PagedKV(k[:1].expand(5, -1, -1, -1), v[:1].expand(5, -1, -1, -1), table),
                lambda: ops.paged_attention_cuda(q.bfloat16(), kv, cu, n), lambda: ops.paged_attention_cuda(q[:, :5], kv, cu, n),
                lambda: ops.paged_attention_cuda(q, kv, cu.long(), n), lambda: ops.paged_attention_cuda(q, kv, cu[:2], n),
                lambda: ops.paged_attention_cuda(q, kv, cu, n.cpu()), lambda: ops.paged_attention_cuda(q, kv, cu, n, max_q_len=-1),
                lambda: ops.paged_attention_cuda(q, kv, cu, n, scale=0.0), lambda: ops.paged_attention_cuda(q, kv, cu, n, out=q[:, :, :64]),
                lambda: ops.paged_attention_cuda(q, kv, cu, n, out=torch.empty(4, 8, 132, dtype=q.dtype, device=DEV)[..., 4:]),
                lambda: ops.cache_weight_sums_cuda(q, kv, cu, n, torch.zeros(4, 7, device=DEV)),
                lambda: ops.cache_weight_sums_cuda(q, kv, cu, n, torch.zeros(4, 8, device=DEV), torch.zeros(2, 2, 5, device=DEV)),
                lambda: ops.cache_evict_cuda(kv, n, torch.zeros(2, 2, kv.max_slots, device=DEV), 0),
                lambda: ops.cache_evict_cuda(kv, n, torch.zeros(2, 2, kv.max_slots, device=DEV), kv.max_slots + 1),
                lambda: ops.cache_evict_cuda(kv, n, torch.zeros(2, 2, kv.max_slots, device=DEV), 10, n_sink=6, n_recent=5),
                lambda: ops.cache_evict_cuda(kv, n, torch.zeros(2, 2, kv.max_slots, device=DEV), 10, into=R.Case([0], [50], 8, 2, 128).kv()),
                lambda: ops.qkv_rope_cache_cuda(c.qkv.to(DEV)[:, :-128], kv, cu, n, *(t.to(DEV) for t in tables(99, 64))),
                lambda: ops.qkv_rope_cache_cuda(c.qkv.to(DEV), kv, cu, n, *(t.to(DEV).half() for t in tables(99, 64))),
                lambda: ops.qkv_rope_cache_cuda(c.qkv.to(DEV), kv, cu, n, *(t.to(DEV) for t in tables(99, 60))),
                lambda: ops.qkv_rope_cache_cuda(c.qkv.to(DEV), kv, cu, n, *(t.to(DEV) for t in tables(99, 64)), q_norm=torch.ones(64, device=DEV).half())):
        with pytest.raises(ValueError):
            bad()
    assert device_error() == 0
    # nothing to do: no tokens, no sequences
    assert ops.paged_attention_cuda(q[:0], kv, cu.zero_(), n).shape == (0, 8, 128)
    none = ops.PagedKV(k, v, table[:0])
    out = ops.paged_attention_cuda(q, none, cu[:1], n[:0], out=torch.full_like(q, 2.0))
    assert (out == 2.0).all()


def test_cache_beyond_32_bit_offsets():
    """Pages whose elements lie beyond 2^31 (and, in bytes, beyond 2^32)."""
    from zip_kernel_b200 import ops
    n_pages = 36000
    k = torch.zeros(n_pages, 8, 64, 128, dtype=torch.float16, device=DEV)
    v = torch.zeros_like(k)
    small = R.Case([1, 40], [130, 200], 32, 8, 128, 64, "fp16", seed=15)
    far = (n_pages - 1 - small.table).to(torch.int32)
    idx = small.table.flatten().long()
    k[(n_pages - 1 - idx).to(DEV)], v[(n_pages - 1 - idx).to(DEV)] = small.k[idx].to(DEV), small.v[idx].to(DEV)
    kv, cu, n, q = ops.PagedKV(k, v, far.to(DEV)), small.cu.to(DEV), small.lengths.to(DEV), small.q.to(DEV)
    want, lse = ops.paged_attention_cuda(q, small.kv(), cu, n, return_lse=True)
    assert torch.equal(ops.paged_attention_cuda(q, kv, cu, n), want)
    assert torch.equal(ops.cache_weight_sums_cuda(q, kv, cu, n, lse), ops.cache_weight_sums_cuda(q, small.kv(), cu, n, lse))
    cos, sin = (t.to(DEV) for t in tables(256, 64))
    near = small.kv()
    ops.qkv_rope_cache_cuda(small.qkv.to(DEV), near, cu, n, cos, sin)
    ops.qkv_rope_cache_cuda(small.qkv.to(DEV), kv, cu, n, cos, sin)
    sums = torch.rand(2, 8, kv.max_slots, generator=torch.Generator(device=DEV).manual_seed(3), device=DEV)
    a, b = ops.cache_evict_cuda(near, n, sums, 100, n_recent=9), ops.cache_evict_cuda(kv, n, sums, 100, n_recent=9)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    for x, y in ((k, near.k_pages), (v, near.v_pages)):
        assert torch.equal(x[(n_pages - 1 - idx).to(DEV)].nan_to_num(9.0), y[idx.to(DEV)].nan_to_num(9.0))
    assert device_error() == 0


def test_long_history_of_one_sequence_and_many_short_ones():
    """Runs that cut one unit into many parts, and runs that hold many units, give what 64 bits give."""
    from zip_kernel_b200 import ops
    for news, lens, heads, kv_heads in (([1], [20011], 8, 1), ([1] * 300, [1 + (7 * b) % 130 for b in range(300)], 2, 2), ([33], [9001], 8, 1)):
        c = R.Case(news, lens, heads, kv_heads, 64, 32, "bf16", seed=16)
        ref, ref_lse, amp, mag = R.attention_ref(c)
        q, kv, cu, n = c.q.to(DEV), c.kv(), c.cu.to(DEV), c.lengths.to(DEV)
        out, lse = ops.paged_attention_cuda(q, kv, cu, n, max_q_len=max(news), return_lse=True)
        R.assert_within(out, ref, R.attention_tolerance(c, ref, amp, mag), "out")
        R.assert_within(lse, ref_lse, R.lse_tolerance(c, ref_lse, mag), "lse")
        want, rel = R.sums_ref(c, lse.cpu())
        R.assert_within(ops.cache_weight_sums_cuda(q, kv, cu, n, lse), want, rel * want, "sums")
    assert device_error() == 0


@pytest.mark.parametrize("news,lens,heads,kv_heads,dim,page", [
    ([2, 1, 40], [70, 33, 200], 130, 1, 64, 16),                          # more heads than a row tile of 128 has rows
    ([40, 1, 0, 9] * 12, [90, 300, 7, 9] * 12, 4, 2, 64, 32),             # more sequences than a warp has lanes, both kernels
    ([17] * 33, [17 + 5 * b for b in range(33)], 8, 4, 64, 16),
    ([0, 0, 3], [5, 0, 3], 2, 2, 128, 16),
])
def test_attention_of_mixed_batches(news, lens, heads, kv_heads, dim, page):
    from zip_kernel_b200 import ops
    c = R.Case(news, lens, heads, kv_heads, dim, page, "fp16", seed=18)
    ref, ref_lse, amp, mag = R.attention_ref(c)
    q, kv, cu, n = c.q.to(DEV), c.kv(), c.cu.to(DEV), c.lengths.to(DEV)
    out, lse = ops.paged_attention_cuda(q, kv, cu, n, return_lse=True)
    R.assert_within(out, ref, R.attention_tolerance(c, ref, amp, mag), "out")
    R.assert_within(lse, ref_lse, R.lse_tolerance(c, ref_lse, mag), "lse")
    if heads // kv_heads <= 128:
        want, rel = R.sums_ref(c, lse.cpu())
        R.assert_within(ops.cache_weight_sums_cuda(q, kv, cu, n, lse), want, rel * want, "sums")
    else:
        with pytest.raises(RuntimeError, match="share"):
            ops.cache_weight_sums_cuda(q, kv, cu, n, lse)
    assert device_error() == 0


def test_scores_that_grow_and_infinities():
    """Maxima that rise by more than 2^8 along a row (the output follows), rows of one weight, and a NaN key that only its
    own sequence's later rows see."""
    from zip_kernel_b200 import ops
    c = R.Case([140, 1], [500, 400], 4, 1, 128, 16, "fp16", seed=17)
    for b in range(2):
        for j in range(c.lens[b]):
            p, i = int(c.table[b, j // 16]), j % 16
            c.k[p, :, i] = (c.k[p, :, i].float() * (0.2 + 6.0 * j / 500)).to(c.dt)
    ref, ref_lse, amp, mag = R.attention_ref(c)
    out, lse = ops.paged_attention_cuda(c.q.to(DEV), c.kv(), c.cu.to(DEV), c.lengths.to(DEV), return_lse=True)
    R.assert_within(out, ref, R.attention_tolerance(c, ref, amp, mag), "out")
    R.assert_within(lse, ref_lse, R.lse_tolerance(c, ref_lse, mag), "lse")
    # sequence 0: key of slot 450 is NaN, seen by new tokens 90 .. 139 (slots 450 .. 499)
    p, i = int(c.table[0, 450 // 16]), 450 % 16
    c.k[p, :, i] = float("nan")
    bad = ops.paged_attention_cuda(c.q.to(DEV), c.kv(), c.cu.to(DEV), c.lengths.to(DEV))
    assert torch.isnan(bad[90:140].float()).all()
    rest = torch.cat((torch.arange(90), torch.tensor([140])))
    R.assert_within(bad[rest], ref[rest], R.attention_tolerance(c, ref, amp, mag)[rest], "rows that do not see it")
    assert device_error() == 0


def small_cfg(**kw):
    from zip_kernel_b200.decoder_stack import StackConfig
    return StackConfig(n_layers=2, hidden=512, n_heads=8, n_kv_heads=2, ffn=512, vocab=1000, density=0.25, page_size=16, **kw)


@pytest.mark.parametrize("qk_norm,evict", [(False, 0), (True, 0), (True, 12)])
def test_paged_stack_graph_decode_equals_eager(qk_norm, evict):
    from zip_kernel_b200 import decoder_stack as ds
    runs = [ds.run(small_cfg(qk_norm=qk_norm), batch=2, prefill_len=40, decode_steps=6, device=DEV, use_graph=g, seed=3, paged=True,
                   chunk=24, evict=evict) for g in (True, False)]
    assert runs[0]["last_tokens"] == runs[1]["last_tokens"]
    assert runs[0]["cache"]["slots"] == (12 if evict else 40) + 6
    assert device_error() == 0


def test_paged_stack_tracks_the_other_cache():
    """The same stack on either cache: the rotation and the weights round differently, and a last bit can flip a 4-bit code
    of the next linear, so the two drift apart by a bounded fraction of the quantisation noise."""
    from zip_kernel_b200 import decoder_stack as ds
    cfg = small_cfg()
    tokens = torch.randint(0, cfg.vocab, (2, 24), generator=torch.Generator().manual_seed(5)).to(DEV)
    with torch.no_grad():
        a = ds.DecoderStack(cfg, 2, 32, DEV, seed=4)
        x = a.embed[tokens]
        for li in range(cfg.n_layers):
            x = a._layer(li, x, 0, 24, None)
        b = ds.DecoderStack(cfg, 2, 32, DEV, seed=4, paged=True)
        y, cu = b.embed[tokens], b.cache.advance(24)
        for li in range(cfg.n_layers):
            y = b._layer_paged(li, y, cu)
    assert torch.isfinite(y).all()
    assert ((y - x).float().norm() / x.float().norm()).item() < 0.3
    with pytest.raises(ValueError, match="paged"):
        ds.DecoderStack(small_cfg(qk_norm=True), 2, 32, DEV)


def test_rotation_of_nothing_needs_no_tables_and_no_positions():
    from zip_kernel_b200 import ops
    c = R.Case([3, 1], [40, 7], 8, 2, 128, 16, "fp16", seed=19)
    q, k, v, err = R.rope_ref(c, torch.zeros(64, 0), torch.zeros(64, 0))
    for max_pos, interleaved in ((0, False), (0, True), (5, False)):
        kv, none = c.kv(), torch.zeros(max_pos, 0, device=DEV)
        got = ops.qkv_rope_cache_cuda(c.qkv.to(DEV), kv, c.cu.to(DEV), c.lengths.to(DEV), none, none, interleaved=interleaved)
        R.assert_within(got, q, 0.0, "queries")
        R.assert_within(kv.k_pages, k, 0.0, "keys")
        R.assert_within(kv.v_pages, v, 0.0, "values")
        assert device_error() == 0


def test_sequences_without_any_page():
    from zip_kernel_b200 import ops
    c = R.Case([2, 1], [4, 7], 8, 2, 128, 16, "fp16", seed=20)
    full, cu, n, q = c.kv(), c.cu.to(DEV), torch.zeros(2, dtype=torch.int32, device=DEV), c.q.to(DEV)
    kv = ops.PagedKV(full.k_pages, full.v_pages, full.block_table[:, :0])
    out, lse = ops.paged_attention_cuda(q, kv, cu, n, return_lse=True)
    assert (out == 0).all() and (lse == float("-inf")).all()
    assert ops.cache_weight_sums_cuda(q, kv, cu, n, lse).shape == (2, 2, 0)
    assert device_error() == 0
    with pytest.raises(ValueError, match="budget"):
        ops.cache_evict_cuda(kv, n, torch.zeros(2, 2, 0, device=DEV), 1)


@pytest.mark.parametrize("news", [[1, 1, 1], [5, 2, 1], [700, 3, 150]])
def test_attention_may_overwrite_its_queries(news):
    from zip_kernel_b200 import ops
    c = R.Case(news, [2000, 77, 900], 10, 2, 128, 16, "bf16", seed=21)
    kv, cu, n = c.kv(), c.cu.to(DEV), c.lengths.to(DEV)
    want, q = ops.paged_attention_cuda(c.q.to(DEV), kv, cu, n), c.q.to(DEV)
    got = ops.paged_attention_cuda(q, kv, cu, n, out=q)
    assert got is q and torch.equal(got, want)


def test_offsets_of_a_captured_step_are_whole_before_its_replay():
    from zip_kernel_b200.paged_cache import PagedKVCache
    cache = PagedKVCache(1, 3, 64, 2, 64, page_size=16, device=DEV)
    torch.empty(1 << 20, device=DEV).fill_(1e30)             # what fresh memory may hold
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        cache.cu_seqlens(5)
    assert cache.cu_seqlens(5).tolist() == [0, 5, 10, 15] and cache.cu_seqlens(1).tolist() == [0, 1, 2, 3]
    for bad in (0, 8, 24, -16):
        with pytest.raises(ValueError, match="page_size"):
            PagedKVCache(1, 3, 64, 2, 64, page_size=bad, device=DEV)


@pytest.mark.parametrize("news,lens,max_pages,tail", [
    ([1, 1, 0, 1], [70, 1, 40, 0], 300, 0),                  # chunks of zeros behind the lengths, a sequence without a new token
    ([0, 40, 3], [128, 300, 9], None, 2), ([0, 0], [20, 0], 2, 3), ([1] * 40, [1 + 7 * b for b in range(40)], 20, 0),
    ([5, 2], [3, 1], 2, 0),
])
def test_sums_that_hold_nothing_yet_are_written_whole(news, lens, max_pages, tail):
    from zip_kernel_b200 import ops
    c = R.Case(news, lens, 8, 2, 128, 16, "fp16", seed=22, max_pages=max_pages, tail=tail)
    q, kv, cu, n = c.q.to(DEV), c.kv(), c.cu.to(DEV), c.lengths.to(DEV)
    lse = ops.paged_attention_cuda(q, kv, cu, n, return_lse=True)[1]
    want = ops.cache_weight_sums_cuda(q, kv, cu, n, lse, torch.zeros(c.n, 2, kv.max_slots, device=DEV))
    hold = torch.full((c.n, 2, kv.max_slots), float("nan"), device=DEV)
    del hold                                                 # the memory that the next sums most likely get
    got = ops.cache_weight_sums_cuda(q, kv, cu, n, lse)
    assert torch.equal(got, want) and device_error() == 0
    assert torch.equal(ops.cache_weight_sums_cuda(q[:0], kv, torch.zeros_like(cu), n, lse[:0]), torch.zeros_like(want))
