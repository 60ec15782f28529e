"""The operators on a paged cache against plain 64-bit forms: head layouts, page sizes, ragged lengths from zero on,
rows that see nothing, strides, and NaN wherever no slot is in use."""

import pytest
import torch

from tests import paged_helpers as R

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_device_error():
    from zip_kernel_b200 import _lib
    dev = torch.device("cuda", 0)
    _lib.device_error(dev)
    yield
    assert _lib.device_error(dev) == 0


def tables(n_pos, half, seed=0):
    ang = torch.arange(n_pos, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(half, dtype=torch.float64) / max(1, half))
    return ang.cos().float(), ang.sin().float()


ROPE = [
    # news, lens, heads, kv heads, dim, page, dtype, half of the rotated width, interleaved, norms, offsets
    ([1, 1, 1], [1, 40, 16], 32, 8, 128, 16, "fp16", 64, True, False, False),
    ([7, 0, 19], [7, 3, 50], 8, 2, 128, 48, "bf16", 64, False, True, True),
    ([5], [5], 4, 4, 64, 32, "fp16", 32, False, True, False),
    ([2, 3], [30, 3], 6, 2, 64, 16, "bf16", 32, True, True, True),
    ([4, 1], [9, 70], 40, 8, 128, 64, "fp16", 24, False, True, False),
    ([4, 1], [9, 70], 3, 1, 128, 64, "fp16", 16, True, False, True),
    ([3], [3], 2, 1, 64, 16, "fp16", 0, False, True, False),
    ([1] * 70, list(range(1, 71)), 4, 2, 128, 16, "bf16", 64, False, False, True),
]


@pytest.mark.parametrize("news,lens,heads,kv_heads,dim,page,dtype,half,interleaved,norms,shifted", ROPE)
@pytest.mark.parametrize("nhd", [False, True])
def test_rope_writes_queries_and_cache(news, lens, heads, kv_heads, dim, page, dtype, half, interleaved, norms, shifted, nhd):
    from zip_kernel_b200 import ops
    c = R.Case(news, lens, heads, kv_heads, dim, page, dtype, seed=1, tail=3, nhd=nhd)
    g = torch.Generator().manual_seed(2)
    qn, kn = ((1 + 0.3 * torch.randn(dim, generator=g)).to(c.dt) for _ in range(2)) if norms else (None, None)
    off = torch.randint(0, 30, (c.n,), generator=g).to(torch.int32) if shifted else None
    cos, sin = tables(128, half)
    q, k, v, err = R.rope_ref(c, cos, sin, qn, kn, 1e-5, interleaved, off)
    kv = c.kv()
    cuda = lambda t: None if t is None else t.cuda()
    wide = torch.full((c.T, c.qkv.shape[1] + 16), 7.0, dtype=c.dt, device="cuda")
    wide[:, 8:-8] = c.qkv.cuda()
    out = torch.full((c.T, heads, dim), float("nan"), dtype=c.dt, device="cuda")
    got = ops.qkv_rope_cache_cuda(wide[:, 8:-8], kv, c.cu.cuda(), c.lengths.cuda(), cos.cuda(), sin.cuda(), q_norm=cuda(qn),
                                  k_norm=cuda(kn), eps=1e-5, interleaved=interleaved, offsets=cuda(off), out=out)
    u = torch.finfo(c.dt).eps / 2
    assert got is out
    R.assert_within(got, q, u * q.abs().nan_to_num(0) + err + 2.0 ** -24, "queries")        # rows behind the last sequence: NaN as before
    R.assert_within(kv.k_pages, k, u * k.abs().nan_to_num(0) + err + 2.0 ** -24, "keys")
    R.assert_within(kv.v_pages, v, 0.0, "values")


def test_rope_in_place_of_the_queries():
    from zip_kernel_b200 import ops
    c = R.Case([3, 4], [10, 4], 8, 2, 128, 16, "fp16", seed=3)
    cos, sin = (t.cuda() for t in tables(64, 64))
    args = (c.cu.cuda(), c.lengths.cuda(), cos, sin)
    want = ops.qkv_rope_cache_cuda(c.qkv.cuda(), c.kv(), *args)
    qkv = c.qkv.cuda()
    got = ops.qkv_rope_cache_cuda(qkv, c.kv(), *args, out=qkv.view(c.T, -1, 128)[:, :8])
    assert torch.equal(got, want) and got.data_ptr() == qkv.data_ptr()


ATTN = [
    # news, lens, heads, kv heads, dim, page, dtype
    ([1], [1], 1, 1, 128, 16, "fp16"),
    ([1, 1, 1, 1], [1, 63, 64, 65], 32, 8, 128, 16, "fp16"),
    ([1, 1, 1], [200, 129, 700], 16, 2, 128, 64, "bf16"),
    ([1, 0, 1], [33, 50, 0], 8, 2, 64, 32, "fp16"),
    ([1, 1], [300, 17], 16, 1, 64, 48, "bf16"),
    ([1] * 40, [1 + 13 * b for b in range(40)], 4, 2, 128, 128, "fp16"),
    ([3, 1, 4], [3, 77, 260], 8, 2, 128, 16, "fp16"),
    ([5, 2], [3, 1], 4, 4, 128, 16, "bf16"),                       # more new tokens than slots: the first see nothing
    ([17], [17], 4, 2, 128, 16, "fp16"),
    ([70, 33], [70, 190], 4, 1, 128, 16, "fp16"),
    ([130, 1, 29], [400, 300, 29], 6, 2, 64, 48, "bf16"),
    ([257], [300], 5, 5, 128, 256, "fp16"),
    ([40, 2], [150, 9], 7, 1, 128, 80, "bf16"),
    ([9, 1], [600, 601], 24, 1, 128, 32, "fp16"),                  # more heads on a key/value head than a row tile of 16
    ([200], [150], 8, 8, 64, 16, "fp16"),                          # 50 rows that see nothing
]


@pytest.mark.parametrize("news,lens,heads,kv_heads,dim,page,dtype", ATTN)
@pytest.mark.parametrize("nhd", [False, True])
def test_attention(news, lens, heads, kv_heads, dim, page, dtype, nhd):
    from zip_kernel_b200 import ops
    c = R.Case(news, lens, heads, kv_heads, dim, page, dtype, seed=4, tail=2, nhd=nhd, q_scale=2.0)
    ref, lse, amp, mag = R.attention_ref(c)
    out = torch.full((c.T, heads, dim), 3.0, dtype=c.dt, device="cuda")
    got, got_lse = ops.paged_attention_cuda(c.q.cuda(), c.kv(), c.cu.cuda(), c.lengths.cuda(), out=out, return_lse=True)
    end = sum(news)
    assert (got[end:] == 3.0).all()                                # rows behind the last sequence are left
    R.assert_within(got[:end], ref[:end], R.attention_tolerance(c, ref, amp, mag)[:end], "out")
    R.assert_within(got_lse[:end], lse[:end], R.lse_tolerance(c, lse, mag)[:end], "lse")
    hinted = ops.paged_attention_cuda(c.q.cuda(), c.kv(), c.cu.cuda(), c.lengths.cuda(), max_q_len=max(news))
    R.assert_within(hinted[:end], ref[:end], R.attention_tolerance(c, ref, amp, mag)[:end], "out with max_q_len")


@pytest.mark.parametrize("news,lens", [([1, 1], [900, 100]), ([64, 3], [900, 100])])
def test_attention_scale_strides_and_repeated_calls(news, lens):
    from zip_kernel_b200 import ops
    c = R.Case(news, lens, 8, 2, 128, 16, "fp16", seed=5)
    ref, _, amp, mag = R.attention_ref(c, scale=0.3)
    wide = torch.zeros(c.T, 12, 136, dtype=c.dt, device="cuda")
    wide[:, 2:10, :128] = c.q.cuda()
    out = torch.zeros(c.T, 8, 256, dtype=c.dt, device="cuda")
    kv, cu, n = c.kv(), c.cu.cuda(), c.lengths.cuda()
    got = ops.paged_attention_cuda(wide[:, 2:10, :128], kv, cu, n, scale=0.3, out=out[..., 128:])
    R.assert_within(got, ref, R.attention_tolerance(c, ref, amp, mag), "strided")
    assert not out[..., :128].any()
    first = got.clone()
    for _ in range(20):                                            # same bits every time: fixed order of all additions
        assert torch.equal(ops.paged_attention_cuda(c.q.cuda(), kv, cu, n, scale=0.3), first)
    odd = torch.zeros(c.T, 8, 129, dtype=c.dt, device="cuda")[..., 1:]          # rows no kernel can read: copied
    odd.copy_(c.q.cuda())
    assert torch.equal(ops.paged_attention_cuda(odd, kv, cu, n, scale=0.3), first)


@pytest.mark.parametrize("news,lens,heads,kv_heads,dim,page,dtype", [a for a in ATTN])
def test_weight_sums(news, lens, heads, kv_heads, dim, page, dtype):
    from zip_kernel_b200 import ops
    c = R.Case(news, lens, heads, kv_heads, dim, page, dtype, seed=6, tail=1)
    lse = R.attention_ref(c)[1].float()
    ref, rel = R.sums_ref(c, lse)
    args = (c.q.cuda(), c.kv(), c.cu.cuda(), c.lengths.cuda(), lse.cuda())
    got = ops.cache_weight_sums_cuda(*args)
    R.assert_within(got, ref, rel * ref, "sums")
    base = torch.rand(ref.shape, generator=torch.Generator().manual_seed(7)).cuda()
    more = base.clone()
    assert ops.cache_weight_sums_cuda(*args, more, max_q_len=max(news)) is more
    R.assert_within(more, base.cpu().double() + ref, rel * ref + 2.0 ** -23 * (base.cpu().double() + ref), "added")
    for b, n in enumerate(lens):
        assert torch.equal(more[b, :, n:], base[b, :, n:])


EVICT = [
    # lens, kv heads, dim, page, budget, sink, recent
    ([100, 5, 0, 33], 2, 128, 16, 32, 2, 7),
    ([1000, 999, 40], 4, 64, 48, 200, 0, 0),
    ([3000], 1, 128, 64, 1500, 4, 100),
    ([64, 65, 66], 8, 128, 16, 64, 32, 32),
    ([17, 300], 3, 64, 16, 1, 1, 0),
    ([2200, 1100], 2, 128, 128, 2048, 4, 500),
]


def evict_sums(c, kind, seed=8):
    g = torch.Generator().manual_seed(seed)
    s = torch.rand(c.n, c.kv_heads, c.cols * c.page, generator=g)
    if kind == "ties":
        s = (s * 4).floor()
    elif kind == "equal":
        s = torch.ones_like(s)
    elif kind == "odd":                                            # negative, both zeros, infinities, NaN
        s = torch.where(s < 0.2, -s, s)
        s[..., ::7], s[..., ::11], s[..., ::13], s[..., ::17], s[..., ::19] = 0.0, -0.0, float("inf"), float("nan"), float("-inf")
    return s


@pytest.mark.parametrize("lens,kv_heads,dim,page,budget,sink,recent", EVICT)
@pytest.mark.parametrize("kind", ["random", "ties", "equal", "odd"])
@pytest.mark.parametrize("where", ["in place", "other"])
def test_evict(lens, kv_heads, dim, page, budget, sink, recent, kind, where):
    from zip_kernel_b200 import ops
    c = R.Case([0] * len(lens), lens, kv_heads, kv_heads, dim, page, "fp16" if dim == 64 else "bf16", seed=9)
    if where == "in place" and budget > c.cols * page:
        budget = c.cols * page
    sums = evict_sums(c, kind)
    kept, new_len, new_sums = R.evict_ref(c, sums, budget, sink, recent)
    kv = c.kv()
    if where == "other":
        o = R.Case([0] * len(lens), [0] * len(lens), kv_heads, kv_heads, dim, 32, "fp16" if dim == 64 else "bf16", seed=10, max_pages=budget // 32 + 1, nhd=True)
        into = o.kv()
    else:
        o, into = c, None
    want_k, want_v = (into or kv).k_pages.cpu().clone(), (into or kv).v_pages.cpu().clone()
    for b in range(c.n):
        for g in range(kv_heads):
            m = int(new_len[b])
            i = torch.arange(m)
            src = kept[b, g, :m].long()
            for want, t in ((want_k, c.k), (want_v, c.v)):
                want[o.table[b, i // o.page].long(), g, i % o.page] = t[c.table[b, src // c.page].long(), g, src % c.page]
    got = ops.cache_evict_cuda(kv, c.lengths.cuda(), sums.cuda(), budget, n_sink=sink, n_recent=recent, into=into)
    assert torch.equal(got[0].cpu(), kept) and torch.equal(got[1].cpu(), new_len)
    assert torch.equal(got[2].cpu()[..., :budget].nan_to_num(123.0), new_sums.nan_to_num(123.0)) and not got[2][..., budget:].any()
    R.assert_within((into or kv).k_pages, want_k, 0.0, "keys")
    R.assert_within((into or kv).v_pages, want_v, 0.0, "values")
