"""Evictions from histories of more than 8192 slots, whose sums a block of the selection does not hold in registers."""

import types

import pytest
import torch

from tests import paged_helpers as R
from tests.test_gpu_paged_ops import evict_sums

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def case(lens, kv_heads, dim, page, seed):
    g = torch.Generator().manual_seed(seed)
    c = types.SimpleNamespace(n=len(lens), lens=lens, kv_heads=kv_heads, page=page, cols=(max(lens) + page - 1) // page,
                              lengths=torch.tensor(lens, dtype=torch.int32))
    pages = c.n * c.cols
    c.table = torch.randperm(pages, generator=g).reshape(c.n, c.cols).to(torch.int32)
    c.k, c.v = (torch.randn(pages, kv_heads, page, dim, generator=g).half() for _ in range(2))
    return c


@pytest.mark.parametrize("lens,kv_heads,budget,sink,recent", [
    ([8193, 300, 8192], 2, 1000, 4, 100), ([20011, 9000], 1, 9500, 0, 0), ([8193], 1, 8192, 3, 5000), ([12000, 0, 8191], 1, 1, 0, 1),
    ([20011], 3, 15000, 7000, 8000),
])
@pytest.mark.parametrize("kind", ["random", "ties", "equal", "odd"])
@pytest.mark.parametrize("where", ["in place", "other"])
def test_evict_from_long_histories(lens, kv_heads, budget, sink, recent, kind, where):
    from zip_kernel_b200 import _lib, ops
    c = case(lens, kv_heads, 64, 64, 50)
    sums = evict_sums(c, kind)
    kept, new_len, new_sums = R.evict_ref(c, sums, budget, sink, recent)
    kv, into, o = ops.PagedKV(c.k.to(DEV), c.v.to(DEV), c.table.to(DEV)), None, c
    want_k, want_v = c.k.clone(), c.v.clone()
    if where == "other":
        o = case([budget] * c.n, kv_heads, 64, 32, 51)
        into = ops.PagedKV(o.k.to(DEV), o.v.to(DEV), o.table.to(DEV))
        want_k, want_v = o.k.clone(), o.v.clone()
    for b in range(c.n):
        for g in range(kv_heads):
            i, src = torch.arange(int(new_len[b])), kept[b, g, :int(new_len[b])].long()
            for want, t in ((want_k, c.k), (want_v, c.v)):
                want[o.table[b, i // o.page].long(), g, i % o.page] = t[c.table[b, src // c.page].long(), g, src % c.page]
    got = ops.cache_evict_cuda(kv, c.lengths.to(DEV), sums.to(DEV), budget, n_sink=sink, n_recent=recent, into=into)
    assert torch.equal(got[0].cpu(), kept) and torch.equal(got[1].cpu(), new_len)
    assert torch.equal(got[2].cpu()[..., :budget].nan_to_num(123.0), new_sums.nan_to_num(123.0)) and not got[2][..., budget:].any()
    assert torch.equal((into or kv).k_pages.cpu(), want_k) and torch.equal((into or kv).v_pages.cpu(), want_v)
    assert _lib.device_error(DEV) == 0


def test_fresh_sums_of_the_longest_table_are_written_whole():
    """2^31 - 2048 slots a row, eight in use: zeros behind them all the same."""
    from zip_kernel_b200 import _lib, ops
    slots = 2 ** 31 - 2048
    k = torch.randn(1, 1, 16, 64, generator=torch.Generator().manual_seed(52)).half().to(DEV)
    kv = ops.PagedKV(k, k, torch.zeros(1, slots // 16, dtype=torch.int32, device=DEV))
    q, cu = torch.randn(1, 2, 64, generator=torch.Generator().manual_seed(53)).half().to(DEV), torch.tensor([0, 1], dtype=torch.int32, device=DEV)
    n = torch.tensor([8], dtype=torch.int32, device=DEV)
    _, lse = ops.paged_attention_cuda(q, kv, cu, n, max_q_len=1, return_lse=True)
    sums = torch.full((1, 1, slots), float("nan"), device=DEV)
    assert _lib.load().w4a4_cache_weight_sums_fresh(kv._ptr, q.data_ptr(), 128, 64, cu.data_ptr(), n.data_ptr(), lse.data_ptr(), sums.data_ptr(),
                                                    slots, slots, 1, 2, 1, 0.125, _lib.stream_ptr(DEV)) == 0
    small = ops.cache_weight_sums_cuda(q, ops.PagedKV(k, k, torch.zeros(1, 1, dtype=torch.int32, device=DEV)), cu, n, lse)
    assert torch.equal(sums[..., :16], small) and not sums[..., 16:].any() and _lib.device_error(DEV) == 0
