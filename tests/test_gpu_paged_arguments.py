"""Calls on a paged cache that are refused, or that must not depend on what was called before."""

import pytest
import torch

from tests import paged_helpers as R

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def test_a_block_table_that_sequences_share_is_refused():
    from zip_kernel_b200 import ops
    c = R.Case([1, 3], [50, 60], 8, 2, 128, 16, "fp16", seed=30)
    kv = c.kv()
    row = kv.block_table[:1]
    for bad in (row.expand(2, -1), kv.block_table.flatten().as_strided((2, 4), (2, 1))):
        with pytest.raises(ValueError, match="apart"):
            ops.PagedKV(kv.k_pages, kv.v_pages, bad)
    # made contiguous it is a table like any other: both sequences read the same pages
    shared = ops.PagedKV(kv.k_pages, kv.v_pages, row.expand(2, -1).contiguous())
    q, cu, n = c.q.to(DEV), torch.tensor([0, 1, 2], dtype=torch.int32, device=DEV), torch.full((2,), 50, dtype=torch.int32, device=DEV)
    out = ops.paged_attention_cuda(q[:1].repeat(2, 1, 1), shared, cu, n, max_q_len=1)
    ref, _, amp, mag = R.attention_ref(c)
    R.assert_within(out, ref[:1].expand(2, -1, -1), R.attention_tolerance(c, ref, amp, mag)[:1].expand(2, -1, -1), "out")


def test_sequences_without_any_page_need_no_earlier_call():
    """A block table without columns has no address; the workspace is this call's own."""
    from zip_kernel_b200 import _lib, ops
    c = R.Case([2, 1], [4, 7], 8, 2, 128, 16, "fp16", seed=20)
    full, cu, n, q = c.kv(), c.cu.to(DEV), torch.zeros(2, dtype=torch.int32, device=DEV), c.q.to(DEV)
    kv = ops.PagedKV(full.k_pages, full.v_pages, torch.zeros(2, 0, dtype=torch.int32, device=DEV))
    for q_len in (2, 1):
        with _lib.use_workspace(_lib.WorkspaceHolder()):
            out, lse = ops.paged_attention_cuda(q, kv, cu if q_len == 2 else torch.tensor([0, 1, 2], dtype=torch.int32, device=DEV), n,
                                                max_q_len=q_len, return_lse=True)
        assert (out[:q_len + 1] == 0).all() and (lse[:q_len + 1] == float("-inf")).all()
    assert _lib.device_error(DEV) == 0


@pytest.mark.parametrize("length,written", [(97, [0, 1]), (98, [0]), (99, []), (200, []), (2 ** 31 - 1, []), (-1, []), (-2 ** 31, []), (2, [1, 2])])
def test_tokens_beyond_the_table_take_no_other_slot(length, written):
    """Sequence 1 has three new tokens and six pages of 16 slots: those whose slot exists are written there, the others nowhere."""
    from zip_kernel_b200 import _lib, ops
    c = R.Case([1, 3], [50, 96], 8, 2, 128, 16, "fp16", seed=35, max_pages=6)
    cos = torch.ones(256, 64, device=DEV)
    sin = torch.zeros(256, 64, device=DEV)
    kv, n = c.kv(), torch.tensor([50, length], dtype=torch.int32, device=DEV)
    want_k, want_v = c.k.clone(), c.v.clone()
    rows = c.qkv.view(4, 12, 128)
    for t, slot in [(0, 49)] + [(1 + i, length - 3 + i) for i in written]:
        b = min(t, 1)
        page, at = int(c.table[b, slot // 16]), slot % 16
        want_k[page, :, at], want_v[page, :, at] = rows[t, 8:10], rows[t, 10:12]
    _lib.device_error(DEV)
    ops.qkv_rope_cache_cuda(c.qkv.to(DEV), kv, c.cu.to(DEV), n, cos, sin)
    assert _lib.device_error(DEV) != 0
    assert torch.equal(kv.k_pages.cpu().nan_to_num(9.0), want_k.nan_to_num(9.0))
    assert torch.equal(kv.v_pages.cpu().nan_to_num(9.0), want_v.nan_to_num(9.0))
