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
