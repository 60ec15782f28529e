"""Checks of the paged-cache operators that look at shapes and strides alone: no GPU."""

import pytest
import torch


def table(rows, cols, strides=None):
    t = torch.zeros(4096, dtype=torch.int32)
    return t[:rows * cols].view(rows, cols) if strides is None else t.as_strided((rows, cols), strides)


@pytest.mark.parametrize("t,stride", [
    (table(4, 6), 6), (table(4, 6, (9, 1)), 9), (table(1, 6, (0, 1)), 6), (table(0, 6), 6), (table(4, 1, (1, 7)), 1), (table(4, 1, (5, 0)), 5),
    (table(4, 6)[:, :0], 6), (table(4, 0), 1), (table(3, 6).expand(3, 6), 6), (table(1, 6).expand(1, 6), 6),
])
def test_row_stride_of_a_block_table(t, stride):
    from zip_kernel_b200 import paged_ops
    assert paged_ops._table_stride(t) >= t.shape[1] and (t.shape[0] < 2 or paged_ops._table_stride(t) == stride)


@pytest.mark.parametrize("t", [
    table(1, 6).expand(4, 6),                               # one row for all sequences: stride 0
    table(4, 6, (5, 1)), table(2, 6, (1, 1)),               # rows that overlap
    table(4, 6, (12, 2)), table(6, 4).T, table(4, 1).expand(4, 3),
])
def test_block_tables_whose_rows_are_not_apart_are_refused(t):
    from zip_kernel_b200 import paged_ops
    with pytest.raises(ValueError, match="apart"):
        paged_ops._table_stride(t)


def test_workspace_query_takes_a_cache_without_pages():
    """It may fail for want of a device, not of a block table; a bad argument is named."""
    from tests.test_paged_refusals import arg
    import ctypes
    from zip_kernel_b200 import _lib
    L = _lib.load()

    def query(kv, T=3, n_heads=32, max_q=1):
        got = L.w4a4_paged_attention_workspace_bytes(ctypes.addressof(kv), T, n_heads, max_q)
        return got, L.w4a4_last_error().decode()

    got, why = query(arg(block_table=None, max_pages=0))
    assert got > 0 or "cuda" in why
    for kw, word in ((dict(T=-1), "negative"), (dict(n_heads=12), "multiple"), (dict(max_q=-1), "max_q_len")):
        got, why = query(arg(), **kw)
        assert got == 0 and word in why


def test_weight_sums_of_more_steps_than_are_counted_are_refused():
    """2^24 slot tiles; a row tile of 8 heads holds 16 tokens, so 2048 tokens make 128 of them: 2^31 steps of a unit."""
    from tests.test_paged_refusals import UNSUPPORTED, arg, sums
    from zip_kernel_b200 import _lib
    slots = ((1 << 27) - 80) * 16
    kv = arg(max_pages=slots // 16, table_stride=slots // 16)
    big = dict(seq=8 * slots, head=slots, n_heads=64, T=1 << 20)
    assert sums(kv, max_q=2048, **big) == UNSUPPORTED and "too many" in _lib.load().w4a4_last_error().decode()


def test_rotation_refuses_tables_of_negative_length_and_misaligned_offsets():
    """Compared as an unsigned number, a negative length would let every position through."""
    import ctypes
    from tests.test_paged_refusals import ALIGN, BAD, P, arg, rope
    from zip_kernel_b200 import _lib
    L, kv = _lib.load(), arg()
    for max_pos in (-1, -2 ** 31):
        assert rope(kv, max_pos=max_pos, T=0) == BAD and "max_pos" in L.w4a4_last_error().decode()
    assert L.w4a4_qkv_rope_cache(ctypes.addressof(kv), P, 48 * 128, P, P, P, P, 64, 128, None, None, 1e-6, 0, P + 2, P, 32 * 128, 128, 0, 32,
                                 None) == ALIGN and "offsets" in L.w4a4_last_error().decode()


def test_outputs_whose_rows_overlap_are_refused():
    """Two blocks would write one place.  Strides that nest either way are taken (nothing to do: no launch)."""
    import ctypes
    from tests.test_paged_refusals import BAD, P, arg, attention, rope, sums
    from zip_kernel_b200 import _lib
    L = _lib.load()

    def out(tok, head, T=3):
        return L.w4a4_paged_attention(ctypes.addressof(arg()), P, 4096, 128, P, P, P, tok, head, None, T, 32, 1, 0.1, P, 1 << 30, None)

    for tok, head in ((128, 128), (4096 - 128, 128), (128, 256), (200, 136)):
        assert out(tok, head) == BAD and "out overlap" in L.w4a4_last_error().decode()
        assert rope(arg(), q_tok=tok, q_head=head) == BAD and "q_out overlap" in L.w4a4_last_error().decode()
    for seq, head in ((64, 64), (8 * 64 - 1, 64), (64, 127)):
        assert sums(arg(), seq=seq, head=head, T=0) == BAD and "sums overlap" in L.w4a4_last_error().decode()
    for seq, head in ((8 * 64, 64), (64, 128), (600, 70)):
        assert sums(arg(), seq=seq, head=head, T=0) == 0
    for st in ((8 * 16 * 128, 16 * 128, 64), (8 * 16 * 128, 128, 128), (128, 9 * 128, 9 * 8 * 64), (8 * 16 * 128 - 8, 16 * 128, 128)):
        for kw in (dict(k_strides=st), dict(v_strides=st)):
            assert attention(arg(**kw), T=0) == BAD and "overlap" in L.w4a4_last_error().decode()
    for st in ((8 * 16 * 128, 128, 8 * 128), (128, 9 * 128, 9 * 8 * 128), (2 * 8 * 16 * 128, 16 * 136, 136)):
        assert attention(arg(k_strides=st, v_strides=st), T=0) == 0
