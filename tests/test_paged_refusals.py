"""Argument errors of the paged-cache entry points are reported before any CUDA call: the C ABI without a GPU."""

import ctypes

import pytest


def arg(**kw):
    from zip_kernel_b200 import _lib
    d = dict(k_pages=1 << 20, v_pages=1 << 21, k_strides=(8 * 16 * 128, 16 * 128, 128), v_strides=(8 * 16 * 128, 16 * 128, 128),
             block_table=1 << 22, table_stride=4, n_pages=9, page_size=16, n_kv_heads=8, head_dim=128, n_seqs=2, max_pages=4, dtype=_lib.F16)
    d.update(kw)
    L3 = ctypes.c_longlong * 3
    return _lib.PagedKVArg(d["k_pages"], d["v_pages"], L3(*d["k_strides"]), L3(*d["v_strides"]), d["block_table"], d["table_stride"],
                           d["n_pages"], d["page_size"], d["n_kv_heads"], d["head_dim"], d["n_seqs"], d["max_pages"], d["dtype"])


P = 1 << 24          # an aligned address that nothing reads


def rope(kv, ld=48 * 128, max_pos=64, rot=128, q_tok=32 * 128, q_head=128, T=3, n_heads=32, qkv=P, cos=P, out=P, cu=P):
    from zip_kernel_b200 import _lib
    L = _lib.load()
    return L.w4a4_qkv_rope_cache(ctypes.addressof(kv), qkv, ld, cu, P, cos, P, max_pos, rot, None, None, 1e-6, 0, None, out, q_tok, q_head, T, n_heads, None)


def attention(kv, q=P, tok=4096, head=128, T=3, n_heads=32, max_q=1, scale=0.1, cu=P, out=P, lse=None):
    from zip_kernel_b200 import _lib
    L = _lib.load()
    return L.w4a4_paged_attention(ctypes.addressof(kv), q, tok, head, cu, P, out, 4096, 128, lse, T, n_heads, max_q, scale, P, 1 << 30, None)


def sums(kv, seq=8 * 64, head=64, T=3, n_heads=32, max_q=1, scale=0.1, lse=P):
    from zip_kernel_b200 import _lib
    L = _lib.load()
    return L.w4a4_cache_weight_sums(ctypes.addressof(kv), P, 4096, 128, P, P, lse, P, seq, head, T, n_heads, max_q, scale, None)


def evict(kv, into, budget=8, sink=0, recent=0, seq=8 * 64, head=64, kept=P):
    from zip_kernel_b200 import _lib
    L = _lib.load()
    return L.w4a4_cache_evict(ctypes.addressof(kv), ctypes.addressof(into), P, P, seq, head, budget, sink, recent, kept, P, P, None)


BAD, ALIGN, UNSUPPORTED = 1, 2, 6

CACHES = [
    (dict(dtype=2), BAD, "dtype"), (dict(head_dim=96), BAD, "head_dim"), (dict(page_size=8), BAD, "page_size"),
    (dict(page_size=24), BAD, "page_size"), (dict(n_kv_heads=0), BAD, "positive"), (dict(n_pages=0), BAD, "positive"),
    (dict(n_seqs=-1), BAD, "negative"), (dict(max_pages=1 << 28), BAD, "too long"), (dict(k_pages=None), BAD, "NULL"),
    (dict(block_table=None), BAD, "NULL"), (dict(table_stride=3), BAD, "table_stride"),
    (dict(k_strides=(0, 2048, 128)), BAD, "positive"), (dict(v_strides=(16384, -2048, 128)), BAD, "positive"),
    (dict(v_strides=(16384, 2048, 132)), ALIGN, "multiples of 8"), (dict(k_pages=(1 << 20) + 8), ALIGN, "16-byte"),
]


@pytest.mark.parametrize("kw,code,word", CACHES)
def test_bad_caches_are_refused_by_every_entry_point(kw, code, word):
    from zip_kernel_b200 import _lib
    L = _lib.load()
    kv = arg(**kw)
    for call in (rope, attention, sums, lambda k: evict(k, arg())):
        assert call(kv) == code and word in L.w4a4_last_error().decode()
    assert evict(arg(), kv) == code
    assert L.w4a4_paged_attention_workspace_bytes(ctypes.addressof(kv), 3, 32, 1) == 0


CALLS = [
    (rope, dict(rot=24), BAD, "rot_dim"), (rope, dict(rot=144), BAD, "rot_dim"), (rope, dict(cos=None), BAD, "NULL"),
    (rope, dict(qkv=None), BAD, "NULL"), (rope, dict(ld=47 * 128), BAD, "ld_qkv"), (rope, dict(n_heads=30), BAD, "n_heads"),
    (rope, dict(T=-1), BAD, "negative"), (rope, dict(ld=48 * 128 + 4), ALIGN, "16-byte"), (rope, dict(qkv=P + 2), ALIGN, "16-byte"),
    (rope, dict(q_head=64), BAD, "head stride"), (rope, dict(q_tok=4100), ALIGN, "multiples of 8"), (rope, dict(cu=None), BAD, "cu_seqlens"),
    (attention, dict(max_q=-1), BAD, "max_q_len"), (attention, dict(scale=0.0), BAD, "scale"), (attention, dict(scale=-1.0), BAD, "scale"),
    (attention, dict(scale=float("nan")), BAD, "scale"), (attention, dict(scale=float("inf")), BAD, "scale"),
    (attention, dict(q=None), BAD, "NULL"), (attention, dict(out=None), BAD, "NULL"), (attention, dict(n_heads=12), BAD, "n_heads"),
    (attention, dict(lse=P + 2), ALIGN, "lse"), (attention, dict(tok=64), BAD, "token stride"),
    (sums, dict(head=63), BAD, "strides"), (sums, dict(seq=10), BAD, "strides"), (sums, dict(lse=None), BAD, "NULL"),
    (sums, dict(scale=0.0), BAD, "scale"), (sums, dict(n_heads=8 * 129), UNSUPPORTED, "share"),
]


@pytest.mark.parametrize("call,kw,code,word", CALLS)
def test_bad_calls_are_refused(call, kw, code, word):
    from zip_kernel_b200 import _lib
    assert call(arg(), **kw) == code
    assert word in _lib.load().w4a4_last_error().decode()


@pytest.mark.parametrize("into,kw,word", [
    (dict(), dict(budget=0), "budget"), (dict(), dict(budget=65), "budget"), (dict(max_pages=2, table_stride=2), dict(budget=33), "budget"),
    (dict(), dict(sink=5, recent=4), "n_sink"), (dict(), dict(sink=-1), "n_sink"), (dict(n_seqs=3), dict(), "differ"),
    (dict(head_dim=64), dict(), "differ"), (dict(dtype=1), dict(), "differ"), (dict(), dict(kept=None), "NULL"), (dict(), dict(head=32), "strides"),
])
def test_bad_evictions_are_refused(into, kw, word):
    from zip_kernel_b200 import _lib
    assert evict(arg(), arg(**into), **kw) == BAD
    assert word in _lib.load().w4a4_last_error().decode()


def test_nothing_to_do_needs_no_gpu():
    assert rope(arg(), T=0) == 0 and attention(arg(), T=0) == 0 and sums(arg(), T=0) == 0
    empty = dict(n_seqs=0, block_table=None)
    assert rope(arg(**empty)) == 0 and attention(arg(**empty)) == 0 and sums(arg(**empty)) == 0 and evict(arg(**empty), arg(**empty)) == 0
    assert attention(arg(), max_q=0) == 0


def test_cache_handle_refuses_host_tensors():
    import torch
    from zip_kernel_b200 import ops
    pages = torch.zeros(4, 2, 16, 128, dtype=torch.float16)
    with pytest.raises(ValueError, match="CUDA"):
        ops.PagedKV(pages, pages, torch.zeros(1, 2, dtype=torch.int32))


@pytest.mark.parametrize("kw,word", [(dict(T=0), "no new token"), (dict(max_q=0), "no new token"), (dict(T=-1), "negative"), (dict(n_heads=12), "multiple")])
def test_sums_that_hold_nothing_need_a_new_token(kw, word):
    from zip_kernel_b200 import _lib
    L, d = _lib.load(), dict(T=3, n_heads=32, max_q=1)
    d.update(kw)
    kv = arg()
    assert L.w4a4_cache_weight_sums_fresh(ctypes.addressof(kv), P, 4096, 128, P, P, P, P, 8 * 64, 64, d["T"], d["n_heads"], d["max_q"], 0.1, None) == BAD
    assert word in L.w4a4_last_error().decode()
