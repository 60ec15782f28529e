"""Operators on a paged key/value cache: what stands between the qkv linear and the o linear of a decoder layer.

* :func:`qkv_rope_cache_cuda`    - norms of queries and keys, position rotation, cache write, in one launch;
* :func:`paged_attention_cuda`   - attention of each sequence's newest tokens (one, or a chunk) over its pages;
* :func:`cache_weight_sums_cuda` - the attention weight every cache slot has received from them;
* :func:`cache_evict_cuda`       - keeps the slots with the most weight, in order, in fewer slots.

They work on a :class:`PagedKV`, the pages of one layer with the block table of the batch, and on two small int32 device
tensors that all layers of a step share: ``cu_seqlens (B + 1)``, the first of the packed new tokens of each sequence and
the end of the last, and ``lengths (B)``, the cache slots in use with the new tokens included.  New token ``i`` of
sequence ``b`` has slot ``lengths[b] - q_len[b] + i`` and sees the slots up to its own.  Their values stay on the device: what
is out of range there is cut or left out and sets the device error word (``_lib.device_error``), see
include/w4a4_b200.h.  Every call is issued on the current stream of the cache's device and can be captured in a graph.
Forward only: no gradient is recorded.

No counterpart in the reference, whose layer harness uses PyTorch here (bench/layer/qwen3_layer_bf16.py:129-241).
"""

from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch

from . import _lib
from .nvtx_shim import traced

_L = _lib.load()

DTYPES = {torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}


def _strides(t: torch.Tensor):
    """Strides in elements; those of dimensions of one entry, which say nothing, as if contiguous."""
    out, inner = [], 1
    for size, stride in zip(reversed(t.shape), reversed(t.stride())):
        out.append(stride if size > 1 else inner)
        inner = out[-1] * size
    return out[::-1]


def _table_stride(table: torch.Tensor) -> int:
    """Row stride of a block table whose rows lie apart."""
    (rows, cols), (row, col) = table.shape, _strides(table)
    if (cols > 1 and col != 1) or (rows > 1 and row < cols):
        raise ValueError(f"the rows of block_table must be contiguous and apart (an expanded one: .contiguous()), got strides {tuple(table.stride())}")
    return max(row, cols)


class PagedKV:
    """Key and value pages ``(n_pages, n_kv_heads, page_size, head_dim)`` fp16 or bf16 and the block table
    ``(B, max_pages)`` int32 of the sequences that use them.  The tensors are referred to, not copied; any strides over
    16-byte multiples go as long as a row's elements are neighbours (a ``(n_pages, page_size, n_kv_heads, head_dim)`` array
    is passed as its transpose).  Keep the object from step to step: the arguments are checked here, once."""

    def __init__(self, k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor):
        for name, t in (("k_pages", k_pages), ("v_pages", v_pages)):
            if not t.is_cuda or t.dim() != 4 or t.dtype not in DTYPES:
                raise ValueError(f"{name} must be a 4-D fp16 or bf16 CUDA tensor, got {t.dtype} {tuple(t.shape)} on {t.device}")
        if v_pages.shape != k_pages.shape or v_pages.dtype != k_pages.dtype or v_pages.device != k_pages.device:
            raise ValueError("k_pages and v_pages differ in shape, dtype or device")
        if block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.device != k_pages.device:
            raise ValueError(f"block_table must be a 2-D int32 tensor on {k_pages.device}, got {block_table.dtype} "
                             f"{tuple(block_table.shape)} on {block_table.device}")
        n_pages, n_kv, page, dim = k_pages.shape
        if dim not in (64, 128):
            raise ValueError(f"head_dim must be 64 or 128, got {dim}")
        if page < 16 or page % 16:
            raise ValueError(f"page_size must be a positive multiple of 16, got {page}")
        if n_pages < 1 or n_kv < 1:
            raise ValueError("there must be a page and a head")
        ks, vs, ts = _strides(k_pages), _strides(v_pages), _table_stride(block_table)
        for name, t, st in (("k_pages", k_pages, ks), ("v_pages", v_pages, vs)):
            if st[3] != 1 or any(s <= 0 or s % 8 for s in st[:3]) or t.data_ptr() % 16:
                raise ValueError(f"{name}: rows must be contiguous, strides positive multiples of 8 elements, the address of 16 bytes; "
                                 f"got strides {tuple(t.stride())}")
        self.k_pages, self.v_pages, self.block_table = k_pages, v_pages, block_table
        self.n_pages, self.n_kv_heads, self.page_size, self.head_dim = (int(x) for x in k_pages.shape)
        self.n_seqs, self.max_pages = (int(x) for x in block_table.shape)
        self.dtype, self.device = k_pages.dtype, k_pages.device
        self.max_slots = self.max_pages * self.page_size
        if self.max_slots >= 2 ** 31 - 1024:
            raise ValueError(f"a sequence of {self.max_pages} pages of {self.page_size} slots is too long")
        self._arg = _lib.PagedKVArg(
            k_pages.data_ptr(), v_pages.data_ptr(), (ctypes.c_longlong * 3)(*ks[:3]), (ctypes.c_longlong * 3)(*vs[:3]),
            block_table.data_ptr(), ts, self.n_pages, self.page_size, self.n_kv_heads, self.head_dim,
            self.n_seqs, self.max_pages, DTYPES[self.dtype])
        self._ptr = ctypes.addressof(self._arg)
        self._cu_shape, self._len_shape = (self.n_seqs + 1,), (self.n_seqs,)
        self._sums_shape = (self.n_seqs, self.n_kv_heads, self.max_slots)
        self._scale = self.head_dim ** -0.5


# The checks below run on every call of a decode loop, whose kernels take a few microseconds: each attribute of a tensor is
# asked for once (a shape or a stride costs a third of a microsecond).

def _check_seqs(kv: PagedKV, cu_seqlens, lengths):
    if cu_seqlens.dtype is not torch.int32 or cu_seqlens.shape != kv._cu_shape or not cu_seqlens.is_contiguous() or cu_seqlens.device != kv.device:
        raise ValueError(f"cu_seqlens must be contiguous int32 of {kv.n_seqs + 1} entries on {kv.device}, got {cu_seqlens.dtype} "
                         f"{tuple(cu_seqlens.shape)} on {cu_seqlens.device}")
    _check_lengths(kv, lengths)


def _check_lengths(kv: PagedKV, lengths):
    if lengths.dtype is not torch.int32 or lengths.shape != kv._len_shape or not lengths.is_contiguous() or lengths.device != kv.device:
        raise ValueError(f"lengths must be contiguous int32 of {kv.n_seqs} entries on {kv.device}, got {lengths.dtype} "
                         f"{tuple(lengths.shape)} on {lengths.device}")


def _row_strides(shape, strides, dim):
    """(token, head) strides, those of dimensions of one entry as if contiguous."""
    return (strides[0] if shape[0] > 1 else shape[1] * dim), (strides[1] if shape[1] > 1 else dim)


def _rows_ok(tok: int, head: int, inner: int, dim: int, ptr: int) -> bool:
    return inner == 1 and head >= dim and tok >= dim and not (tok | head) & 7 and not ptr & 15


def _query_rows(kv: PagedKV, q: torch.Tensor):
    """(q or a copy a kernel can read, T, n_heads, token stride, head stride)"""
    shape = q.shape
    if q.dtype is not kv.dtype or len(shape) != 3 or shape[2] != kv.head_dim or q.device != kv.device:
        raise ValueError(f"q must be (T, n_heads, {kv.head_dim}) {kv.dtype} on {kv.device}, got {q.dtype} {tuple(shape)} on {q.device}")
    T, n_heads, dim = shape
    if n_heads < 1 or n_heads % kv.n_kv_heads:
        raise ValueError(f"q: {n_heads} heads are no multiple of the {kv.n_kv_heads} key/value heads")
    strides = q.stride()
    tok, head = _row_strides(shape, strides, dim)
    if not _rows_ok(tok, head, strides[2], dim, q.data_ptr()):
        q, tok, head = q.clone(memory_format=torch.contiguous_format), n_heads * dim, dim
    return q, T, n_heads, tok, head


def _out_rows(kv: PagedKV, out: Optional[torch.Tensor], T: int, n_heads: int):
    """(output, token stride, head stride)"""
    dim = kv.head_dim
    if out is None:
        return torch.empty((T, n_heads, dim), dtype=kv.dtype, device=kv.device), n_heads * dim, dim
    shape, strides = out.shape, out.stride()
    if shape == (T, n_heads, dim) and out.dtype is kv.dtype and out.device == kv.device:
        tok, head = _row_strides(shape, strides, dim)
        if _rows_ok(tok, head, strides[2], dim, out.data_ptr()):
            return out, tok, head
    raise ValueError(f"out must be ({T}, {n_heads}, {dim}) {kv.dtype} on {kv.device} with contiguous rows over 16-byte strides, got "
                     f"{out.dtype} {tuple(shape)} with strides {tuple(strides)} on {out.device}")


def _aligned(t: Optional[torch.Tensor]):
    """Contiguous and on a 16-byte boundary, copied where it is not."""
    return t if t is None or (t.is_contiguous() and not t.data_ptr() & 15) else t.clone(memory_format=torch.contiguous_format)


def _max_q(max_q_len: Optional[int], T: int) -> int:
    if max_q_len is None:
        return T
    if max_q_len < 0:
        raise ValueError(f"max_q_len must not be negative, got {max_q_len}")
    return min(int(max_q_len), T)


def _check_scale(kv: PagedKV, scale: Optional[float]) -> float:
    if scale is None:
        return kv._scale
    scale = float(scale)
    if not 0.0 < scale < 3e38:
        raise ValueError(f"scale must be positive and finite, got {scale}")
    return scale


@traced("cuda.qkv_rope_cache")
def qkv_rope_cache_cuda(qkv: torch.Tensor, kv: PagedKV, cu_seqlens: torch.Tensor, lengths: torch.Tensor, cos: torch.Tensor,
                        sin: torch.Tensor, *, q_norm: Optional[torch.Tensor] = None, k_norm: Optional[torch.Tensor] = None,
                        eps: float = 1e-6, interleaved: bool = False, offsets: Optional[torch.Tensor] = None,
                        out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """From the output of the fused qkv linear, ``qkv (T, (n_heads + 2 n_kv_heads) * head_dim)``: RMS norms of the query and
    key heads (where ``q_norm`` / ``k_norm (head_dim)`` are given), rotation of their first ``2 * cos.shape[1]`` elements,
    keys and values written to their cache slots.  Returns the queries ``(T, n_heads, head_dim)``.

    ``cos``, ``sin``: float32 ``(max_pos, rot_dim / 2)``; of width 0 nothing is rotated.  A token's position is its cache slot, plus ``offsets[b]`` (int32) where
    that is given: the number of slots evicted from the sequence.  ``interleaved``: pairs are neighbours, else ``i`` and
    ``i + rot_dim / 2``.  Everything is computed in float32 and rounded once.  Tokens behind the last sequence are left as
    ``out`` holds them (undefined without ``out``); ``out`` may be the query columns of ``qkv``."""
    shape, D, device, dtype = qkv.shape, kv.head_dim, kv.device, kv.dtype
    if len(shape) != 2 or qkv.dtype is not dtype or qkv.device != device:
        raise ValueError(f"qkv must be 2-D {dtype} on {device}, got {qkv.dtype} {tuple(shape)} on {qkv.device}")
    T, width = shape
    n_heads = width // D - 2 * kv.n_kv_heads
    if width % D or n_heads < 1 or n_heads % kv.n_kv_heads:
        raise ValueError(f"qkv of width {width} is not n_heads + 2 * {kv.n_kv_heads} heads of {D}, n_heads a multiple of {kv.n_kv_heads}")
    _check_seqs(kv, cu_seqlens, lengths)
    table = cos.shape
    if cos.dtype is not torch.float32 or sin.dtype is not torch.float32 or len(table) != 2 or sin.shape != table:
        raise ValueError("cos and sin must be float32 of one shape (max_pos, rot_dim / 2)")
    if cos.device != device or sin.device != device:
        raise ValueError(f"cos and sin must be on {device}")
    max_pos, half = table
    if half % 8 or 2 * half > D:
        raise ValueError(f"the rotated width must be a multiple of 16 up to {D}, got {2 * half}")
    for name, w in (("q_norm", q_norm), ("k_norm", k_norm)):
        if w is not None and (w.shape != (D,) or w.dtype is not dtype or w.device != device):
            raise ValueError(f"{name} must be ({D},) {dtype} on {device}")
    if offsets is not None:
        _check_lengths(kv, offsets)
    q, tok, head = _out_rows(kv, out, T, n_heads)
    if T == 0 or kv.n_seqs == 0:
        return q
    ld, inner = qkv.stride()
    if T == 1:
        ld = width
    if inner != 1 or ld < width or ld & 7 or qkv.data_ptr() & 15:
        qkv, ld = qkv.clone(memory_format=torch.contiguous_format), width
    cos, sin, q_norm, k_norm = _aligned(cos), _aligned(sin), _aligned(q_norm), _aligned(k_norm)
    with _lib.on_device(device):
        status = _L.w4a4_qkv_rope_cache(
            kv._ptr, qkv.data_ptr(), ld, cu_seqlens.data_ptr(), lengths.data_ptr(), cos.data_ptr(), sin.data_ptr(), max_pos, 2 * half,
            None if q_norm is None else q_norm.data_ptr(), None if k_norm is None else k_norm.data_ptr(), eps, interleaved,
            None if offsets is None else offsets.data_ptr(), q.data_ptr(), tok, head, T, n_heads, _lib.stream_ptr(device))
    if status:
        _lib.check(status, "qkv_rope_cache")
    return q


@traced("cuda.paged_attention")
def paged_attention_cuda(q: torch.Tensor, kv: PagedKV, cu_seqlens: torch.Tensor, lengths: torch.Tensor, *,
                         max_q_len: Optional[int] = None, scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
                         return_lse: bool = False):
    """Causal attention of the new tokens' queries ``q (T, n_heads, head_dim)`` over the cached keys and values, their own
    included: ``out (T, n_heads, head_dim)``, with ``return_lse=True`` ``(out, lse)``, ``lse (T, n_heads)`` float32 the natural
    logarithm of each row's sum of exponentials.

    ``scale``: of the scores, ``head_dim ** -0.5`` by default.  ``max_q_len``: no sequence has more new tokens (``T`` by
    default); pass 1 for a decode step, so that with up to 16 heads on a key/value head only the kernel for few rows is
    launched.  A row that sees no slot is
    zero, its ``lse`` minus infinity.  ``out`` may be ``q``.  Tokens behind the last sequence are left as ``out`` holds them (undefined without
    ``out``, like their ``lse``).  Values within a sequence's length must be finite; what lies behind it does not matter."""
    q, T, n_heads, tok, head = _query_rows(kv, q)
    _check_seqs(kv, cu_seqlens, lengths)
    scale = _check_scale(kv, scale)
    o, o_tok, o_head = _out_rows(kv, out, T, n_heads)
    lse = torch.empty((T, n_heads), dtype=torch.float32, device=kv.device) if return_lse else None
    max_q = _max_q(max_q_len, T)
    if T and kv.n_seqs and max_q:
        device = kv.device
        with _lib.on_device(device):
            stream = _lib.stream_ptr(device)
            ws = _lib.attention_workspace(kv, T, n_heads, max_q, stream)
            status = _L.w4a4_paged_attention(
                kv._ptr, q.data_ptr(), tok, head, cu_seqlens.data_ptr(), lengths.data_ptr(), o.data_ptr(), o_tok, o_head,
                None if lse is None else lse.data_ptr(), T, n_heads, max_q, scale, ws.data_ptr(), ws.numel(), stream)
        if status:
            _lib.check(status, "paged_attention")
    return (o, lse) if return_lse else o


def _check_sums(kv: PagedKV, sums):
    """(sequence stride, head stride)"""
    shape, slots = sums.shape, kv.max_slots
    if sums.dtype is not torch.float32 or shape != kv._sums_shape or sums.device != kv.device:
        raise ValueError(f"sums must be float32 {kv._sums_shape} on {kv.device}, got {sums.dtype} {tuple(shape)} on {sums.device}")
    seq, head, inner = _strides(sums)
    if (shape[2] > 1 and inner != 1) or (shape[1] > 1 and head < slots) or (shape[0] > 1 and seq < slots):
        raise ValueError(f"the rows of sums must be contiguous and apart, got strides {tuple(sums.stride())}")
    return max(seq, slots), max(head, slots)


@traced("cuda.cache_weight_sums")
def cache_weight_sums_cuda(q: torch.Tensor, kv: PagedKV, cu_seqlens: torch.Tensor, lengths: torch.Tensor, lse: torch.Tensor,
                           sums: Optional[torch.Tensor] = None, *, max_q_len: Optional[int] = None,
                           scale: Optional[float] = None) -> torch.Tensor:
    """Adds the attention weight that each cache slot receives from the new tokens to ``sums (B, n_kv_heads, max_slots)``
    float32, in place, and returns it; ``None`` starts from zeros.  ``lse`` is what :func:`paged_attention_cuda` returned for the
    same queries and lengths.  The heads that share a key/value head, 128 at most, are added up.  Slots behind a sequence's length are
    left as they are.  To count the last tokens of a chunk only, pass their rows of ``q`` and ``lse`` and their
    ``cu_seqlens``."""
    q, T, n_heads, tok, head = _query_rows(kv, q)
    _check_seqs(kv, cu_seqlens, lengths)
    if lse.shape != (T, n_heads) or lse.dtype is not torch.float32 or lse.device != kv.device:
        raise ValueError(f"lse must be float32 ({T}, {n_heads}) on {kv.device}, got {lse.dtype} {tuple(lse.shape)} on {lse.device}")
    scale = _check_scale(kv, scale)
    max_q = _max_q(max_q_len, T)
    some, add = T and kv.n_seqs and max_q, _L.w4a4_cache_weight_sums
    if sums is not None:
        seq, group = _check_sums(kv, sums)
    else:
        sums = (torch.empty if some else torch.zeros)(kv._sums_shape, dtype=torch.float32, device=kv.device)
        seq, group, add = kv.n_kv_heads * kv.max_slots, kv.max_slots, _L.w4a4_cache_weight_sums_fresh
    if some:
        lse = lse.contiguous()
        device = kv.device
        with _lib.on_device(device):
            status = add(
                kv._ptr, q.data_ptr(), tok, head, cu_seqlens.data_ptr(), lengths.data_ptr(), lse.data_ptr(), sums.data_ptr(), seq, group,
                T, n_heads, max_q, scale, _lib.stream_ptr(device))
        if status:
            _lib.check(status, "cache_weight_sums")
    return sums


@traced("cuda.cache_evict")
def cache_evict_cuda(kv: PagedKV, lengths: torch.Tensor, sums: torch.Tensor, budget: int, *, n_sink: int = 0, n_recent: int = 0,
                     into: Optional[PagedKV] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Keeps ``budget`` slots of every sequence and key/value head (all of them where a sequence has no more): the first
    ``n_sink``, the last ``n_recent`` and those with the largest ``sums`` in between, equal sums by the lowest slot, NaN least.
    Their keys and values move in their order to the first slots of ``into``, or of ``kv`` itself.

    Returns ``(kept, new_lengths, new_sums)``: the old slot of each new one ``(B, n_kv_heads, budget)`` int32 with -1 behind the
    last, ``min(lengths, budget)``, and the sums that go with the new slots (zero behind the last).  ``lengths`` is not changed, so
    that the layers that share it can follow: assign ``new_lengths`` when all are done, and give
    ``offsets = lengths - new_lengths`` (added up over evictions) to :func:`qkv_rope_cache_cuda` from then on.  Pages that two
    sequences share must not be evicted from; ``into`` must use other pages than ``kv``, or the same ones for the same slots."""
    into = kv if into is None else into
    _check_lengths(kv, lengths)
    seq, head = _check_sums(kv, sums)
    if (into.n_seqs, into.n_kv_heads, into.head_dim, into.dtype, into.device) != (kv.n_seqs, kv.n_kv_heads, kv.head_dim, kv.dtype, kv.device):
        raise ValueError("into differs from kv in sequences, heads, head_dim, dtype or device")
    budget, n_sink, n_recent = int(budget), int(n_sink), int(n_recent)
    if not 1 <= budget <= into.max_slots:
        raise ValueError(f"budget must be 1 .. {into.max_slots}, got {budget}")
    if n_sink < 0 or n_recent < 0 or n_sink + n_recent > budget:
        raise ValueError(f"n_sink ({n_sink}) and n_recent ({n_recent}) must not be negative and fit budget ({budget})")
    kept = torch.empty((kv.n_seqs, kv.n_kv_heads, budget), dtype=torch.int32, device=kv.device)
    new_lengths = torch.empty((kv.n_seqs,), dtype=torch.int32, device=kv.device)
    new_sums = torch.empty((kv.n_seqs, kv.n_kv_heads, into.max_slots), dtype=torch.float32, device=kv.device)
    if kv.n_seqs:
        with _lib.on_device(kv.device):
            status = _L.w4a4_cache_evict(
                kv._ptr, into._ptr, lengths.data_ptr(), sums.data_ptr(), seq, head, budget, n_sink, n_recent, kept.data_ptr(),
                new_lengths.data_ptr(), new_sums.data_ptr(), _lib.stream_ptr(kv.device))
        if status:
            _lib.check(status, "cache_evict")
    return kept, new_lengths, new_sums


__all__ = ["PagedKV", "qkv_rope_cache_cuda", "paged_attention_cuda", "cache_weight_sums_cuda", "cache_evict_cuda"]
