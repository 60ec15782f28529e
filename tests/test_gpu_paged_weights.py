"""Softmax weights of the attention on a paged cache: small ones that are all a row has to see, and
those of scores so large that a step of them is more than a weight can follow."""

import math

import pytest
import torch

from tests import paged_helpers as R

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def cache(n_seqs, slots, heads, dim, dtype, fill):
    """Sequences of `slots` slots, keys zero, values `fill`, pages of 64 in order."""
    from zip_kernel_b200 import ops
    cols = (slots + 63) // 64
    k = torch.zeros(n_seqs * cols, heads, 64, dim, dtype=R.DT[dtype], device=DEV)
    v = torch.full_like(k, fill)
    table = torch.arange(n_seqs * cols, dtype=torch.int32, device=DEV).reshape(n_seqs, cols)
    return ops.PagedKV(k, v, table), k, v


def batch(n_seqs, new, slots):
    return (torch.arange(n_seqs + 1, dtype=torch.int32, device=DEV) * new, torch.full((n_seqs,), slots, dtype=torch.int32, device=DEV))


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new", [1, 4, 64])
@pytest.mark.parametrize("gap", [12, 18, 20])
def test_small_weights_are_all_there_is_to_see(dtype, dim, new, gap):
    """One slot's score is `gap` above all others, its values are zero: the output is what the others, exp(-gap) each, add up
    to.  Enough (sequence, head) pairs that most of them are not split."""
    from zip_kernel_b200 import ops
    B, G, n = 24, 8, 3000
    kv, k, v = cache(B, n, G, dim, dtype, 8.0)
    first = kv.block_table[:, 0].long()
    k[first, :, 0, 0], v[first, :, 0] = gap / 2, 0.0
    q = torch.zeros(B * new, 2 * G, dim, dtype=R.DT[dtype], device=DEV)
    q[..., 0] = 2.0
    cu, lengths = batch(B, new, n)
    out, lse = ops.paged_attention_cuda(q, kv, cu, lengths, max_q_len=new, scale=1.0, return_lse=True)
    others = torch.arange(n - new, n, dtype=torch.float64).repeat(B)          # slots that a row sees besides the first
    w = others * math.exp(-gap)
    u = torch.finfo(R.DT[dtype]).eps / 2
    # half a step of the weights and of the output, the exponentials, the additions; an output below the normal range; and in
    # the kernel for many rows weights below it: they are made 2^7 times as large, so half a step of 2^-24 is 2^-32 of a weight
    rel = 2 * u + 2.0 ** -21 * (1 + gap) + (n + 16) * 2.0 ** -24
    low = others * 8.0 * 2.0 ** -32 if dtype == "fp16" and 2 * new > 32 else torch.zeros_like(others)
    want = (8.0 * w / (1 + w))[:, None, None].expand(out.shape)
    R.assert_within(out, want, rel * want + low[:, None, None] + 2.0 ** -25, "out")
    R.assert_within(lse, (gap + torch.log1p(w))[:, None].expand(lse.shape), 2.0 ** -20 * gap + (n + 16) * 2.0 ** -24, "lse")


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("new", [1, 40, 200])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("log2", list(range(18, 38)))
def test_weights_of_equal_scores_are_equal_however_large_the_scores(dtype, new, sign, log2):
    """All slots have the same key, scores up to 2^39: the output is the mean of the values, a constant."""
    from zip_kernel_b200 import ops
    B, G, n = 3, 2, 700
    kv, k, v = cache(B, n, G, 128, dtype, 3.0)
    a = log2 // 3                                                               # (12 at most: finite as fp16)
    k[...], q = 0.0, torch.zeros(B * new, 2 * G, 128, dtype=R.DT[dtype], device=DEV)
    k[..., 5], q[..., 5] = 1.3 * 2.0 ** a, sign * 1.7 * 2.0 ** a
    scale = 1.1 * 2.0 ** (log2 - 2 * a)                                         # (products that round)
    cu, lengths = batch(B, new, n)
    out = ops.paged_attention_cuda(q, kv, cu, lengths, max_q_len=new, scale=scale)
    # the weights are equal, but for the additions everything cancels; half a step of the weights and of the output
    u = torch.finfo(R.DT[dtype]).eps / 2
    R.assert_within(out, torch.full(out.shape, 3.0), 3.0 * (2 * u + (n + 16) * 2.0 ** -24), "out")


@pytest.mark.parametrize("news,lens,heads,kv_heads,dim,page", [
    ([1, 1, 1, 1], [1, 5, 17, 64], 32, 8, 128, 16),
    ([1, 1], [40, 7], 16, 1, 64, 48),
    ([3, 1, 4], [3, 30, 60], 8, 2, 128, 16),
    ([8], [50], 4, 1, 64, 32),
])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_weights_of_few_rows_are_not_rounded_to_the_type(news, lens, heads, kv_heads, dim, page, dtype):
    """One rounding, that of the output: a weight enters as two terms, which leave (half a step)^2 of it.  Queries and keys are
    small whole numbers, their products and sums exact."""
    from zip_kernel_b200 import ops
    c = R.Case(news, lens, heads, kv_heads, dim, page, dtype, seed=23)
    g = torch.Generator().manual_seed(24)
    c.q = torch.randint(-2, 3, c.q.shape, generator=g).to(c.dt)
    c.k = torch.where(torch.isnan(c.k), c.k, torch.randint(-2, 3, c.k.shape, generator=g).to(c.dt))
    ref, _, amp, mag = R.attention_ref(c)
    out = ops.paged_attention_cuda(c.q.to(DEV), c.kv(), c.cu.to(DEV), c.lengths.to(DEV), max_q_len=max(news))
    u = torch.finfo(c.dt).eps / 2
    # the scale's rounding and the exponentials, the additions
    rel = u * u + 2.0 ** -21 * (1 + mag) + (max(lens) + 16) * 2.0 ** -24
    R.assert_within(out, ref, u * ref.abs() + 1.01 * rel[..., None] * (amp + ref.abs()) + 2.0 ** -25, "out")


@pytest.mark.parametrize("news,lens,heads,kv_heads", [
    ([4, 5, 8, 9, 1, 0, 3, 6], [300, 5, 130, 700, 64, 40, 3, 257], 32, 8),       # 16 rows and fewer, 20, 32, 36 side by side
    ([1] * 64, [1 + (37 * b) % 400 for b in range(64)], 24, 1),                  # 24 rows of one token each
    ([8, 4], [500, 333], 16, 4), ([5] * 15, [20 + 31 * b for b in range(15)], 16, 4),      # fewer than 64 pairs
])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_sequences_on_both_sides_of_the_border(news, lens, heads, kv_heads, dtype):
    from zip_kernel_b200 import _lib, ops
    c = R.Case(news, lens, heads, kv_heads, 64, 16, dtype, seed=25, q_scale=2.0)
    ref, ref_lse, amp, mag = R.attention_ref(c)
    for max_q in (max(news), None):
        out, lse = ops.paged_attention_cuda(c.q.to(DEV), c.kv(), c.cu.to(DEV), c.lengths.to(DEV), max_q_len=max_q, return_lse=True)
        R.assert_within(out, ref, R.attention_tolerance(c, ref, amp, mag), "out")
        R.assert_within(lse, ref_lse, R.lse_tolerance(c, ref_lse, mag), "lse")
    assert _lib.device_error(DEV) == 0
