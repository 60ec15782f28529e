"""The decoder stack on the paged cache: which tokens' weight an eviction goes by, and what the operators are handed."""

import pytest
import torch

from tests import paged_helpers as R
from tests.test_gpu_paged_cache import View, small_cfg

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def stack(max_len, **kw):
    from zip_kernel_b200 import decoder_stack as ds
    return ds.DecoderStack(small_cfg(qk_norm=True), 2, max_len, DEV, seed=6, paged=True, **kw)


def prompt(cfg, n):
    return torch.randint(0, cfg.vocab, (2, n), generator=torch.Generator().manual_seed(7)).to(DEV)


@pytest.mark.parametrize("S", [40, 20])
def test_weight_of_a_prompt_in_chunks_is_that_of_its_last_tokens(S):
    """A token's weights add up to one: every head pair's sums come to the number of counted tokens times the heads that share
    the keys.  With normed heads of 64 elements a score's products add up to 64 / 8 at most, an fp32 score is off by
    72 * 2^-23 * 8 and a weight, whose logarithm takes a score and a sum, by less than 2^-12."""
    s = stack(48, track_weights=True)
    counted, whole = min(S, s.WEIGHT_WINDOW), None
    for chunk in (0, 24, 33, 7, 1):
        s.reset()
        with torch.no_grad():
            s.prefill(prompt(s.cfg, S), chunk)
        got = s.cache.sums.double().sum(-1)
        want = counted * s.cfg.n_heads // s.cfg.n_kv_heads
        assert ((got - want).abs() <= want * 2.0 ** -12).all(), (chunk, got)
        # slot by slot as with the whole prompt: linears of other token counts add in another order, so that queries and keys
        # of the first layer are up to three half steps of 2^-11 off on either side, of scores up to 8: 2.4 %, twice
        first = s.cache.sums[0, ..., :S]
        whole = first.clone() if whole is None else whole
        assert ((first - whole).abs() <= 0.05 * whole).all(), chunk


def test_sums_after_a_run_do_not_depend_on_the_graph(monkeypatch):
    from zip_kernel_b200 import decoder_stack as ds
    made = []

    class Recorded(ds.DecoderStack):
        def __init__(self, *a, **kw):
            super().__init__(*a, **kw)
            made.append(self)

    monkeypatch.setattr(ds, "DecoderStack", Recorded)
    for graph in (True, False):
        ds.run(small_cfg(), batch=2, prefill_len=40, decode_steps=6, device=DEV, use_graph=graph, seed=3, paged=True, chunk=24, evict=12)
    a, b = (s.cache for s in made)
    assert torch.equal(a.sums, b.sums) and torch.equal(a.lengths, b.lengths) and torch.equal(a.offsets, b.offsets)
    assert not a.sums[..., 12:].any()                       # nothing is added once the histories are cut


def test_the_stack_hands_the_operators_the_right_slots_and_positions(monkeypatch):
    """Chunks of a prompt, decode steps, an eviction, decode steps: rotation, cache write and attention of every layer against 64
    bits, at slots and positions that the test counts itself."""
    from zip_kernel_b200 import ops
    s = stack(48, track_weights=True)
    cfg, u = s.cfg, 2.0 ** -11
    slots = seen = calls = 0
    rope, attention = ops.qkv_rope_cache_cuda, ops.paged_attention_cuda

    def checked_rope(qkv, kv, *a, **kw):
        before = kv.k_pages.cpu(), kv.v_pages.cpu()
        q = rope(qkv, kv, *a, **kw)
        n = qkv.shape[0] // 2
        c = View(kv, [n, n], [slots + n] * 2, q)
        c.qkv, (c.k, c.v) = qkv.cpu(), before
        want, k, v, err = R.rope_ref(c, s.cos32.cpu(), s.sin32.cpu(), s.q_norm.cpu(), s.k_norm.cpu(), cfg.rms_eps, True,
                                     torch.tensor([seen - slots] * 2))
        R.assert_within(q, want, u * want.abs() + err + 2.0 ** -24, "queries")
        R.assert_within(kv.k_pages, k, u * k.abs() + err + 2.0 ** -24, "keys")
        R.assert_within(kv.v_pages, v, 0.0, "values")
        return q

    def checked_attention(q, kv, *a, **kw):
        nonlocal calls
        got = attention(q, kv, *a, **kw)
        n = q.shape[0] // 2
        c = View(kv, [n, n], [slots + n] * 2, q)
        ref, _, amp, mag = R.attention_ref(c)
        R.assert_within(got[0] if isinstance(got, tuple) else got, ref, R.attention_tolerance(c, ref, amp, mag), "attention")
        calls += 1
        return got

    monkeypatch.setattr(ops, "qkv_rope_cache_cuda", checked_rope)
    monkeypatch.setattr(ops, "paged_attention_cuda", checked_attention)
    tokens = prompt(cfg, 40)
    with torch.no_grad():
        for c0, n in ((0, 24), (24, 16)):                    # (one at a time: the counts above go on between them)
            s.prefill(tokens[:, c0:c0 + n])
            slots, seen = slots + n, seen + n
        for step in range(4):
            if step == 2:
                s.cache.evict(12, n_sink=2, n_recent=4)
                slots = 12
            s.decode_step(tokens[:, step], None, 0)
            slots, seen = slots + 1, seen + 1
    assert calls == 6 * cfg.n_layers
