"""Calls from several host threads of one process."""

import pytest
import torch

from tests import paged_helpers as R

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def in_threads(*jobs):
    """Runs the jobs at once, on the default stream of each thread, and passes on the first exception."""
    import threading
    errors, start = [], threading.Barrier(len(jobs))

    def work(job):
        try:
            start.wait()
            job()
        except BaseException as e:                                           # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(j,)) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    if errors:
        raise errors[0]


def test_first_cuda_call_of_a_thread():
    """Threads that have no current context yet: all that the calls need is there, so nothing else makes one current."""
    from zip_kernel_b200 import ops, synth
    c = R.Case([1, 40], [50, 60], 8, 2, 128, 16, "fp16", seed=30)
    kv, q, cu, n = c.kv(), c.q.to(DEV), c.cu.to(DEV), c.lengths.to(DEV)
    want, lse = ops.paged_attention_cuda(q, kv, cu, n, return_lse=True)
    want_sums = ops.cache_weight_sums_cuda(q, kv, cu, n, lse, torch.zeros(2, 2, kv.max_slots, device=DEV))
    out, total = torch.zeros_like(want), torch.zeros_like(want_sums)
    X = synth.make_activations(300, 512, seed=1).to(DEV)
    W = [synth.make_container(256, 512, 0.2, seed=2).to(DEV) for _ in range(2)]
    xs4, sx, sumx = ops.activation_quant_cuda(X, W[0].perm)
    codes, group_sums = ops.expand_activations_cuda(xs4, sumx)

    def linear(w):
        return ops.fused_dense_sparse_expanded_cuda(w.W_low_packed, w.W_high_blocks_packed, w.hp_row_offsets, w.hp_col_indices, codes,
                                                    group_sums, w.scale_u4, w.zero_u4, sx, 256, 512)

    want_y, y = linear(W[0]), []
    torch.cuda.synchronize()
    in_threads(lambda: ops.paged_attention_cuda(q, kv, cu, n, out=out))
    in_threads(lambda: ops.cache_weight_sums_cuda(q, kv, cu, n, lse, total))
    in_threads(lambda: y.append(linear(W[1])))               # (weights at addresses that no call has seen)
    assert torch.equal(out, want) and torch.equal(total, want_sums) and torch.equal(y[0], want_y)


def test_attention_of_threads_that_share_a_stream():
    """Prompts whose units are cut (a join after the kernel), a mixed batch and decode steps, issued by four threads on one
    stream with one workspace: the bits that each gives alone."""
    from zip_kernel_b200 import _lib, ops
    cases = [R.Case([64], [3000], 8, 2, 128, 16, "fp16", seed=31), R.Case([200, 3, 90], [900, 40, 2000], 8, 2, 128, 16, "fp16", seed=32),
             R.Case([1] * 9, [700 - 60 * b for b in range(9)], 8, 2, 128, 16, "fp16", seed=33), R.Case([33], [1500], 8, 2, 64, 32, "bf16", seed=34)]
    args = [(c.q.to(DEV), c.kv(), c.cu.to(DEV), c.lengths.to(DEV)) for c in cases]
    want = [ops.paged_attention_cuda(*a, max_q_len=max(c.news)) for a, c in zip(args, cases)]
    got = [[] for _ in cases]

    def job(i):
        return lambda: got[i].extend(ops.paged_attention_cuda(*args[i], max_q_len=max(cases[i].news)) for _ in range(150))

    in_threads(*(job(i) for i in range(len(cases))))
    for w, outs in zip(want, got):
        assert len(outs) == 150 and all(torch.equal(o, w) for o in outs)
    assert _lib.device_error(DEV) == 0


def test_linears_of_threads_that_share_a_stream():
    """Quantisation and GEMM of four threads on one stream with one workspace, few tokens and many: the bits that each gives alone."""
    from zip_kernel_b200 import _lib, synth, v9_linear
    W = synth.make_container(512, 1024, 0.2, seed=3).to(DEV)
    X = [synth.make_activations(t, 1024, seed=40 + t).to(DEV) for t in (4, 40, 300, 301)]
    want = [v9_linear.v9_linear_forward(x, W) for x in X]
    got = [[] for _ in X]

    def job(i):
        return lambda: got[i].extend(v9_linear.v9_linear_forward(X[i], W) for _ in range(150))

    in_threads(*(job(i) for i in range(len(X))))
    for w, outs in zip(want, got):
        assert len(outs) == 150 and all(torch.equal(o, w) for o in outs)
    assert _lib.device_error(DEV) == 0
