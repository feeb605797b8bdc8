"""Packed attention: the kernel of ordinary batches for every kind of head, small gradients, plans that are
dropped, memory that is not aligned.  Oracle and bounds: tests/test_gpu_packed_attention.py."""

import pytest
import torch

from test_gpu_packed_attention import attend, close, inputs, oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_a_dropped_plan_outlives_the_calls_on_another_stream():
    from bastile_b200.ops.packed_attention import pack_sequences, packed_attention

    q, k, v, cu, dout = inputs([200, 3, 60], 4, 2, 64, torch.bfloat16, seed=31)
    want = attend(q, k, v, cu, dout)
    side = torch.cuda.Stream()
    for _ in range(3):
        seqs = pack_sequences(torch.tensor(cu, dtype=torch.int32, device=DEV), 263)
        words = seqs.plan.numel()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            xs = [x.detach().clone().requires_grad_(True) for x in (q, k, v)]
            torch.cuda._sleep(20_000_000)  # about 10 ms
            out = packed_attention(*xs, seqs)
            got = (out.detach(), *torch.autograd.grad(out, xs, dout))
        del seqs, out
        # the first stream's next tensors of that size (zeros: a plan without tiles)
        reuse = [torch.zeros(words, dtype=torch.int32, device=DEV) for _ in range(8)]
        torch.cuda.synchronize()
        for n, x in zip(("out", "dq", "dk", "dv"), got):
            assert torch.equal(x, want[n]), n
        del reuse
