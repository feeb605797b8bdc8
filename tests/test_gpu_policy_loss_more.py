"""The policy loss and the log-probabilities where a batch is unusual: rows behind the last sequence,
types, sizes and magnitudes beyond the ordinary.  Oracle and bounds: tests/test_gpu_policy_loss.py."""

import pytest
import torch

from test_gpu_policy_loss import Oracle, close, make, policy_inputs, policy_oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("chunk", [4096, 40])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_rows_behind_the_last_sequence_may_hold_anything(bad, chunk):
    """Their targets may be vocabulary rows: they count as ignored all the same."""
    from bastile_b200.ops.fused_linear_policy_loss import fused_linear_policy_loss

    x, w, t, _, g = make(90, 128, 700, torch.bfloat16, seed=21)
    o = Oracle(x, w, t)
    old, adv, ref = policy_inputs(o, g)
    cu = torch.tensor([0, 30, 30, 71], dtype=torch.int32, device=DEV)

    def grads():
        xx, ww = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        pl = fused_linear_policy_loss(xx, ww, t, old, adv, ref, kl_coef=0.1, cu_seqlens=cu, chunk_size=chunk)
        return (pl.loss.detach(), pl.log_probs, pl.kl, *torch.autograd.grad(pl.loss, (xx, ww)))

    want = grads()
    assert (t[71:] >= 0).any()
    x[71:], old[71:], adv[71:], ref[71:] = bad, bad, bad, bad
    for a, b in zip(grads(), want):
        assert torch.equal(a, b)
    assert (want[3][71:] == 0).all()


def test_bad_offsets_give_no_gradient_whatever_the_rows_hold():
    from bastile_b200 import _lib
    from bastile_b200.ops.fused_linear_policy_loss import fused_linear_policy_loss

    x, w, t, _, _ = make(20, 64, 50, torch.bfloat16, seed=22)
    x[:] = float("nan")
    x.requires_grad_(True), w.requires_grad_(True)
    got = fused_linear_policy_loss(x, w, t, torch.zeros(20, device=DEV), torch.ones(20, device=DEV),
                                   cu_seqlens=torch.tensor([0, 8, 21], device=DEV))
    assert got.loss == 0
    for grad in torch.autograd.grad(got.loss, (x, w)):
        assert (grad == 0).all()
    with pytest.raises(_lib.BastileB200Error, match="offsets"):
        _lib.check_all_status()
