"""A head weight that two losses share, with a registered gradient destination."""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _losses(x, w, t):
    from bastile_b200.ops.fused_linear_cross_entropy import fused_linear_cross_entropy
    from bastile_b200.ops.fused_linear_policy_loss import fused_linear_log_probs, fused_linear_policy_loss

    old, adv = torch.full(t.shape, -5.0, device=DEV), torch.ones(t.shape, device=DEV)
    return [lambda: fused_linear_policy_loss(x, w, t, old, adv).loss, lambda: fused_linear_log_probs(x, w, t).mean(),
            lambda: fused_linear_cross_entropy(x, w, t)]


@pytest.mark.parametrize("pair", [(0, 1), (0, 0), (1, 2), (0, 2)])
def test_two_losses_on_one_head(pair):
    from bastile_b200 import _lib

    torch.manual_seed(3)
    x = torch.randn(50, 64, device=DEV).to(torch.bfloat16)
    w = (0.2 * torch.randn(300, 64, device=DEV)).to(torch.bfloat16).requires_grad_(True)
    t = torch.randint(0, 300, (50,), device=DEV)
    losses = _losses(x, w, t)
    parts = [torch.autograd.grad(losses[i](), w)[0] for i in pair]
    dest = torch.zeros_like(w)
    _lib.register_grad_sink(w.data, dest)
    try:
        (losses[pair[0]]() + losses[pair[1]]()).backward()
        assert torch.equal(w.grad, parts[0] + parts[1])  # two terms: either order gives the same bits
        w.grad = None
        losses[pair[0]]().backward()
        assert w.grad.data_ptr() == dest.data_ptr()  # one use still writes in place
        losses[pair[1]]().backward()
        assert torch.equal(w.grad, parts[0] + parts[1])
    finally:
        _lib.unregister_grad_sinks([dest])
    _lib.check_all_status()


def test_sharded_adamw_sees_the_sum():
    from bastile_b200.optim import ShardedAdamW

    torch.manual_seed(4)
    x = torch.randn(50, 64, device=DEV).to(torch.bfloat16)
    t = torch.randint(0, 300, (50,), device=DEV)
    start = (0.2 * torch.randn(300, 64, device=DEV)).to(torch.bfloat16)
    seen = []

    def keep(bucket, step, hyper, master):
        seen.append(bucket.flat_g[:start.numel()].view(start.shape).clone())

    w = torch.nn.Parameter(start.clone())
    opt = ShardedAdamW([w], update_fn=keep)
    try:
        for _ in range(2):
            losses = _losses(x, w, t)
            want = sum(torch.autograd.grad(losses[i](), w)[0].clone() for i in (0, 1))
            opt.zero_grad()
            (losses[0]() + losses[1]()).backward()
            torch.autograd.grad(losses[2](), w)  # something else on the weight before the step
            opt.step()
            torch.cuda.synchronize()
            assert torch.equal(seen[-1], want)
    finally:
        opt.close()
