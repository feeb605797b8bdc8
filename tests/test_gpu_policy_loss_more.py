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


def scaled_bounds(o, coef, e_coef, top_weight, shifted):
    """Gradients and bounds where fp16 rows are formed scaled.  A row's coefficient is brought into [1/2, 2^15) by a
    power of two 2^-e: half a step of 2^-24 below the normal range is then at most 2^-24 of the coefficient.  Its row
    of x is multiplied by 2^(e - E), E at most three above the greatest e: off by 2^-25 in those units."""
    u = 2.0 ** -11
    coef, e_coef = (torch.where(o.live, c, 0.0)[:, None] for c in (coef, e_coef))
    rel = coef[:, 0].abs() / top_weight
    ex = torch.frexp(rel)[1].double()
    e = torch.where(ex > 15, ex - 15, ex.clamp(max=0))
    e = torch.where(rel > 0, e, -1000.0)
    top = e.max() + 3
    p = (o.z - o.lse[:, None]).exp()
    dl = -coef * p
    dl.scatter_add_(1, o.col, coef)
    e_p = p * (2 * o.e[:, None] + 2.0 ** -19)
    if shifted:
        n, v = o.z.shape
        zz = torch.nn.functional.pad(o.z, (0, -v % 128), value=-torch.inf).view(n, -1, 128)
        e_p = e_p + p * u * (zz - zz.amax(-1, keepdim=True)).view(n, -1)[:, :v].abs()
    e_dl = coef.abs() * (e_p + 2.0 ** -24) + e_coef * (dl.abs() / coef.abs().clamp(min=1e-300)) + u * dl.abs()
    sums = 2.0 ** -19  # fp32 sums
    dx = (dl @ o.w, 1.01 * (e_dl @ o.w.abs() + sums * (dl.abs() @ o.w.abs()) + u * (dl @ o.w).abs()) + 2.0 ** -24)
    e_x = torch.where(rel > 0, 2.0 ** -25 * 2.0 ** (top - e).clamp(max=200), 0.0)[:, None].expand_as(o.x)
    dw = (dl.t() @ o.x, 1.01 * (e_dl.t() @ (o.x.abs() + e_x) + dl.abs().t() @ e_x + sums * (dl.abs().t() @ o.x.abs())))
    return dx, dw


@pytest.mark.parametrize("chunk", [4096, 40])
@pytest.mark.parametrize("what", ["ratios", "kl", "tiny", "mixed"])
def test_fp16_coefficients_of_any_size(what, chunk):
    """Ratios and KL gaps are exponentials: coefficients beyond 65504 (and far below 2^-24) with gradients that are
    ordinary numbers once they are multiplied with a token's weight."""
    from bastile_b200 import _lib
    from bastile_b200.ops.fused_linear_policy_loss import fused_linear_policy_loss

    x, w, t, _, g = make(90, 64, 700, torch.float16, seed=23)
    w32 = w.float()
    o = Oracle(x, w, t)
    old, adv, ref = policy_inputs(o, g)
    kl = 0.0
    if what == "ratios":
        adv[71], adv[3], old[71], old[3] = -1.0, -0.5, o.logp[71] - 13.0, o.logp[3] - 12.0
    elif what == "kl":
        kl, ref[75], ref[2] = 0.05, o.logp[75] + 15.0, o.logp[2] + 14.0
    elif what == "tiny":
        adv *= 1e-7
    else:
        adv[::2] *= 1e-6
        adv[79], old[79] = -1.0, o.logp[79] - 13.0
    up = 1.0 if what != "tiny" else 1e7
    want, *_ = policy_oracle(o, old, adv, ref if kl else None, 0.2, 0.28, kl, None)
    assert (want["coef"].abs().max() * o.live.sum() > 65504) == (what != "tiny")
    dx, dw = scaled_bounds(o, up * want["coef"], up * want["e_coef"], float(up / o.live.sum()), shifted=True)
    x.requires_grad_(True), w32.requires_grad_(True)
    got = fused_linear_policy_loss(x, w32, t, old, adv, ref if kl else None, 0.2, 0.28, kl, chunk_size=chunk)
    for _ in range(2):
        a, b = torch.autograd.grad(got.loss * up, (x, w32), retain_graph=True)
        close(a, *dx, "dhidden")
        close(b, *dw, "dweight")
    _lib.check_all_status()


def test_fp16_ordinary_coefficients_are_left_alone():
    """The same tokens beside one with a huge coefficient and without it: their rows of d hidden have the same bits."""
    from bastile_b200.ops.fused_linear_policy_loss import fused_linear_policy_loss

    x, w, t, _, g = make(60, 64, 700, torch.float16, seed=24)
    o = Oracle(x, w, t)
    old, adv, _ = policy_inputs(o, g)
    x.requires_grad_(True)

    def rows():
        return torch.autograd.grad(fused_linear_policy_loss(x, w, t, old, adv).loss, x)[0]

    want = rows()
    adv[8], old[8] = -1.0, o.logp[8] - 14.0
    got = rows()
    keep = torch.arange(60, device=DEV) != 8
    assert torch.equal(got[keep], want[keep]) and torch.isfinite(got[8]).all() and (got[8] != 0).any()


@pytest.mark.parametrize("chunk", [4096, 40])
def test_fp16_upstream_gradients_of_different_sizes(chunk):
    """Token weights six orders of magnitude apart: a small one's row of d hidden has its own digits."""
    from bastile_b200 import _lib
    from bastile_b200.ops.fused_linear_policy_loss import fused_linear_log_probs

    x, w, t, up, _ = make(90, 64, 700, torch.float16, seed=25)
    w32 = w.float().requires_grad_(True)
    o = Oracle(x, w, t)
    size = 10.0 ** -(torch.arange(90, device=DEV) % 7)
    up = up * size * 64.0
    x.requires_grad_(True)
    top = 2.0 ** float(torch.frexp((up * o.live).abs().max())[1])  # relative to this the largest is in [1/2, 1)
    dx, dw = scaled_bounds(o, up.double(), torch.zeros_like(o.e), top, shifted=False)
    a, b = torch.autograd.grad(fused_linear_log_probs(x, w32, t, chunk_size=chunk), (x, w32), up)
    close(a, *dx, "dhidden")
    close(b, *dw, "dweight")
    _lib.check_all_status()


@pytest.mark.parametrize("need_w", [False, True])
def test_a_smaller_chunk_keeps_no_more_memory(need_w):
    """What a loss keeps until its backward: fp32 d hidden once, whatever its product is cut into."""
    from bastile_b200 import _lib
    from bastile_b200.ops.fused_linear_policy_loss import fused_linear_policy_loss

    rows, h, v, chunk = 2000, 256, 9001, 64
    assert _lib.get_lib().bt_dhidden_runs(chunk, h, v, _lib.BT_BF16) > 4
    x, w, t, _, g = make(rows, h, v, torch.bfloat16, seed=26)
    zero, one = torch.zeros(rows, device=DEV), torch.ones(rows, device=DEV)
    x.requires_grad_(True), w.requires_grad_(need_w)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    got = fused_linear_policy_loss(x, w, t, zero, one, chunk_size=chunk)
    kept = torch.cuda.memory_allocated() - before
    ld = (v + 7) // 8 * 8
    most = 4 * rows * h + (4 * v * h + 2 * rows * h + 2 * chunk * ld if need_w else 0) + 4 * rows
    assert kept <= most + (1 << 20), (kept, most)
    del got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_dense_tensors_off_a_16_byte_boundary(dtype):
    from bastile_b200.ops.fused_linear_policy_loss import fused_linear_log_probs, fused_linear_policy_loss

    def shifted(a):
        buf = torch.empty(a.numel() + 8, dtype=a.dtype, device=DEV)
        y = buf[1:1 + a.numel()].view(a.shape)
        y.copy_(a)
        assert y.data_ptr() % 16 != 0
        return y

    x, w, t, up, g = make(40, 64, 300, dtype, seed=27)
    o = Oracle(x, w, t)
    old, adv, ref = policy_inputs(o, g)

    def both(move):
        a, b, *rest = (move(i) for i in (x, w, t, up, old, adv, ref))
        a.requires_grad_(True), b.requires_grad_(True)
        tt, u, ol, ad, rf = rest
        lp = fused_linear_log_probs(a, b, tt)
        pl = fused_linear_policy_loss(a, b, tt, ol, ad, rf, kl_coef=0.1)
        return (lp.detach(), pl.loss.detach(), *torch.autograd.grad(lp, (a, b), u), *torch.autograd.grad(pl.loss, (a, b)))

    for a, b in zip(both(shifted), both(lambda i: i.clone())):
        assert torch.equal(a, b)


def test_a_reference_for_the_log_alone_does_not_reach_the_loss():
    """kl_coef = 0: a gap whose exponential is infinite shows in the average, not in loss or gradients."""
    from bastile_b200.ops.fused_linear_policy_loss import fused_linear_policy_loss

    x, w, t, _, g = make(30, 64, 200, torch.bfloat16, seed=28)
    o = Oracle(x, w, t)
    old, adv, ref = policy_inputs(o, g)
    ref[5] = 900.0
    x.requires_grad_(True), w.requires_grad_(True)
    a = fused_linear_policy_loss(x, w, t, old, adv)
    b = fused_linear_policy_loss(x, w, t, old, adv, ref)
    assert b.kl == float("inf") and torch.equal(a.loss, b.loss)
    for p, q in zip(torch.autograd.grad(a.loss, (x, w)), torch.autograd.grad(b.loss, (x, w))):
        assert torch.equal(p, q)


@pytest.mark.parametrize("rows,h,v", [(1, 64, 8), (7, 64, 129), (300, 256, 1000), (513, 128, 4099)])
@pytest.mark.parametrize("chunk,kl,packed", [(4096, 0.0, False), (100, 0.1, False), (128, 0.05, True)])
def test_policy_loss_fp32(rows, h, v, chunk, kl, packed):
    from bastile_b200 import _lib
    from bastile_b200.ops.fused_linear_policy_loss import fused_linear_policy_loss

    x, w, t, _, g = make(rows, h, v, torch.float32, seed=rows + 5 * v)
    cu = None
    if packed:
        cu = [0, 1] if rows == 1 else ([0, 3, 3, rows] if rows < 20 else [0, 10, 20, 20, rows // 2, rows - 5])
    o = Oracle(x, w, t)
    old, adv, ref = policy_inputs(o, g)
    ref = ref if kl else None
    want, want_logp, e_logp = policy_oracle(o, old, adv, ref, 0.2, 0.28, kl, cu)
    x.requires_grad_(True), w.requires_grad_(True)
    cut = None if cu is None else torch.tensor(cu, dtype=torch.int32, device=DEV)
    got = fused_linear_policy_loss(x, w, t, old, adv, ref_log_probs=ref, clip_low=0.2, clip_high=0.28, kl_coef=kl,
                                   cu_seqlens=cut, chunk_size=chunk)
    close(got.loss.detach(), want["loss"], want["e_loss"] + 1e-30, "loss")
    close(got.log_probs, want_logp, e_logp, "log_probs")
    # the oracle has 2^-11 for dlogits and 2^-10 for the operands; the tensor cores cut both operands to tf32's 11 bits,
    # off by up to 2^-10 each: 4 / 3 of that
    bounds = o.grads(want["coef"], want["e_coef"], shifted=True)
    for name, grad, like in zip(("dhidden", "dweight"), torch.autograd.grad(got.loss, (x, w)), (x, w)):
        assert grad.dtype == like.dtype == torch.float32
        close(grad, bounds[name][0], bounds[name][1] * 4 / 3, name)
    _lib.check_all_status()


def test_captured_fp16_steps_start_from_their_own_exponents():
    """Chunks hand the greatest exponent on; a replay begins anew, with other advantages too."""
    from bastile_b200.ops.fused_linear_policy_loss import fused_linear_policy_loss

    x, w, t, _, g = make(150, 64, 600, torch.float16, seed=29)
    o = Oracle(x, w, t)
    old, adv, _ = policy_inputs(o, g)
    x.requires_grad_(True)
    w32 = w.float().requires_grad_(True)

    def step():
        return torch.autograd.grad(fused_linear_policy_loss(x, w32, t, old, adv, chunk_size=40).loss, (x, w32))

    plain = (old.clone(), adv.clone())
    huge = (old.clone(), adv.clone())
    huge[0][50], huge[1][50] = o.logp[50] - 14.0, -1.0
    want = {}
    for name, (ol, ad) in (("plain", plain), ("huge", huge)):
        old.copy_(ol), adv.copy_(ad)
        want[name] = step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = step()
    for name, (ol, ad) in (("plain", plain), ("huge", huge), ("plain", plain)):
        old.copy_(ol), adv.copy_(ad)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(res, want[name]):
            assert torch.equal(a, b), name


@pytest.mark.parametrize("rows,chunk", [(1, 4096), (3, 2), (50, 4096), (50, 17)])
def test_fp16_small_coefficients_in_the_weight_gradient(rows, chunk):
    """Advantages of a few percent: probabilities times them have the steps of a coefficient of 1, seen in an fp32
    weight, for the policy loss and the log-probabilities alike."""
    from bastile_b200.ops.fused_linear_policy_loss import fused_linear_log_probs, fused_linear_policy_loss

    x, w, t, up, g = make(rows, 64, 4099, torch.float16, seed=30, ignored=1000)
    t[0] = 7
    x = (x * 1.5).half()
    o = Oracle(x, w, t)
    old, adv, _ = policy_inputs(o, g)
    adv = adv * 0.03
    w32 = w.float().requires_grad_(True)
    want, *_ = policy_oracle(o, old, adv, None, 0.2, 0.28, 0.0, None)
    got = torch.autograd.grad(fused_linear_policy_loss(x, w32, t, old, adv, None, 0.2, 0.28, chunk_size=chunk).loss, w32)[0]
    close(got, *scaled_bounds(o, want["coef"], want["e_coef"], 1.0 / rows, shifted=True)[1], "policy")
    got = torch.autograd.grad(fused_linear_log_probs(x, w32, t, chunk_size=chunk), w32, up)[0]
    close(got, *scaled_bounds(o, up.double(), torch.zeros_like(o.e), 1.0, shifted=False)[1], "log_probs")
