"""Token log-probabilities and the clipped policy loss through the output head, against a plain
implementation in 64 bits.

Bounds, with u = eps / 2 of the operands' type and e the error of a logit: the tensor cores add the K
products in fp32 and may cut every partial sum, e <= (K / 8 + 8) 2^-23 sum |h w| (fp32 operands are
read as tf32: 2^-9 sum |h w| more).  A log-probability is off by the errors of its logit and of the
log-sum-exp, 2 max e, and FAST = 2^-19 for the fast exponentials and fp32 sums.  dlogits are
c (onehot - p): p is off by p (2 max e + FAST), the rounding to 16 bits adds u; the policy loss keeps
logit - (maximum of its 128 columns) in 16 bits, whose rounding moves p by u |difference|.  The products
of those with weight and hidden follow, and one rounding of the result."""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -11}
FAST = 2.0 ** -19


class Oracle:
    def __init__(self, x, w, target, ignore=-100):
        self.dtype = x.dtype
        self.x, self.w = x.detach().double().reshape(-1, x.shape[-1]), w.detach().double()
        self.t = target.reshape(-1)
        self.live = self.t != ignore
        self.x = torch.where(self.live[:, None], self.x, 0.0)
        self.z = self.x @ self.w.t()
        k = self.x.shape[1]
        cut = (k / 8 + 8) * 2.0 ** -23 + (2.0 ** -9 if x.dtype == torch.float32 else 0.0)
        self.e = (cut * (self.x.abs() @ self.w.abs().t())).amax(-1)  # per row
        self.lse = torch.logsumexp(self.z, -1)
        self.col = torch.where(self.live, self.t, 0)[:, None]
        self.logp = torch.where(self.live, self.z.gather(1, self.col)[:, 0] - self.lse, 0.0)
        self.e_logp = torch.where(self.live, 2 * self.e + FAST * (1 + self.logp.abs()), 0.0)

    def grads(self, coef, e_coef, shifted):
        """Gradients for d loss / d logp = coef (off by e_coef), with bounds."""
        u = U[self.dtype]
        coef = torch.where(self.live, coef, 0.0)[:, None]
        e_coef = torch.where(self.live, e_coef, 0.0)[:, None]
        p = (self.z - self.lse[:, None]).exp()
        dl = -coef * p
        dl.scatter_add_(1, self.col, coef)
        e_p = p * (2 * self.e[:, None] + FAST)
        if shifted:
            n, v = self.z.shape
            pad = -v % 128
            zz = torch.nn.functional.pad(self.z, (0, pad), value=-torch.inf).view(n, -1, 128)
            t = (zz - zz.amax(-1, keepdim=True)).view(n, -1)[:, :v]
            e_p = e_p + p * u * t.abs()
        e_dl = coef.abs() * e_p + e_coef * (dl.abs() / coef.abs().clamp(min=1e-300)) + u * dl.abs()
        if self.dtype == torch.float16:  # steps of 2^-24 below the normal range, relative to the largest coefficient
            e_dl = e_dl + 2.0 ** -24 * coef.abs().max()
        fp32 = 2.0 ** -14 * u  # sums in fp32: far below a rounding
        out = {}
        for name, a, b, e_a in (("dhidden", dl, self.w, e_dl), ("dweight", dl.t(), self.x, e_dl.t())):
            g = a @ b
            operand = 2.0 ** -10 * (a.abs() @ b.abs()) if self.dtype == torch.float32 else 0.0  # tf32 operands
            tiny = 2.0 ** -24 if self.dtype == torch.float16 else 0.0
            out[name] = (g, 1.01 * (e_a @ b.abs() + (u if self.dtype != torch.float32 else 0.0) * g.abs() + operand +
                                    (fp32 + 2.0 ** -20) * (a.abs() @ b.abs())) + tiny)
        return out


def close(got, value, bound, what):
    assert torch.isfinite(got).all(), f"{what}: not finite"
    off = (got.double().reshape(value.shape) - value).abs()
    assert (off <= bound).all(), f"{what}: {int((off > bound).sum())} of {off.numel()} outside, worst by " \
                                 f"{float((off - bound).max()):.3e}"


def make(rows, h, v, dtype, seed=0, ignored=7):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = (torch.randn(rows, h, generator=g, device=DEV) * (8 / h ** 0.5)).to(dtype)
    w = (torch.randn(v, h, generator=g, device=DEV) * 0.2).to(dtype)
    t = torch.randint(0, v, (rows,), generator=g, device=DEV)
    if rows > 1:
        t[::ignored] = -100
    up = torch.randn(rows, generator=g, device=DEV)
    return x, w, t, up, g


SIZES = [(1, 64, 8), (7, 64, 129), (300, 256, 1000), (513, 128, 4099), (65, 1024, 2048)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,h,v", SIZES)
@pytest.mark.parametrize("chunk", [4096, 100])
def test_log_probs(rows, h, v, chunk, dtype):
    from bastile_b200 import _lib
    from bastile_b200.ops.fused_linear_policy_loss import fused_linear_log_probs

    x, w, t, up, _ = make(rows, h, v, dtype, seed=rows + v)
    want = Oracle(x, w, t)
    x.requires_grad_(True), w.requires_grad_(True)
    logp = fused_linear_log_probs(x, w, t, chunk_size=chunk)
    assert logp.dtype == torch.float32 and logp.shape == t.shape
    close(logp.detach(), want.logp, want.e_logp, "logp")
    grads = torch.autograd.grad(logp, (x, w), up)
    ref = want.grads(up.double(), torch.zeros_like(want.e), shifted=False)
    for name, g, like in zip(("dhidden", "dweight"), grads, (x, w)):
        assert g.dtype == like.dtype
        close(g, *ref[name], name)
    with torch.no_grad():
        assert torch.equal(fused_linear_log_probs(x, w, t, chunk_size=chunk), logp)
    _lib.check_all_status()


def policy_oracle(o, old, adv, ref, lo, hi, kl_coef, cu):
    w = o.live.double()
    if cu is None:
        w = w / w.sum().clamp(min=1)
    else:
        share = torch.zeros_like(w)
        spans = [(a, b, int(o.live[a:b].sum())) for a, b in zip(cu[:-1], cu[1:])]
        filled = sum(n > 0 for *_, n in spans)
        for a, b, n in spans:
            if n:
                share[a:b] = w[a:b] / n / filled
        w = share
    on = w > 0
    old, adv = torch.where(on, old.double(), 0.0), torch.where(on, adv.double(), 0.0)
    r = torch.where(on, (o.logp - old).exp(), 0.0)
    over = ((adv > 0) & (r > 1 + hi)) | ((adv < 0) & (r < 1 - lo))
    val = -adv * torch.where(over, r.clamp(1 - lo, 1 + hi), r)
    slope = torch.where(over, 0.0, -adv * r)
    e_slope = slope.abs() * o.e_logp
    kl = torch.zeros_like(r)
    if ref is not None:
        d = torch.where(on, ref.double() - o.logp, 0.0)
        kl = torch.expm1(d) - d
        val, slope = val + kl_coef * kl, slope - kl_coef * torch.expm1(d)
        e_slope = e_slope + abs(kl_coef) * d.exp() * o.e_logp
    res = dict(loss=(val * w).sum(), kl=(kl * w).sum(), clip=(over * w).sum(), coef=slope * w)
    res["e_loss"] = (w * (slope.abs() + e_slope) * o.e_logp).sum() + 2.0 ** -22 * (val.abs() * w).sum()
    res["e_kl"] = (w * (torch.expm1(d).abs() + o.e_logp) * o.e_logp).sum() + 2.0 ** -22 * res["kl"] if ref is not None else 0.0
    res["e_coef"] = e_slope * w + 2.0 ** -22 * (slope * w).abs()
    on_logp = torch.where(on, o.logp, 0.0)
    return res, on_logp, torch.where(on, o.e_logp, 0.0)


def policy_inputs(o, g, spread=0.3):
    n = len(o.t)
    delta = spread * torch.randn(n, generator=g, device=DEV).double()
    for border in (0.8, 1.28):  # off the borders, where either branch would be right
        near = (delta - torch.tensor(border).log().item()).abs() < 0.02
        delta = torch.where(near, delta + 0.05, delta)
    old = (o.logp - delta).float()
    ref = (o.logp + 0.4 * torch.randn(n, generator=g, device=DEV)).float()
    adv = torch.randn(n, generator=g, device=DEV)
    return old, adv, ref


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,h,v", SIZES)
@pytest.mark.parametrize("chunk,kl,packed", [(4096, 0.0, False), (100, 0.1, False), (128, 0.05, True), (4096, 0.0, True)])
def test_policy_loss(rows, h, v, chunk, kl, packed, dtype):
    from bastile_b200 import _lib
    from bastile_b200.ops.fused_linear_policy_loss import fused_linear_policy_loss

    x, w, t, _, g = make(rows, h, v, dtype, seed=rows + 3 * v)
    if rows > 20:
        t[10:20] = -100  # one sequence without a counted token
    cu = None
    if packed:
        cu = [0, 1] if rows == 1 else ([0, 3, 3, rows] if rows < 20 else [0, 10, 20, 20, rows // 2, rows - 5])
    o = Oracle(x, w, t)
    old, adv, ref = policy_inputs(o, g)
    ref = ref if kl else None
    want, want_logp, e_logp = policy_oracle(o, old, adv, ref, 0.2, 0.28, kl, cu)
    x.requires_grad_(True), w.requires_grad_(True)
    cut = None if cu is None else torch.tensor(cu, dtype=torch.int64, device=DEV)
    got = fused_linear_policy_loss(x, w, t, old, adv, ref_log_probs=ref, clip_low=0.2, clip_high=0.28, kl_coef=kl,
                                   cu_seqlens=cut, chunk_size=chunk)
    close(got.loss.detach(), want["loss"], want["e_loss"] + 1e-30, "loss")
    close(got.kl, want["kl"], want["e_kl"] + 1e-30, "kl")
    close(got.clip_fraction, want["clip"], 2.0 ** -20, "clip_fraction")
    close(got.log_probs, want_logp, e_logp, "log_probs")
    assert not got.log_probs.requires_grad and got.loss.shape == ()
    dx, dw = torch.autograd.grad(got.loss * 3.0, (x, w), retain_graph=True)
    ref_g = o.grads(3.0 * want["coef"], 3.0 * want["e_coef"], shifted=True)
    close(dx, *ref_g["dhidden"], "dhidden")
    close(dw, *ref_g["dweight"], "dweight")
    again = torch.autograd.grad(got.loss * 3.0, (x, w))  # the saved state survives a backward
    assert torch.equal(dx, again[0]) and torch.equal(dw, again[1])
    with torch.no_grad():
        quiet = fused_linear_policy_loss(x, w, t, old, adv, ref_log_probs=ref, clip_low=0.2, clip_high=0.28,
                                         kl_coef=kl, cu_seqlens=cut, chunk_size=chunk)
    for a, b in zip(quiet, got):
        assert torch.equal(a, b.detach())
    _lib.check_all_status()


def test_ignored_positions_may_hold_anything():
    from bastile_b200.ops.fused_linear_policy_loss import fused_linear_log_probs, fused_linear_policy_loss

    x, w, t, up, g = make(90, 128, 700, torch.bfloat16, seed=1)
    o = Oracle(x, w, t)
    old, adv, ref = policy_inputs(o, g)

    def both(x):
        x, ww = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        lp = fused_linear_log_probs(x, ww, t)
        pl = fused_linear_policy_loss(x, ww, t, old, adv, ref, kl_coef=0.1)
        return (lp.detach(), *torch.autograd.grad(lp, (x, ww), up), pl.loss.detach(), pl.log_probs, pl.kl,
                pl.clip_fraction, *torch.autograd.grad(pl.loss, (x, ww)))

    want = both(x)
    for k, bad in enumerate((float("nan"), float("inf"), -float("inf"))):
        dead = t == -100
        x[dead], up[dead], old[dead], adv[dead], ref[dead] = bad, bad, bad, bad, bad
        for a, b in zip(both(x), want):
            assert torch.equal(a, b)


def test_clipping_on_both_sides_and_infinite_ratios():
    """Ratios far outside: clipped tokens have no policy gradient; a clipped ratio may overflow."""
    from bastile_b200.ops.fused_linear_policy_loss import fused_linear_policy_loss

    x, w, t, _, _ = make(6, 64, 100, torch.bfloat16, seed=2, ignored=100)
    t[0] = 5
    o = Oracle(x, w, t)
    move = torch.tensor([2.0, 2.0, -2.0, -2.0, 0.0, 800.0], device=DEV, dtype=torch.float64)  # log of the ratio
    adv = torch.tensor([1.0, -1.0, 1.0, -1.0, 0.0, 1.0], device=DEV)
    old = (o.logp - move).float()
    x.requires_grad_(True)
    got = fused_linear_policy_loss(x, w, t, old, adv)
    want, *_ = policy_oracle(o, old, adv, None, 0.2, 0.2, 0.0, None)
    close(got.loss.detach(), want["loss"], want["e_loss"], "loss")
    close(got.clip_fraction, torch.tensor(3 / 6, device=DEV).double(), 1e-6, "clip_fraction")
    (dx,) = torch.autograd.grad(got.loss, x)
    for row, moves in enumerate([False, True, True, False, False, False]):
        assert bool((dx[row] != 0).any()) == moves, row


def test_nothing_counted_and_no_rows():
    from bastile_b200.ops.fused_linear_policy_loss import fused_linear_log_probs, fused_linear_policy_loss

    for rows in (0, 5):
        x, w, t, up, _ = make(rows, 64, 100, torch.bfloat16, seed=3)
        t.fill_(-100)
        x.requires_grad_(True), w.requires_grad_(True)
        zero = torch.zeros(rows, device=DEV)
        lp = fused_linear_log_probs(x, w, t)
        assert (lp == 0).all()
        pl = fused_linear_policy_loss(x, w, t, zero, zero + 1)
        assert pl.loss == 0 and pl.kl == 0 and pl.clip_fraction == 0
        for loss, up_ in ((lp, up), (pl.loss, None)):
            for g, like in zip(torch.autograd.grad(loss, (x, w), up_), (x, w)):
                assert g.shape == like.shape and (g == 0).all()


def test_shapes_strides_and_partial_gradients():
    from bastile_b200.ops.fused_linear_policy_loss import fused_linear_log_probs, fused_linear_policy_loss

    x, w, t, up, g = make(60, 128, 300, torch.bfloat16, seed=4)
    o = Oracle(x, w, t)
    old, adv, ref = policy_inputs(o, g)
    x.requires_grad_(True), w.requires_grad_(True)
    lp = fused_linear_log_probs(x, w, t)
    pl = fused_linear_policy_loss(x, w, t, old, adv)
    want = (*torch.autograd.grad(lp, (x, w), up), *torch.autograd.grad(pl.loss, (x, w)))
    wide = torch.randn(3, 21, 136, device=DEV).to(torch.bfloat16)  # a [3, 20, 128] slice of a larger tensor
    wide[:, :20, 8:] = x.detach().view(3, 20, 128)
    for view in (wide[:, :20, 8:], x.detach().view(20, 3, 128).transpose(0, 1).contiguous().transpose(0, 1)):
        shape = view.shape[:-1]
        v3 = view.requires_grad_(True) if view.is_leaf else view.detach().requires_grad_(True)
        wt = w.detach().t().contiguous().t().requires_grad_(True)
        r = lambda a: a.view(shape)  # noqa: E731
        lp3 = fused_linear_log_probs(v3, wt, r(t).to(torch.int32))
        assert lp3.shape == shape and torch.equal(lp3.reshape(-1), lp)
        got = torch.autograd.grad(lp3, (v3, wt), r(up))
        pl3 = fused_linear_policy_loss(v3, wt, r(t), r(old).double(), r(adv))
        got = (*got, *torch.autograd.grad(pl3.loss, (v3, wt)))
        for a, b in zip(got, want):
            assert torch.equal(a.reshape(b.shape), b)
    for need in ((True, False), (False, True)):
        a, b = x.detach().clone().requires_grad_(need[0]), w.detach().clone().requires_grad_(need[1])
        leaf, i = (a, 0) if need[0] else (b, 1)
        assert torch.equal(torch.autograd.grad(fused_linear_log_probs(a, b, t), leaf, up)[0], want[i])
        assert torch.equal(torch.autograd.grad(fused_linear_policy_loss(a, b, t, old, adv).loss, leaf)[0], want[2 + i])


def test_small_coefficients_keep_their_precision_in_fp16():
    """A mean over many tokens: upstream gradients far below fp16's range, seen in an fp32 weight."""
    from bastile_b200.ops.fused_linear_policy_loss import fused_linear_log_probs

    x, w, t, up, _ = make(50, 64, 400, torch.float16, seed=5)
    w32 = w.float().requires_grad_(True)
    want = Oracle(x, w, t)
    (dw,) = torch.autograd.grad(fused_linear_log_probs(x, w32, t), w32, up * 1e-9)
    value, bound = want.grads(up.double() * 1e-9, torch.zeros_like(want.e), shifted=False)["dweight"]
    assert dw.dtype == torch.float32
    close(dw, value, bound - 2.0 ** -24, "dweight")  # without the allowance for an fp16 result


def test_gradient_against_differences():
    from bastile_b200.ops.fused_linear_policy_loss import fused_linear_policy_loss

    x, w, t, _, g = make(40, 64, 200, torch.float16, seed=6)
    o = Oracle(x, w, t)
    old, adv, ref = policy_inputs(o, g)
    want, *_ = policy_oracle(o, old, adv, ref, 0.2, 0.28, 0.1, None)
    bounds = o.grads(want["coef"], want["e_coef"], shifted=True)
    x.requires_grad_(True), w.requires_grad_(True)
    got = fused_linear_policy_loss(x, w, t, old, adv, ref, 0.2, 0.28, 0.1)
    grads = torch.autograd.grad(got.loss, (x, w))

    def loss(a, b):
        oo = Oracle(a, b, t)
        return policy_oracle(oo, old, adv, ref, 0.2, 0.28, 0.1, None)[0]["loss"]

    step = 1e-6
    for i, name in enumerate(("dhidden", "dweight")):
        way = torch.randn_like((x, w)[i].detach().double())
        args = [[x.detach().double(), w.detach().double()] for _ in range(2)]
        args[0][i] = args[0][i] + step * way
        args[1][i] = args[1][i] - step * way
        slope = (loss(*args[0]) - loss(*args[1])) / (2 * step)
        room = (bounds[name][1] * way.abs()).sum() + 1e-6 * (1 + slope.abs())
        assert (slope - (grads[i].double() * way).sum()).abs() <= room, name


def test_policy_loss_is_the_log_probs_loss():
    """The same loss written with fused_linear_log_probs and torch: same value, same gradients."""
    from bastile_b200.ops.fused_linear_policy_loss import fused_linear_log_probs, fused_linear_policy_loss

    x, w, t, _, g = make(200, 128, 900, torch.bfloat16, seed=7)
    o = Oracle(x, w, t)
    old, adv, ref = policy_inputs(o, g)
    x.requires_grad_(True), w.requires_grad_(True)
    pl = fused_linear_policy_loss(x, w, t, old, adv, ref, 0.2, 0.28, 0.05)
    lp = fused_linear_log_probs(x, w, t)
    assert torch.equal(lp, pl.log_probs)
    r, d = (lp - old).exp(), ref - lp
    terms = -torch.minimum(r * adv, r.clamp(0.8, 1.28) * adv) + 0.05 * (torch.expm1(d) - d)
    live = t != -100
    loss = terms[live].mean()
    assert abs(loss.item() - pl.loss.item()) <= 1e-5
    a, b = torch.autograd.grad(pl.loss, (x, w)), torch.autograd.grad(loss, (x, w))
    want, *_ = policy_oracle(o, old, adv, ref, 0.2, 0.28, 0.05, None)
    for name, p, q in zip(("dhidden", "dweight"), a, b):
        bound = o.grads(want["coef"], want["e_coef"], shifted=True)[name][1]
        assert ((p.double() - q.double()).abs() <= 2 * bound).all(), name


@pytest.mark.parametrize("cu", [[1, 8, 20], [0, 15, 8, 20], [0, 8, 21], [0, -3, 20], [0, 8, 1 << 40]])
def test_bad_offsets_and_targets_are_reported(cu):
    from bastile_b200 import _lib
    from bastile_b200.ops.fused_linear_policy_loss import fused_linear_log_probs, fused_linear_policy_loss

    x, w, t, up, _ = make(20, 64, 50, torch.bfloat16, seed=8)
    x.requires_grad_(True)
    old, adv = torch.zeros(20, device=DEV), torch.ones(20, device=DEV)
    got = fused_linear_policy_loss(x, w, t, old, adv, cu_seqlens=torch.tensor(cu, device=DEV))
    assert got.loss == 0 and (torch.autograd.grad(got.loss, x)[0] == 0).all()
    with pytest.raises(_lib.BastileB200Error, match="offsets"):
        _lib.check_all_status()
    want = fused_linear_log_probs(x, w, torch.where(torch.arange(20, device=DEV) == 4, -100, t))
    for bad in (50, -1, 1 << 40):
        t[4] = bad
        got = fused_linear_log_probs(x, w, t)
        assert torch.equal(got, want) and (torch.autograd.grad(got, x, up)[0][4] == 0).all()
        with pytest.raises(_lib.BastileB200Error, match="neither ignore_index"):
            _lib.check_all_status()


def test_captured_step_replays_and_two_streams():
    from bastile_b200.ops.fused_linear_policy_loss import fused_linear_log_probs, fused_linear_policy_loss

    x, w, t, up, g = make(150, 128, 600, torch.bfloat16, seed=9)
    o = Oracle(x, w, t)
    old, adv, ref = policy_inputs(o, g)
    x.requires_grad_(True), w.requires_grad_(True)

    def step(x, w):
        lp = fused_linear_log_probs(x, w, t, chunk_size=64)
        pl = fused_linear_policy_loss(x, w, t, old, adv, ref, kl_coef=0.1, chunk_size=64)
        return (lp.detach(), *torch.autograd.grad(lp, (x, w), up), pl.loss.detach(),
                *torch.autograd.grad(pl.loss, (x, w)))

    streams = [torch.cuda.Stream() for _ in range(2)]
    results = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            results.append(step(x, w))
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    for a, b in zip(*results):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = step(x, w)
    fresh = torch.randn_like(x)
    want = step(fresh.requires_grad_(True), w)
    with torch.no_grad():
        x.copy_(fresh)
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(res, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("switch,value", [("bt_set_gemm_cta_pairs", 0), ("bt_set_gemm_dynamic_tiles", 1),
                                          ("bt_set_gemm_tile_stores", 0), ("bt_set_dependent_launch", 0)])
def test_other_ways_to_run_the_products(switch, value):
    """The process-wide switches of the products: the contraction over the vocabulary in several runs
    (40 rows x 128 from 9000), several chunks, an odd vocabulary."""
    from bastile_b200 import _lib
    from bastile_b200.ops.fused_linear_policy_loss import fused_linear_log_probs, fused_linear_policy_loss

    lib = _lib.get_lib()
    assert lib.bt_dhidden_runs(40, 128, 9001, _lib.BT_BF16) > 1
    x, w, t, up, g = make(100, 128, 9001, torch.bfloat16, seed=10)
    o = Oracle(x, w, t)
    old, adv, ref = policy_inputs(o, g)
    want, *_ = policy_oracle(o, old, adv, ref, 0.2, 0.28, 0.1, None)
    x.requires_grad_(True), w.requires_grad_(True)
    prev = getattr(lib, switch)(value)
    try:
        lp = fused_linear_log_probs(x, w, t, chunk_size=40)
        a = torch.autograd.grad(lp, (x, w), up)
        pl = fused_linear_policy_loss(x, w, t, old, adv, ref, 0.2, 0.28, 0.1, chunk_size=40)
        b = torch.autograd.grad(pl.loss, (x, w))
        torch.cuda.synchronize()
    finally:
        getattr(lib, switch)(prev)
    close(lp.detach(), o.logp, o.e_logp, "logp")
    close(pl.loss.detach(), want["loss"], want["e_loss"], "loss")
    ref_a = o.grads(up.double(), torch.zeros_like(o.e), shifted=False)
    ref_b = o.grads(want["coef"], want["e_coef"], shifted=True)
    for i, name in enumerate(("dhidden", "dweight")):
        close(a[i], *ref_a[name], name)
        close(b[i], *ref_b[name], name)
    _lib.check_all_status()


def test_second_derivatives_are_refused():
    from bastile_b200.ops.fused_linear_policy_loss import fused_linear_log_probs

    x, w, t, up, _ = make(10, 64, 50, torch.bfloat16, seed=11)
    x.requires_grad_(True)
    (g,) = torch.autograd.grad(fused_linear_log_probs(x, w, t), x, up.requires_grad_(True), create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_log_probs_do_not_depend_on_the_rows_beside_them(dtype):
    """Few rows, and an odd number of 128-row tiles, take another tile shape than full pairs of them: the
    same sums in the same order, so that a policy's ratio to itself is 1 whatever it was batched with."""
    from bastile_b200.ops.fused_linear_policy_loss import fused_linear_log_probs, fused_linear_policy_loss

    x, w, t, _, _ = make(512, 264, 4099, dtype, seed=11)
    with torch.no_grad():
        full = fused_linear_log_probs(x, w, t)
        for n in (1, 61, 128, 129, 300):
            assert torch.equal(fused_linear_log_probs(x[:n], w, t[:n]), full[:n])
        pl = fused_linear_policy_loss(x, w, t, full, torch.ones_like(full), chunk_size=100)
        assert torch.equal(pl.log_probs, full) and pl.clip_fraction.item() == 0.0
