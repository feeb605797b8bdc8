"""Causal attention over packed sequences against a plain implementation in 64 bits.

The bounds follow the kernels' roundings.  With u = eps / 2 of the 16-bit type:
  out   P is rounded to 16 bits for the second product (u P|v|), the result once more (u |out|);
  dv    the same with P^T |dout|;
  dq/dk dS = P (dP - D) is rounded (u |dS|); D = dout . out uses the rounded out, which moves dS by
        P |dout| . (the error of out); then the result is rounded.
Scores, exponentials, statistics and sums are fp32: SLACK relative to the same sums of absolute
values covers them (products of 16-bit values summed over at most 128 terms, then exp2 of arguments
below 2^7 in magnitude with 24-bit rounding: below 2^-15)."""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
SLACK = 2.0 ** -14
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def oracle(q, k, v, cu, scale, dout=None):
    """fp64 results and elementwise error bounds: {name: (value, bound)}."""
    u = U[q.dtype]
    q, k, v = (x.detach().double() for x in (q, k, v))
    g = q.shape[1] // k.shape[1]
    res = {n: [torch.zeros_like(x), torch.zeros_like(x)] for n, x in (("out", q), ("dq", q), ("dk", k), ("dv", v))}
    for a, b in zip(cu[:-1], cu[1:]):
        n = b - a
        if n == 0:
            continue
        mask = torch.ones(n, n, dtype=torch.bool, device=q.device).tril()
        for h in range(q.shape[1]):
            qh, kh, vh = q[a:b, h], k[a:b, h // g], v[a:b, h // g]
            p = torch.softmax((qh @ kh.t() * scale).masked_fill(~mask, -torch.inf), -1)
            out = p @ vh
            e_out = (u + SLACK) * (p @ vh.abs()) + u * out.abs()
            res["out"][0][a:b, h], res["out"][1][a:b, h] = out, e_out
            if dout is None:
                continue
            do = dout[a:b, h].double()
            res["dv"][0][a:b, h // g] += p.t() @ do
            res["dv"][1][a:b, h // g] += (u + SLACK) * (p.t() @ do.abs())
            dp, dd = do @ vh.t(), (do * out).sum(-1, keepdim=True)
            ds = p * (dp - dd)
            room = do.abs() @ vh.abs().t() + (do.abs() * out.abs()).sum(-1, keepdim=True)
            e_ds = u * ds.abs() + p * ((do.abs() * e_out).sum(-1, keepdim=True) + SLACK * room)
            res["dq"][0][a:b, h] = ds @ kh * scale
            res["dq"][1][a:b, h] = (e_ds + SLACK * ds.abs()) @ kh.abs() * scale
            res["dk"][0][a:b, h // g] += ds.t() @ qh * scale
            res["dk"][1][a:b, h // g] += (e_ds + SLACK * ds.abs()).t() @ qh.abs() * scale
    tiny = torch.finfo(torch.float16).smallest_normal * 2.0 ** -10 if u == U[torch.float16] else 0.0
    for n in ("dq", "dk", "dv"):
        res[n][1] = res[n][1] + u * res[n][0].abs()
    # fp16 below its normal range is spaced 2^-24 apart (half a step for each of the summed terms)
    return {n: (x, 1.01 * e + tiny * (1 + q.shape[0])) for n, (x, e) in res.items()}


def inputs(lens, hq, hk, d, dtype, seed=0, tail=0, fused=False):
    g = torch.Generator(device=DEV).manual_seed(seed)
    t = sum(lens) + tail
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    x = torch.randn(t, hq + 2 * hk, d, generator=g, device=DEV)
    x[:, :hq] *= 1.5
    x = x.to(dtype)
    q, k, v = x[:, :hq], x[:, hq:hq + hk], x[:, hq + hk:]
    if not fused:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    dout = torch.randn(t, hq, d, generator=g, device=DEV).to(dtype)
    return q, k, v, cu, dout


def close(got, want, what):
    value, bound = want
    assert got.shape == value.shape, what
    off = (got.double() - value).abs()
    assert torch.isfinite(got).all(), f"{what}: not finite"
    worst = (off - bound).max() if off.numel() else torch.tensor(0.0)
    assert worst <= 0, f"{what}: {int((off > bound).sum())} of {off.numel()} outside, worst by {float(worst):.3e}"


def attend(q, k, v, cu, dout=None, scale=None, total=None):
    from bastile_b200 import _lib
    from bastile_b200.ops.packed_attention import pack_sequences, packed_attention

    seqs = pack_sequences(torch.tensor(cu, dtype=torch.int32, device=DEV), q.shape[0] if total is None else total)
    if dout is None:
        with torch.no_grad():
            got = {"out": packed_attention(q, k, v, seqs, scale)}
    else:
        q, k, v = (x.detach().requires_grad_(True) for x in (q, k, v))
        out = packed_attention(q, k, v, seqs, scale)
        dq, dk, dv = torch.autograd.grad(out, (q, k, v), dout)
        got = {"out": out.detach(), "dq": dq, "dk": dk, "dv": dv}
    _lib.check_all_status()
    return got


HEADS = [(1, 1, 128), (2, 1, 64), (4, 2, 128), (5, 1, 80), (8, 8, 8), (6, 2, 72), (8, 1, 128), (32, 1, 64)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hk,d", HEADS)
@pytest.mark.parametrize("lens", [[1], [128], [129], [7, 0, 1, 250, 0, 33], [300, 64], [127, 1, 128, 257]])
def test_forward_and_gradients(lens, hq, hk, d, dtype):
    q, k, v, cu, dout = inputs(lens, hq, hk, d, dtype, seed=len(lens) + d, tail=3 if len(lens) > 2 else 0,
                               fused=len(lens) % 2 == 0)
    want = oracle(q, k, v, cu, d ** -0.5, dout)
    got = attend(q, k, v, cu, dout)
    for n in ("out", "dq", "dk", "dv"):
        close(got[n], want[n], n)
        assert (got[n][cu[-1]:] == 0).all(), f"{n}: rows behind the last sequence"
    assert torch.equal(attend(q, k, v, cu)["out"], got["out"])  # inference gives training's bits


@pytest.mark.parametrize("lens,hq,hk,d", [([2100], 4, 1, 128), ([900, 1500, 40], 2, 2, 64), ([5] * 150, 4, 2, 64)])
def test_long_and_many(lens, hq, hk, d):
    q, k, v, cu, dout = inputs(lens, hq, hk, d, torch.bfloat16, seed=3)
    want = oracle(q, k, v, cu, 0.3, dout)
    got = attend(q, k, v, cu, dout, scale=0.3)
    for n in got:
        close(got[n], want[n], n)


@pytest.mark.parametrize("lens,hq,hk,d", [([500, 30, 11], 64, 16, 64), ([100] * 4, 80, 40, 64),
                                           ([700, 100], 64, 64, 72)])
def test_key_tiles_of_one_cta_or_two(lens, hq, hk, d):
    """dK and dV of the longest sequence's key tiles by two CTAs each while an even deal would take half their
    time, by one each with sequences of one length or more heads."""
    q, k, v, cu, dout = inputs(lens, hq, hk, d, torch.bfloat16, seed=6, tail=5)
    want = oracle(q, k, v, cu, d ** -0.5, dout)
    got = attend(q, k, v, cu, dout)
    for n in got:
        close(got[n], want[n], n)
    again = attend(q, k, v, cu, dout)
    assert all(torch.equal(got[n], again[n]) for n in got)


def test_more_sequences_than_are_sorted():
    lens = [(i * 7) % 5 for i in range(1500)]
    q, k, v, cu, dout = inputs(lens, 2, 1, 64, torch.float16, seed=4, tail=11)
    want = oracle(q, k, v, cu, 0.125, dout)
    got = attend(q, k, v, cu, dout)
    for n in got:
        close(got[n], want[n], n)


def test_growing_scores_rescale_the_accumulator():
    """Scores that rise along the keys make the running maximum move in every block."""
    q, k, v, cu, dout = inputs([700], 2, 1, 64, torch.bfloat16, seed=5)
    q = torch.ones_like(q)
    k = (torch.arange(700, device=DEV)[:, None, None] / 64.0).expand(700, 1, 64).to(torch.bfloat16).contiguous()
    want = oracle(q, k, v, cu, 1.0, dout)
    got = attend(q, k, v, cu, dout, scale=1.0)
    # scores reach 700 here instead of 2^7: their fp32 rounding is 2^-24 * 700 * log2(e), below 2^-13.9
    for n in got:
        value, bound = want[n]
        close(got[n], (value, bound * (1 + 2.0 ** -13 / U[torch.bfloat16])), n)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_rows_of_others_do_not_leak(bad):
    """What stands behind a sequence - another sequence, or unused rows - is masked, whatever it holds."""
    lens, tail = [150, 60, 90], 40
    q, k, v, cu, dout = inputs(lens, 4, 2, 64, torch.bfloat16, seed=6, tail=tail)
    want = oracle(q, k, v, cu, 0.125, dout)
    for x in (q, k, v, dout):
        x[150:210] = bad
        x[300:] = bad
    got = attend(q, k, v, cu, dout)
    for n in got:
        for a, b in ((0, 150), (210, 300)):
            close(got[n][a:b], (want[n][0][a:b], want[n][1][a:b]), n)
        assert (got[n][300:] == 0).all()


def test_memory_layouts():
    lens = [70, 130]
    q, k, v, cu, dout = inputs(lens, 4, 2, 64, torch.float16, seed=7)
    want = attend(q, k, v, cu, dout)
    t = sum(lens)
    by_head = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v, dout)]  # [heads, tokens, d] storage
    wide = [torch.randn(t, x.shape[1], 96, device=DEV).to(x.dtype) for x in (q, k, v, dout)]
    for w, x in zip(wide, (q, k, v, dout)):
        w[..., 8:72] = x
    odd = [torch.randn(t, x.shape[1], 67, device=DEV).to(x.dtype) for x in (q, k, v, dout)]
    for w, x in zip(odd, (q, k, v, dout)):
        w[..., 3:67] = x
    last = [x.permute(2, 0, 1).contiguous().permute(1, 2, 0) for x in (q, k, v, dout)]
    for views in (by_head, [w[..., 8:72] for w in wide], [w[..., 3:67] for w in odd], last,
                  [q, k, v, dout[:1, :1, :1].expand_as(dout)]):
        ref = want if views[3].stride(0) else attend(q, k, v, cu, views[3].contiguous())
        got = attend(*views[:3], cu, views[3])
        for n in got:
            assert torch.equal(got[n], ref[n]), n


def test_element_offsets_beyond_32_bits():
    t, step = 600, 1 << 22  # 600 * 2^22 elements between the first and the last token
    buf = torch.empty(t * step, dtype=torch.bfloat16, device=DEV)
    q, k, v, cu, dout = inputs([590], 2, 1, 64, torch.bfloat16, seed=8, tail=10)
    want = attend(q, k, v, cu, dout)
    far = []
    for i, x in enumerate((q, k, v, dout)):
        w = torch.as_strided(buf, x.shape, (step, 64, 1), storage_offset=i * 256)
        w.copy_(x)
        far.append(w)
    got = attend(*far[:3], cu, far[3])
    for n in got:
        assert torch.equal(got[n], want[n]), n


def test_gradient_against_differences():
    q, k, v, cu, dout = inputs([45, 3], 2, 1, 64, torch.float16, seed=9)
    got = attend(q, k, v, cu, dout)
    want = oracle(q, k, v, cu, 0.125, dout)

    def loss(qq, kk, vv):
        total = 0.0
        for a, b in zip(cu[:-1], cu[1:]):
            for h in range(2):
                s = (qq[a:b, h] @ kk[a:b, 0].t() * 0.125).masked_fill(
                    ~torch.ones(b - a, b - a, dtype=torch.bool, device=DEV).tril(), -torch.inf)
                total = total + (torch.softmax(s, -1) @ vv[a:b, 0] * dout[a:b, h].double()).sum()
        return total

    xs = [x.double() for x in (q, k, v)]
    step = 1e-5
    for i, n in enumerate(("dq", "dk", "dv")):
        way = torch.randn_like(xs[i])
        up, down = list(xs), list(xs)
        up[i], down[i] = xs[i] + step * way, xs[i] - step * way
        slope = (loss(*up) - loss(*down)) / (2 * step)
        # third derivatives of a softmax of these scores are below 10^3 per unit step along `way`
        room = (want[n][1] * way.abs()).sum() + 1e-10 * 1e3 * way.abs().sum() + 1e-6
        assert (slope - (got[n].double() * way).sum()).abs() <= room, n


def test_partial_gradients():
    from bastile_b200.ops.packed_attention import pack_sequences, packed_attention

    q, k, v, cu, dout = inputs([90, 40], 4, 2, 64, torch.bfloat16, seed=10)
    want = attend(q, k, v, cu, dout)
    seqs = pack_sequences(torch.tensor(cu, dtype=torch.int64, device=DEV), 130)
    for names in (["q"], ["k"], ["v"], ["q", "v"]):
        xs = dict(q=q.detach(), k=k.detach(), v=v.detach())
        for n in names:
            xs[n] = xs[n].clone().requires_grad_(True)
        out = packed_attention(xs["q"], xs["k"], xs["v"], seqs)
        for n, g in zip(names, torch.autograd.grad(out, [xs[n] for n in names], dout)):
            assert torch.equal(g, want["d" + n])


def test_same_bits_every_time_and_on_another_stream():
    from bastile_b200.ops.packed_attention import pack_sequences, packed_attention

    q, k, v, cu, dout = inputs([400, 3, 260], 8, 2, 128, torch.bfloat16, seed=11)
    want = attend(q, k, v, cu, dout)
    seqs = pack_sequences(torch.tensor(cu, dtype=torch.int32, device=DEV), 663)
    results = []
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:  # two calls at once, one plan
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            xs = [x.detach().clone().requires_grad_(True) for x in (q, k, v)]
            out = packed_attention(*xs, seqs)
            results.append((out.detach(), *torch.autograd.grad(out, xs, dout)))
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    for r in results:
        for n, x in zip(("out", "dq", "dk", "dv"), r):
            assert torch.equal(x, want[n]), n


def test_captured_step_replays_on_new_data():
    """Plan, forward and backward in one CUDA graph: a replay takes new values AND new lengths."""
    from bastile_b200.ops.packed_attention import pack_sequences, packed_attention

    q, k, v, cu, dout = inputs([200, 101], 4, 2, 64, torch.bfloat16, seed=12)
    offsets = torch.tensor(cu, dtype=torch.int32, device=DEV)
    xs = [x.clone().requires_grad_(True) for x in (q, k, v)]

    def step():
        out = packed_attention(*xs, pack_sequences(offsets, 301))
        return (out.detach(), *torch.autograd.grad(out, xs, dout))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = step()
    q2, k2, v2, cu2, _ = inputs([57, 210], 4, 2, 64, torch.bfloat16, seed=13, tail=34)
    want = attend(q2, k2, v2, [0, 57, 267], dout)
    with torch.no_grad():
        for x, y in zip(xs, (q2, k2, v2)):
            x.copy_(y)
    offsets.copy_(torch.tensor([0, 57, 267], dtype=torch.int32))
    graph.replay()
    torch.cuda.synchronize()
    for n, x in zip(("out", "dq", "dk", "dv"), res):
        assert torch.equal(x, want[n]), n


@pytest.mark.parametrize("cu", [[1, 20, 40], [0, 30, 20, 40], [0, 20, 41], [0, -4, 40], [0, 20, 1 << 33]])
def test_bad_offsets_are_reported_and_give_zeros(cu):
    from bastile_b200 import _lib
    from bastile_b200.ops.packed_attention import pack_sequences, packed_attention

    q, k, v, _, dout = inputs([40], 4, 2, 64, torch.bfloat16, seed=14)
    seqs = pack_sequences(torch.tensor(cu, dtype=torch.int64, device=DEV), 40)
    with pytest.raises(_lib.BastileB200Error, match="offsets"):
        _lib.check_all_status()
    xs = [x.detach().requires_grad_(True) for x in (q, k, v)]
    out = packed_attention(*xs, seqs)
    for x in (out, *torch.autograd.grad(out, xs, dout)):
        assert (x == 0).all()
    _lib.check_all_status()


def test_no_tokens_and_no_sequences():
    from bastile_b200.ops.packed_attention import pack_sequences, packed_attention

    for t, cu in ((0, [0]), (0, [0, 0, 0]), (5, [0]), (5, [0, 0])):
        seqs = pack_sequences(torch.tensor(cu, dtype=torch.int32, device=DEV), t)
        xs = [torch.randn(t, h, 64, device=DEV).to(torch.bfloat16).requires_grad_(True) for h in (4, 2, 2)]
        out = packed_attention(*xs, seqs)
        assert out.shape == (t, 4, 64) and (out == 0).all()
        for x, g in zip(xs, torch.autograd.grad(out, xs, torch.ones_like(out))):
            assert g.shape == x.shape and (g == 0).all()
