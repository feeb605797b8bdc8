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


def off(got, x):
    return float((got.double() - x).norm() / x.norm())


@pytest.mark.parametrize("size", [1.0, 1e-4, 2e-7])
@pytest.mark.parametrize("big", ["q", "k"])
def test_fp16_small_upstream_gradients_keep_their_digits(big, size):
    """Long rows (probabilities of 1 / 4000) and small upstream gradients: dS lies below fp16's normal range.
    dS and the result are rounded once each, by at most u / sqrt(3) in the mean square; what a result loses in
    its own subnormal steps comes on top.  (q or k are large so that dk or dq are not themselves subnormal.)"""
    n, d, factor = 4000, 64, 64.0
    q, k, v, cu, dout = inputs([n], 2, 1, d, torch.float16, seed=32, tail=7)
    q, k = (q * factor, k) if big == "q" else (q, k * factor)
    v, dout = v * (256.0 if size < 1e-5 else 8.0), (dout * size).half()
    dout[n:] = 3e4  # rows behind the last sequence have no say in the scale
    v[n:] = 6e4
    scale = d ** -0.5 / factor
    want = oracle(q, k, v, cu, scale, dout)
    got = attend(q, k, v, cu, dout, scale=scale)
    name = "dk" if big == "q" else "dq"
    x = want[name][0]
    own = 2.0 ** -24 / 12 ** 0.5 / float(x[:n].square().mean().sqrt())
    bar = 1.25 * (2 * (2.0 ** -11) ** 2 / 3 + own ** 2) ** 0.5
    assert off(got[name], x) <= bar, (off(got[name], x), bar, own)


def test_fp16_large_upstream_gradients():
    """dP far beyond 65504 times a small probability: dS once overflowed where the probability is not small."""
    q, k, v, cu, dout = inputs([300], 2, 1, 64, torch.float16, seed=33)
    v, dout = v * 64.0, dout * 512.0
    scale = 2.0 ** -12
    want = oracle(q, k, v, cu, scale, dout)
    got = attend(q, k, v, cu, dout, scale=scale)
    for n in ("dq", "dk"):
        bar = 1.25 * (2 * (2.0 ** -11) ** 2 / 3) ** 0.5
        assert torch.isfinite(got[n]).all() and off(got[n], want[n][0]) <= bar, n


def test_fp16_infinite_upstream_gradients_stay_where_they_are():
    q, k, v, cu, dout = inputs([100, 90], 2, 1, 64, torch.float16, seed=34)
    want = attend(q, k, v, cu, dout)
    dout[120] = float("inf")
    got = attend(q, k, v, cu, dout)
    for n in ("dq", "dk", "dv"):
        assert torch.equal(got[n][:100], want[n][:100]), n
        assert not torch.isfinite(got[n][100:]).all(), n


def test_fp16_gradients_scale_with_the_upstream_gradient():
    """A power of two on the upstream gradient: the same bits, scaled, while the results stay normal numbers."""
    q, k, v, cu, dout = inputs([130, 70], 4, 2, 64, torch.float16, seed=35)
    a, b = attend(q, k, v, cu, dout * 8.0), attend(q, k, v, cu, dout)
    for n in ("dq", "dk"):
        big = b[n].abs() >= 2.0 ** -14
        assert torch.equal(a[n][big], (b[n] * 8.0)[big]), n


def shifted(x, by=1):
    """The same values, dense, ``by`` elements off an aligned start."""
    buf = torch.empty(x.numel() + 8, dtype=x.dtype, device=x.device)
    y = buf[by:by + x.numel()].view(x.shape)
    y.copy_(x)
    assert y.is_contiguous() and y.data_ptr() % 16 != 0
    return y


def test_dense_tensors_off_a_16_byte_boundary():
    q, k, v, cu, dout = inputs([70, 130], 4, 2, 64, torch.bfloat16, seed=36)
    want = attend(q, k, v, cu, dout)
    got = attend(shifted(q), shifted(k, 3), shifted(v, 4), cu, shifted(dout, 7))
    for n in got:
        assert torch.equal(got[n], want[n]), n


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens,hq,hk,d", [
    ([500, 0, 130, 1, 60], 64, 32, 64), ([1100, 3, 97], 80, 16, 80), ([2000, 450], 32, 8, 128), ([257, 50], 128, 64, 8),
    ([128] * 3 + [20], 48, 48, 128), ([40] * 16, 64, 32, 72),
])
def test_the_kernel_of_ordinary_batches(lens, hq, hk, d, dtype):
    """A key tile per CTA, no clusters: what dK and dV take from 128 tokens times SMs over key/value heads on."""
    q, k, v, cu, dout = inputs(lens, hq, hk, d, dtype, seed=41, tail=5, fused=len(lens) % 2 == 0)
    assert q.shape[0] * hk >= 128 * torch.cuda.get_device_properties(0).multi_processor_count
    want = oracle(q, k, v, cu, d ** -0.5, dout)
    got = attend(q, k, v, cu, dout)
    for n in got:
        close(got[n], want[n], n)
        assert (got[n][cu[-1]:] == 0).all(), n
    again = attend(q, k, v, cu, dout)
    assert all(torch.equal(got[n], again[n]) for n in got)


def test_the_benchmarks_sequence():
    q, k, v, cu, dout = inputs([8192], 32, 8, 128, torch.bfloat16, seed=42)
    want = oracle(q, k, v, cu, 128 ** -0.5, dout)
    got = attend(q, k, v, cu, dout)
    for n in got:
        close(got[n], want[n], n)


def mean_square_errors(q, k, v, cu, scale, dout, u):
    """Per sequence: the 2-norms that dq's and dk's errors have in the mean, {(name, start): (with D from the
    unrounded output, with D from the rounded one)}.  Roundings are independent and at most u / sqrt(3) of their
    value in the mean square: of dS, of the result, and of P in the sum for the output, which moves D by
    P_ij dP_ij each; the output's own rounding moves it by dout_id out_id each."""
    q, k, v, dout = (x.double() for x in (q, k, v, dout))
    g, r2 = q.shape[1] // k.shape[1], u * u / 3
    res = {}
    for a, b in zip(cu[:-1], cu[1:]):
        mask = torch.ones(b - a, b - a, dtype=torch.bool, device=q.device).tril()
        sq = {(n, w): 0.0 for n in ("dq", "dk") for w in (0, 1)}
        dk = [0.0] * k.shape[1]
        for h in range(q.shape[1]):
            qh, kh, vh, do = q[a:b, h], k[a:b, h // g], v[a:b, h // g], dout[a:b, h]
            p = torch.softmax((qh @ kh.t() * scale).masked_fill(~mask, -torch.inf), -1)
            out, dp = p @ vh, do @ vh.t()
            ds = p * (dp - (do * out).sum(-1, keepdim=True))
            move = r2 * (p * dp).square().sum(-1)
            for w, d2 in enumerate((move, move + r2 * (do * out).square().sum(-1))):
                sq["dq", w] += scale ** 2 * (r2 * (ds.square() @ kh.square()).sum() + (d2[:, None] * (p @ kh).square()).sum())
                sq["dk", w] += scale ** 2 * (r2 * (ds.square().t() @ qh.square()).sum()
                                             + (p.square().t() @ (d2[:, None] * qh.square())).sum())
                sq["dq", w] += r2 * (ds @ kh * scale).square().sum()
            dk[h // g] = dk[h // g] + ds.t() @ qh * scale
        for n, w in sq:
            total = sq[n, w] + (r2 * sum(x.square().sum() for x in dk) if n == "dk" else 0.0)
            res.setdefault((n, a), []).append(float(total) ** 0.5)
    return res


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hk", [(4, 2), (1, 1)])
def test_the_outputs_rounding_does_not_reach_the_gradients(hq, hk, dtype):
    """Values far from zero that differ little: D = dout . out from the rounded output alone would be far off."""
    u = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[dtype]
    q, k, v, cu, dout = inputs([300, 77, 128], hq, hk, 64, dtype, seed=43)
    v = (8.0 + 0.25 * v.float()).to(dtype)
    want = oracle(q, k, v, cu, 0.125, dout)
    got = attend(q, k, v, cu, dout)
    for (n, a), (unrounded, rounded) in mean_square_errors(q, k, v, cu, 0.125, dout, u).items():
        b = cu[cu.index(a) + 1]
        error = float((got[n][a:b].double() - want[n][0][a:b]).norm())
        assert error <= 1.25 * unrounded, (n, a, error, unrounded, rounded)
        assert rounded >= 1.5 * unrounded  # so that the bar tells one from the other


@pytest.mark.parametrize("lens,hq,hk", [([600], 2, 1), ([600, 40], 64, 32)])
def test_fp16_keys_that_are_hardly_seen(lens, hq, hk):
    """The first key takes all but a millionth of every row: what dV of the others is formed from lies below fp16's
    normal range.  P and the result are rounded once each."""
    q, k, v, cu, dout = inputs(lens, hq, hk, 64, torch.float16, seed=44)
    dout = dout * 256.0
    q[..., 0], k[..., 0] = 4.0, 0.0
    for a in cu[:-1]:
        k[a, :, 0] = 8.0 * 15.0 / 4.0  # 15 above the others' scores: e^-15 = 2^-21.6
    want = oracle(q, k, v, cu, 0.125, dout)
    got = attend(q, k, v, cu, dout)
    bar = 1.25 * (2 * (2.0 ** -11) ** 2 / 3) ** 0.5
    others = torch.ones(cu[-1], dtype=torch.bool, device=DEV)
    others[cu[:-1]] = False
    x, y = got["dv"][others], want["dv"][0][others]
    own = 2.0 ** -24 / 12 ** 0.5 / float(y.square().mean().sqrt())
    assert off(x, y) <= bar + own, (off(x, y), bar, own)
    for n in got:
        close(got[n], want[n], n)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_two_captured_graphs_share_a_plan_and_replay_at_once(dtype):
    """A plan made outside the graphs, two graphs of a step each on two streams, replayed together."""
    from bastile_b200.ops.packed_attention import pack_sequences, packed_attention

    q, k, v, cu, dout = inputs([200, 101], 4, 2, 64, dtype, seed=45)
    sets = [(q, k, v, dout), (q * 0.5, k, v * 2.0, dout * 0.25)]
    want = [attend(*s[:3], cu, s[3]) for s in sets]
    seqs = pack_sequences(torch.tensor(cu, dtype=torch.int32, device=DEV), 301)
    graphs, results = [], []
    for a, b, c, g in sets:
        xs = [x.clone().requires_grad_(True) for x in (a, b, c)]

        def step():
            out = packed_attention(*xs, seqs)
            return (out.detach(), *torch.autograd.grad(out, xs, g))

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results.append(step())
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(3):
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for got, w in zip(results, want):
        for n, x in zip(("out", "dq", "dk", "dv"), got):
            assert torch.equal(x, w[n]), n


def test_two_backward_passes_of_one_graph():
    from bastile_b200.ops.packed_attention import pack_sequences, packed_attention

    q, k, v, cu, dout = inputs([90, 40], 4, 2, 64, torch.float16, seed=46)
    xs = [x.clone().requires_grad_(True) for x in (q, k, v)]
    out = packed_attention(*xs, pack_sequences(torch.tensor(cu, dtype=torch.int32, device=DEV), 130))
    for factor in (1.0, 2.0 ** -9, 16.0):  # another upstream gradient, another scale of dS
        want = attend(q, k, v, cu, dout * factor)
        for n, x in zip(("dq", "dk", "dv"), torch.autograd.grad(out, xs, dout * factor, retain_graph=True)):
            assert torch.equal(x, want[n]), n
