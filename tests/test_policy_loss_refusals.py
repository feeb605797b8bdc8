"""What the log-probability and policy-loss ops refuse, and their C entry points (no GPU needed)."""

import ctypes as C

import pytest
import torch


def _args(rows=4, h=64, v=100, dtype=torch.bfloat16):
    return torch.zeros(rows, h, dtype=dtype), torch.zeros(v, h, dtype=dtype), torch.zeros(rows, dtype=torch.int64)


def test_log_probs_refusals():
    from bastile_b200.ops.fused_linear_policy_loss import fused_linear_log_probs

    x, w, t = _args()
    for args, error, text in (((x.double(), w, t), TypeError, "dtype"), ((x, w[:, :32], t), ValueError, "vocab, hidden"),
                              ((x, w[0], t), ValueError, "vocab, hidden"), ((x, w, t[:3]), ValueError, "does not match"),
                              ((x, w, t.float()), TypeError, "token ids"), ((x, w, t.bool()), TypeError, "token ids"),
                              ((x[:, :60], w[:, :60], t), ValueError, "16-byte"), ((x, w[:0], t), ValueError, "16-byte"),
                              ((x, w, t), RuntimeError, "CUDA")):
        with pytest.raises(error, match=text):
            fused_linear_log_probs(*args)
    with pytest.raises(ValueError, match="chunk_size"):
        fused_linear_log_probs(x, w, t, chunk_size=0)


def test_policy_loss_refusals():
    from bastile_b200.ops.fused_linear_policy_loss import fused_linear_policy_loss

    x, w, t = _args()
    f = torch.zeros(4)
    cu = torch.zeros(2, dtype=torch.int32)
    for kw, error, text in ((dict(old_log_probs=f[:3]), ValueError, "old_log_probs"),
                            (dict(old_log_probs=t), ValueError, "old_log_probs"),
                            (dict(advantages=f[None]), ValueError, "advantages"),
                            (dict(ref_log_probs=f[:1]), ValueError, "ref_log_probs"),
                            (dict(kl_coef=0.1), ValueError, "needs ref"), (dict(kl_coef=float("nan")), ValueError, "finite"),
                            (dict(clip_low=-0.1), ValueError, "clip_low"), (dict(clip_low=1.5), ValueError, "clip_low"),
                            (dict(clip_high=float("inf")), ValueError, "clip_high"),
                            (dict(clip_high=float("nan")), ValueError, "clip_high"),
                            (dict(cu_seqlens=cu[:0]), ValueError, "cu_seqlens"),
                            (dict(cu_seqlens=cu.float()), TypeError, "cu_seqlens"), ({}, RuntimeError, "CUDA")):
        with pytest.raises(error, match=text):
            fused_linear_policy_loss(x, w, t, **{**dict(old_log_probs=f, advantages=f), **kw})


def test_c_entry_points():
    from bastile_b200 import _lib

    lib = _lib.get_lib()
    one = C.c_void_p(16)  # never dereferenced: validation fails before any launch
    b = _lib.BT_BF16

    def err(rc, text):
        assert rc == -1 and text in lib.bt_last_error(), lib.bt_last_error()

    def fwd(hidden=one, w=one, labels=one, logp=one, ws=one, rows=4, h=64, v=100, ld=64, chunk=4, dtype=b):
        return lib.bt_logp_fwd(hidden, w, labels, logp, None, ws, rows, h, v, ld, chunk, -100, dtype, None, None)

    err(fwd(hidden=None), b"null"), err(fwd(labels=None), b"null"), err(fwd(logp=None), b"null")
    err(fwd(dtype=7), b"dtype"), err(fwd(h=0), b"extents"), err(fwd(rows=-1), b"extents"), err(fwd(chunk=0), b"chunk")
    err(fwd(hidden=C.c_void_p(8)), b"aligned"), err(fwd(ld=60), b"aligned"), err(fwd(ld=56), b"aligned")
    assert fwd(rows=0, hidden=None, labels=None) == 0

    def bwd(dlogp=one, masked=one, parts=one, dw=one, acc=one, rows=4, chunk=4):
        return lib.bt_logp_bwd(dlogp, one, one, one, one, masked, one, one, parts, dw, acc, one, rows, 64, 100, 64, chunk,
                               -100, b, b, None, None)

    err(bwd(dlogp=None), b"null"), err(bwd(masked=None), b"null"), err(bwd(masked=C.c_void_p(24)), b"aligned")
    err(bwd(acc=None, chunk=2), b"accumulator")
    err(bwd(parts=None), b"parts")
    assert bwd(rows=0) == 0
    err(lib.bt_sum_runs(one, one, 6, 1, 6, one, b, None), b"sizes"), err(lib.bt_sum_runs(one, one, 8, 2, 4, one, b, None), b"sizes")
    err(lib.bt_sum_runs(one, None, 8, 1, 8, one, b, None), b"null"), err(lib.bt_sum_runs(one, one, 8, 1, 8, one, 5, None), b"dtype")
    assert lib.bt_dhidden_runs(517, 1024, 32000, b) > 1 and lib.bt_dhidden_runs(8192, 4096, 4096, b) == 1
    assert lib.bt_dhidden_runs(0, 64, 100, b) == 1

    def policy(**kw):
        d = _lib.PolicyDesc()
        for n, t in d._fields_:
            if t is C.c_void_p and n not in ("cu_seqlens", "ref_logp"):
                setattr(d, n, 16)
        d.rows, d.H, d.V, d.ld_hidden, d.chunk, d.n_seq, d.ignore_index, d.dtype = 4, 64, 100, 64, 4, 1, -100, b
        for n, x in kw.items():
            setattr(d, n, x)
        return lib.bt_policy_fwd(C.byref(d), None, None)

    err(lib.bt_policy_fwd(None, None, None), b"null descriptor")
    for kw, text in ((dict(hidden=None), b"null"), (dict(ws=None), b"null"), (dict(adv=None), b"null"),
                     (dict(masked=None), b"buffers"), (dict(logits=24), b"buffers"), (dict(n_seq=2), b"sequence count"),
                     (dict(n_seq=-1, cu_seqlens=16), b"sequence count"), (dict(dtype=9), b"dtype"),
                     (dict(chunk=2, want_dweight=1, dweight_acc=None), b"accumulator"), (dict(ld_hidden=8), b"aligned")):
        err(policy(**kw), text)
    assert lib.bt_logp_fwd_ws_floats(3, 100) == 3 * 2 * 2 + 3 and lib.bt_logp_fwd_ws_floats(-1, 100) == 0
    assert lib.bt_policy_fwd_ws_floats(5, 3, 2, 100) == 26 + 3 * 2 * 2 and lib.bt_policy_fwd_ws_floats(5, 3, 2, 0) == 0
