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

    err(lib.bt_logp_stats(None, one, one, None, one, one, 4, 64, 100, 64, 104, -100, b, None, None), b"null")
    err(lib.bt_logp_stats(one, one, one, one, one, one, 4, 64, 100, 64, 96, -100, b, None, None), b"stride")
    err(lib.bt_logp_stats(one, one, one, None, one, one, 4, 64, 100, 64, 104, -100, 7, None, None), b"dtype")
    err(lib.bt_logp_stats(one, one, one, None, one, one, 4, 0, 100, 64, 104, -100, b, None, None), b"extents")
    err(lib.bt_logp_rows(one, one, one, None, None, 4, 100, -100, None, None), b"null")
    err(lib.bt_logp_coef(one, one, 4, 100, -100, None, one, None), b"null")
    err(lib.bt_logp_dlogits(one, one, one, one, None, one, 4, 64, 100, 64, 104, b, None, None), b"null")
    err(lib.bt_logp_dlogits(one, one, one, one, one, one, 4, 64, 100, 64, 99, b, None, None), b"stride")
    err(lib.bt_logp_mask_rows(one, one, one, 4, 60, 60, 100, -100, b, None), b"aligned")
    err(lib.bt_policy_weights(one, 4, None, 2, 100, -100, one, one, None, None), b"sequence count")
    err(lib.bt_policy_weights(one, 4, one, 2, 100, -100, None, one, None, None), b"null")
    err(lib.bt_policy_rows(*[one] * 13, 4, 2, 5, 1, 100, -100, 0.2, 0.2, 0.0, None), b"outside")
    err(lib.bt_policy_rows(None, *[one] * 12, 4, 0, 5, 1, 100, -100, 0.2, 0.2, 0.0, None), b"null")
    err(lib.bt_policy_dlogits(one, one, one, one, one, 4, 101, 103, b, None), b"aligned")
    err(lib.bt_policy_reduce(None, 4, one, None), b"bad args")
    for rc in (lib.bt_logp_rows(None, None, None, None, None, 0, 100, -100, None, None),
               lib.bt_policy_dlogits(None, None, None, None, None, 0, 100, 104, b, None)):
        assert rc == 0  # no rows: nothing to do
