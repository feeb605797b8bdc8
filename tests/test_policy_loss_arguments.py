"""Coefficients of the policy loss that fp32 does not hold (no GPU needed)."""

import pytest
import torch


@pytest.mark.parametrize("kl_coef", [1e39, -1e300])
def test_kl_coefficients_beyond_fp32_are_refused(kl_coef):
    from bastile_b200.ops.fused_linear_policy_loss import fused_linear_policy_loss

    x, w, t, f = torch.zeros(4, 64), torch.zeros(100, 64), torch.zeros(4, dtype=torch.int64), torch.zeros(4)
    with pytest.raises(ValueError, match="kl_coef must be finite"):
        fused_linear_policy_loss(x, w, t, f, f, f, kl_coef=kl_coef)


def test_c_entry_point_with_several_chunks():
    import ctypes as C

    from bastile_b200 import _lib

    lib = _lib.get_lib()
    rows, chunk, h, v = 40, 20, 128, 9001
    assert lib.bt_dhidden_runs(chunk, h, v, _lib.BT_BF16) > 1

    def policy(**kw):
        d = _lib.PolicyDesc()
        for n, t in d._fields_:
            if t is C.c_void_p and n not in ("cu_seqlens", "ref_logp"):
                setattr(d, n, 16)  # never dereferenced: validation fails before any launch
        d.rows, d.H, d.V, d.ld_hidden, d.chunk, d.n_seq, d.ignore_index, d.dtype = rows, h, v, h, chunk, 1, -100, _lib.BT_BF16
        for n, x in kw.items():
            setattr(d, n, x)
        return lib.bt_policy_fwd(C.byref(d), None, None), lib.bt_last_error()

    for kw, text in ((dict(dhidden_parts=None), b"parts"), (dict(dhidden_parts=24), b"parts"), (dict(dhidden=20), b"parts"),
                     (dict(want_dweight=1, dweight_acc=20), b"accumulator")):
        rc, message = policy(**kw)
        assert rc == -1 and text in message, (kw, message)


def test_c_sizes_of_attention_scratch():
    from bastile_b200 import _lib

    lib = _lib.get_lib()
    assert lib.bt_attn_delta_floats(7, 3, _lib.BT_BF16) == 21
    assert lib.bt_attn_delta_floats(7, 3, _lib.BT_FP16) >= 22 + 2 * 148 and lib.bt_attn_delta_floats(-1, 3, 0) == 0


def test_c_entry_points_refuse_unaligned_statistics_and_missing_strides():
    import ctypes as C

    from bastile_b200 import _lib

    lib = _lib.get_lib()
    one, odd, b = C.c_void_p(16), C.c_void_p(20), _lib.BT_BF16  # never dereferenced

    rc = lib.bt_logp_fwd(one, one, one, one, None, odd, 4, 64, 100, 64, 4, -100, b, None, None)
    assert rc == -1 and b"8-byte" in lib.bt_last_error()
    d = _lib.PolicyDesc()
    for n, t in d._fields_:
        if t is C.c_void_p and n not in ("cu_seqlens", "ref_logp"):
            setattr(d, n, 16)
    d.rows, d.H, d.V, d.ld_hidden, d.chunk, d.n_seq, d.ignore_index, d.dtype, d.ws = 4, 64, 100, 64, 4, 1, -100, b, 20
    assert lib.bt_policy_fwd(C.byref(d), None, None) == -1 and b"8-byte" in lib.bt_last_error()
    st = _lib.I64x2(256, 64)
    rc = lib.bt_attn_fwd(one, one, one, one, None, None, one, 1, 4, 4, 2, 64, st, st, None, st, 0.1, b, None, None)
    assert rc == -1 and b"strides" in lib.bt_last_error()
    for missing in range(8):
        s = [st] * 8
        s[missing] = None
        rc = lib.bt_attn_bwd(one, one, one, one, one, None, one, one, one, one, one, one, 1, 4, 4, 2, 64, *s, 0.1, b, None, None)
        assert rc == -1 and b"strides" in lib.bt_last_error(), missing
