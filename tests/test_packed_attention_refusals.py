"""What packed attention refuses, and the argument checks of its C entry points (no GPU needed)."""

import ctypes as C

import pytest
import torch


def _seqs(t):
    from bastile_b200.ops.packed_attention import PackedSequences

    return PackedSequences(torch.zeros(16, dtype=torch.int32), 1, t)


def _qkv(t=4, hq=4, hk=2, d=64, dtype=torch.bfloat16):
    return (torch.zeros(t, hq, d, dtype=dtype), torch.zeros(t, hk, d, dtype=dtype), torch.zeros(t, hk, d, dtype=dtype))


@pytest.mark.parametrize("change,error,text", [
    (dict(d=12), ValueError, "multiple of 8"), (dict(d=136), ValueError, "up to 128"), (dict(d=0), ValueError, "head_dim"),
    (dict(hq=3), ValueError, "multiple of 2"), (dict(hk=0), ValueError, "multiple"),
    (dict(dtype=torch.float32), TypeError, "bf16 or fp16"), (dict(t=5), ValueError, "4"),
])
def test_bad_tensors(change, error, text):
    from bastile_b200.ops.packed_attention import packed_attention

    with pytest.raises(error, match=text):
        packed_attention(*_qkv(**change), _seqs(4))


def test_mismatched_tensors_and_plans():
    from bastile_b200.ops.packed_attention import pack_sequences, packed_attention

    q, k, v = _qkv()
    with pytest.raises(TypeError, match="pack_sequences"):
        packed_attention(q, k, v, torch.tensor([0, 4], dtype=torch.int32))
    with pytest.raises(ValueError, match="disagree"):
        packed_attention(q, k, v[:3], _seqs(4))
    with pytest.raises(ValueError, match="heads, head_dim"):
        packed_attention(q[0], k, v, _seqs(4))
    with pytest.raises(TypeError, match="share"):
        packed_attention(q, k.half(), v, _seqs(4))
    for scale in (-0.1, 0.0, float("inf"), float("nan")):
        with pytest.raises(ValueError, match="scale"):
            packed_attention(q, k, v, _seqs(4), scale=scale)
    with pytest.raises(RuntimeError, match="CUDA"):
        packed_attention(q, k, v, _seqs(4))
    with pytest.raises(ValueError, match="batch"):
        pack_sequences(torch.zeros(2, 2, dtype=torch.int32), 4)
    with pytest.raises(ValueError, match="batch"):
        pack_sequences(torch.zeros(0, dtype=torch.int32), 4)
    with pytest.raises(TypeError, match="int32 or int64"):
        pack_sequences(torch.zeros(2), 4)
    with pytest.raises(ValueError, match="total_tokens"):
        pack_sequences(torch.zeros(2, dtype=torch.int32), 1 << 30)
    with pytest.raises(RuntimeError, match="CUDA"):
        pack_sequences(torch.zeros(2, dtype=torch.int32), 4)


def test_c_entry_points():
    from bastile_b200 import _lib

    lib = _lib.get_lib()
    one = C.c_void_p(16)  # never dereferenced: validation fails before any launch
    good, bad = _lib.I64x2(256, 64), _lib.I64x2(250, 64)

    def fwd(q=one, batch=1, total=4, hq=4, hk=2, d=64, qs=good, dtype=_lib.BT_BF16, plan=one, scale=0.1):
        return lib.bt_attn_fwd(q, one, one, one, None, None, plan, batch, total, hq, hk, d, qs, good, good, good, scale,
                               dtype, None, None)

    for kw, text in ((dict(q=None), b"null"), (dict(plan=None), b"null plan"), (dict(hq=3), b"multiple"),
                     (dict(d=68), b"head_dim"), (dict(d=256), b"head_dim"), (dict(dtype=_lib.BT_FP32), b"dtype"),
                     (dict(qs=bad), b"strides"), (dict(q=C.c_void_p(8)), b"aligned"), (dict(total=0), b"token count"),
                     (dict(total=1 << 30), b"token count"), (dict(batch=-1), b"batch"), (dict(scale=-1.0), b"scale"),
                     (dict(scale=0.0), b"scale"), (dict(scale=float("nan")), b"scale")):
        assert fwd(**kw) == -1 and text in lib.bt_last_error(), (kw, lib.bt_last_error())

    def bwd(dk=one, dv=one, lse=one):
        return lib.bt_attn_bwd(one, one, one, one, one, None, lse, one, one, dk, dv, one, 1, 4, 4, 2, 64, good, good, good,
                               good, good, good, good, bad, 0.1, _lib.BT_BF16, None, None)

    assert bwd(lse=None) == -1 and b"null" in lib.bt_last_error()
    assert bwd(dv=None) == -1 and b"together" in lib.bt_last_error()
    assert bwd() == -1 and b"dv" in lib.bt_last_error()
    assert lib.bt_attn_plan(None, 1, 4, one, None, None) == -1 and b"null" in lib.bt_last_error()
    assert lib.bt_attn_plan(one, -1, 4, one, None, None) == -1
    assert lib.bt_attn_plan_words(-1) == 0 and lib.bt_attn_plan_words(3) == 4 * 2 + 5 * 5 + 2
