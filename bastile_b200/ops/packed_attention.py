"""Causal attention over packed sequences with grouped heads, on the sm_100a kernels.

The reference leaves attention to torch (its patches stop at q/k-norm + RoPE); here the op stands
between ``qk_norm_rope`` and ``o_proj``.  A batch of sequences of different lengths lies one behind
the other along the token axis, without padding, and ``pack_sequences`` turns their offsets into
what the kernels need, on the device and without a host synchronisation.
"""

from __future__ import annotations

import inspect

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from .. import _lib

_DTYPES = (torch.bfloat16, torch.float16)
MAX_HEAD_DIM = 128


class PackedSequences:
    """The layout of one packed batch (made by ``pack_sequences``): usable by any number of
    attention calls, forward and backward, on any stream on work ordered behind its creation; it may be
    dropped as soon as the calls have been made."""

    __slots__ = ("plan", "batch", "total_tokens", "device", "stream")

    def __init__(self, plan: Tensor, batch: int, total_tokens: int):
        self.plan, self.batch, self.total_tokens, self.device = plan, batch, total_tokens, plan.device
        self.stream = _lib.stream_ptr(plan.device) if plan.is_cuda else None

    def keep_for(self, dev: torch.device) -> None:
        """The plan's memory belongs to the stream that made it: not given to its next user before the work
        that other streams have queued is done (kernels take addresses from it)."""
        if _lib.stream_ptr(dev) != self.stream:
            self.plan.record_stream(torch.cuda.current_stream(dev))


def pack_sequences(cu_seqlens: Tensor, total_tokens: int) -> PackedSequences:
    """``cu_seqlens`` [batch + 1] (int32 or int64, on the GPU): sequence ``b`` is tokens
    ``cu_seqlens[b] .. cu_seqlens[b + 1]`` of ``total_tokens``; the first offset is 0, sequences may be
    empty, tokens behind the last one belong to no sequence.  Offsets that start elsewhere, fall or
    run past ``total_tokens`` are noticed on the device: attention then gives zeros, and
    ``bastile_b200._lib.check_all_status()`` raises."""
    if cu_seqlens.dim() != 1 or cu_seqlens.numel() < 1:
        raise ValueError(f"pack_sequences: cu_seqlens must be [batch + 1], got {tuple(cu_seqlens.shape)}")
    if cu_seqlens.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"pack_sequences: cu_seqlens must be int32 or int64, got {cu_seqlens.dtype}")
    total_tokens = int(total_tokens)
    if not 0 <= total_tokens < 1 << 30:
        raise ValueError(f"pack_sequences: total_tokens must be in [0, 2^30), got {total_tokens}")
    dev = _lib.require_cuda(cu_seqlens)
    lib = _lib.get_lib()
    if cu_seqlens.dtype == torch.int64:
        # an offset that does not fit 32 bits is past the tokens in either type
        cu_seqlens = cu_seqlens.clamp(-1, 1 << 30).to(torch.int32)
    cu = cu_seqlens.contiguous()
    batch = cu.numel() - 1
    with _lib.device_of(dev), _lib.timed("attn_plan", 1, dev):
        plan = torch.empty(int(lib.bt_attn_plan_words(batch)), dtype=torch.int32, device=dev)
        rc = lib.bt_attn_plan(cu.data_ptr(), batch, total_tokens, plan.data_ptr(), _lib.status_word(dev).data_ptr(),
                              _lib.stream_ptr(dev))
    _lib.check(rc, "bt_attn_plan")
    return PackedSequences(plan, batch, total_tokens)


def _strides(t: Tensor):
    return _lib.I64x2(*t.stride()[:2])


def _rows(t: Tensor) -> Tensor:
    """``t`` if the kernels can read it where it lies (unit stride along the head, 16-byte rows), else a copy."""
    (n, heads, _), (st, sh, sd) = t.shape, t.stride()
    if sd == 1 and (n <= 1 or (st > 0 and st % 8 == 0)) and (heads <= 1 or (sh > 0 and sh % 8 == 0)) \
            and t.data_ptr() % 16 == 0:
        return t
    c = t.contiguous()
    return c if c.data_ptr() % 16 == 0 else c.clone()  # (dense rows off a 16-byte boundary are returned as they are)


def _forward(q, k, v, sequences, scale, keep: bool):
    """(out, what the backward needs if ``keep``)."""
    lib = _lib.get_lib()
    dev = q.device
    t, hq, d = q.shape
    q, k, v = _rows(q), _rows(k), _rows(v)
    out = torch.empty((t, hq, d), dtype=q.dtype, device=dev)
    lse2 = torch.empty((hq, t), dtype=torch.float32, device=dev) if keep else None
    lo = torch.empty_like(out) if keep else None  # what rounding cut off: dout . out is formed from both
    if t > 0:
        st = _lib.status_word(dev)
        sequences.keep_for(dev)  # (the backward runs on this stream too)
        with _lib.device_of(dev), _lib.timed("attn_fwd", 1, dev):
            rc = lib.bt_attn_fwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
                                 lo.data_ptr() if keep else None, lse2.data_ptr() if keep else None,
                                 sequences.plan.data_ptr(), sequences.batch, t, hq, k.shape[1], d, _strides(q), _strides(k), _strides(v), _strides(out), scale,
                                 _lib.dtype_code(q.dtype), st.data_ptr(), _lib.stream_ptr(dev))
        _lib.check(rc, "bt_attn_fwd")
    return out, (q, k, v, out, lo, lse2, sequences.plan)


class PackedAttentionFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, sequences, scale):
        out, saved = _forward(q, k, v, sequences, scale, True)
        ctx.save_for_backward(*saved)
        ctx.meta = (sequences.batch, scale)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, out, lo, lse2, plan = ctx.saved_tensors
        batch, scale = ctx.meta
        dev = q.device
        lib = _lib.get_lib()
        t, hq, d = q.shape
        hk = k.shape[1]
        dout = _rows(dout if dout.dtype == q.dtype else dout.to(q.dtype))
        need_q, need_kv = ctx.needs_input_grad[0], ctx.needs_input_grad[1] or ctx.needs_input_grad[2]
        dq = torch.empty((t, hq, d), dtype=q.dtype, device=dev) if need_q else None
        dk = torch.empty((t, hk, d), dtype=q.dtype, device=dev) if need_kv else None
        dv = torch.empty((t, hk, d), dtype=q.dtype, device=dev) if need_kv else None
        if q.numel() > 0:
            code = _lib.dtype_code(q.dtype)
            delta = torch.empty(int(lib.bt_attn_delta_floats(t, hq, code)), dtype=torch.float32, device=dev)
            st = _lib.status_word(dev)
            none = _lib.I64x2(0, 0)
            with _lib.device_of(dev), _lib.timed("attn_bwd", 1 + int(need_q) + int(need_kv), dev):
                rc = lib.bt_attn_bwd(dout.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
                                     lo.data_ptr(), lse2.data_ptr(), delta.data_ptr(),
                                     dq.data_ptr() if need_q else None, dk.data_ptr() if need_kv else None, dv.data_ptr() if need_kv else None,
                                     plan.data_ptr(), batch, t, hq, hk, d, _strides(dout), _strides(q), _strides(k),
                                     _strides(v), _strides(out), _strides(dq) if need_q else none,
                                     _strides(dk) if need_kv else none, _strides(dv) if need_kv else none, scale,
                                     code, st.data_ptr(), _lib.stream_ptr(dev))
            _lib.check(rc, "bt_attn_bwd")
        return dq, dk, dv, None, None


def packed_attention(q: Tensor, k: Tensor, v: Tensor, sequences: PackedSequences, scale: float | None = None) -> Tensor:
    """``out[t, h] = sum_s softmax_s(scale * q[t, h] . k[s, h // group]) v[s, h // group]`` over the tokens
    ``s <= t`` of ``t``'s own sequence; q [tokens, Hq, D], k and v [tokens, Hk, D] with Hq a multiple of Hk
    and D a multiple of 8 up to 128, bf16 or fp16 (scores, softmax statistics and sums are fp32).
    Strided views are read where they lie as long as heads are contiguous and 16-byte aligned.  Rows
    behind the last sequence are zeros and get zero gradients.  ``scale`` defaults to ``D ** -0.5``."""
    if not isinstance(sequences, PackedSequences):
        raise TypeError("packed_attention: sequences must come from pack_sequences()")
    if q.dim() != 3 or k.dim() != 3 or v.dim() != 3:
        raise ValueError("packed_attention: q, k and v must be [tokens, heads, head_dim]")
    t, hq, d = q.shape
    if k.shape != v.shape or k.shape[0] != t or k.shape[2] != d:
        raise ValueError(f"packed_attention: q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} disagree")
    if k.shape[1] < 1 or hq % k.shape[1] != 0 or hq < 1:
        raise ValueError(f"packed_attention: {hq} query heads are not a multiple of {k.shape[1]} key/value heads")
    if d < 8 or d % 8 != 0 or d > MAX_HEAD_DIM:
        raise ValueError(f"packed_attention: head_dim must be a multiple of 8 up to {MAX_HEAD_DIM}, got {d}")
    if q.dtype not in _DTYPES or k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError(f"packed_attention: q, k and v must share bf16 or fp16, got {q.dtype}, {k.dtype}, {v.dtype}")
    if t != sequences.total_tokens:
        raise ValueError(f"packed_attention: q has {t} tokens, the packed sequences {sequences.total_tokens}")
    scale = d ** -0.5 if scale is None else float(scale)
    if not 1e-30 <= scale <= 1e30:
        raise ValueError(f"packed_attention: scale must be between 1e-30 and 1e30, got {scale}")
    _lib.require_cuda(q, k, v, sequences.plan)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return PackedAttentionFunction.apply(q, k, v, sequences, scale)
    return _forward(q, k, v, sequences, scale, False)[0]


# ------------------------------------------------------------------ as an attention of HF transformers
#: ``attn_implementation`` under which ``apply(packed_attention=True)`` makes the op known to transformers.
HF_NAME = "bastile_packed"


def _padded_offsets(mask: Tensor) -> Tensor:
    """Offsets of a padded batch: every row of the [B, T] mask is up to three sequences, the padding in
    front, the tokens, the padding behind (each attends to itself only).  Tokens that are not one run
    are reported like bad offsets."""
    b, t = mask.shape
    m = mask != 0
    lead = m.to(torch.int32).argmax(dim=1)
    count = m.sum(dim=1)
    lead = torch.where(count > 0, lead, torch.zeros_like(lead))
    start = torch.arange(b, device=mask.device) * t
    cu = torch.stack((start, start + lead, start + lead + count), dim=1).reshape(-1)
    pos = torch.arange(t, device=mask.device)
    holes = (m != ((pos >= lead[:, None]) & (pos < (lead + count)[:, None]))).any()
    _report(holes)
    return torch.nn.functional.pad(cu, (0, 1), value=b * t).to(torch.int32)


def _report(bad: Tensor, what: int = _lib.STATUS_BAD_SEQUENCES) -> None:
    """Set ``what`` in the stream's status word where ``bad`` - without waiting for it."""
    _lib.status_word(bad.device).bitwise_or_(bad.to(torch.int32) * what)


def _mask_leaves(function) -> list:
    """The mask functions of which transformers put ``function`` together by intersection."""
    if getattr(function, "__qualname__", "").startswith("and_masks.<locals>"):
        parts = inspect.getclosurevars(function).nonlocals.get("mask_functions", ())
        return [leaf for part in parts for leaf in _mask_leaves(part)]
    return [function]


def _packed_offsets(same_sequence, b: int, t: int, device) -> Tensor:
    """Offsets of the sequences of a [B, T] batch: a row begins one, and so does a token that ``same_sequence``
    keeps apart from the one before it.  Their number is read from the device, as transformers itself does to
    find out that there are several."""
    rows, at = torch.arange(b, device=device)[:, None], torch.arange(1, t, device=device)[None]
    first = torch.ones(b, t, dtype=torch.bool, device=device)
    if t > 1:
        first[:, 1:] = ~same_sequence(rows, 0, at, at - 1)
    cu = torch.nn.functional.pad(first.reshape(-1).nonzero()[:, 0], (0, 1), value=b * t).to(torch.int32)
    cu.implied = True
    return cu


def hf_packed_mask(batch_size, q_length, kv_length, *args, attention_mask=None, mask_function=None, device=None,
                   **kwargs):
    """The mask that transformers prepares once per forward: nothing, or the offsets of a padded batch or of
    rows whose position ids start several sequences (``mask_function`` then keeps these apart).  Any other
    mask function - bidirectional, windows, chunks, overlays - is refused."""
    from transformers import masking_utils

    packed = None
    for leaf in [] if mask_function is None else _mask_leaves(mask_function):
        if getattr(leaf, "__qualname__", "").startswith("packed_sequence_mask_function.<locals>"):
            packed = leaf
        elif leaf is not masking_utils.causal_mask_function:
            raise ValueError(f"{HF_NAME}: full causal attention only, got the mask function "
                             f"{getattr(leaf, '__qualname__', leaf)}")
    if attention_mask is None:
        return None if packed is None else _packed_offsets(packed, batch_size, q_length, device)
    if packed is not None or attention_mask.dim() != 2 or attention_mask.shape[1] != q_length or kv_length != q_length:
        raise ValueError(f"{HF_NAME}: takes [batch, tokens] padding masks and no cached tokens, got a mask of "
                         f"{tuple(attention_mask.shape)} for {q_length} queries and {kv_length} keys")
    return _padded_offsets(attention_mask)


def hf_packed_attention(module, query, key, value, attention_mask, dropout: float = 0.0, scaling: float | None = None,
                        sliding_window=None, is_causal=None, cu_seq_lens_q=None, position_ids=None, **kwargs):
    """``packed_attention`` with the signature of ``ALL_ATTENTION_FUNCTIONS``: query [B, Hq, T, D], key and
    value [B, Hk, T, D] -> ([B, T, Hq, D], None).  A packed row (B = 1) brings its offsets as
    ``cu_seq_lens_q`` (transformers' ``DataCollatorWithFlattening(return_flash_attn_kwargs=True)``);
    otherwise each batch row is a sequence, or what its padding mask leaves of it, or the sequences that its
    position ids start.  The last are kept apart and reported through the status word, since finding them
    waits for the device.  transformers looks for them only in a forward without a cache; with one it takes a
    row as one sequence, which is reported too where position ids restart."""
    b, hq, t, d = query.shape
    if dropout:
        raise ValueError(f"{HF_NAME}: attention dropout is not supported")
    if is_causal is None:
        is_causal = getattr(module, "is_causal", True)
    if sliding_window is not None or kwargs.get("softcap") is not None or not is_causal:
        raise ValueError(f"{HF_NAME}: full causal attention only")
    if kwargs.get("s_aux") is not None:
        raise ValueError(f"{HF_NAME}: attention sinks are not supported")
    if key.shape[2] != t:
        raise ValueError(f"{HF_NAME}: {t} queries against {key.shape[2]} keys: a cache is not supported, use 'sdpa'")
    if cu_seq_lens_q is not None:
        if b != 1:
            raise ValueError(f"{HF_NAME}: cu_seq_lens_q describes one packed row, got a batch of {b}")
        cu = cu_seq_lens_q
    elif attention_mask is not None:
        if attention_mask.dim() != 1:
            raise ValueError(f"{HF_NAME}: takes the mask that hf_packed_mask prepares, got one of "
                             f"{tuple(attention_mask.shape)}")
        cu = attention_mask
        if getattr(cu, "implied", False) and getattr(module, "layer_idx", 0) == 0:
            _report(torch.ones((), dtype=torch.bool, device=cu.device), _lib.STATUS_IMPLIED_SEQUENCES)
    else:
        cu = torch.arange(0, (b + 1) * t, max(t, 1), dtype=torch.int32, device=query.device)[:b + 1]
        if position_ids is not None and t > 1 and getattr(module, "layer_idx", 0) == 0:
            _report((position_ids[..., 1:] <= position_ids[..., :-1]).any())
    seqs = pack_sequences(cu, b * t)
    rows = [x.transpose(1, 2).reshape(b * t, x.shape[1], d) for x in (query, key, value)]
    return packed_attention(*rows, seqs, scale=scaling).view(b, t, hq, d), None


def register_with_transformers() -> str:
    """Make ``attn_implementation="bastile_packed"`` known to transformers; returns the name."""
    from transformers import AttentionInterface, AttentionMaskInterface

    AttentionInterface.register(HF_NAME, hf_packed_attention)
    AttentionMaskInterface.register(HF_NAME, hf_packed_mask)
    return HF_NAME
