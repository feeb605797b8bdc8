"""Token log-probabilities and the clipped policy loss through the output head, on sm_100a.

The reference's only loss is the mean or summed cross-entropy; these are the two next to it that
post-training needs, built the same way: ``[tokens, vocab]`` logits exist one chunk of rows at a time
(``fused_linear_policy_loss``) or not at all (``fused_linear_log_probs`` without gradients).

* The softmax statistics and the target logit come from the fp32 accumulators of the logits product.
  ``fused_linear_cross_entropy`` rounds the logits to 16 bits first, as ``lm_head`` would; the ratio
  of two log-probabilities would carry that rounding as a relative error of a percent.
* ``fused_linear_log_probs`` recomputes the logits in its backward, where the epilogue turns them into
  ``dlogits`` before they are rounded; its forward keeps one log-sum-exp per row.
* ``fused_linear_policy_loss`` knows its gradient with respect to a row's logits as soon as the row's
  statistics are complete (no other row's result enters), so one logits product serves loss and
  gradients: three products instead of four, with the logits kept in 16 bits as differences to the
  maximum of their 128 columns.
* Nothing waits for the host; ignored rows are never computed with (their hidden state, old
  log-probability or advantage may hold anything, NaN included).
"""

from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from .. import _lib
from .fused_linear_cross_entropy import _GEMM_DTYPES, AUTO_CHUNK_BYTES, AUTO_CHUNK_ROWS, DEFAULT_CHUNK

_F32_MAX = torch.finfo(torch.float32).max


class PolicyLoss(NamedTuple):
    """``loss`` is differentiable; the others are for the log: ``log_probs`` (fp32, the target's shape, 0
    where ignored), ``kl`` and ``clip_fraction`` (averages with the loss's own token weights; ``kl`` is 0
    without ``ref_log_probs``)."""

    loss: Tensor
    log_probs: Tensor
    kl: Tensor
    clip_fraction: Tensor


def _check(what: str, hidden: Tensor, weight: Tensor, target: Tensor, chunk_size: int) -> None:
    if hidden.dtype not in _GEMM_DTYPES:
        raise TypeError(f"{what}: unsupported hidden-state dtype {hidden.dtype}")
    if hidden.dim() < 1 or weight.dim() != 2 or weight.shape[1] != hidden.shape[-1]:
        raise ValueError(f"{what}: weight {tuple(weight.shape)} must be [vocab, hidden] for hidden states "
                         f"{tuple(hidden.shape)}")
    if target.shape != hidden.shape[:-1]:
        raise ValueError(f"{what}: target {tuple(target.shape)} does not match hidden states {tuple(hidden.shape)}")
    if target.dtype.is_floating_point or target.dtype == torch.bool:
        raise TypeError(f"{what}: target must hold token ids, got {target.dtype}")
    if hidden.shape[-1] % (16 // hidden.element_size()) != 0 or hidden.shape[-1] == 0 or weight.shape[0] == 0:
        raise ValueError(f"{what}: rows of {hidden.shape[-1]} {hidden.dtype} are not whole 16-byte vectors")
    if int(chunk_size) < 1:
        raise ValueError(f"{what}: chunk_size must be positive, got {chunk_size}")
    _lib.require_cuda(hidden, weight, target)


def _rows_of(x: Tensor) -> Tensor:
    """[..., H] -> [rows, H] with unit inner stride and 16-byte rows."""
    x2 = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    vec = 16 // x2.element_size()
    if x2.stride(-1) != 1 or x2.data_ptr() % 16 != 0 or (x2.shape[0] > 1 and
                                                         (x2.stride(0) % vec != 0 or x2.stride(0) < x2.shape[1])):
        x2 = x2.contiguous()
    return x2 if x2.data_ptr() % 16 == 0 else x2.clone()  # (dense rows may lie off a 16-byte boundary)


def _head_weight(weight: Tensor, dtype) -> Tensor:
    if weight.dtype == dtype and weight.is_contiguous() and weight.data_ptr() % 16 == 0:
        return weight
    w = weight.detach()
    w = w if w.dtype == dtype else w.to(dtype)
    w = w.contiguous()
    return w if w.data_ptr() % 16 == 0 else w.clone()


def _flat(t: Tensor, dtype) -> Tensor:
    """``t``'s values one behind the other in ``dtype`` (itself if they lie that way)."""
    return t if t.dtype == dtype and t.is_contiguous() else t.detach().to(dtype).contiguous()


def _ld(x2: Tensor) -> int:
    return x2.stride(0) if x2.shape[0] > 1 else x2.shape[1]


def _ld_logits(vocab: int) -> int:
    return (vocab + 7) // 8 * 8  # whole 16-byte vectors


def _chunk_rows(chunk_size: int, rows: int, ld_logits: int) -> int:
    """The rule of fused_linear_cross_entropy: the default may grow to AUTO_CHUNK_ROWS rows."""
    want = int(chunk_size)
    if want == DEFAULT_CHUNK and AUTO_CHUNK_ROWS * ld_logits * 2 <= AUTO_CHUNK_BYTES:
        want = AUTO_CHUNK_ROWS
    return max(1, min(want, rows))


def _f32(dev, *shape) -> Tensor:
    return torch.empty(shape, dtype=torch.float32, device=dev)


def _runs(dev, rows: int, hdim: int, vocab: int, code: int) -> int:
    """Partial sums of d hidden that the product of ``rows`` rows writes: counted for ``dev``'s SMs."""
    with _lib.device_of(dev):
        return int(_lib.get_lib().bt_dhidden_runs(rows, hdim, vocab, code))


def _dweight_out(w: Tensor, w_dtype) -> Tensor:
    """The weight gradient's buffer: a registered destination if there is one."""
    out_dtype = w_dtype if w_dtype in (w.dtype, torch.float32) else w.dtype
    out = _lib.grad_sink(w, out_dtype) if w.dtype == w_dtype else None
    return out if out is not None else torch.empty(w.shape, dtype=out_dtype, device=w.device)


def _log_probs(hidden, weight, target, ignore_index: int, chunk_size: int, keep: bool):
    """(log-probabilities, what the backward needs if ``keep``)."""
    lib = _lib.get_lib()
    x, w, labels = _rows_of(hidden), _head_weight(weight, hidden.dtype), _flat(target, torch.int64)
    dev, rows = x.device, x.shape[0]
    vocab, hdim = w.shape
    logp = _f32(dev, rows)
    lse = _f32(dev, rows) if keep else None
    # without logits in memory a chunk only bounds the statistics (8 bytes per 128 columns)
    step = max(1, min(rows, max(chunk_size, AUTO_CHUNK_ROWS)))
    ws = _f32(dev, int(lib.bt_logp_fwd_ws_floats(step, vocab)))
    st = _lib.status_word(dev)
    with _lib.device_of(dev), _lib.timed("logp_fwd", 2 * -(-rows // step), dev):
        rc = lib.bt_logp_fwd(x.data_ptr(), w.data_ptr(), labels.data_ptr(), logp.data_ptr(),
                             lse.data_ptr() if keep else None, ws.data_ptr(), rows, hdim, vocab, _ld(x), step,
                             ignore_index, _lib.dtype_code(x.dtype), st.data_ptr(), _lib.stream_ptr(dev))
    _lib.check(rc, "bt_logp_fwd")
    return logp.view(target.shape), (x, w, labels, lse)


class LinearLogProbsFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, target, ignore_index, chunk_size):
        logp, saved = _log_probs(hidden, weight, target, ignore_index, chunk_size, True)
        ctx.save_for_backward(*saved)
        ctx.meta = (hidden.shape, weight.dtype, ignore_index, chunk_size)
        return logp

    @staticmethod
    @once_differentiable
    def backward(ctx, dlogp):
        lib = _lib.get_lib()
        x, w, labels, lse = ctx.saved_tensors
        shape, w_dtype, ignore_index, chunk_size = ctx.meta
        need_x, need_w = ctx.needs_input_grad[0], ctx.needs_input_grad[1]
        dev, rows = x.device, x.shape[0]
        vocab, hdim = w.shape
        dx = torch.empty((rows, hdim), dtype=x.dtype, device=dev) if need_x else None
        dw = _dweight_out(w, w_dtype) if need_w else None
        if rows == 0:
            return (dx.view(shape) if need_x else None, dw.zero_().to(w_dtype) if need_w else None, None, None, None)
        g = _flat(dlogp, torch.float32)
        ld = _ld_logits(vocab)
        step = _chunk_rows(chunk_size, rows, ld)
        n_chunks = -(-rows // step)
        dlogits = torch.empty((step, ld), dtype=x.dtype, device=dev)
        masked = torch.empty((rows, hdim), dtype=x.dtype, device=dev)
        code = _lib.dtype_code(x.dtype)
        parts = _f32(dev, _runs(dev, step, hdim, vocab, code), step, hdim) if need_x else None
        acc = _f32(dev, vocab, hdim) if need_w and n_chunks > 1 else None
        ws = _f32(dev, 2 * rows + 1)
        st = _lib.status_word(dev)
        with _lib.device_of(dev), _lib.timed("logp_bwd", 2 + n_chunks * (1 + 2 * int(need_x) + int(need_w)), dev):
            rc = lib.bt_logp_bwd(g.data_ptr(), x.data_ptr(), w.data_ptr(), labels.data_ptr(), lse.data_ptr(),
                                 masked.data_ptr(), dlogits.data_ptr(), dx.data_ptr() if need_x else None,
                                 parts.data_ptr() if need_x else None, dw.data_ptr() if need_w else None,
                                 acc.data_ptr() if acc is not None else None, ws.data_ptr(), rows, hdim, vocab,
                                 _ld(x), step, ignore_index, code, _lib.dtype_code(dw.dtype) if need_w else 0,
                                 st.data_ptr(), _lib.stream_ptr(dev))
        _lib.check(rc, "bt_logp_bwd")
        return (dx.view(shape) if need_x else None, dw.to(w_dtype) if need_w else None, None, None, None)


def _policy(hidden, weight, target, old, adv, ref, cu, clip_low, clip_high, kl_coef, ignore_index, chunk_size, need_x,
            need_w):
    """((loss, log-probabilities, averages), what the backward needs)."""
    lib = _lib.get_lib()
    x, w, labels = _rows_of(hidden), _head_weight(weight, hidden.dtype), _flat(target, torch.int64)
    dev, rows = x.device, x.shape[0]
    vocab, hdim = w.shape
    grad = need_x or need_w
    old, adv, ref = (None if t is None else _flat(t, torch.float32) for t in (old, adv, ref))
    n_seq = 1 if cu is None else cu.numel() - 1
    ld = _ld_logits(vocab)
    step = _chunk_rows(chunk_size, rows, ld)
    n_chunks = -(-rows // step)
    loss, averages, logp = _f32(dev), _f32(dev, 8), _f32(dev, rows)
    ws = _f32(dev, int(lib.bt_policy_fwd_ws_floats(rows, step, n_seq, vocab)))
    logits = torch.empty((step, ld), dtype=x.dtype, device=dev) if grad else None
    masked = torch.empty((rows, hdim), dtype=x.dtype, device=dev) if grad else None
    code = _lib.dtype_code(x.dtype)
    # fp32 until the upstream gradient is known: one rounding to the hidden states' type.  The runs of a single
    # chunk are added up then; those of several at once, so that only the sums are kept.
    runs = _runs(dev, step, hdim, vocab, code) if need_x else 1
    dx = _f32(dev, runs if n_chunks <= 1 else 1, rows, hdim) if need_x else None
    parts = _f32(dev, runs, step, hdim) if n_chunks > 1 and runs > 1 else None
    acc = _f32(dev, vocab, hdim) if need_w and n_chunks > 1 else None
    ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    d = _lib.PolicyDesc(ptr(x), ptr(w), ptr(labels), ptr(old), ptr(adv), ptr(ref), ptr(cu), ptr(logp), ptr(loss),
                        ptr(averages), ptr(dx), ptr(acc), ptr(masked), ptr(logits), ptr(ws), rows, hdim, vocab, _ld(x),
                        step, n_seq, ignore_index, clip_low, clip_high, kl_coef, int(need_w), code, ptr(parts))
    st = _lib.status_word(dev)
    with _lib.device_of(dev), _lib.timed("policy_fwd", 2 + int(grad) + n_chunks *
                                         (2 + int(grad) + int(need_x) + int(need_w) + int(parts is not None)) -
                                         int(need_w), dev):
        rc = lib.bt_policy_fwd(ctypes.byref(d), st.data_ptr(), _lib.stream_ptr(dev))
    _lib.check(rc, "bt_policy_fwd")
    last = masked[(n_chunks - 1) * step:] if need_w and n_chunks else None
    return (loss, logp.view(target.shape), averages), (w, averages, dx, logits if need_w else None, last, acc)


class LinearPolicyLossFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, *args):
        out, saved = _policy(hidden, weight, *args, ctx.needs_input_grad[0], ctx.needs_input_grad[1])
        ctx.save_for_backward(*saved)
        ctx.meta = (hidden.shape, hidden.dtype, weight.dtype)
        ctx.mark_non_differentiable(out[1], out[2])
        ctx.set_materialize_grads(False)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss, *_):
        none = (None,) * 10
        if dloss is None:
            return (None, None, *none)
        lib = _lib.get_lib()
        w, averages, dx, dlogits, x_last, acc = ctx.saved_tensors
        shape, x_dtype, w_dtype = ctx.meta
        need_x, need_w = ctx.needs_input_grad[0], ctx.needs_input_grad[1]
        dev = w.device
        vocab, hdim = w.shape
        stream, code = _lib.stream_ptr(dev), _lib.dtype_code(x_dtype)
        # the coefficients were stored relative to the largest token weight; fp16 has a scale of its own for d weight
        alphas = dloss.detach().to(torch.float32) * averages[2:5:2]
        alpha_x, alpha_w = alphas.data_ptr(), alphas.data_ptr() + 4
        dx_out = dw = None
        with _lib.device_of(dev), _lib.timed("policy_bwd", int(need_x) + int(need_w and x_last is not None), dev):
            if need_x:
                dx_out = torch.empty(shape, dtype=x_dtype, device=dev)
                n = dx_out.numel()
                _lib.check(lib.bt_sum_runs(dx.data_ptr(), dx_out.data_ptr(), n, dx.shape[0], n, alpha_x, code,
                                           stream), "bt_sum_runs(dhidden)")
            if need_w:
                dw = _dweight_out(w, w_dtype)
                if x_last is None:
                    dw.zero_()
                else:
                    # dW = alpha (dlogits^T x + the other chunks)
                    st = _lib.status_word(dev)
                    _lib.check(lib.bt_gemm(dlogits.data_ptr(), x_last.data_ptr(), dw.data_ptr(), vocab, hdim,
                                           x_last.shape[0], dlogits.shape[1], hdim, hdim, 0, 0, code,
                                           _lib.dtype_code(dw.dtype), acc.data_ptr() if acc is not None else None,
                                           hdim, alpha_w, st.data_ptr(), stream), "bt_gemm(dweight)")
                dw = dw.to(w_dtype)
        return (dx_out, dw, *none)


def fused_linear_log_probs(hidden_states: Tensor, weight: Tensor, target: Tensor, ignore_index: int = -100,
                           chunk_size: int = DEFAULT_CHUNK) -> Tensor:
    """``log_softmax(hidden_states @ weight.T)[..., target]`` in fp32, without ``[tokens, vocab]`` logits in
    the forward: hidden_states [..., H], weight [vocab, H], target [...] token ids; 0 (and no gradient)
    where ``target == ignore_index``.  ``chunk_size`` rows of logit gradients are held at a time in the
    backward.  fp32 tensors are multiplied as tf32.  A target that is neither ``ignore_index`` nor a
    vocabulary row counts as ignored and sets ``BT_STATUS_BAD_LABEL`` (see ``check_all_status``)."""
    _check("fused_linear_log_probs", hidden_states, weight, target, chunk_size)
    if torch.is_grad_enabled() and (hidden_states.requires_grad or weight.requires_grad):
        return LinearLogProbsFunction.apply(hidden_states, weight, target, int(ignore_index), int(chunk_size))
    return _log_probs(hidden_states, weight, target, int(ignore_index), int(chunk_size), False)[0]


def fused_linear_policy_loss(hidden_states: Tensor, weight: Tensor, target: Tensor, old_log_probs: Tensor,
                             advantages: Tensor, ref_log_probs: Tensor | None = None, clip_low: float = 0.2,
                             clip_high: float = 0.2, kl_coef: float = 0.0, ignore_index: int = -100,
                             cu_seqlens: Tensor | None = None, chunk_size: int = DEFAULT_CHUNK) -> PolicyLoss:
    """The clipped policy loss of tokens under ``softmax(hidden_states @ weight.T)``.

    With ``r = exp(logp - old_log_probs)`` and ``d = ref_log_probs - logp`` a token's loss is
    ``-min(r A, clip(r, 1 - clip_low, 1 + clip_high) A) + kl_coef (exp(d) - d - 1)``; the result is the
    mean over tokens whose target is not ``ignore_index``, or with ``cu_seqlens`` [sequences + 1] (packed
    offsets as for ``pack_sequences``) the mean over sequences of their tokens' means - sequences
    without a counted token are left out, tokens behind the last sequence count as ignored.
    ``old_log_probs``, ``advantages`` and ``ref_log_probs`` have the target's shape and get no gradients.
    Gradients of logits are formed in the hidden states' type relative to the largest token weight (with
    fp16, rows of very large or small coefficients scaled by a power of two)."""
    what = "fused_linear_policy_loss"
    for name, t in (("old_log_probs", old_log_probs), ("advantages", advantages), ("ref_log_probs", ref_log_probs)):
        if t is None and name == "ref_log_probs":
            continue
        if t.shape != target.shape or not t.dtype.is_floating_point:
            raise ValueError(f"{what}: {name} must be floating-point values in the target's shape "
                             f"{tuple(target.shape)}, got {t.dtype} {tuple(t.shape)}")
    clip_low, clip_high, kl_coef = float(clip_low), float(clip_high), float(kl_coef)
    if not (0.0 <= clip_low <= 1.0 and 0.0 <= clip_high < float("inf")):
        raise ValueError(f"{what}: need 0 <= clip_low <= 1 and clip_high >= 0, got {clip_low} and {clip_high}")
    if not abs(kl_coef) <= _F32_MAX:
        raise ValueError(f"{what}: kl_coef must be finite in fp32, got {kl_coef}")
    if kl_coef != 0.0 and ref_log_probs is None:
        raise ValueError(f"{what}: kl_coef = {kl_coef} needs ref_log_probs")
    if cu_seqlens is not None:
        if cu_seqlens.dim() != 1 or cu_seqlens.numel() < 1:
            raise ValueError(f"{what}: cu_seqlens must be [sequences + 1], got {tuple(cu_seqlens.shape)}")
        if cu_seqlens.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"{what}: cu_seqlens must be int32 or int64, got {cu_seqlens.dtype}")
    _check(what, hidden_states, weight, target, chunk_size)
    _lib.require_cuda(hidden_states, old_log_probs, advantages,
                      *(t for t in (ref_log_probs, cu_seqlens) if t is not None))
    if cu_seqlens is not None:
        if cu_seqlens.dtype == torch.int64:
            cu_seqlens = cu_seqlens.clamp(-1, (1 << 31) - 1).to(torch.int32)
        cu_seqlens = cu_seqlens.contiguous()
    args = (hidden_states, weight, target, old_log_probs, advantages, ref_log_probs, cu_seqlens, clip_low, clip_high,
            kl_coef, int(ignore_index), int(chunk_size))
    if torch.is_grad_enabled() and (hidden_states.requires_grad or weight.requires_grad):
        loss, log_probs, averages = LinearPolicyLossFunction.apply(*args)
    else:
        loss, log_probs, averages = _policy(*args, False, False)[0]
    return PolicyLoss(loss, log_probs, averages[0], averages[1])
