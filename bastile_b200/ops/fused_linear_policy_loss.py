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

from typing import NamedTuple

import torch
from torch import Tensor

from .. import _lib
from .fused_linear_cross_entropy import _GEMM_DTYPES, AUTO_CHUNK_BYTES, AUTO_CHUNK_ROWS, DEFAULT_CHUNK


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
    x2 = x.reshape(-1, x.shape[-1])
    vec = 16 // x2.element_size()
    if x2.stride(-1) != 1 or x2.data_ptr() % 16 != 0 or (x2.shape[0] > 1 and
                                                         (x2.stride(0) % vec != 0 or x2.stride(0) < x2.shape[1])):
        x2 = x2.contiguous()
    return x2


def _head_weight(weight: Tensor, dtype) -> Tensor:
    w = weight.detach()
    w = w if w.dtype == dtype else w.to(dtype)
    w = w.contiguous()
    return w if w.data_ptr() % 16 == 0 else w.clone()


def _labels(target: Tensor) -> Tensor:
    return target.reshape(-1).to(torch.int64).contiguous()


def _ld(x2: Tensor) -> int:
    return x2.stride(0) if x2.shape[0] > 1 else x2.shape[1]


def _chunk_rows(chunk_size: int, rows: int, ld_logits: int) -> int:
    """The rule of fused_linear_cross_entropy: the default may grow to AUTO_CHUNK_ROWS rows."""
    want = int(chunk_size)
    if want == DEFAULT_CHUNK and AUTO_CHUNK_ROWS * ld_logits * 2 <= AUTO_CHUNK_BYTES:
        want = AUTO_CHUNK_ROWS
    return max(1, min(want, rows))


class _Head:
    """One call's view of the C entry points: device, stream, sizes and types filled in."""

    def __init__(self, x: Tensor, w: Tensor, ignore_index: int):
        self.lib, self.dev = _lib.get_lib(), x.device
        self.stream = _lib.stream_ptr(self.dev)
        self.st = _lib.status_word(self.dev)
        self.code = _lib.dtype_code(x.dtype)
        self.w, self.hdim, self.vocab = w, w.shape[1], w.shape[0]
        self.ignore = int(ignore_index)
        self.ld = (self.vocab + 7) // 8 * 8
        self.n_vt = int(self.lib.bt_lce_num_vtiles(self.vocab))

    def f32(self, *shape) -> Tensor:
        return torch.empty(shape, dtype=torch.float32, device=self.dev)

    def stats(self, xc, labels, logits, tile_stats, tgt) -> None:
        _lib.check(self.lib.bt_logp_stats(xc.data_ptr(), self.w.data_ptr(), labels.data_ptr(),
                                          logits.data_ptr() if logits is not None else None, tile_stats.data_ptr(),
                                          tgt.data_ptr(), xc.shape[0], self.hdim, self.vocab, _ld(xc), self.ld,
                                          self.ignore, self.code, self.st.data_ptr(), self.stream), "bt_logp_stats")

    def mask_rows(self, x2, labels) -> Tensor:
        out = torch.empty(x2.shape, dtype=x2.dtype, device=self.dev)
        _lib.check(self.lib.bt_logp_mask_rows(x2.data_ptr(), out.data_ptr(), labels.data_ptr(), x2.shape[0], self.hdim,
                                              _ld(x2), self.vocab, self.ignore, self.code, self.stream),
                   "bt_logp_mask_rows")
        return out

    def dhidden(self, dlogits, rows, out, alpha) -> None:
        """out[rows, H] = alpha dlogits[rows, V] W[V, H]"""
        _lib.check(self.lib.bt_gemm(dlogits.data_ptr(), self.w.data_ptr(), out.data_ptr(), rows, self.hdim, self.vocab,
                                    self.ld, self.hdim, self.hdim, 1, 0, self.code, _lib.dtype_code(out.dtype), None,
                                    0, alpha.data_ptr() if alpha is not None else None, self.st.data_ptr(),
                                    self.stream), "bt_gemm(dhidden)")

    def dweight(self, dlogits, xc, out, addend, alpha) -> None:
        """out[V, H] = alpha (dlogits^T x + addend)"""
        _lib.check(self.lib.bt_gemm(dlogits.data_ptr(), xc.data_ptr(), out.data_ptr(), self.vocab, self.hdim,
                                    xc.shape[0], self.ld, _ld(xc), self.hdim, 0, 0, self.code,
                                    _lib.dtype_code(out.dtype), addend.data_ptr() if addend is not None else None,
                                    self.hdim, alpha.data_ptr() if alpha is not None else None, self.st.data_ptr(),
                                    self.stream), "bt_gemm(dweight)")

    def dweight_out(self, w_dtype) -> Tensor:
        """The weight gradient's buffer: a registered destination if there is one."""
        out_dtype = w_dtype if w_dtype in (self.w.dtype, torch.float32) else self.w.dtype
        out = _lib.grad_sink(self.w, out_dtype) if self.w.dtype == w_dtype else None
        return out if out is not None else torch.empty((self.vocab, self.hdim), dtype=out_dtype, device=self.dev)


class LinearLogProbsFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, target, ignore_index, chunk_size):
        x, w, labels = _rows_of(hidden), _head_weight(weight, hidden.dtype), _labels(target)
        rows = x.shape[0]
        h = _Head(x, w, ignore_index)
        grad = any(ctx.needs_input_grad[:2])
        logp = h.f32(rows)
        lse = h.f32(rows) if grad else None
        # without logits in memory a chunk only bounds the statistics (8 bytes per 128 columns)
        step = max(1, min(rows, max(int(chunk_size), AUTO_CHUNK_ROWS)))
        tile_stats, tgt = h.f32(step, h.n_vt, 2), h.f32(step)
        with _lib.device_of(h.dev), _lib.timed("logp_fwd", 2 * -(-rows // step), h.dev):
            for s in range(0, rows, step):
                xc, lc = x[s:s + step], labels[s:s + step]
                h.stats(xc, lc, None, tile_stats, tgt)
                _lib.check(h.lib.bt_logp_rows(tile_stats.data_ptr(), tgt.data_ptr(), lc.data_ptr(),
                                              logp[s:].data_ptr(), lse[s:].data_ptr() if grad else None, xc.shape[0],
                                              h.vocab, h.ignore, h.st.data_ptr(), h.stream), "bt_logp_rows")
        if grad:
            ctx.save_for_backward(x, w, labels, lse)
            ctx.meta = (hidden.shape, weight.dtype, int(ignore_index), int(chunk_size))
        return logp.view(target.shape)

    @staticmethod
    def backward(ctx, dlogp):
        x, w, labels, lse = ctx.saved_tensors
        shape, w_dtype, ignore_index, chunk_size = ctx.meta
        need_x, need_w = ctx.needs_input_grad[0], ctx.needs_input_grad[1]
        rows = x.shape[0]
        h = _Head(x, w, ignore_index)
        dx = torch.empty((rows, h.hdim), dtype=x.dtype, device=h.dev) if need_x else None
        dw = h.dweight_out(w_dtype) if need_w else None
        if rows == 0:
            return (dx.view(shape) if need_x else None, dw.zero_().to(w_dtype) if need_w else None, None, None, None)
        g = dlogp.reshape(-1).to(torch.float32).contiguous()
        coef, scal = h.f32(rows), h.f32(1)
        step = _chunk_rows(chunk_size, rows, h.ld)
        n_chunks = -(-rows // step)
        dlogits = torch.empty((step, h.ld), dtype=x.dtype, device=h.dev)
        acc = h.f32(h.vocab, h.hdim) if need_w and n_chunks > 1 else None
        with _lib.device_of(h.dev), _lib.timed("logp_bwd", 2 + n_chunks * (1 + int(need_x) + int(need_w)), h.dev):
            _lib.check(h.lib.bt_logp_coef(g.data_ptr(), labels.data_ptr(), rows, h.vocab, h.ignore, coef.data_ptr(),
                                          scal.data_ptr(), h.stream), "bt_logp_coef")
            xm = h.mask_rows(x, labels)
            for i in range(n_chunks):
                s = i * step
                xc = xm[s:s + step]
                n = xc.shape[0]
                _lib.check(h.lib.bt_logp_dlogits(xc.data_ptr(), w.data_ptr(), labels[s:].data_ptr(),
                                                 lse[s:].data_ptr(), coef[s:].data_ptr(), dlogits.data_ptr(), n,
                                                 h.hdim, h.vocab, _ld(xc), h.ld, h.code, h.st.data_ptr(), h.stream),
                           "bt_logp_dlogits")
                if need_x:
                    h.dhidden(dlogits, n, dx[s:], scal)
                if need_w:
                    last = i == n_chunks - 1
                    h.dweight(dlogits, xc, dw if last else acc, acc if i > 0 else None, scal if last else None)
        return (dx.view(shape) if need_x else None, dw.to(w_dtype) if need_w else None, None, None, None)


class LinearPolicyLossFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, target, old, adv, ref, cu, clip_low, clip_high, kl_coef, ignore_index, chunk_size):
        x, w, labels = _rows_of(hidden), _head_weight(weight, hidden.dtype), _labels(target)
        rows = x.shape[0]
        h = _Head(x, w, ignore_index)
        need_x, need_w = ctx.needs_input_grad[0], ctx.needs_input_grad[1]
        grad = need_x or need_w
        old, adv, ref = (t if t is None else t.detach().reshape(-1).to(torch.float32).contiguous()
                         for t in (old, adv, ref))
        n_seq = 1 if cu is None else cu.numel() - 1
        seq_w, scal, sums = h.f32(max(n_seq, 1)), h.f32(2), h.f32(3)
        logp, terms = h.f32(rows), h.f32(3, rows)
        step = _chunk_rows(chunk_size, rows, h.ld)
        n_chunks = -(-rows // step)
        lse, coef, tgt, tile_stats = h.f32(step), h.f32(step), h.f32(step), h.f32(step, h.n_vt, 2)
        logits = torch.empty((step, h.ld), dtype=x.dtype, device=h.dev) if grad else None
        # fp32 until the upstream gradient is known: one rounding to the hidden states' type
        dx = h.f32(rows, h.hdim) if need_x else None
        acc = h.f32(h.vocab, h.hdim) if need_w and n_chunks > 1 else None
        x_last = x
        cu_ptr = cu.data_ptr() if cu is not None else None
        with _lib.device_of(h.dev), _lib.timed("policy_fwd", 2 + int(grad) + n_chunks *
                                               (2 + int(grad) + int(need_x) + int(need_w)) - int(need_w), h.dev):
            _lib.check(h.lib.bt_policy_weights(labels.data_ptr(), rows, cu_ptr, n_seq, h.vocab, h.ignore,
                                               seq_w.data_ptr(), scal.data_ptr(), h.st.data_ptr(), h.stream),
                       "bt_policy_weights")
            xm = h.mask_rows(x, labels) if grad and rows > 0 else x
            for i in range(n_chunks):
                s = i * step
                xc, lc = xm[s:s + step], labels[s:s + step]
                n = xc.shape[0]
                h.stats(xc, lc, logits, tile_stats, tgt)
                _lib.check(h.lib.bt_policy_rows(tile_stats.data_ptr(), tgt.data_ptr(), lc.data_ptr(), old.data_ptr(),
                                                adv.data_ptr(), ref.data_ptr() if ref is not None else None, cu_ptr,
                                                seq_w.data_ptr(), scal.data_ptr(), logp[s:].data_ptr(),
                                                lse.data_ptr(), coef.data_ptr(), terms.data_ptr(), n, s, rows, n_seq,
                                                h.vocab, h.ignore, clip_low, clip_high, kl_coef, h.stream),
                           "bt_policy_rows")
                if not grad:
                    continue
                _lib.check(h.lib.bt_policy_dlogits(logits.data_ptr(), tile_stats.data_ptr(), lse.data_ptr(),
                                                   lc.data_ptr(), coef.data_ptr(), n, h.vocab, h.ld, h.code, h.stream),
                           "bt_policy_dlogits")
                if need_x:
                    h.dhidden(logits, n, dx[s:], None)
                if need_w:
                    if i < n_chunks - 1:
                        h.dweight(logits, xc, acc, acc if i > 0 else None, None)
                    else:
                        x_last = xc
            _lib.check(h.lib.bt_policy_reduce(terms.data_ptr(), rows, sums.data_ptr(), h.stream), "bt_policy_reduce")
        if grad:
            empty = scal[:0]
            ctx.save_for_backward(w, scal, dx if need_x else empty, logits if need_w else empty, x_last,
                                  acc if acc is not None else empty)
            ctx.meta = (hidden.shape, hidden.dtype, weight.dtype, n_chunks, int(ignore_index))
        loss, kl, clipped = sums[0].clone(), sums[1].clone(), sums[2].clone()
        logp = logp.view(target.shape)
        ctx.mark_non_differentiable(logp, kl, clipped)
        ctx.set_materialize_grads(False)
        return loss, logp, kl, clipped

    @staticmethod
    def backward(ctx, dloss, *_):
        none = (None,) * 10
        if dloss is None:
            return (None, None, *none)
        w, scal, dx, dlogits, x_last, acc = ctx.saved_tensors
        shape, x_dtype, w_dtype, n_chunks, ignore_index = ctx.meta
        need_x, need_w = ctx.needs_input_grad[0], ctx.needs_input_grad[1]
        h = _Head(x_last, w, ignore_index)
        # the coefficients were stored relative to the largest token weight (scal[0])
        alpha = (dloss.detach().to(torch.float32) * scal[0]).reshape(1)
        dx_out = dw = None
        with _lib.device_of(h.dev), _lib.timed("policy_bwd", int(need_x) + int(need_w and n_chunks > 0), h.dev):
            if need_x:
                dx_out = torch.empty(dx.shape, dtype=x_dtype, device=h.dev)
                _lib.check(h.lib.bt_scale_cast(dx.data_ptr(), dx_out.data_ptr(), dx.numel(), alpha.data_ptr(),
                                               _lib.BT_FP32, h.code, h.stream), "bt_scale_cast(dhidden)")
                dx_out = dx_out.view(shape)
            if need_w:
                dw = h.dweight_out(w_dtype)
                if n_chunks == 0:
                    dw.zero_()
                else:
                    h.dweight(dlogits, x_last, dw, acc if n_chunks > 1 else None, alpha)
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
    return LinearLogProbsFunction.apply(hidden_states, weight, target, int(ignore_index), int(chunk_size))


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
    ``old_log_probs``, ``advantages`` and ``ref_log_probs`` have the target's shape and get no gradients."""
    what = "fused_linear_policy_loss"
    for name, t in (("old_log_probs", old_log_probs), ("advantages", advantages), ("ref_log_probs", ref_log_probs)):
        if t is None and name == "ref_log_probs":
            continue
        if t.shape != target.shape or not t.dtype.is_floating_point:
            raise ValueError(f"{what}: {name} must be floating-point values in the target's shape {tuple(target.shape)}, "
                             f"got {t.dtype} {tuple(t.shape)}")
    clip_low, clip_high, kl_coef = float(clip_low), float(clip_high), float(kl_coef)
    if not (0.0 <= clip_low <= 1.0 and 0.0 <= clip_high < float("inf")):
        raise ValueError(f"{what}: need 0 <= clip_low <= 1 and clip_high >= 0, got {clip_low} and {clip_high}")
    if kl_coef != kl_coef or abs(kl_coef) == float("inf"):
        raise ValueError(f"{what}: kl_coef must be finite, got {kl_coef}")
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
    return PolicyLoss(*LinearPolicyLossFunction.apply(hidden_states, weight, target, old_log_probs, advantages,
                                                      ref_log_probs, cu_seqlens, clip_low, clip_high, kl_coef,
                                                      int(ignore_index), int(chunk_size)))
