"""Registered gradient destinations: lent to one contribution at a time."""

import torch


class Scaled(torch.autograd.Function):
    """sum(w) * c, its gradient written into the weight's registered destination where that is free."""

    @staticmethod
    def forward(ctx, w, c):
        ctx.save_for_backward(w)
        ctx.c = c
        return w.sum() * c

    @staticmethod
    def backward(ctx, up):
        from bastile_b200 import _lib

        (w,) = ctx.saved_tensors
        out = _lib.grad_sink(w, w.dtype)
        out = out if out is not None else torch.empty_like(w)
        return out.fill_(ctx.c).mul_(up), None


def _sunk(shape=(4, 8)):
    from bastile_b200 import _lib

    w = torch.zeros(shape, requires_grad=True)
    dest = torch.full(shape, -1.0)
    _lib.register_grad_sink(w.data, dest)
    return _lib, w, dest


def test_two_uses_in_one_backward_add_up():
    _lib, w, dest = _sunk()
    try:
        (Scaled.apply(w, 3.0) + Scaled.apply(w, 4.0) + Scaled.apply(w, 0.5)).backward()
        assert (w.grad == 7.5).all()
    finally:
        _lib.unregister_grad_sinks([dest])


def test_accumulation_over_two_backward_passes():
    _lib, w, dest = _sunk()
    try:
        Scaled.apply(w, 3.0).backward()
        assert w.grad.data_ptr() == dest.data_ptr()  # in place
        Scaled.apply(w, 4.0).backward()
        assert (w.grad == 7.0).all()
    finally:
        _lib.unregister_grad_sinks([dest])


def test_a_gradient_in_a_users_hands_is_not_overwritten():
    _lib, w, dest = _sunk()
    try:
        (a,) = torch.autograd.grad(Scaled.apply(w, 3.0), w)
        (b,) = torch.autograd.grad(Scaled.apply(w, 4.0), w)
        assert (a == 3.0).all() and (b == 4.0).all()
        del a, b
        Scaled.apply(w, 5.0).backward()  # both are gone: in place again
        assert w.grad.data_ptr() == dest.data_ptr()
    finally:
        _lib.unregister_grad_sinks([dest])


def test_a_gradient_that_waits_for_its_optimizer_is_not_overwritten():
    """What an optimizer took out of ``.grad`` lies in the destination until its step."""
    _lib, w, dest = _sunk()
    try:
        for _ in range(2):
            Scaled.apply(w, 3.0).backward()
            assert w.grad.data_ptr() == dest.data_ptr()
            w.grad = None
            _lib.hold_grad_sink(w)
            torch.autograd.grad(Scaled.apply(w, 4.0), w)
            assert (dest == 3.0).all()
            _lib.release_grad_sinks([w])
    finally:
        _lib.unregister_grad_sinks([dest])
    assert w.data_ptr() not in _lib._grad_held and w.data_ptr() not in _lib._grad_lent
