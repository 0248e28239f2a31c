"""Modes of torch that the decoder operators do not support are refused, before a device is used."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from wfe_amd import decoder


@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_is_refused(grad):
    """A tangent that a call dropped would be a silent zero derivative."""
    h, w, y = torch.randn(2, 3, 8), torch.randn(5, 8), torch.zeros(2, 3, dtype=torch.int64)
    if grad:
        h.requires_grad_(), w.requires_grad_()
    with fwd.dual_level():
        dual_h, dual_w = fwd.make_dual(h, torch.randn(2, 3, 8)), fwd.make_dual(w, torch.randn(5, 8))
        for call in (lambda: decoder.linear_cross_entropy(dual_h, w, y), lambda: decoder.linear_cross_entropy(h, dual_w, y),
                     lambda: decoder.token_embedding(y, dual_w)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
            with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                call()


def test_function_transforms_are_refused():
    h, w, y = torch.randn(2, 3, 8), torch.randn(5, 8), torch.zeros(2, 3, dtype=torch.int64)
    calls = [lambda: torch.func.jvp(lambda a: decoder.linear_cross_entropy(a, w, y), (h,), (h,)),
             lambda: torch.func.grad(lambda a: decoder.linear_cross_entropy(h, a, y))(w),
             lambda: torch.func.grad(lambda a: decoder.token_embedding(y, a).sum())(w),
             lambda: torch.vmap(lambda a, b: decoder.linear_cross_entropy(a, w, b))(h, y),
             lambda: torch.vmap(lambda b: decoder.token_embedding(b, w))(y)]
    for call in calls:
        with pytest.raises(NotImplementedError, match="forward-mode|transform"):
            call()
