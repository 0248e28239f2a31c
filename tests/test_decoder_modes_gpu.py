"""Tensors in unusual states, given to the decoder operators: tangents, negated views."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

pytestmark = pytest.mark.gpu


def case():
    g = torch.Generator(device="cuda").manual_seed(0)
    h = torch.randn(6, 64, generator=g, device="cuda")
    w = torch.randn(50, 64, generator=g, device="cuda") / 8
    return h, w, torch.randint(0, 50, (6,), generator=g, device="cuda")


def test_tangents_are_refused_in_both_directions():
    from wfe_amd import decoder as d
    h, w, y = case()
    h, w = h.requires_grad_(), w.requires_grad_()
    calls = [(d.linear_cross_entropy(h, w, y, reduction="none"), h), (d.token_embedding(y, w), w)]
    with fwd.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            d.linear_cross_entropy(fwd.make_dual(h.detach(), torch.ones_like(h)), w, y)
        for out, of in calls:
            up = fwd.make_dual(torch.ones_like(out), torch.ones_like(out))
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(out, of, up, retain_graph=True)
            assert torch.autograd.grad(out, of, torch.ones_like(out))[0].shape == of.shape
        assert d.linear_cross_entropy(h, w, y).dim() == 0          # no tangent, no refusal
