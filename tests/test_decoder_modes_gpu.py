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


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=["bf16", "f16", "f32"])
def test_saved_tensors_moved_by_hooks(dtype):
    """What a call saves may come back as another tensor (offloading hooks bring back contiguous copies), whatever strides it
    had: the gradients are the same bits."""
    from wfe_amd import decoder as d
    g = torch.Generator(device="cuda").manual_seed(1)
    base = torch.randn(300, 200, generator=g, device="cuda").to(dtype)
    y = torch.randint(0, 100, (40,), generator=g, device="cuda")
    h = torch.randn(40, 64, generator=g, device="cuda").to(dtype).requires_grad_()
    views = {"wide rows": lambda: base[:, :64], "off its alignment": lambda: base[:, 3:67], "every third": lambda: base[::3, 8:72],
             "one row": lambda: base[:1, :64].expand(120, 64), "columns": lambda: base[:64, :150].T, "dense": lambda: base[:, :64].clone()}

    def moved(t):
        return t.detach().cpu()

    def back(t):
        return t.to("cuda")

    def spread(t):
        """Comes back with other strides than it was saved with."""
        room = torch.full((*t.shape[:-1], t.shape[-1] + 8), 7, dtype=t.dtype, device=t.device)
        room[..., :t.shape[-1]] = t.detach()
        return room[..., :t.shape[-1]]
    for name, view in views.items():
        w = view().detach().requires_grad_()

        def step():
            out = d.token_embedding(y, w, scale=0.5)
            loss = d.linear_cross_entropy(h + out, w, y)
            return torch.autograd.grad(loss, (h, w))
        want = step()
        with torch.autograd.graph.save_on_cpu():
            offloaded = step()
        with torch.autograd.graph.saved_tensors_hooks(moved, back):
            again = step()
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, spread):
            strided = step()
        for other in (offloaded, again, strided):
            for a, b in zip(want, other):
                assert torch.equal(a, b), name


def test_saved_tensors_changed_by_hooks_are_refused():
    """Hooks that bring back less than was saved, or another type of it, get an error and no kernel."""
    from wfe_amd import decoder as d
    h, w, y = case()
    h, w = h.requires_grad_(), w.requires_grad_()
    for call in (lambda: d.linear_cross_entropy(h, w, y), lambda: d.token_embedding(y, w).sum()):
        for change in (lambda t: t[:-1] if t.dim() else t, lambda t: t.to(torch.float16), lambda t: t.cpu(),
                       lambda t: t.reshape(-1)[:0]):
            with torch.autograd.graph.saved_tensors_hooks(lambda t: t, change):
                out = call()
            with pytest.raises((RuntimeError, ValueError), match="saved"):
                torch.autograd.grad(out, w)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=["bf16", "f16", "f32"])
def test_lazily_negated_views(dtype):
    """torch keeps the sign of some views (the imaginary part of a conjugate) apart from their memory."""
    from wfe_amd import decoder as d
    h, w, y = case()
    h, w = h.to(dtype), w.to(dtype)
    up = torch.linspace(-1, 1, 6, device="cuda")

    def step(h, w, y, up):
        h, w = h.detach().requires_grad_(), w.detach().requires_grad_()
        loss = d.linear_cross_entropy(h, w, y, reduction="none")
        out = d.token_embedding(y, w)
        with torch.no_grad():
            plain = d.linear_cross_entropy(h, w, y), d.token_embedding(y, w)
        return (loss, out, *plain, *torch.autograd.grad(loss, (h, w), up),
                *torch.autograd.grad(out, w, up[:, None].to(dtype).expand_as(out)))
    want = step(h, w, y, up)
    neg = torch._neg_view
    for given in ((neg(-h), w, y, up), (h, neg(-w), y, up), (h, w, neg(-y), up), (h, w, y, neg(-up)),
                  (neg(-h.expand(6, 64)), neg((-w).T.contiguous()).T, neg(-y), neg(-up))):
        for a, b in zip(want, step(*given)):
            assert torch.equal(a, b)
    if dtype == torch.float32:
        z = torch.complex(torch.zeros_like(h), -h)
        assert z.conj().imag.is_neg()
        assert torch.equal(d.linear_cross_entropy(z.conj().imag, w, y), d.linear_cross_entropy(h.clone(), w, y))
