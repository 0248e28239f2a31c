"""Capturing a training step the way torch documents it: warm up on a side stream, whose last loss stays alive, then capture."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("how", ["backward", "grad"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_warm_up_on_a_side_stream(dtype, how):
    from wfe_amd import decoder as d
    g = torch.Generator(device="cuda").manual_seed(0)
    h = torch.randn(40, 64, generator=g, device="cuda").to(dtype).requires_grad_()
    w = (torch.randn(300, 64, generator=g, device="cuda") / 8).to(dtype).requires_grad_()
    y = torch.randint(0, 300, (40,), generator=g, device="cuda")
    ids = torch.randint(0, 300, (40,), generator=g, device="cuda")

    def step():
        loss = d.linear_cross_entropy(h + d.token_embedding(ids, w), w, y)
        if how == "grad":
            return (loss, *torch.autograd.grad(loss, (h, w), retain_graph=True))
        h.grad = w.grad = None
        loss.backward()
        return loss, h.grad, w.grad
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            alive = step()                       # its graph, and with it the parameters' nodes on this stream, live on
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(4):
        y.copy_(torch.randint(0, 300, (40,), generator=g, device="cuda"))
        ids.copy_(torch.randint(0, 300, (40,), generator=g, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.detach().clone() for t in out]
        h2, w2 = h.detach().clone().requires_grad_(), w.detach().clone().requires_grad_()
        loss = d.linear_cross_entropy(h2 + d.token_embedding(ids, w2), w2, y)
        for a, b in zip(got, (loss, *torch.autograd.grad(loss, (h2, w2)))):
            assert torch.equal(a, b)
    assert alive[0].grad_fn is not None
