"""Gradients of the vocabulary cross entropy where the rows are cut into shares: narrow models and many rows.  A share holds at
most 256 MB of d over a usefully wide piece of the vocabulary: 4864 rows of the narrowest models, 2304 in float32."""
import pytest
import torch

from test_decoder_gpu import BF16, F16, F32, check, close, make, oracle

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,dim,vocab,dtype,ignored", [
    (12000, 64, 35003, BF16, 0.1),     # three shares by two pieces
    (5000, 72, 34999, F16, 0.0),       # two shares, rows of 72
    (30000, 40, 5003, BF16, 0.2),      # one piece, two shares
    (30000, 40, 5003, F16, 0.97),      # kept rows in the first share only
    (5200, 64, 28001, F32, 0.1),       # float32: three shares
    (5200, 65, 27999, F32, 0.7),
    (20000, 384, 14003, BF16, 0.3),    # a wider model, three shares
    (150000, 16, 1000, BF16, 0.4)], ids=str)
def test_shares(rows, dim, vocab, dtype, ignored):
    h, w, y = make(rows, dim, vocab, dtype, seed=rows, ignored=ignored)
    check(h, w, y, "mean")
    check(h, w, y, "none")
    check(h, w, y, "sum", grads=(True, False))
    check(h, w, y, "none", grads=(False, True))


def test_shares_without_a_kept_row_and_whole_ones():
    from wfe_amd import decoder as d
    h, w, y = make(12000, 64, 35003, BF16, ignored=0.0)       # shares of 4096
    for kept in (0, 1, 4095, 4096, 4097, 8192, 8193):
        labels = torch.where(torch.arange(12000, device="cuda") < kept, y, -100)
        if kept:
            check(h, w, labels, "mean")
            continue
        a, b = h.clone().requires_grad_(), w.clone().requires_grad_()
        for reduction in ("sum", "mean", "none"):
            loss = d.linear_cross_entropy(a, b, labels, reduction=reduction)
            for g in torch.autograd.grad(loss, (a, b), torch.ones_like(loss)):
                assert not bool(g.any())


def test_shares_under_autocast_and_captured():
    """Gradients written in float32, and a captured pass replayed with other labels (shares that empty and fill)."""
    from wfe_amd import decoder as d
    h, w, y = make(8000, 64, 35003, F32, ignored=0.2)
    a, b = h.clone().requires_grad_(), w.clone().requires_grad_()

    def step():
        with torch.autocast("cuda", dtype=BF16):
            loss = d.linear_cross_entropy(a, b, y)
        return (loss.detach(), *torch.autograd.grad(loss, (a, b)))
    got = step()
    want = oracle(h.to(BF16), w.to(BF16), y, "mean", torch.ones((), device="cuda"))
    for g, at in zip(got, (0, 2, 4)):
        close(g, want[at], want[at + 1], "loss dh dW".split()[at // 2])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed, ignored in enumerate((0.0, 0.9, 0.2, 0.6)):
        y.copy_(make(8000, 64, 35003, F32, seed=seed, ignored=ignored)[2])
        graph.replay()
        torch.cuda.synchronize()
        for x, z in zip([t.clone() for t in out], step()):
            assert torch.equal(x, z)
