"""The decoder's vocabulary operators (wfe_amd/decoder.py) against plain float64 formulas.

Tolerances are sums of what each step can lose, with u = 2^-24 (float32, half a step) and e the half step of the
16-bit type (bfloat16 2^-8, float16 2^-11):
  logits   products of 16-bit values are exact in float32 and of float32 values lose u each; dim additions lose u each:
           dz = (dim + 1) u max_{n,v} sum_k |h_nk W_vk|
  losses   2 dz, the exponential's argument times log2(e) rounded (|z| < 100: 100 * 1.44 * 2 u), sums over the vocabulary
           in chunks of at most 128 (128 u + joins), one logarithm
  dh       d rounded (e), its exponent (2 dz + 300 u), products summed in float32 (vocab u), then the output's rounding
  dW       the same over the rows, one more e where rows carry their own weights"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -149}
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def decoder():
    from wfe_amd import decoder as d
    return d


def make(rows, dim, vocab, dtype, seed=0, ignored=0.3, lean=6.0, ignore_index=-100):
    g = torch.Generator(device="cuda").manual_seed(seed)
    w = (torch.randn(vocab, dim, generator=g, device="cuda") / math.sqrt(dim)).to(dtype)
    shape = rows if isinstance(rows, tuple) else (rows,)
    y = torch.randint(0, vocab, shape, generator=g, device="cuda")
    h = torch.randn(*shape, dim, generator=g, device="cuda") + lean * torch.rand(*shape, 1, generator=g,
                                                                                 device="cuda") * w[y].float()
    drop = torch.rand(shape, generator=g, device="cuda") < ignored
    return h.to(dtype), w, torch.where(drop, ignore_index, y)


def oracle(h, w, y, reduction, upstream, ignore_index=-100):
    """losses, dh, dW in float64, and their tolerances apart from the output's own rounding."""
    dim, vocab = w.shape[1], w.shape[0]
    p_half = HALF[w.dtype]
    shape = y.shape
    y = y.reshape(-1)
    keep = torch.nonzero(y != ignore_index).flatten()
    hd, wd = h.reshape(-1, dim).double(), w.double()
    loss = torch.zeros(y.numel(), dtype=torch.float64, device=y.device)
    loss_tol = torch.zeros_like(loss)
    dh, dh_tol = torch.zeros_like(hd), torch.zeros_like(hd)
    dw, dw_tol = torch.zeros_like(wd), torch.zeros_like(wd)
    dz = 0.0
    parts = keep.split(1024) if keep.numel() else ()
    for part in parts:
        dz = max(dz, float((hd[part].abs() @ wd.abs().T).max()) * (dim + 1) * U)
    for part in parts:
        logp = torch.log_softmax(hd[part] @ wd.T, -1)
        loss[part] = -logp.gather(1, y[part][:, None].long())[:, 0]
        loss_tol[part] = 2 * dz + (300 + 128 + 300) * U + 4 * U * loss[part].abs() + 16 * U
        d = logp.exp()
        d[torch.arange(part.numel(), device=y.device), y[part].long()] -= 1
        if reduction == "none":
            g = upstream.reshape(-1).double()[part]
        else:
            g = upstream.double().reshape(1) / (keep.numel() if reduction == "mean" else 1)
            g = g.expand(part.numel())
        lost = p_half + 2 * dz + 300 * U
        # (the label's d = p - 1 cancels: p's error stays as it is)
        size = d.abs() * (lost + vocab * U) + torch.where(d < 0, 1.0 + d, d) * (2 * dz + 400 * U)
        dh[part] = (d * g[:, None]) @ wd
        dh_tol[part] = (size * g.abs()[:, None]) @ wd.abs() + 4 * U * dh[part].abs()
        dw += (d * g[:, None]).T.contiguous() @ hd[part]
        size = size + d.abs() * (y.numel() * U + (p_half if reduction == "none" else 0))
        dw_tol += (size * g.abs()[:, None]).T.contiguous() @ hd[part].abs()
    count = keep.numel()
    if reduction == "none":
        return loss.view(shape), loss_tol.view(shape), dh.view(h.shape), dh_tol.view(h.shape), dw, dw_tol
    total = loss.sum() / (count if reduction == "mean" else 1)
    tol = loss_tol.sum() / max(count if reduction == "mean" else 1, 1) + U * total.abs()
    return total, tol, dh.view(h.shape), dh_tol.view(h.shape), dw, dw_tol


def close(got, want, tol, what):
    bound = tol + HALF[got.dtype] * want.abs() + TINY[got.dtype]
    err = (got.double() - want).abs()
    bad = ~(err <= bound)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((err / bound).max()):.3f} of the bound"


def check(h, w, y, reduction, grads=(True, True), ignore_index=-100):
    d = decoder()
    h = h.detach().requires_grad_(grads[0])
    w = w.detach().requires_grad_(grads[1])
    loss = d.linear_cross_entropy(h, w, y, reduction=reduction, ignore_index=ignore_index)
    assert loss.dtype == torch.float32 and loss.shape == (y.shape if reduction == "none" else ())
    up = torch.rand(loss.shape, generator=torch.Generator(device="cuda").manual_seed(5), device="cuda") + 0.5
    want = oracle(h.detach(), w.detach(), y, reduction, up, ignore_index)
    close(loss.detach(), want[0], want[1], "loss")
    wanted = [t for t, need in zip((h, w), grads) if need]
    if wanted:
        got = torch.autograd.grad(loss, wanted, up)
        for g, t, at in zip(got, wanted, [i for i, need in zip((2, 4), grads) if need]):
            assert g.dtype == t.dtype and g.shape == t.shape
            close(g, want[at], want[at + 1], "dh" if at == 2 else "dW")
    return loss


SIZES = [  # rows, dim, vocab
    (1, 1, 1), (1, 64, 2), (2, 8, 127), (3, 250, 128), (16, 384, 129), (17, 96, 1000), (64, 72, 257), (65, 33, 255),
    (127, 128, 256), (128, 192, 5003), (129, 320, 300), (300, 40, 777), (513, 65, 129), ((3, 41), 1280, 515)]


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,dim,vocab", SIZES, ids=[str(s).replace(" ", "") for s in SIZES])
def test_loss_and_gradients(rows, dim, vocab, dtype):
    h, w, y = make(rows, dim, vocab, dtype)
    for reduction in ("mean", "sum", "none"):
        if reduction == "mean" and not bool((y != -100).any()):
            continue
        check(h, w, y, reduction)


@pytest.mark.parametrize("rows", [1, 5, 16, 33, 64, 100, 200, 257, 700])
def test_whisper_vocabulary(rows):
    """The real vocabulary sizes, few rows and many; only one gradient wanted."""
    for vocab, dim, dtype in ((51865, 384, BF16), (51866, 1280, F16)):
        h, w, y = make(rows, dim, vocab, dtype, seed=rows)
        check(h, w, y, "none", grads=(False, False))
        check(h, w, y, "sum", grads=(True, False))
        check(h, w, y, "none", grads=(False, True))


def test_several_pieces_of_the_vocabulary():
    h, w, y = make(40000, 32, 7001, BF16, ignored=0.1)
    check(h, w, y, "mean")
    h, w, y = make(20000, 40, 5003, F32, ignored=0.5)
    check(h, w, y, "none")


@pytest.mark.parametrize("rows,dim,vocab,dtype,reduction", [
    (9001, 1280, 16001, BF16, "mean"), (9000, 1273, 15999, F16, "none"), (5003, 640, 14003, F32, "sum")], ids=str)
def test_pieces_of_a_wide_model(rows, dim, vocab, dtype, reduction):
    """Many rows and a wide model: d in three pieces of the vocabulary, the last of them ragged."""
    h, w, y = make(rows, dim, vocab, dtype, ignored=0.05)
    check(h, w, y, reduction)
    check(h, w, y, reduction, grads=(True, False))


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows", [9, 70, 300])
@pytest.mark.parametrize("dim", [8, 40, 72, 104, 136, 1224])
def test_widths_that_end_inside_a_tile(rows, dim, dtype):
    """Rows of W are read in place up to their end: what lies between them does not matter, nor does an infinity in their
    last values."""
    h, w, y = make(rows, dim, 391, dtype, seed=dim, ignored=0.1)
    base = torch.full((391, dim + 8), float("nan"), device="cuda", dtype=dtype)
    base[:, :dim] = w
    gaps = base[:, :dim]
    want = check(h, w, y, "none")
    got = check(h, gaps, y, "none")
    assert torch.equal(want, got)
    y[y == 17] = 18
    h[:, -1] = 1.0
    z = h.double() @ w.double().T
    z[:, 17] = -float("inf")
    gaps[17, -1] = -float("inf")
    loss = decoder().linear_cross_entropy(h, gaps, y, reduction="none")
    keep = y != -100
    ref = torch.logsumexp(z, 1) - z.gather(1, y.clamp_min(0)[:, None])[:, 0]
    assert float((loss.double() - ref)[keep].abs().max()) < 2e-5 * max(1.0, float(ref.max()))


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows", [20, 300])
def test_weights_of_rows_far_apart(rows, dtype):
    """Upstream gradients of zero, of either sign, tiny all together and of many sizes: every row of dh is exact relative to
    itself, dW to its largest rows."""
    d = decoder()
    h, w, y = make(rows, 104, 391, dtype, seed=rows, ignored=0.1)
    g = torch.Generator(device="cuda").manual_seed(rows)
    sign = torch.where(torch.rand(rows, generator=g, device="cuda") < 0.5, -1.0, 1.0)
    sizes = torch.rand(rows, generator=g, device="cuda") + 0.5
    far = sizes * 2.0 ** torch.randint(-12, 1, (rows,), generator=g, device="cuda").float()
    some = torch.where(torch.arange(rows, device="cuda") % 3 == 0, 0.0, sizes)
    for up in (sign * sizes * 2.0 ** -20, sign * far, some * 2.0 ** -10, some * 2.0 ** 10, torch.zeros_like(some)):
        if dtype == F16 and float(up.abs().max()) > 100:
            continue                                           # (its gradients leave the type's range)
        a, b = h.clone().requires_grad_(), w.float().requires_grad_()
        with torch.autocast("cuda", dtype=dtype, enabled=dtype != F32):
            loss = d.linear_cross_entropy(a.float(), b, y, reduction="none")
        ga, gb = torch.autograd.grad(loss, (a, b), up)
        want = oracle(h, w, y, "none", up)
        tiny = 2.0 ** -24 * float(up.abs().max()) * want[4].shape[1] if dtype == F16 else 0.0
        close(ga.float() if dtype != F16 else ga, want[2], want[3] + HALF[dtype] * want[2].abs() + TINY[dtype], "dh")
        close(gb, want[4], want[5] + tiny * float(h.abs().max()), "dW")


def test_views_strides_and_index_types():
    h, w, y = make((4, 23), 128, 1003, BF16, seed=3)
    g = torch.Generator(device="cuda").manual_seed(1)
    base = torch.randn(4, 30, 160, generator=g, device="cuda").to(BF16)
    base[:, 3:26, :128] = h
    view = base[:, 3:26, :128]
    assert not view.is_contiguous()
    big = torch.randn(1003, 200, generator=g, device="cuda").to(BF16)
    for at in (0, 8, 3):                                   # in place, in place, misaligned: copied
        big[:, at:at + 128] = w
        check(view, big[:, at:at + 128], y.to(torch.int32), "mean")
    check(h.transpose(0, 1), w, y.T, "none")               # rows in another order
    check(h.permute(0, 1, 2)[..., ::2], w[:, ::2], y, "sum")      # inner step of 2
    check(h[:1, :1].expand(4, 23, 128), w, y, "none")      # every row the same memory
    deep = torch.randn(2, 3, 2, 5, 128, generator=g, device="cuda").to(BF16)[:, 1:, :, ::2]
    yy = torch.randint(0, 1003, deep.shape[:-1], generator=g, device="cuda")
    check(deep, w, yy, "none")
    check(h[0, 0], w, y[0, 1], "sum")                      # one token without dimensions


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=["bf16", "f16", "f32"])
def test_ignored_rows_may_hold_anything(dtype):
    h, w, y = make(150, 64, 333, dtype, ignored=0.5)
    clean = [t.clone() for t in (h, w, y)]
    drop = y == -100
    fill = torch.tensor([float("nan"), float("inf"), -float("inf"), torch.finfo(dtype).min], device="cuda").to(dtype)
    h[drop] = fill[torch.arange(int(drop.sum()), device="cuda") % 4][:, None]
    for reduction in ("mean", "none"):
        up = torch.ones((150,) if reduction == "none" else (), device="cuda")
        out = []
        for hh in (clean[0], h):
            a, b = hh.clone().requires_grad_(), w.clone().requires_grad_()
            loss = decoder().linear_cross_entropy(a, b, y, reduction=reduction)
            if reduction == "none":
                up[drop] = float("nan")                    # what flows into an ignored row's loss does not matter
            out.append((loss, *torch.autograd.grad(loss, (a, b), up)))
        for x, z in zip(*out):
            assert torch.equal(x, z) and bool(torch.isfinite(x).all())
        assert not bool(out[1][1][drop].any())


def test_every_row_ignored_and_no_rows():
    h, w, _ = make(40, 64, 100, BF16)
    for rows in (40, 0):
        y = torch.full((rows,), -100, device="cuda")
        for reduction in ("none", "sum", "mean"):
            a, b = h[:rows].clone().requires_grad_(), w.clone().requires_grad_()
            loss = decoder().linear_cross_entropy(a, b, y, reduction=reduction)
            if reduction == "mean":
                assert bool(torch.isnan(loss))
            else:
                assert float(loss.sum()) == 0.0
            ga, gb = torch.autograd.grad(loss, (a, b), torch.ones_like(loss))
            assert not bool(ga.any()) and not bool(gb.any())


def test_ignore_index_inside_the_vocabulary_and_labels_outside():
    h, w, y = make(90, 64, 500, BF16, ignore_index=7)
    check(h, w, y, "mean", ignore_index=7)
    y[3] = 500
    y[11] = -5
    a = h.clone().requires_grad_()
    loss = decoder().linear_cross_entropy(a, w, y, ignore_index=7, reduction="none")
    bad = torch.zeros(90, dtype=torch.bool, device="cuda")
    bad[[3, 11]] = True
    assert torch.equal(torch.isnan(loss), bad)
    assert bool(torch.isnan(decoder().linear_cross_entropy(h, w, y, ignore_index=7)))
    grad, = torch.autograd.grad(loss.sum(), a)
    assert torch.equal(torch.isnan(grad).any(-1), bad)


def test_infinite_logits():
    """A logit of -inf has no probability; the label's own makes the loss inf; +inf makes it NaN, as the formula has it."""
    w = torch.zeros(300, 64, device="cuda", dtype=BF16)
    w[:, 0] = torch.linspace(-3, 3, 300, device="cuda").to(BF16)
    w[5, 1] = -float("inf")
    h = torch.zeros(3, 64, device="cuda", dtype=BF16)
    h[:, 0] = 1
    h[:, 1] = 1
    y = torch.tensor([0, 5, 299], device="cuda")
    loss = decoder().linear_cross_entropy(h, w, y, reduction="none")
    z = w[:, 0].double()
    z[5] = -float("inf")
    want = torch.logsumexp(z, 0) - z[y]
    assert float(loss[1]) == float("inf")
    assert torch.allclose(loss[[0, 2]].double(), want[[0, 2]], rtol=1e-5)
    w[5, 1] = float("inf")
    assert bool(torch.isnan(decoder().linear_cross_entropy(h, w, y, reduction="none")).all())
    # a whole tile of -inf
    w[5, 1] = 0
    w[0:256, 1] = -float("inf")
    loss = decoder().linear_cross_entropy(h, w, y, reduction="none")
    want = torch.logsumexp(w[256:, 0].double(), 0) - z[299]
    assert abs(float(loss[2]) - float(want)) < 1e-5 and float(loss[0]) == float("inf")


def test_confident_rows_keep_their_small_gradients():
    """Labels with probability 1 - 1e-6: float32 logits give the loss to dz, not to the type of the inputs."""
    h, w, y = make(64, 256, 2000, F32, ignored=0.0)
    h = torch.randn(64, 256, device="cuda") * 0.1 + 26 * w[y]
    check(h, w, y, "sum")


def test_gradient_against_differences():
    """Directional differences of the loss itself.  Step s: error of the difference quotient is s^2 / 6 |f'''| (f''' of
    a log-sum-exp along a direction u is at most 6 max|u . W|^3 per row) plus the losses' own errors over s."""
    h, w, y = make(37, 48, 211, F32, seed=9)
    g = torch.Generator(device="cuda").manual_seed(2)
    a, b = h.clone().requires_grad_(), w.clone().requires_grad_()
    loss = decoder().linear_cross_entropy(a, b, y, reduction="sum")
    ga, gb = torch.autograd.grad(loss, (a, b))
    s = 2.0 ** -5
    kept = int((y != -100).sum())
    for which in ("h", "w"):
        u = torch.randn((h if which == "h" else w).shape, generator=g, device="cuda")
        u /= u.norm()
        f = [decoder().linear_cross_entropy(h + k * s * u if which == "h" else h, w + k * s * u if which == "w" else w,
                                            y, reduction="sum").double() for k in (1, -1)]
        quotient = float((f[0] - f[1]) / (2 * s))
        slope = float((u.double() * (ga if which == "h" else gb).double()).sum())
        reach = float((u @ w.T if which == "h" else h @ u.T).abs().max())
        dz = float((h.abs() @ w.abs().T).max()) * 49 * U
        bound = s * s * kept * reach ** 3 + kept * (2 * dz + 800 * U) / s + 1e-4 * abs(slope)
        assert abs(quotient - slope) <= bound, (which, quotient, slope, bound)


def test_autocast_casts_as_linear_does():
    h, w, y = make((3, 50), 128, 700, F32)
    for dtype in (BF16, F16):
        a, b = h.clone().requires_grad_(), w.clone().requires_grad_()
        with torch.autocast("cuda", dtype=dtype):
            loss = decoder().linear_cross_entropy(a, b, y)
        ga, gb = torch.autograd.grad(loss, (a, b))
        assert ga.dtype == gb.dtype == torch.float32
        want = oracle(h.to(dtype), w.to(dtype), y, "mean", torch.ones((), device="cuda"))
        close(loss.detach(), want[0], want[1], "loss")
        close(ga, want[2], want[3], "dh")
        close(gb, want[4], want[5], "dW")
        half = h.to(dtype).requires_grad_()                # a hidden state that is 16-bit already, W's master in 32
        with torch.autocast("cuda", dtype=dtype):
            loss = decoder().linear_cross_entropy(half, b, y)
        ga, gb = torch.autograd.grad(loss, (half, b))
        assert ga.dtype == dtype and gb.dtype == torch.float32
        close(ga, want[2], want[3], "dh")
        close(gb, want[4], want[5], "dW")


def _step(h, w, y, ids):
    d = decoder()
    emb = d.token_embedding(ids, w, scale=0.5, padding_idx=3)
    loss = d.linear_cross_entropy(h + emb, w, y)
    return (loss.detach(), *torch.autograd.grad(loss, (h, w)))


def test_capture_beside_a_living_eager_graph_is_refused():
    d = decoder()
    h, w, y = make(20, 64, 300, BF16)
    w = w.requires_grad_()
    for call in (lambda: d.linear_cross_entropy(h, w, y), lambda: d.token_embedding(y.clamp_min(0), w)):
        alive = call()
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="alive"), torch.cuda.graph(graph):
            call()
        del alive
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
            grad, = torch.autograd.grad(out, w, torch.ones_like(out))
            del out
        graph.replay()
        torch.cuda.synchronize()
        again = call()
        assert torch.equal(grad, torch.autograd.grad(again, w, torch.ones_like(again))[0])
        del again


def test_together_in_a_captured_graph_and_on_a_side_stream():
    """Embedding into loss over one matrix: eager, on another stream, and captured and replayed with new inputs between
    the replays, with eager work beside it; the same bits each time."""
    h, w, y = make((4, 60), 192, 3001, BF16)
    h, w = h.requires_grad_(), w.requires_grad_()
    ids = torch.where(y == -100, 3, y)
    want = _step(h, w, y, ids)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = _step(h, w, y, ids)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(want, again):
        assert torch.equal(a, b)
    del again
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _step(h, w, y, ids)
    for seed in range(4):
        h2, _, y2 = make((4, 60), 192, 3001, BF16, seed=seed, ignored=(0.0, 0.9, 1.0, 0.3)[seed])
        with torch.no_grad():
            h.copy_(h2)
            y.copy_(y2)
            ids.copy_(torch.where(y2 == -100, 3, y2))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        for a, b in zip(got, _step(h, w, y, ids)):
            assert torch.equal(a, b) or (seed == 2 and bool(torch.isnan(a).all()) and bool(torch.isnan(b).all()))


def test_two_calls_at_once_share_nothing():
    cases = [make(500, 128, 3000, BF16, seed=s) for s in range(2)]
    want = [decoder().linear_cross_entropy(*c, reduction="none") for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, (s, c) in enumerate(zip(streams, cases)):
            with torch.cuda.stream(s):
                got[i].append(decoder().linear_cross_entropy(*c, reduction="none"))
    torch.cuda.synchronize()
    for w, gs in zip(want, got):
        assert all(torch.equal(w, g) for g in gs)


# rows around every strip and tile edge; vocabularies around the tiles'
@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows", [31, 32, 33, 63, 64, 65, 96, 97, 128, 160, 192, 255, 256, 257, 320, 321, 384, 385, 512])
def test_every_row_kept_at_tile_edges(rows, dtype):
    for vocab, dim in ((255, 64), (512, 192), (769, 96)):
        h, w, y = make(rows, dim, vocab, dtype, seed=rows, ignored=0.0)
        check(h, w, y, "sum")
        check(h, w, y, "none")


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=["bf16", "f16", "f32"])
def test_infinite_weights(dtype):
    """Products with infinities follow float32: -inf logits drop out of the softmax, other rows stay exact."""
    h, w, y = make(40, 64, 500, dtype, ignored=0.0)
    y[y == 17] = 18
    h[:, 0] = 1.0
    clean = w.clone()
    w[17, 0] = -float("inf")
    loss = decoder().linear_cross_entropy(h, w, y, reduction="none")
    z = h.double() @ clean.double().T
    z[:, 17] = -float("inf")
    want = torch.logsumexp(z, 1) - z.gather(1, y[:, None])[:, 0]
    assert float((loss.double() - want).abs().max()) < 2e-5 * max(1.0, float(want.max()))
    w[17, 0] = float("inf")
    assert bool(torch.isnan(decoder().linear_cross_entropy(h, w, y, reduction="none")).all())


def test_differentiable_once_and_again_on_the_same_graph():
    d = decoder()
    h, w, y = make(70, 64, 300, F32)
    ids = y.clamp_min(0)
    a, b = h.requires_grad_(), w.requires_grad_()
    for out, of in ((d.linear_cross_entropy(a, b, y), (a, b)), (d.token_embedding(ids, b).sum(), (b,))):
        first = torch.autograd.grad(out, of, retain_graph=True)
        again = torch.autograd.grad(out, of, create_graph=True)
        for x, z in zip(first, again):
            assert torch.equal(x, z)
        with pytest.raises(RuntimeError):                              # no path from the gradient to its input
            torch.autograd.grad(again[-1].sum(), of, retain_graph=True)
        with pytest.raises(RuntimeError, match="differentiated once"):
            again[-1].sum().backward()


def test_hidden_off_its_alignment_and_weights_with_strides():
    g = torch.Generator(device="cuda").manual_seed(6)
    for dtype in (BF16, F32):
        base = torch.randn(50, 200, generator=g, device="cuda").to(dtype)
        w = (torch.randn(333, 130, generator=g, device="cuda") / 11).to(dtype)
        y = torch.randint(0, 333, (50,), generator=g, device="cuda")
        check(base[:, 1:129], w[:, 1:129], y, "mean")                 # both off 16 bytes
        check(base[:, 8:136], w[:, :128], y, "none")                  # rows of W 130 apart
        check(base[:, 8:72].flip(0), w[1:2, :64].expand(333, 64), y, "sum", grads=(True, False))
        check(base[:, 8:136][::2], w[::3, :128], y[::2] % 111, "mean")


def test_two_captured_graphs_share_a_pool_and_threads_share_nothing():
    import threading
    d = decoder()
    cases = [[t.requires_grad_() if t.is_floating_point() else t for t in make(n, 128, 1111, BF16, seed=n)] for n in (90, 400)]

    def step(h, w, y):
        loss = d.linear_cross_entropy(h, w, y)
        return (loss.detach(), *torch.autograd.grad(loss, (h, w)))
    want = [[t.clone() for t in step(*c)] for c in cases]
    graphs = [torch.cuda.CUDAGraph() for _ in cases]
    outs = []
    for i, (graph, c) in enumerate(zip(graphs, cases)):
        with torch.cuda.graph(graph, pool=graphs[0].pool() if i else None):
            outs.append(step(*c))
    for i in (0, 1, 1, 0, 1):
        graphs[i].replay()
        torch.cuda.synchronize()
        for a, b in zip(outs[i], want[i]):
            assert torch.equal(a, b)
    got, errors = [None, None], []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(8):
                    got[i] = step(*cases[i])
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001 -- reported below
            errors.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for g, w in zip(got, want):
        assert all(torch.equal(a, b) for a, b in zip(g, w))


def test_offsets_past_32_bits():
    """W of 4.5 GB and hidden states of 4.5 GB: addresses behind 2^32 bytes; spot checks against float64."""
    d = decoder()
    vocab, dim = 2_200_000, 1024
    w = torch.empty(vocab, dim, device="cuda", dtype=BF16).normal_(0, 0.03)
    y = torch.tensor([vocab - 1, 5, vocab // 2, vocab - 300, -100], device="cuda")
    h = torch.randn(5, dim, device="cuda").to(BF16)
    a, b = h.clone().requires_grad_(), w.requires_grad_()
    loss = d.linear_cross_entropy(a, b, y, reduction="sum")
    ga, gb = torch.autograd.grad(loss, (a, b))
    z = torch.cat([h[:4].double() @ part.T.double() for part in w.detach().split(1 << 18)], dim=1)
    logp = torch.log_softmax(z, 1)
    want = -logp.gather(1, y[:4, None]).sum()
    assert abs(float(loss) - float(want)) < 1e-4 * float(want)
    p = logp.exp()
    p[torch.arange(4), y[:4]] -= 1
    for rows in (slice(vocab - 400, vocab), slice(0, 300), slice(1 << 21, (1 << 21) + 9)):
        ref = p[:, rows].T @ h[:4].double()
        assert float((gb[rows].double() - ref).abs().max()) < 0.02 * float(ref.abs().max()) + 1e-9
    ref = sum(p[:, at:at + part.shape[0]] @ part.double() for at, part in
              zip(range(0, vocab, 1 << 18), w.detach().split(1 << 18)))
    assert float((ga[:4].double() - ref).abs().max()) < 0.02 * float(ref.abs().max())
    ids = torch.tensor([vocab - 1, 0, vocab - 2, vocab - 1], device="cuda")
    out = d.token_embedding(ids, b)
    assert torch.equal(out, w.detach()[ids])
    up = torch.randn(4, dim, device="cuda").to(BF16)
    grad, = torch.autograd.grad(out, b, up)
    assert torch.equal(grad[vocab - 2], up[2]) and torch.equal(grad[vocab - 1], (up[0].float() + up[3].float()).to(BF16))
    assert not bool(grad[1:vocab - 2].any())
    del w, b, gb, grad, z, logp, p, out
    rows, vocab = 2_200_000, 257
    h = torch.empty(rows, dim, device="cuda", dtype=BF16).normal_()
    w = torch.randn(vocab, dim, device="cuda").mul_(0.03).to(BF16)
    y = torch.randint(0, vocab, (rows,), device="cuda")
    y[::7] = -100
    a, b = h.requires_grad_(), w.requires_grad_()
    loss = d.linear_cross_entropy(a, b, y, reduction="none")
    ga, = torch.autograd.grad(loss, a, torch.ones_like(loss))
    for part in (slice(0, 500), slice(rows - 700, rows), slice(1 << 21, (1 << 21) + 100)):
        keep = y[part] != -100
        z = h.detach()[part].double() @ w.detach().double().T
        logp = torch.log_softmax(z, 1)
        t = y[part].clamp_min(0)
        ref = torch.where(keep, -logp.gather(1, t[:, None])[:, 0], 0.0)
        assert float((loss[part].double() - ref).abs().max()) < 1e-3
        p = logp.exp()
        p[torch.arange(t.numel()), t] -= 1
        ref = (p * keep[:, None]) @ w.detach().double()
        assert float((ga[part].double() - ref).abs().max()) < 0.02 * float(ref.abs().max())
    del ga, loss
    up = h.detach()
    ids = y.clamp_min(0)
    grad, = torch.autograd.grad(d.token_embedding(ids, b), b, up)
    ref = torch.zeros(vocab, dim, device="cuda", dtype=torch.float64)
    for part, i in zip(up.split(1 << 18), ids.split(1 << 18)):
        ref.index_add_(0, i, part.double())
    assert float((grad.double() - ref).abs().max()) < 0.01 * float(ref.abs().max())


# ---- embedding ---------------------------------------------------------------------------------------------
def tokens(rows, vocab, seed=0, heavy=0.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    ids = torch.randint(0, vocab, rows if isinstance(rows, tuple) else (rows,), generator=g, device="cuda")
    if heavy:
        ids = torch.where(torch.rand(ids.shape, generator=g, device="cuda") < heavy, vocab // 2, ids)
    return ids


def embed_oracle(ids, up, vocab, scale, padding):
    """dW in float64 and its tolerance: a float32 sum of c terms, one product with the scale."""
    dim = up.shape[-1]
    flat, up = ids.reshape(-1).long(), up.reshape(-1, dim).double()
    ok = (flat >= 0) & (flat < vocab)
    if padding is not None:
        ok &= flat != padding
    flat, up = flat[ok], up[ok]
    grad = torch.zeros(vocab, dim, dtype=torch.float64, device=ids.device).index_add_(0, flat, up) * scale
    size = torch.zeros(vocab, dim, dtype=torch.float64, device=ids.device).index_add_(0, flat, up.abs()) * abs(scale)
    count = torch.bincount(flat, minlength=vocab).double()
    return grad, size * (count[:, None] + 2) * U


EMBED = [  # rows, vocab, dim, heavy
    (1, 1, 1, 0), (5, 300, 7, 0), (64, 51865, 384, 0), ((16, 48), 51866, 1280, 0.4), (1000, 257, 24, 0), (3000, 50, 65, 0),
    (70, 256, 128, 1.0), (5000, 1000, 40, 0.9), (29000, 5003, 72, 0.3), (129, 513, 1, 0)]


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,vocab,dim,heavy", EMBED, ids=[str(s[:3]).replace(" ", "") for s in EMBED])
def test_embedding_and_its_gradient(rows, vocab, dim, heavy, dtype):
    d = decoder()
    ids = tokens(rows, vocab, heavy=heavy)
    g = torch.Generator(device="cuda").manual_seed(4)
    w = torch.randn(vocab, dim, generator=g, device="cuda").to(dtype).requires_grad_()
    for scale, padding in ((1.0, None), (math.sqrt(dim), int(ids.reshape(-1)[0]))):
        out = d.token_embedding(ids, w, scale=scale, padding_idx=padding)
        exact = (w.detach().float() * torch.tensor(scale, dtype=torch.float32)).to(dtype)[ids]
        assert torch.equal(out, exact)
        up = torch.randn(out.shape, generator=g, device="cuda").to(dtype)
        got, = torch.autograd.grad(out, w, up)
        want, tol = embed_oracle(ids, up, vocab, float(torch.tensor(scale, dtype=torch.float32)), padding)
        close(got, want, tol, "dW")
        again, = torch.autograd.grad(d.token_embedding(ids, w, scale=scale, padding_idx=padding), w, up)
        assert torch.equal(got, again)


def test_embedding_strides_types_and_bad_ids():
    d = decoder()
    g = torch.Generator(device="cuda").manual_seed(8)
    big = torch.randn(500, 100, generator=g, device="cuda").to(BF16)
    ids = tokens((6, 20), 500)
    ids[0, 0], ids[1, 2], ids[2, 2] = -1, 500, 2 ** 40
    bad = torch.zeros_like(ids, dtype=torch.bool)
    bad[0, 0] = bad[1, 2] = bad[2, 2] = True
    for w in (big[:, :64], big[:, 3:70], big[:, ::3], big[::2].T.contiguous().T[:250].repeat(2, 1)):
        w = w.detach().requires_grad_()
        out = d.token_embedding(ids, w, padding_idx=-1)
        assert torch.equal(torch.isnan(out).any(-1), bad)
        assert torch.equal(out[~bad], w.detach()[ids[~bad]])
        up = torch.randn(20, 6, w.shape[1] + 5, generator=g, device="cuda").to(BF16).transpose(0, 1)[..., :w.shape[1]]
        for grad in (up, up[:1, :1].expand(out.shape), up[:, :1].expand(out.shape),
                     torch.ones((), device="cuda", dtype=BF16).expand(out.shape)):
            got, = torch.autograd.grad(out, w, grad, retain_graph=True)
            want, tol = embed_oracle(ids, grad, 500, 1.0, 499)
            close(got, want, tol, "dW")
    small = tokens((3, 9), 500).to(torch.int32)[:, ::2]
    assert torch.equal(d.token_embedding(small, big), big[small.long()])
    none = torch.zeros((0, 4), dtype=torch.int64, device="cuda")
    w = big.clone().requires_grad_()
    out = d.token_embedding(none, w)
    assert out.shape == (0, 4, 100)
    assert not bool(torch.autograd.grad(out, w, torch.zeros_like(out))[0].any())


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows", [1023, 1024, 1025, 2309])
@pytest.mark.parametrize("dim", [7, 64, 1288])
def test_embedding_gradient_with_bad_ids_and_strides(rows, dim, dtype):
    """Ids out of range, padding, a common token, upstream gradients that are strided or the same for every token."""
    d = decoder()
    g = torch.Generator(device="cuda").manual_seed(rows + dim)
    vocab = 1003
    ids = tokens(rows, vocab, heavy=0.4)
    ids[3], ids[700], ids[-1] = -1, vocab, 2 ** 40
    padding = int(ids[0])
    w = torch.randn(vocab, dim, generator=g, device="cuda").to(dtype).requires_grad_()
    up = torch.randn(rows, dim + 9, generator=g, device="cuda").to(dtype)
    for grad in (up[:, :dim].contiguous(), up[:, 8:8 + dim], up[:, 1:1 + dim], up[:1, :dim].expand(rows, dim)):
        out = d.token_embedding(ids, w, padding_idx=padding)
        got, = torch.autograd.grad(out, w, grad)
        want, tol = embed_oracle(ids, grad, vocab, 1.0, padding)
        close(got, want, tol, "dW")


def test_embedding_gradient_leaves_masked_tokens_alone():
    """Gradients of padding tokens are dropped whatever they hold."""
    w = torch.randn(300, 64, device="cuda").requires_grad_()
    ids = tokens(200, 300)
    ids[::3] = 299
    up = torch.randn(200, 64, device="cuda")
    clean, = torch.autograd.grad(decoder().token_embedding(ids, w, padding_idx=299), w, up)
    up[::3] = float("nan")
    up[3] = float("inf")
    got, = torch.autograd.grad(decoder().token_embedding(ids, w, padding_idx=299), w, up)
    assert torch.equal(got, clean)


# ---- in a model ----------------------------------------------------------------------------------------------
def whisper(vocab=603, d_model=64):
    from transformers import WhisperConfig, WhisperForConditionalGeneration
    torch.manual_seed(0)
    cfg = WhisperConfig(vocab_size=vocab, num_mel_bins=8, d_model=d_model, encoder_layers=1, decoder_layers=2,
                        encoder_attention_heads=2, decoder_attention_heads=2, encoder_ffn_dim=96, decoder_ffn_dim=96,
                        max_source_positions=20, max_target_positions=32, pad_token_id=600, bos_token_id=600,
                        eos_token_id=600, decoder_start_token_id=601, dropout=0.0)
    return WhisperForConditionalGeneration(cfg).cuda()


def test_whisper_training_step_on_the_operators():
    """Loss and every gradient (the tied vocabulary matrix's among them) of a float32 model with and without the
    operators; evaluation and generation stay as they were."""
    import copy
    d = decoder()
    stock = whisper().train()
    model = copy.deepcopy(stock)
    assert d.install(model) is model and d.install(model) is model
    feats = torch.randn(3, 8, 40, device="cuda")
    labels = torch.randint(0, 600, (3, 17), device="cuda")
    labels[0, 9:] = -100
    labels[2, 3:] = -100
    outs = [m(input_features=feats, labels=labels) for m in (stock, model)]
    assert outs[0].logits is not None and outs[1].logits is None
    assert abs(float(outs[0].loss) - float(outs[1].loss)) < 1e-5
    for o in outs:
        o.loss.backward()
    for (name, p), q in zip(stock.named_parameters(), model.parameters()):
        assert (p.grad is None) == (q.grad is None), name
        if p.grad is not None:
            # float32 on both sides, sums in another order over at most 603 x 51 terms
            assert float((p.grad - q.grad).abs().max()) <= 1e-4 * float(p.grad.abs().max()) + 1e-7, name
    with torch.autocast("cuda", dtype=BF16):
        mixed = model(input_features=feats, labels=labels).loss
    mixed.backward()
    assert abs(float(mixed) - float(outs[0].loss)) < 0.05
    twin = copy.deepcopy(model)
    with torch.no_grad():
        twin.get_output_embeddings().weight.mul_(0.0)
    assert abs(float(twin(input_features=feats, labels=labels).loss) - math.log(603)) < 1e-5   # its own weights
    stock.eval(), model.eval()
    a, b = (m(input_features=feats, labels=labels) for m in (stock, model))
    assert torch.equal(a.logits, b.logits) and torch.equal(a.loss, b.loss)
    with torch.no_grad():
        ids = [m.generate(feats, max_new_tokens=5, do_sample=False) for m in (stock, model)]
    assert torch.equal(*ids)
    frugal = d.install(copy.deepcopy(stock), logits_in_eval=False)
    out = frugal(input_features=feats, labels=labels)
    assert out.logits is None and abs(float(out.loss) - float(a.loss)) < 1e-5
