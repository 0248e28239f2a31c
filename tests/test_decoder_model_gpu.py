"""An installed model on the GPU: the output's forms under mixed precision, a Trainer's steps, two threads on one model, and a
process whose first call is captured."""
import copy
import os
import subprocess
import sys
import threading

import pytest
import torch

from test_decoder_gpu import BF16, F16, F32, HALF, whisper
from test_decoder_model_cpu import batch, stock_model, trainer_losses

pytestmark = pytest.mark.gpu


def inputs(seed=0, length=17):
    g = torch.Generator(device="cuda").manual_seed(seed)
    labels = torch.randint(0, 600, (3, length), generator=g, device="cuda")
    labels[0, 9:] = -100
    labels[2, 3:] = -100
    return {"input_features": torch.randn(3, 8, 40, generator=g, device="cuda"), "labels": labels}


def pair():
    from wfe_amd import decoder
    stock = whisper().train()
    return stock, decoder.install(copy.deepcopy(stock))


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
def test_mixed_precision_outputs_have_no_logits(dtype):
    operations = pytest.importorskip("accelerate.utils.operations")
    stock, model = pair()
    given = inputs()
    with torch.autocast("cuda", dtype=dtype):
        want = stock(**given)
        out = operations.convert_outputs_to_fp32(model.forward)(**given)
        plain = model(**given)
    for o in (out, plain):
        assert o.logits is None and "logits" not in o and o[0] is o.loss and o["loss"] is o.loss
        assert list(o.keys()) == [k for k in want.keys() if k != "logits"]
    assert torch.equal(out.loss, plain.loss)
    # the decoder in `dtype` on both sides; the stock logits (under 8 in size here) are rounded to it, ours are not
    assert float(want.logits.abs().max()) < 8
    assert abs(float(out.loss.detach()) - float(want.loss.detach())) <= 2 * 8 * HALF[dtype]


@pytest.mark.parametrize("how", [{}, {"fp16": True}, {"bf16": True}], ids=["f32", "fp16", "bf16"])
def test_trainer_steps(how, tmp_path):
    """The Trainer's own path: outputs by key, GradScaler, clipping.  float32 steps follow the stock model's to rounding."""
    from wfe_amd import decoder
    stock = stock_model()
    model = decoder.install(copy.deepcopy(stock))
    (_, want), (_, got) = (trainer_losses(m, tmp_path, **how) for m in (stock, model))
    assert len(got) == 2
    if not how:
        assert got == pytest.approx(want, abs=1e-4)
        for (name, p), q in zip(stock.named_parameters(), model.parameters()):
            assert torch.allclose(p, q, atol=2e-3), name       # (Adam: at most the learning rate a step, whatever the gradient)
    else:
        assert all(x == pytest.approx(y, abs=2 * 8 * HALF[F16 if "fp16" in how else BF16]) for x, y in zip(got, want))


def test_two_threads_train_and_score_on_one_model():
    stock, model = pair()
    cases = [inputs(0), inputs(1, 30)]
    tokens = {"input_features": cases[0]["input_features"], "decoder_input_ids": torch.full((3, 4), 601, device="cuda")}
    params = [p for p in model.parameters() if p.requires_grad]

    def train(i):
        loss = model(**cases[i]).loss
        return (loss.detach(), *torch.autograd.grad(loss, params, allow_unused=True))
    want = [train(0), train(1), (model(**tokens).logits,)]
    assert torch.equal(want[2][0], stock(**tokens).logits)
    got, errors = [[], [], []], []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(5):
                    got[i].append(train(i) if i < 2 else (model(**tokens).logits,))
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001 -- reported below
            errors.append(e)
    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for w, runs in zip(want, got):
        for run in runs:
            assert all(a is b is None or a.shape == b.shape for a, b in zip(w, run))
            assert torch.allclose(w[0], run[0], atol=1e-5)


def test_first_call_of_a_process_may_be_captured():
    """Nothing that a first call sets up (devices, kernels' attributes) disturbs a capture."""
    code = """
import torch
from wfe_amd import decoder as d
decoder_loaded = d._ext()
for dtype in (torch.bfloat16, torch.float16, torch.float32):
    h = torch.randn(300, 64, device="cuda").to(dtype).requires_grad_()
    w = (torch.randn(700, 64, device="cuda") / 8).to(dtype).requires_grad_()
    y = torch.randint(0, 700, (300,), device="cuda")
    def step():
        x = d.token_embedding(y, w)
        loss = d.linear_cross_entropy(h + x, w, y)
        return (loss.detach(), *torch.autograd.grad(loss, (h, w)))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        for a, b in zip(got, step()):
            assert torch.equal(a, b), dtype
print("same")
"""
    import wfe_amd
    package = os.path.dirname(list(wfe_amd.__path__)[0])
    done = subprocess.run([sys.executable, "-c", code], env={**os.environ, "PYTHONPATH": package}, capture_output=True,
                          text=True, timeout=100)
    assert done.returncode == 0 and done.stdout.strip().endswith("same"), done.stderr[-2000:]


def test_losses_may_be_added_to_in_place():
    stock, model = pair()
    given = inputs()
    out = model(**given)
    out.loss += 2.0
    out["loss"].backward()
    want = stock(**given)
    want.loss.backward()
    a, b = (m.get_output_embeddings().weight.grad for m in (stock, model))
    assert float((a - b).abs().max()) <= 1e-4 * float(a.abs().max()) + 1e-7
