"""The model path of the decoder operators (decoder.install) without a GPU: the two operators' places are taken by their
formulas in torch, everything around them is the code that runs on one."""
import pytest
import torch
import torch.nn.functional as F
import torch.nn.utils.parametrize

from wfe_amd import decoder


@pytest.fixture
def plain(monkeypatch):
    """The operators as formulas, for tensors on the CPU."""
    def loss(hidden, weight, labels, ignore_index=-100, reduction="mean"):
        assert hidden.shape[:-1] == labels.shape and hidden.shape[-1] == weight.shape[1]
        return F.cross_entropy((hidden @ weight.T).float().flatten(0, -2), labels.flatten(), ignore_index=ignore_index,
                               reduction=reduction)

    def embedding(ids, weight, scale=1.0, padding_idx=None):
        return scale * F.embedding(ids, weight, padding_idx)
    monkeypatch.setattr(decoder, "_fits", lambda weight: True)
    monkeypatch.setattr(decoder, "linear_cross_entropy", loss)
    monkeypatch.setattr(decoder, "token_embedding", embedding)


def stock_model():
    from transformers import WhisperConfig, WhisperForConditionalGeneration
    torch.manual_seed(0)
    cfg = WhisperConfig(vocab_size=103, num_mel_bins=8, d_model=16, encoder_layers=1, decoder_layers=1,
                        encoder_attention_heads=2, decoder_attention_heads=2, encoder_ffn_dim=16, decoder_ffn_dim=16,
                        max_source_positions=10, max_target_positions=8, pad_token_id=100, bos_token_id=100,
                        eos_token_id=100, decoder_start_token_id=101, dropout=0.0, attn_implementation="eager")
    return WhisperForConditionalGeneration(cfg).train()


def pair():
    """A model as it comes, and its twin with the operators."""
    import copy
    stock = stock_model()
    return stock, decoder.install(copy.deepcopy(stock))


def batch(seed=1):
    g = torch.Generator().manual_seed(seed)
    labels = torch.randint(0, 100, (2, 5), generator=g)
    labels[0, 3:] = -100
    return {"input_features": torch.randn(2, 8, 20, generator=g), "labels": labels}


def test_output_of_a_training_call_has_a_loss_and_no_logits_in_every_form(plain):
    stock, model = pair()
    more = {"output_hidden_states": True, "output_attentions": True}
    for extra in ({}, more, {"use_cache": False}):
        want, out = stock(**batch(), **extra), model(**batch(), **extra)
        assert type(out) is type(want)
        assert list(out.keys()) == [k for k in want.keys() if k != "logits"]       # the loss first, as ever
        assert "logits" not in out and out.logits is None
        assert out[0] is out.loss and out["loss"] is out.loss and out.to_tuple()[0] is out.loss
        assert torch.allclose(out.loss, want.loss, atol=1e-6)
        again = type(out)(**dict(out.items()))                                     # as wrappers rebuild it from its items
        assert again.logits is None and again.loss is out.loss
        for k in out.keys():
            if torch.is_tensor(out[k]):
                assert torch.allclose(out[k], want[k], atol=1e-6), k
        for k in ("decoder_hidden_states", "encoder_hidden_states", "decoder_attentions", "cross_attentions"):
            assert (getattr(out, k) is None) == (getattr(want, k) is None)
            for a, b in zip(getattr(out, k) or (), getattr(want, k) or ()):
                assert torch.equal(a, b)


def test_output_survives_the_conversion_of_mixed_precision_training(plain):
    operations = pytest.importorskip("accelerate.utils.operations")
    _, model = pair()
    model.forward = operations.convert_outputs_to_fp32(model.forward)
    out = model(**batch())
    assert out.logits is None and "logits" not in out and out["loss"].dtype == torch.float32


def test_evaluation_without_logits_predicts_nothing(plain):
    """What the Trainer takes for predictions are the output's items apart from the loss: none of them may pass for logits."""
    stock, model = pair()
    decoder.install(model, logits_in_eval=False)
    stock.eval(), model.eval()
    with torch.no_grad():
        want, out = stock(**batch()), model(**batch())
    assert "logits" not in out and not any(torch.is_tensor(v) and v.shape == (2, 5, 16) for v in out.values())
    assert torch.allclose(out.loss, want.loss, atol=1e-6)


def test_a_call_for_tuples_is_as_before(plain):
    stock, model = pair()
    a, b = (m(**batch(), return_dict=False) for m in (stock, model))
    assert isinstance(b, tuple) and len(a) == len(b) and torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


class Wrapped(torch.nn.Module):
    """An output projection with an adapter around it."""

    def __init__(self, inner):
        super().__init__()
        self.inner, self.more = inner, torch.nn.Linear(inner.in_features, inner.out_features, bias=False)

    @property
    def weight(self):
        return self.inner.weight

    def forward(self, x):
        return self.inner(x) + self.more(x)


def other_head(model, how):
    head = model.get_output_embeddings()
    torch.manual_seed(3)
    if how == "resized":
        model.resize_token_embeddings(110)
    elif how == "bias":
        model.set_output_embeddings(torch.nn.Linear(16, 103))
    elif how == "bias on the same":
        head.bias = torch.nn.Parameter(torch.randn(103))
    elif how == "adapter":
        model.set_output_embeddings(Wrapped(head))
    elif how == "forward replaced":
        head.forward = lambda x: torch.nn.functional.linear(x, 2 * head.weight)
    elif how == "hook":
        head.register_forward_hook(lambda module, args, out: 2 * out)
    elif how == "pre-hook":
        head.register_forward_pre_hook(lambda module, args: (2 * args[0],))
    elif how == "parametrized":
        class Doubled(torch.nn.Module):
            def forward(self, w):
                return 2 * w
        torch.nn.utils.parametrize.register_parametrization(head, "weight", Doubled())


@pytest.mark.parametrize("how", ["resized", "bias", "bias on the same", "adapter", "forward replaced", "hook", "pre-hook",
                                 "parametrized"])
def test_an_output_projection_changed_after_install_counts(plain, how):
    """What install found may be replaced, wrapped or hooked later on; the loss is that of the projection as it then is."""
    stock, model = pair()
    for m in (stock, model):
        other_head(m, how)
    want, out = stock(**batch()), model(**batch())
    assert torch.allclose(out.loss, want.loss, atol=1e-5), (out.loss.detach(), want.loss.detach())
    for o in (want, out):
        o.loss.backward()
    for (name, p), q in zip(stock.named_parameters(), model.parameters()):
        assert (p.grad is None) == (q.grad is None), name
        assert p.grad is None or torch.allclose(p.grad, q.grad, atol=1e-5), name


def test_weights_that_are_no_plain_matrix():
    """A matrix that another library holds in pieces, or as a tensor type of its own, is only that library's to read."""
    class Fake:
        is_cuda, dtype, shape = True, torch.float32, (4, 4)

        def dim(self):
            return 2

    class Own(torch.nn.Parameter):
        is_cuda = True
    assert not decoder._fits(torch.nn.Parameter(torch.zeros(4, 4)))               # on the CPU
    assert not decoder._fits(Fake()) and not decoder._fits(Own(torch.zeros(4, 4)))


def test_two_threads_on_one_model(plain):
    """A training call waits in the middle of the decoder while another thread asks the same model for logits, or trains."""
    import threading
    for second in ("logits", "loss"):
        stock, model = pair()
        inputs, other = batch(), batch(2)
        if second == "logits":
            other = {"input_features": other["input_features"], "decoder_input_ids": torch.tensor([[101, 1, 2], [101, 3, 4]])}
        inside, go_on = threading.Event(), threading.Event()
        first = []

        def wait(module, args, output):
            if threading.current_thread() is first[0]:
                inside.set()
                assert go_on.wait(60)
        model.model.decoder.register_forward_hook(wait)
        got, errors = {}, []

        def train():
            try:
                got["first"] = model(**inputs)
            except Exception as e:  # noqa: BLE001 -- reported below
                errors.append(e)
        first.append(threading.Thread(target=train))
        first[0].start()
        try:
            assert inside.wait(60)
            got["second"] = model(**other)
        finally:
            go_on.set()
            first[0].join()
        assert not errors, errors
        assert torch.allclose(got["first"].loss, stock(**inputs).loss, atol=1e-6)
        want = stock(**other)
        if second == "logits":
            assert torch.equal(got["second"].logits, want.logits)
        else:
            assert torch.allclose(got["second"].loss, want.loss, atol=1e-6)


def test_arguments_by_position(plain):
    """Every argument of a call may come by position, labels among them."""
    import inspect
    stock, model = pair()
    names = list(inspect.signature(stock.forward).parameters)
    given = batch()
    by_position = [given.get(name) for name in names[:names.index("labels") + 1]]
    want, out = stock(**given), model(*by_position)
    assert torch.allclose(out.loss, want.loss, atol=1e-6) and "logits" not in out
    out = model(given["input_features"], labels=given["labels"], num_items_in_batch=7)     # as a Trainer calls it
    assert torch.allclose(out.loss, want.loss, atol=1e-6) and "logits" not in out
    seen = {}
    model.model.register_forward_pre_hook(lambda module, args, kwargs: seen.update(kwargs), with_kwargs=True)
    model(**given, num_items_in_batch=7, use_cache=False)
    assert set(seen) == {"input_features", "decoder_input_ids", "num_items_in_batch", "use_cache", "return_dict"}
    with pytest.raises(TypeError):
        model(given["input_features"], input_features=given["input_features"], labels=given["labels"])


def test_installed_models_pickle_and_save_whole(plain, tmp_path):
    import copy
    import io
    import pickle
    stock, model = pair()
    decoder.install(model, logits_in_eval=False)
    want = model(**batch())
    buffer = io.BytesIO()
    torch.save(model, buffer)
    buffer.seek(0)
    for twin in (pickle.loads(pickle.dumps(model)), torch.load(buffer, weights_only=False), copy.deepcopy(model)):
        assert type(twin) is type(model) and twin.wfe_logits_in_eval is False
        out = twin(**batch())
        assert torch.equal(out.loss, want.loss) and "logits" not in out
    # in a process that has not installed anything
    path = tmp_path / "model.pkl"
    path.write_bytes(pickle.dumps(model.cpu()))
    import os
    import subprocess
    import sys
    package = os.path.dirname(os.path.dirname(decoder.__file__))
    code = ("import pickle, sys; m = pickle.load(open(sys.argv[1], 'rb')); from wfe_amd import decoder; "
            "assert type(m) is decoder._model_class() and m.wfe_logits_in_eval is False; print(type(m).__name__)")
    done = subprocess.run([sys.executable, "-c", code, str(path)], env={**os.environ, "PYTHONPATH": package},
                          capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and done.stdout.strip() == "WhisperForConditionalGeneration", done.stderr
    model.save_pretrained(tmp_path / "saved")
    from transformers import WhisperForConditionalGeneration
    again = WhisperForConditionalGeneration.from_pretrained(tmp_path / "saved").train()
    assert type(again) is WhisperForConditionalGeneration
    assert torch.allclose(again(**batch()).loss, want.loss, atol=1e-6)
    with pytest.raises(AttributeError):
        decoder.no_such_name


def trainer_losses(model, tmp_path, **kw):
    """Two steps of the Seq2SeqTrainer that finetune.py uses, on batches as the collator makes them; -> losses, weights."""
    from transformers import Seq2SeqTrainer, Seq2SeqTrainingArguments
    torch.manual_seed(0)
    data = [{k: v[i] for k, v in batch(s).items()} for s in range(4) for i in range(2)]
    args = Seq2SeqTrainingArguments(output_dir=str(tmp_path), per_device_train_batch_size=2, max_steps=2, logging_steps=1,
                                    learning_rate=1e-3, report_to=[], save_strategy="no", disable_tqdm=True,
                                    dataloader_pin_memory=False, remove_unused_columns=False, **kw)
    trainer = Seq2SeqTrainer(model=model, args=args, train_dataset=data, eval_dataset=data,
                             data_collator=lambda rows: {k: torch.stack([r[k] for r in rows]) for k in rows[0]})
    trainer.train()
    losses = [e["loss"] for e in trainer.state.log_history if "loss" in e]
    return trainer, losses


def test_trainer_steps_and_evaluation(plain, tmp_path):
    stock, model = pair()
    decoder.install(model, logits_in_eval=False)
    (_, want), (trainer, got) = (trainer_losses(m, tmp_path, use_cpu=True) for m in (stock, model))
    assert len(want) == 2 and got == pytest.approx(want, abs=1e-4)
    for (name, p), q in zip(stock.named_parameters(), model.named_parameters()):
        assert torch.allclose(p, q[1], atol=1e-4), name
    # a Trainer's predictions: nothing passes for logits (of 103 columns) that is none
    found = trainer.predict(trainer.eval_dataset)
    flat = found.predictions if isinstance(found.predictions, tuple) else (found.predictions,)
    assert all(getattr(x, "shape", (0,))[-1] != 16 or x.shape[1] == 10 for x in flat if x is not None)     # (the encoder's states)


def test_losses_may_be_added_to_in_place(plain):
    """As adapter libraries do with their regularisation."""
    _, model = pair()
    out = model(**batch())
    out.loss += 2.0
    assert out["loss"] is out.loss and out[0] is out.loss
    out.loss.backward()
    assert model.get_output_embeddings().weight.grad is not None
