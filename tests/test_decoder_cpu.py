"""What the decoder's vocabulary operators refuse, checked without a GPU: nothing here reaches a device call."""
import ctypes as C

import pytest
import torch

from wfe_amd import _lib, decoder


def test_python_entry_points_refuse():
    h, w, y = torch.zeros(2, 3, 8), torch.zeros(5, 8), torch.zeros(2, 3, dtype=torch.int64)
    lce, emb = decoder.linear_cross_entropy, decoder.token_embedding
    with pytest.raises(ValueError, match="reduction"):
        lce(h, w, y, reduction="batchmean")
    with pytest.raises(ValueError, match="weight must be"):
        lce(h, w[0], y)
    with pytest.raises(ValueError, match="float64"):
        lce(h.double(), w.double(), y)
    with pytest.raises(ValueError, match="int16"):
        lce(h, w, y.to(torch.int16))
    with pytest.raises(ValueError, match="outside 1"):
        lce(torch.zeros(1, 0), torch.zeros(5, 0), y[0, :1])
    with pytest.raises(ValueError, match="outside 1"):
        emb(y, torch.zeros(0, 8))
    with pytest.raises(ValueError, match="outside 1"):
        emb(y, torch.empty(1, 16385))
    with pytest.raises(ValueError, match="on meta"):
        lce(h, w, y.to("meta"))
    with pytest.raises(ValueError, match="2\\^37 logits"):
        lce(h[:1, 0].expand(1 << 24, 8), w[:1].expand((1 << 13) + 1, 8), y[:1, 0].expand(1 << 24))
    with pytest.raises(ValueError, match="int32 or int64"):
        emb(y.bool(), w)
    for call in (lambda: lce(h, w, y), lambda: emb(y, w)):
        with pytest.raises(_lib.WfeError, match="no CPU path"):
            call()


def test_shapes_are_checked_before_the_device_is_used():
    meta = torch.device("meta")          # (a stand-in for another device: refused like the CPU, but after the types)
    with pytest.raises(_lib.WfeError, match="no CPU path"):
        decoder.linear_cross_entropy(torch.zeros(2, 8, device=meta), torch.zeros(5, 8, device=meta),
                                     torch.zeros(2, dtype=torch.int64, device=meta))


def _ce(**kw):
    d = _lib.WfeLinearCe(0, 2, 10, 10, 0, 64, 64, 64, 100, 64, 2, -100, 2, 2)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def _emb(**kw):
    d = _lib.WfeEmbedding(0, 2, 10, 64, 64, 64, 100, 64, 2, -1, 1.0)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


BAD_CE = [dict(dtype=3), dict(dtype=-1), dict(rows=-1), dict(rows=(1 << 24) + 1), dict(dim=0), dict(dim=16385),
          dict(vocab=0), dict(vocab=(1 << 24) + 1), dict(inner=0), dict(outer_stride=-1), dict(inner_stride=-64),
          dict(weight_stride=-1), dict(weight_stride=1 << 47), dict(label_bits=16), dict(reduction=3),
          dict(grad_hidden_dtype=1), dict(grad_weight_dtype=1),
          dict(rows=1 << 24, vocab=(1 << 13) + 1, inner=1 << 24), dict(rows=2650000, vocab=51866, inner=2650000)]


@pytest.mark.parametrize("bad", BAD_CE, ids=str)
def test_c_linear_ce_refuses(bad):
    lib, d = _lib.lib(), _ce(**bad)
    assert lib.wfe_linear_ce_state_bytes(C.byref(d)) == _lib.ERR_ARG
    assert lib.wfe_linear_ce_workspace_bytes(C.byref(d), None, 1, 3) == _lib.ERR_ARG
    assert lib.wfe_linear_ce_forward(C.byref(d), 64, 64, 64, 64, 64, 64, 1 << 40, None) == _lib.ERR_ARG
    assert lib.wfe_linear_ce_backward(C.byref(d), 64, 64, 64, 64, 64, 64, 1 << 40, None) == _lib.ERR_ARG
    assert b"linear_ce" in lib.wfe_last_error(None)


BAD_EMB = [dict(dtype=5), dict(rows=-1), dict(rows=1 << 25), dict(dim=0), dict(dim=1 << 15), dict(vocab=0),
           dict(vocab=1 << 25), dict(weight_stride=-1), dict(grad_stride=-8), dict(id_bits=8), dict(grad_weight_dtype=1)]


@pytest.mark.parametrize("bad", BAD_EMB, ids=str)
def test_c_embedding_refuses(bad):
    lib, d = _lib.lib(), _emb(**bad)
    assert lib.wfe_embedding(C.byref(d), 64, 64, 64, None) == _lib.ERR_ARG
    assert lib.wfe_embedding_workspace_bytes(C.byref(d)) == _lib.ERR_ARG
    assert lib.wfe_embedding_backward(C.byref(d), 64, 64, 64, 64, 1 << 40, None) == _lib.ERR_ARG
    assert b"embedding" in lib.wfe_last_error(None)


def test_c_pointers_and_workspaces():
    lib = _lib.lib()
    d = _ce()
    need = lib.wfe_linear_ce_workspace_bytes(C.byref(d), 64, 0, 0)
    assert need > 0 and lib.wfe_linear_ce_state_bytes(C.byref(d)) > 0
    # rows of W that cannot be read in place cost a copy of W
    assert lib.wfe_linear_ce_workspace_bytes(C.byref(d), 66, 0, 0) >= need + 100 * 64 * 2
    assert lib.wfe_linear_ce_workspace_bytes(C.byref(_ce(weight_stride=65)), 64, 0, 0) >= need + 100 * 64 * 2
    both = lib.wfe_linear_ce_workspace_bytes(C.byref(d), 64, 1, 3)
    assert both >= lib.wfe_linear_ce_workspace_bytes(C.byref(d), 64, 1, 2)
    fwd = lib.wfe_linear_ce_forward
    assert fwd(C.byref(d), None, 64, 64, 64, 64, 64, need, None) == _lib.ERR_ARG
    assert fwd(C.byref(d), 64, 64, 64, None, 64, 64, need, None) == _lib.ERR_ARG
    assert fwd(C.byref(d), 64, 64, 68, 64, 64, 64, need, None) == _lib.ERR_ARG          # labels off 8 bytes
    assert fwd(C.byref(d), 64, 64, 64, 64, 64, 64, need - 1, None) == _lib.ERR_ARG
    assert b"workspace" in lib.wfe_last_error(None)
    assert fwd(C.byref(d), 64, 64, 64, 64, 64, None, need, None) == _lib.ERR_ARG
    assert fwd(C.byref(d), 64, 64, 64, 64, 64, 72, need, None) == _lib.ERR_ARG
    assert fwd(None, 64, 64, 64, 64, 64, 64, need, None) == _lib.ERR_ARG
    bwd = lib.wfe_linear_ce_backward
    assert bwd(C.byref(d), 64, 64, 64, None, None, None, 0, None) == 0               # nothing wanted
    assert bwd(C.byref(d), 64, 64, 64, 66, None, 64, both, None) == _lib.ERR_ARG
    assert bwd(C.byref(d), 64, None, 64, 64, None, 64, both, None) == _lib.ERR_ARG
    assert bwd(C.byref(d), 64, 64, 64, 64, 64, 64, both - 1, None) == _lib.ERR_ARG
    e = _emb()
    need = lib.wfe_embedding_workspace_bytes(C.byref(e))
    assert lib.wfe_embedding(C.byref(e), 64, None, 64, None) == _lib.ERR_ARG
    assert lib.wfe_embedding(C.byref(_emb(rows=0)), None, None, None, None) == 0
    assert lib.wfe_embedding_backward(C.byref(e), 64, 64, 64, 64, need - 1, None) == _lib.ERR_ARG
    assert lib.wfe_embedding_backward(C.byref(e), 64, 64, 68, 64, need, None) == _lib.ERR_ARG


@pytest.mark.skipif(torch.cuda.is_available(), reason="a machine without a GPU")
def test_c_entries_without_a_gpu():
    lib, d = _lib.lib(), _ce()
    need = lib.wfe_linear_ce_workspace_bytes(C.byref(d), 64, 0, 0)
    assert lib.wfe_linear_ce_forward(C.byref(d), 64, 64, 64, 64, 64, 64, need, None) == _lib.ERR_HIP
    assert b"no HIP device" in lib.wfe_last_error(None)


def test_install_refuses_what_it_does_not_know_and_leaves_a_cpu_model_alone():
    import copy
    from transformers import WhisperConfig, WhisperForConditionalGeneration
    with pytest.raises(ValueError, match="not a WhisperForConditionalGeneration"):
        decoder.install(torch.nn.Linear(2, 2))
    cfg = WhisperConfig(vocab_size=103, num_mel_bins=8, d_model=16, encoder_layers=1, decoder_layers=1,
                        encoder_attention_heads=2, decoder_attention_heads=2, encoder_ffn_dim=16, decoder_ffn_dim=16,
                        max_source_positions=10, max_target_positions=8, pad_token_id=100, bos_token_id=100,
                        eos_token_id=100, decoder_start_token_id=101)
    stock = WhisperForConditionalGeneration(cfg).eval()
    model = decoder.install(copy.deepcopy(stock))
    import inspect
    assert inspect.signature(model.forward) == inspect.signature(stock.forward)
    feats, labels = torch.randn(2, 8, 20), torch.randint(0, 100, (2, 5))
    a, b = (m(input_features=feats, labels=labels) for m in (stock, model))
    assert torch.equal(a.loss, b.loss) and torch.equal(a.logits, b.logits)
    import pickle
    again = pickle.loads(pickle.dumps(model.get_output_embeddings()))
    assert torch.equal(again(torch.ones(1, 16)), stock.get_output_embeddings()(torch.ones(1, 16)))
    assert type(model).__name__ == type(stock).__name__ and decoder.install(model) is model
    hooked = copy.deepcopy(stock)
    hooked.forward = hooked.forward
    with pytest.raises(ValueError, match="replaced already"):
        decoder.install(hooked)
    odd = copy.deepcopy(stock)
    odd.set_output_embeddings(torch.nn.Linear(16, 103, bias=True))
    with pytest.raises(ValueError, match="not a plain one"):
        decoder.install(odd)


def test_launcher_installs_the_operators_on_request(tmp_path, monkeypatch):
    """wfe_amd.launch with WFE_INSTALL_DECODER=1: from_pretrained returns a model with the operators in place."""
    import sys
    from transformers import WhisperConfig, WhisperForConditionalGeneration
    from wfe_amd import launch
    cfg = WhisperConfig(vocab_size=103, num_mel_bins=8, d_model=16, encoder_layers=1, decoder_layers=1,
                        encoder_attention_heads=2, decoder_attention_heads=2, encoder_ffn_dim=16, decoder_ffn_dim=16,
                        max_source_positions=10, max_target_positions=8, pad_token_id=100, bos_token_id=100,
                        eos_token_id=100, decoder_start_token_id=101)
    WhisperForConditionalGeneration(cfg).save_pretrained(tmp_path / "model")
    script = tmp_path / "script.py"
    script.write_text("import os, transformers\n"
                      "m = transformers.WhisperForConditionalGeneration.from_pretrained(os.environ['MODEL_DIR'])\n"
                      "open(os.environ['MODEL_DIR'] + '/seen', 'w').write(str(hasattr(m, 'wfe_logits_in_eval')))\n")
    monkeypatch.setenv("MODEL_DIR", str(tmp_path / "model"))
    before = WhisperForConditionalGeneration.__dict__.get("from_pretrained")
    try:
        for flag, want in (("0", "False"), ("1", "True")):
            monkeypatch.setenv("WFE_INSTALL_DECODER", flag)
            monkeypatch.setattr(sys, "argv", list(sys.argv))
            monkeypatch.setattr(sys, "path", list(sys.path))
            monkeypatch.setattr(sys, "meta_path", list(sys.meta_path))
            launch.main([str(script)])
            assert (tmp_path / "model" / "seen").read_text() == want
    finally:
        if before is None:
            del WhisperForConditionalGeneration.from_pretrained
        else:
            WhisperForConditionalGeneration.from_pretrained = before
