"""The two ends of the decoder's vocabulary matrix W (vocab, dim), as HIP kernels:

* ``token_embedding``      rows of W for the input tokens, times a scale, and the gradient of W;
* ``linear_cross_entropy`` the loss of the labels under ``hidden @ W.T`` without the logits ever being kept, and the
  gradients of ``hidden`` and W;
* ``install``              puts both into a ``WhisperForConditionalGeneration``, whose training step
  (the Seq2SeqTrainer of finetune.py:144-150 calls ``model(**batch)`` with the collator's labels) then runs on them.

They work on the current stream of the tensors' device, allocate their workspace from torch's allocator and never
synchronise, so they can be captured into a graph (not while the graph of an earlier call on the default stream over the
same parameters is alive: that is refused, since torch would end the process).  There is no CPU path: tensors elsewhere
raise.

The kernels and their C ABI are in libwfe_hip.so; ``_decoder.so`` (csrc/wfe_torch.cpp) makes them differentiable.
"""
from __future__ import annotations

import ctypes as C
import functools
import inspect
import os
from typing import Optional

import torch

from . import _lib

_REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}                         # wfe_reduction
_ENTRIES = ("wfe_last_error", "wfe_linear_ce_state_bytes", "wfe_linear_ce_workspace_bytes", "wfe_linear_ce_forward",
            "wfe_linear_ce_backward", "wfe_embedding", "wfe_embedding_workspace_bytes", "wfe_embedding_backward")

_module = None


def _ext():
    global _module
    if _module is None:
        try:
            from . import _decoder
        except ImportError as e:
            raise _lib.WfeError(f"{os.path.join(os.path.dirname(__file__), '_decoder.so')} cannot be loaded ({e}): build it "
                                "with `make -C whisper-finetune_amd/csrc` (or __graft_entry__.build())") from e
        lib = _lib.lib()
        _decoder.bind([C.cast(getattr(lib, name), C.c_void_p).value for name in _ENTRIES], _lib.WfeError)
        _module = _decoder
    return _module


def linear_cross_entropy(hidden: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor, *,
                         ignore_index: int = -100, reduction: str = "mean") -> torch.Tensor:
    """``F.cross_entropy(hidden @ weight.T, labels)`` without the logits: float32, ``labels``' shape for ``"none"``,
    one value for ``"sum"`` and ``"mean"`` (NaN where no label is kept, as torch has it).

    ``hidden`` (..., dim) and ``weight`` (vocab, dim) are both float32, float16 or bfloat16; ``labels`` (...) int32 or
    int64.  Logits, exponentials and sums are float32; a float32 call multiplies to float32 accuracy.  Under
    ``torch.autocast`` both are cast to its type, as ``F.linear`` casts them, and gradients come in the inputs' own
    types.  Tokens whose label is ``ignore_index`` cost nothing and contribute nothing, whatever ``hidden`` holds there.
    A label outside the vocabulary makes the loss (and the gradients) NaN.  Differentiable once, in ``hidden`` and
    ``weight``, in reverse mode (forward-mode tangents and ``torch.func`` transforms raise).  At most 2^24 tokens, a vocabulary of 2^24, a dim of 16384 and 2^37 logits."""
    code = _REDUCTIONS.get(reduction)
    if code is None:
        raise ValueError(f"linear_cross_entropy: reduction {reduction!r} is not 'none', 'sum' or 'mean'")
    return (_module or _ext()).linear_cross_entropy(hidden, weight, labels, ignore_index, code)


def token_embedding(ids: torch.Tensor, weight: torch.Tensor, *, scale: float = 1.0,
                    padding_idx: Optional[int] = None) -> torch.Tensor:
    """``scale * F.embedding(ids, weight, padding_idx)``, rounded once: (..., dim) of ``weight``'s type.

    ``ids`` (...) int32 or int64, ``weight`` (vocab, dim) float32, float16 or bfloat16.  The gradient of ``weight`` is
    summed in float32 over a token's occurrences in their order, the same bits every time; ``padding_idx`` (negative:
    from the end) gets none.  An id outside the vocabulary gives a row of NaN and no gradient.  Differentiable once, in
    reverse mode, as above."""
    return (_module or _ext()).token_embedding(ids, weight, scale, padding_idx)


# ---- a Whisper model on them -------------------------------------------------------------------------------
_TYPES = (torch.float32, torch.float16, torch.bfloat16)


def _fits(weight: torch.Tensor) -> bool:
    # (libraries that shard or quantise hold weights as flat pieces or as tensor types of their own)
    return type(weight) in (torch.Tensor, torch.nn.Parameter) and weight.dim() == 2 and weight.is_cuda \
        and weight.dtype in _TYPES


def _plain(module, kind) -> bool:
    """Whether ``module`` computes what a ``kind`` does and nothing beside it."""
    return type(module) is kind and "forward" not in module.__dict__ and not (
        module._forward_hooks or module._forward_pre_hooks or module._backward_hooks or module._backward_pre_hooks)


class _Embedding(torch.nn.Embedding):
    def forward(self, ids):
        if not _fits(self.weight):
            return super().forward(ids)
        return token_embedding(ids, self.weight, padding_idx=self.padding_idx)


@functools.lru_cache(maxsize=None)
def _model_class():
    from transformers import WhisperForConditionalGeneration
    from transformers.modeling_outputs import Seq2SeqLMOutput
    from transformers.models.whisper.modeling_whisper import shift_tokens_right
    signature = inspect.signature(WhisperForConditionalGeneration.forward)
    more = next((p.name for p in signature.parameters.values() if p.kind is p.VAR_KEYWORD), None)

    class Model(WhisperForConditionalGeneration):
        wfe_logits_in_eval = True

        @functools.wraps(WhisperForConditionalGeneration.forward)
        def forward(self, *args, **kwargs):
            if self.training or not self.wfe_logits_in_eval:
                given = dict(signature.bind(self, *args, **kwargs).arguments)
                given.update(given.pop(more, {}))
                labels, return_dict, head = given.get("labels"), given.get("return_dict"), self.get_output_embeddings()
                as_tuple = not (self.config.return_dict if return_dict is None else return_dict)
                # the projection may have been replaced, wrapped or hooked since install: then it is called as it is
                if labels is not None and not as_tuple and _plain(head, torch.nn.Linear) and head.bias is None \
                        and _fits(head.weight):
                    del given["self"], given["labels"]
                    return self._wfe_loss(head.weight, labels, {**given, "return_dict": True})
            return super().forward(*args, **kwargs)

        def _wfe_loss(self, weight, labels, given):
            """The call with labels: the decoder's last hidden states into the loss, the projection itself not called."""
            if labels.shape[1] > self.max_target_positions:
                raise ValueError(f"labels of {labels.shape[1]} tokens are longer than max_target_positions "
                                 f"({self.max_target_positions})")
            if given.get("decoder_input_ids") is None and given.get("decoder_inputs_embeds") is None:
                given["decoder_input_ids"] = shift_tokens_right(labels, self.config.pad_token_id,
                                                                self.config.decoder_start_token_id)
            out = self.model(**given)
            hidden = out.last_hidden_state
            loss = linear_cross_entropy(hidden, weight, labels.to(hidden.device))
            return Seq2SeqLMOutput(loss=loss, **{k: v for k, v in out.items() if k != "last_hidden_state"})

    # saved configurations and the Trainer know a model by its class's name; pickles find it here by that (__getattr__)
    Model.__name__ = Model.__qualname__ = "WhisperForConditionalGeneration"
    return Model


def __getattr__(name):
    if name == "WhisperForConditionalGeneration":
        return _model_class()
    raise AttributeError(f"module {__name__!r} has no attribute {name!r}")


def install(model, logits_in_eval: bool = True):
    """Puts the two operators into ``model``, a ``WhisperForConditionalGeneration`` (or a wrapper whose
    ``get_base_model()`` is one), in place, and returns it: the decoder's token embedding, and the loss of a call with
    ``labels``.  Such a call returns its loss and no logits (no such entry); in evaluation mode it computes both
    as before unless ``logits_in_eval`` is False.  Calls without labels or for tuples, generation, copies, pickles and
    saved files are as before, and so is everything while the weights are on the CPU or in 64 bits, or the output
    projection is another module than it was, or hooked.  Installing twice only sets ``logits_in_eval``."""
    base = model.get_base_model() if hasattr(model, "get_base_model") else model
    from transformers import WhisperForConditionalGeneration
    if isinstance(base, _model_class()):
        base.wfe_logits_in_eval = logits_in_eval
        return model
    if type(base) is not WhisperForConditionalGeneration:
        raise ValueError(f"install: {type(base).__name__} is not a WhisperForConditionalGeneration")
    embed, head = base.get_input_embeddings(), base.get_output_embeddings()
    if type(embed) is not torch.nn.Embedding or type(head) is not torch.nn.Linear or head.bias is not None \
            or embed.max_norm is not None or embed.sparse or embed.scale_grad_by_freq:
        raise ValueError("install: the model's token embedding or output projection is not a plain one")
    if any("forward" in module.__dict__ for module in (base, embed, head)):
        raise ValueError("install: the model's forward has been replaced already (by hooks of another library, as "
                         "device_map leaves them); install before that")
    # subclasses, not bound functions: copies, pickles and replicas of the modules keep their own weights
    embed.__class__, base.__class__ = _Embedding, _model_class()
    base.wfe_logits_in_eval = logits_in_eval
    return model
