"""The two ends of the decoder's vocabulary matrix W (vocab, dim), as HIP kernels:

* ``token_embedding``      rows of W for the input tokens, times a scale, and the gradient of W;
* ``linear_cross_entropy`` the loss of the labels under ``hidden @ W.T`` without the logits ever being kept, and the
  gradients of ``hidden`` and W;
* ``install``              puts both into a ``WhisperForConditionalGeneration``, whose training step
  (finetune.py:143-153, finetune_all.py:143-153: the Trainer calls ``model(**batch)`` with the collator's labels) then
  runs on them.

They work on the current stream of the tensors' device, allocate their workspace from torch's allocator and never
synchronise, so they can be captured into a graph (not while an eager call's graph over the same parameters is alive: that
is refused, since torch would end the process).  There is no CPU path: tensors elsewhere raise.
"""
from __future__ import annotations

import ctypes as C
import functools
import types
import weakref
from typing import Optional

import torch

from . import _lib

_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}      # wfe_dtype
_REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}                         # wfe_reduction
_INDEX_BITS = {torch.int32: 32, torch.int64: 64}
_MAX_ROWS = _MAX_VOCAB = 1 << 24
_MAX_DIM = 16384


def _check_matrix(name: str, weight: torch.Tensor, index_name: str, index: torch.Tensor) -> None:
    if weight.dim() != 2:
        raise ValueError(f"{name}: weight must be (vocab, dim), got {tuple(weight.shape)}")
    if weight.dtype not in _DTYPES:
        raise ValueError(f"{name}: weight is {weight.dtype}; float32, float16 or bfloat16 is needed")
    if not 1 <= weight.shape[0] <= _MAX_VOCAB or not 1 <= weight.shape[1] <= _MAX_DIM:
        raise ValueError(f"{name}: weight of {tuple(weight.shape)} outside 1..{_MAX_VOCAB} x 1..{_MAX_DIM}")
    if index.dtype not in _INDEX_BITS:
        raise ValueError(f"{name}: {index_name} are {index.dtype}; int32 or int64 is needed")
    if index.numel() > _MAX_ROWS:
        raise ValueError(f"{name}: {index.numel()} tokens are more than {_MAX_ROWS}")
    if index.device != weight.device:
        raise ValueError(f"{name}: {index_name} are on {index.device}, weight on {weight.device}")
    if weight.device.type != "cuda":
        raise _lib.WfeError(f"{name}: tensors are on {weight.device}; an MI355X is needed, there is no CPU path")


def _stream(device: torch.device) -> int:
    return torch._C._cuda_getCurrentRawStream(device.index)


def _workspace(nbytes: int, device: torch.device) -> torch.Tensor:
    if nbytes < 0:
        _lib.check(int(nbytes))
    return torch.empty(nbytes, dtype=torch.uint8, device=device)


def _dense_rows(t: torch.Tensor) -> torch.Tensor:
    """t with its last dimension contiguous and no negative step (torch has none)."""
    return t if t.shape[-1] == 1 or t.stride(-1) == 1 else t.contiguous()


class _Call:
    """A differentiable call whose graph is alive: the graph holds this, _CALLS only knows of it."""
    __slots__ = ("leaves", "stream", "__weakref__")

    def __init__(self, leaves, stream):
        self.leaves, self.stream = leaves, stream


_CALLS: "weakref.WeakSet[_Call]" = weakref.WeakSet()


def _note(name: str, *inputs: torch.Tensor) -> _Call:
    """Refuses to record a call on parameters that the graph of an earlier eager call, still alive, holds on to.
    Autograd keeps one accumulation node per parameter while any graph refers to it, on the stream it was made on; a
    captured backward pass would draw that stream into the capture, never to leave it, which ends the process."""
    leaves = [t for t in inputs if t.requires_grad and t.is_leaf]
    call = _Call(leaves, _stream(inputs[-1].device))
    if leaves and torch.cuda.is_current_stream_capturing():
        for other in list(_CALLS):
            if other.stream != call.stream and any(a is b for a in leaves for b in other.leaves):
                raise RuntimeError(f"{name}: captured while the autograd graph of an eager call with the same parameter "
                                   "is alive; drop that call's results (or detach them) before capturing")
    _CALLS.add(call)
    return call


# ---- cross entropy -----------------------------------------------------------------------------------------
def _two_strides(hidden: torch.Tensor):
    """(hidden or a copy, inner, outer stride, inner stride): row n of hidden lies at n // inner outer strides and n % inner
    inner ones."""
    hidden = _dense_rows(hidden)
    levels: list = []                           # (size, stride), merged from the last leading dimension on
    for size, stride in zip(reversed(hidden.shape[:-1]), reversed(hidden.stride()[:-1])):
        if size == 1:
            continue
        if levels and stride == levels[-1][0] * levels[-1][1]:
            levels[-1] = (levels[-1][0] * size, levels[-1][1])
        else:
            levels.append((size, stride))
    if len(levels) > 2:
        hidden = hidden.contiguous()
        levels = [(hidden.numel() // hidden.shape[-1], hidden.shape[-1])] if hidden.numel() else []
    inner, inner_stride = levels[0] if levels else (1, hidden.shape[-1])
    outer_stride = levels[1][1] if len(levels) == 2 else 0
    return hidden, max(inner, 1), outer_stride, inner_stride


def _describe(hidden, weight, labels, ignore_index, reduction):
    hidden, inner, outer_stride, inner_stride = _two_strides(hidden)
    weight = _dense_rows(weight)
    desc = _lib.WfeLinearCe(weight.device.index, _DTYPES[weight.dtype], labels.numel(), inner, outer_stride,
                            inner_stride, weight.stride(0), weight.shape[1], weight.shape[0],
                            _INDEX_BITS[labels.dtype], _REDUCTIONS[reduction], ignore_index,
                            _DTYPES[weight.dtype], _DTYPES[weight.dtype])
    return desc, hidden, weight


def _ce_forward(hidden, weight, labels, ignore_index, reduction, keep):
    """(loss, what the backward pass needs if ``keep``)"""
    desc, hidden, weight = _describe(hidden, weight, labels, ignore_index, reduction)
    lib, device, ref = _lib.lib(), weight.device, C.byref(desc)
    labels = labels.contiguous()
    loss = torch.empty(labels.shape if reduction == "none" else (), dtype=torch.float32, device=device)
    address = weight.data_ptr()
    state_bytes = lib.wfe_linear_ce_state_bytes(ref)
    nbytes = lib.wfe_linear_ce_workspace_bytes(ref, address, 0, 0)
    if keep:
        state, workspace = _workspace(state_bytes, device), _workspace(nbytes, device)
        at = workspace.data_ptr()
    else:                                       # one buffer for both
        at = (state_bytes + 255) & -256
        state = _workspace(at + nbytes if state_bytes >= 0 else state_bytes, device)
        at += state.data_ptr()
    _lib.check(lib.wfe_linear_ce_forward(ref, hidden.data_ptr(), address, labels.data_ptr(), loss.data_ptr(),
                                         state.data_ptr(), at, nbytes, _stream(device)))
    return loss, (state, desc, weight) if keep else None


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, labels, dtype, ignore_index, reduction, call):
        ctx.call = call
        ctx.types = (hidden.dtype, weight.dtype)
        ctx.shape = hidden.shape
        loss, (state, ctx.desc, weight) = _ce_forward(hidden.to(dtype), weight.to(dtype), labels, ignore_index,
                                                      reduction, True)
        ctx.save_for_backward(weight, state)
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, upstream):
        weight, state = ctx.saved_tensors
        need_hidden, need_weight = ctx.needs_input_grad[:2]
        desc, device, lib = ctx.desc, weight.device, _lib.lib()
        # a gradient in float32 is written as such; any other type is the products' own, cast where the input's differs
        kinds = [t if t == torch.float32 else weight.dtype for t in ctx.types]
        desc.grad_hidden_dtype, desc.grad_weight_dtype = _DTYPES[kinds[0]], _DTYPES[kinds[1]]
        grad_hidden = torch.empty(ctx.shape, dtype=kinds[0], device=device) if need_hidden else None
        grad_weight = torch.empty(weight.shape, dtype=kinds[1], device=device) if need_weight else None
        ref = C.byref(desc)
        upstream = upstream.to(torch.float32).contiguous()
        nbytes = lib.wfe_linear_ce_workspace_bytes(ref, weight.data_ptr(), 1, int(need_hidden) + 2 * int(need_weight))
        workspace = _workspace(nbytes, device)
        _lib.check(lib.wfe_linear_ce_backward(
            ref, weight.data_ptr(), state.data_ptr(), upstream.data_ptr(),
            grad_hidden.data_ptr() if need_hidden else None, grad_weight.data_ptr() if need_weight else None,
            workspace.data_ptr(), nbytes, _stream(device)))
        if need_hidden:
            grad_hidden = grad_hidden.to(ctx.types[0])
        if need_weight:
            grad_weight = grad_weight.to(ctx.types[1])
        return grad_hidden, grad_weight, None, None, None, None, None


def linear_cross_entropy(hidden: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor, *,
                         ignore_index: int = -100, reduction: str = "mean") -> torch.Tensor:
    """``F.cross_entropy(hidden @ weight.T, labels)`` without the logits: float32, ``labels``' shape for ``"none"``,
    one value for ``"sum"`` and ``"mean"`` (NaN where no label is kept, as torch has it).

    ``hidden`` (..., dim) and ``weight`` (vocab, dim) are both float32, float16 or bfloat16; ``labels`` (...) int32 or
    int64.  Logits, exponentials and sums are float32; a float32 call multiplies in float32.  Under ``torch.autocast``
    both are cast to its type, as ``F.linear`` casts them, and gradients come in the inputs' own types.  Tokens whose
    label is ``ignore_index`` cost nothing and contribute nothing, whatever ``hidden`` holds there.  A label outside
    the vocabulary makes the loss (and the gradients) NaN.  Differentiable once, in ``hidden`` and ``weight``."""
    name = "linear_cross_entropy"
    if reduction not in _REDUCTIONS:
        raise ValueError(f"{name}: reduction {reduction!r} is not 'none', 'sum' or 'mean'")
    _check_matrix(name, weight, "labels", labels)
    if hidden.dim() < 1 or hidden.shape[-1] != weight.shape[1] or hidden.shape[:-1] != labels.shape:
        raise ValueError(f"{name}: hidden {tuple(hidden.shape)} does not fit labels {tuple(labels.shape)} and weight "
                         f"{tuple(weight.shape)}")
    if hidden.device != weight.device:
        raise ValueError(f"{name}: hidden is on {hidden.device}, weight on {weight.device}")
    dtype = weight.dtype
    if torch.is_autocast_enabled("cuda"):
        dtype = torch.get_autocast_dtype("cuda")
        if hidden.dtype not in _DTYPES or dtype not in _DTYPES:
            raise ValueError(f"{name}: {hidden.dtype} under autocast to {dtype}")
    elif hidden.dtype != dtype:
        raise ValueError(f"{name}: hidden is {hidden.dtype}, weight {dtype}; outside autocast they must agree")
    if torch.is_grad_enabled() and (hidden.requires_grad or weight.requires_grad):
        return _LinearCrossEntropy.apply(hidden, weight, labels, dtype, int(ignore_index), reduction,
                                         _note(name, hidden, weight))
    return _ce_forward(hidden.to(dtype), weight.to(dtype), labels, int(ignore_index), reduction, False)[0]


# ---- embedding ---------------------------------------------------------------------------------------------
def _embed_desc(ids, weight, scale, padding_idx):
    return _lib.WfeEmbedding(weight.device.index, _DTYPES[weight.dtype], ids.numel(), weight.stride(0), weight.shape[1],
                             weight.shape[1], weight.shape[0], _INDEX_BITS[ids.dtype], _DTYPES[weight.dtype],
                             -1 if padding_idx is None else padding_idx, scale)


def _embed_forward(ids, weight, scale, padding_idx):
    weight, ids = _dense_rows(weight), ids.contiguous()
    desc = _embed_desc(ids, weight, scale, padding_idx)
    out = torch.empty((*ids.shape, weight.shape[1]), dtype=weight.dtype, device=weight.device)
    _lib.check(_lib.lib().wfe_embedding(C.byref(desc), ids.data_ptr(), weight.data_ptr(), out.data_ptr(),
                                        _stream(weight.device)))
    return out, ids, desc


class _TokenEmbedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, weight, scale, padding_idx, call):
        ctx.call = call
        out, ids, ctx.desc = _embed_forward(ids, weight, scale, padding_idx)
        ctx.save_for_backward(ids)
        ctx.weight_shape = weight.shape
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_out):
        ids, = ctx.saved_tensors
        desc, lib, device = ctx.desc, _lib.lib(), grad_out.device
        dim = ctx.weight_shape[1]
        rows = _dense_rows(grad_out)
        if not rows.is_contiguous():
            rows = rows.reshape(-1, dim)        # a view where the leading dimensions allow one
        desc.grad_stride = dim if rows.is_contiguous() else rows.stride(0)
        grad_weight = torch.empty(ctx.weight_shape, dtype=grad_out.dtype, device=device)
        nbytes = lib.wfe_embedding_workspace_bytes(C.byref(desc))
        workspace = _workspace(nbytes, device)
        _lib.check(lib.wfe_embedding_backward(C.byref(desc), ids.data_ptr(), rows.data_ptr(), grad_weight.data_ptr(),
                                              workspace.data_ptr(), nbytes, _stream(device)))
        return None, grad_weight, None, None, None


def token_embedding(ids: torch.Tensor, weight: torch.Tensor, *, scale: float = 1.0,
                    padding_idx: Optional[int] = None) -> torch.Tensor:
    """``scale * F.embedding(ids, weight, padding_idx)``, rounded once: (..., dim) of ``weight``'s type.

    ``ids`` (...) int32 or int64, ``weight`` (vocab, dim) float32, float16 or bfloat16.  The gradient of ``weight`` is
    summed in float32 over a token's occurrences in their order, the same bits every time; ``padding_idx`` (negative:
    from the end) gets none.  An id outside the vocabulary gives a row of NaN and no gradient.  Differentiable once."""
    name = "token_embedding"
    _check_matrix(name, weight, "ids", ids)
    if padding_idx is not None:
        if not -weight.shape[0] <= padding_idx < weight.shape[0]:
            raise ValueError(f"{name}: padding_idx {padding_idx} outside a vocabulary of {weight.shape[0]}")
        padding_idx = int(padding_idx) % weight.shape[0]
    if torch.is_grad_enabled() and weight.requires_grad:
        return _TokenEmbedding.apply(ids, weight, float(scale), padding_idx, _note(name, weight))
    return _embed_forward(ids, weight, float(scale), padding_idx)[0]


# ---- a Whisper model on them -------------------------------------------------------------------------------
def _stock(module):
    """The module's forward as a function of (module, ...): its class's, so that copies of the module keep working, or
    the one that hooks have put into the instance."""
    own = module.__dict__.get("forward")
    return type(module).forward if own is None else lambda self, *args, **kwargs: own(*args, **kwargs)


def install(model, logits_in_eval: bool = True):
    """Puts the two operators into ``model``, a ``WhisperForConditionalGeneration`` (or a wrapper whose
    ``get_base_model()`` is one), in place, and returns it: the decoder's token embedding, and the loss of a call with
    ``labels``.  Such a call returns its loss and no logits (``logits`` is None); in evaluation mode it computes both
    as before unless ``logits_in_eval`` is False.  Calls without labels, generation and saved files are untouched.
    Weights may sit on the CPU until the first call.  Installing twice does nothing."""
    base = model.get_base_model() if hasattr(model, "get_base_model") else model
    from transformers import WhisperForConditionalGeneration
    if not isinstance(base, WhisperForConditionalGeneration):
        raise ValueError(f"install: {type(base).__name__} is not a WhisperForConditionalGeneration")
    if getattr(base, "_wfe_decoder", False):
        return model
    from transformers.models.whisper.modeling_whisper import shift_tokens_right
    embed, head = base.get_input_embeddings(), base.get_output_embeddings()
    if type(embed) is not torch.nn.Embedding or type(head) is not torch.nn.Linear or head.bias is not None \
            or embed.max_norm is not None or embed.sparse or embed.scale_grad_by_freq:
        raise ValueError("install: the model's token embedding or output projection is not a plain one")
    stock_forward, stock_embed, stock_head = _stock(base), _stock(embed), _stock(head)

    def embed_forward(self, ids):
        if not self.weight.is_cuda:
            return stock_embed(self, ids)
        return token_embedding(ids, self.weight, padding_idx=self.padding_idx)

    def head_forward(self, hidden):
        return hidden if getattr(self, "_wfe_pass_hidden", False) else stock_head(self, hidden)

    @functools.wraps(type(base).forward)
    def forward(self, *args, **kwargs):
        labels, head = kwargs.get("labels"), self.get_output_embeddings()
        fused = labels is not None and head.weight.is_cuda and (self.training or not logits_in_eval)
        if not fused or kwargs.get("return_dict") is False:
            return stock_forward(self, *args, **kwargs)
        if labels.shape[1] > self.max_target_positions:
            raise ValueError(f"Labels' sequence length {labels.shape[1]} cannot exceed the maximum allowed length of "
                             f"{self.max_target_positions} tokens.")
        kwargs["labels"] = None
        if kwargs.get("decoder_input_ids") is None and kwargs.get("decoder_inputs_embeds") is None:
            kwargs["decoder_input_ids"] = shift_tokens_right(labels, self.config.pad_token_id,
                                                             self.config.decoder_start_token_id)
        head._wfe_pass_hidden = True            # the call's "logits" are the head's input
        try:
            out = stock_forward(self, *args, **kwargs)
        finally:
            head._wfe_pass_hidden = False
        out.loss = linear_cross_entropy(out.logits, head.weight, labels.to(out.logits.device))
        out.logits = None
        return out

    embed.forward = types.MethodType(embed_forward, embed)
    head.forward = types.MethodType(head_forward, head)
    base.forward = types.MethodType(forward, base)
    base._wfe_decoder = True
    return model
