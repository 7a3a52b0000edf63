"""The two ends of a student's training step on torch tensors: embeddings with their
gradient, and the gradients' norm and clipping.

For programs that distil into a model of their own with scores.distill_loss: what
comes before its first layer and after its last gradient.  The calls enqueue the
library's kernels (dtl_embedding*, dtl_grad_norm, dtl_clip_grads of
include/detllm.h, which define every result) on the current stream of the tensors'
device, do not wait, and can be captured into a graph, as those of scores.py.
Reverse mode only.

    hidden = train.embedding(weight, tokens, scale=weight.shape[1] ** 0.5)
    logits = student(hidden)
    loss, grad = scores.distill_loss_and_grad(logits, teacher.top_ids, teacher.top_log_probs, weights)
    logits.backward(grad)
    norm = train.clip_grad_norm([p.grad for p in parameters], 1.0)
"""
from __future__ import annotations

import ctypes as C
from functools import lru_cache
from typing import Optional

import torch

from . import _lib
from ._lib import DetllmError, lib
from .scores import _DTYPES, _INDEX, _call, _incoming, _no_tangent, _ptr, _scratch, _tracing

MAX_TOKENS = 1 << 20  # of an embedding's gradient

_embed_scratch = lru_cache(maxsize=256)(lib.dtl_embedding_backward_scratch)


# ---- embeddings ---------------------------------------------------------------------


def _need_floats(t: torch.Tensor, name: str) -> None:
    if not isinstance(t, torch.Tensor) or t.dtype not in _DTYPES:
        raise TypeError(f"{name} must be a float32, bfloat16 or float16 tensor")
    _no_tangent(t, name)
    if _tracing():
        raise RuntimeError("calls of the library cannot be recorded by torch.jit.trace")
    if not t.is_cuda:
        raise ValueError(f"{name} must be on the GPU")


def _table(t: torch.Tensor, name: str) -> _lib.Table:
    """A matrix's rows as a dtl_table."""
    if t.dim() != 2 or not t.numel():
        raise ValueError(f"{name} must be a matrix [vocab, width]")
    (vocab, width), (stride, step) = t.shape, t.stride()
    if width > 1 and step != 1:
        raise ValueError(f"the last dimension of {name} must be contiguous")
    if vocab > 1 and stride < width:
        raise ValueError(f"the rows of {name} overlap: call .contiguous()")
    return _lib.Table(t.data_ptr(), _DTYPES[t.dtype], vocab, width, max(stride, width))


def _token_ids(tokens, device) -> torch.Tensor:
    if not isinstance(tokens, torch.Tensor) or tokens.dtype not in _INDEX:
        raise TypeError("tokens must be a tensor of torch.int64 or torch.int32")
    if tokens.device != device:
        raise ValueError("tokens and the table are on different devices")
    return tokens.contiguous()


def _lookup(weight, tokens, scale):
    t = _table(weight, "weight")
    out = torch.empty((*tokens.shape, t.width), dtype=weight.dtype, device=weight.device)
    _call(weight.device, lib.dtl_embedding, C.byref(t), _ptr(tokens), tokens.element_size(), tokens.numel(), scale,
          _ptr(out), t.width)
    return out


def _gradient(tokens, grad, scale, out, add):
    g, n = _table(out, "out"), tokens.numel()
    need = _embed_scratch(n, g.vocab, g.width)
    scratch = _scratch(need, out.device)
    _call(out.device, lib.dtl_embedding_backward, _ptr(tokens), tokens.element_size(), n, _ptr(grad), _DTYPES[grad.dtype],
          g.width, scale, C.byref(g), int(add), _ptr(scratch), need)
    return out


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, weight, tokens, scale):
        ctx.save_for_backward(tokens)
        ctx.like, ctx.scale = (weight.shape, weight.dtype, weight.device), scale
        return _lookup(weight, tokens, scale)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        tokens, = ctx.saved_tensors
        shape, dtype, device = ctx.like
        return _gradient(tokens, _incoming(g), ctx.scale, torch.empty(shape, dtype=dtype, device=device), False), None, None


def embedding(weight: torch.Tensor, tokens: torch.Tensor, *, scale: float = 1.0) -> torch.Tensor:
    """dtl_embedding: scale * weight[tokens] for weight[vocab, width] (float32, bfloat16
    or float16) and tokens[...] (int64 or int32; -1 is padding: a row of zeros),
    differentiable in weight: a dense gradient, the same bits every time."""
    _need_floats(weight, "weight")
    tokens = _token_ids(tokens, weight.device)
    if torch.is_grad_enabled() and weight.requires_grad:
        if tokens.numel() > MAX_TOKENS:
            raise DetllmError(1, "embedding: more tokens than a gradient takes")
        return _Embedding.apply(weight, tokens, float(scale))
    return _lookup(weight, tokens, float(scale))


def embedding_grad(tokens: torch.Tensor, grad: torch.Tensor, vocab: Optional[int] = None, *, scale: float = 1.0,
                   out: Optional[torch.Tensor] = None, add: bool = False) -> torch.Tensor:
    """dtl_embedding_backward: the gradient of embedding's weight for that of its rows,
    grad[..., width], for loops that run their own backward pass.  out: where it goes
    ([vocab, width], of grad's type or float32); with add, on top of what it holds (an
    output matrix that shares its weight, say), its other rows left alone."""
    _need_floats(grad, "grad")
    tokens = _token_ids(tokens, grad.device)
    if not grad.dim() or grad.shape[:-1] != tokens.shape:
        raise ValueError(f"grad has shape {tuple(grad.shape)}, expected {(*tokens.shape, 'width')}")
    grad = grad.contiguous()
    if out is None:
        if vocab is None or add:
            raise ValueError("embedding_grad needs a vocab or an out, and out for add")
        out = torch.empty((vocab, grad.shape[-1]), dtype=grad.dtype, device=grad.device)
        return _gradient(tokens, grad, float(scale), out, False)
    _need_floats(out, "out")
    if out.requires_grad and torch.is_grad_enabled():
        raise ValueError("out has no gradient")
    if out.device != grad.device or out.dim() != 2 or out.shape != (vocab or out.shape[0], grad.shape[-1]):
        raise ValueError("out must have grad's device and width, and the vocab")
    if out.dtype not in (grad.dtype, torch.float32):
        raise TypeError("out must have the type of grad, or be float32")
    _gradient(tokens, grad, float(scale), out, add)
    torch.autograd.graph.increment_version(out)  # autograd is told that it was written
    return out
