"""The two ends of a student's training step on torch tensors: embeddings with their
gradient, and the gradients' norm and clipping.

For programs that distil into a model of their own with scores.distill_loss: what
comes before its first layer and after its last gradient.  The calls enqueue the
library's kernels (dtl_embedding*, dtl_grad_norm, dtl_clip_grads of
include/detllm.h, which define every result) on the current stream of the tensors'
device, do not wait, and can be captured into a graph, as those of scores.py (a
captured backward needs a leaf of its own, `weight.detach().requires_grad_()`).
Reverse mode only.

    hidden = train.embedding(weight, tokens, scale=weight.shape[1] ** 0.5)
    logits = student(hidden)
    loss, grad = scores.distill_loss_and_grad(logits, teacher.top_ids, teacher.top_log_probs, weights)
    logits.backward(grad)
    norm = train.clip_grad_norm([p.grad for p in parameters], 1.0)
"""
from __future__ import annotations

import ctypes as C
import math
from array import array
from functools import lru_cache
from operator import attrgetter
from typing import Iterable, List, Optional, Tuple, Union

import torch
from torch.autograd import forward_ad

from . import _lib
from ._lib import DetllmError, lib
from .scores import _DTYPES, _INDEX, _call, _no_tangent, _once, _ptr, _tracing

MAX_TOKENS = 1 << 20  # of an embedding's gradient

_dtype_of, _layout_of, _shape_of, _requires_grad_of = map(attrgetter, ("dtype", "layout", "shape", "requires_grad"))
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
    out = weight.new_empty((*tokens.shape, t.width))
    _call(weight.device, lib.dtl_embedding, C.byref(t), _ptr(tokens), tokens.element_size(), tokens.numel(), scale,
          _ptr(out), t.width)
    return out


def _gradient(tokens, grad, scale, out, add):
    g, n = _table(out, "out"), tokens.numel()
    if grad.dim() == 2 and grad.stride(1) == 1 and grad.stride(0) >= g.width:  # rows of a wider tensor are not copied
        spacing = grad.stride(0)
    else:
        grad, spacing = grad.contiguous(), g.width
    need = _embed_scratch(n, g.vocab, g.width)
    scratch = out.new_empty(need, dtype=torch.uint8)
    _call(out.device, lib.dtl_embedding_backward, _ptr(tokens), tokens.element_size(), n, _ptr(grad), _DTYPES[grad.dtype],
          spacing, scale, C.byref(g), int(add), _ptr(scratch), need)
    return out


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, weight, tokens, scale):
        ctx.save_for_backward(tokens)
        ctx.shape, ctx.scale = weight.shape, scale
        return _lookup(weight, tokens, scale)

    @staticmethod
    @_once
    def backward(ctx, g):
        tokens, = ctx.saved_tensors
        _no_tangent(g, "the gradient")
        return _gradient(tokens, g, ctx.scale, g.new_empty(ctx.shape), False), None, None


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
    grad[..., width] (a constant to autograd), for loops that run their own backward
    pass.  out: where it goes ([vocab, width], of grad's type or float32); with add, on
    top of what it holds (an output matrix that shares its weight, say), its other rows
    left alone."""
    _need_floats(grad, "grad")
    if grad.requires_grad and torch.is_grad_enabled():
        raise ValueError("grad is a constant to autograd: detach it")
    tokens = _token_ids(tokens, grad.device)
    if not grad.dim() or grad.shape[:-1] != tokens.shape:
        raise ValueError(f"grad has shape {tuple(grad.shape)}, expected {(*tokens.shape, 'width')}")
    if out is None:
        if vocab is None or add:
            raise ValueError("embedding_grad needs a vocab or an out, and out for add")
        out = grad.new_empty((vocab, grad.shape[-1]))
        return _gradient(tokens, grad, float(scale), out, False)
    _need_floats(out, "out")
    if out.requires_grad and torch.is_grad_enabled():
        raise ValueError("out has no gradient")
    if out.device != grad.device or out.dim() != 2 or out.shape != (out.shape[0] if vocab is None else vocab, grad.shape[-1]):
        raise ValueError("out must have grad's device and width, and the vocab")
    if out.dtype not in (grad.dtype, torch.float32):
        raise TypeError("out must have the type of grad, or be float32")
    _gradient(tokens, grad, float(scale), out, add)
    torch.autograd.graph.increment_version(out)  # autograd is told that it was written
    return out


# ---- the gradients' norm, and clipping ---------------------------------------------------


def _dense(t: torch.Tensor) -> bool:
    """Whether the tensor's elements fill their memory, in whatever order."""
    if t.is_contiguous():
        return True
    n = 1
    for stride, size in sorted((s, k) for k, s in zip(t.shape, t.stride()) if k != 1):
        if stride != n:
            return False
        n *= size
    return True


def _check_tensors(tensors, name: str) -> None:
    """Says what is wrong with a list that _tensor_list does not take."""
    for t in tensors:
        if not isinstance(t, torch.Tensor) or t.dtype not in _DTYPES or t.layout is not torch.strided:
            raise TypeError(f"{name} must be dense float32, bfloat16 or float16 tensors")
        if not t.is_cuda or t.device != tensors[0].device:
            raise ValueError(f"{name} must be on one GPU")
        if torch.is_grad_enabled() and t.requires_grad:
            raise ValueError(f"{name} need a gradient, which a norm here does not have: detach them")
        if not _dense(t):
            raise ValueError(f"{name} must fill their memory: call .contiguous()")


_PLAIN = {torch.Tensor, torch.nn.Parameter}


def _tensor_list(tensors, name: str) -> Tuple[List[torch.Tensor], array]:
    """The tensors and an array of dtl_tensor.  A model has hundreds of them: each
    attribute is read by one map over the list."""
    if isinstance(tensors, torch.Tensor):
        tensors = [tensors]
    tensors = [t for t in tensors if t is not None]
    if _tracing():
        raise RuntimeError("calls of the library cannot be recorded by torch.jit.trace")
    if getattr(forward_ad, "_current_level", 0) >= 0:
        for t in tensors:
            _no_tangent(t, name)
    table = array("Q", bytes(24 * len(tensors)))
    if not tensors:
        return tensors, table
    plain = set(map(type, tensors)) <= _PLAIN
    dtypes = set(map(_dtype_of, tensors)) if plain else ()
    if (not plain or not dtypes <= _DTYPES.keys() or set(map(_layout_of, tensors)) != {torch.strided}
            or len(places := set(map(torch.Tensor.get_device, tensors))) != 1 or -1 in places
            or torch.is_grad_enabled() and any(map(_requires_grad_of, tensors))
            or not all(map(torch.Tensor.is_contiguous, tensors))):
        _check_tensors(tensors, name)
        dtypes = set(map(_dtype_of, tensors))
    table[0::3] = array("Q", map(torch.Tensor.data_ptr, tensors))
    table[1::3] = array("Q", map(torch.Tensor.numel, tensors))
    if len(dtypes) == 1:
        table[2::3] = array("Q", [_DTYPES[tensors[0].dtype]]) * len(tensors)
    else:
        table[2::3] = array("Q", [_DTYPES[t.dtype] for t in tensors])
    return tensors, table


def _norm(grads, norm_type, scale, max_norm=None, out=None):
    grads, table = _tensor_list(grads, "grads")
    if norm_type not in (2, math.inf):
        raise ValueError("norm_type must be 2 or inf")
    if grads:
        beside = grads[0]
    else:  # the scale's device, or the current one
        beside = torch.empty(0, device=scale.device if isinstance(scale, torch.Tensor) and scale.is_cuda else "cuda")
    device = beside.device
    at = None
    if isinstance(scale, torch.Tensor):
        if scale.dtype != torch.float32 or scale.numel() != 1 or scale.device != device:
            raise ValueError("scale must be a number or one float32 on the gradients' device")
        _no_tangent(scale, "scale")
        if scale.requires_grad and torch.is_grad_enabled():
            raise ValueError("scale is a constant to autograd: detach it")
        at, scale = scale.data_ptr(), 0.0
    written = grads
    to = None
    if out is not None:
        written, to = _tensor_list(out, "out")
        if len(written) != len(grads):
            raise ValueError("out must have a tensor for each gradient")
        if written and written[0].device != device:
            raise ValueError("out must be on the gradients' device")
        if list(map(_shape_of, written)) != list(map(_shape_of, grads)):
            raise ValueError("out must have the gradients' shapes")
        if any(o != t and o != _lib.DTL_F32 for t, o in zip(table[2::3], to[2::3])):
            raise TypeError("out must have the gradients' types, or be float32")
        if list(map(torch.Tensor.stride, written)) != list(map(torch.Tensor.stride, grads)):
            for t, o in zip(grads, written):
                if o.stride() != t.stride() and not (o.is_contiguous() and t.is_contiguous()):
                    raise ValueError("out must have the gradients' strides")
    address = table.buffer_info()[0]
    norm = beside.new_empty((), dtype=torch.float32)
    need = lib.dtl_grad_norm_scratch(address, len(grads))
    scratch = beside.new_empty(need, dtype=torch.uint8)
    kind = int(norm_type == math.inf)
    if max_norm is None:
        _call(device, lib.dtl_grad_norm, address, len(grads), kind, scale, at, _ptr(norm), _ptr(scratch), need)
        return norm
    _call(device, lib.dtl_clip_grads, address, len(grads), kind, scale, at, max_norm,
          None if to is None else to.buffer_info()[0], _ptr(norm), _ptr(scratch), need)
    torch.autograd.graph.increment_version(written)  # autograd is told that they were written
    return norm


def grad_norm(grads: Union[torch.Tensor, Iterable[Optional[torch.Tensor]]], *, norm_type: float = 2.0,
              scale: Union[float, torch.Tensor] = 1.0) -> torch.Tensor:
    """dtl_grad_norm: scale times the norm over all elements of the tensors (float32,
    bfloat16 or float16, mixed as they come; None is left out), on the device: the 2-norm,
    summed in 64 bits, or with norm_type=inf the largest magnitude; 0 (on the scale's
    device, or the current one) where there are no tensors.  scale: what the gradients
    are to be multiplied by (1 / the loss scale), a number or one float32 on the device,
    a constant to autograd as the gradients are."""
    return _norm(grads, norm_type, scale if isinstance(scale, torch.Tensor) else float(scale))


def clip_grad_norm(grads: Union[torch.Tensor, Iterable[Optional[torch.Tensor]]], max_norm: float, *,
                   norm_type: float = 2.0, scale: Union[float, torch.Tensor] = 1.0,
                   out: Optional[Iterable[torch.Tensor]] = None) -> torch.Tensor:
    """dtl_clip_grads: the gradients times scale and, where grad_norm is above max_norm,
    times max_norm / (norm + 1e-6), in place; returns the norm on the device, without
    waiting for it.  out: where they go instead, a tensor for each, of their shapes and
    types or float32 (what an optimizer of float32 weights takes)."""
    return _norm(grads, norm_type, scale if isinstance(scale, torch.Tensor) else float(scale),
                 float(max_norm), out)
