"""Scores of given tokens and distillation on logits held in torch tensors.

For programs that have a model's logits on the GPU as a torch tensor: what the
rows say of given tokens (log probability, entropy, top alternatives), and the
loss that moves a student towards a teacher's top alternatives, both with
gradients.  The calls enqueue the library's kernels (dtl_token_scores*,
dtl_distill* of include/detllm.h, which define every result) on the current
stream of the logits' device, do not wait, and can be captured into a graph (a
captured backward needs a leaf of its own, `logits.detach().requires_grad_()`: one
whose eager graph is still alive belongs to that graph's stream).  Reverse mode only:
tensors with a forward-mode tangent and torch.jit.trace are refused; in a function
given to torch.compile they stand inside torch.compiler.disable.

    teacher = scores.token_scores(teacher_logits, tokens, top=32, temperature=2.0)
    loss = scores.distill_loss(student_logits, teacher.top_ids, teacher.top_log_probs,
                               temperature=2.0, rest=True).mean()
    loss.backward()

`Session.token_scores` and `F32Llama.scores_for_tokens_chunked` (model.py) give
the same for this library's own sessions, without torch.
"""
from __future__ import annotations

import ctypes as C
from functools import lru_cache
from typing import NamedTuple, Optional, Tuple

import torch
from torch.autograd import forward_ad

from . import _lib
from ._lib import DetllmError, check, lib


def _one_hip_runtime() -> None:
    """torch brings a HIP runtime of its own; the library shares it if torch was
    loaded first.  Streams of one runtime mean nothing to another."""
    with open("/proc/self/maps") as f:
        found = sorted({line.split(None, 5)[5].strip() for line in f if "libamdhip64" in line})
    if len(found) > 1:
        raise ImportError(f"two HIP runtimes are loaded ({', '.join(found)}): import torch before detllm_amd")


_one_hip_runtime()

MAX_TOP = 128
MAX_TEACHER = 256

_DTYPES = {torch.float32: _lib.DTL_F32, torch.bfloat16: _lib.DTL_BF16, torch.float16: _lib.DTL_F16}


class TokenScores(NamedTuple):
    """Per row (the logits' leading dimensions): log probability of the row's
    token, entropy, ids and log probabilities of the `top` largest logits."""

    log_probs: Optional[torch.Tensor]
    entropy: torch.Tensor
    top_ids: Optional[torch.Tensor]
    top_log_probs: Optional[torch.Tensor]


def _no_tangent(t: torch.Tensor, name: str) -> None:
    """The kernels see a tensor's values alone: the tangent of a dual tensor would be
    lost, and torch takes a missing one for zero."""
    if getattr(forward_ad, "_current_level", 0) >= 0 and forward_ad.unpack_dual(t).tangent is not None:
        raise NotImplementedError(f"{name} has a tangent: there is no forward-mode derivative")


# Without its wrapper, as _device_now below.
_tracing = getattr(torch._C, "_is_tracing", None) or torch.jit.is_tracing


def _need_logits(t: torch.Tensor) -> None:
    """What a call asks of its logits first, before autograd unpacks them."""
    if not isinstance(t, torch.Tensor) or t.dtype not in _DTYPES:
        raise TypeError("logits must be a float32, bfloat16 or float16 tensor")
    _no_tangent(t, "logits")
    if _tracing():
        raise RuntimeError("calls of the library cannot be recorded by torch.jit.trace")


def _logits_view(t: torch.Tensor, name: str = "logits") -> _lib.Logits:
    """The tensor's rows as a dtl_logits."""
    if not t.is_cuda:
        raise ValueError(f"{name} must be on the GPU")
    shape, strides = t.shape, t.stride()
    if not shape or shape[-1] == 0:
        raise ValueError(f"{name} needs a vocabulary in its last dimension")
    vocab = shape[-1]
    if vocab > 1 and strides[-1] != 1:
        raise ValueError(f"the last dimension of {name} must be contiguous")
    rows, stride = 1, vocab
    for n, s in zip(reversed(shape[:-1]), reversed(strides[:-1])):
        if n == 1:
            continue
        if rows == 1:
            stride = s
        elif s != rows * stride and n and rows:
            raise ValueError(f"the rows of {name} are not evenly spaced: call .contiguous()")
        rows *= n
    if rows > 1 and stride < vocab:
        raise ValueError(f"the rows of {name} overlap: call .contiguous()")
    return _lib.Logits(t.data_ptr(), _DTYPES[t.dtype], rows, vocab, stride)


def _beside(t: torch.Tensor, logits: torch.Tensor, shape, dtypes, name: str) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or t.dtype not in dtypes:
        raise TypeError(f"{name} must be a tensor of {' or '.join(str(d) for d in dtypes)}")
    _no_tangent(t, name)
    if t.device != logits.device:
        raise ValueError(f"{name} and logits are on different devices")
    if t.shape != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    return t.contiguous()


_INDEX = (torch.int64, torch.int32)
_FLOAT = (torch.float32,)


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


# Without their wrappers: a call on a few rows is as short as its host side.
_device_now = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
_stream_of = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def _call(device: torch.device, entry, *args) -> None:
    """The entry point on the current stream of `device`."""
    index = device.index
    if index == _device_now():
        status = entry(*args, _stream_of(index))
    else:
        with torch.cuda.device(index):
            status = entry(*args, _stream_of(index))
    if status:
        check(status, entry.__name__)


_scores_scratch = lru_cache(maxsize=256)(lib.dtl_token_scores_scratch)
_distill_scratch = lru_cache(maxsize=256)(lib.dtl_distill_scratch)


def _scratch(n: int, device: torch.device) -> Optional[torch.Tensor]:
    return torch.empty(n, dtype=torch.uint8, device=device) if n else None


def _incoming(g: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """The gradient that a backward is given."""
    if g is None:
        return None
    _no_tangent(g, "the gradient")
    return g.contiguous()


# ---- scores ------------------------------------------------------------------


def _scores(logits, tokens, top, temperature, stats):
    z = _logits_view(logits)
    if not 0 <= top <= min(MAX_TOP, z.vocab):
        raise DetllmError(1, "token_scores: top")
    lead, dev = logits.shape[:-1], logits.device
    log_probs = torch.empty(lead, dtype=torch.float32, device=dev) if tokens is not None else None
    entropy = torch.empty(lead, dtype=torch.float32, device=dev)
    ids = lps = st = None
    if top:
        ids = torch.empty((*lead, top), dtype=torch.int32, device=dev)
        lps = torch.empty((*lead, top), dtype=torch.float32, device=dev)
    if stats:
        st = torch.empty((z.rows, 2), dtype=torch.float32, device=dev)
    n = _scores_scratch(z.rows, z.vocab, top)
    scratch = _scratch(n, dev)
    _call(dev, lib.dtl_token_scores, C.byref(z), _ptr(tokens), 0 if tokens is None else tokens.element_size(),
          temperature, top, _ptr(log_probs), _ptr(entropy), _ptr(st), _ptr(ids), _ptr(lps), _ptr(scratch), n)
    return log_probs, entropy, ids, lps, st


class _TokenScores(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, top, temperature):
        log_probs, entropy, ids, lps, stats = _scores(logits, tokens, top, temperature, True)
        ctx.save_for_backward(logits, tokens, stats, entropy)
        ctx.temperature = temperature
        ctx.set_materialize_grads(False)
        if top:
            ctx.mark_non_differentiable(ids, lps)
        return log_probs, entropy, ids, lps

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g, h, _ids, _lps):
        logits, tokens, stats, entropy = ctx.saved_tensors
        grad = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        g = _incoming(g)
        h = _incoming(h)
        z = _logits_view(logits)
        _call(logits.device, lib.dtl_token_scores_backward, C.byref(z), _ptr(tokens),
              0 if tokens is None else tokens.element_size(), ctx.temperature, _ptr(stats), _ptr(entropy), _ptr(g),
              _ptr(h), _ptr(grad), z.vocab)
        return grad, None, None, None


def token_scores(logits: torch.Tensor, tokens: Optional[torch.Tensor] = None, *, top: int = 0,
                 temperature: float = 1.0) -> TokenScores:
    """dtl_token_scores of logits[..., vocab] (float32, bfloat16 or float16) and
    tokens[...] (int64 or int32; -1 is padding): log probabilities and entropy in
    float32, differentiable, and the `top` (up to 128) alternatives of each row,
    which are constants to autograd.  With p = softmax(logits / temperature)."""
    _need_logits(logits)
    if tokens is not None:
        tokens = _beside(tokens, logits, logits.shape[:-1], _INDEX, "tokens")
    if torch.is_grad_enabled() and logits.requires_grad:
        return TokenScores(*_TokenScores.apply(logits, tokens, int(top), float(temperature)))
    return TokenScores(*_scores(logits, tokens, int(top), float(temperature), False)[:4])


# ---- distillation ---------------------------------------------------------------


def _teacher(logits, ids, log_probs, rest):
    k = ids.shape[-1] if isinstance(ids, torch.Tensor) and ids.dim() else 0
    shape = (*logits.shape[:-1], k)
    ids = _beside(ids, logits, shape, _INDEX, "teacher_ids")
    log_probs = _beside(log_probs, logits, shape, _FLOAT, "teacher_log_probs")
    return _teacher_view(ids, log_probs, rest), ids, log_probs


def _teacher_view(ids, log_probs, rest) -> _lib.Teacher:
    return _lib.Teacher(ids.data_ptr(), ids.element_size(), log_probs.data_ptr(), ids.shape[-1], int(bool(rest)))


def _distill(logits, ids, log_probs, temperature, rest, stats):
    z = _logits_view(logits)
    t, ids, log_probs = _teacher(logits, ids, log_probs, rest)
    dev = logits.device
    loss = torch.empty(logits.shape[:-1], dtype=torch.float32, device=dev)
    st = torch.empty(z.rows, 5, dtype=torch.float32, device=dev) if stats else None
    n = _distill_scratch(z.rows, z.vocab)
    scratch = _scratch(n, dev)
    _call(dev, lib.dtl_distill, C.byref(z), C.byref(t), temperature, _ptr(loss), _ptr(st), _ptr(scratch), n)
    return loss, ids, log_probs, st


class _Distill(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, ids, log_probs, temperature, rest):
        loss, ids, log_probs, stats = _distill(logits, ids, log_probs, temperature, rest, True)
        ctx.save_for_backward(logits, ids, log_probs, stats)
        ctx.temperature, ctx.rest = temperature, rest
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        logits, ids, log_probs, stats = ctx.saved_tensors
        grad = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        z = _logits_view(logits)
        t = _teacher_view(ids, log_probs, ctx.rest)
        g = _incoming(g)
        _call(logits.device, lib.dtl_distill_backward, C.byref(z), C.byref(t), ctx.temperature, _ptr(stats), _ptr(g),
              _ptr(grad), z.vocab)
        return grad, None, None, None, None


def distill_loss(logits: torch.Tensor, teacher_ids: torch.Tensor, teacher_log_probs: torch.Tensor, *,
                 temperature: float = 1.0, rest: bool = False) -> torch.Tensor:
    """dtl_distill: each row's loss of logits[..., vocab] against teacher_ids
    and teacher_log_probs[..., k] (k up to 256), differentiable in the logits.

    teacher_log_probs (float32) are at this temperature, as token_scores with
    the same temperature gives them, and constants to autograd.  rest=False
    compares within the list's renormalised probabilities; rest=True keeps them as
    they are and compares what lies outside the list as one more outcome."""
    _need_logits(logits)
    if torch.is_grad_enabled() and logits.requires_grad:
        return _Distill.apply(logits, teacher_ids, teacher_log_probs, float(temperature), bool(rest))
    return _distill(logits, teacher_ids, teacher_log_probs, float(temperature), rest, False)[0]


def distill_loss_and_grad(logits: torch.Tensor, teacher_ids: torch.Tensor, teacher_log_probs: torch.Tensor,
                          weights: Optional[torch.Tensor] = None, *, temperature: float = 1.0, rest: bool = False,
                          out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """dtl_distill_step: (weights * distill_loss, the gradient of its sum), for
    loops that know the rows' weights (1 / rows for a mean, 0 for padding; None:
    ones) before the loss.  One pass instead of a forward and a backward; pass the
    gradient on with `logits.backward(grad)`.  out: where the gradient goes, of the
    logits' shape and type; the logits themselves if nothing needs them again, but
    not memory that holds other rows' or only a part of them."""
    _need_logits(logits)
    z = _logits_view(logits)
    t, teacher_ids, teacher_log_probs = _teacher(logits, teacher_ids, teacher_log_probs, rest)
    dev = logits.device
    if weights is not None:
        weights = _beside(weights, logits, logits.shape[:-1], _FLOAT, "weights")
    given = out is not None
    if not given:
        out = torch.empty(logits.shape, dtype=logits.dtype, device=dev)
        stride = z.vocab
    else:
        if out.shape != logits.shape or out.dtype != logits.dtype or out.device != dev:
            raise ValueError("out must have the shape, type and device of logits")
        _no_tangent(out, "out")
        stride = _logits_view(out, "out").stride
    loss = torch.empty(logits.shape[:-1], dtype=torch.float32, device=dev)
    n = _distill_scratch(z.rows, z.vocab)
    scratch = _scratch(n, dev)
    _call(dev, lib.dtl_distill_step, C.byref(z), C.byref(t), float(temperature), _ptr(weights), _ptr(loss),
          out.data_ptr(), stride, _ptr(scratch), n)
    if given:  # autograd is told that it was written
        torch.autograd.graph.increment_version(out)
    return loss, out
