"""Scores of given tokens, distillation, and penalties and masks on logits held in
torch tensors.

For programs that have a model's logits on the GPU as a torch tensor: what the
rows say of given tokens (log probability, entropy, top alternatives), the
loss that moves a student towards a teacher's top alternatives, and what is done
to the rows before either (penalties for repeated tokens, biases, masks), all with
gradients.  The calls enqueue the library's kernels (dtl_token_scores*,
dtl_distill*, dtl_adjust_logits* of include/detllm.h, which define every result) on
the current stream of the logits' device, do not wait, and can be captured into a graph (a
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
from functools import lru_cache, wraps
from typing import NamedTuple, Optional, Tuple, Union

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
_MASK = (torch.int32, torch.bool)


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


# ---- penalties, biases, masks -------------------------------------------------------


def _spaced(t):
    """A tensor whose rows are used as they lie, and how far they are apart (0: one for all):
    the first places of a longer buffer are not copied."""
    if t.dim() == 2 and t.stride(1) == 1:
        return t, t.stride(0)
    return t.contiguous(), 0 if t.dim() == 1 else t.shape[-1]


class _By:
    """A dtl_adjust and the tensors that it points to."""

    def __init__(self, logits, vocab, history, prompt, repetition, presence, frequency, bias_ids, bias, allowed):
        a = self.struct = _lib.Adjust()
        self.lead, self.device = logits.shape[:-1], logits.device
        self.dual = getattr(forward_ad, "_current_level", 0) >= 0
        rows = presences = frequencies = None
        if history is not None:
            history, n, a.history_stride = self.rows(history, _INDEX, "history")
            a.history, a.history_bytes, a.history_len = history.data_ptr(), history.element_size(), n
            if prompt is not None:
                prompt = self.tensor(prompt, _INDEX, "prompt", self.lead)
                if prompt.dtype == torch.int64:  # a place past 32 bits stays behind the history's last
                    prompt = prompt.clamp(0, n).int()
                prompt = prompt.contiguous()
                a.prompt = prompt.data_ptr()
        elif prompt is not None:
            raise ValueError("prompt counts places of a history")
        if isinstance(repetition, torch.Tensor):
            rows = self.constant(repetition, "repetition", self.lead)
            a.repetitions = rows.data_ptr()
        else:
            a.repetition = float(repetition)
        if isinstance(presence, torch.Tensor):
            presences = self.constant(presence, "presence", self.lead)
            a.presences = presences.data_ptr()
        else:
            a.presence = float(presence)
        if isinstance(frequency, torch.Tensor):
            frequencies = self.constant(frequency, "frequency", self.lead)
            a.frequencies = frequencies.data_ptr()
        else:
            a.frequency = float(frequency)
        if (bias_ids is None) != (bias is None):
            raise ValueError("bias_ids and bias belong together")
        if bias is not None:
            bias = self.constant(bias, "bias", bias_ids.shape if isinstance(bias_ids, torch.Tensor) else None)
            bias_ids, a.bias_len, _ = self.rows(bias_ids, _INDEX, "bias_ids")
            bias_ids = bias_ids.contiguous()  # one spacing for both
            a.bias_stride = 0 if bias_ids.dim() == 1 else a.bias_len
            a.bias_ids, a.bias_bytes, a.biases = bias_ids.data_ptr(), bias_ids.element_size(), bias.data_ptr()
        if allowed is not None:
            allowed, n, a.allowed_stride = self.rows(allowed, _MASK, "allowed")
            a.allowed_bits = 1 if allowed.dtype == torch.int32 else 8
            if n != (vocab if a.allowed_bits == 8 else -(-vocab // 32)):
                raise ValueError(f"allowed has {n} entries in a row, expected one for each logit or 32")
            a.allowed = allowed.data_ptr()
        self.tensors = (history, prompt, rows, presences, frequencies, bias_ids, bias, allowed)

    def tensor(self, t, dtypes, name, shape=None) -> torch.Tensor:
        """As _beside; of any shape where none is given."""
        if not isinstance(t, torch.Tensor) or t.dtype not in dtypes:
            raise TypeError(f"{name} must be a tensor of {' or '.join(str(d) for d in dtypes)}")
        if self.dual:
            _no_tangent(t, name)
        if t.device != self.device:
            raise ValueError(f"{name} and logits are on different devices")
        if shape is not None and t.shape != shape:
            raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
        return t

    def rows(self, t, dtypes, name):
        """A tensor of the logits' leading dimensions and one more, or of one dimension for
        every row; its row's length, and how far rows are apart."""
        shape = self.tensor(t, dtypes, name).shape
        if len(shape) != 1 and (not shape or shape[:-1] != self.lead):
            raise ValueError(f"{name} has shape {tuple(shape)}, expected {(*self.lead, 'n')} or ('n',)")
        t, stride = _spaced(t)
        return t, shape[-1], stride

    def constant(self, t, name, shape):
        t = self.tensor(t, _FLOAT, name, shape)
        if t.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"{name} is a constant to autograd: detach it")
        return t.contiguous()

    def for_backward(self):
        """What the gradient needs: whether a token stood in the history, and the mask."""
        history, _, rows, _, _, _, _, allowed = self.tensors
        if history is None or self.struct.repetition == 1.0 and rows is None:
            return None, None, allowed
        return history, rows, allowed


def _adjust(z, by, out, stride, device):
    _call(device, lib.dtl_adjust_logits, C.byref(z), C.byref(by.struct), out.data_ptr(), stride)


def _once(backward):
    """once_differentiable, without its wrapper where no second derivative can follow."""
    guarded = torch.autograd.function.once_differentiable(backward)

    @wraps(backward)
    def run(ctx, g):
        return guarded(ctx, g) if torch.is_grad_enabled() else backward(ctx, g)

    return run


class _Adjust(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, z, by):
        out = logits.new_empty(logits.shape)
        _adjust(z, by, out, z.vocab, logits.device)
        history, rows, allowed = by.for_backward()
        # without repetitions a logit's sign does not matter, only where it is
        ctx.save_for_backward(logits if history is not None else None, history, rows, allowed)
        ctx.repetition = by.struct.repetition
        return out

    @staticmethod
    @_once
    def backward(ctx, g):
        logits, history, rows, allowed = ctx.saved_tensors
        g = _incoming(g)
        if history is None and allowed is None:
            return g, None, None
        shape = g.shape
        grad = g.new_empty(shape)
        a, V = _lib.Adjust(), shape[-1]
        a.repetition = ctx.repetition
        if history is not None:
            history, a.history_stride = _spaced(history)
            a.history, a.history_bytes, a.history_len = history.data_ptr(), history.element_size(), history.shape[-1]
            a.repetitions = _ptr(rows)
        if allowed is not None:
            allowed, a.allowed_stride = _spaced(allowed)
            a.allowed, a.allowed_bits = allowed.data_ptr(), 8 if allowed.dtype == torch.bool else 1
        gv = _lib.Logits(g.data_ptr(), _DTYPES[g.dtype], g.numel() // V, V, V)
        z = gv if logits is None else _logits_view(logits)
        _call(g.device, lib.dtl_adjust_logits_backward, C.byref(z), C.byref(a), gv.data, V, grad.data_ptr(), V)
        return grad, None, None


def adjust_logits(logits: torch.Tensor, *, history: Optional[torch.Tensor] = None, prompt: Optional[torch.Tensor] = None,
                  repetition: Union[float, torch.Tensor] = 1.0, presence: Union[float, torch.Tensor] = 0.0,
                  frequency: Union[float, torch.Tensor] = 0.0, bias_ids: Optional[torch.Tensor] = None,
                  bias: Optional[torch.Tensor] = None, allowed: Optional[torch.Tensor] = None,
                  out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """dtl_adjust_logits of logits[..., vocab]: what is done to rows before they are
    scored, drawn from or trained on; differentiable in the logits.

    history[..., n] or [n] (int64 or int32; -1 is no token): a token in it is
    divided by `repetition` (multiplied, where its logit is negative), and loses
    presence + frequency * its count.  The first prompt[...] places are a prompt,
    which counts for the repetition alone.  The three are numbers, or float32 tensors
    with one for each row.  bias_ids and bias[..., k] or [k]: what is added to listed
    tokens (of an id listed twice the later place).  allowed: int32 words of
    32 bits [..., ceil(vocab / 32)], or bool [..., vocab], or of one row for all;
    what it does not allow becomes -inf.

    out: where the result goes, of the logits' shape and type; the logits themselves,
    whose unchanged places are then not written.  It has no gradient."""
    _need_logits(logits)
    z = _logits_view(logits)
    by = _By(logits, z.vocab, history, prompt, repetition, presence, frequency, bias_ids, bias, allowed)
    grad = torch.is_grad_enabled() and logits.requires_grad
    if out is None:
        if grad:
            return _Adjust.apply(logits, z, by)
        out = logits.new_empty(logits.shape)
        _adjust(z, by, out, z.vocab, logits.device)
        return out
    if grad or out.requires_grad and torch.is_grad_enabled():
        raise ValueError("out has no gradient: leave it out, or call under torch.no_grad()")
    if out.shape != logits.shape or out.dtype != logits.dtype or out.device != logits.device:
        raise ValueError("out must have the shape, type and device of logits")
    _no_tangent(out, "out")
    _adjust(z, by, out, _logits_view(out, "out").stride, logits.device)
    torch.autograd.graph.increment_version(out)  # autograd is told that it was written
    return out
