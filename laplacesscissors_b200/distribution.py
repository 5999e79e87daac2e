"""Distributions over tokens from rows of logits on the device: log probabilities of
given tokens with the entropy and the top alternatives, distillation from a teacher's
top logits, and the gradients of both (lsx_token_logprobs_device and the entries
beside it, which state the formulas).

The reference scores one target per row on the host (attribution::loss,
src/attribution.rs:49-60); these work on torch CUDA tensors: `logits` [rows, vocab]
of float32, float16 or bfloat16 with unit stride along the vocabulary and any stride
between rows, token ids as int32 (-1 for an unused slot; another id outside the
vocabulary makes the results it enters NaN).  Calls enqueue on torch's current stream
on the Gpu's device, as torch's own operations do, copy nothing to the host and may be
captured into a CUDA graph.  `out` takes tensors to write instead of new ones, in the
order of the results (None where a result is not wanted); they count as modified in
place, so that torch's autograd notices where it had saved one.  A gradient is written
fastest into rows that lie to 16 bytes as the logits' do: for logits of padded rows into
an `out` of the same row stride, or over the logits (1000 x 50257 f16: 38 us, 137 into
contiguous rows).

Autograd does not record the calls.  Logits that require grad are refused where their
gradient would be lost without a word; a training step passes them on itself,
    step = distill(gpu, logits.detach(), ids, values, weights=w, gradient=True)
    logits.backward(step.gradient)
and likewise with token_logprobs and token_logprobs_backward."""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple

import torch

from ._lib import BF16, F16, F32, check, lib
from .gpu import Gpu

_KINDS = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}
_DEFAULT_STREAM = 1  # cudaStreamLegacy
# The raw handle that torch.cuda.current_stream wraps in an object, where torch has it by this name.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
    (lambda device: torch.cuda.current_stream(device).cuda_stream)
_F32, _I32 = torch.float32, torch.int32
_Tensor = torch.Tensor
_logprobs = lib.lsx_token_logprobs_device
_written = torch.autograd.graph.increment_version
MAX_SLOTS = 128  # given tokens, alternatives or teacher tokens per row


class TokenLogprobs(NamedTuple):
    logprob: torch.Tensor | None       # f32 [rows, n]: ln q of the given tokens
    entropy: torch.Tensor | None       # f32 [rows]
    stats: torch.Tensor | None         # f32 [rows, 2]: m and ln sum exp((z - m) / T)
    top_ids: torch.Tensor | None       # int32 [rows, k]
    top_logits: torch.Tensor | None    # f32 [rows, k]
    top_logprobs: torch.Tensor | None  # f32 [rows, k]


class Distillation(NamedTuple):
    loss: torch.Tensor | None      # f32 [rows]
    stats: torch.Tensor | None     # f32 [rows, 3]: m, ln sum, ln of the sum outside the teacher's list
    gradient: torch.Tensor | None  # [rows, vocab], the logits' dtype


def _rows(gpu: Gpu, logits: torch.Tensor, name: str = "logits"):
    """(rows, vocab, stride, kind) of a matrix of rows on the Gpu's device."""
    kind = _KINDS.get(logits.dtype) if isinstance(logits, _Tensor) and logits.dim() == 2 else None
    if kind is None:
        raise ValueError(f"{name} must be a [rows, vocab] tensor of float32, float16 or bfloat16")
    if logits.get_device() != gpu.device:
        raise ValueError(f"{name} must be on the Gpu's device")
    rows, vocab = logits.shape
    stride, unit = logits.stride()
    if vocab < 1:
        raise ValueError("check the vocabulary size")
    if unit != 1 and vocab > 1:
        raise ValueError(f"{name} must have unit stride along the vocabulary")
    if rows <= 1:
        stride = vocab
    elif stride < vocab:
        raise ValueError(f"rows of {name} must not overlap")
    return rows, vocab, stride, kind


def _vector(device: int, t: torch.Tensor, shape: tuple, dtype: torch.dtype, name: str) -> int:
    """Address of a contiguous tensor of this shape and type on the device."""
    if isinstance(t, _Tensor) and t.dtype is dtype and t.shape == shape and t.get_device() == device \
            and t.is_contiguous():
        return t.data_ptr()
    raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {list(shape)} on the Gpu's device")


def _count(t: torch.Tensor, rows: int, name: str) -> int:
    shape = t.shape if isinstance(t, _Tensor) else ()
    if len(shape) != 2 or shape[0] != rows or shape[1] > MAX_SLOTS:
        raise ValueError(f"{name} must be [rows, at most {MAX_SLOTS}]")
    return shape[1]


def _unrecorded(name: str):
    """Refuses a tensor that requires grad while gradients are recorded: autograd would not get this one."""
    if torch.is_grad_enabled():
        raise ValueError(f"{name} require grad, which autograd does not record here: pass {name}.detach(); gradients "
                         "with respect to the logits come from the calls that return them")


def _gradient(gpu: Gpu, logits: torch.Tensor, out: torch.Tensor | None):
    """The gradient's tensor and row stride; a new one is contiguous."""
    if out is None:
        out = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    elif out.shape != logits.shape or out.dtype != logits.dtype:
        raise ValueError("the gradient must have the logits' shape and dtype")
    return out, _rows(gpu, out, "the gradient")[2]


def _stream(device: int) -> int:
    """torch's current stream on the device, as lsx.h takes it."""
    return _raw_stream(device) or _DEFAULT_STREAM


def token_logprobs(gpu: Gpu, logits: torch.Tensor, tokens: torch.Tensor | None = None, *, alternatives: int = 0,
                   temperature: float = 1.0, out=None) -> TokenLogprobs:
    """Log probabilities of `tokens` (int32 [rows, n]), the entropy, the statistics
    (m, s) and the `alternatives` largest logits of each row, in descending order
    with the lower id first among equals (lsx_token_logprobs_device)."""
    rows, vocab, stride, kind = _rows(gpu, logits)
    if logits.requires_grad:
        _unrecorded("logits")
    n = _count(tokens, rows, "tokens") if tokens is not None else 0
    k = int(alternatives)
    if not 0 <= k <= MAX_SLOTS or k > vocab:
        raise ValueError(f"alternatives must be at most {MAX_SLOTS} and at most the vocabulary")
    if out is None:
        def new(wanted, *shape, dtype=_F32):
            return torch.empty(shape, dtype=dtype, device=logits.device) if wanted else None
        out = (new(n, rows, n), new(True, rows), new(True, rows, 2), new(k, rows, k, dtype=_I32), new(k, rows, k),
               new(k, rows, k))
    elif len(out) != 6:
        raise ValueError("out holds the six results")
    d = gpu.device
    logprob, entropy, stats, ids, values, logprobs = out
    if rows:
        check(_logprobs(
            gpu.handle, logits.data_ptr(), kind, rows, vocab, stride, temperature,
            _vector(d, tokens, (rows, n), _I32, "tokens") if n else None, n, k,
            None if logprob is None or not n else _vector(d, logprob, (rows, n), _F32, "out[0]"),
            None if entropy is None else _vector(d, entropy, (rows,), _F32, "out[1]"),
            None if stats is None else _vector(d, stats, (rows, 2), _F32, "out[2]"),
            None if ids is None or not k else _vector(d, ids, (rows, k), _I32, "out[3]"),
            None if values is None or not k else _vector(d, values, (rows, k), _F32, "out[4]"),
            None if logprobs is None or not k else _vector(d, logprobs, (rows, k), _F32, "out[5]"), _stream(d)))
        if n and k and not (logprob is None or entropy is None or stats is None or ids is None or values is None
                            or logprobs is None):
            _written(out)
        else:
            _written([t for t, count in zip(out, (n, 1, 1, k, k, k)) if count and t is not None])
    return TokenLogprobs(logprob, entropy, stats, ids, values, logprobs)


def token_logprobs_backward(gpu: Gpu, logits: torch.Tensor, tokens: torch.Tensor | None, stats: torch.Tensor,
                            entropy: torch.Tensor | None, logprob_gradient: torch.Tensor | None,
                            entropy_gradient: torch.Tensor | None = None, *, temperature: float = 1.0,
                            out: torch.Tensor | None = None) -> torch.Tensor:
    """Gradient with respect to the logits of sum(logprob_gradient * logprob) +
    sum(entropy_gradient * entropy), from token_logprobs' stats and entropy
    (lsx_token_logprobs_backward_device).  `out` may be the logits themselves."""
    rows, vocab, stride, kind = _rows(gpu, logits)
    n = _count(tokens, rows, "tokens") if tokens is not None else 0
    out, out_stride = _gradient(gpu, logits, out)
    if entropy_gradient is None:
        entropy = None
    at = (_vector(gpu.device, tokens, (rows, n), _I32, "tokens") if n else None, n,
          _vector(gpu.device, stats, (rows, 2), _F32, "stats"),
          _vector(gpu.device, entropy, (rows,), _F32, "entropy") if entropy_gradient is not None else None,
          _vector(gpu.device, logprob_gradient, (rows, n), _F32, "logprob_gradient") if n else None,
          _vector(gpu.device, entropy_gradient, (rows,), _F32, "entropy_gradient") if entropy_gradient is not None else None)
    if rows:
        check(lib.lsx_token_logprobs_backward_device(gpu.handle, logits.data_ptr(), kind, rows, vocab, stride,
                                                     temperature, *at, out.data_ptr(), out_stride, _stream(gpu.device)))
        _written((out,))
    return out


def _teacher(gpu: Gpu, rows: int, ids, values, stats):
    k = _count(ids, rows, "teacher_ids")
    if k < 1:
        raise ValueError("the teacher lists at least one token")
    return (_vector(gpu.device, ids, (rows, k), _I32, "teacher_ids"),
            _vector(gpu.device, values, (rows, k), _F32, "teacher_logits"), k,
            _vector(gpu.device, stats, (rows, 2), _F32, "teacher_stats") if stats is not None else None)


def distill(gpu: Gpu, logits: torch.Tensor, teacher_ids: torch.Tensor, teacher_logits: torch.Tensor, *,
            teacher_stats: torch.Tensor | None = None, weights: torch.Tensor | None = None, temperature: float = 1.0,
            gradient: bool = False, out=None) -> Distillation:
    """Divergence of the student's rows from a teacher's top tokens
    (lsx_distill_device): teacher_ids int32 and teacher_logits f32 [rows, k],
    teacher_stats [rows, 2] the teacher's statistics at the same temperature (with
    them the tokens outside the list count as one outcome, left out only where the
    student masks them all; without them the teacher is normalised over its list).  With `gradient` also the gradient of
    weights * loss with respect to the logits, which out[2] may be."""
    rows, vocab, stride, kind = _rows(gpu, logits)
    teacher = _teacher(gpu, rows, teacher_ids, teacher_logits, teacher_stats)
    if not gradient and (logits.requires_grad or teacher_logits.requires_grad):
        _unrecorded("logits" if logits.requires_grad else "teacher_logits")
    if weights is not None and not gradient:
        raise ValueError("weights scale the gradient only")
    if out is None:
        out = (torch.empty(rows, dtype=_F32, device=logits.device),
               torch.empty((rows, 3), dtype=_F32, device=logits.device), None)
    elif len(out) != 3 or (out[2] is not None and not gradient):
        raise ValueError("out holds the three results, the last only with the gradient")
    grad, grad_stride = _gradient(gpu, logits, out[2]) if gradient else (None, 0)
    at = (_vector(gpu.device, weights, (rows,), _F32, "weights") if weights is not None else None,
          _vector(gpu.device, out[0], (rows,), _F32, "out[0]") if out[0] is not None else None,
          _vector(gpu.device, out[1], (rows, 3), _F32, "out[1]") if out[1] is not None else None)
    if rows:
        check(lib.lsx_distill_device(gpu.handle, logits.data_ptr(), kind, rows, vocab, stride, temperature, *teacher,
                                     *at, grad.data_ptr() if gradient else None, grad_stride, _stream(gpu.device)))
        if out[0] is None or out[1] is None:
            _written([t for t in (*out[:2], grad) if t is not None])
        else:
            _written((out[0], out[1], grad) if gradient else out[:2])
    return Distillation(out[0], out[1], grad)


def distill_backward(gpu: Gpu, logits: torch.Tensor, teacher_ids: torch.Tensor, teacher_logits: torch.Tensor,
                     stats: torch.Tensor, loss_gradient: torch.Tensor, *, teacher_stats: torch.Tensor | None = None,
                     temperature: float = 1.0, out: torch.Tensor | None = None) -> torch.Tensor:
    """Gradient of sum(loss_gradient * loss) with respect to the logits, from
    distill's stats (lsx_distill_backward_device).  `out` may be the logits."""
    rows, vocab, stride, kind = _rows(gpu, logits)
    teacher = _teacher(gpu, rows, teacher_ids, teacher_logits, teacher_stats)
    out, out_stride = _gradient(gpu, logits, out)
    at = (_vector(gpu.device, stats, (rows, 3), _F32, "stats"),
          _vector(gpu.device, loss_gradient, (rows,), _F32, "loss_gradient"))
    if rows:
        check(lib.lsx_distill_backward_device(gpu.handle, logits.data_ptr(), kind, rows, vocab, stride, temperature,
                                              *teacher, *at, out.data_ptr(), out_stride, _stream(gpu.device)))
        _written((out,))
    return out


__all__ = ["TokenLogprobs", "Distillation", "token_logprobs", "token_logprobs_backward", "distill",
           "distill_backward", "MAX_SLOTS"]
