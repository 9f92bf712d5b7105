"""Log probabilities of chosen tokens, and the preference loss on them (``csrc/token_logprob.hip``,
``csrc/preference.hip``; ``keras.losses.PreferenceLoss`` is the loss object).

``token_log_probs`` turns logits over a vocabulary -- or over the items of a ranked list -- into the log probability of
the token (item) that was chosen; sums of them over an answer are what preferences between answers are trained on.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib
from . import _ops
from ._ops import _ptr, _stream, require_device
from .embedding import _dtype_code, _same_device

KINDS = {'logistic': 0, 'hinge': 1, 'squared': 2}                          # TFR_PREFERENCE_*
MAX_ANSWERS = 64


def _rows(logits: torch.Tensor, targets: torch.Tensor):
    """(logits, per, stride_b, stride_t, dense int64 targets): the rows of logits [..., V] as two strided axes."""
    require_device(logits, 'logits')
    require_device(targets, 'targets')
    _same_device(logits, targets, 'logits', 'targets')
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError('logits must be [..., vocab], got shape %s' % (tuple(logits.shape),))
    if targets.dtype not in (torch.int32, torch.int64):
        raise ValueError('targets must be int32 or int64, got %s' % targets.dtype)
    if tuple(targets.shape) != tuple(logits.shape[:-1]):
        raise ValueError('targets of shape %s do not fit logits of shape %s' % (tuple(targets.shape), tuple(logits.shape)))
    if logits.stride(-1) != 1 and logits.shape[-1] > 1 or logits.dim() > 3:
        logits = logits.contiguous()
    if logits.dim() > 3:
        logits = logits.reshape(-1, logits.shape[-1])
    if logits.dim() == 1:
        per, stride_b, stride_t = 1, 0, 0
    elif logits.dim() == 2:
        per, stride_b, stride_t = max(1, logits.shape[0]), 0, logits.stride(0)
    else:
        per, stride_b, stride_t = max(1, logits.shape[1]), logits.stride(0), logits.stride(1)
    return logits, per, stride_b, stride_t, targets.to(torch.int64).contiguous()


def _temperature(t) -> float:
    t = float(t)
    if not 1e-30 <= t <= 1e30:
        raise ValueError('temperature must be positive, got %r' % t)
    return t


def _limits(n: int, vocab: int) -> None:
    if n >= 1 << 24 or vocab > 1 << 28:
        raise ValueError('at most 2^24 - 1 rows of 2^28 logits, got %d of %d' % (n, vocab))


@_ops.device_guarded
def _log_probs(logits, targets, temperature, want_stats):
    code = _dtype_code(logits, 'logits')
    shape, vocab = tuple(logits.shape[:-1]), logits.shape[-1]
    logits, per, sb, st, targets = _rows(logits, targets)
    n = targets.numel()
    _limits(n, vocab)
    lib = _lib.load()
    logp = torch.empty(shape, dtype=torch.float32, device=logits.device)
    stats = torch.empty(shape + (2,), dtype=torch.float32, device=logits.device) if want_stats else None
    nbytes = lib.tfr_token_logprob_workspace_bytes(n, vocab)
    workspace = torch.empty((nbytes,), dtype=torch.uint8, device=logits.device) if nbytes > 0 else None
    rc = lib.tfr_token_logprob(_ptr(logits), code, per, sb, st, _ptr(targets), n, vocab, _temperature(temperature), _ptr(logp), _ptr(stats),
                               _ptr(workspace), nbytes, _stream())
    _lib.check(rc, 'tfr_token_logprob')
    return logp, stats


def token_log_probs_with_stats(logits: torch.Tensor, targets: torch.Tensor, temperature: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """``token_log_probs`` without autograd, and the row statistics ``[..., 2]`` that ``token_log_probs_grad`` takes."""
    return _log_probs(logits.detach(), targets, temperature, True)


@_ops.device_guarded
def token_log_probs_grad(grad: torch.Tensor, logits: torch.Tensor, targets: torch.Tensor, stats: torch.Tensor,
                         temperature: float = 1.0) -> torch.Tensor:
    """``d sum(grad * token_log_probs) / d logits`` as a dense tensor of ``logits``' shape and type."""
    require_device(grad, 'grad')
    code = _dtype_code(logits, 'logits')
    shape, vocab = tuple(logits.shape), logits.shape[-1]
    logits, per, sb, st, targets = _rows(logits, targets)
    _same_device(grad, logits, 'grad', 'logits')
    if tuple(grad.shape) != shape[:-1] or tuple(stats.shape) != shape[:-1] + (2,) or stats.dtype != torch.float32:
        raise ValueError('grad of shape %s and stats of shape %s do not fit logits of shape %s'
                         % (tuple(grad.shape), tuple(stats.shape), shape))
    _same_device(require_device(stats, 'stats'), logits, 'stats', 'logits')
    grad, stats = _ops._f32(grad, 'grad'), stats.contiguous()
    n = targets.numel()
    _limits(n, vocab)
    out = torch.empty(shape, dtype=logits.dtype, device=logits.device)
    rc = _lib.load().tfr_token_logprob_grad(_ptr(logits), code, per, sb, st, _ptr(targets), _ptr(stats), _ptr(grad), n, vocab,
                                            _temperature(temperature), _ptr(out), _stream())
    _lib.check(rc, 'tfr_token_logprob_grad')
    return out


class _TokenLogProbsFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, temperature):
        logp, stats = _log_probs(logits, targets, temperature, True)
        ctx.save_for_backward(logits, targets, stats)
        ctx.temperature = temperature
        return logp

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        logits, targets, stats = ctx.saved_tensors
        return token_log_probs_grad(g, logits, targets, stats, ctx.temperature), None, None


def token_log_probs(logits: torch.Tensor, targets: torch.Tensor, temperature: float = 1.0) -> torch.Tensor:
    """``log softmax(logits / temperature)[targets]``: logits ``[..., vocab]`` (float32, bfloat16, float16; rows of any
    stride), targets ``[...]`` -> float32 ``[...]``.  A target below 0 is no target: 0, no gradient, its row is not read.
    A target beyond the vocabulary gives NaN.  Differentiable with respect to ``logits``."""
    require_device(logits, 'logits')
    if torch.is_grad_enabled() and logits.requires_grad:
        return _TokenLogProbsFn.apply(logits, targets, temperature)
    return _log_probs(logits, targets, temperature, False)[0]


@_ops.device_guarded
def preference_loss(log_probs: torch.Tensor, labels: torch.Tensor, reference: Optional[torch.Tensor] = None,
                    mask: Optional[torch.Tensor] = None, list_weights: Optional[torch.Tensor] = None, kind: str = 'logistic',
                    beta: float = 0.1, label_smoothing: float = 0.0, length_normalized: bool = False,
                    scale: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """(loss ``[B]``, coefficients ``[B, L]`` of ``preference_grad``) of token log probabilities ``[B, L, T]`` fp32."""
    B, L, T = log_probs.shape
    lib = _lib.load()
    loss = torch.empty((B,), dtype=torch.float32, device=log_probs.device)
    coef = torch.empty((B, L), dtype=torch.float32, device=log_probs.device)
    nbytes = lib.tfr_preference_workspace_bytes(B, L, T)
    if nbytes < 0:
        raise ValueError('log_probs of shape %s: at most %d answers a list, 2^24 - 1 answers and 2^28 tokens an answer'
                         % (tuple(log_probs.shape), MAX_ANSWERS))
    workspace = torch.empty((nbytes,), dtype=torch.uint8, device=log_probs.device) if nbytes else None
    rc = lib.tfr_preference_loss_f32(_ptr(log_probs), _ptr(reference), _ptr(mask), _ptr(labels), _ptr(list_weights), B, L, T, KINDS[kind],
                                     float(beta), float(label_smoothing), int(length_normalized), float(scale), _ptr(loss), _ptr(coef),
                                     _ptr(workspace), nbytes, _stream())
    _lib.check(rc, 'tfr_preference_loss_f32')
    return loss, coef


@_ops.device_guarded
def preference_grad(coef: torch.Tensor, mask: Optional[torch.Tensor], tokens: int, upstream: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``[B, L, tokens]``: the coefficients on the unmasked tokens, times ``upstream`` ``[B]``."""
    B, L = coef.shape
    out = torch.empty((B, L, tokens), dtype=torch.float32, device=coef.device)
    rc = _lib.load().tfr_preference_grad_f32(_ptr(coef), _ptr(upstream), _ptr(mask), B, L, tokens, _ptr(out), _stream())
    _lib.check(rc, 'tfr_preference_grad_f32')
    return out


class _PreferenceFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, log_probs, labels, reference, mask, list_weights, how):
        loss, coef = preference_loss(log_probs, labels, reference, mask, list_weights, **how)
        ctx.save_for_backward(coef, *([] if mask is None else [mask]))
        ctx.tokens = log_probs.shape[2]
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        coef, *mask = ctx.saved_tensors
        return preference_grad(coef, mask[0] if mask else None, ctx.tokens, g.contiguous()), None, None, None, None, None
