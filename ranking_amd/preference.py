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
from ._ops import _raw_stream, require_device
from .embedding import _device_of, _differentiated, _dtype_code

KINDS = {'logistic': 0, 'hinge': 1, 'squared': 2}                          # TFR_PREFERENCE_*
MAX_ANSWERS = 64


def _rows(logits: torch.Tensor, targets: torch.Tensor):
    """(logits, rows, vocab, per, stride_b, stride_t, dense int64 targets): the rows of [..., vocab] as two strided axes."""
    shape = tuple(logits.shape)
    if not shape or shape[-1] < 1:
        raise ValueError('logits must be [..., vocab], got shape %s' % (shape,))
    if targets.dtype is not torch.int64 and targets.dtype is not torch.int32:
        raise ValueError('targets must be int32 or int64, got %s' % targets.dtype)
    if tuple(targets.shape) != shape[:-1]:
        raise ValueError('targets of shape %s do not fit logits of shape %s' % (tuple(targets.shape), shape))
    n, vocab = targets.numel(), shape[-1]
    if n >= 1 << 24 or vocab > 1 << 28:
        raise ValueError('at most 2^24 - 1 rows of 2^28 logits, got %d of %d' % (n, vocab))
    if len(shape) > 3 or (logits.stride(-1) != 1 and vocab > 1):
        logits = logits.contiguous()
        per, stride_b, stride_t = 1, vocab, 0
    elif len(shape) == 2:
        per, stride_b, stride_t = 1, logits.stride(0), 0
    elif len(shape) == 1:
        per, stride_b, stride_t = 1, 0, 0
    else:
        per, stride_b, stride_t = max(1, shape[1]), logits.stride(0), logits.stride(1)
    if targets.dtype is not torch.int64:
        targets = targets.to(torch.int64)
    return logits, n, vocab, per, stride_b, stride_t, targets.contiguous()


def _temperature(t) -> float:
    if not 1e-30 <= t <= 1e30:
        raise ValueError('temperature must be positive, got %r' % t)
    return t


def _log_probs(logits, targets, temperature, want_stats):
    index = _device_of('logits', logits, targets=targets)
    code = _dtype_code(logits, 'logits')
    logits, n, vocab, per, stride_b, stride_t, targets = _rows(logits, targets)
    lib = _lib.load()
    with _ops.device_of(index):
        logp = torch.empty_like(targets, dtype=torch.float32)
        stats = targets.new_empty(targets.shape + (2,), dtype=torch.float32) if want_stats else None
        nbytes = lib.tfr_token_logprob_workspace_bytes(n, vocab)
        workspace = targets.new_empty((nbytes,), dtype=torch.uint8) if nbytes > 0 else None
        rc = lib.tfr_token_logprob(logits.data_ptr(), code, per, stride_b, stride_t, targets.data_ptr(), n, vocab, _temperature(temperature),
                                   logp.data_ptr(), stats.data_ptr() if want_stats else None, workspace.data_ptr() if nbytes > 0 else None, nbytes,
                                   _raw_stream(index))
    if rc:
        _lib.check(rc, 'tfr_token_logprob')
    return logp, stats


def token_log_probs_with_stats(logits: torch.Tensor, targets: torch.Tensor, temperature: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """``token_log_probs`` without autograd, and the row statistics ``[..., 2]`` that ``token_log_probs_grad`` takes."""
    return _log_probs(logits.detach() if torch.is_tensor(logits) else logits, targets, temperature, True)


def token_log_probs_grad(grad: torch.Tensor, logits: torch.Tensor, targets: torch.Tensor, stats: torch.Tensor,
                         temperature: float = 1.0) -> torch.Tensor:
    """``d sum(grad * token_log_probs) / d logits`` as a dense tensor of ``logits``' shape and type."""
    index = _device_of('logits', logits, targets=targets, grad=grad, stats=stats)
    code = _dtype_code(logits, 'logits')
    shape = logits.shape
    logits, n, vocab, per, stride_b, stride_t, targets = _rows(logits, targets)
    if grad.shape != shape[:-1] or stats.shape != shape[:-1] + (2,) or stats.dtype is not torch.float32:
        raise ValueError('grad of shape %s and stats of shape %s do not fit logits of shape %s'
                         % (tuple(grad.shape), tuple(stats.shape), tuple(shape)))
    if grad.dtype is not torch.float32:
        grad = grad.to(torch.float32)
    grad, stats = grad.contiguous(), stats.contiguous()
    with _ops.device_of(index):
        out = torch.empty_like(logits) if logits.is_contiguous() else logits.new_empty(shape)
        rc = _lib.load().tfr_token_logprob_grad(logits.data_ptr(), code, per, stride_b, stride_t, targets.data_ptr(), stats.data_ptr(),
                                                grad.data_ptr(), n, vocab, _temperature(temperature), out.data_ptr(), _raw_stream(index))
    if rc:
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
    if _differentiated(logits):
        return _TokenLogProbsFn.apply(logits, targets, temperature)
    return _log_probs(logits, targets, temperature, False)[0]


def _address(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _check_dense(index, t, name, shape, dtypes=(torch.float32,)):
    require_device(t, name)
    if tuple(t.shape) != tuple(shape) or t.dtype not in dtypes or t.get_device() != index or not t.is_contiguous():
        raise ValueError('%s must be a dense %s tensor of shape %s on device %d, got %s of shape %s on %s'
                         % (name, ' or '.join(map(str, dtypes)), tuple(shape), index, t.dtype, tuple(t.shape), t.device))


def _check_loss(log_probs, labels, reference, mask, list_weights, kind):
    """Refuses what the loss kernels would not read as it is meant (``keras.losses.PreferenceLoss`` makes its tensors fit)."""
    if kind not in KINDS:
        raise ValueError('Invalid kind: {}. Expected "{}"'.format(kind, tuple(KINDS)))
    require_device(log_probs, 'log_probs')
    if log_probs.dim() != 3:
        raise ValueError('log_probs must be [batch, answers, tokens], got shape %s' % (tuple(log_probs.shape),))
    index, shape = log_probs.get_device(), log_probs.shape
    _check_dense(index, log_probs, 'log_probs', shape)
    _check_dense(index, labels, 'labels', shape[:2])
    if reference is not None:
        _check_dense(index, reference, 'reference', shape)
    if mask is not None:
        _check_dense(index, mask, 'mask', shape, (torch.uint8, torch.bool))
    if list_weights is not None:
        _check_dense(index, list_weights, 'list_weights', shape[:1])


def _loss_args(log_probs, labels, reference, mask, list_weights, kind, beta, label_smoothing, length_normalized, scale):
    """(B, L, T, workspace, its bytes, the arguments that both forms of the loss share)."""
    B, L, T = log_probs.shape
    nbytes = _lib.load().tfr_preference_workspace_bytes(B, L, T)
    if nbytes < 0:
        raise ValueError('log_probs of shape %s: at most %d answers a list, 2^24 - 2 answers and 2^28 tokens an answer'
                         % (tuple(log_probs.shape), MAX_ANSWERS))
    workspace = log_probs.new_empty((nbytes,), dtype=torch.uint8)
    return B, L, T, workspace, nbytes, (log_probs.data_ptr(), _address(reference), _address(mask), labels.data_ptr(), _address(list_weights),
                                        B, L, T, KINDS[kind], beta, label_smoothing, int(length_normalized), scale)


def preference_loss(log_probs: torch.Tensor, labels: torch.Tensor, reference: Optional[torch.Tensor] = None,
                    mask: Optional[torch.Tensor] = None, list_weights: Optional[torch.Tensor] = None, kind: str = 'logistic',
                    beta: float = 0.1, label_smoothing: float = 0.0, length_normalized: bool = False,
                    scale: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """(loss ``[B]``, coefficients ``[B, L]`` of ``preference_grad``).  Dense device tensors: ``log_probs`` and ``reference``
    ``[B, L, T]``, ``labels`` ``[B, L]``, ``list_weights`` ``[B]`` in float32, ``mask`` ``[B, L, T]`` uint8 or bool (what
    ``keras.losses.PreferenceLoss`` makes of its arguments)."""
    _check_loss(log_probs, labels, reference, mask, list_weights, kind)
    return _loss(log_probs, labels, reference, mask, list_weights, kind, beta, label_smoothing, length_normalized, scale)


def _loss(log_probs, labels, reference, mask, list_weights, kind, beta, label_smoothing, length_normalized, scale):
    index = log_probs.get_device()
    with _ops.device_of(index):
        B, L, T, workspace, nbytes, args = _loss_args(log_probs, labels, reference, mask, list_weights, kind, beta, label_smoothing,
                                                      length_normalized, scale)
        loss = torch.empty((B,), dtype=torch.float32, device=log_probs.device)
        coef = torch.empty((B, L), dtype=torch.float32, device=log_probs.device)
        rc = _lib.load().tfr_preference_loss_f32(*args, loss.data_ptr(), coef.data_ptr(), workspace.data_ptr(), nbytes, _raw_stream(index))
    if rc:
        _lib.check(rc, 'tfr_preference_loss_f32')
    return loss, coef


def preference_loss_and_grad(log_probs: torch.Tensor, labels: torch.Tensor, reference: Optional[torch.Tensor] = None,
                             mask: Optional[torch.Tensor] = None, list_weights: Optional[torch.Tensor] = None, kind: str = 'logistic',
                             beta: float = 0.1, label_smoothing: float = 0.0, length_normalized: bool = False,
                             scale: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """(sum of the lists' losses, its gradient ``[B, L, T]``) of the same arguments as ``preference_loss``."""
    _check_loss(log_probs, labels, reference, mask, list_weights, kind)
    return _loss_and_grad(log_probs, labels, reference, mask, list_weights, kind, beta, label_smoothing, length_normalized, scale)


def _loss_and_grad(log_probs, labels, reference, mask, list_weights, kind, beta, label_smoothing, length_normalized, scale):
    index = log_probs.get_device()
    with _ops.device_of(index):
        B, L, T, workspace, nbytes, args = _loss_args(log_probs, labels, reference, mask, list_weights, kind, beta, label_smoothing,
                                                      length_normalized, scale)
        total = log_probs.new_empty(())
        grad = torch.empty_like(log_probs)
        rc = _lib.load().tfr_preference_loss_and_grad_f32(*args, total.data_ptr(), grad.data_ptr(), workspace.data_ptr(), nbytes,
                                                          _raw_stream(index))
    if rc:
        _lib.check(rc, 'tfr_preference_loss_and_grad_f32')
    return total, grad


def preference_grad(coef: torch.Tensor, mask: Optional[torch.Tensor], tokens: int, upstream: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``[B, L, tokens]``: the coefficients ``[B, L]`` on the unmasked tokens, times ``upstream`` ``[B]`` (dense float32)."""
    require_device(coef, 'coef')
    if coef.dim() != 2 or not 1 <= coef.shape[1] <= MAX_ANSWERS or tokens < 0:
        raise ValueError('coef must be [batch, answers] with at most %d answers and tokens a length, got shape %s and %r'
                         % (MAX_ANSWERS, tuple(coef.shape), tokens))
    index = coef.get_device()
    _check_dense(index, coef, 'coef', coef.shape)
    if mask is not None:
        _check_dense(index, mask, 'mask', tuple(coef.shape) + (tokens,), (torch.uint8, torch.bool))
    if upstream is not None:
        _check_dense(index, upstream, 'upstream', coef.shape[:1])
    return _grad(coef, mask, tokens, upstream)


def _grad(coef, mask, tokens, upstream):
    B, L = coef.shape
    index = coef.get_device()
    with _ops.device_of(index):
        out = torch.empty((B, L, tokens), dtype=torch.float32, device=coef.device)
        rc = _lib.load().tfr_preference_grad_f32(coef.data_ptr(), _address(upstream), _address(mask), B, L, tokens, out.data_ptr(),
                                                 _raw_stream(index))
    if rc:
        _lib.check(rc, 'tfr_preference_grad_f32')
    return out


def _total(loss):
    index = loss.get_device()
    with _ops.device_of(index):
        total = loss.new_empty(())
        rc = _lib.load().tfr_preference_total_f32(loss.data_ptr(), loss.shape[0], total.data_ptr(), _raw_stream(index))
    if rc:
        _lib.check(rc, 'tfr_preference_total_f32')
    return total


class _PreferenceFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, log_probs, labels, reference, mask, list_weights, how, total):
        loss, coef = _loss(log_probs, labels, reference, mask, list_weights, **how)
        ctx.save_for_backward(coef, *([] if mask is None else [mask]))
        ctx.tokens, ctx.total = log_probs.shape[2], total
        return _total(loss) if total else loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        coef, *mask = ctx.saved_tensors
        if ctx.total:
            g = g.expand(coef.shape[0])
        return (_grad(coef, mask[0] if mask else None, ctx.tokens, g.contiguous()),) + (None,) * 6
