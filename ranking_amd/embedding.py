"""Embedding lookup with scaling and its gradient by sorted tokens (``csrc/embedding.hip``): what turns token or
category ids of a query or a document into dense features (``keras.layers.Embedding`` holds the table).

``embedding_lookup`` is differentiable with respect to the table.  ``embedding_grad`` is the same gradient as a plain
call, for loops that place gradients themselves (and for stream captures).
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib
from . import _ops
from ._ops import _ptr, _stream, require_device

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}          # TFR_DTYPE_*
_COMBINERS = {None: 0, 'sum': 1, 'mean': 2}                                # TFR_COMBINER_*
_MOST = 1 << 25                                                            # rows, bags and lookups of one call


def _dtype_code(t: torch.Tensor, name: str) -> int:
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise ValueError('%s must be float32, bfloat16 or float16, got %s' % (name, t.dtype))
    return code


def _same_device(a: torch.Tensor, b: torch.Tensor, na: str, nb: str) -> None:
    if a.device != b.device:
        raise ValueError('%s is on %s, %s on %s' % (na, a.device, nb, b.device))


def _ids(ids: torch.Tensor, combiner: Optional[str]):
    """(dense ids, id type, bags, tokens, shape of the lookup without its last axis)."""
    require_device(ids, 'ids')
    if ids.dtype not in (torch.int32, torch.int64):
        raise ValueError('ids must be int32 or int64, got %s' % ids.dtype)
    if combiner not in _COMBINERS:
        raise ValueError("combiner must be None, 'sum' or 'mean', got %r" % (combiner,))
    if combiner is None:
        bags, tokens, shape = ids.numel(), 1, tuple(ids.shape)
    else:
        if ids.dim() < 1:
            raise ValueError('a combiner needs ids of [..., tokens]')
        tokens, shape = ids.shape[-1], tuple(ids.shape[:-1])
        bags = 1
        for n in shape:
            bags *= n
    if max(bags, bags * tokens) > _MOST:
        raise ValueError('at most %d lookups a call, got ids of shape %s' % (_MOST, tuple(ids.shape)))
    return ids.contiguous(), (0 if ids.dtype == torch.int32 else 1), bags, tokens, shape


@_ops.device_guarded
def _lookup(table, ids, scale, combiner):
    code = _dtype_code(table, 'table')
    ids, id_type, bags, tokens, shape = _ids(ids, combiner)
    rows, dim = table.shape
    if table.stride(1) != 1 or table.stride(0) < dim:
        table = table.contiguous()
    out = torch.empty(shape + (dim,), dtype=table.dtype, device=table.device)
    rc = _lib.load().tfr_embedding_lookup(_ptr(table), max(table.stride(0), dim), rows, dim, code, _ptr(ids), id_type, bags, tokens,
                                          _COMBINERS[combiner], float(scale), _ptr(out), _stream())
    _lib.check(rc, 'tfr_embedding_lookup')
    return out


@_ops.device_guarded
def embedding_grad(grad: torch.Tensor, ids: torch.Tensor, num_embeddings: int, scale: float = 1.0,
                   combiner: Optional[str] = None) -> torch.Tensor:
    """Gradient of ``embedding_lookup(table, ids, scale, combiner)`` with respect to the table:
    ``[num_embeddings, dim]`` in ``grad``'s type, sums in fp32, every row written.  The order of the sums depends on
    the ids alone: equal calls give equal bits."""
    require_device(grad, 'grad')
    code = _dtype_code(grad, 'grad')
    ids, id_type, bags, tokens, shape = _ids(ids, combiner)
    _same_device(grad, ids, 'grad', 'ids')
    if tuple(grad.shape[:-1]) != shape or grad.dim() < 1 or grad.shape[-1] < 1:
        raise ValueError('grad of shape %s does not fit ids of shape %s' % (tuple(grad.shape), tuple(ids.shape)))
    rows, dim = int(num_embeddings), grad.shape[-1]
    if not 0 <= rows <= _MOST:
        raise ValueError('num_embeddings must be in [0, %d], got %d' % (_MOST, rows))
    grad = grad.contiguous()
    lib = _lib.load()
    out = torch.empty((rows, dim), dtype=grad.dtype, device=grad.device)
    nbytes = lib.tfr_embedding_grad_workspace_bytes(rows, dim, bags, tokens, _COMBINERS[combiner])
    workspace = torch.empty((nbytes,), dtype=torch.uint8, device=grad.device) if nbytes > 0 else None
    rc = lib.tfr_embedding_grad(_ptr(grad), code, _ptr(ids), id_type, bags, tokens, _COMBINERS[combiner], float(scale), rows, dim, _ptr(out),
                                _ptr(workspace), nbytes, _stream())
    _lib.check(rc, 'tfr_embedding_grad')
    return out


class _EmbeddingFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, ids, scale, combiner):
        ctx.save_for_backward(ids)
        ctx.rows, ctx.scale, ctx.combiner = table.shape[0], scale, combiner
        return _lookup(table, ids, scale, combiner)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        (ids,) = ctx.saved_tensors
        return embedding_grad(g, ids, ctx.rows, ctx.scale, ctx.combiner), None, None, None


def embedding_lookup(table: torch.Tensor, ids: torch.Tensor, scale: float = 1.0, combiner: Optional[str] = None) -> torch.Tensor:
    """Rows of ``table`` ``[rows, dim]`` (float32, bfloat16 or float16) times ``scale``.

    ``combiner=None``: ``ids`` of any shape -> ``ids.shape + (dim,)``.  ``'sum'`` / ``'mean'``: the rows of the last axis
    are added (averaged over the ids that are not padding), in fp32, and rounded once: ``ids.shape[:-1] + (dim,)``.
    Ids below 0 are padding: zeros, no gradient.  An id beyond the table gives NaN and no gradient.  Differentiable with
    respect to ``table``; the gradient is a dense tensor of the table's type."""
    require_device(table, 'table')
    if table.dim() != 2 or table.shape[1] < 1:
        raise ValueError('table must be [rows, dim], got shape %s' % (tuple(table.shape),))
    if table.shape[0] > _MOST:
        raise ValueError('a table of at most %d rows, got %d' % (_MOST, table.shape[0]))
    require_device(ids, 'ids')
    _same_device(table, ids, 'table', 'ids')
    if torch.is_grad_enabled() and table.requires_grad:
        return _EmbeddingFn.apply(table, ids, scale, combiner)
    return _lookup(table, ids, scale, combiner)
