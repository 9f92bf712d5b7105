"""Embedding lookup with scaling and its gradient by sorted tokens (``csrc/embedding.hip``): what turns token or
category ids of a query or a document into dense features (``keras.layers.Embedding`` holds the table).

``embedding_lookup`` is differentiable with respect to the table.  ``embedding_grad`` is the same gradient as a plain
call, for loops that place gradients themselves (and for stream captures).
"""
from __future__ import annotations

import math
from typing import Optional

import torch
from torch.autograd import forward_ad

from . import _lib
from . import _ops
from ._ops import _raw_stream, require_device

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}          # TFR_DTYPE_*
_COMBINERS = {None: 0, 'sum': 1, 'mean': 2}                                # TFR_COMBINER_*
_MOST = 1 << 25                                                            # rows, bags and lookups of one call


def _dtype_code(t: torch.Tensor, name: str) -> int:
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise ValueError('%s must be float32, bfloat16 or float16, got %s' % (name, t.dtype))
    return code


def _device_of(name: str, t: torch.Tensor, **others) -> int:
    """Index of the HIP device that all these tensors are on."""
    if not torch.is_tensor(t) or not t.is_cuda:
        require_device(t, name)
    index = t.get_device()
    for other, u in others.items():
        if not torch.is_tensor(u) or not u.is_cuda:
            require_device(u, other)
        if u.get_device() != index:
            raise ValueError('%s is on %s, %s on %s' % (name, t.device, other, u.device))
    return index


def _ids(ids: torch.Tensor, combiner: Optional[str]):
    """(dense ids, id type, bags, tokens, combiner code, shape of the lookup without its last axis)."""
    if ids.dtype is torch.int64:
        id_type = 1
    elif ids.dtype is torch.int32:
        id_type = 0
    else:
        raise ValueError('ids must be int32 or int64, got %s' % ids.dtype)
    code = _COMBINERS.get(combiner)
    if code is None:
        raise ValueError("combiner must be None, 'sum' or 'mean', got %r" % (combiner,))
    shape = tuple(ids.shape)
    if code == 0:
        bags, tokens = ids.numel(), 1
    else:
        if not shape:
            raise ValueError('a combiner needs ids of [..., tokens]')
        tokens, shape = shape[-1], shape[:-1]
        bags = ids.numel() // tokens if tokens else math.prod(shape)
    if bags > _MOST or bags * tokens > _MOST:
        raise ValueError('at most %d lookups a call, got ids of shape %s' % (_MOST, tuple(ids.shape)))
    return ids.contiguous(), id_type, bags, tokens, code, shape


def _lookup(table, ids, scale, combiner):
    index = _device_of('table', table, ids=ids)
    code = _dtype_code(table, 'table')
    if table.dim() != 2 or table.shape[1] < 1:
        raise ValueError('table must be [rows, dim], got shape %s' % (tuple(table.shape),))
    rows, dim = table.shape
    if rows > _MOST:
        raise ValueError('a table of at most %d rows, got %d' % (_MOST, rows))
    ids, id_type, bags, tokens, how, shape = _ids(ids, combiner)
    pitch, step = table.stride()
    if step != 1 or pitch < dim:
        table = table.contiguous()
        pitch = dim
    with _ops.device_of(index):
        out = table.new_empty(shape + (dim,))
        rc = _lib.load().tfr_embedding_lookup(table.data_ptr(), pitch, rows, dim, code, ids.data_ptr(), id_type, bags, tokens, how,
                                              float(scale), out.data_ptr(), _raw_stream(index))
    if rc:
        _lib.check(rc, 'tfr_embedding_lookup')
    return out


def embedding_grad(grad: torch.Tensor, ids: torch.Tensor, num_embeddings: int, scale: float = 1.0,
                   combiner: Optional[str] = None) -> torch.Tensor:
    """Gradient of ``embedding_lookup(table, ids, scale, combiner)`` with respect to the table:
    ``[num_embeddings, dim]`` in ``grad``'s type, sums in fp32, every row written.  The order of the sums depends on
    the ids alone: equal calls give equal bits."""
    index = _device_of('grad', grad, ids=ids)
    code = _dtype_code(grad, 'grad')
    ids, id_type, bags, tokens, how, shape = _ids(ids, combiner)
    if grad.dim() < 1 or tuple(grad.shape[:-1]) != shape or grad.shape[-1] < 1:
        raise ValueError('grad of shape %s does not fit ids of shape %s' % (tuple(grad.shape), tuple(ids.shape)))
    rows, dim = int(num_embeddings), grad.shape[-1]
    if not 0 <= rows <= _MOST:
        raise ValueError('num_embeddings must be in [0, %d], got %d' % (_MOST, rows))
    grad = grad.contiguous()
    lib = _lib.load()
    with _ops.device_of(index):
        out = grad.new_empty((rows, dim))
        nbytes = lib.tfr_embedding_grad_workspace_bytes(rows, dim, bags, tokens, how)
        workspace = grad.new_empty((max(nbytes, 0),), dtype=torch.uint8)
        rc = lib.tfr_embedding_grad(grad.data_ptr(), code, ids.data_ptr(), id_type, bags, tokens, how, float(scale), rows, dim, out.data_ptr(),
                                    workspace.data_ptr(), nbytes, _raw_stream(index))
    if rc:
        _lib.check(rc, 'tfr_embedding_grad')
    return out


def _differentiated(t) -> bool:
    """Whether autograd has to see a call on ``t``: a gradient is wanted, or ``t`` carries a forward-mode tangent (which the autograd
    functions here refuse; the kernels, called on its address, would drop it)."""
    return torch.is_tensor(t) and ((t.requires_grad and torch.is_grad_enabled()) or forward_ad.unpack_dual(t).tangent is not None)


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
    if _differentiated(table):
        return _EmbeddingFn.apply(table, ids, scale, combiner)
    return _lookup(table, ids, scale, combiner)
