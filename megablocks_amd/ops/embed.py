"""Rows of a table by token, and the table's gradient by sorted tokens.  The reference has neither: its models' embedding is the trainer's."""
from typing import Any, Optional

import torch

from megablocks_amd import _lib
from megablocks_amd._lib import lib
from megablocks_amd.ops.choose import _has_memory


def _rows(ids, table, scale):
    out = torch.empty((*ids.shape, table.shape[1]), dtype=table.dtype, device=table.device)
    with _lib.device_of(table):
        _lib.check(lib.mbx_embedding(ids.data_ptr(), _lib.ITYPE[ids.dtype], ids.numel(), table.data_ptr(), _lib.DTYPE[table.dtype], table.shape[0], table.shape[1],
                                     scale, out.data_ptr(), _lib.stream()), 'embedding')
    return out


def _table_gradient(grad, ids, words, scale, padding):
    hidden = grad.shape[-1]
    grad = grad.contiguous()
    out = grad.new_empty((words, hidden))
    with _lib.device_of(grad):
        nbytes = lib.mbx_embedding_gradient_scratch_bytes(ids.numel(), words, hidden)
        scratch = torch.empty(nbytes, dtype=torch.uint8, device=grad.device) if nbytes else None      # none for a few tokens
        _lib.check(lib.mbx_embedding_gradient(grad.data_ptr(), ids.data_ptr(), _lib.ITYPE[ids.dtype], ids.numel(), _lib.DTYPE[grad.dtype], words, hidden, padding, scale,
                                              out.data_ptr(), _lib.ptr(scratch), nbytes, _lib.stream()), 'embedding_gradient')
    return out


def _plain_rows(ids, table, scale):
    """_rows in torch's operations, of a batch of tables (is_grads_batched), which has no memory of its own."""
    words = table.shape[0]
    if words == 0:
        return table.new_zeros((*ids.shape, table.shape[1]))
    inside = (ids >= 0) & (ids < words)
    rows = table.index_select(0, torch.where(inside, ids, 0).long().flatten()).double() * scale
    return rows.masked_fill(~inside.flatten().unsqueeze(1), 0.).to(table.dtype).reshape(*ids.shape, table.shape[1])


def _plain_table_gradient(grad, ids, words, scale, padding):
    """_table_gradient in torch's operations, of a batch of gradients: sums in 64 bits, the same from run to run."""
    ids, hidden = ids.flatten().long(), grad.shape[-1]
    counts = (ids >= 0) & (ids < words) & (ids != padding)
    zeros = torch.zeros((words + 1, hidden), dtype=torch.float64, device=ids.device)       # the last row: tokens that do not count
    sums = zeros.index_put((torch.where(counts, ids, words),), grad.reshape(len(ids), hidden).double(), accumulate=True)
    return (sums.narrow(0, 0, words) * scale).to(grad.dtype)


class EmbeddingOp(torch.autograd.Function):

    @staticmethod
    def forward(ctx: Any, ids, table, scale, padding):
        ctx.save_for_backward(ids)
        ctx.sizes = table.shape[0], scale, padding
        return _rows(ids, table, scale)

    @staticmethod
    def backward(ctx: Any, grad):
        ids, = ctx.saved_tensors
        # a node of its own only where the backward is differentiated itself; a batch of gradients at once (is_grads_batched) by torch
        gradient = _plain_table_gradient if not _has_memory(grad) else EmbeddingGradientOp.apply if torch.is_grad_enabled() else _table_gradient
        return None, gradient(grad, ids, *ctx.sizes), None, None


class EmbeddingGradientOp(torch.autograd.Function):
    """The table's gradient, which is linear in the rows': its own gradient is rows of a table again."""

    @staticmethod
    def forward(ctx: Any, grad, ids, words, scale, padding):
        ctx.save_for_backward(ids)
        ctx.choice = scale, padding
        return _table_gradient(grad, ids, words, scale, padding)

    @staticmethod
    def backward(ctx: Any, grad):
        ids, = ctx.saved_tensors
        scale, padding = ctx.choice
        if padding >= 0:
            ids = ids.masked_fill(ids == padding, -1)      # rows of zeros
        rows = EmbeddingOp.apply(ids, grad.contiguous(), scale, -1) if _has_memory(grad) else _plain_rows(ids, grad, scale)
        return rows, None, None, None, None


def embedding(ids: torch.Tensor, table: torch.Tensor, scale: float = 1.0, padding_idx: Optional[int] = None) -> torch.Tensor:
    """scale * table[ids], [*ids.shape, hidden], for int32 or int64 ids of any shape and a table [words, hidden] in bf16, fp16 or fp32, rounded once.  An id outside
    [0, words) gives a row of zeros.

    The table's gradient is dense, its sums in fp32 (of an fp32 table in 64 bits) in the order of the tokens, rounded once, the same from run to run; a row that no id names gets zeros, and so does
    that of padding_idx (from the end if negative), whose values are given out like any other's.  It is differentiable itself;
    several gradients at once (is_grads_batched) are computed by torch's operations.  Forward and backward can be captured into a
    graph; as with all of torch's operations no eager graph of the same table may be alive then."""
    scale = float(scale)
    if table.ndim != 2:
        raise ValueError('embedding: the table must be [words, hidden]')
    if not abs(scale) <= torch.finfo(torch.float32).max:
        raise ValueError('embedding: the scale must be finite, in fp32')
    words = table.shape[0]
    padding = -1
    if padding_idx is not None:
        padding = int(padding_idx)
        if not -words <= padding < words:
            raise ValueError(f'embedding: a table of {words} words has no padding_idx {padding}')
        padding %= words
    if not ids.is_cuda or table.device != ids.device:
        raise RuntimeError(f'embedding: expected ids and table on one GPU but got them on {ids.device} and {table.device}')
    if ids.dtype not in (torch.int32, torch.int64):
        raise RuntimeError(f'embedding: expected int32 or int64 ids but got {ids.dtype}')
    if table.dtype not in _lib.DTYPE:
        raise RuntimeError(f'embedding: expected a bfloat16, float16 or float32 table but got {table.dtype}')
    ids, table = ids.contiguous(), table.contiguous()
    # a node is some us of the host's time; one in forward differentiation says that it has none
    if (table.requires_grad and torch.is_grad_enabled()) or getattr(torch.autograd.forward_ad, '_current_level', 0) >= 0:
        return EmbeddingOp.apply(ids, table, scale, padding)
    return _rows(ids, table, scale)
