"""Scaled token embedding with its gradient on B200 (tb_embedding_fwd / tb_embedding_grad), for
steps that train the table or scale the embedding; model.embed_rows is the frozen, unscaled form
the fused QLoRA forward uses (reference: solution/model.py:220-225).

    y[t] = scale * W[id_t]        dW[v] = scale * sum over t with id_t = v of dy[t]

The gradient sorts the tokens by id and adds each id's rows in fp32 in that order: the same inputs
give the same bits. Ids outside the table give zero rows and no gradient, and are counted
(tb_embed_invalid_ids), as in model.embed_rows.
"""

import torch
from torch.autograd.function import once_differentiable

from . import _lib


def _check_ids(ids, what):
    if ids.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"{what}: ids must be int64 or int32, got {ids.dtype}")
    return ids if ids.is_contiguous() else ids.contiguous()


def _grad(ids, dy, dw, scale, padding_idx, accumulate):
    n, (vocab, hidden) = ids.numel(), dw.shape
    nbytes = _lib.workspace_bytes(dw, "tb_embedding_grad_workspace", n, hidden)
    ws = dw.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    _lib.call_on(dw, "tb_embedding_grad", ids.data_ptr(), int(ids.dtype == torch.int64),
                 dy.data_ptr(), _lib.TYPE_CODES[dy.dtype], dw.data_ptr(),
                 _lib.TYPE_CODES[dw.dtype], scale, padding_idx, int(accumulate), n, hidden, vocab,
                 _lib.addr(ws), nbytes)
    return dw


def _forward(ids, weight, scale, out_dtype):
    vocab, hidden = weight.shape
    out = weight.new_empty((*ids.shape, hidden), dtype=out_dtype)
    if ids.numel():
        _lib.call_on(weight, "tb_embedding_fwd", ids.data_ptr(), int(ids.dtype == torch.int64),
                     weight.data_ptr(), _lib.TYPE_CODES[weight.dtype],
                     weight.stride(0) if vocab > 1 else hidden, out.data_ptr(),
                     _lib.TYPE_CODES[out_dtype], scale, ids.numel(), hidden, vocab)
    return out


class ScaledEmbedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, weight, scale, padding_idx, out_dtype):
        ctx.save_for_backward(ids)
        ctx.rest = (weight.shape, weight.dtype, scale, padding_idx)
        return _forward(ids, weight, scale, out_dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        (ids,) = ctx.saved_tensors
        shape, dtype, scale, padding_idx = ctx.rest
        dw = dy.new_empty(shape, dtype=dtype)
        return None, _grad(ids, dy.contiguous(), dw, scale, padding_idx, False), None, None, None


def embedding(ids, weight, scale=1.0, padding_idx=None, out_dtype=None):
    """scale * weight[ids] in `out_dtype` (weight's dtype, the default, or fp32), rounded once, for
    int64 or int32 ids of any shape and a [vocab, hidden] fp16, bf16 or fp32 table; differentiable
    in weight (a dense gradient). `padding_idx`: an id whose row gets no gradient."""
    _lib.require_cuda(ids, weight, what="embedding")
    ids = _check_ids(ids, "embedding")
    if weight.dtype not in _lib.TYPE_CODES or weight.dim() != 2 or 0 in weight.shape:
        raise ValueError(f"embedding: weight must be fp16, bf16 or fp32 [vocab, hidden], got "
                         f"{tuple(weight.shape)} {weight.dtype}")
    if ids.get_device() != weight.get_device():
        raise ValueError(f"embedding: ids on {ids.device}, weight on {weight.device}")
    out_dtype = weight.dtype if out_dtype is None else out_dtype
    if out_dtype not in (weight.dtype, torch.float32):
        raise TypeError(f"embedding: out_dtype {out_dtype} for a {weight.dtype} table")
    if padding_idx is not None and not 0 <= padding_idx < weight.shape[0]:
        raise ValueError(f"embedding: padding_idx {padding_idx} outside [0, {weight.shape[0]})")
    if weight.stride(1) != 1 or (weight.shape[0] > 1 and weight.stride(0) < weight.shape[1]):
        weight = weight.contiguous()
    if _lib.needs_grad(weight):
        return ScaledEmbedding.apply(ids, weight, float(scale),
                                     -1 if padding_idx is None else int(padding_idx), out_dtype)
    return _forward(ids, weight, float(scale), out_dtype)


def embedding_grad(ids, dy, vocab, scale=1.0, padding_idx=None, out=None, dtype=None):
    """embedding's weight gradient [vocab, hidden] for dy [*ids.shape, hidden], in `dtype` (dy's by
    default; dy's, or either of the two fp32). With `out` (contiguous, its dtype such a one) the
    sums are added to it in place, each touched row rounded once more, and it is returned: the
    form for a table tied to the head, whose gradient holds the head's share already. Not
    differentiable itself: dy and out are taken as values."""
    _lib.require_cuda(ids, dy, out, what="embedding_grad")
    ids = _check_ids(ids, "embedding_grad")
    if dy.dtype not in _lib.TYPE_CODES or dy.dim() != ids.dim() + 1 or \
            dy.shape[:-1] != ids.shape or dy.shape[-1] == 0:
        raise ValueError(f"embedding_grad: dy {tuple(dy.shape)} {dy.dtype} for ids "
                         f"{tuple(ids.shape)}")
    hidden, vocab = dy.shape[-1], int(vocab)
    if vocab <= 0:
        raise ValueError(f"embedding_grad: vocab {vocab}")
    if padding_idx is not None and not 0 <= padding_idx < vocab:
        raise ValueError(f"embedding_grad: padding_idx {padding_idx} outside [0, {vocab})")
    if out is not None:
        if tuple(out.shape) != (vocab, hidden) or not out.is_contiguous() or \
                (dtype is not None and out.dtype != dtype):
            raise ValueError(f"embedding_grad: out {tuple(out.shape)} {out.dtype}, expected "
                             f"contiguous {(vocab, hidden)}")
    dtype = out.dtype if out is not None else dy.dtype if dtype is None else dtype
    if dtype not in _lib.TYPE_CODES or (dtype != dy.dtype and
                                        torch.float32 not in (dtype, dy.dtype)):
        raise TypeError(f"embedding_grad: {dy.dtype} -> {dtype}")
    for t in (ids, out):
        if t is not None and t.device != dy.device:
            raise ValueError(f"embedding_grad: operands on {t.device} and {dy.device}")
    _lib.refuse_tangents("embedding_grad", dy, out)
    accumulate = out is not None
    dw = out if accumulate else torch.empty((vocab, hidden), dtype=dtype, device=dy.device)
    _grad(ids, dy.contiguous(), dw, float(scale), -1 if padding_idx is None else int(padding_idx),
          accumulate)
    if accumulate:
        torch.autograd.graph.increment_version(out)  # autograd sees the write
    return dw
