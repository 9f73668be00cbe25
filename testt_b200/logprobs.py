"""Log-probabilities of given tokens, with entropy and the top alternatives, from given logits on
B200 (tb_token_logprobs_fwd / tb_token_logprobs_bwd): what a policy-gradient, preference or
distillation loss and a scoring pass read from the head. head.fused_head_loss is the
cross-entropy form that never holds the logits (reference: solution/head.py).

    z = logits / temperature     logprob = z[id] - logsumexp z     entropy = logsumexp z - sum p z
One read of the logits forward; the gradient is one read and one write.
"""

from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib

MAX_TOP = 32


class TokenLogprobs(NamedTuple):
    logprob: torch.Tensor       # fp32 [...]: 0 where the id is outside the vocabulary
    entropy: torch.Tensor       # fp32 [...]
    top_logprobs: torch.Tensor  # fp32 [..., top_k], descending
    top_ids: torch.Tensor       # int64 [..., top_k]; equal logits by the lowest id


def _ld(logits):
    """Elements between rows (a single row's stride may be anything)."""
    return logits.stride(0) if logits.shape[0] > 1 else logits.shape[1]


def _grad_like(logits):
    """An empty gradient whose rows lie modulo 16 bytes as the logits' rows do, so that both are
    read and written in whole 16-byte words (at most 7 spare columns a row)."""
    rows, vocab = logits.shape
    if logits.is_contiguous() and logits.data_ptr() % 16 == 0:
        return torch.empty_like(logits)
    per = 16 // logits.element_size()
    ld = vocab + (_ld(logits) - vocab) % per
    lead = logits.data_ptr() % 16 // logits.element_size()
    flat = torch.empty(lead + rows * ld, dtype=logits.dtype, device=logits.device)
    return flat.as_strided((rows, vocab), (ld, 1), lead)


def _forward(logits, ids, top_k, temperature):
    """(logprob, entropy, top_lp, top_ids) and the buffer that ends with the backward's
    statistics."""
    rows, vocab = logits.shape
    code = _lib.TYPE_CODES[logits.dtype]
    logprob = logits.new_empty(rows, dtype=torch.float32)
    entropy = torch.empty_like(logprob)
    top_lp = logprob.new_empty((rows, top_k))
    top_ids = logprob.new_empty((rows, top_k), dtype=torch.int64)
    if not rows:
        return logprob, entropy, top_lp, top_ids, logprob.new_empty(0)
    # the workspace with the backward's statistics [rows, 3] behind it, as one allocation
    nbytes = _lib.workspace_bytes(logits, "tb_token_logprobs_workspace", rows, vocab, code, top_k)
    stats = logprob.new_empty(nbytes // 4 + 3 * rows)
    at = stats.data_ptr()
    _lib.call_on(logits, "tb_token_logprobs_fwd", logits.data_ptr(), code, _ld(logits),
                 ids.data_ptr(), int(ids.dtype == torch.int64), temperature, top_k,
                 logprob.data_ptr(), entropy.data_ptr(), top_lp.data_ptr(), top_ids.data_ptr(),
                 at + nbytes, rows, vocab, at if nbytes else None, nbytes)
    return logprob, entropy, top_lp, top_ids, stats


class TokenLogprobsFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, ids, top_k, temperature):
        logprob, entropy, top_lp, top_ids, stats = _forward(logits, ids, top_k, temperature)
        ctx.save_for_backward(logits, ids, top_ids, stats)
        ctx.rest = (top_k, temperature)
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(top_ids)
        return logprob, entropy, top_lp, top_ids

    @staticmethod
    @once_differentiable
    def backward(ctx, g_lp, g_ent, g_top, _g_ids):
        logits, ids, top_ids, stats = ctx.saved_tensors
        top_k, temperature = ctx.rest
        if g_lp is None and g_ent is None and g_top is None:
            return None, None, None, None
        rows, vocab = logits.shape
        g_lp, g_ent, g_top = (None if g is None else g.contiguous() for g in (g_lp, g_ent, g_top))
        grad = _grad_like(logits)
        if rows:
            _lib.call_on(logits, "tb_token_logprobs_bwd", logits.data_ptr(),
                         _lib.TYPE_CODES[logits.dtype], _ld(logits), ids.data_ptr(),
                         int(ids.dtype == torch.int64), temperature, top_k, top_ids.data_ptr(),
                         stats.data_ptr() + 4 * (stats.numel() - 3 * rows), _lib.addr(g_lp),
                         _lib.addr(g_ent), _lib.addr(g_top), grad.data_ptr(),
                         grad.stride(0) if rows > 1 else vocab, rows, vocab)
        return grad, None, None, None


def token_logprobs(logits, ids, top_k=0, temperature=1.0):
    """TokenLogprobs of fp16, bf16 or fp32 `logits` [..., vocab] (unit column stride is taken as it
    is, rows may be views) at int64 or int32 `ids` [...]; `top_k` 0 to 32. Differentiable in the
    logits through logprob, entropy and top_logprobs. An id outside [0, vocab) (IGNORE_INDEX) has
    logprob 0 and no gradient; -inf logits have probability 0, beside the type's lowest value too (a
    row of that value is one of equal logits); a row of -inf only has logprob -inf, entropy 0 and no
    gradient; a NaN or +inf makes its row NaN. Fewer than 2^21 rows."""
    _lib.require_cuda(logits, ids, what="token_logprobs")
    if logits.dtype not in _lib.TYPE_CODES or logits.dim() < 1 or logits.shape[-1] == 0:
        raise ValueError(f"token_logprobs: logits must be fp16, bf16 or fp32 [..., vocab], got "
                         f"{tuple(logits.shape)} {logits.dtype}")
    if ids.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"token_logprobs: ids must be int64 or int32, got {ids.dtype}")
    lead, vocab = logits.shape[:-1], logits.shape[-1]
    if ids.shape != lead or ids.get_device() != logits.get_device():
        raise ValueError(f"token_logprobs: ids {tuple(ids.shape)} on {ids.device} for logits "
                         f"{tuple(logits.shape)} on {logits.device}")
    top_k = int(top_k)
    if not 0 <= top_k <= min(MAX_TOP, vocab):
        raise ValueError(f"token_logprobs: top_k {top_k} outside [0, {min(MAX_TOP, vocab)}]")
    temperature = float(temperature)
    if not 1e-4 <= temperature <= 1e4:
        raise ValueError(f"token_logprobs: temperature {temperature} outside [1e-4, 1e4]")
    flat = logits if len(lead) == 1 else logits.reshape(-1, vocab)
    if flat.stride(1) != 1 or _ld(flat) < vocab:
        flat = flat.contiguous()
    ids = (ids if len(lead) == 1 else ids.reshape(-1)).contiguous()
    if _lib.needs_grad(flat):
        out = TokenLogprobsFn.apply(flat, ids, top_k, temperature)
    else:
        out = _forward(flat, ids, top_k, temperature)[:4]
    if len(lead) == 1:
        return TokenLogprobs(*out)
    return TokenLogprobs(out[0].view(lead), out[1].view(lead), out[2].view(*lead, top_k),
                         out[3].view(*lead, top_k))
