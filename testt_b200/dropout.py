"""Dropout from a counter-based generator, with an optional residual add, on B200 (tb_dropout).

    y = residual + keep * x / (1 - p)

keep[i] is a function of (seed, offset, i) alone: word i % 4 of Philox4x32-10 (Salmon, Moraes,
Dror, Shaw, SC 2011) at counter offset + i / 4, i counting the elements of x in row-major order,
is at least round(p 2^32). No mask is stored: the backward draws it again. A call uses
counters(n) counters, so the next call under the same seed takes offset + counters(n); calls with
the same (seed, offset) draw the same mask. The reference runs PyTorch's dropout with a stored
byte mask (solution/model.py:195-206); lora.lora_pair keeps that, for equal draws.
"""

import torch
from torch.autograd.function import once_differentiable

from . import _lib


def counters(n):
    """Counters a call over n elements uses: what to add to `offset` for the next one."""
    return (int(n) + 3) // 4


def _launch(x, residual, out, threshold, scale, seed, offset, state=None, used=None):
    if x.numel():
        _lib.call_on(x, "tb_dropout", x.data_ptr(), _lib.TYPE_CODES[x.dtype], _lib.addr(residual),
                     out.data_ptr(), _lib.TYPE_CODES[out.dtype], x.numel(), threshold, scale, seed,
                     offset, _lib.addr(state), _lib.addr(used))
    return out


class CounterDropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, threshold, scale, seed, offset, state):
        ctx.dtype = x.dtype
        ctx.draw = (threshold, scale, seed, offset)
        out = torch.empty_like(x if residual is None else residual)
        if state is None:
            return _launch(x, residual, out, threshold, scale, seed, offset)
        # the caller may move its state on before the backward: keep what this call used
        used = torch.empty_like(state)
        ctx.save_for_backward(used)
        ctx.draw = (threshold, scale, 0, 0)
        return _launch(x, residual, out, threshold, scale, seed, offset, state, used)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        dx = None
        if ctx.needs_input_grad[0]:
            g = dy.contiguous()
            dx = torch.empty_like(g, dtype=ctx.dtype)
            _launch(g, None, dx, *ctx.draw, *ctx.saved_tensors)
        return dx, dy if ctx.needs_input_grad[1] else None, None, None, None, None, None


def dropout(x, p, seed, offset=0, residual=None):
    """residual + keep * x / (1 - p) (the residual optional) for fp16, bf16 or fp32 x of any shape;
    differentiable in x and residual. `residual` has x's shape and x's dtype or fp32; the output
    has its dtype (x's without one). `seed`: an int (its low 64 bits), or an int64 CUDA tensor of
    two elements (seed, offset) read when the kernel runs, which a captured graph's caller moves
    on between replays; `offset` is added to it. p 1 drops everything, p 0 keeps everything."""
    _lib.require_cuda(x, residual, what="dropout")
    if x.dtype not in _lib.TYPE_CODES:
        raise TypeError(f"dropout: x must be fp16, bf16 or fp32, got {x.dtype}")
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"dropout: p {p} outside [0, 1]")
    offset = int(offset)
    if not 0 <= offset < 2 ** 63:
        raise ValueError(f"dropout: offset {offset} outside [0, 2^63)")
    if residual is not None:
        if residual.shape != x.shape or residual.device != x.device:
            raise ValueError(f"dropout: residual {tuple(residual.shape)} on {residual.device} "
                             f"beside x {tuple(x.shape)} on {x.device}")
        if residual.dtype not in (x.dtype, torch.float32):
            raise TypeError(f"dropout: residual {residual.dtype} beside x {x.dtype}")
        residual = residual.contiguous()
    state = None
    if torch.is_tensor(seed):
        if seed.dtype != torch.int64 or seed.numel() != 2 or seed.device != x.device:
            raise ValueError("dropout: a seed tensor is int64 (seed, offset) on x's device")
        state, seed = seed.contiguous(), 0
    else:
        seed = int(seed) & 0xFFFFFFFFFFFFFFFF
        seed -= (seed >> 63) << 64
    x = x.contiguous()
    threshold, scale = round(p * 2 ** 32), 1.0 / (1.0 - p) if p < 1.0 else 0.0
    if _lib.needs_grad(x, residual):
        return CounterDropout.apply(x, residual, threshold, scale, seed, offset, state)
    return _launch(x, residual, torch.empty_like(x if residual is None else residual), threshold,
                   scale, seed, offset, state)
