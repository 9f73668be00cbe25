"""Per-head RMS norms of queries and keys, the LoRA add and the rotary embedding in one pass on
B200 (tb_norm_rope_fwd / tb_norm_rope_bwd): rope.rope_tokens (reference: solution/rope.py) for
decoders that norm each query and key head before the rotation.

    x = qkv + lora                                            fp32
    q, k: n = x * rsqrt(mean(x^2 over the head) + eps) * (weight_offset + weight)
          y = n cos + half-turned n sin on the first rot dims, n past them
    v = x
Outputs are token-major (q [rows, n_heads, d], k and v [rows, n_kv, d]), the layout
attention.varlen_attention takes. The forward keeps nothing but its inputs: the backward forms
the norms again from them.
"""

import torch
from torch.autograd.function import once_differentiable

from . import _lib


def _ld(qkv):
    """Elements between rows (a single row's stride may be anything)."""
    return qkv.stride(0) if qkv.shape[0] > 1 else qkv.shape[1]


def _code(t, default):
    return default if t is None else _lib.TYPE_CODES[t.dtype]


def _forward(qkv, lora_q, lora_v, q_weight, k_weight, eps, cos, sin, pos_idx, batch, seq, n_heads,
             n_kv, head_dim, weight_offset):
    rows = qkv.shape[0]
    code = _lib.TYPE_CODES[qkv.dtype]
    q = qkv.new_empty((rows, n_heads, head_dim))
    k = qkv.new_empty((rows, n_kv, head_dim))
    v = torch.empty_like(k)
    if rows:
        _lib.call_on(qkv, "tb_norm_rope_fwd", qkv.data_ptr(), code, _ld(qkv), _lib.addr(lora_q),
                     _lib.addr(lora_v), _code(lora_q if lora_q is not None else lora_v, code),
                     _lib.addr(q_weight), _lib.addr(k_weight),
                     _code(q_weight if q_weight is not None else k_weight, code), weight_offset,
                     eps, cos.data_ptr(), sin.data_ptr(), cos.shape[1], pos_idx.data_ptr(),
                     q.data_ptr(), k.data_ptr(), v.data_ptr(), rows, batch, seq, n_heads, n_kv,
                     head_dim)
    return q, k, v


class NormRopeTokens(torch.autograd.Function):
    @staticmethod
    def forward(ctx, qkv, lora_q, lora_v, q_weight, k_weight, eps, cos, sin, pos_idx, *dims):
        ctx.save_for_backward(qkv, lora_q, q_weight, k_weight, cos, sin, pos_idx)
        ctx.dims = (eps, *dims)
        ctx.set_materialize_grads(False)
        return _forward(qkv, lora_q, lora_v, q_weight, k_weight, eps, cos, sin, pos_idx, *dims)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_q, grad_k, grad_v):
        qkv, lora_q, q_weight, k_weight, cos, sin, pos_idx = ctx.saved_tensors
        eps, batch, seq, n_heads, n_kv, head_dim, weight_offset = ctx.dims
        need = ctx.needs_input_grad
        rows = qkv.shape[0]
        code = _lib.TYPE_CODES[qkv.dtype]
        grads = [None if g is None else g.contiguous() for g in (grad_q, grad_k, grad_v)]
        dqkv = qkv.new_empty((rows, (n_heads + 2 * n_kv) * head_dim))
        dqw = torch.empty_like(q_weight) if need[3] else None
        dkw = torch.empty_like(k_weight) if need[4] else None
        ws, nbytes = None, 0
        if need[3] or need[4]:
            nbytes = _lib.workspace_bytes(qkv, "tb_norm_rope_bwd_workspace", rows, n_heads, n_kv,
                                          head_dim)
            ws = cos.new_empty(max(nbytes // 4, 1))
        _lib.call_on(qkv, "tb_norm_rope_bwd", *(_lib.addr(g) for g in grads), qkv.data_ptr(), code,
                     _ld(qkv), _lib.addr(lora_q), _code(lora_q, code), _lib.addr(q_weight),
                     _lib.addr(k_weight),
                     _code(q_weight if q_weight is not None else k_weight, code), weight_offset,
                     eps, cos.data_ptr(), sin.data_ptr(), cos.shape[1], pos_idx.data_ptr(),
                     dqkv.data_ptr(), _lib.addr(dqw), _lib.addr(dkw),
                     _lib.addr(ws), nbytes, rows, batch, seq, n_heads, n_kv, head_dim)
        q_cols, v_start = n_heads * head_dim, (n_heads + n_kv) * head_dim
        return (dqkv if need[0] else None, dqkv[:, :q_cols] if need[1] else None,
                dqkv[:, v_start:] if need[2] else None, dqw, dkw, None, None, None, None, None,
                None, None, None, None, None)


def _pair(a, b, dtype):
    """Two optional tensors contiguous and in one type the kernels take (`dtype`'s or fp32)."""
    if (a is None or a.dtype == dtype) and (b is None or b.dtype == dtype):
        return None if a is None else a.contiguous(), None if b is None else b.contiguous()
    return (None if a is None else a.to(torch.float32).contiguous(),
            None if b is None else b.to(torch.float32).contiguous())


def _check(t, name, shape, index):
    if t.shape != shape or t.get_device() != index:
        raise ValueError(f"norm_rope_tokens: {name} {tuple(t.shape)} on {t.device}, expected "
                         f"{shape} beside qkv")
    if t.dtype not in _lib.TYPE_CODES:
        raise TypeError(f"norm_rope_tokens: {name} must be fp16, bf16 or fp32, got {t.dtype}")


def norm_rope_tokens(qkv, lora_q, lora_v, q_weight, k_weight, eps, cos, sin, pos_idx, batch, seq,
                     n_heads, n_kv, head_dim, weight_offset=0.0):
    """(q, k, v) token-major in qkv's dtype (fp16, bf16 or fp32), as rope.rope_tokens with each
    query and key head normed first. `lora_q` [rows, n_heads * head_dim] and `lora_v` [rows,
    n_kv * head_dim] are added in fp32 (None: none); `q_weight`, `k_weight` [head_dim] (None: 1);
    `cos`, `sin` [>= seq, rot] with rot <= head_dim; a token's table row is pos_idx % seq, and one
    whose pos_idx is outside [0, batch * seq) gets zero rows and no gradient. qkv's rows may be
    views of wider rows; in 16-bit types rows that do not start on 16 bytes are several times slower
    than a contiguous copy. Differentiable in qkv, lora_q, lora_v, q_weight and k_weight. Gradients
    of the LoRA rows are qkv's gradient's columns, as in rope.rope_tokens: fp32 rows beside 16-bit
    qkv get values rounded to qkv's type (beside fp16, 0 below 3e-8 and infinite above 65504)."""
    _lib.require_cuda(qkv, lora_q, lora_v, q_weight, k_weight, cos, sin, pos_idx,
                      what="norm_rope_tokens")
    dtype, rows = qkv.dtype, qkv.shape[0] if qkv.dim() else 0
    if dtype not in _lib.TYPE_CODES:
        raise TypeError(f"norm_rope_tokens: qkv must be fp16, bf16 or fp32, got {dtype}")
    if n_heads <= 0 or n_kv < 0 or head_dim <= 0 or head_dim % 2:
        raise ValueError(f"norm_rope_tokens: {n_heads} / {n_kv} heads of {head_dim}")
    width = (n_heads + 2 * n_kv) * head_dim
    if qkv.dim() != 2 or qkv.shape[1] != width:
        raise ValueError(f"norm_rope_tokens: qkv {tuple(qkv.shape)}, expected [rows, {width}]")
    index = qkv.get_device()
    if lora_q is not None:
        _check(lora_q, "lora_q", (rows, n_heads * head_dim), index)
    if lora_v is not None:
        _check(lora_v, "lora_v", (rows, n_kv * head_dim), index)
    if q_weight is not None:
        _check(q_weight, "q_weight", (head_dim,), index)
    if k_weight is not None:
        _check(k_weight, "k_weight", (head_dim,), index)
    rot = cos.shape[-1] if cos.dim() == 2 else -1
    if rot < 0 or rot % 2 or rot > head_dim or cos.shape != sin.shape or cos.shape[0] < seq or \
            cos.get_device() != index or sin.get_device() != index:
        raise ValueError(f"norm_rope_tokens: tables {tuple(cos.shape)} and {tuple(sin.shape)} for "
                         f"seq {seq}, head_dim {head_dim}")
    if pos_idx.dtype != torch.int64:
        if pos_idx.dtype != torch.int32:
            raise TypeError(f"norm_rope_tokens: pos_idx must be int64 or int32, got "
                            f"{pos_idx.dtype}")
        pos_idx = pos_idx.to(torch.int64)
    if pos_idx.dim() != 1 or pos_idx.shape[0] != rows or pos_idx.get_device() != index:
        raise ValueError(f"norm_rope_tokens: pos_idx {tuple(pos_idx.shape)} on {pos_idx.device}, "
                         f"expected {(rows,)} on {qkv.device}")
    if qkv.stride(1) != 1 or _ld(qkv) < width:
        qkv = qkv.contiguous()
    if lora_q is not None or lora_v is not None:
        lora_q, lora_v = _pair(lora_q, lora_v, dtype)
    q_weight, k_weight = _pair(q_weight, k_weight, dtype)
    if cos.dtype != torch.float32 or sin.dtype != torch.float32:
        cos, sin = cos.to(torch.float32), sin.to(torch.float32)
    args = (qkv, lora_q, lora_v, q_weight, k_weight, float(eps), cos.contiguous(),
            sin.contiguous(), pos_idx.contiguous(), int(batch), int(seq), int(n_heads), int(n_kv),
            int(head_dim), float(weight_offset))
    if _lib.needs_grad(qkv, lora_q, lora_v, q_weight, k_weight):
        return NormRopeTokens.apply(*args)
    return _forward(*args)
