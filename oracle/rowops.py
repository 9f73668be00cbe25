"""fp64 restatements of the row operators around a training step's GEMMs: the scaled embedding and
its gradient, the per-head norms with the rotation, the token log-probabilities and the
counter-based dropout. Plain torch / numpy on the CPU; `mag` results are the sums of the absolute
terms behind each value, which the tests' error bounds are built from."""

import numpy as np
import torch


def philox_words(seed, offset, n):
    """Words 0 .. n - 1 of Philox4x32-10 (Salmon, Moraes, Dror, Shaw, SC 2011), uint64 array."""
    low, half = np.uint64(0xFFFFFFFF), np.uint64(32)
    ctr = np.arange((n + 3) // 4, dtype=np.uint64) + np.uint64(offset)
    x = [ctr & low, ctr >> half, np.zeros_like(ctr), np.zeros_like(ctr)]
    k = [np.uint64(seed & 0xFFFFFFFF), np.uint64((seed >> 32) & 0xFFFFFFFF)]
    for _ in range(10):
        a, b = x[0] * np.uint64(0xD2511F53), x[2] * np.uint64(0xCD9E8D57)
        x = [(b >> half) ^ x[1] ^ k[0], b & low, (a >> half) ^ x[3] ^ k[1], a & low]
        k = [(k[0] + np.uint64(0x9E3779B9)) & low, (k[1] + np.uint64(0xBB67AE85)) & low]
    return np.stack(x, 1).reshape(-1)[:n]


def keep_mask(shape, p, seed, offset):
    n = int(np.prod(shape))
    return torch.from_numpy(philox_words(seed, offset, n) >= np.uint64(round(p * 2 ** 32))) \
        .reshape(shape)


def dropout(x, p, seed, offset=0, residual=None):
    keep = keep_mask(x.shape, p, seed, offset)
    y = torch.where(keep, x.double() / (1 - p) if p < 1 else torch.zeros(()).double(),
                    torch.zeros(()).double())
    return (y if residual is None else residual.double() + y), keep


def embedding(ids, table, scale):
    ids = ids.reshape(-1).long()
    ok = (ids >= 0) & (ids < table.shape[0])
    y = table.double()[ids.clamp(0, table.shape[0] - 1)] * scale
    return torch.where(ok[:, None], y, torch.zeros(()).double())


def embedding_grad(ids, dy, vocab, scale, padding_idx=None):
    """(gradient, mag, tokens of each id), all [vocab, ...]."""
    ids = ids.reshape(-1).long()
    dy = dy.reshape(ids.numel(), -1).double()
    ok = (ids >= 0) & (ids < vocab)
    if padding_idx is not None:
        ok &= ids != padding_idx
    dw = torch.zeros(vocab, dy.shape[1], dtype=torch.float64)
    mag, count = dw.clone(), torch.zeros(vocab, dtype=torch.long)
    for t in ok.nonzero()[:, 0].tolist():
        dw[ids[t]] += dy[t]
        mag[ids[t]] += dy[t].abs()
        count[ids[t]] += 1
    return dw * scale, mag * abs(scale), count


def _tables(cos, sin, pos, seq, slots, back):
    """The two dims each dim of a rotated head is made of: (partner index, own factor, partner's
    factor) per token, padded past rot with 1 and 0."""
    rot = cos.shape[1]
    h = rot // 2
    inside = (pos >= 0) & (pos < slots)
    t = torch.where(inside, pos, torch.zeros_like(pos)) % seq
    c, s = cos.double()[t], sin.double()[t]
    partner = torch.cat([torch.arange(h, rot), torch.arange(h)])
    if back:  # the transpose: y_i = g_i c_i + g_{i+h} s_{i+h}, y_{i+h} = g_{i+h} c_{i+h} - g_i s_i
        other = torch.cat([s[:, h:], -s[:, :h]], 1)
    else:
        other = torch.cat([-s[:, :h], s[:, h:]], 1)
    return rot, partner, c, other, inside


def _turn(x, tables):
    rot, partner, own, other, _ = tables
    y = x.clone()
    y[..., :rot] = x[..., :rot] * own[:, None] + x[..., partner] * other[:, None]
    return y


def _turn_mag(x, tables):
    rot, partner, own, other, _ = tables
    y = x.abs().clone()
    y[..., :rot] = (x[..., :rot] * own[:, None]).abs() + (x[..., partner] * other[:, None]).abs()
    return y


def norm_rope(qkv, lora_q, lora_v, q_weight, k_weight, eps, cos, sin, pos, batch, seq, nh, nkv, d,
              w0=0.0, grads=None):
    """dict of q, k, v (and their mags) and, for grads = (dq, dk, dv), dqkv, dqw, dkw and mags."""
    n = qkv.shape[0]
    x = qkv.double().reshape(n, nh + 2 * nkv, d).clone()
    if lora_q is not None:
        x[:, :nh] += lora_q.double().reshape(n, nh, d)
    if lora_v is not None:
        x[:, nh + nkv:] += lora_v.double().reshape(n, nkv, d)
    fwd = _tables(cos, sin, pos, seq, batch * seq, False)
    bwd = _tables(cos, sin, pos, seq, batch * seq, True)
    live = fwd[4][:, None, None].double()
    out = {"v": x[:, nh + nkv:] * live}
    dx, dxm = torch.zeros_like(x), torch.zeros_like(x)
    for name, a, b, w, i in (("q", 0, nh, q_weight, 0), ("k", nh, nh + nkv, k_weight, 1)):
        xx = x[:, a:b]
        ww = torch.ones(d, dtype=torch.float64) if w is None else w.double() + w0
        r = 1.0 / torch.sqrt((xx * xx).mean(-1, keepdim=True) + eps)
        out[name] = _turn(xx * r * ww, fwd) * live
        out[name + "_mag"] = _turn_mag(xx * r * ww, fwd) * live
        if grads is not None:
            g = grads[i]
            g = torch.zeros_like(xx) if g is None else g.double()
            dn, dnm = _turn(g, bwd) * live, _turn_mag(g, bwd) * live
            dot = (dn * ww * xx).mean(-1, keepdim=True)
            dotm = (dnm * ww.abs() * xx.abs()).mean(-1, keepdim=True)
            dx[:, a:b] = r * (dn * ww - xx * r * r * dot)
            dxm[:, a:b] = r * (dnm * ww.abs() + xx.abs() * r * r * dotm)
            out["d%sw" % name] = (dn * xx * r).sum((0, 1))
            out["d%sw_mag" % name] = (dnm * xx.abs() * r).sum((0, 1))
    if grads is not None:
        dv = grads[2]
        if dv is not None:
            dx[:, nh + nkv:] = dv.double() * live
        dxm[:, nh + nkv:] = dx[:, nh + nkv:].abs()
        out["dqkv"], out["dqkv_mag"] = dx.reshape(n, -1), dxm.reshape(n, -1)
    return out


def token_logprobs(logits, ids, top_k=0, temperature=1.0, grads=None):
    """dict of lp, ent, top_lp, top_ids and, for grads = (g_lp, g_ent, g_top) (each or None), dz and
    its mag. A row of -inf only: lp -inf, ent 0, no gradient; an id outside: lp 0."""
    x = logits.double()
    n, vocab = x.shape
    z = x / temperature
    empty = torch.isneginf(x).all(1)
    logp = torch.where(empty[:, None], torch.full_like(z, -np.inf), torch.log_softmax(z, 1))
    p = torch.where(empty[:, None], torch.zeros_like(z), logp.exp())
    logp0 = torch.where(p == 0, torch.zeros_like(z), logp)
    ok = (ids >= 0) & (ids < vocab)
    at = ids.long().clamp(0, vocab - 1)[:, None]
    out = {"lp": torch.where(ok, logp.gather(1, at)[:, 0], torch.zeros(n).double()),
           "ent": -(p * logp0).sum(1), "spread": (z.amax(1, keepdim=True) - z)}
    order = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :top_k]
    out["top_ids"], out["top_lp"] = order, logp.gather(1, order)
    if grads is not None:
        g_lp, g_ent, g_top = (None if g is None else g.double() for g in grads)
        hot = torch.zeros_like(z)
        if g_lp is not None:
            hot.scatter_add_(1, at, torch.where(ok, g_lp, torch.zeros_like(g_lp))[:, None])
        if g_top is not None and top_k:
            hot.scatter_add_(1, order, g_top)
        ge = torch.zeros(n).double() if g_ent is None else g_ent
        total = hot.sum(1, keepdim=True)
        slope = p * (total + ge[:, None] * (logp0 + out["ent"][:, None]))
        keep = (~empty)[:, None].double()
        out["dz"] = (hot - slope) / temperature * keep
        hotm = torch.zeros_like(z)
        if g_top is not None and top_k:
            hotm.scatter_add_(1, order, g_top.abs())
        if g_lp is not None:
            hotm.scatter_add_(1, at, torch.where(ok, g_lp.abs(), torch.zeros_like(g_lp))[:, None])
        out["dz_mag"] = (hotm + p * (hotm.sum(1, keepdim=True) + ge.abs()[:, None] *
                                     (logp0.abs() + out["ent"][:, None]))) / temperature * keep
        out["p"] = p
    return out
