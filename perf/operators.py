"""The cases by which the row operators of a training step are timed, and their plain forms.

Four operators: the scaled embedding with its gradient (testt_b200.embed), the per-head norms of
queries and keys with the rotation (testt_b200.norm_rope), the log-probabilities of given tokens
with entropy and top alternatives (testt_b200.logprobs) and dropout from a counter-based generator
(testt_b200.dropout). `own` False: elementary torch operations in 32 bits, rounded once; True: the
calls a user makes of the package.
"""

import math

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
SIZE = {"fp16": 2, "bf16": 2, "fp32": 4}


def listed():
    return [
        # a handful of tokens looked up while scoring or sampling: latency alone
        dict(name="embed few", op="embed", n=17, vocab=151936, hidden=1536, dtype="fp16",
             out="fp32", scale=1.0, pad=-1, grad=False),
        # the embedding of a training step's real tokens, its table trained: the dense gradient
        dict(name="embed step", op="embed", n=621, vocab=151936, hidden=1536, dtype="fp16",
             out="fp32", scale=39.1918359, pad=-1, grad=True),
        # a long packed batch on a smaller, odd vocabulary, with a padding id without gradient
        dict(name="embed long", op="embed", n=32749, vocab=50021, hidden=2056, dtype="bf16",
             out="bf16", scale=45.25, pad=7, grad=True),
        # q|k|v of a few tokens, forward only
        dict(name="heads few", op="heads", n=5, nh=12, nkv=2, d=128, rot=128, table=2048,
             dtype="fp16", lora=False, grad=False),
        # a training step's q|k|v with the LoRA rows of q and v
        dict(name="heads step", op="heads", n=621, nh=12, nkv=2, d=128, rot=128, table=512,
             dtype="fp16", lora=True, grad=True),
        # a long packed batch, many heads, half of each head rotated
        dict(name="heads long", op="heads", n=16411, nh=32, nkv=8, d=128, rot=64, table=32768,
             dtype="bf16", lora=False, grad=True),
        # the next token's alternatives for a few sequences
        dict(name="tokens few", op="tokens", n=3, vocab=151936, dtype="fp16", k=20, temp=1.0,
             masked=0, grad=False),
        # a policy-gradient step: log-probability and entropy, both with gradients
        dict(name="tokens step", op="tokens", n=621, vocab=151936, dtype="fp16", k=0, temp=1.0,
             masked=267, grad=True),
        # distillation on the top alternatives, fp32 logits, an odd vocabulary, a temperature
        dict(name="tokens top", op="tokens", n=1531, vocab=50021, dtype="fp32", k=8, temp=0.7,
             masked=21, grad=True),
        # scoring and training a long batch
        dict(name="tokens long", op="tokens", n=2048, vocab=151936, dtype="bf16", k=5, temp=1.0,
             masked=267, grad=True),
        # the adapter input of a training step
        dict(name="dropout step", op="dropout", rows=621, cols=1536, dtype="fp32", res="none",
             p=0.05, offset=0, grad=True),
        # a long batch's block output dropped and added to the fp32 residual stream
        dict(name="dropout long", op="dropout", rows=16411, cols=2048, dtype="fp16", res="fp32",
             p=0.1, offset=2 ** 33 + 5, grad=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["embed", "heads", "tokens", "dropout"])
    dtype = rng.choice(["fp16", "bf16", "fp32"])
    grad = rng.random() < 0.7
    if op == "embed":
        hidden = 8 * _log(rng, 8, 512) if rng.random() < 0.7 else _log(rng, 65, 2500)
        vocab = _log(rng, 500, min(151936, 240000000 // hidden))
        n = _log(rng, 1, max(2, min(40000, 67000000 // hidden)))
        return dict(op=op, n=n, vocab=vocab, hidden=hidden, dtype=dtype,
                    out=rng.choice([dtype, "fp32"]), scale=rng.choice([1.0, math.sqrt(hidden)]),
                    pad=rng.choice([-1, 0]), grad=grad)
    if op == "heads":
        d = rng.choice([64, 80, 96, 128, 160, 256])
        nkv = rng.choice([1, 2, 4, 8])
        nh = nkv * rng.choice([1, 3, 4, 6])
        n = _log(rng, 1, max(2, min(40000, 100000000 // ((nh + 2 * nkv) * d))))
        return dict(op=op, n=n, nh=nh, nkv=nkv, d=d, rot=rng.choice([d, d, d // 2]),
                    table=_log(rng, 64, 40000), dtype=dtype, lora=rng.random() < 0.4, grad=grad)
    if op == "tokens":
        vocab = _log(rng, 1000, 200000)
        n = _log(rng, 1, max(2, min(8192, 150000000 // vocab)))
        return dict(op=op, n=n, vocab=vocab, dtype=dtype, k=rng.choice([0, 1, 2, 5, 8, 20, 32]),
                    temp=rng.choice([1.0, 0.7, 1.3]), masked=rng.choice([0, vocab // 9]), grad=grad)
    cols = _log(rng, 1, 8000)
    rows = _log(rng, 1, max(2, min(40000, 50000000 // cols)))
    return dict(op=op, rows=rows, cols=cols, dtype=dtype, res=rng.choice(["none", dtype, "fp32"]),
                p=rng.choice([0.05, 0.1, 0.5]), offset=rng.choice([0, 77, 2 ** 32 - 3]), grad=grad)


# ---- inputs -----------------------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed) * 7919 + 13)


def _randn(g, *shape, dtype=torch.float32, std=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * std).to(dtype)


def prepare(case, seed):
    g = _gen(seed)
    dt = TYPES[case["dtype"]]
    s = dict(case=case)
    if case["op"] == "embed":
        n, v, h = case["n"], case["vocab"], case["hidden"]
        # token ids as text has them: a few very frequent ones, a long tail
        u = torch.rand(n, generator=g, device=DEV, dtype=torch.float64)
        s["ids"] = ((v + 1.0) ** u - 1.0).long().clamp_(0, v - 1)
        s["table"] = _randn(g, v, h, dtype=dt, std=0.02).requires_grad_(case["grad"])
        if case["grad"]:
            s["dy"] = _randn(g, n, h, dtype=TYPES[case["out"]], std=0.01)
    elif case["op"] == "heads":
        n, nh, nkv, d, rot = (case[k] for k in ("n", "nh", "nkv", "d", "rot"))
        s["qkv"] = _randn(g, n, (nh + 2 * nkv) * d, dtype=dt).requires_grad_(case["grad"])
        s["lq"] = _randn(g, n, nh * d, dtype=dt, std=0.1) if case["lora"] else None
        s["lv"] = _randn(g, n, nkv * d, dtype=dt, std=0.1) if case["lora"] else None
        s["qw"] = (1 + _randn(g, d, std=0.2)).to(dt).requires_grad_(case["grad"])
        s["kw"] = (1 + _randn(g, d, std=0.2)).to(dt).requires_grad_(case["grad"])
        # the angles of far positions need 64 bits
        freq = 1e6 ** (-torch.arange(0, rot, 2, device=DEV, dtype=torch.float64) / rot)
        ang = torch.arange(case["table"], device=DEV, dtype=torch.float64)[:, None] * freq
        s["cos"] = torch.cat([ang.cos(), ang.cos()], 1).float()
        s["sin"] = torch.cat([ang.sin(), ang.sin()], 1).float()
        # positions run on from a place of the table and wrap to its start
        start = torch.randint(0, case["table"], (1,), generator=g, device=DEV)
        s["pos"] = (torch.arange(n, device=DEV) + start) % case["table"]
        if case["grad"]:
            s["dq"] = _randn(g, n, nh, d, dtype=dt)
            s["dk"] = _randn(g, n, nkv, d, dtype=dt)
            s["dv"] = _randn(g, n, nkv, d, dtype=dt)
    elif case["op"] == "tokens":
        n, v, k = case["n"], case["vocab"], case["k"]
        z = torch.empty(n, v, device=DEV, dtype=dt).normal_(generator=g) * 3
        if case["masked"]:  # a vocabulary padded to a rounder size
            z[:, v - case["masked"]:] = -math.inf
        s["logits"] = z.requires_grad_(case["grad"])
        s["ids"] = torch.randint(0, v - case["masked"], (n,), generator=g, device=DEV)
        if case["grad"]:
            s["g_lp"] = _randn(g, n)
            s["g_ent"] = _randn(g, n, std=0.01)
            s["g_top"] = _randn(g, n, k) if k else None
    else:
        r, c = case["rows"], case["cols"]
        s["x"] = _randn(g, r, c, dtype=dt).requires_grad_(case["grad"])
        s["res"] = None if case["res"] == "none" else _randn(g, r, c, dtype=TYPES[case["res"]])
        if case["grad"]:
            s["dy"] = _randn(g, r, c, dtype=dt if s["res"] is None else s["res"].dtype)
        s["seed"] = int(seed) * 0x9E3779B97F4A7C15 % 2 ** 63
    return s


# ---- one pass ---------------------------------------------------------------------------------


def run(state):
    case = state["case"]
    if own:
        return {"embed": _own_embed, "heads": _own_heads, "tokens": _own_tokens,
                "dropout": _own_dropout}[case["op"]](state, case)
    with torch.no_grad():
        return {"embed": _plain_embed, "heads": _plain_heads, "tokens": _plain_tokens,
                "dropout": _plain_dropout}[case["op"]](state, case)


def _own_embed(s, c):
    from testt_b200.embed import embedding

    y = embedding(s["ids"], s["table"], scale=c["scale"],
                  padding_idx=c["pad"] if c["pad"] >= 0 else None, out_dtype=TYPES[c["out"]])
    if not c["grad"]:
        return {"y": y}
    (dw,) = torch.autograd.grad(y, s["table"], s["dy"])
    return {"y": y, "dw": dw}


def _plain_embed(s, c):
    ids, table = s["ids"], s["table"]
    out = {"y": (table[ids].float() * c["scale"]).to(TYPES[c["out"]])}
    if c["grad"]:
        dy = s["dy"].float() * c["scale"]
        if c["pad"] >= 0:
            dy = dy * (ids != c["pad"]).float()[:, None]
        dw = torch.zeros(table.shape, device=DEV)
        dw.index_add_(0, ids, dy)
        out["dw"] = dw.to(table.dtype)
    return out


def _own_heads(s, c):
    from testt_b200.norm_rope import norm_rope_tokens

    q, k, v = norm_rope_tokens(s["qkv"], s["lq"], s["lv"], s["qw"], s["kw"], 1e-6, s["cos"],
                               s["sin"], s["pos"], 1, c["table"], c["nh"], c["nkv"], c["d"])
    out = {"q": q, "k": k, "v": v}
    if c["grad"]:
        out["dqkv"], out["dqw"], out["dkw"] = torch.autograd.grad(
            (q, k, v), (s["qkv"], s["qw"], s["kw"]), (s["dq"], s["dk"], s["dv"]))
    return out


def _turn(x, cos, sin, sign=1.0):
    """x cos + half-turned x sin on the first rot dims; sign -1: the transposed rotation (the
    tables' two halves are alike)."""
    rot = cos.shape[-1]
    a, b, rest = x[..., :rot // 2], x[..., rot // 2:rot], x[..., rot:]
    ca, cb, sa, sb = cos[..., :rot // 2], cos[..., rot // 2:], sin[..., :rot // 2], sin[..., rot // 2:]
    return torch.cat([a * ca - sign * (b * sa), b * cb + sign * (a * sb), rest], -1)


def _plain_heads(s, c):
    n, nh, nkv, d = c["n"], c["nh"], c["nkv"], c["d"]
    dt = s["qkv"].dtype
    x = s["qkv"].float().reshape(n, nh + 2 * nkv, d)
    xq, xk, v = x[:, :nh], x[:, nh:nh + nkv], x[:, nh + nkv:]
    if s["lq"] is not None:
        xq = xq + s["lq"].float().reshape(n, nh, d)
        v = v + s["lv"].float().reshape(n, nkv, d)
    cos, sin = s["cos"][s["pos"]][:, None], s["sin"][s["pos"]][:, None]
    out = {"v": v.to(dt)}
    grads = []
    for name, xx, w, dy in (("q", xq, s["qw"], s.get("dq")), ("k", xk, s["kw"], s.get("dk"))):
        r = torch.rsqrt((xx * xx).mean(-1, keepdim=True) + 1e-6)
        hat = xx * r
        out[name] = _turn(hat * w.float(), cos, sin).to(dt)
        if c["grad"]:
            dn = _turn(dy.float(), cos, sin, -1.0)
            g = dn * w.float()
            grads.append(r * (g - hat * (g * hat).mean(-1, keepdim=True)))
            out["d%sw" % name] = (dn * hat).sum((0, 1)).to(dt)
    if c["grad"]:
        out["dqkv"] = torch.cat(grads + [s["dv"].float()], 1).reshape(n, -1).to(dt)
    return out


def _own_tokens(s, c):
    from testt_b200.logprobs import token_logprobs

    o = token_logprobs(s["logits"], s["ids"], top_k=c["k"], temperature=c["temp"])
    out = {"lp": o.logprob, "ent": o.entropy}
    if c["k"]:
        out["top_lp"], out["top_ids"] = o.top_logprobs, o.top_ids
    if c["grad"]:
        outs, gs = [o.logprob, o.entropy], [s["g_lp"], s["g_ent"]]
        if c["k"]:
            outs.append(o.top_logprobs)
            gs.append(s["g_top"])
        (out["dlogits"],) = torch.autograd.grad(outs, s["logits"], gs)
    return out


def _plain_tokens(s, c):
    logits, k = s["logits"], c["k"]
    z = logits.float()
    out = {}
    if k:
        # the ordered bits of the value above the reversed index: equal values, lowest index first
        bits = z.view(torch.int32).long()
        bits = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
        key = bits * 2 ** 32 + torch.arange(c["vocab"] - 1, -1, -1, device=DEV)
        out["top_ids"] = (c["vocab"] - 1) - (key.topk(k).values & 0xFFFFFFFF)
        del bits, key
    z = z * (1.0 / c["temp"])
    z = z - z.amax(-1, keepdim=True)
    p = torch.exp(z)
    total = p.sum(-1, keepdim=True)
    p = p / total
    lp = z - torch.log(total)
    out["lp"] = lp.gather(1, s["ids"][:, None])[:, 0]
    plp = torch.where(p > 0, p * lp, torch.zeros_like(p))
    out["ent"] = -plp.sum(-1)
    if k:
        out["top_lp"] = lp.gather(1, out["top_ids"])
    if c["grad"]:
        del lp
        sum_g = s["g_lp"] if not k else s["g_lp"] + s["g_top"].sum(-1)
        d = -p * sum_g[:, None] - s["g_ent"][:, None] * (plp + p * out["ent"][:, None])
        d.scatter_add_(1, s["ids"][:, None], s["g_lp"][:, None])
        if k:
            d.scatter_add_(1, out["top_ids"], s["g_top"])
        out["dlogits"] = (d * (1.0 / c["temp"])).to(logits.dtype)
    return out


def _own_dropout(s, c):
    from testt_b200.dropout import dropout

    y = dropout(s["x"], c["p"], s["seed"], c["offset"], residual=s["res"])
    if not c["grad"]:
        return {"y": y}
    (dx,) = torch.autograd.grad(y, s["x"], s["dy"])
    return {"y": y, "dx": dx}


def _plain_words(seed, offset, n):
    """The generator's 32-bit words 0 .. n - 1: four for each counter (Philox 4x32, 10 rounds;
    Salmon, Moraes, Dror, Shaw 2011). int64 products wrap modulo 2^64, which leaves both halves
    of a 32 x 32 bit product right."""
    low = 0xFFFFFFFF
    ctr = offset + torch.arange((n + 3) // 4, device=DEV)
    c0, c1 = ctr & low, (ctr >> 32) & low
    c2 = c3 = torch.zeros_like(c0)
    k0, k1 = seed & low, (seed >> 32) & low
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = (((b >> 32) & low) ^ c1 ^ k0, b & low, ((a >> 32) & low) ^ c3 ^ k1, a & low)
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return torch.stack([c0, c1, c2, c3], 1).reshape(-1)[:n]


def _plain_dropout(s, c):
    x, res, p = s["x"], s["res"], c["p"]
    keep = (_plain_words(s["seed"], c["offset"], x.numel()) >= round(p * 2 ** 32)).reshape(x.shape)
    scale = 1.0 / (1.0 - p)
    y = torch.where(keep, x.float() * scale, torch.zeros((), device=DEV))
    out = {"y": y.to(x.dtype) if res is None else (res.float() + y).to(res.dtype)}
    if c["grad"]:
        out["dx"] = torch.where(keep, s["dy"].float() * scale, torch.zeros((), device=DEV)).to(x.dtype)
    return out


# ---- what a pass cannot do without -------------------------------------------------------------


def work(case):
    e = SIZE[case["dtype"]]
    if case["op"] == "embed":
        n, v, h, eo = case["n"], case["vocab"], case["hidden"], SIZE[case["out"]]
        r = np.arange(v, dtype=np.float64)
        p = np.log1p(1.0 / (r + 1.0)) / math.log(v + 1.0)
        distinct = float(-np.expm1(n * np.log1p(-p)).sum())
        b = 8 * n + distinct * h * e + n * h * eo
        if case["grad"]:
            b += n * h * eo + v * h * e
        return {"bytes": b, "flops": n * h * (3 if case["grad"] else 1)}
    if case["op"] == "heads":
        n, d = case["n"], case["d"]
        qk, w = (case["nh"] + case["nkv"]) * d, (case["nh"] + 2 * case["nkv"]) * d
        table = 2 * 4 * case["rot"] * min(n, case["table"])
        lora = n * (case["nh"] + case["nkv"]) * d * e if case["lora"] else 0
        b, f = 2 * n * w * e + lora + table + 8 * n, 8 * n * qk
        if case["grad"]:
            b += n * (2 * w + qk) * e + lora
            f += 18 * n * qk
        return {"bytes": b, "flops": f}
    if case["op"] == "tokens":
        cells = case["n"] * case["vocab"]
        return {"bytes": cells * e * (3 if case["grad"] else 1) + case["n"] * (16 + 12 * case["k"]),
                "flops": cells * (12 if case["grad"] else 6)}
    cells = case["rows"] * case["cols"]
    eo = e if case["res"] == "none" else SIZE[case["res"]]
    b = cells * (e + eo + (0 if case["res"] == "none" else eo))
    if case["grad"]:
        b += cells * (eo + e)
    return {"bytes": b, "flops": cells * (30 if case["grad"] else 16)}


# ---- the definitions in 64 bits ----------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"embed": _exact_embed, "heads": _exact_heads, "tokens": _exact_tokens,
                "dropout": _exact_dropout}[case["op"]](s, case)


def _exact_embed(s, c):
    ids = s["ids"]
    out = {"y": s["table"].index_select(0, ids).double().mul_(c["scale"])}
    if c["grad"]:
        dw = torch.zeros(s["table"].shape, device=DEV, dtype=torch.float64)
        dy = s["dy"].double()
        order = torch.argsort(ids, stable=True)
        vals, counts = torch.unique_consecutive(ids[order], return_counts=True)
        # the rows of each id are consecutive in the sorted order: sums by lengths
        sums = torch.segment_reduce(dy[order], "sum", lengths=counts, axis=0)
        dw[vals] = sums * c["scale"]
        if c["pad"] >= 0:
            dw[c["pad"]] = 0
        out["dw"] = dw
    return out


def _exact_heads(s, c):
    n, nh, nkv, d, rot = c["n"], c["nh"], c["nkv"], c["d"], c["rot"]
    x = s["qkv"].double().view(n, -1, d).clone()
    if c["lora"]:
        x[:, :nh] += s["lq"].double().view(n, nh, d)
        x[:, nh + nkv:] += s["lv"].double().view(n, nkv, d)
    cos = s["cos"].double().index_select(0, s["pos"])
    sin = s["sin"].double().index_select(0, s["pos"])
    turn = torch.zeros(n, d, d, device=DEV, dtype=torch.float64) if n * d * d <= 5e7 else None
    i = torch.arange(rot // 2, device=DEV)
    j = i + rot // 2

    def rotate(v, back):  # v [n, heads, d]
        if turn is not None:  # as a matrix of each position
            return torch.einsum("nab,nhb->nha" if not back else "nba,nhb->nha", turn, v)
        r = v.clone()
        ci, cj, si, sj = cos[:, None, i], cos[:, None, j], sin[:, None, i], sin[:, None, j]
        r[..., i] = v[..., i] * ci + (v[..., j] * sj if back else -v[..., j] * si)
        r[..., j] = v[..., j] * cj + (-v[..., i] * si if back else v[..., i] * sj)
        return r

    if turn is not None:
        rest = torch.arange(rot, d, device=DEV)
        turn[:, rest, rest] = 1.0
        turn[:, i, i], turn[:, j, j] = cos[:, i], cos[:, j]
        turn[:, i, j], turn[:, j, i] = -sin[:, i], sin[:, j]
    out = {"v": x[:, nh + nkv:]}
    if c["grad"]:
        dx = torch.empty_like(x)
        dx[:, nh + nkv:] = s["dv"].double()
    for name, lo, hi in (("q", 0, nh), ("k", nh, nh + nkv)):
        xx, w = x[:, lo:hi], s[name + "w"].double()
        ms = xx.pow(2).sum(-1, keepdim=True) / d + 1e-6
        out[name] = rotate(xx / ms.sqrt() * w, False)
        if c["grad"]:
            dn = rotate(s["d" + name].double(), True)
            out["d%sw" % name] = (dn * xx / ms.sqrt()).sum(1).sum(0)
            dot = (dn * w * xx).sum(-1, keepdim=True)
            dx[:, lo:hi] = dn * w / ms.sqrt() - xx * dot / (d * ms.pow(1.5))
    if c["grad"]:
        out["dqkv"] = dx.view(n, -1)
    return out


def _exact_tokens(s, c):
    n, v, k = c["n"], c["vocab"], c["k"]
    step = max(1, int(6e7) // v)
    parts = []
    for a in range(0, n, step):
        x = s["logits"][a:a + step].double()
        ids = s["ids"][a:a + step]
        r = torch.arange(x.shape[0], device=DEV)
        z = x / c["temp"]
        logp = torch.log_softmax(z, -1)
        prob = logp.exp()
        safe = logp.masked_fill(prob == 0, 0.0)
        ent = -(prob * safe).sum(-1)
        part = {"lp": logp[r, ids], "ent": ent}
        if k:
            order = x.sort(stable=True, dim=-1, descending=True).indices[:, :k]
            part["top_lp"], part["top_ids"] = logp.gather(1, order), order
        if c["grad"]:
            g = torch.zeros_like(x)  # the gradient that reaches each log-probability
            g[r, ids] += s["g_lp"][a:a + step].double()
            if k:
                g.scatter_add_(1, order, s["g_top"][a:a + step].double())
            g -= s["g_ent"][a:a + step].double()[:, None] * prob * (safe + 1.0)
            part["dlogits"] = (g - prob * g.sum(-1, keepdim=True)) / c["temp"]
        parts.append(part)
    return {key: torch.cat([p[key] for p in parts]) for key in parts[0]}


def _exact_dropout(s, c):
    n = c["rows"] * c["cols"]
    m0, m1, w0, w1 = (np.uint64(v) for v in (0xD2511F53, 0xCD9E8D57, 0x9E3779B9, 0xBB67AE85))
    low, half = np.uint64(0xFFFFFFFF), np.uint64(32)
    keep = np.empty(((n + 3) // 4, 4), dtype=bool)
    bar = np.uint64(round(c["p"] * 2 ** 32))
    for a in range(0, keep.shape[0], 1 << 20):
        ctr = np.arange(a, min(a + (1 << 20), keep.shape[0]), dtype=np.uint64) + np.uint64(c["offset"])
        x = [ctr & low, ctr >> half, np.zeros_like(ctr), np.zeros_like(ctr)]
        key = [np.uint64(s["seed"]) & low, np.uint64(s["seed"]) >> half]
        for rnd in range(10):
            if rnd:
                key = [(key[0] + w0) & low, (key[1] + w1) & low]
            p0, p1 = x[0] * m0, x[2] * m1
            x = [(p1 >> half) ^ x[1] ^ key[0], p1 & low, (p0 >> half) ^ x[3] ^ key[1], p0 & low]
        for w in range(4):
            keep[a:a + ctr.size, w] = x[w] >= bar
    mask = torch.from_numpy(keep.reshape(-1)[:n]).to(DEV).view(c["rows"], c["cols"])
    kept = mask.double() / (1.0 - c["p"])
    y = s["x"].double() * kept
    out = {"y": y if s["res"] is None else y + s["res"].double()}
    if c["grad"]:
        out["dx"] = s["dy"].double() * kept
    return out
