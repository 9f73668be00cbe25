"""The row operators as one run, the way a training step with a trained table, normed heads and a
loss of token log-probabilities uses them: ids -> scaled embedding -> dropout onto the residual
stream -> q|k|v -> head norms with the rotation -> variable-length attention -> dropout + residual
-> logits -> log-probability and entropy. Gradients of every parameter against a plain fp64 run on
the same masks, and a captured step against the eager one."""

import pytest
import torch

from oracle import rowops

pytestmark = pytest.mark.gpu
DEV = "cuda"
NH, NKV, D, HID, V = 4, 2, 128, 96, 301
LENS = [5, 1, 23, 12]
P, SEED = 0.1, 77


def _setup():
    g = torch.Generator().manual_seed(5)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    rows = sum(LENS)
    pos = torch.cat([torch.arange(n) + 64 * i for i, n in enumerate(LENS)])
    inv = 1e4 ** (-torch.arange(0, D, 2).double() / D)
    ang = torch.arange(64).double()[:, None] * inv
    return dict(ids=torch.randint(0, V, (rows,), generator=g), pos=pos,
                cu=torch.tensor([0, *torch.tensor(LENS).cumsum(0).tolist()], dtype=torch.int32),
                cos=torch.cat([ang.cos()] * 2, 1).float(), sin=torch.cat([ang.sin()] * 2, 1).float(),
                targets=torch.randint(0, V, (rows,), generator=g), adv=r(rows)), \
        dict(table=r(V, HID) * 0.5, wqkv=r((NH + 2 * NKV) * D, HID) / HID ** 0.5,
             qw=1 + 0.2 * r(D), kw=1 + 0.2 * r(D), wo=r(HID, NH * D) / (NH * D) ** 0.5)


def _kernels(x, p, state=None):
    from testt_b200.attention import varlen_attention
    from testt_b200.dropout import counters, dropout
    from testt_b200.embed import embedding
    from testt_b200.logprobs import token_logprobs
    from testt_b200.norm_rope import norm_rope_tokens

    seed = SEED if state is None else state
    h = embedding(x["ids"], p["table"], scale=HID ** 0.5, padding_idx=3)
    h = dropout(h, P, seed)
    qkv = h @ p["wqkv"].t()
    q, k, v = norm_rope_tokens(qkv, None, None, p["qw"], p["kw"], 1e-6, x["cos"], x["sin"],
                               x["pos"], len(LENS), 64, NH, NKV, D)
    a = varlen_attention(q, k, v, x["cu"], max(LENS), D ** -0.5)
    o = a.reshape(-1, NH * D) @ p["wo"].t()
    s = dropout(o, P, seed, counters(h.numel()), residual=h)
    o = token_logprobs(s @ p["table"].t(), x["targets"], top_k=2, temperature=0.8)
    return (x["adv"] * o.logprob).sum() + 0.01 * o.entropy.sum()


def _plain(x, p):
    rows = x["ids"].numel()
    keep1 = rowops.keep_mask((rows, HID), P, SEED, 0)
    keep2 = rowops.keep_mask((rows, HID), P, SEED, (rows * HID + 3) // 4)
    table = p["table"]
    emb = table[x["ids"]]
    h = torch.where((x["ids"] == 3)[:, None], emb.detach(), emb) * HID ** 0.5
    h = h * keep1 / (1 - P)
    qkv = (h @ p["wqkv"].t()).reshape(rows, NH + 2 * NKV, D)
    c, s = (x[n].double()[x["pos"] % 64][:, None] for n in ("cos", "sin"))

    def turn(z, w):
        z = z * (z.pow(2).mean(-1, keepdim=True) + 1e-6).rsqrt() * w
        return z * c + torch.cat([-z[..., D // 2:], z[..., :D // 2]], -1) * s

    q, k, v = turn(qkv[:, :NH], p["qw"]), turn(qkv[:, NH:NH + NKV], p["kw"]), qkv[:, NH + NKV:]
    outs, at = [], 0
    for n in LENS:
        qs, ks, vs = (t[at:at + n].transpose(0, 1) for t in (q, k, v))
        ks, vs = (t.repeat_interleave(NH // NKV, 0) for t in (ks, vs))
        w = qs @ ks.transpose(1, 2) * D ** -0.5
        w = w.masked_fill(torch.ones(n, n).triu(1).bool(), -float("inf")).softmax(-1)
        outs.append((w @ vs).transpose(0, 1).reshape(n, NH * D))
        at += n
    s_ = h + (torch.cat(outs) @ p["wo"].t()) * keep2 / (1 - P)
    logp = torch.log_softmax(s_ @ table.t() / 0.8, 1)
    lp = logp.gather(1, x["targets"][:, None])[:, 0]
    ent = -(logp.exp() * logp).sum(1)
    return (x["adv"].double() * lp).sum() + 0.01 * ent.sum()


def test_loss_and_gradients():
    x, p = _setup()
    gx = {k: v.to(DEV) for k, v in x.items()}
    gp = {k: v.half().to(DEV).requires_grad_() for k, v in p.items()}
    loss = _kernels(gx, gp)
    grads = torch.autograd.grad(loss, list(gp.values()))
    dp = {k: v.half().double().requires_grad_() for k, v in p.items()}
    want = _plain(x, dp)
    wgrads = torch.autograd.grad(want, list(dp.values()))
    # every fp16 value on the way (about ten deep) is off by half a step (2^-11) of the values it
    # came from; relative to the tensor's norm the roundings add up as independent ones
    assert abs(float(loss.detach()) - float(want.detach())) < 12 * 2.0 ** -11 * float(x["adv"].abs().sum())
    for name, a, b in zip(gp, grads, wgrads):
        err = (a.cpu().double() - b).norm() / b.norm()
        assert err < 12 * 2.0 ** -11, (name, float(err))


def test_captured_step_repeats_the_eager_one():
    x, p = _setup()
    gx = {k: v.to(DEV) for k, v in x.items()}
    gp = {k: v.half().to(DEV).requires_grad_() for k, v in p.items()}
    leaves = list(gp.values())
    eager = [t.detach().clone() for t in torch.autograd.grad(_kernels(gx, gp), leaves)]
    state = torch.tensor([SEED, 0], device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(_kernels(gx, gp, state), leaves)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = torch.autograd.grad(_kernels(gx, gp, state), leaves)
    for _ in range(2):
        for t in out:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, eager):
            assert torch.equal(a, b)
    state[1] += 10000  # another mask on the next replay
    graph.replay()
    torch.cuda.synchronize()
    assert not torch.equal(out[1], eager[1])
