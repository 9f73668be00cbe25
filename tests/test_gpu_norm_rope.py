"""Head norms with the rotation (tb_norm_rope_fwd / _bwd) against the fp64 oracle. Bounds: a sum
of d fp32 products is off by at most d half steps of its absolute terms, a value takes under 16
more roundings, a weight gradient one per token and head on top; then one rounding to the type."""

import pytest
import torch

from helpers import assert_rounded
from oracle import rowops

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
TYPES = [torch.float16, torch.bfloat16, torch.float32]


def _case(n, nh, nkv, d, rot, seq, dtype, lora=None, weights=None, seed=0, outside=False):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    ang = r(seq, max(rot // 2, 1))[:, :rot // 2] * 3
    pos = torch.randint(0, 2 * seq, (n,), generator=g)
    if outside and n > 2:
        pos[0], pos[n // 2] = -1, 2 * seq
    return dict(qkv=r(n, (nh + 2 * nkv) * d).to(dtype),
                lora_q=None if lora is None else (r(n, nh * d) * 0.3).to(lora),
                lora_v=None if lora is None else (r(n, nkv * d) * 0.3).to(lora),
                q_weight=None if weights is None else (1 + 0.3 * r(d)).to(weights),
                k_weight=None if weights is None else (1 + 0.3 * r(d)).to(weights), eps=1e-6,
                cos=torch.cat([ang.cos(), ang.cos()], 1), sin=torch.cat([ang.sin(), ang.sin()], 1),
                pos_idx=pos, batch=2, seq=seq, n_heads=nh, n_kv=nkv, head_dim=d), \
        [r(n, h, d).to(dtype) for h in (nh, nkv, nkv)]


def _gpu(c):
    return {k: v.to(DEV) if torch.is_tensor(v) else v for k, v in c.items()}


def _oracle(c, w0, grads):
    return rowops.norm_rope(c["qkv"], c["lora_q"], c["lora_v"], c["q_weight"], c["k_weight"],
                            c["eps"], c["cos"], c["sin"], c["pos_idx"], c["batch"], c["seq"],
                            c["n_heads"], c["n_kv"], c["head_dim"], w0, grads)


def _check(c, grads, w0=0.0, gpu=None):
    from testt_b200.norm_rope import norm_rope_tokens

    g = _gpu(c) if gpu is None else gpu
    names = [k for k in ("qkv", "lora_q", "lora_v", "q_weight", "k_weight") if g[k] is not None]
    for k in names:
        g[k].requires_grad_()
    q, k, v = norm_rope_tokens(**g, weight_offset=w0)
    got = torch.autograd.grad((q, k, v), [g[x] for x in names], [t.to(DEV) for t in grads])
    got = dict(zip(names, got))
    want = _oracle(c, w0, grads)
    n, nh, nkv, d = c["qkv"].shape[0], c["n_heads"], c["n_kv"], c["head_dim"]
    tol = (d + 16) * U
    assert_rounded(q, want["q"], want["q_mag"] * tol, "q")
    assert_rounded(k, want["k"], want["k_mag"] * tol, "k")
    assert_rounded(v, want["v"], want["v"].abs() * U + (0.5 * U if c["lora_v"] is not None else 0),
                   "v")
    assert_rounded(got["qkv"], want["dqkv"], want["dqkv_mag"] * (2 * d + 32) * U, "dqkv")
    if "q_weight" in got:
        for name, heads in (("q", nh), ("k", nkv)):
            assert_rounded(got[name + "_weight"], want[f"d{name}w"],
                           want[f"d{name}w_mag"] * (n * heads + d + 32) * U, name + "_weight")
    if "lora_q" in got:
        lt = c["lora_q"].dtype
        assert torch.equal(got["lora_q"], got["qkv"][:, :nh * d].to(lt))
        assert torch.equal(got["lora_v"], got["qkv"][:, (nh + nkv) * d:].to(lt))
    return q, k, v, got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,nh,nkv,d,rot,seq", [
    (1, 1, 1, 16, 16, 1), (5, 12, 2, 128, 128, 40), (37, 4, 4, 64, 32, 50), (300, 32, 8, 128, 64, 9),
    (19, 6, 1, 80, 80, 33), (11, 3, 3, 96, 48, 20), (9, 24, 8, 256, 256, 30), (3, 2, 1, 512, 128, 5),
    (7, 4, 2, 80, 40, 11), (7, 2, 2, 20, 6, 11), (6, 3, 1, 2, 2, 4), (5, 2, 1, 64, 0, 4),
    (2, 70, 1, 128, 128, 3)])
def test_against_oracle(n, nh, nkv, d, rot, seq, dtype):
    _check(*_case(n, nh, nkv, d, rot, seq, dtype, weights=dtype, outside=True))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lora,weights", [(torch.float16, torch.float32), (torch.float32, None),
                                          (torch.bfloat16, torch.bfloat16), (None, None)])
@pytest.mark.parametrize("d", [64, 20])
def test_lora_weight_types_and_offset(dtype, lora, weights, d):
    _check(*_case(23, 6, 2, d, d, 12, dtype, lora, weights, seed=3), w0=1.0)


@pytest.mark.parametrize("width,start", [(1100, 0), (1100, 8), (1100, 3)])
def test_rows_of_a_wider_buffer(width, start):
    c, grads = _case(21, 4, 2, 128, 128, 7, torch.float16, weights=torch.float16, seed=4)
    wide = torch.full((21, width), float("nan"), dtype=torch.float16, device=DEV)
    wide = torch.cat([wide, wide[:, :start]], 1)
    wide[:, start:start + 1024] = c["qkv"].to(DEV)
    g = _gpu(c)
    g["qkv"] = wide[:, start:start + 1024]
    _check(c, grads, gpu=g)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,rot", [(64, 64), (80, 40), (20, 20), (20, 6)])
def test_several_tokens_a_warp(d, rot, dtype):
    """As many tokens as make every warp of every kernel walk on from one to the next (at most 3,552
    and 18,944 warps forward, 2,368 and 1,184 backward on 148 SMs), on tables whose halves differ,
    with LoRA rows, weights and positions outside."""
    n, nh, nkv = 9001, 2, 1
    c, grads = _case(n, nh, nkv, d, rot, 700, dtype, torch.float32 if d == 64 else dtype, dtype,
                     seed=17, outside=True)
    c["pos_idx"][5::97] = 2 * 700
    g = torch.Generator().manual_seed(18)
    c["cos"], c["sin"] = torch.randn(2, 700, rot, generator=g)
    got = _check(c, grads, w0=0.5)[3]
    want = _oracle(c, 0.5, grads)
    # a weight's sum: at most 8 tokens of 2 heads in a lane, 64 lanes' sums, 37 CTAs', 32 groups'
    for name in "qk":
        assert_rounded(got[name + "_weight"], want[f"d{name}w"],
                       want[f"d{name}w_mag"] * (16 + 64 + 37 + 32 + d + 32) * U, name + "_weight")


def test_no_key_value_heads_and_missing_gradients():
    from testt_b200.norm_rope import norm_rope_tokens

    c, grads = _case(13, 4, 0, 64, 64, 8, torch.bfloat16, weights=torch.bfloat16, seed=5)
    g = _gpu(c)
    g["qkv"].requires_grad_()
    g["k_weight"].requires_grad_()
    q, k, v = norm_rope_tokens(**g)
    assert k.shape == (13, 0, 64) and v.shape == (13, 0, 64)
    dqkv, dkw = torch.autograd.grad(q, [g["qkv"], g["k_weight"]], grads[0].to(DEV))
    want = _oracle(c, 0.0, (grads[0], None, None))
    assert_rounded(dqkv, want["dqkv"], want["dqkv_mag"] * 160 * U)
    assert torch.all(dkw == 0)


@pytest.mark.parametrize("n,nkv", [(1, 2), (5, 0), (1, 0)])
def test_gradients_share_no_memory(n, nkv):
    """The LoRA rows' gradients are qkv's columns: where those are whole, autograd keeps what it is
    given, and a later change of one leaf's gradient must not reach another's."""
    from testt_b200.norm_rope import norm_rope_tokens

    c, grads = _case(n, 4, nkv, 64, 64, 8, torch.float32, torch.float32, torch.float32, seed=15)
    g = _gpu(c)
    leaves = [g[x].requires_grad_() for x in ("qkv", "lora_q", "lora_v")]
    out = norm_rope_tokens(**g)
    torch.autograd.backward(out, [t.to(DEV) for t in grads])
    want = [t.grad.clone() for t in leaves]
    for i, t in enumerate(leaves):
        t.grad.add_(1.0)
        want[i] += 1.0
        for u, v in zip(leaves, want):
            assert torch.equal(u.grad, v)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d", [64, 20])
def test_small_heads_without_eps(dtype, d):
    """Heads of 1e-14 with eps 0: 1 / rms is 1e14, whose cube is no fp32 number."""
    c, grads = _case(9, 4, 2, d, d, 8, dtype, weights=dtype, seed=16)
    c["qkv"] = (c["qkv"].float() * 1e-14).to(dtype)
    c["eps"] = 0.0
    _check(c, grads)


def test_only_values_used():
    from testt_b200.norm_rope import norm_rope_tokens

    c, grads = _case(13, 4, 2, 64, 64, 8, torch.float16, weights=torch.float16, seed=6)
    g = _gpu(c)
    g["qkv"].requires_grad_()
    _, _, v = norm_rope_tokens(**g)
    (dqkv,) = torch.autograd.grad(v, g["qkv"], grads[2].to(DEV))
    assert torch.all(dqkv[:, :6 * 64] == 0)
    inside = (c["pos_idx"] >= 0)[:, None, None]
    assert torch.equal(dqkv[:, 6 * 64:].reshape(13, 2, 64).cpu(),
                       torch.where(inside, grads[2], torch.zeros((), dtype=torch.float16)))


def test_zero_rows_and_extremes():
    """A head of zeros stays zero (r = 1 / sqrt(eps)); large fp16 values do not overflow the fp32
    sum; a NaN stays in its head."""
    from testt_b200.norm_rope import norm_rope_tokens

    c, _ = _case(4, 2, 1, 64, 64, 8, torch.float16, seed=7)
    c["qkv"][0] = 0
    c["qkv"][1] = 60000.0
    c["qkv"][2, 3] = float("nan")
    q, k, v = norm_rope_tokens(**_gpu(c))
    want = _oracle(c, 0.0, None)
    assert_rounded(q[:2], want["q"][:2], want["q_mag"][:2] * 80 * U)
    assert torch.all(q[0] == 0) and torch.all(k[0] == 0)
    assert torch.isnan(q[2, 0]).all() and not torch.isnan(q[2, 1]).any()


def test_same_bits_twice_and_in_a_graph():
    c, grads = _case(700, 12, 2, 128, 128, 500, torch.float16, torch.float16, torch.float32, seed=8)
    a = _check(c, grads)
    b = _check(c, grads)
    for x, y in zip((*a[:3], *a[3].values()), (*b[:3], *b[3].values())):
        assert torch.equal(x, y)
    from testt_b200.norm_rope import norm_rope_tokens

    g, dg = _gpu(c), [t.to(DEV) for t in grads]
    leaves = [g[k].requires_grad_() for k in ("qkv", "q_weight", "k_weight")]

    def step():
        return torch.autograd.grad(norm_rope_tokens(**g), leaves, dg)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(2):
        for t in out:
            t.detach().zero_()
        graph.replay()
        torch.cuda.synchronize()
        for t, k in zip(out, ("qkv", "q_weight", "k_weight")):
            assert torch.equal(t, a[3][k])


def test_gradient_against_differences():
    """The kernels' gradient in fp32 against central differences of the kernels' own forward: a
    step of 2^-6 in a random direction leaves a cubic term and the forward's rounding."""
    from testt_b200.norm_rope import norm_rope_tokens

    c, grads = _case(6, 3, 1, 32, 16, 8, torch.float32, weights=torch.float32, seed=9)
    g = _gpu(c)
    dg = [t.to(DEV).double() for t in grads]
    direction = torch.randn(c["qkv"].shape, generator=torch.Generator().manual_seed(1)).to(DEV)

    def value(step):
        h = dict(g, qkv=g["qkv"].detach() + step * direction)
        return sum(float((o.double() * d).sum()) for o, d in zip(norm_rope_tokens(**h), dg))

    g["qkv"].requires_grad_()
    (dx,) = torch.autograd.grad(norm_rope_tokens(**g), g["qkv"], [d.float() for d in dg])
    h = 2.0 ** -6
    slope = (8 * (value(h) - value(-h)) - (value(2 * h) - value(-2 * h))) / (12 * h)
    got = float((dx.double() * direction.double()).sum())
    terms = sum(float((o.abs().double() * d.abs()).sum())
                for o, d in zip(norm_rope_tokens(**{**g, "qkv": g["qkv"].detach()}), dg))
    assert abs(slope - got) <= terms * (60 * U / h + 32 * h ** 4)


def test_refusals_and_empty():
    from testt_b200.norm_rope import norm_rope_tokens

    c, _ = _case(5, 4, 2, 64, 64, 8, torch.float16, weights=torch.float16, seed=2)
    g = _gpu(c)
    for change in (dict(qkv=g["qkv"].double()), dict(qkv=g["qkv"][:, :-1]), dict(n_heads=5),
                   dict(head_dim=63), dict(seq=9), dict(pos_idx=g["pos_idx"][:4]),
                   dict(pos_idx=g["pos_idx"].float()), dict(q_weight=g["q_weight"][:32]),
                   dict(k_weight=g["k_weight"].double()), dict(lora_q=g["qkv"]),
                   dict(cos=g["cos"][:, :62]), dict(sin=g["sin"][:7])):
        with pytest.raises((TypeError, ValueError)):
            norm_rope_tokens(**{**g, **change})
    with pytest.raises(RuntimeError, match="CUDA tensors"):
        norm_rope_tokens(**{**g, "cos": c["cos"]})
    e = {**g, "qkv": g["qkv"][:0].requires_grad_(), "pos_idx": g["pos_idx"][:0],
         "q_weight": g["q_weight"].requires_grad_()}
    q, k, v = norm_rope_tokens(**e)
    assert q.shape == (0, 4, 64)
    dqkv, dqw = torch.autograd.grad(q.sum() + v.sum(), [e["qkv"], e["q_weight"]])
    assert dqkv.shape == e["qkv"].shape and torch.all(dqw == 0)


def test_offsets_past_32_bits():
    """More than 2^31 elements of q|k|v, outputs and gradient: the last tokens equal the same
    tokens alone."""
    from testt_b200.norm_rope import norm_rope_tokens

    if torch.cuda.mem_get_info()[0] < 40e9:
        pytest.skip("needs 40 GB of device memory")
    rows, nh, nkv, d = 280001, 48, 8, 128
    g = torch.Generator().manual_seed(3)
    tail = torch.randn(5, (nh + 2 * nkv) * d, generator=g).half().to(DEV)
    cos, sin = torch.randn(2, 16, d, generator=g).to(DEV)
    w = torch.rand(d, generator=g).half().to(DEV)
    qkv = torch.zeros(rows, (nh + 2 * nkv) * d, dtype=torch.float16, device=DEV)
    qkv[-5:] = tail
    pos = torch.arange(rows, device=DEV) % 16
    grads = [torch.randn(5, h, d, generator=g).half().to(DEV) for h in (nh, nkv, nkv)]

    def run(x, at, weight):
        x, weight = x.requires_grad_(), weight.clone().requires_grad_()
        outs = norm_rope_tokens(x, None, None, weight, None, 1e-6, cos, sin, at, 1, 16, nh, nkv, d)
        full = [torch.zeros_like(o) for o in outs]
        for f, t in zip(full, grads):
            f[-5:] = t
        return outs, torch.autograd.grad(outs, [x, weight], full)

    outs, (dx, dw) = run(qkv, pos, w)
    alone, (dx5, dw5) = run(tail, pos[-5:], w)
    for a, b in zip(outs, alone):
        assert torch.equal(a[-5:], b) and not a[:-5].any()
    assert torch.equal(dx[-5:], dx5) and not dx[:-5].any()
    assert torch.allclose(dw.float(), dw5.float(), rtol=2.0 ** -9)
