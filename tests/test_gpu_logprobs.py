"""Token log-probabilities (tb_token_logprobs_fwd / _bwd) against the fp64 oracle; top ids exactly.

Bounds (U = 2^-24, n the vocabulary): S is a sum of n positive terms in fp32, at most n / 256 + 64
of them one after the other, each term off by the rounding of its exponent d (up to 2 U |d|,
weighted by the term: at most log2 n on average) and by the 2 ulp of 2^x: S is off by
(n / 256 + 64 + 2 log2 n + 8) U relative, log S by as much absolutely."""

import math

import numpy as np
import pytest
import torch

from helpers import assert_rounded
from oracle import rowops

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
TYPES = [torch.float16, torch.bfloat16, torch.float32]


def _sum_tol(vocab):
    return (vocab / 256 + 64 + 2 * math.log2(vocab + 1) + 8) * U


def _logits(rows, vocab, dtype, seed, std=3.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, vocab, generator=g) * std).to(dtype)


def _check(logits, ids, k=0, temp=1.0, which=(True, True, True), gpu=None, seed=1):
    from testt_b200.logprobs import token_logprobs

    rows, vocab = logits.shape
    g = torch.Generator().manual_seed(seed)
    grads = [torch.randn(rows, generator=g), torch.randn(rows, generator=g),
             torch.randn(rows, k, generator=g)]
    use = [w and (i < 2 or k > 0) for i, w in enumerate(which)]
    z = (logits.to(DEV) if gpu is None else gpu).requires_grad_()
    o = token_logprobs(z, ids.to(DEV), top_k=k, temperature=temp)
    w = rowops.token_logprobs(logits, ids, k, temp, [t if u else None for t, u in zip(grads, use)])
    tol = _sum_tol(vocab)
    assert torch.equal(o.top_ids.cpu(), w["top_ids"])
    fin = lambda t: torch.nan_to_num(t.abs(), nan=0.0, posinf=0.0, neginf=0.0)  # noqa: E731
    # lp = t c ln2 - log S: the difference, c and the products round (6 U of it)
    assert_rounded(o.logprob, w["lp"], tol + 6 * U * (fin(w["lp"]) + math.log(vocab)), "lp")
    assert_rounded(o.top_logprobs, w["top_lp"], tol + 6 * U * (fin(w["top_lp"]) + math.log(vocab)),
                   "top")
    # H = log S - U / (S T): U's terms round like S's, and log S - H is at most log n
    h_tol = (2 * tol + 8 * U) * (1 + math.log(vocab))
    assert_rounded(o.entropy, w["ent"], h_tol, "entropy")
    if any(use):
        outs = [o.logprob, o.entropy, o.top_logprobs]
        (dz,) = torch.autograd.grad([t for t, u in zip(outs, use) if u], z,
                                    [t.to(DEV) for t, u in zip(grads, use) if u])
        assert dz.shape == z.shape and dz.dtype == z.dtype
        # p = 2^d: off by tol, 2 ulp and the rounding of d (4 U |d|); the entropy in it by h_tol
        p = w["p"]
        d = torch.where(p > 0, p.clamp_min(1e-300).log2().abs(), torch.zeros_like(p))
        ge = grads[1].double().abs()[:, None] if use[1] else 0.0
        extra = w["dz_mag"] * (tol + (4 * d + 16 + k) * U) + p * ge * h_tol / temp
        extra = extra + 2.0 ** -126 / temp * (1 + ge)  # results of 2^x below the normal numbers are 0
        assert_rounded(dz, w["dz"], extra, "dz")
        return o, dz
    return o, None


def _ids(rows, vocab, seed=2):
    ids = torch.randint(0, vocab, (rows,), generator=torch.Generator().manual_seed(seed))
    if rows > 2:
        ids[rows // 2] = -100
    return ids


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab,k,temp", [
    (1, 1, 0, 1.0), (1, 1, 1, 1.0), (3, 2, 2, 0.5), (5, 7, 7, 1.0), (4, 40, 32, 1.3),
    (3, 333, 5, 0.7), (9, 4096, 20, 1.0), (2, 50021, 32, 1.0), (700, 1003, 3, 2.0),
    (1, 151936, 20, 1.0), (7, 151936, 0, 1.0), (600, 2056, 1, 1.0), (5, 9000, 2, 1e-3)])
def test_against_oracle(rows, vocab, k, temp, dtype):
    _check(_logits(rows, vocab, dtype, rows + vocab), _ids(rows, vocab), k, temp)


@pytest.mark.parametrize("which", [(True, False, False), (False, True, False), (False, False, True),
                                   (True, False, True)])
def test_each_gradient_alone(which):
    _check(_logits(5, 3001, torch.float32, 3), _ids(5, 3001), 6, 0.9, which)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [4, 700])
def test_ties_go_to_the_lowest_index(dtype, rows):
    """Few distinct values, all equal, and the largest ones next to each other (all in the vectors
    of a few threads)."""
    v = 3 * 2048 + 5
    g = torch.Generator().manual_seed(4)
    few = torch.randint(-2, 3, (rows, v), generator=g).to(dtype)
    few[few == 0] = 0.0
    few[1] = torch.where(torch.arange(v) % 2 == 0, 0.0, -0.0).to(dtype)  # +0 and -0 are equal
    _check(few, _ids(rows, v), 32)
    _check(torch.full((rows, v), 1.5).to(dtype), _ids(rows, v), 20)
    run = torch.zeros(rows, v).to(dtype)
    run[:, 4000:4040] = torch.arange(40).to(dtype) / 8
    _check(run, _ids(rows, v), 32)
    _check(torch.arange(v).expand(rows, v).div(2048).to(dtype), _ids(rows, v), 32)
    _check(torch.arange(v).flip(0).expand(rows, v).div(2048).to(dtype), _ids(rows, v), 32)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [6, 700])
def test_masks(dtype, rows):
    """-inf columns, a row of -inf only, a row with one finite logit, the type's lowest value as a
    mask (everywhere it is a row of equal logits), large offsets."""
    v = 5003
    z = _logits(rows, v, dtype, 5)
    z[:, 4000:] = -math.inf
    z[0] = -math.inf
    z[1] = -math.inf
    z[1, 77] = 2.0
    z[2] = torch.finfo(dtype).min
    z[3, ::2] = torch.finfo(dtype).min
    z[4] = (z[4].float() + 40000.0).to(dtype)
    z[5, :-3] = -math.inf
    z[5, -3:] = torch.tensor([1.0, 2.0, 1.0]).to(dtype)
    ids = _ids(rows, v)
    ids[1], ids[2], ids[3], ids[5] = 77, 4999, 11, 5001
    o, dz = _check(z, ids, 3)
    assert o.logprob[0] == -math.inf and o.entropy[0] == 0 and torch.all(dz[0] == 0)
    assert o.top_ids[0].tolist() == [0, 1, 2]
    assert o.logprob[1] == 0 and o.entropy[1] == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("temp", [1.0, 1e-4, 1e4])
@pytest.mark.parametrize("rows", [5, 700])
def test_lowest_values_beside_minus_infinities(dtype, temp, rows):
    """Rows whose largest logit is the type's lowest value or lies far below the usual ones, with
    -inf columns beside it: those have probability 0 and no gradient, the finite ones their own
    differences. Columns 0 to 2 and the last lie outside the whole 16-byte vectors of some rows."""
    v = 5003
    low = torch.finfo(dtype).min
    z = torch.full((rows, v), -math.inf)
    z[:, :3] = low
    z[1::5, 100:4000] = low
    z[2::5, v - 1] = low
    z[3::5, 50:3000] = low / 2
    z[3::5, 60:70] = low / 4
    z[4::5, 7:v:2] = -3e4 if dtype == torch.float16 else -2e20
    ids = _ids(rows, v)
    ids[:2] = torch.tensor([1, 4500])  # a finite logit, a -inf one
    ids[3::5] = 65
    z = z.to(dtype)
    o, dz = _check(z, ids, 3, temp)
    zero = torch.isneginf(z)
    zero[torch.arange(rows)[ids >= 0], ids[ids >= 0]] = False
    assert torch.all(dz.cpu()[zero] == 0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_large_gradients_of_masked_rows(dtype):
    """Masked columns add nothing to a gradient of any size: powers of two times the incoming
    gradients give that times the outgoing one, bit for bit (no probability here is near the
    smallest normal number)."""
    from testt_b200.logprobs import token_logprobs

    z = _logits(5, 2000, dtype, 12)
    z[:, 1500:] = -math.inf
    z[2, ::3] = torch.finfo(dtype).min
    z = z.to(DEV).requires_grad_()
    o = token_logprobs(z, _ids(5, 1500).to(DEV), temperature=0.7)
    gs = torch.randn(2, 5, device=DEV)
    (small,) = torch.autograd.grad(o[:2], z, list(gs), retain_graph=True)
    for e in (20, 66, 100):
        (big,) = torch.autograd.grad(o[:2], z, list(gs * 2.0 ** e), retain_graph=True)
        assert torch.equal(big.double(), small.double() * 2.0 ** e)


@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_nan_and_infinity_stay_in_their_row(bad):
    from testt_b200.logprobs import token_logprobs

    for rows in (3, 700):
        z = _logits(rows, 3000, torch.float16, 6)
        z[1, 1500] = bad
        zz = z.to(DEV).requires_grad_()
        o = token_logprobs(zz, _ids(rows, 3000).to(DEV).clamp_min(0), top_k=4)
        (dz,) = torch.autograd.grad(o.logprob.sum(), zz)
        for t in (o.logprob, o.entropy, o.top_logprobs, dz):
            assert torch.isnan(t[1]).any() and not torch.isnan(t[0]).any()
            assert not torch.isnan(t[2:]).any()
        assert torch.isnan(o.logprob[1]) and torch.isnan(o.entropy[1])
        assert int(o.top_ids.min()) >= 0 and int(o.top_ids.max()) < 3000
    all_nan = torch.full((2, 100), math.nan, device=DEV)
    o = token_logprobs(all_nan, torch.tensor([1, 2], device=DEV), top_k=5)
    assert torch.isnan(o.top_logprobs).all() and int(o.top_ids.max()) < 100


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("temp", [1.0, 1e-4, 1e4])
@pytest.mark.parametrize("rows", [3, 700])
def test_spreads_past_fp32(dtype, temp, rows):
    """Logits whose differences, or whose differences over the temperature, are no fp32 numbers:
    those far below the largest have probability 0 and leave no NaN."""
    from testt_b200.logprobs import token_logprobs

    vocab, k = 2500, 3
    logits = _logits(rows, vocab, dtype, 8, std=1e37)
    logits[:, 7], logits[:, 2049], logits[:, 1300] = -3e38, 3e38, 1e38
    logits[1] = _logits(1, vocab, dtype, 9, std=1e12)[0]
    ids = torch.tensor([7, 2049, 1300]).repeat(rows)[:rows]
    z = logits.to(DEV).requires_grad_()
    o = token_logprobs(z, ids.to(DEV), top_k=k, temperature=temp)
    g = torch.Generator().manual_seed(3)
    grads = [torch.randn(rows, generator=g), torch.randn(rows, generator=g),
             torch.randn(rows, k, generator=g)]
    w = rowops.token_logprobs(logits, ids, k, temp, grads)
    as_fp32 = lambda t: t.float().double()  # noqa: E731  (-inf past its range)
    tol = _sum_tol(vocab)
    fin = lambda t: torch.nan_to_num(t.abs(), posinf=0.0)  # noqa: E731
    # the difference, 1 / T, the products and the sum with log S round: 6 U of it
    assert_rounded(o.logprob, as_fp32(w["lp"]), tol + 6 * U * fin(as_fp32(w["lp"])), "lp")
    assert_rounded(o.top_logprobs, as_fp32(w["top_lp"]), tol + 6 * U * fin(as_fp32(w["top_lp"])),
                   "top")
    assert torch.equal(o.top_ids.cpu(), w["top_ids"])
    assert_rounded(o.entropy, w["ent"], (2 * tol + 8 * U) * (1 + math.log(vocab)), "entropy")
    (dz,) = torch.autograd.grad([o.logprob, o.entropy, o.top_logprobs], z, [t.to(DEV) for t in grads])
    # the spreads leave one logit of probability 1 or gaps of at least 1e5 U below it (1e12 / 1e4)
    ge = grads[1].double().abs()[:, None]
    d = torch.where(w["p"] > 0, w["p"].clamp_min(1e-300).log2().abs(), torch.zeros_like(w["p"]))
    extra = w["dz_mag"] * (tol + (4 * d + 16 + k) * U) + \
        w["p"] * ge * (2 * tol + 8 * U) * (1 + math.log(vocab)) / temp + 2.0 ** -126 / temp * (1 + ge)
    assert_rounded(dz, w["dz"], extra, "dz")


@pytest.mark.parametrize("rows", [2, 700])
def test_nan_among_minus_infinities(rows):
    from testt_b200.logprobs import token_logprobs

    z = torch.full((rows, 900), -math.inf)
    z[0, 333] = math.nan
    o = token_logprobs(z.to(DEV), torch.zeros(rows, dtype=torch.long, device=DEV), top_k=2)
    for t in (o.logprob, o.top_logprobs[:, 0]):
        assert torch.isnan(t[0]) and torch.isneginf(t[1:]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("a,b", [(0, 1001), (3, 1004), (8, 1009), (5, 9)])
def test_rows_of_a_wider_buffer(dtype, a, b):
    """Views whose rows start anywhere modulo 16 bytes; what lies around them is NaN."""
    z = _logits(9, b - a, dtype, 7)
    wide = torch.full((9, 1013), math.nan, device=DEV, dtype=dtype)
    wide[:, a:b] = z.to(DEV)
    _check(z, _ids(9, b - a), min(4, b - a), gpu=wide[:, a:b])


def test_last_positions_and_batches():
    """Logits of [batch, seq, vocab] taken at the last position (a row stride of seq * vocab), and
    whole, with ids of the same leading shape."""
    from testt_b200.logprobs import token_logprobs

    z = _logits(12, 777, torch.bfloat16, 8).view(3, 4, 777)
    zz = z.to(DEV).requires_grad_()
    ids = torch.randint(0, 777, (3, 4))
    last = token_logprobs(zz[:, -1], ids[:, -1].to(DEV), top_k=2)
    whole = token_logprobs(zz, ids.to(DEV).int(), top_k=2)
    assert whole.logprob.shape == (3, 4) and whole.top_ids.shape == (3, 4, 2)
    assert torch.equal(whole.top_ids[:, -1], last.top_ids)
    w = rowops.token_logprobs(z.reshape(12, 777), ids.reshape(-1), 2)
    assert_rounded(whole.logprob, w["lp"], _sum_tol(777) + 100 * U)
    (g,) = torch.autograd.grad(last.logprob.sum(), zz)
    assert torch.all(g[:, :-1] == 0) and torch.all(g[:, -1].float().abs().sum(-1) > 0)
    turned = zz.detach().reshape(12, 777).t().contiguous().t()
    again = token_logprobs(turned, ids.to(DEV).reshape(-1), top_k=2)
    assert torch.equal(again.top_ids, whole.top_ids.reshape(12, 2))
    one = token_logprobs(zz[0, 0], ids[0, 0].to(DEV), top_k=1)
    assert one.logprob.shape == () and one.top_ids.shape == (1,)


def test_offsets_past_32_bits():
    """Rows whose element offsets pass 2^31 (a row stride of 2^31 / 3 + elements)."""
    from testt_b200.logprobs import token_logprobs

    if torch.cuda.mem_get_info()[0] < 24e9:
        pytest.skip("needs 24 GB of device memory")
    rows, vocab, ld = 5, 4001, 2 ** 30 + 8
    flat = torch.empty((rows - 1) * ld + vocab, dtype=torch.float16, device=DEV)
    z = flat.as_strided((rows, vocab), (ld, 1))
    src = _logits(rows, vocab, torch.float16, 9)
    z.copy_(src)
    ids = _ids(rows, vocab)
    o = token_logprobs(z, ids.to(DEV), top_k=4)
    w = rowops.token_logprobs(src, ids, 4)
    assert torch.equal(o.top_ids.cpu(), w["top_ids"])
    assert_rounded(o.logprob, w["lp"], _sum_tol(vocab) + 120 * U)


def test_same_bits_twice_streams_and_graphs():
    from testt_b200.logprobs import token_logprobs

    sets = []
    for rows, vocab in ((2, 151936), (640, 5001)):
        z = _logits(rows, vocab, torch.float16, rows).to(DEV).requires_grad_()
        sets.append((z, _ids(rows, vocab).to(DEV), torch.randn(rows, device=DEV)))

    def step(z, ids, g):
        o = token_logprobs(z, ids, top_k=8)
        # detached: PyTorch cannot capture a backward while an eager graph of its leaves lives
        return [t.detach() for t in (*o, *torch.autograd.grad([o.logprob, o.entropy], z, [g, g]))]

    want = [step(*s) for s in sets]
    for s, w in zip(sets, want):
        assert all(torch.equal(a, b) for a, b in zip(step(*s), w))
    side = torch.cuda.Stream()
    graphs, outs = [], []
    for s in sets:
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(*s)
        torch.cuda.current_stream().wait_stream(side)
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(step(*s))
    for _ in range(2):
        for g, o, w in zip(graphs, outs, want):
            for t in o:
                t.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(o, w))


def test_gradient_against_differences():
    """fp32, central differences of the kernels' own outputs along a random direction (fourth
    order, step 2^-5: the forward's error over the step, and the fifth derivative's term)."""
    from testt_b200.logprobs import token_logprobs

    z = _logits(4, 500, torch.float32, 10).to(DEV).requires_grad_()
    ids = _ids(4, 500).to(DEV)
    dirs = torch.randn(4, 500, generator=torch.Generator().manual_seed(11)).to(DEV)
    gs = [torch.randn(4, device=DEV).double(), torch.randn(4, device=DEV).double(),
          torch.randn(4, 3, device=DEV).double()]

    def value(step):
        # the top ids of the middle: two logits that pass each other would be a kink
        zs = z.detach() + step * dirs
        at = token_logprobs(zs, ids)
        top = torch.stack([token_logprobs(zs, o.top_ids[:, j]).logprob for j in range(3)], 1)
        return sum(float((a.double() * b).sum())
                   for a, b in zip((at.logprob, at.entropy, top), gs))

    o = token_logprobs(z, ids, top_k=3)
    (dz,) = torch.autograd.grad(list(o[:3]), z, [g.float() for g in gs])
    h = 2.0 ** -5
    slope = (8 * (value(h) - value(-h)) - (value(2 * h) - value(-2 * h))) / (12 * h)
    weight = sum(float(g.abs().sum()) for g in gs)
    noise = 2 * weight * (2 * _sum_tol(500) + 40 * U) * (1 + math.log(500)) / h
    assert abs(slope - float((dz.double() * dirs.double()).sum())) <= noise + weight * 400 * h ** 4


def test_refusals_and_empty():
    from testt_b200.logprobs import token_logprobs

    z = torch.randn(3, 20, device=DEV)
    ids = torch.tensor([1, 2, 3], device=DEV)
    for bad in (lambda: token_logprobs(z.double(), ids), lambda: token_logprobs(z, ids[:2]),
                lambda: token_logprobs(z, ids.float()), lambda: token_logprobs(z[:, :0], ids),
                lambda: token_logprobs(z, ids, top_k=21), lambda: token_logprobs(z, ids, top_k=-1),
                lambda: token_logprobs(z.repeat(1, 9), ids, top_k=33),
                lambda: token_logprobs(z, ids, temperature=0.0),
                lambda: token_logprobs(z, ids, temperature=math.nan)):
        with pytest.raises((TypeError, ValueError)):
            bad()
    with pytest.raises(RuntimeError, match="CUDA tensors"):
        token_logprobs(z, ids.cpu())
    e = z[:0].requires_grad_()
    o = token_logprobs(e, ids[:0], top_k=4)
    assert o.logprob.shape == (0,) and o.top_ids.shape == (0, 4)
    (g,) = torch.autograd.grad(o.logprob.sum(), e)
    assert g.shape == (0, 20)
    same = token_logprobs(z[:1].expand(3, 20), ids)
    assert np.allclose(same.entropy.cpu(), same.entropy[0].cpu())
