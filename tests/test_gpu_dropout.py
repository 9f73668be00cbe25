"""Dropout from the counter-based generator (tb_dropout) against the generator restated in numpy:
the mask exactly, the values to one rounding (of x * scale in fp32, then of the output type)."""

import numpy as np
import pytest
import torch

from helpers import assert_rounded
from oracle import rowops

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24  # fp32 half step
TYPES = [torch.float16, torch.bfloat16, torch.float32]


def _x(shape, dtype, seed):
    x = torch.randn(shape, generator=torch.Generator().manual_seed(seed))
    x = torch.where(x.abs() < 1e-3, torch.full_like(x, 1e-3), x)  # no zeros: the mask shows
    return x.to(dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1,), (7,), (3, 5), (8, 64), (257, 1536), (2, 3, 333)])
@pytest.mark.parametrize("seed,offset,p", [(0, 0, 0.1), (2 ** 63 + 11, 2 ** 32 - 3, 0.5),
                                           (-1, 2 ** 62, 0.95)])
def test_values_and_gradient(dtype, shape, seed, offset, p):
    from testt_b200.dropout import dropout

    x = _x(shape, dtype, 1).to(DEV).requires_grad_()
    dy = _x(shape, dtype, 2).to(DEV)
    y = dropout(x, p, seed, offset)
    y.backward(dy)
    want, keep = rowops.dropout(x.detach().cpu(), p, seed % 2 ** 64, offset)
    assert torch.equal(y.detach().cpu() != 0, keep)
    # scale = 1/(1-p) is rounded to fp32, and so is the product
    assert_rounded(y, want, want.abs() * 2 * U, "y")
    gx, _ = rowops.dropout(dy.cpu(), p, seed % 2 ** 64, offset)
    assert_rounded(x.grad, gx, gx.abs() * 2 * U, "dx")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("own", [True, False])
def test_residual(dtype, own):
    from testt_b200.dropout import dropout

    res_type = dtype if own else torch.float32
    x = _x((33, 130), dtype, 3).to(DEV).requires_grad_()
    res = _x((33, 130), res_type, 4).to(DEV).requires_grad_()
    dy = _x((33, 130), res_type, 5).to(DEV)
    y = dropout(x, 0.25, 9, 4, residual=res)
    assert y.dtype == res_type
    y.backward(dy)
    want, keep = rowops.dropout(x.detach().cpu(), 0.25, 9, 4, res.detach().cpu())
    mag = res.detach().cpu().double().abs() + x.detach().cpu().double().abs() * 2
    assert_rounded(y, want, mag * 3 * U, "y")
    assert torch.equal(res.grad, dy)
    gx, _ = rowops.dropout(dy.cpu(), 0.25, 9, 4)
    assert_rounded(x.grad, gx, gx.abs() * 2 * U, "dx")


@pytest.mark.parametrize("p", [0.0, 1.0])
def test_all_and_nothing(p):
    from testt_b200.dropout import dropout

    x = _x((5, 77), torch.float16, 6).to(DEV)
    x[0, 0], x[1, 1] = float("inf"), float("nan")
    y = dropout(x, p, 3)
    if p == 0.0:
        assert torch.equal(y.isnan(), x.isnan())
        assert torch.equal(y.nan_to_num(), x.nan_to_num())
    else:
        assert torch.all(y == 0)
        assert torch.equal(dropout(x, p, 3, residual=x[2:3].expand(5, 77)),
                           x[2:3].expand(5, 77))


def test_known_words_and_layout_independence():
    """Counter 0 under key 0 gives the generator's published words; the mask does not depend on
    type, alignment or how a tensor is strided, and consecutive offsets continue it."""
    from testt_b200.dropout import counters, dropout

    words = [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]
    one = torch.ones(4, device=DEV)
    for i, w in enumerate(words):
        p_keep, p_drop = w / 2 ** 32, (w + 1) / 2 ** 32
        assert dropout(one, p_keep, 0)[i] != 0 and dropout(one, p_drop, 0)[i] == 0
    n = 4096
    base = dropout(torch.ones(n, device=DEV), 0.3, 5, 7) != 0
    assert torch.equal(base, dropout(torch.ones(n, device=DEV).half(), 0.3, 5, 7) != 0)
    odd = torch.ones(n + 1, device=DEV).half()[1:]  # 2-byte aligned only
    assert torch.equal(base, dropout(odd, 0.3, 5, 7) != 0)
    turned = torch.ones(64, 64, device=DEV).t()
    assert torch.equal(base, dropout(turned, 0.3, 5, 7).reshape(-1) != 0)
    rest = dropout(torch.ones(n - 400, device=DEV), 0.3, 5, 7 + counters(400)) != 0
    assert torch.equal(base[400:], rest)
    assert abs(float(base.float().mean()) - 0.7) < 4 * (0.21 / n) ** 0.5


def test_state_tensor_in_a_captured_graph():
    """With the seed and offset in device memory a replay draws what they then hold; the backward
    uses what its forward used though the state has moved on."""
    from testt_b200.dropout import dropout

    x = torch.ones(1000, device=DEV, requires_grad=True)
    state = torch.tensor([11, 0], device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        dropout(x, 0.5, state)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = dropout(x, 0.5, state, 3)
        state[1] += 250
        (dx,) = torch.autograd.grad(y, x, torch.ones_like(y))
    for i in range(3):
        graph.replay()
        torch.cuda.synchronize()
        keep = rowops.keep_mask((1000,), 0.5, 11, 3 + 250 * i)
        assert torch.equal(y.detach().cpu() != 0, keep) and torch.equal(dx.cpu() != 0, keep)


def test_another_stream_and_broadcast_gradient():
    from testt_b200.dropout import dropout

    x = torch.randn(300, 40, device=DEV).requires_grad_()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        y = dropout(x, 0.5, 1)
        (g,) = torch.autograd.grad(y.sum(), x)  # an expanded gradient
    stream.synchronize()
    keep = rowops.keep_mask((300, 40), 0.5, 1, 0)
    assert torch.equal(g.cpu(), keep.float() * 2)
    row = torch.randn(1, 40, device=DEV).requires_grad_()
    (gr,) = torch.autograd.grad(dropout(row.expand(300, 40), 0.5, 1).sum(), row)
    assert torch.equal(gr.cpu()[0], keep.float().sum(0) * 2)


def test_refusals():
    from testt_b200.dropout import dropout

    x = torch.ones(4, device=DEV)
    for bad in (lambda: dropout(x.double(), 0.1, 0), lambda: dropout(x, 1.5, 0),
                lambda: dropout(x, float("nan"), 0), lambda: dropout(x, 0.1, 0, -1),
                lambda: dropout(x, 0.1, 0, residual=x[:3]),
                lambda: dropout(x, 0.1, 0, residual=x.half()),
                lambda: dropout(x, 0.1, torch.zeros(2, dtype=torch.int32, device=DEV)),
                lambda: dropout(x, 0.1, torch.zeros(2, dtype=torch.int64))):
        with pytest.raises((TypeError, ValueError)):
            bad()
    with pytest.raises(RuntimeError, match="CUDA tensors"):
        dropout(x.cpu(), 0.1, 0)
    assert dropout(x[:0], 0.1, 0).numel() == 0
    assert np.array_equal(dropout(x[:0].reshape(0, 4), 0.1, 0).shape, (0, 4))


def test_offsets_past_32_bits():
    """More than 2^32 elements: the last ones draw the words of their own numbers."""
    from testt_b200.dropout import dropout

    if torch.cuda.mem_get_info()[0] < 40e9:
        pytest.skip("needs 40 GB of device memory")
    n = 2 ** 32 + 1003
    x = torch.ones(n, dtype=torch.float16, device=DEV)
    y = dropout(x, 0.5, 21, 5)
    first = n - 1003
    words = rowops.philox_words(21, 5 + first // 4, 1003)
    assert np.array_equal((y[first:] != 0).cpu().numpy(), words >= np.uint64(2 ** 31))
    assert torch.equal(y[:1000].cpu() != 0, rowops.keep_mask((1000,), 0.5, 21, 5))
