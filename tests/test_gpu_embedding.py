"""The scaled embedding (tb_embedding_fwd) and its gradient by sorted tokens (tb_embedding_grad)
against the fp64 oracle. Bounds: the forward rounds the scale and one product in fp32; an id's
gradient takes one fp32 rounding per token, two more for the scale; then one rounding to the type
(two with an existing gradient: the fp32 sum with it)."""

import pytest
import torch

from helpers import assert_rounded
from oracle import rowops

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
TYPES = [torch.float16, torch.bfloat16, torch.float32]


def _ids(n, vocab, seed, kind="zipf"):
    g = torch.Generator().manual_seed(seed)
    if kind == "same":
        return torch.full((n,), vocab - 1)
    if kind == "uniform":
        return torch.randint(0, vocab, (n,), generator=g)
    return ((vocab + 1.0) ** torch.rand(n, generator=g, dtype=torch.float64) - 1).long() \
        .clamp(0, vocab - 1)


def _table(vocab, hidden, dtype, seed):
    return torch.randn(vocab, hidden, generator=torch.Generator().manual_seed(seed)).to(dtype)


def _check_grad(got, ids, dy, vocab, scale, pad=None, old=None, what=""):
    want, mag, count = rowops.embedding_grad(ids.cpu(), dy.cpu(), vocab, scale, pad)
    extra = mag * (count[:, None] + 4) * U
    if old is not None:
        want = want + old.double()
        extra = extra + (mag + old.double().abs()) * U
    assert_rounded(got, want, extra, what)
    if old is not None:
        assert torch.equal(got.cpu()[count == 0], old[count == 0])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,vocab,hidden,kind", [
    (1, 1, 1, "same"), (1, 17, 8, "uniform"), (7, 5, 65, "uniform"), (621, 1000, 136, "zipf"),
    (2048, 31, 24, "uniform"), (2049, 300, 8, "zipf"), (5000, 40, 40, "same"),
    (9001, 2000, 72, "zipf"), (300, 11, 4104, "zipf"), (40, 70000, 33, "uniform"),
    (256, 90, 40, "zipf"), (257, 90, 40, "zipf"), (255, 3, 2112, "same"), (64, 64, 16, "uniform"),
    (65, 500, 9, "zipf"), (33, 40, 264, "uniform")])
def test_forward_and_gradient(n, vocab, hidden, kind, dtype):
    from testt_b200.embed import embedding

    ids = _ids(n, vocab, n, kind)
    table = _table(vocab, hidden, dtype, 1).to(DEV).requires_grad_()
    scale = hidden ** 0.5
    for out in {dtype, torch.float32}:
        y = embedding(ids.to(DEV), table, scale=scale, out_dtype=out)
        want = rowops.embedding(ids, table.detach().cpu(), scale)
        assert y.dtype == out
        assert_rounded(y, want, want.abs() * 2 * U, "y")
        dy = torch.randn(n, hidden, generator=torch.Generator().manual_seed(2)).to(out).to(DEV)
        (dw,) = torch.autograd.grad(y, table, dy)
        assert dw.dtype == dtype and dw.is_contiguous()
        _check_grad(dw, ids, dy, vocab, scale, what="dw")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,hidden", [(1301, 4104), (701, 1001)])
def test_forward_of_many_vectors(n, hidden, dtype):
    """More vectors (of 8 columns, of one) than the persistent forward has threads for at a time
    (606,208 on 148 SMs), with ids outside."""
    from testt_b200 import _lib
    from testt_b200.embed import embedding

    vocab = 2000
    ids = _ids(n, vocab, n, "uniform")
    ids[::50], ids[7::300] = vocab, -5
    outside = int(((ids < 0) | (ids >= vocab)).sum())
    table = _table(vocab, hidden, dtype, 14)
    want = rowops.embedding(ids, table, 3.3)
    for out, index in ((dtype, torch.int64), (torch.float32, torch.int32)):
        before = _lib.load().tb_embed_invalid_ids()
        y = embedding(ids.to(DEV, index), table.to(DEV), scale=3.3, out_dtype=out)
        assert_rounded(y, want, want.abs() * 2 * U, "y")
        assert _lib.load().tb_embed_invalid_ids() == before + outside


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [2 ** 21 - 2, 2 ** 21 - 1, 2 ** 22 + 77])
@pytest.mark.parametrize("hidden", [8, 3])
def test_large_vocabularies(vocab, hidden, dtype):
    """Vocabularies around the one from which on a tile's keys take 64 bits: ids that differ in
    their high bits alone, repeated, the last ones, the padding id and ids outside."""
    from testt_b200.embed import embedding_grad

    n = 4500
    ids = _ids(n, vocab, 15)
    ids[::3] = torch.randint(0, 7, (n // 3,), generator=torch.Generator().manual_seed(16)) \
        + 2 ** 20 * torch.arange(n // 3).remainder(2)
    ids[1::9], ids[2::90], ids[4::90] = vocab - 1, vocab, -1
    ids[5::30] = vocab - 2 - torch.arange(n // 30).remainder(3)
    dy = torch.randn(n, hidden, generator=torch.Generator().manual_seed(17)).to(dtype)
    got = embedding_grad(ids.to(DEV), dy.to(DEV), vocab, scale=1.5, padding_idx=2)
    _check_grad(got, ids, dy, vocab, 1.5, pad=2)


@pytest.mark.parametrize("n,kind", [(33000, "zipf"), (33000, "same"), (70001, "uniform")])
def test_many_tiles_merge(n, kind):
    """More tokens than one merge takes (16 tiles of 2048), ids over many chunks."""
    from testt_b200.embed import embedding_grad

    ids = _ids(n, 777, 3, kind)
    dy = torch.randn(n, 16, generator=torch.Generator().manual_seed(4)).half()
    dw = embedding_grad(ids.to(DEV), dy.to(DEV), 777, dtype=torch.float32)
    _check_grad(dw, ids, dy, 777, 1.0)
    again = embedding_grad(ids.to(DEV).int(), dy.to(DEV), 777, dtype=torch.float32)
    assert torch.equal(dw, again)


@pytest.mark.parametrize("dtype", TYPES)
def test_padding_and_ids_outside(dtype):
    from testt_b200 import _lib
    from testt_b200.embed import embedding, embedding_grad

    ids = torch.tensor([[3, 9, -1, 3], [10, 2 ** 40, 3, 0]], device=DEV)
    table = _table(10, 48, dtype, 5).to(DEV).requires_grad_()
    before = _lib.load().tb_embed_invalid_ids()
    y = embedding(ids, table, scale=2.0, padding_idx=3)
    assert y.shape == (2, 4, 48)
    torch.cuda.synchronize()
    assert _lib.load().tb_embed_invalid_ids() == before + 3
    assert torch.all(y[0, 2] == 0) and torch.all(y[1, :2] == 0)
    assert torch.equal(y[0, 0].float(), (table[3].float() * 2).to(dtype).float())
    dy = torch.randn(2, 4, 48, device=DEV).to(dtype)
    (dw,) = torch.autograd.grad(y, table, dy)
    _check_grad(dw, ids, dy, 10, 2.0, pad=3)
    assert torch.all(dw[3] == 0)
    assert torch.equal(dw, embedding_grad(ids, dy, 10, scale=2.0, padding_idx=3))


@pytest.mark.parametrize("dtype,dy_dtype", [(torch.float16, torch.float16),
                                            (torch.float32, torch.bfloat16),
                                            (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("hidden", [40, 37])
def test_added_to_an_existing_gradient(dtype, dy_dtype, hidden):
    from testt_b200.embed import embedding_grad

    ids = _ids(3000, 900, 6)
    ids[::7] = 13
    dy = torch.randn(3000, hidden, generator=torch.Generator().manual_seed(7)).to(dy_dtype)
    old = _table(900, hidden, dtype, 8)
    out = old.clone().to(DEV)
    assert embedding_grad(ids.to(DEV), dy.to(DEV), 900, scale=0.5, out=out) is out
    _check_grad(out, ids, dy, 900, 0.5, old=old)
    assert out._version > 0
    empty = embedding_grad(ids[:0].to(DEV), dy[:0].to(DEV), 900, out=out)
    assert empty is out


def test_views_and_unaligned_tables():
    from testt_b200.embed import embedding

    ids = _ids(50, 30, 9).to(DEV)
    wide = _table(30, 200, torch.float16, 10).to(DEV)
    for a, b in ((0, 64), (8, 72), (3, 67), (5, 6)):
        w = wide[:, a:b]
        assert torch.equal(embedding(ids, w), w[ids])
    assert torch.equal(embedding(ids, wide.t()[:30]), wide.t()[:30][ids])
    strided = ids.repeat(2)[::2]
    assert torch.equal(embedding(strided, wide), wide[strided])
    flat = torch.randn(30 * 64 + 1, device=DEV).half()[1:].view(30, 64)
    assert torch.equal(embedding(ids.int(), flat), flat[ids])


def test_unaligned_gradient_rows_keep_their_neighbours():
    """The zero fill and the sums of a gradient that starts off a 16-byte boundary end inside it."""
    from testt_b200 import _lib

    for vocab, hidden in ((3, 5), (7, 8), (40, 33)):
        for lead in (0, 1, 3):
            buf = torch.full((lead + vocab * hidden + 9,), 7.0, dtype=torch.float16, device=DEV)
            dw = buf[lead:lead + vocab * hidden]
            ids = torch.tensor([1, 2, 1], device=DEV)
            dy = torch.ones(3, hidden, dtype=torch.float16, device=DEV)
            want = torch.zeros(vocab, hidden)
            want[1], want[2] = 2, 1
            for copies in (1, 100):  # one launch; the sort, the sums and the join
                n, dw_of = 3 * copies, dw.fill_(9.0)
                nbytes = _lib.load().tb_embedding_grad_workspace(n, hidden)
                ws = torch.empty(nbytes, dtype=torch.uint8, device=DEV) if nbytes else None
                many, rows = ids.repeat(copies), dy.repeat(copies, 1)
                _lib.call("tb_embedding_grad", _lib.ptr(many), 1, _lib.ptr(rows), 0,
                          _lib.ptr(dw_of), 0, 1.0, -1, 0, n, hidden, vocab, _lib.ptr(ws), nbytes,
                          _lib.stream_of(dw))
                assert torch.equal(dw.cpu().float().view(vocab, hidden), want * copies)
                assert torch.all(buf[:lead] == 7) and torch.all(buf[lead + vocab * hidden:] == 7)


def test_no_tokens_and_same_bits():
    from testt_b200.embed import embedding

    table = _table(60, 24, torch.float16, 11).to(DEV).requires_grad_()
    y = embedding(torch.empty((0,), dtype=torch.int64, device=DEV), table)
    assert y.shape == (0, 24)
    (dw,) = torch.autograd.grad(y.sum(), table)
    assert torch.all(dw == 0)
    ids = _ids(4000, 60, 12).to(DEV)
    dy = torch.randn(4000, 24, device=DEV).half()
    runs = [torch.autograd.grad(embedding(ids, table), table, dy)[0] for _ in range(3)]
    assert torch.equal(runs[0], runs[1]) and torch.equal(runs[0], runs[2])


def test_two_captured_graphs_and_a_stream():
    """Two graphs of the gradient, replayed by turns, and an eager call between them on another
    stream: each keeps its own workspace."""
    from testt_b200.embed import embedding

    table = _table(5000, 64, torch.float16, 13).to(DEV).requires_grad_()
    sets = [(_ids(n, 5000, n).to(DEV), torch.randn(n, 64, device=DEV).half()) for n in (900, 4500)]

    def step(ids, dy):
        return torch.autograd.grad(embedding(ids, table, scale=3.0), table, dy)[0]

    want = [step(*s) for s in sets]
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
            o.detach().fill_(1)
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                eager = step(*sets[0])
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(o, w) and torch.equal(eager, want[0])


def test_refusals():
    from testt_b200.embed import embedding, embedding_grad

    ids = torch.tensor([0, 1], device=DEV)
    w = torch.ones(4, 8, device=DEV).half()
    dy = torch.ones(2, 8, device=DEV).half()
    for bad in (lambda: embedding(ids.float(), w), lambda: embedding(ids, w.double()),
                lambda: embedding(ids, w[0]), lambda: embedding(ids, w, out_dtype=torch.bfloat16),
                lambda: embedding(ids, w, padding_idx=4), lambda: embedding(ids, w[:0]),
                lambda: embedding_grad(ids, dy[:1], 4), lambda: embedding_grad(ids, dy, 0),
                lambda: embedding_grad(ids, dy, 4, out=w[:, :4]),
                lambda: embedding_grad(ids, dy, 4, out=w.bfloat16()),
                lambda: embedding_grad(ids, dy, 4, padding_idx=-2),
                lambda: embedding_grad(ids, dy, 4, dtype=torch.bfloat16)):
        with pytest.raises((TypeError, ValueError)):
            bad()
    with pytest.raises(RuntimeError, match="CUDA tensors"):
        embedding(ids.cpu(), w)


def test_offsets_past_32_bits():
    """A table and a gradient of more than 2^31 elements: rows at their far end."""
    from testt_b200.embed import embedding

    if torch.cuda.mem_get_info()[0] < 24e9:
        pytest.skip("needs 24 GB of device memory")
    vocab, hidden = 140001, 16384
    table = torch.zeros(vocab, hidden, dtype=torch.float16, device=DEV).requires_grad_()
    rows = torch.randn(3, hidden, device=DEV).half()
    ids = torch.tensor([vocab - 1, 131072, 5, vocab - 1], device=DEV)
    with torch.no_grad():
        table[ids[:3]] = rows
    y = embedding(ids, table, scale=2.0)
    assert torch.equal(y, (rows * 2)[[0, 1, 2, 0]])
    for copies in (1, 100):  # one launch; the sort, the sums and the join
        many = ids.repeat(copies)
        dy = torch.ones(many.numel(), hidden, dtype=torch.float16, device=DEV)
        (dw,) = torch.autograd.grad(embedding(many, table, scale=2.0), table, dy)
        sums = dw.sum(1, dtype=torch.float32)
        want = torch.zeros(vocab, device=DEV)
        want.index_add_(0, ids, torch.full((4,), 2.0 * copies * hidden, device=DEV))
        assert torch.equal(sums, want)
        del dw
