"""The row operators' C entry points refuse bad arguments before any CUDA call (no GPU needed), and
their oracle agrees with autograd on its own formulas."""

import ctypes

import numpy as np
import pytest
import torch

from oracle import rowops

TB_EINVAL, TB_EALIGN = -1, -2
P = ctypes.c_void_p


@pytest.fixture(scope="module")
def lib():
    from testt_b200 import _lib

    return _lib.load()


def _refuses(lib, name, args, code, text):
    assert getattr(lib, name)(*args) == code, name
    assert text in lib.tb_last_error(), lib.tb_last_error()


def test_dropout(lib):
    ok = [P(256), 0, None, P(512), 0, 8, 5, 1.0, 0, 0, None, None, None]

    def bad(i, v, code, text):
        _refuses(lib, "tb_dropout", ok[:i] + [v] + ok[i + 1:], code, text)

    bad(1, 3, TB_EINVAL, b"types")
    bad(4, 1, TB_EINVAL, b"types")      # fp16 -> bf16
    bad(5, -1, TB_EINVAL, b"n -1")
    bad(6, 2 ** 32 + 1, TB_EINVAL, b"threshold")
    bad(0, None, TB_EINVAL, b"required")
    bad(3, P(513), TB_EALIGN, b"aligned")
    bad(10, P(12), TB_EALIGN, b"aligned")
    assert lib.tb_dropout(None, 0, None, None, 0, 0, 0, 1.0, 0, 0, None, None, None) == 0


def test_norm_rope(lib):
    ok = [P(256), 0, 1024, None, None, 0, None, None, 0, 0.0, 1e-6, P(256), P(256), 64, P(256),
          P(256), P(256), P(256), 4, 1, 8, 4, 2, 128, None]

    def bad(i, v, code, text):
        _refuses(lib, "tb_norm_rope_fwd", ok[:i] + [v] + ok[i + 1:], code, text)

    bad(1, 7, TB_EINVAL, b"types")
    bad(2, 1023, TB_EINVAL, b"row stride")
    bad(13, 130, TB_EINVAL, b"dims")    # rot > head_dim
    bad(13, 63, TB_EINVAL, b"dims")
    bad(20, 0, TB_EINVAL, b"dims")      # seq
    bad(23, 127, TB_EINVAL, b"dims")
    bad(23, 8192, TB_EINVAL, b"head_dim")
    bad(19, 2 ** 31, TB_EINVAL, b"too many")
    bad(0, None, TB_EINVAL, b"required")
    bad(14, P(260), TB_EALIGN, b"aligned")
    bwd = [P(256)] * 4 + [0, 1024, None, 0, P(256), P(256), 0, 0.0, 1e-6, P(256), P(256), 64,
                          P(256), P(256), P(256), P(256), P(256), 0, 4, 1, 8, 4, 2, 128, None]
    _refuses(lib, "tb_norm_rope_bwd", bwd, TB_EINVAL, b"workspace of 0")
    assert lib.tb_norm_rope_bwd_workspace(4, 4, 2, 128) >= 2 * 128 * 4
    assert lib.tb_norm_rope_bwd_workspace(0, 4, 2, 128) == 0


def test_embedding(lib):
    fwd = [P(256), 1, P(256), 0, 64, P(256), 2, 1.0, 4, 64, 100, None]
    for i, v, code, text in ((6, 1, TB_EINVAL, b"types"), (4, 63, TB_EINVAL, b"row stride"),
                             (8, -1, TB_EINVAL, b"n -1"), (10, 2 ** 31, TB_EINVAL, b"vocab"),
                             (2, None, TB_EINVAL, b"required"), (0, P(257), TB_EALIGN, b"aligned")):
        _refuses(lib, "tb_embedding_fwd", fwd[:i] + [v] + fwd[i + 1:], code, text)
    nbytes = lib.tb_embedding_grad_workspace(300, 64)
    assert nbytes >= 2 * 300 * 8 and lib.tb_embedding_grad_workspace(0, 64) == 0
    assert lib.tb_embedding_grad_workspace(256, 64) == 0  # one launch
    assert lib.tb_embedding_grad_workspace(257, 64) > 0
    grad = [P(256), 1, P(256), 0, P(256), 0, 1.0, -1, 0, 300, 64, 100, P(256), nbytes, None]
    for i, v, code, text in ((3, 1, TB_EINVAL, b"types"), (13, nbytes - 1, TB_EINVAL, b"workspace"),
                             (12, None, TB_EINVAL, b"workspace"), (12, P(8), TB_EALIGN, b"aligned"),
                             (4, None, TB_EINVAL, b"required")):
        _refuses(lib, "tb_embedding_grad", grad[:i] + [v] + grad[i + 1:], code, text)


def test_embedding_token_limit(lib):
    """More tokens than a launch's grid can merge are refused before any launch."""
    n = 0x7fff0001
    for name, args in (("tb_embedding_fwd", [P(256), 1, P(256), 0, 64, P(256), 2, 1.0, n, 64, 100, None]),
                       ("tb_embedding_grad", [P(256), 1, P(256), 0, P(256), 0, 1.0, -1, 0, n, 64, 100,
                                              P(256), 2 ** 62, None])):
        _refuses(lib, name, args, TB_EINVAL, b"n 2147418113")


def test_token_logprobs_gradient_is_not_the_logits(lib):
    """The columns with a one-hot term are read again after the row is written."""
    args = [P(256), 0, 1000, P(256), 1, 1.0, 0, None, P(256), P(256), None, None, P(256), 1000, 4,
            1000, None]
    _refuses(lib, "tb_token_logprobs_bwd", args, TB_EINVAL, b"the logits themselves")


def test_token_logprobs(lib):
    need = lib.tb_token_logprobs_workspace(4, 100000, 0, 4)  # few long rows are split
    assert need > 0 and lib.tb_token_logprobs_workspace(0, 100000, 0, 4) == 0
    fwd = [P(256), 0, 100000, P(256), 1, 1.0, 4, P(256), P(256), P(256), P(256), P(256), 4, 100000,
           P(256), need, None]
    for i, v, code, text in ((1, 5, TB_EINVAL, b"type"), (2, 99999, TB_EINVAL, b"row stride"),
                             (5, 0.0, TB_EINVAL, b"temperature"),
                             (5, float("nan"), TB_EINVAL, b"temperature"),
                             (6, 33, TB_EINVAL, b"top"), (13, 3, TB_EINVAL, b"top"),
                             (12, 2 ** 22, TB_EINVAL, b"rows"), (9, None, TB_EINVAL, b"missing"),
                             (15, need - 1, TB_EINVAL, b"workspace"), (0, P(257), TB_EALIGN, b"aligned")):
        _refuses(lib, "tb_token_logprobs_fwd", fwd[:i] + [v] + fwd[i + 1:], code, text)
    bwd = [P(256), 0, 1000, P(256), 1, 1.0, 0, None, P(256), P(256), None, None, P(256), 1000, 4,
           1000, None]
    _refuses(lib, "tb_token_logprobs_bwd", bwd[:12] + [P(258)] + bwd[13:], TB_EALIGN, b"modulo 16")
    _refuses(lib, "tb_token_logprobs_bwd", bwd[:13] + [1001] + bwd[14:], TB_EALIGN, b"modulo 16")
    _refuses(lib, "tb_token_logprobs_bwd", bwd[:13] + [999] + bwd[14:], TB_EINVAL, b"stride")


def test_gradient_buffer_lies_as_the_logits_do():
    """Every row of the log-probabilities' gradient starts modulo 16 bytes where its logits row
    does, with at most 7 spare columns a row."""
    from testt_b200.logprobs import _grad_like

    for dtype in (torch.float16, torch.float32):
        base = torch.empty(40 * 64, dtype=dtype)
        for start, ld, vocab in ((0, 64, 64), (3, 61, 57), (5, 64, 9), (1, 1000, 7), (2, 33, 33)):
            rows = (base.numel() - start - vocab) // ld + 1
            z = base.as_strided((rows, vocab), (ld, 1), start)
            g = _grad_like(z)
            assert g.shape == z.shape and g.stride(1) == 1
            for r in range(rows):
                assert (g[r].data_ptr() - z[r].data_ptr()) % 16 == 0
            assert rows == 1 or vocab <= g.stride(0) <= vocab + 7


def test_oracle_gradients_against_autograd():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(5, 37, generator=g, dtype=torch.float64, requires_grad=True)
    ids = torch.tensor([3, -100, 36, 0, 7])
    o = torch.log_softmax(x / 0.7, 1)
    lp = o.gather(1, ids.clamp(0, 36)[:, None])[:, 0] * (ids >= 0)
    outs = [lp, -(o.exp() * o).sum(1), o.topk(4, 1).values]
    gs = [torch.randn(t.shape, generator=g, dtype=torch.float64) for t in outs]
    (gx,) = torch.autograd.grad(outs, x, gs)
    r = rowops.token_logprobs(x.detach(), ids, 4, 0.7, gs)
    assert torch.allclose(r["dz"], gx, rtol=0, atol=1e-13)
    assert [hex(int(v)) for v in rowops.philox_words(0, 0, 4)] == \
        ["0x6627e8d5", "0xe169c58d", "0xbc57ac4c", "0x9b00dbd8"]
    dw, mag, count = rowops.embedding_grad(torch.tensor([1, 1, 5, 9]), torch.ones(4, 2), 6, 2.0)
    assert np.array_equal(dw[:, 0].numpy(), [0, 4, 0, 0, 0, 2]) and count.tolist() == [0, 2, 0, 0, 0, 1]
