"""Forward-mode differentiation: the row operators have no jvp, and a call on tensors with a tangent
raises instead of returning an output without one. The launches are left out: no GPU needed."""

import pytest
import torch
from torch.autograd import forward_ad

from testt_b200 import _lib
from testt_b200.dropout import dropout
from testt_b200.embed import embedding, embedding_grad
from testt_b200.logprobs import token_logprobs
from testt_b200.norm_rope import norm_rope_tokens

IDS = torch.tensor([1, 0, 3])
TABLE = torch.ones(2, 4)


def _heads(qkv, weight=None):
    return norm_rope_tokens(qkv, None, None, weight, None, 1e-6, TABLE, TABLE, IDS, 2, 2, 2, 1, 4)


CALLS = {
    "embedding": (lambda x: embedding(IDS, x), (5, 8)),
    "embedding_grad": (lambda x: embedding_grad(IDS, x, 5), (3, 8)),
    "embedding_grad out": (lambda x: embedding_grad(IDS, torch.ones(3, 8), 5, out=x), (5, 8)),
    "norm_rope": (_heads, (3, 16)),
    "norm_rope weight": (lambda w: _heads(torch.ones(3, 16), w), (4,)),
    "token_logprobs": (lambda x: token_logprobs(x, IDS, top_k=2), (3, 8)),
    "token_logprobs of a batch": (lambda x: token_logprobs(x, IDS.view(1, 3)), (1, 3, 8)),
    "dropout": (lambda x: dropout(x, 0.5, 1), (3, 8)),
    "dropout residual": (lambda r: dropout(torch.ones(3, 8), 0.5, 1, residual=r), (3, 8)),
}


@pytest.fixture
def launches(monkeypatch):
    names = []
    monkeypatch.setattr(_lib, "require_cuda", lambda *t, what: None)
    monkeypatch.setattr(_lib, "call_on", lambda t, name, *args: names.append(name))
    monkeypatch.setattr(_lib, "workspace_bytes", lambda t, name, *args: 0)
    return names


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("grad", [True, False])
def test_a_tangent_is_refused(name, grad, launches):
    call, shape = CALLS[name]
    x = torch.ones(shape)
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        with pytest.raises(NotImplementedError):
            call(forward_ad.make_dual(x, torch.ones(shape)))
        launches.clear()
        call(x)  # without a tangent, inside a level
        assert len(launches) == 1
    launches.clear()
    call(x)
    assert len(launches) == 1
