"""Which rows the final norm and the LM head are given (host logic, on CPU tensors)."""
import types

import pytest
import torch

from plaquant_b200 import forward_pass


@pytest.fixture
def model(monkeypatch):
    m = object.__new__(forward_pass.ResQForwardB200)
    m.cfg, m.layers, m.kv = forward_pass.LlamaConfig(rms_eps=1e-6), [], []
    m.ctx, m.scatter, m.peer = types.SimpleNamespace(size=2, rank=0), None, types.SimpleNamespace(rows=64)
    g = torch.Generator().manual_seed(0)
    m.embed = torch.randn(50, 16, generator=g).to(torch.bfloat16)
    m.final_norm, m.lm_head = torch.ones(16, dtype=torch.bfloat16), torch.randn(50, 16, generator=g).to(torch.bfloat16)
    m._rope_rows = lambda pos0, t: None
    m.given, finish, logits = [], m._finish, m._logits
    m._finish = lambda h, delta: h * 2 if delta is forward_pass._IN_PEER_BUFFER else finish(h, delta)

    def watched(h):
        m.given.append(tuple(h.shape))
        return logits(h)
    m._logits = watched
    return m


@pytest.mark.parametrize("b,t", [(1, 1), (3, 5), (2, 1)])
@pytest.mark.parametrize("where", ["peer", "tensor"])
def test_last_position_only(model, b, t, where):
    """The last MLP output in the peer buffers or at hand: the head sees one row per sequence, and gives what it gives those
    rows of a whole pass."""
    ids = torch.arange(b * t).view(b, t) % 50
    model._run_layers = lambda h, *a, **kw: (h, forward_pass._IN_PEER_BUFFER if where == "peer" else h)
    last = model.forward(ids)
    assert model.given == [(b, 16)] and last.shape == (b, 50)
    assert torch.equal(last, model._logits(model.embed[ids[:, -1]] * 2))
    model.given.clear()
    every = model.forward(ids, all_positions=True)
    assert model.given == [(b, t, 16)] and every.shape == (b, t, 50)
    assert torch.allclose(every[:, -1], last, rtol=2.0 ** -7, atol=2.0 ** -6)


def test_a_decode_step_of_no_sequence(model):
    model._run_layers = lambda h, *a, **kw: (h, h)
    assert model.forward(torch.zeros(0, 3, dtype=torch.int64)).shape == (0, 50)
