"""Operators that go past their autograd function where nothing is differentiated are recorded all the same where a call is traced.

The launches are replaced by something that a trace sees as little of as of a launch: memory is allocated by PyTorch, its values come from elsewhere.  (A trace without the function holds the
allocations alone and returns whatever they find.)"""
import ctypes

import pytest
import torch

from easyllm_amd import functional as F, kernels as K


def unseen(value):
    out = torch.empty_like(value)
    ctypes.memmove(out.data_ptr(), value.numpy().ctypes.data, value.numel() * value.element_size())
    return out


@pytest.fixture
def host(monkeypatch):
    monkeypatch.setattr(K, "rotary", lambda q, k, inv_freq, ids=None, interleaved=False, scale=1.0, backward=False: (unseen(q.detach() * 2), None if k is None else unseen(k.detach() * 3)))
    monkeypatch.setattr(K, "gated_mlp_fwd", lambda act, x, gate, up, down, keep=False: (unseen((x @ gate.t() * (x @ up.t()) @ down.t()).detach()), None))
    monkeypatch.setattr(K, "gated_fwd", lambda act, x, gate, up, keep=False: (unseen((x @ gate.t() * (x @ up.t())).detach()), None))


CALLS = {"RotaryEmbedFunction": (lambda q, k: F.rotary_embed(q, k, torch.ones(4)), (3, 1, 2, 8), (3, 1, 1, 8)),
         "RotaryEmbedFunction alone": (lambda q: F.rotary_embed(q, None, torch.ones(4))[0], (3, 1, 2, 8)),
         "GatedMLPFunction": (F.gated_mlp, (5, 8), (16, 8), (16, 8), (8, 16)),
         "GatedLinearFunction": (F.gated_linear, (5, 8), (16, 8), (16, 8))}


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("name", CALLS)
def test_an_evaluation_is_recorded(host, name):
    call, *shapes = CALLS[name]
    values = lambda seed: [torch.randn(s, generator=torch.Generator().manual_seed(seed + i)) for i, s in enumerate(shapes)]  # noqa: E731
    with torch.no_grad():
        traced = torch.jit.trace(call, values(1), check_trace=False)
        assert "^" + name.split()[0] in str(traced.graph)
        for seed in (2, 3):
            got, want = traced(*values(seed)), call(*values(seed))
            got, want = ((t,) if torch.is_tensor(t) else t for t in (got, want))
            assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_an_evaluation_that_is_not_traced_makes_no_node(host, monkeypatch):
    monkeypatch.setattr(F.RotaryEmbedFunction, "apply", None)
    monkeypatch.setattr(F.GatedMLPFunction, "apply", None)
    with torch.no_grad():
        F.rotary_embed(torch.ones(3, 1, 2, 8), None, torch.ones(4))
        F.gated_mlp(torch.ones(5, 8), torch.ones(16, 8), torch.ones(16, 8), torch.ones(8, 16))
