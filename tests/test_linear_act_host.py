"""What a product with an epilogue keeps for its backward pass (CPU, the kernels replaced)."""
import pytest
import torch

from easyllm_amd import functional as F


@pytest.fixture
def kept(monkeypatch):
    """whether each call asked the kernel for the activation's input"""
    asked = []

    def product(x, w, bias, act, residual, want_pre=False):
        asked.append(bool(want_pre))
        y = x @ w.t()
        return y, y.clone() if want_pre else None
    monkeypatch.setattr(F.K, "linear_act_fwd", product)
    return asked


@pytest.mark.parametrize("leaf", ["x", "w", "b", "r"])
def test_the_activations_input_is_kept_for_a_backward_pass_only(kept, leaf):
    t = {"x": torch.ones(4, 8), "w": torch.ones(16, 8), "b": torch.ones(16), "r": torch.ones(4, 16)}
    t[leaf].requires_grad_(True)
    F.linear_act(t["x"], t["w"], t["b"], "gelu", t["r"])
    F.linear_act(t["x"], t["w"], t["b"], None, t["r"])
    with torch.no_grad():  # an evaluation, whose parameters need gradients all the same
        F.linear_act(t["x"], t["w"], t["b"], "gelu", t["r"])
    assert kept == [leaf != "r", False, False]
