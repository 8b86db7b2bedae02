"""What a gated block kept has to be memory of the GPU that reads it."""
import pytest
import torch

from easyllm_amd import kernels as K


def test_kept_values_that_lie_elsewhere_are_refused(monkeypatch):
    kept = torch.zeros(K._kept_bytes(4, 16), dtype=torch.uint8)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0)
    with pytest.raises(ValueError, match="not on the current GPU"):
        K._kept(kept, 4, 16)


@pytest.mark.gpu
def test_backward_calls_refuse_them():
    bf16 = lambda *shape: torch.zeros(*shape, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    kept = torch.zeros(K._kept_bytes(4, 16), dtype=torch.uint8)
    with pytest.raises(ValueError, match="not on the current GPU"):
        K.gate_bwd("silu", bf16(4, 16), kept)
    with pytest.raises(ValueError, match="not on the current GPU"):
        K.gated_mlp_bwd("silu", bf16(4, 8), bf16(4, 8), bf16(16, 8), bf16(16, 8), bf16(8, 16), kept, True, (None, None, None))
