"""States of the 8-bit step whose tensors do not all lie in one place."""
import pytest
import torch

from easyllm_amd import kernels as K


def state(master_device, device="cpu", n=600):
    g = torch.Generator().manual_seed(1)
    codes = lambda k, low=0, high=256: torch.randint(low, high, (k,), generator=g, dtype=torch.uint8).to(device)  # noqa: E731
    return {"master": torch.zeros(20, n // 20, device=master_device), "number": 0, "exp_avg": codes(n), "exp_avg_sq": codes(n), "exp_avg_scale": codes((n + 255) // 256, 100, 130),
            "exp_avg_sq_scale": codes((n + 255) // 256, 100, 130)}


def test_values_lie_where_the_codes_do(monkeypatch):
    """The kernel writes to the codes' device: results anywhere else would be an address that it may not write to."""
    seen = []
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: -1)  # (what tensors in host memory say, too)
    monkeypatch.setattr(K, "_stream", lambda: 0)
    monkeypatch.setattr(K._lib, "call", lambda name, count, tensors, m, v, stream: seen.append((name, m[0], v[0])))
    (m, v), = K.moments8_list([state("meta")])
    assert m.device.type == v.device.type == "cpu" and m.shape == v.shape == (20, 30) and m.dtype is v.dtype is torch.bfloat16
    assert seen == [("ezl_moments8_list", m.data_ptr(), v.data_ptr())]


@pytest.mark.gpu
def test_values_of_a_state_whose_master_weights_lie_on_the_host():
    from easyllm_amd import optimizer
    there, here = state("cpu", "cuda"), state("cuda", "cuda")
    for a, b in zip(*(optimizer.moments_8bit([s])[0] for s in (there, here))):
        assert a.is_cuda and a.shape == (20, 30) and torch.equal(a, b)
