"""The norm backward writes nothing past the workspace that it asks for."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,h", [(0, 264), (1, 8), (1, 8192), (3, 4104), (7, 8192), (255, 264), (300, 2056), (1030, 2048), (8200, 2048), (4100, 4096), (4096, 5120)])
def test_what_stands_behind_the_workspace_stays(rows, h):
    from easyllm_amd import _lib
    from easyllm_amd import kernels as K
    print("workspace", rows, h, flush=True)
    g = torch.Generator(device="cuda").manual_seed(1)
    s, dy = (torch.randn(rows, h, generator=g, device="cuda").bfloat16() for _ in range(2))
    w = torch.randn(h, generator=g, device="cuda").bfloat16()
    mean, rstd = s.float().mean(1), s.float().var(1, correction=0).add(1e-5).rsqrt()
    size = _lib.norm_bwd_workspace_bytes(rows, h)
    room = torch.full((size // 4 + 3 * h,), 7.0, device="cuda")
    grads = [torch.empty(h, device="cuda") for _ in range(3)]
    to = [ctypes.byref(_lib.LayerGrad(t.data_ptr(), None, 0)) for t in grads]
    dx, dres = torch.empty_like(s), torch.empty_like(s)
    drop = ctypes.byref(_lib.Dropout(1, 2, 6554, None))
    _lib.call("ezl_norm_bwd", K.LAYER_NORM, dy.data_ptr(), None, s.data_ptr(), w.data_ptr(), mean.data_ptr(), rstd.data_ptr(), drop, dx.data_ptr(), dres.data_ptr(), *to,
              room.data_ptr(), size, rows, h, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert (room[size // 4:] == 7).all()
    want = [torch.empty(h, device="cuda") for _ in range(3)]
    wx, wr = K.norm_bwd(K.LAYER_NORM, dy, s, w, mean, rstd, (want[0], None, False), (want[1], None, False), None, 6554, (1, 2), (want[2], None, False))
    assert torch.equal(dx, wx) and torch.equal(dres, wr) and all(torch.equal(a, b) for a, b in zip(grads, want))
