"""The weights of the 8-bit step are its definition's bit by bit: products, sums, the root and the quotient one correctly rounded fp32 operation each, here and in numpy."""
import numpy as np
import pytest
import torch

import _adam8 as R
from test_adam8_gpu import HOW, gradient, random_state

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [1, 700, 4096, 100003, 1 << 20])
@pytest.mark.parametrize("decay", [0.0, 0.1])
def test_weights_bit_by_bit(n, decay):
    from easyllm_amd import optimizer as O
    state, gpu = random_state(n, n, number=3)
    weight = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    for k in (1, 2, 50, 10000):
        how = dict(HOW, weight_decay=decay, step=k)
        g = gradient(n, n + k)
        R.step(state, g, how)
        O.adamw_8bit_step([gpu], [torch.from_numpy(g).cuda()], [weight], **how)
        got = gpu["master"].cpu().numpy()
        wrong = np.flatnonzero(got.view(np.uint32) != state["master"].view(np.uint32))
        assert not len(wrong), (k, wrong[:5])
        assert torch.equal(weight, gpu["master"].bfloat16())


def test_second_moments_of_every_size():
    """Roots of values from the smallest a code stands for (far below the smallest normal number) to the largest, and eps as large as they are."""
    from easyllm_amd import optimizer as O
    n = 256 * 256
    for eps in (0.0, 1e-8, 1.0):
        state, gpu = random_state(n, 5)
        scales = np.arange(256).clip(0, 250).astype(np.uint8)
        codes = np.random.default_rng(1).integers(1, 256, n).astype(np.uint8)
        state["exp_avg_sq"][:], state["exp_avg_sq_scale"][:] = codes, scales
        gpu["exp_avg_sq"].copy_(torch.from_numpy(codes)), gpu["exp_avg_sq_scale"].copy_(torch.from_numpy(scales))
        how = dict(HOW, eps=eps, step=7)
        g = np.zeros(n, np.float32)
        R.step(state, g, how)
        O.adamw_8bit_step([gpu], [torch.from_numpy(g).cuda()], [None], **how)
        got, want = gpu["master"].cpu().numpy(), state["master"]
        same = (got.view(np.uint32) == want.view(np.uint32)) | (np.isnan(got) & np.isnan(want))
        assert same.all(), (eps, np.flatnonzero(~same)[:5], got[~same][:5], want[~same][:5])
