"""Residuals of products that the kernel cannot read where they lie: far apart, on odd addresses, a single row with a stride that means nothing."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def rnd(*shape, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").bfloat16()


LAYOUTS = {
    "the last token of a long sequence": lambda: rnd(1, 4100, 520, seed=3)[:, -1],
    "the last tokens of two": lambda: rnd(2, 4100, 520, seed=3)[:, -1],
    "a row of one expanded": lambda: rnd(520, seed=3).expand(1, 520),
    "an odd first column": lambda: rnd(5, 528, seed=3)[:, 3:523],
    "an odd row length": lambda: rnd(5, 523, seed=3)[:, :520],
    "one vector without a batch": lambda: rnd(520, 2, seed=3)[:, 0],
}


@pytest.mark.parametrize("name", LAYOUTS)
def test_residuals_that_have_to_be_copied(name):
    from easyllm_amd import functional as F
    r = LAYOUTS[name]()
    x, w = rnd(*r.shape[:-1], 64, seed=1), rnd(520, 64, seed=2)
    whole = torch.empty(r.shape, dtype=r.dtype, device="cuda").copy_(r)
    rr, want_r = r.requires_grad_(True), whole.requires_grad_(True)
    y, want = F.linear_act(x, w, None, "gelu", rr), F.linear_act(x, w, None, "gelu", want_r)
    assert torch.equal(y, want)
    dy = rnd(*y.shape, seed=4)
    assert torch.equal(torch.autograd.grad(y, rr, dy)[0], torch.autograd.grad(want, want_r, dy)[0])
