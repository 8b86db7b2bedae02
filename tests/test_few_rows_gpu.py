"""Products of up to 16 rows with an epilogue on both sides of each bound of their kernel's rule: 8 and 16 rows, 4096 and 8192 columns, K of 2560, 4096 and 5120, and every
number of K blocks that a wave owns.

Tolerances, before any run, as in the other tests of these products: a sum of K products is off by at most K 2^-24 of the sum of magnitudes S (taken twice too
large), a slope below 1.13 passes 1.2 of it on, the activation adds 2^-15 of its value, rounding to bf16 2^-8 of the result."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -24


def rnd(*shape, seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).bfloat16()


def close(got, ref, slack, what):
    off = (got.double() - ref).abs() - ref.abs() * 2.0 ** -8 - slack
    assert got.shape == ref.shape and bool((off <= 0).all()), "%s: %g beyond its tolerance" % (what, off.max().item())


@pytest.mark.parametrize("M,N,K", [
    (8, 520, 5120), (8, 520, 5128), (1, 4096, 5120), (7, 4104, 5120), (8, 8192, 5120), (8, 8200, 5120), (3, 1032, 4616), (9, 1032, 4616), (9, 4096, 4096), (16, 4096, 4096),
    (16, 4096, 4104), (9, 4104, 4096), (16, 8192, 2560), (16, 8200, 2560), (16, 8192, 2568), (12, 72, 3080), (2, 8192, 3592), (8, 264, 512), (8, 264, 1024), (8, 264, 1032),
    (13, 264, 2048), (17, 264, 2048)])
def test_both_sides_of_every_bound(M, N, K):
    from easyllm_amd import kernels
    print("few rows", M, N, K, flush=True)
    x, w, b, r = rnd(M, K, seed=1), rnd(N, K, seed=2, scale=K ** -0.5), rnd(N, seed=3), rnd(M, N, seed=4, scale=4)
    y, pre = kernels.linear_act_fwd(x, w, b, "gelu", r, True)
    v = x.double() @ w.double().t() + b.double()
    err = (x.double().abs() @ w.double().abs().t() + b.double().abs()) * (2 * (K + 4) * EPS)
    close(pre, v, err, "pre")
    a = v * 0.5 * torch.special.erfc(-v / math.sqrt(2))
    close(y, a + r.double(), 1.2 * err + a.abs() * 2.0 ** -15 + ((a + r.double()).abs() + r.double().abs()) * EPS, "y")
