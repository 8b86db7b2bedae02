"""A product with an epilogue, and the activation's backward, whose results have more than 2^31 elements: the last rows against 64 bits, and sums over all rows.

Tolerances, before any run, as in the other tests of these products: 2^-8 of the result for its rounding, 2^-15 of an activation's value or slope, K 2^-24 of the sum of
magnitudes twice, and for a sum of n rows n 2^-24 of the sum of magnitudes."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -24


def rnd(*shape, seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).bfloat16()


@pytest.mark.parametrize("rows,n,k", [(262400, 8192, 64), (1100, 2097144, 8)])
def test_more_than_2_31_elements(rows, n, k):
    from easyllm_amd import kernels
    print("long", rows, n, k, flush=True)
    assert rows * n > 2 ** 31
    x, w, b = rnd(rows, k, seed=1), rnd(n, k, seed=2, scale=k ** -0.5), rnd(n, seed=3)
    r = torch.empty(rows, n, dtype=torch.bfloat16, device="cuda")
    r.copy_(rnd(rows, 1, seed=4).expand(rows, n))
    y, pre = kernels.linear_act_fwd(x, w, b, "gelu", r, True)
    last, cols = slice(rows - 5, rows), slice(n - 1000, n)
    v = x[last].double() @ w[cols].double().t() + b[cols].double()
    err = (x[last].double().abs() @ w[cols].double().abs().t() + b[cols].double().abs()) * (2 * (k + 4) * EPS)
    assert ((pre[last, cols].double() - v).abs() <= v.abs() * 2.0 ** -8 + err).all()
    cdf = 0.5 * torch.special.erfc(-v / math.sqrt(2))
    want = v * cdf + r[last, cols].double()
    assert ((y[last, cols].double() - want).abs() <= want.abs() * 2.0 ** -8 + 1.2 * err + (v * cdf).abs() * 2.0 ** -15 + (want.abs() + r[last, cols].double().abs()) * EPS).all()
    del y
    db = torch.empty(n, device="cuda")
    d = kernels.act_bwd("gelu", r, pre, (db, None, False))
    p = pre[last, cols].double()
    slope = 0.5 * torch.special.erfc(-p / math.sqrt(2)) + p * torch.exp(-0.5 * p * p) / math.sqrt(2 * math.pi)
    want = r[last, cols].double() * slope
    assert ((d[last, cols].double() - want).abs() <= want.abs() * 2.0 ** -8 + r[last, cols].double().abs() * 2.0 ** -15).all()
    # every column's sum lies as near the sum of the rounded terms as their roundings and the summation allow
    some = torch.arange(0, n, max(1, n // 64), device="cuda")
    terms = d[:, some].double()
    assert ((db[some].double() - terms.sum(0)).abs() <= terms.abs().sum(0) * (2.0 ** -8 + (rows + 64) * EPS)).all()
