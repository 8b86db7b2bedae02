"""Layer norm, dropout with bias and residual sum, and both in one pass, against 64-bit arithmetic.

Tolerances, before any run: a result rounded to bf16 is off by half a step, 2^-8 of its value; fp32 arithmetic in front of it adds a share of the
magnitudes M it combines, 2^-24 per operation in a chain of at most SLOP of them (sums of h <= 8192 terms: 16 in a lane, 6 steps across a
wave, 4 across waves, and the mean, the square root and the products behind them); sums over n rows add n 2^-24 of the sum of magnitudes."""
import numpy as np
import pytest
import torch

import _draw

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -24
SLOP = 64


@pytest.fixture(scope="module")
def F():
    from easyllm_amd import functional
    return functional


@pytest.fixture(scope="module")
def K():
    from easyllm_amd import kernels
    return kernels


def rnd(*shape, seed=0, scale=1.0, mean=0.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale + mean).bfloat16()


def factor(shape, p, seed, offset, step=0):
    return torch.from_numpy(_draw.factor(shape, int(p * 65536 + 0.5), seed, offset, step)).cuda()


def near(got, ref, magnitude, what, rounded=2.0 ** -8, slop=SLOP):
    assert got.shape == ref.shape, what
    off = (got.double() - ref).abs() - ref.abs() * rounded - magnitude * (slop * EPS)
    assert bool((off <= 0).all()), "%s: %g beyond its tolerance" % (what, off.max().item())


def sum_near(got, terms, noise, what):
    """A column sum: fp32 over the rows, then one rounding (bf16) or none (fp32); `noise`: what each term may be off by."""
    n = terms.shape[0]
    slack = (terms.abs().sum(0) * (n + SLOP) * EPS + noise.sum(0) if n else torch.zeros_like(got.double()))
    rounded = 2.0 ** -8 if got.dtype == torch.bfloat16 else 2.0 ** -24
    off = (got.double() - terms.sum(0)).abs() - terms.sum(0).abs() * rounded - slack
    assert bool((off <= 0).all()), "%s: %g beyond its tolerance" % (what, off.max().item())


def oracle(kind, s, w, b, eps):
    """y, mean, rstd, xhat of fp64 rows, and the magnitude that y's fp32 arithmetic combines"""
    mean = s.mean(1, keepdim=True) if kind == 0 else torch.zeros_like(s[:, :1])
    rstd = ((s - mean).square().mean(1, keepdim=True) + eps).rsqrt()
    xhat = (s - mean) * rstd
    y = xhat * w + (0 if b is None else b)
    # xhat's relative error grows with what the mean takes away: (|s| + |mean|) rstd
    return y, mean[:, 0], rstd[:, 0], xhat, ((s.abs() + mean.abs()) * rstd + xhat.abs()) * w.abs() + (0 if b is None else b.abs())


def oracle_grads(kind, dy, s, mean, rstd, w, dsum):
    xhat = (s - mean[:, None]) * rstd[:, None]
    g = dy * w
    ds = g - xhat * (g * xhat).mean(1, keepdim=True)
    if kind == 0:
        ds = ds - g.mean(1, keepdim=True)
    size = (s.abs() + mean.abs()[:, None]) * rstd[:, None]
    big = g.abs() + size * (g.abs() * size).mean(1, keepdim=True) + g.abs().mean(1, keepdim=True)
    return ds * rstd[:, None] + dsum, xhat, big * rstd[:, None] + dsum.abs(), size


# widths at each side of every rule: threads of a row (512, 1024, 1536, 2048 columns), chunks, waves of a row backward (2048, 4096, 6144)
SHAPES = [(1, 8), (3, 64), (7, 504), (5, 520), (2, 1000), (9, 1032), (3, 1544), (2, 2040), (3, 2056), (2, 4096), (3, 4104), (2, 6152), (3, 8184), (1, 8192),
          (1167, 256), (513, 768), (1030, 2048), (517, 5120)]


def test_the_oracles_gradient_is_the_derivative():
    """The formula above against autograd and against differences, in 64 bits."""
    torch.manual_seed(0)
    for kind in (0, 1):
        s = torch.randn(3, 16, dtype=torch.float64, requires_grad=True)
        w, b = torch.randn(16, dtype=torch.float64), torch.randn(16, dtype=torch.float64)
        dy = torch.randn(3, 16, dtype=torch.float64)
        y, mean, rstd, _, _ = oracle(kind, s, w, b if kind == 0 else None, 1e-5)
        (auto,) = torch.autograd.grad(y, s, dy)
        ds = oracle_grads(kind, dy, s.detach(), mean.detach(), rstd.detach(), w, torch.zeros_like(dy))[0]
        assert torch.allclose(auto, ds, rtol=1e-10, atol=1e-12)
        d = torch.randn_like(s) * 1e-5
        up, down = (oracle(kind, s.detach() + e, w, None, 1e-5)[0] for e in (d, -d))
        assert torch.allclose(((up - down) * dy).sum(), 2 * (ds * d).sum(), rtol=1e-6)


@pytest.mark.parametrize("rows,h", SHAPES)
@pytest.mark.parametrize("bias", [True, False])
def test_layer_norm_forward(K, rows, h, bias):
    print("layer norm", rows, h, bias, flush=True)
    x, w, b = rnd(rows, h, seed=1, mean=0.5), rnd(h, seed=2, scale=0.1, mean=1.0), rnd(h, seed=3, scale=0.1) if bias else None
    y, s, mean, rstd = K.norm_fwd(K.LAYER_NORM, x, w, b, 1e-5)
    ref, rmean, rrstd, _, big = oracle(0, x.double(), w.double(), None if b is None else b.double(), 1e-5)
    assert s is None
    near(y, ref, big, "y")
    near(mean, rmean, x.double().abs().mean(1), "mean", rounded=0)
    near(rstd, rrstd, rrstd * (1 + rmean.abs() * rrstd), "rstd", rounded=0)


@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("rows,h", SHAPES)
@pytest.mark.parametrize("p,bias", [(0.0, False), (0.0, True), (0.1, True), (0.5, False)])
def test_norm_behind_dropout_and_sum_forward(K, kind, rows, h, p, bias):
    print("norm", kind, rows, h, p, bias, flush=True)
    x, r, w = rnd(rows, h, seed=1), rnd(rows, h, seed=2, mean=0.3), rnd(h, seed=3, scale=0.1, mean=1.0)
    b, xb = rnd(h, seed=4, scale=0.1) if kind == 0 else None, rnd(h, seed=5) if bias else None
    t = int(p * 65536 + 0.5)
    y, s, mean, rstd = K.norm_fwd(kind, x, w, b, 1e-5, r, xb, t, (2 ** 40 + 5, 77))
    f = factor((rows, h), p, 2 ** 40 + 5, 77)
    inner = (x.double() + (0 if xb is None else xb.double())) * f
    ref_s = r.double() + inner
    size = r.double().abs() + f * (x.double().abs() + (0 if xb is None else xb.double().abs()))
    near(s, ref_s, size, "sum", slop=4)
    if p:
        only = K.norm_fwd(kind, x, w, b, 1e-5, torch.zeros_like(r), xb, t, (2 ** 40 + 5, 77))[1]
        assert torch.equal(only == 0, inner == 0)  # the mask itself
    ref, rmean, rrstd, _, big = oracle(kind, ref_s, w.double(), None if b is None else b.double(), 1e-5)
    near(y, ref, big + size * rrstd[:, None] * w.double().abs(), "y")
    near(rstd, rrstd, rrstd * (2 + rmean.abs() * rrstd), "rstd", rounded=0)
    assert (mean is None) == (kind == 1)


@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("rows,h", SHAPES)
@pytest.mark.parametrize("p,bias,dsum", [(0.0, False, False), (0.0, True, True), (0.1, True, True), (0.5, False, False)])
def test_norm_backward(K, kind, rows, h, p, bias, dsum):
    """The kernel on an s and statistics of its own: everything it reads is exact."""
    print("norm backward", kind, rows, h, p, bias, dsum, flush=True)
    s, dy, w = rnd(rows, h, seed=1, mean=0.3), rnd(rows, h, seed=2), rnd(h, seed=3, scale=0.1, mean=1.0)
    d = rnd(rows, h, seed=4) if dsum else None
    _, mean, rstd, _, _ = oracle(kind, s.double(), w.double(), None, 1e-5)
    mean, rstd = mean.float(), rstd.float()
    dw, db, dxb = (torch.empty(h, dtype=torch.bfloat16, device="cuda"), torch.full((h,), 3.0, device="cuda"), torch.empty(h, dtype=torch.bfloat16, device="cuda"))
    t = int(p * 65536 + 0.5)
    dx, dres = K.norm_bwd(kind, dy, s, w, None if kind else mean, rstd, (None, dw, False), (db, None, True) if kind == 0 else None, d, t, (9, 4),
                          (None, dxb, False) if bias else None)
    ref, xhat, big, size = oracle_grads(kind, dy.double(), s.double(), mean.double(), rstd.double(), w.double(), d.double() if dsum else torch.zeros(rows, h, device="cuda").double())
    f = factor((rows, h), p, 9, 4)
    near(dres, ref, big, "dresidual")
    near(dx, ref * f, big * f, "dx")
    assert (dx.data_ptr() == dres.data_ptr()) == (t == 0)
    sum_near(dw, dy.double() * xhat, dy.double().abs() * size * (4 * EPS), "dweight")
    if kind == 0:
        sum_near(db - 3.0, dy.double(), torch.full_like(ref, 3 * EPS), "dbias")
    if bias:
        sum_near(dxb, ref * f, big * f * (SLOP * EPS), "dx_bias")


def test_a_row_far_from_zero_and_a_constant_one(K):
    """Mean 1000, spread 4: the variance as a difference of mean squares would lose it.  A constant row has no variance: y is the bias."""
    h = 4096
    x = rnd(3, h, seed=1, scale=4.0, mean=1000.0)
    x[1] = 7.0
    w, b = rnd(h, seed=2, mean=1.0), rnd(h, seed=3)
    y, _, mean, rstd = K.norm_fwd(K.LAYER_NORM, x, w, b, 1e-5)
    ref, _, _, _, big = oracle(0, x.double(), w.double(), b.double(), 1e-5)
    near(y, ref, big, "y")
    assert torch.equal(y[1], b) and mean[1].item() == 7.0


def test_no_rows(K):
    x, w = torch.empty(0, 64, dtype=torch.bfloat16, device="cuda"), rnd(64)
    assert K.norm_fwd(K.LAYER_NORM, x, w, w, 1e-5)[0].shape == (0, 64)
    assert K.norm_fwd(K.RMS_NORM, x, w, None, 1e-5, x, w, 100, (1, 2))[1].shape == (0, 64)
    dw, db, dxb = (torch.full((64,), 5.0, dtype=torch.bfloat16, device="cuda") for _ in range(3))
    stat = torch.empty(0, device="cuda")
    K.norm_bwd(K.LAYER_NORM, x, x, w, stat, stat, (None, dw, False), (None, db, False), None, 100, (1, 2), (None, dxb, False))
    assert not dw.any() and not db.any() and not dxb.any()
    dxb.fill_(5)
    assert K.dropout_add_fwd(x, w, None, 100, (1, 2)).shape == (0, 64)
    K.dropout_add_bwd(x, 100, (1, 2), (None, dxb, False))
    assert not dxb.any()
    dxb.fill_(5)
    K.dropout_add_bwd(x, 0, None, (None, dxb, False))
    assert not dxb.any()


def test_one_row_without_a_batch(F):
    x, r, w, b = (rnd(264, seed=i).requires_grad_(True) for i in range(4))
    s, y = F.dropout_add_layer_norm(x, r, w, b, p=0.5, rng=(1, 2))
    two = [t.detach().view(1, -1).requires_grad_(True) for t in (x, r)]
    s2, y2 = F.dropout_add_layer_norm(*two, w, b, p=0.5, rng=(1, 2))
    assert torch.equal(s, s2[0]) and torch.equal(y, y2[0])
    got, want = torch.autograd.grad((y, s), (x, r, w, b), (x, r)), torch.autograd.grad((y2, s2), (*two, w, b), two)
    for a, c in zip(got, want):
        assert torch.equal(a, c.view_as(a))


@pytest.mark.parametrize("rows,n", [(1, 8), (3, 64), (5, 520), (1167, 1000), (7, 8192), (2, 13704), (517, 5120), (4099, 256)])
@pytest.mark.parametrize("bias,residual", [(False, False), (True, False), (False, True), (True, True)])
@pytest.mark.parametrize("p", [0.0, 0.1, 1.0])
def test_dropout_add(K, rows, n, bias, residual, p):
    print("dropout", rows, n, bias, residual, p, flush=True)
    x = rnd(rows, n, seed=1)
    b, r = rnd(n, seed=2) if bias else None, rnd(rows, n, seed=3) if residual else None
    t = int(p * 65536 + 0.5)
    seed, offset = 0xFEDCBA9876543210, 0xFFFFFFFF
    out = K.dropout_add_fwd(x, b, r, t, (seed, offset))
    f = factor((rows, n), p, seed, offset)
    zero = torch.zeros((), device="cuda").double()
    bd, rd = zero if b is None else b.double(), zero if r is None else r.double()
    near(out, rd + (x.double() + bd) * f, rd.abs() + (x.double().abs() + bd.abs()) * f, "out", slop=4)
    dy = rnd(rows, n, seed=4)
    for target in [None] + [dict(f32=True), dict(f32=False)] * bias:
        dbias = None
        if target:
            buf = torch.full((n,), 2.0, device="cuda") if target["f32"] else torch.empty(n, dtype=torch.bfloat16, device="cuda")
            dbias = (buf, None, True) if target["f32"] else (None, buf, False)
        dx = K.dropout_add_bwd(dy, t, (seed, offset), dbias)
        near(dx, dy.double() * f, dy.double().abs() * f, "dx", slop=2)
        if target:
            sum_near(buf - 2.0 if target["f32"] else buf, dy.double() * f, dy.double().abs() * f * (2 * EPS) + 2 * EPS, "dbias")


def test_what_is_dropped_is_zero_whatever_it_held(K):
    x = rnd(64, 256, seed=1)
    f = factor((64, 256), 0.5, 3, 0)
    x[f == 0] = float("nan")
    r = rnd(64, 256, seed=2)
    assert torch.isfinite(K.dropout_add_fwd(x, None, r, 32768, (3, 0))).all()
    y, s, _, _ = K.norm_fwd(K.LAYER_NORM, x, rnd(256), None, 1e-5, r, None, 32768, (3, 0))
    assert torch.isfinite(y).all() and torch.isfinite(s).all()


def test_masks_differ_by_seed_offset_and_step(K):
    x = torch.ones(64, 1024, dtype=torch.bfloat16, device="cuda")
    step = torch.tensor([5], device="cuda")
    draws = [(1, 0), (2, 0), (1, 1), (1, 0, step), (1 + 2 ** 32, 0)]
    masks = [K.dropout_add_fwd(x, None, None, 32768, d) != 0 for d in draws]
    assert torch.equal(masks[3], factor((64, 1024), 0.5, 1, 0, step=5) != 0)
    for i in range(len(masks)):
        for j in range(i):
            share = (masks[i] == masks[j]).double().mean().item()
            assert abs(share - 0.5) < 5 * 0.5 / 256, (i, j, share)  # 65536 independent bits
    step += 1
    assert not torch.equal(K.dropout_add_fwd(x, None, None, 32768, draws[3]) != 0, masks[3])
    neighbours = masks[0].double()
    for lag in (1, 2, 8, 1024):
        a = neighbours.flatten()
        assert abs((a[lag:] * a[:-lag]).mean().item() - 0.25) < 5 * 0.5 / 256


def test_more_than_2_31_elements(K):
    """262208 rows of 8192: byte offsets past 32 bits and group numbers that the rows' end needs; the last rows against the definition."""
    rows, h = 262208, 8192
    x = torch.empty(rows, h, dtype=torch.bfloat16, device="cuda")
    x.copy_(rnd(h, seed=1).expand(rows, h))
    last = 4
    f = torch.from_numpy(_draw.factor((last, h), 6554, 11, 2, first_group=(rows - last) * h // 8)).cuda()
    out = K.dropout_add_fwd(x, None, x, 6554, (11, 2))
    ref = x[-last:].double() * (1 + f)
    near(out[-last:], ref, ref.abs() * 2, "out", slop=4)
    w = rnd(h, seed=2, mean=1.0)
    y, s, mean, rstd = K.norm_fwd(K.LAYER_NORM, x, w, None, 1e-5, x, None, 6554, (11, 2))
    assert torch.equal(s, out)
    want, _, _, _, big = oracle(0, ref, w.double(), None, 1e-5)
    near(y[-last:], want, big * 2, "y")
    del y, out
    dw = torch.empty(h, device="cuda")
    dx, dres = K.norm_bwd(K.LAYER_NORM, x, s, w, mean, rstd, (dw, None, False), None, None, 6554, (11, 2))
    want, _, big, _ = oracle_grads(0, x[-last:].double(), s[-last:].double(), mean[-last:].double(), rstd[-last:].double(), w.double(), torch.zeros_like(ref))
    near(dres[-last:], want, big, "dresidual")
    near(dx[-last:], want * f, big * f, "dx")
    assert torch.isfinite(dw).all()


# ---- through autograd ------------------------------------------------------------------------------------------------
def grads_of(outs, leaves, dys):
    return torch.autograd.grad(outs, leaves, dys)


@pytest.mark.parametrize("kind,p,bias", [(0, 0.1, True), (0, 0.0, False), (1, 0.25, False), (1, 0.0, True)])
def test_gradients_through_the_public_call(F, kind, p, bias):
    """Strided inputs, a bias that several rows share, both outputs used; the definition's gradient, s rounded where the call keeps it."""
    s_len, b_len, h = 37, 3, 776
    x = rnd(b_len, s_len, h, seed=1).transpose(0, 1).requires_grad_(True)
    r = rnd(s_len, b_len, 2 * h, seed=2)[..., h:].requires_grad_(True)
    w, nb = rnd(h, seed=3, mean=1.0).requires_grad_(True), rnd(h, seed=4).requires_grad_(True) if kind == 0 else None
    xb = rnd(h, seed=5).requires_grad_(True) if bias else None
    d_s, d_y = rnd(s_len, b_len, h, seed=6), rnd(h, seed=7).expand(s_len, b_len, h)
    if kind == 0:
        s, y = F.dropout_add_layer_norm(x, r, w, nb, 1e-5, bias=xb, p=p, rng=(5, 6))
    else:
        s, y = F.dropout_add_rmsnorm(x, r, w, 1e-5, bias=xb, p=p, rng=(5, 6))
    leaves = [t for t in (x, r, w, nb, xb) if t is not None]
    got = dict(zip([n for n, t in zip("xrwnb", (x, r, w, nb, xb)) if t is not None], grads_of([s, y], leaves, [d_s, d_y])))
    f = factor((s_len * b_len, h), p, 5, 6)
    flat = lambda t: t.detach().reshape(-1, h).double()  # noqa: E731
    ref_s = flat(r) + (flat(x) + (0 if xb is None else xb.double())) * f
    _, mean, rstd, _, _ = oracle(kind, ref_s, w.double(), None, 1e-5)
    stored = flat(s)
    ref, xhat, big, size = oracle_grads(kind, flat(d_y), stored, mean, rstd, w.double(), flat(d_s))
    near(flat(got["r"]), ref, big, "dresidual")
    near(flat(got["x"]), ref * f, big * f, "dx")
    sum_near(got["w"], flat(d_y) * xhat, flat(d_y).abs() * size * (SLOP * EPS), "dweight")
    if kind == 0:
        sum_near(got["n"], flat(d_y), torch.zeros_like(ref), "dbias")
    if bias:
        sum_near(got["b"], ref * f, big * f * (SLOP * EPS), "dx_bias")
    assert got["x"].shape == x.shape and got["r"].shape == r.shape


def test_main_grads_and_frozen_parameters(F):
    """fp32 buffers are overwritten when fresh and added to otherwise; what needs no gradient gets none, and its buffer stays as it is."""
    h = 264
    x, r = rnd(50, h, seed=1).requires_grad_(True), rnd(50, h, seed=2)
    params = [rnd(h, seed=i, mean=1.0).requires_grad_(True) for i in (3, 4, 5)]
    w, nb, xb = params
    for q in params:
        q.main_grad, q.main_grad_fresh = torch.full((h,), 9.0, device="cuda"), True
    dy = rnd(50, h, seed=6)
    once = []
    for _ in range(2):
        s, y = F.dropout_add_layer_norm(x, r, w, nb, bias=xb, p=0.1, rng=(1, 1))
        (s * 0 + y).backward(dy)
        once.append([q.main_grad.clone() for q in params])
    assert all(q.grad is None for q in params)
    for a, b in zip(*once):
        assert torch.allclose(b, 2 * a, rtol=1e-6, atol=1e-6) and not (a == 9.0).any()
    nb.requires_grad_(False)
    xb.requires_grad_(False)
    kept = [q.main_grad.clone() for q in params]
    s, y = F.dropout_add_layer_norm(x, r, w, nb, bias=xb, p=0.1, rng=(1, 1))
    y.backward(dy)
    assert torch.equal(nb.main_grad, kept[1]) and torch.equal(xb.main_grad, kept[2]) and not torch.equal(w.main_grad, kept[0])
    out = F.dropout_add(x, bias=xb, p=0.5, rng=(1, 1))
    out.backward(dy)
    assert torch.equal(xb.main_grad, kept[2])
    xb.requires_grad_(True)
    xb.main_grad_fresh = True
    F.dropout_add(x, bias=xb, p=0.5, rng=(1, 1)).backward(dy)
    sum_near(xb.main_grad, dy.double() * factor((50, h), 0.5, 1, 1), torch.zeros(50, h, device="cuda").double() + 1e-6, "dbias")


def test_one_parameter_in_several_places(F):
    """Its fp32 buffer takes the gradients one after the other: overwritten once where it is fresh, then added to."""
    h = 2056
    x, r, p = rnd(300, h, seed=1).requires_grad_(True), rnd(300, h, seed=2), rnd(h, seed=3).requires_grad_(True)
    d = rnd(300, h, seed=4)

    def call(q):
        s, y = F.dropout_add_layer_norm(x, r, q[0], q[1], bias=q[2], p=0.1, rng=(1, 1))
        return torch.autograd.grad((y, s), q, (d, d))
    apart = [p.detach().clone().requires_grad_(True) for _ in range(3)]
    want = sum(g.double() for g in call(apart))
    for fresh in (True, False):
        p.main_grad, p.main_grad_fresh = torch.full((h,), 7.0, device="cuda"), fresh
        s, y = F.dropout_add_layer_norm(x, r, p, p, bias=p, p=0.1, rng=(1, 1))
        torch.autograd.backward((y, s), (d, d))
        off = (p.main_grad.double() - want - (0 if fresh else 7)).abs()
        # the three are rounded to bf16 in `want`, 2^-8 each of at most
        assert bool((off <= 2.0 ** -8 * sum(g.double().abs() for g in call(apart)) + 1e-3).all()), off.max()
        p.main_grad = None


@pytest.mark.parametrize("frozen", ["w", "nb", "xb", "x", "r", "w nb xb"])
def test_gradients_do_not_change_with_what_is_frozen(F, frozen):
    names = ("x", "r", "w", "nb", "xb")
    t = dict(zip(names, (rnd(70, 1032, seed=1), rnd(70, 1032, seed=2), rnd(1032, seed=3), rnd(1032, seed=4), rnd(1032, seed=5))))
    d = rnd(70, 1032, seed=6), rnd(70, 1032, seed=7)

    def grads(wanted):
        v = {n: a.clone().requires_grad_(n in wanted) for n, a in t.items()}
        s, y = F.dropout_add_layer_norm(v["x"], v["r"], v["w"], v["nb"], bias=v["xb"], p=0.25, rng=(8, 9))
        return dict(zip(wanted, torch.autograd.grad((s, y), [v[n] for n in wanted], d)))
    every, some = grads(names), grads([n for n in names if n not in frozen.split()])
    for n, g in some.items():
        assert torch.equal(g, every[n]), n


def test_results_do_not_depend_on_the_launch_or_the_stream(F):
    x, r, w, nb = rnd(1500, 1032, seed=1).requires_grad_(True), rnd(1500, 1032, seed=2), rnd(1032, seed=3).requires_grad_(True), rnd(1032, seed=4)
    dy = rnd(1500, 1032, seed=5)

    def call():
        s, y = F.dropout_add_layer_norm(x, r, w, nb, p=0.1, rng=(1, 1))
        return (s, y) + torch.autograd.grad((y, s), (x, w), (dy, dy))
    first = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = call()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(first, other):
        assert torch.equal(a, b)


def test_the_wrappers_refuse(F, K):
    x, w = rnd(4, 64), rnd(64)
    for bad in (lambda: F.layer_norm(x.float(), w), lambda: F.layer_norm(x.cpu(), w.cpu()), lambda: F.layer_norm(x, rnd(72)), lambda: F.layer_norm(x, w, rnd(72)),
                lambda: F.add_layer_norm(x, rnd(3, 64), w), lambda: F.dropout_add(x, rnd(1, 64), p=0.1), lambda: F.dropout_add(x, bias=rnd(8)),
                lambda: F.dropout_add(x, p=1.5), lambda: F.dropout_add(x, p=0.1, rng=(1, 2 ** 32)), lambda: F.dropout_add(x, p=0.1, rng=(1, 0, torch.zeros(1, device="cuda"))),
                lambda: F.dropout_add(x, p=0.1, rng=(1, 0, torch.zeros(1, dtype=torch.int64)))):
        with pytest.raises((ValueError, TypeError)):
            bad()
    with pytest.raises(RuntimeError, match="8192"):
        F.layer_norm(rnd(2, 8200), rnd(8200))
    with pytest.raises(RuntimeError, match="aligned"):
        F.layer_norm(rnd(4 * 64 + 1)[1:].view(4, 64), w)


def test_a_captured_pass_draws_anew_on_every_replay(F):
    """Forward and backward in one graph, its step advanced between the replays, eager work of the program's own in between."""
    from easyllm_amd import dropout
    x, r, w = rnd(300, 512, seed=1).requires_grad_(True), rnd(300, 512, seed=2), rnd(512, seed=3).requires_grad_(True)
    dy = rnd(300, 512, seed=4)

    def call(rng=None):
        s, y = F.dropout_add_layer_norm(x, r, w, None, p=0.2, rng=rng)
        return (s, y) + torch.autograd.grad((y, s), (x, w), (dy, dy))
    step = torch.zeros(1, dtype=torch.int64, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with dropout.recording() as draws, dropout.stepping(step), torch.cuda.graph(graph):
        outs = call()
    assert len(draws) == 1 and draws[0].step is step
    for i in range(1, 5):
        step.add_(1)
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in outs]
        want = call(rng=(draws[0].seed, draws[0].offset, torch.tensor([i], device="cuda")))
        for a, b in zip(got, want):
            assert torch.equal(a, b), i
        masks = factor((300, 512), 0.2, draws[0].seed, draws[0].offset, step=i)
        assert torch.equal((got[2] == 0) & (masks != 0), (got[2] == 0) & (want[2] == 0) & (masks != 0))
    kept = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="stepping"):
        with torch.cuda.graph(kept):
            call()
