"""act(x W^T + bias) + residual, forward and backward, against 64-bit arithmetic, on every tile shape a forward product takes.

Tolerances, before any run: products of bf16 values are exact in fp32 and a sum of K of them is off by at most K 2^-24 of the sum of magnitudes S
(taken twice too large, for partial sums); an activation's slope is below 1.13, so the error it is given goes on as 1.2 times itself, and its own
arithmetic adds 2^-15 of its value (the fit of the normal distribution's tail is 5.2e-6 off, exponentials of arguments up to 100 add three times 2^-24 of them); bf16
rounding adds 2^-8 of the result."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -24


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


def act64(v, act):
    """act(v), act'(v) in fp64"""
    if act == "gelu":
        cdf = 0.5 * torch.special.erfc(-v / math.sqrt(2))
        return v * cdf, cdf + v * torch.exp(-0.5 * v * v) / math.sqrt(2 * math.pi)
    if act == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        s = torch.sigmoid(2 * c * (v + 0.044715 * v ** 3))
        return v * s, s + v * s * (1 - s) * 2 * c * (1 + 3 * 0.044715 * v * v)
    return v, torch.ones_like(v)


def close(got, ref, slack, what):
    off = (got.double() - ref).abs() - ref.abs() * 2.0 ** -8 - slack
    assert got.shape == ref.shape and bool((off <= 0).all()), "%s: %g beyond its tolerance" % (what, off.max().item())


def check_forward(K, M, N, Kd, act, bias, residual, seed=0, want_pre=True, strided=False):
    x = rnd(M, 2 * Kd, seed=seed)[:, Kd:] if strided else rnd(M, Kd, seed=seed)
    w = rnd(N, Kd + 8, seed=seed + 1, scale=Kd ** -0.5)[:, :Kd] if strided else rnd(N, Kd, seed=seed + 1, scale=Kd ** -0.5)
    b = rnd(N, seed=seed + 2) if bias else None
    r = (rnd(M, N + 16, seed=seed + 3, scale=4)[:, 8:N + 8] if strided else rnd(M, N, seed=seed + 3, scale=4)) if residual else None
    y, pre = K.linear_act_fwd(x, w, b, act, r, want_pre)
    v = x.double() @ w.double().t()
    size = x.double().abs() @ w.double().abs().t()
    if b is not None:
        v, size = v + b.double(), size + b.double().abs()
    err = size * (2 * (Kd + 4) * EPS)
    if want_pre:
        close(pre, v, err, "pre")
    a, _ = act64(v, act)
    slack = 1.2 * err + a.abs() * 2.0 ** -15
    if r is not None:
        a = a + r.double()
        slack = slack + (a.abs() + r.double().abs()) * EPS
    close(y, a, slack, "y")


# up to 16 rows (a kernel of their own up to K = 6144) at each number of K blocks a wave owns, the smallest, odd ones, and every tile shape, whole and
# split, with and without a K tail (asked for below)
ROWS = [(1, 8, 8), (1, 11008, 4096), (8, 264, 1000), (16, 16, 512), (16, 24, 520), (5, 520, 1032), (3, 16384, 64), (16, 4104, 1544), (2, 72, 2560), (7, 1000, 3080),
        (9, 8200, 4104), (16, 520, 5128), (15, 4096, 6144), (16, 520, 6152), (16, 32776, 72)]
SHAPES = ROWS + [(17, 72, 4104), (64, 64, 64), (100, 520, 688), (389, 520, 256), (1000, 1032, 776), (389, 520, 1024),
          (389, 520, 4096), (389, 5120, 256), (389, 5120, 776), (600, 2048, 4096), (389, 5120, 1024), (389, 8192, 776), (1000, 1032, 4096), (4104, 2048, 256),
          (600, 5120, 4096), (1000, 5504, 1024), (1000, 5504, 776), (389, 2752, 4096), (4000, 8192, 256), (4000, 8192, 776), (2500, 5120, 256), (4104, 2048, 776),
          (389, 5120, 11008), (4096, 4096, 4096)]


def test_the_sizes_reach_every_tile_shape():
    from easyllm_amd import _lib
    seen = {(p[1], p[2], p[3] > 1, p[4]) for p in (_lib.gemm_plan("forward", [M], [N], Kd) for M, N, Kd in SHAPES)}
    assert {(rows, cols, split, 4) for rows, cols in ((256, 256), (192, 256), (256, 128), (192, 128), (128, 128), (64, 64)) for split in (False, True)} <= seen, seen
    assert {(64, 64, False, 8), (256, 256, False, 8)} <= seen, seen


@pytest.mark.parametrize("M,N,Kd", SHAPES)
@pytest.mark.parametrize("act", ["none", "gelu", "gelu_tanh"])
def test_forward(K, M, N, Kd, act):
    print("linear_act", M, N, Kd, act, flush=True)
    check_forward(K, M, N, Kd, act, True, True)


@pytest.mark.parametrize("bias,residual,want_pre", [(False, False, False), (True, False, False), (False, True, False), (False, False, True)])
@pytest.mark.parametrize("M,N,Kd", [(5, 64, 72), (300, 520, 1000), (2048, 4096, 4096), (1000, 8200, 2048)])
def test_forward_without_some_of_it(K, M, N, Kd, bias, residual, want_pre):
    print("linear_act", M, N, Kd, bias, residual, want_pre, flush=True)
    check_forward(K, M, N, Kd, "gelu", bias, residual, want_pre=want_pre)


@pytest.mark.parametrize("M,N,Kd", [(3, 264, 64), (16, 4104, 1000), (300, 520, 1000), (1100, 4096, 4096)])
def test_forward_of_strided_rows(K, M, N, Kd):
    print("strided", M, N, Kd, flush=True)
    check_forward(K, M, N, Kd, "gelu_tanh", True, True, strided=True)


def test_nothing_is_written_past_the_results_edges(K):
    """Rows and columns next to a result that is a part of a larger buffer stay as they are (through the C ABI: row strides of its own)."""
    import ctypes
    from easyllm_amd import _lib
    for M, N, Kd in ((5, 72, 136), (16, 8200, 4096), (70, 72, 128), (300, 520, 1000), (1000, 4104, 4096)):
        x, w, b = rnd(M, Kd, seed=1), rnd(N, Kd, seed=2), rnd(N, seed=3)
        full = torch.full((2, M + 300, N + 24), 77.0, dtype=torch.bfloat16, device="cuda")
        res = full[0].clone()
        y, pre = full[0, :M, 8:N + 8], full[1, :M, 8:N + 8]
        e = _lib.Epilogue(b.data_ptr(), res[:M, 8:N + 8].data_ptr(), pre.data_ptr(), N + 24, N + 24, 1)
        size = _lib.gemm_workspace_bytes(M, N, Kd)
        ws = torch.empty(size, dtype=torch.uint8, device="cuda")
        _lib.call("ezl_gemm_bf16_epilogue", x.data_ptr(), w.data_ptr(), y.data_ptr(), M, N, Kd, Kd, Kd, N + 24, ctypes.byref(e), ws.data_ptr(), size, None)
        torch.cuda.synchronize()
        want, want_pre = K.linear_act_fwd(x, w, b, "gelu", res[:M, 8:N + 8].contiguous(), True)
        assert torch.equal(y, want) and torch.equal(pre, want_pre)
        y.fill_(77)
        pre.fill_(77)
        assert (full == 77).all()


def test_the_residual_may_be_the_result(K):
    import ctypes
    from easyllm_amd import _lib
    for M, N, Kd in ((9, 4104, 1000), (70, 72, 128), (1000, 1032, 776), (2048, 4096, 4096), (1531, 4096, 11008)):
        x, w, r = rnd(M, Kd, seed=1), rnd(N, Kd, seed=2), rnd(M, N, seed=3)
        want, _ = K.linear_act_fwd(x, w, None, "none", r)
        size = _lib.gemm_workspace_bytes(M, N, Kd)
        ws = torch.empty(size, dtype=torch.uint8, device="cuda")
        _lib.call("ezl_gemm_bf16_epilogue", x.data_ptr(), w.data_ptr(), r.data_ptr(), M, N, Kd, Kd, Kd, N, ctypes.byref(_lib.Epilogue(None, r.data_ptr(), None, N, 0, 0)),
                  ws.data_ptr(), size, None)
        assert torch.equal(r, want)


def test_activations_over_their_whole_range(K):
    """Every bf16 value up to the largest, through an identity product; slopes from the backward kernel."""
    v = torch.arange(-2 ** 15, 2 ** 15, dtype=torch.int32, device="cuda").to(torch.int16).view(torch.bfloat16)
    v = v[torch.isfinite(v)]
    v = torch.cat([v, v[:(-v.numel()) % 64]]).view(-1, 64)
    eye = torch.eye(64, dtype=torch.bfloat16, device="cuda")
    for act in ("gelu", "gelu_tanh"):
        y, pre = K.linear_act_fwd(v, eye, None, act, None, True)
        assert torch.equal(pre, v)
        ref, _ = act64(v.double(), act)
        ref = torch.where(torch.isnan(ref), v.double().clamp(min=0), ref)
        # tails below 2^-100 and exponentials of arguments beyond 100 may come out as zero
        close(y, ref, ref.abs() * 2.0 ** -14 + 2.0 ** -100, act)
        d = K.act_bwd(act, torch.ones_like(v), v)
        slope = act64(v.double().clamp(-200, 200), act)[1]
        close(d, slope, 2.0 ** -18 + slope.abs() * 2.0 ** -14, act + " slope")


def test_what_is_not_finite_stays_in_its_place(K):
    """An infinity in a weight or an input reaches the results it is part of, as itself, and no other; rows and columns and k past the operands' ends count for nothing."""
    for M, N, Kd in ((5, 40, 72), (16, 520, 1000), (40, 72, 72), (300, 520, 1000)):
        x, w = rnd(M, Kd, seed=1).abs() + 1, rnd(N, Kd, seed=2).abs() + 1
        w[N - 1, 0] = float("inf")
        x[M - 1, Kd - 1] = float("nan")
        y, _ = K.linear_act_fwd(x, w, None, "gelu", None)
        want = torch.full((M, N), False, device="cuda")
        want[:, N - 1] = True
        want[M - 1] = True
        assert torch.equal(~torch.isfinite(y), want) and (y[:M - 1, N - 1] == float("inf")).all() and torch.isnan(y[M - 1]).all()


def test_slopes_against_differences(K):
    v = torch.linspace(-6, 6, 4096, device="cuda").bfloat16().view(8, 512)
    for act in ("gelu", "gelu_tanh"):
        d = K.act_bwd(act, torch.ones_like(v), v).double()
        h = 1e-4
        num = (act64(v.double() + h, act)[0] - act64(v.double() - h, act)[0]) / (2 * h)
        close(d, num, 1e-6 + 2.0 ** -14 * num.abs(), act)


@pytest.mark.parametrize("rows,n", [(1, 8), (3, 520), (1167, 1000), (130, 11008)])
@pytest.mark.parametrize("act", ["gelu", "gelu_tanh"])
def test_activation_backward(K, rows, n, act):
    dy, pre = rnd(rows, n, seed=1), rnd(rows, n, seed=2, scale=2)
    ref = dy.double() * act64(pre.double(), act)[1]
    slack = dy.double().abs() * 2.0 ** -15
    buf, grad = torch.full((n,), 5.0, device="cuda"), torch.empty(n, dtype=torch.bfloat16, device="cuda")
    for target in (None, (buf, None, True), (None, grad, False)):
        close(K.act_bwd(act, dy, pre, target), ref, slack, "dpre")
    sums = slack.sum(0) + ref.abs().sum(0) * (rows + 8) * EPS
    assert ((buf.double() - 5 - ref.sum(0)).abs() <= sums + (5 + ref.sum(0).abs()) * EPS).all()
    close(grad, ref.sum(0), sums, "dbias")
    empty = torch.empty(0, n, dtype=torch.bfloat16, device="cuda")
    K.act_bwd(act, empty, empty, (None, grad, False))
    assert not grad.any()


@pytest.mark.parametrize("act", ["none", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("bias,residual", [(True, True), (False, False)])
def test_gradients_through_the_public_call(F, act, bias, residual):
    s, b, n_in, n = 41, 3, 520, 776
    x = rnd(b, s, n_in, seed=1).transpose(0, 1).requires_grad_(True)
    w = rnd(n, n_in, seed=2, scale=n_in ** -0.5).requires_grad_(True)
    bi = rnd(n, seed=3).requires_grad_(True) if bias else None
    r = rnd(s, b, n, seed=4).requires_grad_(True) if residual else None
    y = F.linear_act(x, w, bi, act, r)
    dy = rnd(s, b, n, seed=5)
    leaves = [t for t in (x, w, bi, r) if t is not None]
    got = dict(zip([k for k, t in zip("xwbr", (x, w, bi, r)) if t is not None], torch.autograd.grad(y, leaves, dy)))
    xd, wd, dyd = x.detach().reshape(-1, n_in).double(), w.detach().double(), dy.reshape(-1, n).double()
    v = xd @ wd.t() + (bi.detach().double() if bias else 0)
    close(y.detach().reshape(-1, n), act64(v, act)[0] + (r.detach().reshape(-1, n).double() if residual else 0), 1e-3, "y")
    slope = act64(v, act)[1]
    d = dyd * slope
    # what goes into the products: dy times the slope at v rounded to bf16 (|act''| < 1.13), rounded itself
    off = d.abs() * 2.0 ** -8 + (dyd.abs() * 1.13 * (v.abs() * 2.0 ** -8 + 1e-3) if act != "none" else 0)
    close(got["x"].reshape(-1, n_in), d @ wd, off @ wd.abs() + d.abs() @ wd.abs() * (n * 2 * EPS), "dx")
    close(got["w"], d.t() @ xd, off.t() @ xd.abs() + d.abs().t() @ xd.abs() * (s * b * 2 * EPS), "dw")
    if bias:
        close(got["b"], d.sum(0), off.sum(0) + d.abs().sum(0) * s * b * EPS, "dbias")
    if residual:
        assert torch.equal(got["r"], dy)


def test_residuals_of_other_layouts(F):
    x, w = rnd(40, 64, seed=1), rnd(72, 64, seed=2)
    for r in (rnd(72, seed=3).expand(40, 72), rnd(72, 40, seed=3).t(), rnd(40, 144, seed=3)[:, ::2]):
        assert torch.equal(F.linear_act(x, w, None, "gelu", r), F.linear_act(x, w, None, "gelu", r.contiguous()))


def test_main_grads_and_frozen_parameters(F):
    x, w, b = rnd(50, 64, seed=1).requires_grad_(True), rnd(72, 64, seed=2).requires_grad_(True), rnd(72, seed=3).requires_grad_(True)
    dy = rnd(50, 72, seed=4)
    plain = torch.autograd.grad(F.linear_act(x, w, b, "gelu"), (x, w, b), dy)
    for p in (w, b):
        p.main_grad, p.main_grad_fresh = torch.full(p.shape, 3.0, device="cuda"), True
    for times in (1, 2):
        F.linear_act(x, w, b, "gelu").backward(dy)
        for p, g in zip((w, b), plain[1:]):
            assert torch.allclose(p.main_grad, times * g.float(), rtol=2 ** -7, atol=2 ** -7) and p.grad is None
    w.requires_grad_(False)
    kept = w.main_grad.clone()
    x.grad = None
    F.linear_act(x, w, b, "gelu").backward(dy)
    assert torch.equal(w.main_grad, kept) and torch.equal(x.grad, plain[0])
    with torch.no_grad():
        assert torch.equal(F.linear_act(x, w, b, "gelu"), F.linear_act(x, w, b, "gelu").detach())


def test_the_wrappers_refuse(F):
    x, w = rnd(4, 64), rnd(72, 64)
    for bad in (lambda: F.linear_act(x, w, activation="relu"), lambda: F.linear_act(x.float(), w), lambda: F.linear_act(x, rnd(72, 72)), lambda: F.linear_act(x, rnd(76, 64)),
                lambda: F.linear_act(x, w, rnd(64)), lambda: F.linear_act(x, w, residual=rnd(4, 64)), lambda: F.linear_act(x, w, residual=rnd(72)),
                lambda: F.linear_act(x.cpu(), w.cpu())):
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            bad()


def test_an_empty_batch(F):
    x, w, b, r = (rnd(*s, seed=i).requires_grad_(True) for i, s in enumerate(((0, 64), (72, 64), (72,), (0, 72))))
    for act in (None, "gelu"):
        y = F.linear_act(x, w, b, act, r)
        got = torch.autograd.grad(y, (x, w, b, r), torch.empty_like(y))
        assert y.shape == (0, 72) and [g.shape for g in got] == [t.shape for t in (x, w, b, r)] and not got[1].any() and not got[2].any()


def test_a_captured_product_on_another_stream(F):
    x, w, b, r = rnd(300, 4096, seed=1).requires_grad_(True), rnd(1032, 4096, seed=2).requires_grad_(True), rnd(1032, seed=3).requires_grad_(True), rnd(300, 1032, seed=4)
    dy = rnd(300, 1032, seed=5)

    def call():
        y = F.linear_act(x, w, b, "gelu", r)
        return (y.detach(),) + torch.autograd.grad(y, (x, w, b), dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = call()
    for i in range(3):
        with torch.no_grad():
            x.copy_(rnd(300, 4096, seed=10 + i))
        graph.replay()
        torch.cuda.synchronize()
        for a, e in zip(outs, call()):
            assert torch.equal(a, e), i
