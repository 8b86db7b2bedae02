"""act(x gate^T) * (x up^T), times down^T, forward and backward, against 64-bit arithmetic.

Tolerances, before any run.  E = 2^-24.  A sum of K products of bf16 values is off by at most 2 (K + 4) E times the sum of their magnitudes ("size").  An activation's slope is
below 1.13 and its second derivative below 1.2 (ReLU's jumps: gates within their error of zero are left out by taking the larger of both slopes), its own arithmetic adds 2^-15 of its value.
Roundings to bf16 are 2^-8 of a value: of the products between the launches, of the results.  gate and up, where the backward pass reads them, have 12 bits of mantissa: 2^-12."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
E, H, KEPT = 2.0 ** -24, 2.0 ** -8, 2.0 ** -12


@pytest.fixture(scope="module")
def F():
    from easyllm_amd import functional
    return functional


def rnd(*shape, seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).bfloat16()


def act64(a, act):
    """act(a), act'(a) in fp64"""
    if act == "silu":
        s = torch.sigmoid(a)
        return a * s, s * (1 + a * (1 - s))
    if act == "gelu":
        cdf = 0.5 * torch.special.erfc(-a / math.sqrt(2))
        return a * cdf, cdf + a * torch.exp(-0.5 * a * a) / math.sqrt(2 * math.pi)
    if act == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        s = torch.sigmoid(2 * c * (a + 0.044715 * a ** 3))
        return a * s, s + a * s * (1 - s) * 2 * c * (1 + 3 * 0.044715 * a * a)
    return a.clamp_min(0), (a > 0).double()


def near(got, ref, slack, what):
    off = (got.double() - ref).abs() - ref.abs() * H - slack * (1 + H)
    assert got.shape == ref.shape and bool((off <= 0).all()), "%s: %g beyond its tolerance" % (what, off.max().item())


def product(a, a_err, b, b_err=None):
    """a b in fp64, and how far a product in fp32 of values that far off may be from it"""
    k = a.shape[1]
    err = a_err @ b.abs() if a_err is not None else 0
    if b_err is not None:
        err = err + (a.abs() + (0 if a_err is None else a_err)) @ b_err
    return a @ b, err + (a.abs() @ b.abs()) * (2 * (k + 4) * E)


def kept_values(kept, T, f, rows=slice(None)):
    """the two products of what K.gated_fwd kept, in fp64"""
    rows = torch.arange(T, device="cuda")[rows]
    blocks = kept.view((T + 15) // 16, (f + 31) // 32, 2560)[rows // 16]
    place = torch.tensor([16 * (c // 2 + 2 * (c % 2)) for c in range(4)], device="cuda") + (rows % 16)[:, None]  # [row, eight columns of a block's 32]
    here = torch.arange(len(rows), device="cuda")[:, None]
    of = lambda part: part.unflatten(-1, (64, 8)).transpose(1, 2)[here, place].transpose(1, 2).reshape(len(rows), -1)[:, :f]  # noqa: E731
    gate, up = (of(blocks[..., 1024 * i:1024 * (i + 1)].contiguous().view(torch.int16)) for i in range(2))
    low = of(blocks[..., 2048:]).int()
    bits = lambda upper, last: (upper.int() << 16 | last << 12).view(torch.float32).double()  # noqa: E731
    return bits(gate, low & 15), bits(up, low >> 4)


def expected(x, wg, wu, wd, dy, act):
    """name -> (reference, slack)"""
    x, wg, wu, wd = (t.detach().double() for t in (x, wg, wu, wd))
    (g, g_err), (u, u_err) = product(x, None, wg.t()), product(x, None, wu.t())
    a, slope = act64(g, act)
    mid = a * u

    def middle(g1, u1):
        """what act(g) and mid, rounded, are off by where g and u are off by g1 and u1"""
        a_err = 1.2 * g1 + a.abs() * 2.0 ** -15
        err = a_err * u.abs() + (a.abs() + a_err) * u1
        return a_err, err + (mid.abs() + err) * H

    out = {"y": product(mid, middle(g_err, u_err)[1], wd.t())}
    g1, u1 = g_err + (g.abs() + g_err) * KEPT, u_err + (u.abs() + u_err) * KEPT  # (as the backward pass reads them)
    a_err, mid_err = middle(g1, u1)
    if dy is not None:
        dy = dy.double()
        d, d_err = product(dy, None, wd)
        slope_err = 1.2 * g1 + slope.abs() * 2.0 ** -15
        if act == "relu":
            slope_err = slope_err * 0 + (g.abs() <= g1)
        du = d * a
        du_err = d_err * a.abs() + (d.abs() + d_err) * a_err
        du_err = du_err + (du.abs() + du_err) * H
        dg = d * u * slope
        dg_err = d_err * (u * slope).abs() + (d.abs() + d_err) * (u1 * slope.abs() + (u.abs() + u1) * slope_err)
        dg_err = dg_err + (dg.abs() + dg_err) * H
        one, two = product(dg, dg_err, wg), product(du, du_err, wu)
        out.update(x=(one[0] + two[0], one[1] + two[1]), gate=product(dg.t(), dg_err.t(), x), up=product(du.t(), du_err.t(), x),
                   down=product(dy.t(), None, mid, mid_err))
    return out


def check(F, T, h, f, act, h_out=None, seed=0, train=True, shape=None):
    h_out = h_out or h
    x = rnd(T, h, seed=seed).view(*(shape or (T,)), h).requires_grad_(train)
    wg, wu = (rnd(f, h, seed=seed + 1 + i, scale=1.5 * h ** -0.5).requires_grad_(train) for i in range(2))
    wd = rnd(h_out, f, seed=seed + 3, scale=f ** -0.5).requires_grad_(train)
    dy = rnd(T, h_out, seed=seed + 4) if train else None
    with torch.set_grad_enabled(train):
        y = F.gated_mlp(x, wg, wu, wd, activation=act)
    assert y.shape == (*x.shape[:-1], h_out)
    want = expected(x.reshape(-1, h), wg, wu, wd, dy, act)
    near(y.reshape(-1, h_out), *want["y"], "y")
    if train:
        grads = torch.autograd.grad(y, (x, wg, wu, wd), dy.view(y.shape))
        for name, g in zip(("x", "gate", "up", "down"), grads):
            near(g.reshape(want[name][0].shape), *want[name], name)


SMALL = [(1, 8, 8), (1, 64, 64), (2, 256, 688), (5, 1000, 24), (8, 512, 1368), (16, 264, 1000), (17, 72, 520), (33, 128, 16), (64, 64, 136), (100, 520, 264), (257, 768, 2048),
         (389, 256, 688), (389, 1032, 2776), (300, 72, 1048), (1000, 776, 1032)]
# the other tile shapes, whole and split, either way (asked for below); the last of them with a down projection to another width
LARGE = [(513, 4096, 1024, 4096), (389, 4096, 512, 4096), (600, 4096, 1024, 4096), (1000, 1024, 2752, 1024), (4104, 256, 1024, 256), (389, 4096, 2560, 4096), (600, 4096, 2560, 4096),
         (1531, 4096, 5504, 4096), (4000, 264, 4096, 264), (4096, 1024, 4104, 1032), (2500, 520, 4104, 520), (389, 256, 2560, 8192), (1300, 256, 2560, 4096), (1000, 256, 3136, 8192),
         (4096, 64, 2048, 64), (1024, 256, 5504, 2048)]


def test_the_sizes_reach_every_tile_shape():
    from easyllm_amd import _lib
    plan = lambda form, T, n, k: _lib.gemm_plan(form, [T], [n], k)[1:]  # noqa: E731
    ways = [(*s, s[1]) for s in SMALL] + LARGE
    fwd = {(p[0], p[1], p[2] > 1, p[0] == 64 and p[3]) for p in (plan("forward", T, (f + 15) // 16 * 32, h) for T, h, f, _ in ways)}
    bwd = {(p[0], p[1], p[2] > 1, p[0] == 64 and p[3]) for p in (plan("input gradient", T, f, h_out) for T, _, f, h_out in ways)}
    every = {(rows, cols, split, rows == 64 and 4) for rows, cols in ((256, 256), (192, 256), (256, 128), (192, 128), (128, 128), (64, 64)) for split in (False, True)} | {(64, 64, False, 8)}
    assert every <= fwd, every - fwd
    assert every <= bwd, every - bwd


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh", "relu"])
@pytest.mark.parametrize("T,h,f,h_out", LARGE)
def test_every_tile_shape(F, T, h, f, h_out, act):
    print("gated", T, h, f, h_out, act, flush=True)
    check(F, T, h, f, act, h_out=h_out)


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh", "relu"])
@pytest.mark.parametrize("T,h,f", SMALL)
def test_forward_and_backward(F, T, h, f, act):
    print("gated", T, h, f, act, flush=True)
    check(F, T, h, f, act)


@pytest.mark.parametrize("T,h,f", [(1, 8, 8), (5, 264, 1000), (8, 4096, 264), (17, 72, 520), (100, 520, 264), (257, 4096, 2048), (389, 4096, 512), (2500, 520, 4104), (4096, 1024, 4104)])
def test_what_is_kept_has_12_bits(F, T, h, f):
    """Either product within its own error and half a step of 12 bits, and not biased; infinities stay infinities."""
    from easyllm_amd import kernels as K
    x, wg, wu = rnd(T, h), rnd(f, h, seed=1, scale=h ** -0.5), rnd(f, h, seed=2, scale=h ** -0.5)
    mid, kept = K.gated_fwd("silu", x, wg, wu, True)
    alone, nothing = K.gated_fwd("silu", x, wg, wu)
    assert nothing is None and torch.equal(mid, alone)
    for got, w in zip(kept_values(kept, T, f), (wg, wu)):
        ref, err = product(x.double(), None, w.double().t())
        assert bool(((got - ref).abs() <= err + (ref.abs() + err) * KEPT).all())
        # an error's mean over n values, each at most KEPT of its own and even about zero, lies within 6 KEPT |ref| / sqrt(n) of zero but for one in 10^8 (what the sums' own bias adds: err)
        assert abs(float((got.abs() - ref.abs()).sum())) <= 6 * KEPT * float(ref.norm()) + float(err.sum())
    x[0, 0] = float("inf")
    gate, up = kept_values(K.gated_fwd("silu", x, wg, wu, True)[1], T, f)
    assert bool((gate[0].abs() == float("inf")).all()) and bool((up[0] == wu[:, 0].double().sign() * float("inf")).all())


@pytest.mark.parametrize("T,h,f,h_out", [(1, 4096, 11008, 4096), (4, 5120, 13696, 5120), (16, 4096, 4096, 1024), (40, 2048, 5504, 512), (1531, 1024, 2816, 1024)])
def test_forward_alone(F, T, h, f, h_out):
    print("gated", T, h, f, h_out, flush=True)
    for act in ("silu", "gelu"):
        check(F, T, h, f, act, h_out=h_out, train=False)


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh", "relu"])
@pytest.mark.parametrize("T,h,f", [(1, 8, 8), (100, 520, 264), (389, 256, 688), (2500, 520, 4104)])
def test_the_gate_alone(F, T, h, f, act):
    print("gated linear", T, h, f, act, flush=True)
    x = rnd(T, h).requires_grad_()
    wg, wu = (rnd(f, h, seed=1 + i, scale=1.5 * h ** -0.5).requires_grad_() for i in range(2))
    dmid = rnd(T, f, seed=4)
    mid = F.gated_linear(x, wg, wu, activation=act)
    (g, g_err), (u, u_err) = product(x.double(), None, wg.double().t()), product(x.double(), None, wu.double().t())
    (g, g_err, u, u_err) = (t.detach() for t in (g, g_err, u, u_err))
    a, slope = act64(g, act)
    a_err = 1.2 * g_err + a.abs() * 2.0 ** -15
    near(mid, a * u, a_err * u.abs() + (a.abs() + a_err) * u_err, "mid")
    got = torch.autograd.grad(mid, (x, wg, wu), dmid)
    g1, u1, d = g_err + (g.abs() + g_err) * KEPT, u_err + (u.abs() + u_err) * KEPT, dmid.double()
    a_err, slope_err = 1.2 * g1 + a.abs() * 2.0 ** -15, 1.2 * g1 + slope.abs() * 2.0 ** -15
    if act == "relu":
        slope_err = (g.abs() <= g1).double()
    du, dg = d * a, d * u * slope
    du_err = d.abs() * a_err
    dg_err = d.abs() * (u1 * slope.abs() + (u.abs() + u1) * slope_err)
    du_err, dg_err = du_err + (du.abs() + du_err) * H, dg_err + (dg.abs() + dg_err) * H
    xd, wgd, wud = (t.detach().double() for t in (x, wg, wu))
    one, two = product(dg, dg_err, wgd), product(du, du_err, wud)
    for name, t, (ref, slack) in (("x", got[0], (one[0] + two[0], one[1] + two[1])), ("gate", got[1], product(dg.t(), dg_err.t(), xd)), ("up", got[2], product(du.t(), du_err.t(), xd))):
        near(t, ref, slack, name)


def test_shapes_around_the_rows(F):
    check(F, 6 * 35, 64, 80, "silu", shape=(6, 35))
    check(F, 30, 64, 80, "silu", shape=(2, 3, 5))
    x = rnd(0, 4, 64).requires_grad_()
    ws = [rnd(80, 64).requires_grad_(), rnd(80, 64).requires_grad_(), rnd(64, 80).requires_grad_()]
    y = F.gated_mlp(x, *ws)
    assert y.shape == (0, 4, 64)
    grads = torch.autograd.grad(y.float().sum(), [x, *ws])
    assert grads[0].shape == x.shape and all(not bool(g.any()) and g.shape == w.shape for g, w in zip(grads[1:], ws))


# up to 8 rows: a kernel of their own for the gate's products, and for the down projection up to rows x width = 48 K (otherwise, and where the tokens do not fit LDS, the tiles)
@pytest.mark.parametrize("T,h,f,h_out", [(1, 8, 8, 8), (3, 24, 40, 16), (8, 4096, 264, 72), (7, 8712, 72, 8), (2, 20488, 136, 24), (1, 72, 8, 4104), (5, 520, 2056, 520), (1, 64, 11008, 4096),
                                        (4, 1032, 11008, 264), (8, 256, 5512, 520), (6, 1024, 8200, 1032), (1, 64, 49160, 16), (8, 9224, 64, 64), (9, 4096, 264, 72)])
@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh", "relu"])
def test_a_handful_of_tokens(F, T, h, f, h_out, act):
    print("gated rows", T, h, f, h_out, act, flush=True)
    check(F, T, h, f, act, h_out=h_out)
    check(F, T, h, f, act, h_out=h_out, train=False, seed=50)


def test_strides_and_views(F):
    """x and the weights as parts of wider tensors (the two first with strides of their own, or not), an output gradient of any layout."""
    T, h, f = 70, 64, 136
    for rows in (T, 5):
        x = rnd(rows, 3 * h, seed=1)[:, h:2 * h].detach().requires_grad_()
        both = rnd(f, 2 * h, seed=2, scale=h ** -0.5)
        wide = rnd(f, 4 * h, seed=3, scale=h ** -0.5)
        down = rnd(h, f + 24, seed=4, scale=f ** -0.5)[:, 16:16 + f].detach().requires_grad_()
        for wg, wu in ((both[:, :h], both[:, h:]), (both[:, :h], wide[:, h:2 * h])):
            wg, wu = wg.detach().requires_grad_(), wu.detach().requires_grad_()
            y = F.gated_mlp(x, wg, wu, down)
            for dy in (rnd(rows, 2 * h, seed=5)[:, h:], rnd(h, rows, seed=6).t(), rnd(1, h, seed=7).expand(rows, h)):
                want = expected(x, wg, wu, down, dy, "silu")
                near(y, *want["y"], "y")
                for name, g in zip(("x", "gate", "up", "down"), torch.autograd.grad(y, (x, wg, wu, down), dy, retain_graph=True)):
                    near(g, *want[name], name)


@pytest.mark.parametrize("leaf", range(4))
def test_one_gradient_alone(F, leaf):
    tensors = [rnd(40, 64), rnd(72, 64, seed=1, scale=0.125), rnd(72, 64, seed=2, scale=0.125), rnd(64, 72, seed=3, scale=0.11)]
    dy = rnd(40, 64, seed=4)
    tensors[leaf].requires_grad_()
    (g,) = torch.autograd.grad(F.gated_mlp(*tensors), [tensors[leaf]], dy)
    near(g, *expected(*tensors, dy, "silu")[("x", "gate", "up", "down")[leaf]], "gradient")
    if leaf < 3:
        (g,) = torch.autograd.grad(F.gated_linear(*tensors[:3]), [tensors[leaf]], rnd(40, 72, seed=5))
        assert g.shape == tensors[leaf].shape


def test_main_grads_accumulate_in_fp32(F):
    """Overwritten where fresh, then added to; one weight in two places is added to twice."""
    x, dy = rnd(300, 64), rnd(300, 64, seed=1)
    ws = [torch.nn.Parameter(w) for w in (rnd(72, 64, seed=2, scale=0.125), rnd(72, 64, seed=3, scale=0.125), rnd(64, 72, seed=4, scale=0.11))]
    want = expected(x, *ws, dy, "gelu")
    for w in ws:
        w.main_grad, w.main_grad_fresh = torch.full(w.shape, 7.0, device="cuda"), True
    for times in (1, 2):
        F.gated_mlp(x, *ws, activation="gelu").backward(dy)
        for name, w in zip(("gate", "up", "down"), ws):
            ref, slack = want[name]
            off = (w.main_grad.double() - times * ref).abs() - times * slack - ref.abs() * 2.0 ** -20
            assert w.grad is None and bool((off <= 0).all()), (name, times, off.max().item())
    tied = torch.nn.Parameter(ws[0].detach().clone())
    tied.main_grad, tied.main_grad_fresh = torch.full(tied.shape, 7.0, device="cuda"), True
    F.gated_mlp(x, tied, tied, ws[2].detach()).backward(dy)
    want = expected(x, tied, tied, ws[2], dy, "silu")
    off = (tied.main_grad.double() - want["gate"][0] - want["up"][0]).abs() - want["gate"][1] - want["up"][1] - 2.0 ** -20 * want["gate"][0].abs()
    assert bool((off <= 0).all())


def test_an_evaluation_keeps_nothing(F):
    x, ws = rnd(40, 64), [rnd(72, 64, seed=1).requires_grad_(), rnd(72, 64, seed=2).requires_grad_(), rnd(64, 72, seed=3).requires_grad_()]
    with torch.no_grad():
        assert F.gated_mlp(x, *ws).grad_fn is None and F.gated_linear(x, *ws[:2]).grad_fn is None
    before = torch.cuda.memory_allocated()
    with torch.no_grad():
        y = F.gated_mlp(x, *ws)
    assert torch.cuda.memory_allocated() - before <= 512 * (1 + y.numel() * 2 // 512)
    with torch.no_grad():
        assert torch.equal(y, F.gated_mlp(x, *ws))
    assert torch.equal(y, F.gated_mlp(x, *ws).detach())


@pytest.mark.parametrize("T", [3, 500])
def test_another_stream_and_captured_steps(F, T):
    x, dy = rnd(T, 264), rnd(T, 264, seed=1)
    ws = [rnd(520, 264, seed=2, scale=0.06), rnd(520, 264, seed=3, scale=0.06), rnd(264, 520, seed=4, scale=0.04)]
    leaves = [t.requires_grad_() for t in (x, *ws)]

    def step():
        y = F.gated_mlp(*leaves)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    del got
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in (5, 6, 7):
        with torch.no_grad():
            x.copy_(rnd(T, 264, seed=seed))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, step()))


def test_results_of_more_than_two_to_the_31_elements(F):
    """Each way, the first and last rows of T x f > 2^31."""
    from easyllm_amd import kernels as K
    T, h, f = (1 << 18) + 24, 64, 8200
    x, dy = rnd(T, h), rnd(T, h, seed=1)
    wg, wu, wd = rnd(f, h, seed=2, scale=0.125), rnd(f, h, seed=3, scale=0.125), rnd(h, f, seed=4, scale=f ** -0.5)
    mid, kept = K.gated_fwd("silu", x, wg, wu, True)
    rows = [*range(3), *range(T - 300, T)]
    g, u = x[rows].double() @ wg.double().t(), x[rows].double() @ wu.double().t()
    g_err, u_err = (2 * (h + 4) * E * (x[rows].double().abs() @ w.double().abs().t()) for w in (wg, wu))
    a, slope = act64(g, "silu")
    for got, ref, err in zip(kept_values(kept, T, f, rows), (g, u), (g_err, u_err)):
        assert bool(((got - ref).abs() <= err + (ref.abs() + err) * KEPT).all())
    near(mid[rows], a * u, (1.2 * g_err + a.abs() * 2.0 ** -15) * (u.abs() + u_err) + a.abs() * u_err, "mid")
    del mid
    y, _ = K.gated_mlp_fwd("silu", x, wg, wu, wd)
    near(y[rows], *expected(x[rows], wg, wu, wd, None, "silu")["y"], "y")
    dx = K.gated_mlp_bwd("silu", dy, x, wg, wu, wd, kept, True, (None, None, None))
    near(dx[rows], *expected(x[rows], wg, wu, wd, dy[rows], "silu")["x"], "dx")


def test_values_that_are_not_finite(F):
    """Infinities and NaN of a token stay in its row."""
    for T in (4, 100):
        x, ws = rnd(T, 64), [rnd(72, 64, seed=1), rnd(72, 64, seed=2), rnd(64, 72, seed=3)]
        want = F.gated_mlp(x, *ws)
        x[1, 5], x[2, 7] = float("inf"), float("nan")
        got = F.gated_mlp(x, *ws)
        keep = [i for i in range(T) if i not in (1, 2)]
        assert torch.equal(got[keep], want[keep]) and bool(got[2].isnan().all()) and not bool(torch.isfinite(got[1]).any())


def test_second_derivatives_are_refused(F):
    x, ws = rnd(8, 64).requires_grad_(), [rnd(72, 64, seed=1), rnd(72, 64, seed=2), rnd(64, 72, seed=3)]
    for y in (F.gated_mlp(x, *ws), F.gated_linear(x, *ws[:2])):
        (dx,) = torch.autograd.grad(y.float().sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="cannot be differentiated twice"):
            dx.float().sum().backward()


def test_refusals(F):
    x, wg, wu, wd = rnd(8, 64), rnd(72, 64), rnd(72, 64), rnd(64, 72)
    for args in ((x.float(), wg, wu, wd), (x, wg.float(), wu, wd), (x, wg, wu.half(), wd), (x, wg, wu, wd.float()), (x, wg, wu[:64], wd), (x[:, :56], wg, wu, wd), (x, wg, wu, wd[:, :64]),
                 (x.cpu(), wg, wu, wd), (x, wg.cpu(), wu.cpu(), wd), (x, rnd(76, 64), rnd(76, 64), rnd(64, 76)), (rnd(8, 60), rnd(72, 60), rnd(72, 60), wd), (x, wg, wu, rnd(60, 72)),
                 (x, wg[:0], wu[:0], wd[:, :0]), (rnd(8, 0), wg[:, :0], wu[:, :0], wd)):
        for leaf in (False, True):
            with pytest.raises((ValueError, RuntimeError)):
                F.gated_mlp(args[0].detach().requires_grad_(leaf), *args[1:])
    for activation in (None, "none", "tanh"):
        with pytest.raises(ValueError, match="activation"):
            F.gated_mlp(x, wg, wu, wd, activation)
        with pytest.raises(ValueError, match="activation"):
            F.gated_linear(x, wg, wu, activation)
    with pytest.raises((ValueError, RuntimeError)):
        F.gated_linear(x, wg, rnd(72, 56))


@pytest.mark.parametrize("T,h,f", [(100, 72, 136), (1024, 256, 688), (1000, 768, 2048), (4000, 1536, 4096), (4100, 1544, 4104)])
def test_weight_gradients_in_one_list(F, T, h, f):
    """All three in fp32 and in bf16, on small tiles and 256 x 256 ones, and where one of them is of the other type (then they are no list)."""
    x, dy = rnd(T, h), rnd(T, h, seed=1)
    weights = [rnd(f, h, seed=2, scale=h ** -0.5), rnd(f, h, seed=3, scale=h ** -0.5), rnd(h, f, seed=4, scale=f ** -0.5)]
    want = expected(x, *weights, dy, "silu")
    for with_main in ((), (0, 1, 2), (2,), (0, 1), (1,)):
        ws = [torch.nn.Parameter(w) for w in weights]
        for i in with_main:
            ws[i].main_grad = torch.full(ws[i].shape, 0.5, device="cuda")
        F.gated_mlp(x, *ws).backward(dy)
        for i, name in enumerate(("gate", "up", "down")):
            ref, slack = want[name]
            if i in with_main:
                assert ws[i].grad is None and bool(((ws[i].main_grad.double() - 0.5 - ref).abs() <= slack + (ref.abs() + 0.5) * 2.0 ** -22).all()), (with_main, name)
            else:
                near(ws[i].grad, ref, slack, name)


@pytest.mark.parametrize("T", [3, 100, 1024])
def test_one_weight_in_all_three_places(F, T):
    """Its gradients are written one behind the other, the first over what is there."""
    n = 256
    x, dy = rnd(T, n), rnd(T, n, seed=1)
    w = torch.nn.Parameter(rnd(n, n, seed=2, scale=n ** -0.5))
    want = expected(x, w, w, w, dy, "silu")
    w.main_grad, w.main_grad_fresh = torch.full(w.shape, 7.0, device="cuda"), True
    F.gated_mlp(x, w, w, w).backward(dy)
    ref, slack = (sum(want[name][i] for name in ("down", "gate", "up")) for i in range(2))
    size = sum(want[name][0].abs() for name in ("down", "gate", "up"))
    assert bool(((w.main_grad.double() - ref).abs() <= slack + size * 2.0 ** -20).all())
    (g,) = torch.autograd.grad(F.gated_mlp(x, u := w.detach().requires_grad_(), u, u), [u], dy)
    assert bool(((g.double() - ref).abs() <= slack + 3 * H * (size + slack) + 2 * H * size).all())  # (three roundings of the parts, two of their sums)
