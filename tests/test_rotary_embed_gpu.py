"""Rotary positions of either pairing against 64-bit arithmetic.

Tolerances, before any run: an angle comes out of 64 bits as a share of a turn in fp32, half of 2^-24 off at most (2 pi 2^-25 = 1.9e-7 of an angle), the hardware's sine and
cosine of it are off by less than 1e-6; products and the sum in fp32 add 3 2^-24 of what they add up.  With |x1| + |x2| = S that is 1.5e-6 S scale, and the
rounding to bf16 half a step, 2^-8 of the result at most."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def F():
    from easyllm_amd import functional
    return functional


def rnd(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").bfloat16()


def frequencies(turned, base=10000.0, dtype=torch.float32):
    j = torch.arange(0, turned, 2, device="cuda", dtype=torch.float64)
    return (base ** (-j / turned)).to(dtype)


def turned64(x, inv_freq, positions, interleaved, scale, back=False):
    """(the result in fp64, the magnitudes that went into it); positions [b, s]"""
    n = 2 * inv_freq.numel()
    angle = (positions.double()[..., None] * inv_freq.double()).transpose(0, 1).unsqueeze(2)
    c, s = torch.cos(angle) * scale, torch.sin(angle) * scale * (-1 if back else 1)
    y, size = x.double().clone(), torch.zeros_like(x, dtype=torch.float64)
    one, two = (slice(0, n, 2), slice(1, n, 2)) if interleaved else (slice(0, n // 2), slice(n // 2, n))
    a, b = x[..., one].double(), x[..., two].double()
    y[..., one], y[..., two] = a * c - b * s, b * c + a * s
    size[..., one] = size[..., two] = (a.abs() + b.abs()) * abs(scale)
    return y, size


def check(got, x, inv_freq, positions, interleaved, scale, back=False):
    ref, size = turned64(x, inv_freq, positions, interleaved, scale, back)
    assert got.shape == x.shape and got.dtype is torch.bfloat16 and got.is_contiguous()
    off = (got.double() - ref).abs() - size * 1.5e-6 - ref.abs() * 2.0 ** -8 * (size > 0)
    assert bool((off <= 0).all()), off.max().item()


SHAPES = [  # s, b, nq, nk, d, turned
    (1, 1, 1, 1, 8, 8), (1, 1, 32, 8, 128, 128), (1, 3, 4, 4, 64, 2), (7, 2, 3, 1, 80, 80), (5, 1, 2, 2, 96, 32), (33, 2, 6, 2, 64, 24), (16, 1, 5, 5, 72, 40),
    (100, 1, 8, 2, 256, 64), (3, 4, 1, 7, 128, 126), (257, 1, 2, 2, 128, 96), (64, 2, 12, 12, 64, 64), (11, 1, 64, 8, 128, 64), (2, 1, 3, 3, 512, 512), (9, 1, 1, 1, 8, 6)]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("s,b,nq,nk,d,turned", SHAPES)
def test_forward_and_backward(F, s, b, nq, nk, d, turned, interleaved):
    print("rotary", s, b, nq, nk, d, turned, interleaved, flush=True)
    q, k = rnd(s, b, nq, d, seed=1).requires_grad_(), rnd(s, b, nk, d, seed=2).requires_grad_()
    inv_freq = frequencies(turned)
    positions = torch.randint(0, 1 << 20, (b, s), device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))
    yq, yk = F.rotary_embed(q, k, inv_freq, positions, interleaved=interleaved, scale=1.25)
    check(yq, q.detach(), inv_freq, positions, interleaved, 1.25)
    check(yk, k.detach(), inv_freq, positions, interleaved, 1.25)
    dq, dk = rnd(s, b, nq, d, seed=4), rnd(s, b, nk, d, seed=5)
    gq, gk = torch.autograd.grad((yq, yk), (q, k), (dq, dk))
    check(gq, dq, inv_freq, positions, interleaved, 1.25, back=True)
    check(gk, dk, inv_freq, positions, interleaved, 1.25, back=True)


def test_a_rotation_alone_and_its_place_in_the_sequence(F):
    q = rnd(37, 2, 3, 64)
    inv_freq = frequencies(64, dtype=torch.float64)
    y, none = F.rotary_embed(q, None, inv_freq)
    assert none is None
    check(y, q, inv_freq, torch.arange(37, device="cuda").expand(2, 37), False, 1.0)


@pytest.mark.parametrize("interleaved", [False, True])
def test_backward_is_the_transpose(F, interleaved):
    """sum of y times dy = sum of x times dx, for a linear map: both sides are rounded, so by sums of 2^-8 of the terms."""
    q, dy = rnd(64, 2, 4, 128, seed=1).requires_grad_(), rnd(64, 2, 4, 128, seed=2)
    y, _ = F.rotary_embed(q, None, frequencies(96), torch.arange(64, device="cuda").expand(2, 64) * 1001, interleaved=interleaved, scale=0.7)
    (dx,) = torch.autograd.grad(y, q, dy)
    left, right = (y.detach().double() * dy.double()).sum(), (q.detach().double() * dx.double()).sum()
    slack = 2.0 ** -8 * ((y.detach().double() * dy.double()).abs().sum() + (q.detach().double() * dx.double()).abs().sum())
    assert abs(left - right) <= slack


def test_strides_of_every_kind(F):
    """A packed projection's parts, heads apart, batches first, a row used by all: read in place, or copied where the kernel cannot."""
    s, b, d, inv_freq = 19, 2, 64, frequencies(64)
    positions = torch.arange(s, device="cuda").expand(b, s) + 5
    packed = rnd(s, b, 10 * d, seed=1)
    views = [packed[..., :6 * d].unflatten(-1, (6, d)), packed[..., 6 * d:8 * d].unflatten(-1, (2, d)), rnd(b, s, 4, d, seed=2).transpose(0, 1),
             rnd(s, b, 4, 2 * d, seed=3)[..., d:], rnd(s, 1, 3, d, seed=4).expand(s, b, 3, d), rnd(s, b, 3, d + 4, seed=5)[..., :d], rnd(s, b, d, 4, seed=6).transpose(2, 3),
             rnd(s, b * 3 * d + 1, seed=7)[:, 1:].unflatten(-1, (b, 3, d))]
    for x in views:
        y, z = F.rotary_embed(x, views[0], inv_freq, positions)
        check(y, x, inv_freq, positions, False, 1.0)
        check(z, views[0], inv_freq, positions, False, 1.0)
    x = views[0].detach().requires_grad_()
    y, _ = F.rotary_embed(x, None, inv_freq, positions)
    for dy in (rnd(b, s, 6, d, seed=8).transpose(0, 1), rnd(s, b, d, 6, seed=9).transpose(2, 3), rnd(1, 1, 1, d, seed=10).expand(s, b, 6, d)):
        (dx,) = torch.autograd.grad(y, x, dy, retain_graph=True)
        check(dx, dy.contiguous(), inv_freq, positions, False, 1.0, back=True)


def test_positions_far_apart_negative_and_shared(F):
    q, inv_freq = rnd(6, 2, 3, 64), frequencies(64)
    for positions in (torch.tensor([[0, 1, 2 ** 26 - 1, 2 ** 26, 12345678, 3], [7, 7, 7, 7, 7, 7]], device="cuda"), torch.tensor([[-1, -5, -100000, 0, 1, 2]], device="cuda").expand(2, 6),
                      torch.arange(12, device="cuda").view(6, 2).t()):
        y, _ = F.rotary_embed(q, None, inv_freq, positions)
        check(y, q, inv_freq, positions, False, 1.0)


def test_the_rest_of_a_head_passes_through_bit_by_bit(F):
    q = rnd(5, 1, 2, 64)
    q[..., 40:] = torch.tensor([float("inf"), float("nan"), -0.0], device="cuda").bfloat16().repeat(8)
    for interleaved in (False, True):
        y, _ = F.rotary_embed(q, None, frequencies(40), interleaved=interleaved)
        assert torch.equal(y[..., 40:].contiguous().view(torch.int16), q[..., 40:].contiguous().view(torch.int16))
        assert bool(torch.isfinite(y[..., :40]).all())


@pytest.mark.parametrize("s,b,nq,nk", [(0, 1, 2, 2), (3, 0, 2, 2), (3, 1, 0, 2), (3, 1, 2, 0), (0, 0, 0, 0)])
def test_nothing_to_turn(F, s, b, nq, nk):
    yq, yk = F.rotary_embed(rnd(s, b, nq, 64), rnd(s, b, nk, 64), frequencies(64))
    assert yq.shape == (s, b, nq, 64) and yk.shape == (s, b, nk, 64)


def test_offsets_beyond_two_to_the_31_elements(F):
    """Rows far apart in a buffer of more than 2^31 elements, and more than 2^31 elements turned."""
    big = torch.zeros(3, 1, (1 << 30) + 8, dtype=torch.bfloat16, device="cuda")
    x = big[..., :2 * 64].unflatten(-1, (2, 64))
    x.copy_(rnd(3, 1, 2, 64))
    positions = torch.tensor([[5, 6, 7]], device="cuda")
    y, _ = F.rotary_embed(x, None, frequencies(64), positions)
    check(y, x, frequencies(64), positions, False, 1.0)
    del big, x, y
    q = torch.zeros((1 << 17) + 3, 1, 128, 128, dtype=torch.bfloat16, device="cuda")
    last = rnd(2, 1, 128, 128, seed=1)
    q[-2:] = last
    y, _ = F.rotary_embed(q, None, frequencies(128))
    check(y[-2:], last, frequencies(128), torch.arange(len(q) - 2, len(q), device="cuda").view(1, 2), False, 1.0)


def test_another_stream_and_a_captured_call(F):
    q, k, inv_freq = rnd(300, 2, 4, 64, seed=1), rnd(300, 2, 2, 64, seed=2), frequencies(48)
    positions = torch.arange(300, device="cuda").expand(2, 300) * 17
    want = F.rotary_embed(q, k, inv_freq, positions, interleaved=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = F.rotary_embed(q, k, inv_freq, positions, interleaved=True)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = F.rotary_embed(q, k, inv_freq, positions, interleaved=True)
    for seed in (3, 4, 5):
        q.copy_(rnd(300, 2, 4, 64, seed=seed))
        positions_now = torch.arange(300, device="cuda").expand(2, 300) * 17
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, F.rotary_embed(q, k, inv_freq, positions_now, interleaved=True)))


def test_refusals(F):
    q, f = rnd(4, 2, 3, 64), frequencies(64)
    pos = torch.zeros(2, 4, dtype=torch.int64, device="cuda")
    for args in ((q.float(), None, f), (q[0], None, f), (q.cpu(), None, f), (q, rnd(4, 2, 3, 128), f), (q, rnd(5, 2, 3, 64), f), (q, None, frequencies(66)), (q, None, f[:0]),
                 (q, None, f.half()), (q, None, f.cpu()), (q, None, f.view(2, 16)), (q, None, f[::2]), (q, None, f, pos.int()), (q, None, f, pos.t()), (q, None, f, pos[:1]),
                 (q, None, f, pos.cpu()), (rnd(4, 2, 3, 60), None, frequencies(40))):
        with pytest.raises((ValueError, RuntimeError)):
            F.rotary_embed(*args)
    with pytest.raises(ValueError, match="not learnt"):
        F.rotary_embed(q, None, f.clone().requires_grad_())


def test_forward_mode_derivatives_are_an_error(F):
    from easyllm_amd import functional
    q, f = rnd(4, 2, 3, 64), frequencies(64)
    w = rnd(72, 64), rnd(72, 64, seed=1), rnd(64, 72, seed=2)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(q, torch.ones_like(q))
        for call in (lambda: F.rotary_embed(dual, None, f), lambda: functional.gated_mlp(dual, *w), lambda: functional.gated_linear(dual, *w[:2])):
            with pytest.raises((RuntimeError, NotImplementedError)):
                call()


def test_rows_that_lie_anywhere(F):
    """Views whose rows do not begin on 16 bytes, and single rows whose strides are of the tensor they were cut from."""
    inv_freq = frequencies(64)
    whole = rnd(1, 1, 1, 129, seed=1)
    for q in (whole[..., :128], whole[..., 1:], whole[0, :, :, 1:].unsqueeze(0), rnd(1 + 5 * 2 * 3 * 128, seed=2)[1:].view(5, 2, 3, 128), rnd(5, 2, 3, 136, seed=3)[..., 4:132],
              rnd(128, 3, 2, 5, seed=4).permute(3, 2, 1, 0)):
        q = q.detach().requires_grad_()
        s, b = q.shape[:2]
        positions = 77 * torch.arange(1, 1 + s * b, device="cuda").view(s, b).t()
        y, _ = F.rotary_embed(q, None, inv_freq, positions)
        check(y, q.detach(), inv_freq, positions, False, 1.0)
        for dy in (rnd(*q.shape, seed=5), rnd(1, 1, 1, 129, seed=6)[..., 1:].expand(q.shape)):
            (dq,) = torch.autograd.grad(y, q, dy, retain_graph=True)
            check(dq, dy, inv_freq, positions, False, 1.0, back=True)
