"""AdamW with 8-bit moments: every code against the definition in numpy, and what the random rounding is for.

Moments need no tolerance: their products and sums are one fp32 operation each here and there, rounded the same way, and codes are integers.  A weight's change d = lr (update + decay p) has
a root, a reciprocal and a product that are off by 2^-23 of themselves at most, in numpy a root and a quotient by half of that, so d by 2^-21 d; then the weight itself may be rounded to the
other side, one step of it: 2^-23 p, and of d, 2^-23 d."""
import numpy as np
import pytest
import torch

import _adam8 as R

pytestmark = pytest.mark.gpu
HOW = dict(lr=3e-3, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.1, seed=0x123456789ABCDEF0)


@pytest.fixture(scope="module")
def O():
    from easyllm_amd import optimizer
    return optimizer




def random_state(n, seed, number=0):
    """Codes and scales of all kinds, master weights, as numpy and GPU tensors"""
    rng = np.random.default_rng(seed)
    b = (n + 255) // 256
    ms = rng.integers(90, 130, b)
    state = {"master": rng.standard_normal(n).astype(np.float32), "exp_avg": rng.integers(0, 256, n).astype(np.uint8), "exp_avg_sq": rng.integers(0, 256, n).astype(np.uint8),
             "exp_avg_scale": ms.astype(np.uint8), "exp_avg_sq_scale": (2 * ms - 126).astype(np.uint8), "number": number}
    return state, {k: v if k == "number" else torch.from_numpy(v.copy()).cuda() for k, v in state.items()}


def gradient(n, seed):
    rng = np.random.default_rng(seed)
    g = (rng.standard_normal(n) * np.exp(2 * rng.standard_normal(n) - 6)).astype(np.float32)
    g[rng.random(n) < 0.05] = 0
    return g


def same(state, gpu, before, weight=None, between=()):
    """between: what a weight was behind the earlier ones of several steps, each of which adds what it may be off by (and shrinks what it is given by 1 - lr decay)"""
    for name in ("exp_avg_scale", "exp_avg_sq_scale", "exp_avg", "exp_avg_sq"):
        got, want = gpu[name].cpu().numpy(), state[name]
        assert np.array_equal(got, want), (name, np.flatnonzero(got != want)[:5], got[got != want][:5], want[got != want][:5])
    got, want = gpu["master"].cpu().numpy().reshape(-1).astype(np.float64), state["master"].astype(np.float64)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    off = np.abs(got - want)
    for old, new in zip((before, *between), (*between, want)):
        off -= np.abs(new - old) * (2.0 ** -21 + 2.0 ** -23) + np.abs(new) * 2.0 ** -23
    assert not bool((off > 0).any()), np.nanmax(off)
    state["master"][:] = gpu["master"].cpu().numpy().reshape(-1)  # (the next step starts from the same)
    if weight is not None:
        assert torch.equal(weight.view(-1).float().nan_to_num(1e9), gpu["master"].view(-1).bfloat16().float().nan_to_num(1e9))


@pytest.mark.parametrize("n", [1, 3, 4, 255, 256, 257, 511, 513, 1000, 4095, 4096, 4097, 8191, 12288 + 700, 100003])
def test_every_size(O, n):
    print("adam8", n, flush=True)
    state, gpu = random_state(n, n, number=7)
    weight = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    for k in (1, 2, 1000):
        g = gradient(n, n + k)
        before = state["master"].astype(np.float64)
        R.step(state, g, dict(HOW, step=k))
        O.adamw_8bit_step([gpu], [torch.from_numpy(g).cuda()], [weight], step=k, **HOW)
        same(state, gpu, before, weight)


def test_a_list_of_tensors_is_each_by_itself(O):
    """More tensors than a launch takes, sizes of all kinds, empty ones, without a bf16 weight, one that shares its memory with another."""
    sizes = [0, 1, 300, 5000, 256, 4096, 70000, 0, 9] + list(range(100, 160)) + [20000]
    pairs = [random_state(n, i, number=i) for i, n in enumerate(sizes)]
    grads = [gradient(n, 100 + i) for i, n in enumerate(sizes)]
    weights = [None if i % 3 == 0 else torch.zeros(n, dtype=torch.bfloat16, device="cuda") for i, n in enumerate(sizes)]
    gpu = [g for _, g in pairs] + [pairs[3][1]]
    grads.append(gradient(5000, 999))
    coef = torch.tensor([77.0, 0.5], device="cuda")
    O.adamw_8bit_step(gpu, [torch.from_numpy(g).cuda() for g in grads], weights + [None], step=3, norm_coef=coef, bias_correction=False, **HOW)
    before = [state["master"].astype(np.float64) for state, _ in pairs]
    for (state, _), g in zip(pairs, grads):
        R.step(state, g, dict(HOW, step=3, bias_correction=False), np.float32(0.5))
    between = pairs[3][0]["master"].astype(np.float64)
    R.step(pairs[3][0], grads[-1], dict(HOW, step=3, bias_correction=False), np.float32(0.5))
    for i, (state, g) in enumerate(pairs):
        same(state, g, before[i], weights[i] if i != 3 else None, (between,) if i == 3 else ())


def test_moments_as_values(O):
    states = [random_state(n, n) for n in (1, 255, 256, 257, 5000, 0, 4096, 12345)]
    for (state, gpu), (m, v) in zip(states, O.moments_8bit([g for _, g in states])):
        assert m.dtype is v.dtype is torch.bfloat16
        assert np.array_equal(m.double().cpu().numpy(), R.values(state["exp_avg"], state["exp_avg_scale"], 15, 7))
        assert np.array_equal(v.double().cpu().numpy(), R.values(state["exp_avg_sq"], state["exp_avg_sq_scale"], 31, 8))
    _, gpu = random_state(600, 1)
    gpu["master"] = gpu["master"].view(20, 30)
    assert O.moments_8bit([gpu])[0][0].shape == (20, 30)


def test_every_code_and_scale_as_a_value(O):
    """All codes in blocks of all scales, the lowest (where bf16 has fewer bits: values below 2^-130 are rounded to its multiples of 2^-133) and 255 (not a number)."""
    codes = np.tile(np.arange(256, dtype=np.uint8), 256)
    scales = np.arange(256, dtype=np.uint8)
    gpu = {"master": torch.zeros(65536, device="cuda"), "number": 0, "exp_avg": torch.from_numpy(codes).cuda(), "exp_avg_sq": torch.from_numpy(codes).cuda(),
           "exp_avg_scale": torch.from_numpy(scales).cuda(), "exp_avg_sq_scale": torch.from_numpy(scales).cuda()}
    (m, v), = O.moments_8bit([gpu])
    for got, top, bits in ((m, 15, 7), (v, 31, 8)):
        want = R.values(codes, scales, top, bits)
        got = got.double().cpu().numpy()
        assert np.array_equal(np.isnan(got), np.isnan(want))
        large = np.abs(want) >= 2.0 ** -126
        assert np.array_equal(got[large], want[large])
        assert np.nanmax(np.abs(got - want)[~large]) <= 2.0 ** -134


def test_values_that_are_not_finite_stay_visible(O):
    n = 1024
    state, gpu = random_state(n, 5)
    g = gradient(n, 6)
    g[10], g[300], g[1000] = np.inf, np.nan, 3e38
    weight = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    before = state["master"].astype(np.float64)
    R.step(state, g, dict(HOW, step=2))
    O.adamw_8bit_step([gpu], [torch.from_numpy(g).cuda()], [weight], step=2, **HOW)
    same(state, gpu, before, weight)
    assert list(state["exp_avg_sq_scale"]) [0] == 255 and state["exp_avg_sq_scale"][1] == 255 and state["exp_avg_scale"][2] != 255
    m, v = O.moments_8bit([gpu])[0]
    assert bool(m[:512].isnan().all()) and bool(v[:512].isnan().all()) and not bool(m[512:768].isnan().any())


def test_zero_gradients_leave_zero_moments_and_weights(O):
    gpu = O.new_8bit_state(torch.full((700,), 2.0, device="cuda").bfloat16(), 0)
    O.adamw_8bit_step([gpu], [torch.zeros(700, device="cuda")], [None], lr=1e-2, step=1)
    assert bool((gpu["master"] == 2).all()) and not bool(gpu["exp_avg"].any()) and not bool(gpu["exp_avg_sq"].any())


def test_moments_are_right_on_average(O):
    """What 16-bit random numbers make of a moment: its mean over n seeds is off from the fp32 value by up to 2^-17 of a code's step (of their resolution; half a step of 2^-16)
    and by chance.  The chance: a rounded value is one of two a step apart, its deviation half a step at most, so the mean's over n = 512 is step / (2 sqrt n), and six of those are not seen
    by 1024 values (2e-9 each)."""
    n, seeds = 1024, 512
    state, _ = random_state(n, 3)
    g = gradient(n, 4)
    m, v = R.step({k: v.copy() if k != "number" else v for k, v in state.items()}, g, dict(HOW, step=5))
    total_m, total_v = torch.zeros(n, dtype=torch.float64, device="cuda"), torch.zeros(n, dtype=torch.float64, device="cuda")
    for seed in range(seeds):
        gpu = {k: x if k == "number" else torch.from_numpy(x.copy()).cuda() for k, x in state.items()}
        O.adamw_8bit_step([gpu], [torch.from_numpy(g).cuda()], [None], step=5, **dict(HOW, seed=seed))
        (a, b), = O.moments_8bit([gpu])
        total_m += a.double()
        total_v += b.double()
    scale_m, scale_v = gpu["exp_avg_scale"].cpu().numpy().astype(np.float64), gpu["exp_avg_sq_scale"].cpu().numpy().astype(np.float64)
    for total, want, scale, top in ((total_m, m, scale_m, 15), (total_v, v, scale_v, 31)):
        want = want.astype(np.float64)
        lowest = 2.0 ** (np.repeat(scale, 256) - 126 - top)  # of the lowest binade with eighths of its own
        step = np.maximum(2.0 ** np.floor(np.log2(np.maximum(np.abs(want), 1e-300))), lowest) / 8
        kept = np.abs(want) >= step if top == 31 else np.ones(n, bool)  # (a second moment below the least code is held as that)
        off = np.abs(total.cpu().numpy() / seeds - want)
        assert np.all((off <= step * (2.0 ** -17 + 6 / (2 * seeds ** 0.5)))[kept])


def test_a_slow_second_moment_follows_its_gradients(O):
    """beta2 = 0.999 and gradients of one size s after a start at 16 s^2: after 3000 steps the average of fp32 moments is 1 + 15 * 0.999^3000 = 1.75 s^2.  (Rounded to the
    nearest code they would still stand at 16.)  A moment's own deviation: a step moves it by d = 0.001 (v - s^2), which as random rounding adds a variance of at most d times a code's step
    (an eighth of its binade), d v / 8, forgotten at 0.002 a step: below v sqrt(0.001 / 8 / 0.002) = v / 4; over 65536 of them the mean's is v / 1024, and 0.1 is sixty of those."""
    n = 65536
    gpu = O.new_8bit_state(torch.zeros(n, device="cuda").bfloat16(), 0)
    grad = torch.full((n,), 4.0, device="cuda")
    O.adamw_8bit_step([gpu], [grad], [None], lr=0.0, betas=(0.9, 0.0), step=1)
    assert bool((O.moments_8bit([gpu])[0][1] == 16).all())
    grad.fill_(1.0)
    for k in range(3000):
        O.adamw_8bit_step([gpu], [grad], [None], lr=0.0, betas=(0.9, 0.999), step=2 + k, seed=5)
    m, v = O.moments_8bit([gpu])[0]
    assert abs(v.double().mean().item() - (1 + 15 * 0.999 ** 3000)) < 0.1
    assert abs(m.double().mean().item() - 1) < 0.01


def test_another_stream_captured_and_repeated(O):
    n = 10000
    state, gpu = random_state(n, 8)
    g = torch.from_numpy(gradient(n, 9)).cuda()
    start = {k: v if k == "number" else v.clone() for k, v in gpu.items()}

    def reset():
        for k, v in start.items():
            if k != "number":
                gpu[k].copy_(v)

    want = {k: v if k == "number" else torch.from_numpy(v.copy()).cuda() for k, v in state.items()}
    O.adamw_8bit_step([want], [g], [None], step=4, **HOW)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        O.adamw_8bit_step([gpu], [g], [None], step=4, **HOW)
    torch.cuda.synchronize()
    assert all(k == "number" or torch.equal(gpu[k], want[k]) for k in gpu)
    reset()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        O.adamw_8bit_step([gpu], [g], [None], step=4, **HOW)
    for _ in range(3):
        reset()
        graph.replay()
        torch.cuda.synchronize()
        assert all(k == "number" or torch.equal(gpu[k], want[k]) for k in gpu)


def test_a_tensor_of_more_than_two_to_the_31_elements(O):
    """Its last blocks, and some on both sides of 2^31, against the definition."""
    n = (1 << 31) + 1000
    gpu = {"master": torch.zeros(n, device="cuda"), "number": 3}
    for name, k in (("exp_avg", n), ("exp_avg_sq", n), ("exp_avg_scale", (n + 255) // 256), ("exp_avg_sq_scale", (n + 255) // 256)):
        gpu[name] = torch.zeros(k, dtype=torch.uint8, device="cuda")
    grad = torch.zeros(n, device="cuda")
    first = (1 << 31) - 1024
    g = gradient(n - first, 2)
    grad[first:] = torch.from_numpy(g).cuda()
    O.adamw_8bit_step([gpu], [grad], [None], step=1, **HOW)
    m, v = g * np.float32(1 - 0.9), g * g * np.float32(1 - 0.95)
    i = np.arange(first // 512 * 64, (n + 511) // 512 * 64, dtype=np.uint64)
    full = lambda x: np.full(len(i), x, dtype=np.uint64)  # noqa: E731
    words = R.philox([i & np.uint64(0xFFFFFFFF), i >> np.uint64(32), full(3), full(1)], (HOW["seed"] % 2 ** 32, HOW["seed"] >> 32))
    r = np.stack([(w >> np.uint64(s)) & np.uint64(0xFFFF) for w in words for s in (0, 16)], 1).reshape(-1, 64, 2, 4).swapaxes(1, 2).reshape(-1)[:n - first].astype(np.int64)
    for name, x, top, bits, least in (("exp_avg", m, 15, 7, 0), ("exp_avg_sq", v, 31, 8, 1)):
        codes, scales = R.encode(x.astype(np.float32), r, top, bits, least)
        assert np.array_equal(gpu[name][first:].cpu().numpy(), codes) and np.array_equal(gpu[name + "_scale"][first // 256:].cpu().numpy(), scales)
    assert not bool(gpu["exp_avg"][:first].any()) and not bool(gpu["master"][:first].any())


def test_refusals(O):
    _, gpu = random_state(1000, 1)
    g, w = torch.zeros(1000, device="cuda"), torch.zeros(1000, dtype=torch.bfloat16, device="cuda")
    before = {k: v if k == "number" else v.clone() for k, v in gpu.items()}

    def refused(state=None, grad=g, weight=w, **kw):
        with pytest.raises((ValueError, RuntimeError)):
            O.adamw_8bit_step([dict(gpu, **(state or {}))], [grad], [weight], **dict(dict(lr=1e-3, step=1), **kw))

    refused(grad=g[:999]); refused(grad=g.bfloat16()); refused(grad=g.cpu()); refused(weight=w[:999]); refused(weight=w.float())
    for name in ("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale"):
        refused({name: gpu[name][:-1]}); refused({name: gpu[name].int()}); refused({name: gpu[name].cpu()})
    refused({"master": gpu["master"].double()}); refused({"master": gpu["master"][:999]}); refused({"number": -1}); refused({"number": 2 ** 32})
    refused(step=0); refused(step=2 ** 32); refused(norm_coef=torch.zeros(3, device="cuda"))
    big = torch.zeros(1004, dtype=torch.uint8, device="cuda")
    refused({"exp_avg": big[4:]}); refused(grad=torch.zeros(1001, device="cuda")[1:])
    with pytest.raises((ValueError, RuntimeError)):
        O.adamw_8bit_step([gpu, gpu], [g], [w], lr=1e-3, step=1)
    assert all(k == "number" or torch.equal(gpu[k], before[k]) for k in gpu)
    O.adamw_8bit_step([], [], [], lr=1e-3, step=1)
    assert O.moments_8bit([]) == []
