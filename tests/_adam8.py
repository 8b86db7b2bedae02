"""AdamW with 8-bit moments restated in numpy: fp32 numbers with every operation rounded by itself, codes from their bits."""
import numpy as np

from _draw import philox


def random_numbers(n, number, step, seed):
    """A 16-bit number for each of n elements."""
    pairs = (n + 511) // 512
    i = np.arange(64 * pairs, dtype=np.uint64)
    full = lambda v: np.full(64 * pairs, v, dtype=np.uint64)  # noqa: E731
    words = philox([i & np.uint64(0xFFFFFFFF), i >> np.uint64(32), full(number), full(step)], (seed % 2 ** 32, seed >> 32))
    numbers = np.stack([(w >> np.uint64(s)) & np.uint64(0xFFFF) for w in words for s in (0, 16)], 1)
    return numbers.reshape(pairs, 64, 2, 4).swapaxes(1, 2).reshape(-1)[:n].astype(np.int64)


def blocks(x):
    return np.pad(x, (0, -len(x) % 256)).reshape(-1, 256)


def values(codes, scales, top, bits):
    """fp64 values (NaN in blocks that are not finite)"""
    c, e = codes.astype(np.int64), np.repeat(scales.astype(np.int64), 256)[:len(codes)]
    c, negative = c & ((1 << bits) - 1), c >> bits != 0
    x = ((c << 20).astype(np.uint32)).view(np.float32).astype(np.float64) * 2.0 ** (e - top)
    return np.where(e == 255, np.nan, np.where(negative, -x, x))


def encode(x, r, top, bits, least):
    """fp32 x -> (codes, scales)"""
    n = len(x)
    magnitude = (blocks(x).view(np.uint32) & np.uint32(0x7FFFFFFF)).astype(np.int64)
    e = np.minimum((magnitude.max(1) + (1 << 20)) >> 23, 255)
    with np.errstate(invalid="ignore", over="ignore"):  # blocks that are not finite
        scaled = (magnitude.astype(np.uint32).view(np.float32).astype(np.float64) * 2.0 ** (top - e[:, None])).astype(np.float32)  # (one rounding, of denormals)
    code = ((scaled.view(np.uint32).astype(np.int64) + 16 * blocks(r) + 8) >> 20).reshape(-1)[:n]
    code = np.where((x > 0) & (code < least), least, code)
    code = np.where(np.signbit(x), code | (1 << bits) & 0xFF, code)
    return np.where(np.repeat(e, 256)[:n] == 255, 0, code).astype(np.uint8), e.astype(np.uint8)


def step(state, grad, how, coef=np.float32(1)):
    """state: dict of numpy arrays (master fp32, codes, scales), changed in place -> the fp32 moments before they are rounded"""
    f = np.float32
    b1, b2 = how["betas"]
    k, n = how["step"], len(grad)
    bc = how.get("bias_correction", True)
    g = grad * coef
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        m = values(state["exp_avg"], state["exp_avg_scale"], 15, 7).astype(f) * f(b1) + g * f(1 - b1)
        v = values(state["exp_avg_sq"], state["exp_avg_sq_scale"], 31, 8).astype(f) * f(b2) + g * g * f(1 - b2)
        ibc1, ibc2 = (f(1 / (1 - b ** k)) if bc else f(1) for b in (b1, b2))
        update = (m * ibc1) / (np.sqrt(v * ibc2) + f(how["eps"]))
        state["master"][:] = state["master"] - (update + state["master"] * f(how["weight_decay"])) * f(how["lr"])
    r = random_numbers(n, state["number"], k, how["seed"])
    state["exp_avg"], state["exp_avg_scale"] = encode(m, r, 15, 7, 0)
    state["exp_avg_sq"], state["exp_avg_sq_scale"] = encode(v, r, 31, 8, 1)
    return m, v
