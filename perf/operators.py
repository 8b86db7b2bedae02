"""What stands around the products of a transformer layer, measured through the framework's public entry points.

  norm     layer norm of an activation, alone or of its sum with the residual stream (`functional.layer_norm`, `add_layer_norm`)
  dropout  out = residual + dropout(x + bias), the mask drawn from a counter and never stored (`functional.dropout_add`)
  block    sum = residual + dropout(x + bias), y = norm(sum): layer norm or RMSNorm (`functional.dropout_add_layer_norm`,
           `dropout_add_rmsnorm`)
  linear   act(x W^T + bias) + residual (`functional.linear_act`)

each forward, or forward and backward (`train`).  Activations and weights are bf16.  Widths are those of the repository's presets and
workloads, or generic ones.

The random draw is part of the definition: element e of a tensor belongs to group e / 8; the 128 bits that Philox-4x32-10 (Salmon, Moraes, Dror,
Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011) makes of the counter (group low, group high, offset, 0) under the key (seed low,
seed high) are eight 16-bit numbers, the low half of a word first, and element e is dropped if number e % 8 is below round(65536 p).  The
others are scaled by 65536 / (65536 - round(65536 p)).  seed and offset are inputs.
"""
import math

import numpy as np
import torch

own = False

LEAVES = {"norm": ("x", "residual", "weight", "norm_bias"), "dropout": ("x", "residual", "bias"),
          "block": ("x", "residual", "bias", "weight", "norm_bias"), "linear": ("x", "weight", "bias", "residual")}


def _case(name, op, rows, h, **kw):
    case = dict(op=op, rows=rows, h=h, train=True, bias=True, residual=True)
    if op != "linear":
        case.update(kind="layer")
    if op in ("dropout", "block"):
        case.update(p=0.1)
    if op == "linear":
        case.update(out=h, act="none")
    case.update(kw)
    return dict(case, name=name) if name else case


def listed():
    return [
        # One token through a narrow stack, nothing to train: the time of a call.
        _case("norm_token", "norm", 1, 256, train=False, residual=False),
        # Three conversations of odd length at an odd width, fine-tuned.
        _case("norm_odd", "norm", 3 * 389, 1000),
        # The packed 16384-token batch at 7B width: the norm behind the residual sum, in training.
        _case("norm_packed", "norm", 16384, 4096),
        # The embeddings' dropout of the tiny stack: no bias, no residual.
        _case("dropout_tiny", "dropout", 2 * 512, 256, bias=False, residual=False),
        # The last sum of a layer whose down projection has a bias, an odd number of tokens at 13B width.
        _case("dropout_odd", "dropout", 1531, 5120),
        # The same over a micro-batch at 70B width.
        _case("dropout_large", "dropout", 8192, 8192),
        # Between attention and MLP of a small stack with layer norm.
        _case("block_small", "block", 2 * 1024, 768),
        # The same place of a llama stack (RMSNorm, no biases) that is trained with dropout.
        _case("block_rms", "block", 4 * 1000, 2048, kind="rms", bias=False, p=0.05),
        # 16384 tokens at 13B width.
        _case("block_large", "block", 16384, 5120),
        # The first product of an MLP on a handful of tokens, answered, not trained: the weights' way from memory.
        _case("linear_tokens", "linear", 8, 4096, out=11008, act="gelu", train=False, residual=False),
        # The same on one conversation of an odd length, fine-tuned.
        _case("linear_odd", "linear", 1531, 4096, out=11008, act="gelu_tanh", residual=False),
        # The second product of a wide MLP, with its bias and the residual stream, in training.
        _case("linear_residual", "linear", 4096, 13696, out=5120),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """One more case of the same ranges: 1 to 16384 rows, widths of 64 to 8192 that are multiples of 8."""
    op = rng.choice(["norm", "dropout", "block", "linear"])
    rows = _spread(rng, 1, 16384)
    h = 8 * _spread(rng, 8, 1024)
    train = rng.random() < 0.75
    if op == "linear":
        out = 8 * _spread(rng, 8, 1712)
        while rows * h * out > 4096 * 13696 * 5120:
            rows = max(1, rows // 2)
        return _case(None, op, rows, h, out=out, act=rng.choice(["none", "gelu", "gelu_tanh"]), train=train,
                     bias=rng.random() < 0.75, residual=rng.random() < 0.5)
    while rows * h > 16384 * 4096:
        rows = max(1, rows // 2)
    if op == "norm":
        return _case(None, op, rows, h, train=train, residual=rng.random() < 0.5, bias=rng.random() < 0.75)
    p = rng.choice([0.05, 0.1, 0.2, 0.5])
    if op == "dropout":
        return _case(None, op, rows, h, train=train, residual=rng.random() < 0.75, bias=rng.random() < 0.5, p=p)
    kind = rng.choice(["layer", "layer", "rms"])
    return _case(None, op, rows, h, kind=kind, train=train, bias=rng.random() < 0.5, p=p)


def _inputs(case, seed):
    """The tensors of a case, bf16 on the GPU, and the two numbers that the mask is drawn from."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, rows, h = case["op"], case["rows"], case["h"]
    out = case.get("out", h)

    def normal(*shape, scale=1.0, mean=0.0):
        return torch.randn(*shape, device="cuda", generator=g).mul_(scale).add_(mean).bfloat16()

    def stream(n):  # a residual stream: some channels are ten times the others
        wide = 1 + 9 * (torch.rand(n, device="cuda", generator=g) < 0.01).float()
        return torch.randn(rows, n, device="cuda", generator=g).mul_(wide).add_(0.1).bfloat16()

    t = {}
    if op == "linear":
        t["x"] = normal(rows, h)
        t["weight"] = normal(out, h, scale=h ** -0.5)
        if case["bias"]:
            t["bias"] = normal(out, scale=0.5)
        if case["residual"]:
            t["residual"] = stream(out)
    else:
        t["x"] = stream(h) if op == "norm" and not case["residual"] else normal(rows, h)
        if case["residual"]:
            t["residual"] = stream(h)
        if op in ("dropout", "block") and case["bias"]:
            t["bias"] = normal(h, scale=0.5)
        if op in ("norm", "block"):
            t["weight"] = normal(h, scale=0.1, mean=1.0)
            if case["kind"] == "layer" and (op == "block" or case["bias"]):
                t["norm_bias"] = normal(h, scale=0.1)
    grads = []
    if case["train"]:
        grads.append(normal(rows, out))
        if op == "block" or (op == "norm" and case["residual"]):
            grads.append(normal(rows, out))  # of the sum, from the residual stream behind it
    return t, grads, (seed * 1000003 + 12345, seed % 9973)


def _eps(case):
    return 1e-6 if case.get("kind") == "rms" else 1e-5


def prepare(case, seed):
    t, grads, rng = _inputs(case, seed)
    if case["train"]:
        for v in t.values():
            v.requires_grad_(True)
    return {"case": case, "t": t, "grads": grads, "rng": rng, "names": [n for n in LEAVES[case["op"]] if n in t]}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- the framework's calls -------------------------------------------------------------------------------------------
def _run_own(state):
    from easyllm_amd import functional as F

    case, t = state["case"], state["t"]
    x, residual, bias = t["x"], t.get("residual"), t.get("bias")
    with torch.set_grad_enabled(case["train"]):
        if case["op"] == "norm" and residual is None:
            outs = (F.layer_norm(x, t["weight"], t.get("norm_bias"), _eps(case)),)
        elif case["op"] == "norm":
            outs = F.add_layer_norm(x, residual, t["weight"], t.get("norm_bias"), _eps(case))
        elif case["op"] == "dropout":
            outs = (F.dropout_add(x, residual, bias, p=case["p"], rng=state["rng"]),)
        elif case["op"] == "block" and case["kind"] == "layer":
            outs = F.dropout_add_layer_norm(x, residual, t["weight"], t.get("norm_bias"), _eps(case), bias=bias, p=case["p"], rng=state["rng"])
        elif case["op"] == "block":
            outs = F.dropout_add_rmsnorm(x, residual, t["weight"], _eps(case), bias=bias, p=case["p"], rng=state["rng"])
        else:
            outs = (F.linear_act(x, t["weight"], bias, activation=case["act"], residual=residual),)
    if not case["train"]:
        return list(outs)
    grads = torch.autograd.grad(outs, [t[n] for n in state["names"]], state["grads"][::-1])
    return [o.detach() for o in outs] + list(grads)


# ---- the plain forms: elementary operations in 32 bits, rounded once -------------------------------------------------
def _low(a, b):
    return (a * b) & 0xFFFFFFFF


def _high(a, b):
    return ((a * b) >> 32) & 0xFFFFFFFF  # (the product's bits are right modulo 2^64, the mask drops the sign's)


def _kept(n, h, threshold, rng, device):
    """Whether each of n * h elements is kept, as a [n, h] mask."""
    seed, offset = rng
    group = torch.arange(n * h // 8, device=device)
    c0, c1 = group & 0xFFFFFFFF, group >> 32
    c2, c3 = torch.full_like(c0, offset & 0xFFFFFFFF), torch.zeros_like(c0)
    k0, k1 = seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF
    for _ in range(10):
        c0, c1, c2, c3 = (_high(c2, 0xCD9E8D57) ^ c1 ^ k0, _low(c2, 0xCD9E8D57), _high(c0, 0xD2511F53) ^ c3 ^ k1, _low(c0, 0xD2511F53))
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    words = torch.stack((c0, c1, c2, c3), 1)
    return (torch.stack((words & 0xFFFF, words >> 16), 2) >= threshold).view(n, h)


def _threshold(p):
    return int(p * 65536 + 0.5)


def _dropout(v, case, rng):
    """dropout(v) and what it multiplied v by."""
    t = _threshold(case["p"])
    factor = _kept(v.shape[0], v.shape[1], t, rng, v.device).float() * (65536.0 / (65536 - t))
    return v * factor, factor


def _normalised(s, case):
    if case["kind"] == "layer":
        s = s - s.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt((s * s).mean(1, keepdim=True) + _eps(case))
    return s * rstd, rstd


def _normalised_grad(g, xhat, rstd, case):
    dx = g - xhat * (g * xhat).mean(1, keepdim=True)
    if case["kind"] == "layer":
        dx = dx - g.mean(1, keepdim=True)
    return dx * rstd


def _activation(a, case):
    """act(a) and its derivative"""
    if case["act"] == "gelu":
        cdf = 0.5 * torch.special.erfc(a * -math.sqrt(0.5))
        return a * cdf, cdf + a * torch.exp(-0.5 * a * a) / math.sqrt(2 * math.pi)
    if case["act"] == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        sig = 1 / (1 + torch.exp(-2 * c * (a + 0.044715 * a * a * a)))  # (1 + tanh u) / 2 = 1 / (1 + exp(-2 u))
        return a * sig, sig + a * sig * (1 - sig) * 2 * c * (1 + 3 * 0.044715 * a * a)
    return a, None


@torch.no_grad()
def _run_plain(state):
    case, rng = state["case"], state["rng"]
    t = {n: v.detach().float() for n, v in state["t"].items()}
    grads = [g.float() for g in state["grads"]]
    x, residual, bias = t["x"], t.get("residual"), t.get("bias")
    outs, back = [], {}
    if case["op"] == "linear":
        pre = x @ t["weight"].t()
        if bias is not None:
            pre = pre + bias
        y, slope = _activation(pre, case)
        outs = [y if residual is None else y + residual]
        if grads:
            dy = grads[0]
            d = dy if slope is None else dy * slope
            back = {"x": d @ t["weight"], "weight": d.t() @ x, "bias": d.sum(0), "residual": dy}
    else:
        s = x if bias is None or case["op"] == "norm" else x + bias
        factor = None
        if case["op"] != "norm":
            s, factor = _dropout(s, case, rng)
        if residual is not None:
            s = s + residual
        ds = None
        if case["op"] == "dropout":
            outs = [s]
            ds = grads[0] if grads else None
        else:
            xhat, rstd = _normalised(s, case)
            y = xhat * t["weight"]
            if "norm_bias" in t:
                y = y + t["norm_bias"]
            outs = [s, y] if residual is not None else [y]
            if grads:
                dy = grads[0]
                back = {"weight": (dy * xhat).sum(0), "norm_bias": dy.sum(0)}
                ds = _normalised_grad(dy * t["weight"], xhat, rstd, case)
                if residual is not None:
                    ds = ds + grads[1]
        if grads:
            back["residual"] = ds
            back["x"] = ds if factor is None else ds * factor
            back["bias"] = back["x"].sum(0)
    return [v.bfloat16() for v in outs] + [back[n].bfloat16() for n in state["names"] if grads]


# ---- the definition in 64 bits ---------------------------------------------------------------------------------------
def _exact_factor(case, rng):
    """What each element is multiplied by: the generator in numpy's unsigned integers."""
    seed, offset = rng
    n = case["rows"] * case["h"]
    group = np.arange(n // 8, dtype=np.uint64)
    mask, half = np.uint64(0xFFFFFFFF), np.uint64(32)
    c = [group & mask, group >> half, np.full_like(group, offset & 0xFFFFFFFF), np.zeros_like(group)]
    key = [seed % 2 ** 32, seed // 2 ** 32 % 2 ** 32]
    for i in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        keys = [np.uint64((k + i * w) % 2 ** 32) for k, w in zip(key, (0x9E3779B9, 0xBB67AE85))]
        c = [(b >> half) ^ c[1] ^ keys[0], b & mask, (a >> half) ^ c[3] ^ keys[1], a & mask]
    numbers = np.stack([(w >> np.uint64(s)).astype(np.uint16) for w in c for s in (0, 16)], 1).reshape(case["rows"], case["h"])
    t = int(np.floor(65536 * case["p"] + 0.5))
    return torch.from_numpy(numbers >= t).cuda().double() * (65536 / (65536 - t))


def exact(case, seed):
    """The outputs in 64 bits: the operator's definition, and what differentiating it gives."""
    inputs, grads, rng = _inputs(case, seed)
    t = {n: v.double().requires_grad_(case["train"]) for n, v in inputs.items()}
    if case["op"] == "linear":
        y = torch.nn.functional.linear(t["x"], t["weight"], t.get("bias"))
        if case["act"] == "gelu":
            y = y * (1 + torch.erf(y / 2 ** 0.5)) / 2
        elif case["act"] == "gelu_tanh":
            y = y / 2 * (1 + torch.tanh((2 / math.pi) ** 0.5 * (y + 0.044715 * y ** 3)))
        outs = [y + t["residual"] if "residual" in t else y]
    else:
        s = t["x"]
        if case["op"] != "norm":
            s = (s + t["bias"] if "bias" in t else s) * _exact_factor(case, rng)
        if "residual" in t:
            s = s + t["residual"]
        outs = [s]
        if case["op"] != "dropout":
            if case["kind"] == "layer":
                var, mean = torch.var_mean(s, 1, correction=0, keepdim=True)
                y = (s - mean) / (var + _eps(case)) ** 0.5 * t["weight"]
            else:
                y = s / (s.square().mean(1, keepdim=True) + _eps(case)) ** 0.5 * t["weight"]
            y = y + t["norm_bias"] if "norm_bias" in t else y
            outs = [s, y] if "residual" in t else [y]
    back = ()
    if case["train"]:
        back = torch.autograd.grad(outs, [t[n] for n in LEAVES[case["op"]] if n in t], [g.double() for g in grads[::-1]])
    return [o.detach() for o in outs] + list(back)


def work(case):
    """Each input read once, each output written once, two bytes a value."""
    op, n, h = case["op"], case["rows"], case["h"]
    out = case.get("out", h)
    acts = n * h + n * out * (1 + case["residual"])  # x, the residual, the result
    weights = (out * h if op == "linear" else 0) + out * case["bias"]
    if op in ("norm", "block"):
        acts += n * h * case["residual"]  # the sum is a result too
        weights = 2 * h
    flops = {"norm": 10, "dropout": 6, "block": 15}.get(op, 0) * n * h + (2 * n * h * out if op == "linear" else 0)
    values = acts + weights
    if case["train"]:  # the inputs and the gradients of the outputs read, those of the inputs written
        values += acts + weights
        flops *= 3 if op == "linear" else 2
    return {"bytes": 2 * values, "flops": flops}
