"""A stack with rotary positions of another pairing, part of the head and stretched, a fused gated MLP, stepped with 8-bit moments: as a user builds and trains it, against the same
computation in 64 bits.

Tolerance, before any run: a gradient has passed some 25 tensors that are stored in bf16, each off by 2^-9 / sqrt(3) of its values in the mean, independently: sqrt(25) * 0.0011 = 0.6 %; five
times that, 3 %, in the 2-norm.  The loss, a mean over all rows, 1e-3 of itself.  q's and k's gradients are small differences of large values: they may be twice as far off as the same
arithmetic with every stored tensor and its gradient rounded to bf16 and nothing else (two such evaluations, which round independently, are as far apart as either is from 64 bits)."""
import math

import numpy as np
import pytest
import torch

import _adam8
from test_layer_options_gpu import StoredOutputAttention

pytestmark = pytest.mark.gpu

H, HEADS, KV, FFN, VOCAB, S = 256, 4, 2, 712, 520, 96
YARN = {"type": "yarn", "factor": 4.0, "original_length": 32}
STACKS = {
    "neighbours, part of the head, yarn, a GELU gate": (dict(rotary_dim=32, interleaved=True, scaling=YARN), "gelu"),
    "halves, linear, a tanh gate": (dict(scaling={"type": "linear", "factor": 2.0}), "gelu_tanh"),
    "a larger base, a SiLU gate": (dict(rotary_dim=48, scaling={"type": "dynamic", "factor": 2.0, "original_length": 48}), "silu"),
    "neighbours, a ReLU gate": (dict(interleaved=True), "relu"),
}


def build(name, **kw):
    from easyllm_amd import runner
    torch.manual_seed(5)
    positions, gate = STACKS[name]
    cfg = dict(num_layers=2, hidden_size=H, num_attention_heads=HEADS, num_kv_attention_heads=KV, intermediate_size=FFN, vocab_size=VOCAB, seq_length=S, bf16=True,
               checkpoint_activations=False, fp32_logits=False, position_embedding_kwargs=dict(positions), transformer_layer_params=dict(glu_activation=gate, glu_fusion=True))
    cfg.update(kw)
    return runner.build_model({"type": "llama_custom", "kwargs": cfg}).cuda()


def batch(b=3, seed=1, packed=False):
    g = torch.Generator().manual_seed(seed)
    tokens, labels = torch.randint(0, VOCAB, (b, S), generator=g).cuda(), torch.randint(0, VOCAB, (b, S), generator=g).cuda()
    if not packed:
        return (tokens, torch.arange(S).expand(b, S).contiguous().cuda(), None), (labels, torch.ones(b, S, device="cuda"))
    cu = torch.tensor([0, 50, S, S + 31, 2 * S, 3 * S][:2 * b])
    positions = torch.cat([torch.arange(n) + 1000 * i for i, n in enumerate((cu[1:] - cu[:-1]).tolist())]).view(b, S)  # (documents from the middle of longer texts)
    return (tokens, positions.cuda(), None, cu.cuda()), (labels, torch.ones(b, S, device="cuda"))


def reference(model, inputs, labels, name, storage=None):
    """loss and {name: gradient} in fp64; storage: with every tensor that the step keeps rounded to that type"""
    from oracle import llama_oracle as O
    W = {n: v.detach().double().requires_grad_(True) for n, v in model.named_parameters()}
    st = lambda t: O.stored(t, storage)  # noqa: E731
    options, gate = STACKS[name]
    ids, positions = inputs[0], inputs[1]
    b, s = ids.shape
    d = H // HEADS
    n = options.get("rotary_dim", d)
    rope = model.get_submodule("3").self_attn.rotary_emb
    inv_freq, factor = rope.frequencies(s, ids.device)
    angle = positions.t().double()[:, :, None, None] * inv_freq
    cos, sin = torch.cos(angle) * factor, torch.sin(angle) * factor
    cu = inputs[3].tolist() if len(inputs) == 4 else [i * s for i in range(b + 1)]
    doc = torch.zeros(b * s, dtype=torch.long, device="cuda")
    for i in range(len(cu) - 1):
        doc[cu[i]:cu[i + 1]] = i
    doc = doc.view(b, s)
    masked = (doc[:, :, None] != doc[:, None, :]) | torch.ones(s, s, dtype=torch.bool, device="cuda").triu(1)

    def turned(x):
        if options.get("interleaved"):
            p, q = x[..., 0:n:2], x[..., 1:n:2]
            y = torch.stack((p * cos - q * sin, q * cos + p * sin), -1).flatten(-2)
        else:
            p, q = x[..., :n // 2], x[..., n // 2:n]
            y = torch.cat((p * cos - q * sin, q * cos + p * sin), -1)
        return st(torch.cat((y, x[..., n:]), -1))

    def norm(x, name):
        return x * (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * W[name + ".weight"]

    def linear(x, name):
        return x @ W[name + ".weight"].t()

    def act(x):
        f = torch.nn.functional
        return f.silu(x) if gate == "silu" else f.relu(x) if gate == "relu" else f.gelu(x, approximate="tanh" if gate == "gelu_tanh" else "none")
    x = st(W["1.word_embeddings.weight"][ids]).transpose(0, 1)
    for i in (3, 4):
        ln = st(norm(x, "%d.input_layernorm" % i))
        q = st(linear(ln, "%d.self_attn.q_proj" % i)).reshape(s, b, HEADS, d)
        k, v = (st(linear(ln, "%d.self_attn.%s_proj" % (i, c))).reshape(s, b, KV, d) for c in "kv")
        q, k = turned(q), turned(k)
        k, v = (t.repeat_interleave(HEADS // KV, 2).permute(1, 2, 0, 3) for t in (k, v))
        scores = (q.permute(1, 2, 0, 3) @ k.transpose(-1, -2)) / math.sqrt(d)
        scores = scores.masked_fill(masked[:, None], -math.inf)
        ctx = scores.softmax(-1) @ v if storage is None else StoredOutputAttention.apply(scores, v, storage)
        s1 = st(x + st(linear(ctx.permute(2, 0, 1, 3).reshape(s, b, H), "%d.self_attn.o_proj" % i)))
        ln2 = st(norm(s1, "%d.post_attention_layernorm" % i))
        mid = st(act(st(linear(ln2, "%d.mlp.gate_proj" % i))) * st(linear(ln2, "%d.mlp.up_proj" % i)))
        x = st(s1 + st(linear(mid, "%d.mlp.down_proj" % i)))
    logits = st(st(norm(x.transpose(0, 1), "6")) @ W["7.word_embeddings.weight"].t())
    loss = torch.nn.functional.cross_entropy(logits.reshape(-1, VOCAB), labels[0].reshape(-1))
    loss.backward()
    return loss.item(), {n: w.grad for n, w in W.items()}


def far(a, b):
    return ((a.double() - b).norm() / b.norm()).item()


@pytest.mark.parametrize("name", STACKS)
@pytest.mark.parametrize("packed", [False, True])
def test_loss_and_gradients(name, packed):
    from easyllm_amd import runner
    model = build(name)
    inputs, labels = batch(packed=packed)
    runner.attach_main_grads(model)
    loss = runner.forward_step(model, inputs, labels)
    want, grads = reference(model, inputs, labels, name)
    assert abs(loss.item() - want) <= 1e-3 * want
    rounded = None
    for n, p in model.named_parameters():
        off = far(p.main_grad, grads[n])
        if off > 0.03:
            rounded = rounded or reference(model, inputs, labels, name, torch.bfloat16)[1]
            assert off <= 2 * far(rounded[n], grads[n]), (n, off, far(rounded[n], grads[n]))


def test_whatever_is_recomputed_or_captured_gives_the_same_bits():
    from easyllm_amd import runner
    name = next(iter(STACKS))
    inputs, labels = batch(packed=True)
    got = []
    for kw in (dict(), dict(checkpoint_activations=True)):
        model = build(name, **kw)
        runner.attach_main_grads(model)
        loss = runner.forward_step(model, inputs, labels)
        assert model.recompute_count == (2 if kw else 0)
        got.append((loss.item(), {n: p.main_grad.clone() for n, p in model.named_parameters()}))
    assert got[0][0] == got[1][0] and all(torch.equal(got[0][1][n], got[1][1][n]) for n in got[0][1])
    step = runner.GraphedStep(model, inputs, labels)
    for seed in (2, 3, 4):
        inputs, labels = batch(seed=seed, packed=True)
        loss = step(inputs, labels)
        torch.cuda.synchronize()
        step.flush()
        captured = loss.item(), {n: p.main_grad.clone() for n, p in model.named_parameters()}
        runner.zero_main_grads(model)
        eager = runner.forward_step(model, inputs, labels)
        assert eager.item() == captured[0] and all(torch.equal(p.main_grad, captured[1][n]) for n, p in model.named_parameters())
        del eager


def test_hooks_see_what_they_saw():
    """A hook on a projection of a fused block gets that projection's own result; the block's result does not change beyond the roundings in between (three of 2^-9 each, and the sums')."""
    model = build("halves, linear, a tanh gate")
    inputs, _ = batch()
    mlp = model.get_submodule("3").mlp
    with torch.no_grad():
        want = model(inputs)
        for name in ("gate_proj", "up_proj", "down_proj"):
            seen = []
            hook = getattr(mlp, name).register_forward_hook(lambda m, i, o: seen.append((i[0], o[0])))
            got = model(inputs)
            hook.remove()
            (x, y), = seen
            ref = x.double() @ getattr(mlp, name).weight.double().t()
            assert far(y, ref) <= 2.0 ** -8 and far(got, want.double()) <= 1e-2
        assert torch.equal(model(inputs), want)


def test_position_ids_have_no_limit():
    """A document far behind the sequence's own length, which a model with tables refuses."""
    name = "neighbours, a ReLU gate"
    model = build(name)
    (tokens, positions, mask, cu), labels = batch(packed=True)
    with torch.no_grad():
        far_away = model((tokens, positions + (1 << 22), mask, cu))
    assert bool(torch.isfinite(far_away.float()).all())
    from easyllm_amd import runner
    plain = runner.build_model({"type": "llama_custom", "kwargs": dict(num_layers=1, hidden_size=H, num_attention_heads=HEADS, intermediate_size=FFN, vocab_size=VOCAB, seq_length=S, bf16=True)}).cuda()
    with pytest.raises(IndexError):
        plain((tokens, positions + (1 << 22), mask, cu))


@pytest.mark.parametrize("clip", [0.0, 0.25])
def test_training_iterations_with_8_bit_moments(clip):
    """Three iterations of build_optimizer's AdamW8bit: small parameters follow the 32-bit rule, the others' codes are those of the definition fed with the same gradients, bit by bit."""
    from easyllm_amd import optimizer, runner
    from oracle import llama_oracle as O
    name = next(iter(STACKS))
    model = build(name)
    runner.attach_main_grads(model)
    kwargs = {"lr": 1e-3, "betas": [0.9, 0.95], "eps": 1e-8, "weight_decay": 0.1, "seed": 11}
    opt = optimizer.build_optimizer({"type": "AdamW8bit", "kwargs": dict(kwargs)}, model)
    params = [p for g in opt.param_groups for p in g["params"]]
    eight = [p for p in params if "number" in opt.state[p]]
    assert all((p.numel() >= 4096) == ("number" in opt.state[p]) for p in params) and len(eight) > 10 and len(params) > len(eight)
    states = {p: {k: v if k == "number" else v.cpu().numpy().reshape(-1).copy() for k, v in opt.state[p].items()} for p in eight}
    wide = {p: tuple(opt.state[p][k].cpu().clone() for k in ("master", "exp_avg", "exp_avg_sq")) for p in params if p not in states}
    for k in (1, 2, 3):
        inputs, labels = batch(seed=k, packed=k == 2)
        runner.zero_main_grads(model)
        runner.forward_step(model, inputs, labels)
        norm_coef = opt.step(clip_grad=clip)
        coef = np.float32(1 if norm_coef is None else norm_coef[1].item())
        assert (clip > 0) == (norm_coef is not None) and (clip == 0 or coef < 1)
        how = dict(lr=1e-3, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.1, seed=11, step=k)
        for p in eight:
            mine, state = opt.state[p], states[p]
            before = state["master"].astype(np.float64)
            _adam8.step(state, p.main_grad.cpu().numpy().reshape(-1), how, coef)
            for n in ("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale"):
                assert np.array_equal(mine[n].cpu().numpy(), state[n]), (k, n, tuple(p.shape))
            got = mine["master"].cpu().numpy().reshape(-1)
            off = np.abs(got.astype(np.float64) - state["master"]) - np.abs(state["master"] - before) * (2.0 ** -21 + 2.0 ** -23) - np.abs(state["master"].astype(np.float64)) * 2.0 ** -23
            assert not (off > 0).any()
            state["master"][:] = got
            assert torch.equal(p.data, mine["master"].view(p.shape).bfloat16())
            m, v = opt.moments(p)
            assert m.shape == p.shape and np.array_equal(m.double().cpu().numpy().reshape(-1), _adam8.values(state["exp_avg"], state["exp_avg_scale"], 15, 7))
        for p, (master, m, v) in wide.items():
            wide[p] = O.adamw_step(master, m, v, p.main_grad.cpu() * coef, 1e-3, 0.9, 0.95, 1e-8, 0.1, k, True)
            assert torch.allclose(opt.state[p]["master"].cpu(), wide[p][0], rtol=2e-6, atol=1e-6) and opt.moments(p)[0] is opt.state[p]["exp_avg"]


def test_a_run_goes_on_from_a_copy_of_its_state():
    from easyllm_amd import optimizer, runner
    name = next(iter(STACKS))

    def run(steps, model=None, opt=None, first=1):
        if model is None:
            model = build(name)
            runner.attach_main_grads(model)
            opt = optimizer.build_optimizer({"type": "AdamW8bit", "kwargs": {"lr": 1e-3, "seed": 3}}, model)
        for k in range(first, first + steps):
            runner.zero_main_grads(model)
            runner.forward_step(model, *batch(seed=k))
            opt.step(clip_grad=1.0)
        return model, opt
    whole, whole_opt = run(4)
    part, opt = run(2)
    again = build(name)
    again.load_state_dict(part.state_dict())
    runner.attach_main_grads(again)
    fresh = optimizer.build_optimizer({"type": "AdamW8bit", "kwargs": {"lr": 1e-3, "seed": 3}}, again)
    for g, h in zip(opt.param_groups, fresh.param_groups):
        h["step"] = g["step"]
        for p, q in zip(g["params"], h["params"]):
            for n, v in opt.state[p].items():
                if n != "number":
                    fresh.state[q][n].copy_(v)
    run(2, again, fresh, first=3)
    assert all(torch.equal(a, b) for a, b in zip(whole.state_dict().values(), again.state_dict().values()))
    for g, h in zip(whole_opt.param_groups, fresh.param_groups):
        assert all(torch.equal(whole_opt.state[p][n], fresh.state[q][n]) for p, q in zip(g["params"], h["params"]) for n in whole_opt.state[p] if n != "number")
