"""Stacks with layer norm, dropout, biases and a plain GELU MLP, as a user builds them, against the same computation in 64 bits with the masks of the draws
that the step made.

Tolerance, before any run: a gradient has passed some 25 tensors that are stored in bf16, each off by 2^-9 / sqrt(3) of its values in the mean, independently:
sqrt(25) * 0.0011 = 0.6 %; five times that, 3 %, in the 2-norm.  The loss, a mean over all rows, 1e-3 of itself as in the rest of the tests.

Where a value is a small difference of large ones, 3 % is not what storing bf16 costs: a score's gradient is P (dP - sum P dP), whose two terms nearly cancel where
attention is even, so what their inputs are off by comes out magnified in q's and k's gradients.  How much follows from the same arithmetic with every stored
tensor (and its gradient) rounded to bf16 and nothing else: `reference(storage=torch.bfloat16)`, where sum P dP is, as in any backward pass that keeps
no P, the row sum of the output's gradient times the output as it is stored.  A gradient beyond 3 % may be
twice as far off as that evaluation is: what row sums are off by goes into k's gradient along the queries' common part (their bias), as one number for each of
the 12 pairs of sequence and head; a sum of 12 such squares has a relative deviation of sqrt(2 / 12) = 0.41, and two of them, independent since the
evaluations round differently, are a factor of 4 apart (2 in the norm) at 2.4 deviations of their ratio's logarithm, sqrt(2) * 0.41."""
import math

import pytest
import torch

import _draw

pytestmark = pytest.mark.gpu

H, HEADS, FFN, VOCAB = 256, 4, 712, 520


def build(**kw):
    from easyllm_amd import runner
    torch.manual_seed(5)
    layer = dict(kw.pop("layer", {}))
    cfg = dict(num_layers=2, hidden_size=H, num_attention_heads=HEADS, intermediate_size=FFN, vocab_size=VOCAB, seq_length=96, bf16=True,
               checkpoint_activations=False, fp32_logits=False, transformer_layer_params=layer)
    cfg.update(kw)
    model = runner.build_model({"type": "llama_custom", "kwargs": cfg}).cuda()
    with torch.no_grad():
        for p in model.parameters():
            if p.dim() == 1:
                p.add_(0.2 * torch.randn_like(p))
    return model


def batch(b=3, s=96, seed=1):
    g = torch.Generator().manual_seed(seed)
    tokens, labels = torch.randint(0, VOCAB, (b, s), generator=g).cuda(), torch.randint(0, VOCAB, (b, s), generator=g).cuda()
    return (tokens, torch.arange(s).expand(b, s).contiguous().cuda(), None), (labels, torch.ones(b, s, device="cuda"))


class StoredOutputAttention(torch.autograd.Function):
    """softmax(scores) v in fp64, rounded; backward with sum_j P dP = sum dO O of the rounded O, and P and dS rounded for the products."""

    @staticmethod
    def forward(ctx, scores, v, dtype):
        p = scores.softmax(-1)
        o = (p @ v).to(dtype).double()
        ctx.save_for_backward(p, v, o)
        ctx.dtype = dtype
        return o

    @staticmethod
    def backward(ctx, do):
        p, v, o = ctx.saved_tensors
        do = do.to(ctx.dtype).double()
        ds = p * (do @ v.transpose(-1, -2) - (do * o).sum(-1, keepdim=True))
        return ds.to(ctx.dtype).double(), p.to(ctx.dtype).double().transpose(-1, -2) @ do, None


def reference(model, inputs, labels, draws, p, act, post_ln=False, storage=None):
    """loss and {name: gradient} in fp64; storage: with every tensor that the step keeps rounded to that type"""
    from oracle import llama_oracle as O
    W = {n: v.detach().double().requires_grad_(True) for n, v in model.named_parameters()}
    draws = iter(draws)
    st = lambda t: O.stored(t, storage)  # noqa: E731

    def drop(x):
        if p == 0:
            return x
        d = next(draws)
        step = 0 if d.step is None else int(d.step.item())
        return x * torch.from_numpy(_draw.factor(tuple(x.shape), int(p * 65536 + 0.5), d.seed, d.offset, step)).to(x.device)

    def norm(x, name):
        w, b = W[name + ".weight"], W.get(name + ".bias")
        if b is None:
            return x * (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w
        return torch.nn.functional.layer_norm(x, (H,), w, b, 1e-6)

    def linear(x, name):
        y = x @ W[name + ".weight"].t()
        return y if name + ".bias" not in W else y + W[name + ".bias"]
    ids = inputs[0]
    b, s = ids.shape
    x = st(drop(W["1.word_embeddings.weight"][ids])).transpose(0, 1)  # [s, b, h]
    d = H // HEADS
    cos, sin = O.rope_cos_sin(O.positions_sb(s, b, None), d, 10000.0, dtype=torch.float64)
    cos, sin = cos[:, :, None, :].cuda(), sin[:, :, None, :].cuda()
    for i in (3, 4):
        ln = st(norm(x, "%d.input_layernorm" % i))
        q, k, v = (st(linear(ln, "%d.self_attn.%s_proj" % (i, c))).reshape(s, b, HEADS, d) for c in "qkv")
        q, k = st(O.apply_rope(q, cos, sin)), st(O.apply_rope(k, cos, sin))
        scores = (q.permute(1, 2, 0, 3) @ k.permute(1, 2, 3, 0)) / math.sqrt(d)
        scores = scores.masked_fill(torch.ones(s, s, dtype=torch.bool, device="cuda").triu(1), -math.inf)
        vh = v.permute(1, 2, 0, 3)
        ctx = scores.softmax(-1) @ vh if storage is None else StoredOutputAttention.apply(scores, vh, storage)
        ctx = ctx.permute(2, 0, 1, 3).reshape(s, b, H)
        s1 = st((ln if post_ln else x) + drop(st(linear(ctx, "%d.self_attn.o_proj" % i))))
        ln2 = st(norm(s1, "%d.post_attention_layernorm" % i))
        up = st(linear(ln2, "%d.mlp.up_proj" % i))
        if act == "silu":
            up = st(torch.nn.functional.silu(st(linear(ln2, "%d.mlp.gate_proj" % i))) * up)
        else:
            up = st(torch.nn.functional.gelu(up, approximate="tanh" if act == "gelu_tanh" else "none"))
        x = st((ln2 if post_ln else s1) + drop(st(linear(up, "%d.mlp.down_proj" % i))))
    logits = st(st(norm(x.transpose(0, 1), "6")) @ W["7.word_embeddings.weight"].t())
    loss = torch.nn.functional.cross_entropy(logits.reshape(-1, VOCAB), labels[0].reshape(-1))
    loss.backward()
    return loss.item(), {n: w.grad for n, w in W.items()}


LN = {"type": "mixed_fused_norm"}
PLAIN = dict(glu_activation=None, mlp_bias=True, attention_qkv_bias=True, attention_o_bias=True)
CASES = {
    "layer norm, gelu, biases, dropout": (dict(layer_norm_params=LN, hidden_dropout=0.1, layer=PLAIN), 0.1, "gelu"),
    "the same without dropout": (dict(layer_norm_params=LN, layer=dict(PLAIN, use_openai_gelu=True)), 0, "gelu_tanh"),
    "layer norm, gelu, no biases": (dict(layer_norm_params=LN, hidden_dropout=0.2, layer=dict(glu_activation=None, bias_gelu_fusion=True)), 0.2, "gelu_tanh"),
    "llama with dropout": (dict(hidden_dropout=0.1), 0.1, "silu"),
    "llama with dropout and an output bias": (dict(hidden_dropout=0.1, layer=dict(attention_o_bias=True)), 0.1, "silu"),
    "layer norm, gated MLP": (dict(layer_norm_params=LN, layer=dict(attention_o_bias=True)), 0, "silu"),
    "RMSNorm, plain MLP": (dict(layer=dict(glu_activation=None)), 0, "gelu"),
    "residual behind the norm": (dict(layer_norm_params=LN, hidden_dropout=0.1, layer=dict(PLAIN, apply_residual_connection_post_layernorm=True)), 0.1, "gelu"),
    "residual behind the norm, no dropout": (dict(layer_norm_params=LN, layer=dict(PLAIN, apply_residual_connection_post_layernorm=True)), 0, "gelu"),
}


@pytest.mark.parametrize("name", CASES)
@pytest.mark.parametrize("main_grads", [True, False])
def test_loss_and_gradients(name, main_grads):
    from easyllm_amd import dropout, runner
    print(name, main_grads, flush=True)
    kw, p, act = CASES[name]
    model = build(**kw)
    if main_grads:
        runner.attach_main_grads(model)
    inputs, labels = batch()
    with dropout.recording() as draws:
        loss = runner.forward_step(model, inputs, labels)
    assert len(draws) == (5 if p else 0) and len(set(draws)) == len(draws)
    post_ln = kw.get("layer", {}).get("apply_residual_connection_post_layernorm", False)
    ref, grads = reference(model, inputs, labels, draws, p, act, post_ln)
    _, rounded = reference(model, inputs, labels, draws, p, act, post_ln, torch.bfloat16)
    assert abs(loss.item() - ref) <= 1e-3 * ref, (loss.item(), ref)
    for n, w in model.named_parameters():
        got = (w.main_grad if main_grads else w.grad).double()
        off = ((got - grads[n]).norm() / grads[n].norm()).item()
        if n.endswith("k_proj.bias"):  # (a softmax does not change with its key bias: what is left of the gradient is rounding)
            assert got.norm() <= 2e-2 * grads[n.replace("k_proj", "q_proj")].norm() + 2e-2 * grads[n.replace("k_proj", "v_proj")].norm()
            continue
        floor = ((rounded[n] - grads[n]).norm() / grads[n].norm()).item()
        assert off <= max(3e-2, 2 * floor), (n, off, floor)


def test_nothing_is_dropped_in_evaluation():
    from easyllm_amd import dropout
    model = build(layer_norm_params=LN, hidden_dropout=0.3, layer=PLAIN).eval()
    plain = build(layer_norm_params=LN, layer=PLAIN)
    plain.load_state_dict(model.state_dict())
    inputs, _ = batch()
    with torch.no_grad(), dropout.recording() as draws:
        assert torch.equal(model(inputs), model(inputs))
        off = (model(inputs).double() - plain(inputs).double()).norm() / plain(inputs).double().norm()
    assert not draws and off <= 1e-2


@pytest.mark.parametrize("kw", [dict(layer_norm_params=LN, hidden_dropout=0.1, layer=PLAIN), dict(hidden_dropout=0.1)])
def test_recomputed_layers_give_the_same_bits(kw):
    from easyllm_amd import dropout, runner
    inputs, labels = batch()
    seen = []
    for recompute in (False, True):
        model = build(**dict(kw, checkpoint_activations=recompute))
        runner.attach_main_grads(model)
        dropout.manual_seed(99)
        loss = runner.forward_step(model, inputs, labels)
        assert (model.recompute_count > 0) == recompute
        seen.append((loss.item(), {n: w.main_grad.clone() for n, w in model.named_parameters()}))
    assert seen[0][0] == seen[1][0]
    for n, g in seen[0][1].items():
        assert torch.equal(g, seen[1][1][n]), n


def test_a_captured_step_draws_anew_and_matches_the_eager_one():
    from easyllm_amd import dropout, runner
    model = build(layer_norm_params=LN, hidden_dropout=0.2, layer=PLAIN, checkpoint_activations=True)
    runner.attach_main_grads(model)
    batches = [batch(seed=s) for s in (1, 2)]
    step = runner.GraphedStep(model, *batches[0])
    draws = list(step._draws)
    assert len(draws) == 5
    losses = []
    for i in range(1, 5):
        inputs, labels = batches[i % 2]
        loss = step(inputs, labels).item()
        got = {n: w.main_grad.clone() for n, w in model.named_parameters()}
        now = torch.tensor([i], device="cuda")
        runner.zero_main_grads(model)
        with dropout.replaying([d._replace(step=now) for d in draws]):
            eager = runner.forward_step(model, inputs, labels)
        assert eager.item() == loss, i
        for n, w in model.named_parameters():
            assert torch.equal(w.main_grad, got[n]), (i, n)
        del eager
        losses.append(loss)
    assert len(set(losses)) == 4


def test_hooks_see_what_they_saw():
    """A hook on a part of a plain MLP gets that part's own result; the layer's result does not change beyond a rounding."""
    model = build(layer_norm_params=LN, layer=PLAIN)
    inputs, _ = batch()
    with torch.no_grad():
        want = model(inputs)
        mlp = model.get_submodule("3").mlp
        seen = []
        hooks = [mlp.register_forward_hook(lambda m, i, o: seen.append(o)), mlp.down_proj.register_forward_hook(lambda m, i, o: seen.append(o))]
        got = model(inputs)
        for h in hooks:
            h.remove()
    assert len(seen) == 2 and all(o[1] is mlp.down_proj.bias for o in seen) and torch.equal(seen[0][0], seen[1][0])
    assert ((got.double() - want.double()).norm() / want.double().norm()).item() <= 1e-2


def test_options_that_do_not_exist_are_refused():
    for kw, error in ((dict(hidden_dropout=1.5), ValueError), (dict(hidden_dropout=-0.1), ValueError), (dict(layer=dict(mlp_bias=True)), NotImplementedError),
                      (dict(layer=dict(glu_activation="relu")), NotImplementedError), (dict(layer=dict(bias_gelu_fusion=True)), ValueError),
                      (dict(layer_norm_params={"type": "scale_norm"}), NotImplementedError), (dict(layer=dict(attention_dropout=0.1)), AssertionError)):
        with pytest.raises(error):
            build(**kw)
