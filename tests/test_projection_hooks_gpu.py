"""Hooks on a layer's projections and norms, and modules that stand in for them, are not passed by.

Tolerance, before any run: without a hook the two differ by a few roundings to bf16 in what is stored between the products, 2^-9 of its size each: 1 % of the
result's norm is five times that and more."""
import pytest
import torch

pytestmark = pytest.mark.gpu

PLAIN = dict(glu_activation=None, mlp_bias=True)
STACKS = {"plain MLP, biases": (dict(PLAIN), "up_proj"), "plain MLP, tanh": (dict(glu_activation=None, use_openai_gelu=True), "up_proj"),
          "gated MLP, gate": ({}, "gate_proj"), "gated MLP, up": ({}, "up_proj"), "attention, q": ({}, "q_proj"), "attention, v": ({}, "v_proj"),
          "attention, k with a bias": (dict(attention_qkv_bias=True), "k_proj"), "packed projections": (dict(qkv_pack=True), "wqkv")}


def build(layer, **kw):
    from easyllm_amd import runner
    torch.manual_seed(5)
    cfg = dict(num_layers=1, hidden_size=256, num_attention_heads=4, intermediate_size=712, vocab_size=520, seq_length=96, bf16=True,
               checkpoint_activations=False, fp32_logits=False, transformer_layer_params=dict(layer), **{k: dict(v) if isinstance(v, dict) else v for k, v in kw.items()})
    model = runner.build_model({"type": "llama_custom", "kwargs": cfg}).cuda()
    with torch.no_grad():
        for p in model.parameters():
            if p.dim() == 1:
                p.add_(0.2 * torch.randn_like(p))
    return model


def find(layer, name):
    return next(getattr(m, name) for m in (layer, layer.mlp, layer.self_attn) if hasattr(m, name))


def close(a, b):
    return ((a.double() - b.double()).norm() / b.double().norm()).item() <= 1e-2


def run(layer, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(40, 2, 256, generator=g, device="cuda").bfloat16().requires_grad_(True)
    y = layer(x)
    grads = torch.autograd.grad(y, [x, *layer.parameters()], torch.ones_like(y))
    return y.detach(), grads


@pytest.mark.parametrize("name", STACKS)
def test_a_hook_sees_the_projections_own_call(name):
    params, part = STACKS[name]
    layer = build(params).get_submodule("3")
    want, want_grads = run(layer)
    seen = []
    module = find(layer, part)
    hooks = [module.register_forward_pre_hook(lambda m, i: seen.append(i[0].detach().clone())),
             module.register_forward_hook(lambda m, i, o: seen.append((o[0].detach().clone(), o[1])))]
    got, grads = run(layer)
    for h in hooks:
        h.remove()
    assert len(seen) == 2
    x, (y, bias) = seen
    product = x.double() @ module.weight.double().t()
    if bias is None and module.bias is not None:
        product = product + module.bias.double()
    assert close(y, product) and (bias is module.bias if module.skip_bias_add else bias is None)
    assert close(got, want) and all(close(a, b) for a, b in zip(grads, want_grads))
    assert torch.equal(run(layer)[0], want)


@pytest.mark.parametrize("name", STACKS)
def test_what_a_hook_returns_counts(name):
    """Twice the projection, against the projection itself through a hook: the same launches, other values."""
    params, part = STACKS[name]
    layer = build(params).get_submodule("3")
    results = []
    for factor in (1, 2):
        hook = find(layer, part).register_forward_hook(lambda m, i, o: (o[0] * factor, o[1]))
        results.append(run(layer))
        hook.remove()
    (one, _), (two, grads) = results
    assert not torch.equal(one, two) and all(torch.isfinite(g).all() for g in grads)


@pytest.mark.parametrize("name", STACKS)
def test_a_projection_of_another_class_is_called(name):
    params, part = STACKS[name]
    layer = build(params).get_submodule("3")
    module = find(layer, part)

    class Adapted(type(module)):
        share = 0

        def forward(self, x):
            y, bias = super().forward(x)
            return y + self.share * y.detach().roll(1, -1), bias
    module.__class__ = Adapted
    without, _ = run(layer)
    Adapted.share = 3
    assert not torch.equal(run(layer)[0], without)


@pytest.mark.parametrize("name", [*STACKS, "gated MLP, down", "attention, o"])
def test_a_projection_that_wraps_another_is_called(name):
    """It has no weight of its own to go by."""
    params, part = STACKS.get(name) or ({}, {"gated MLP, down": "down_proj", "attention, o": "o_proj"}[name])
    layer = build(params).get_submodule("3")
    want, want_grads = run(layer)
    module, calls = find(layer, part), []

    class Wrapped(torch.nn.Module):
        def __init__(self, inner):
            super().__init__()
            self.inner = inner

        def forward(self, x):
            calls.append(x.shape)
            return self.inner(x)
    holder = next(m for m in (layer.mlp, layer.self_attn) if hasattr(m, part))
    setattr(holder, part, Wrapped(module))
    got, grads = run(layer)
    assert len(calls) == 1 and close(got, want) and all(close(a, b) for a, b in zip(grads, want_grads))


def test_a_residual_does_not_pass_a_hooked_down_projection_by():
    mlp = build(PLAIN).get_submodule("3").mlp
    x, r = (torch.randn(40, 256, device="cuda").bfloat16() for _ in range(2))
    want, bias = mlp(x, residual=r)
    seen = []
    hook = mlp.down_proj.register_forward_hook(lambda m, i, o: seen.append(o))
    got, bias2 = mlp(x, residual=r)
    hook.remove()
    assert len(seen) == 1 and bias is None and bias2 is None and close(got, want)


LN = dict(layer_norm_params={"type": "mixed_fused_norm"})
NORMED = {"RMSNorm": ({}, {}), "layer norm": (LN, {}), "layer norm, output bias": (LN, dict(PLAIN, attention_o_bias=True)),
          "RMSNorm, dropout": (dict(hidden_dropout=0.25), {}), "layer norm, dropout, output bias": (dict(LN, hidden_dropout=0.25), dict(PLAIN, attention_o_bias=True)),
          "layer norm, residual behind it": (LN, dict(apply_residual_connection_post_layernorm=True))}


@pytest.mark.parametrize("part", ["input_layernorm", "post_attention_layernorm"])
@pytest.mark.parametrize("name", NORMED)
def test_a_hook_sees_the_norms_own_call(name, part):
    """What goes in (for the second the residual sum, rounded), what comes out, and what the hook makes of it."""
    from easyllm_amd import dropout
    model, params = NORMED[name]
    layer = build(params, **model).get_submodule("3")
    with dropout.recording() as draws:
        want, want_grads = run(layer)
    norm, seen, factor = find(layer, part), [], 1

    def hook(m, i, o):
        seen.append((i[0].detach().clone(), o.detach().clone()))
        return o * factor
    handle = norm.register_forward_hook(hook)
    with dropout.replaying(draws):
        got, grads = run(layer)
    factor = 2
    with dropout.replaying(draws):
        twice, _ = run(layer)
    handle.remove()
    assert len(seen) == 2
    x, y = seen[0]
    x = x.double()
    if type(norm).__name__ == "RMSNorm":
        ref = x * (x.square().mean(-1, keepdim=True) + norm.eps).rsqrt() * norm.weight.double()
    else:
        ref = torch.nn.functional.layer_norm(x, (256,), norm.weight.double(), norm.bias.double(), norm.eps)
    assert close(y, ref) and close(got, want) and all(close(a, b) for a, b in zip(grads, want_grads))
    assert not torch.equal(twice, got)  # (the same launches; behind another norm twice as much may be nearly the same)


@pytest.mark.parametrize("name", NORMED)
def test_a_norm_of_another_class_is_called(name):
    """One that knows none of the fused forms."""
    model, params = NORMED[name]
    layer = build(params, **model).get_submodule("3")

    class Scale(torch.nn.Module):
        def forward(self, x):
            return x * 0.5
    layer.input_layernorm, layer.post_attention_layernorm = Scale(), Scale()
    y, grads = run(layer)
    assert torch.isfinite(y).all() and all(torch.isfinite(g).all() for g in grads)


@pytest.mark.parametrize("part", ["input_layernorm", "post_attention_layernorm"])
@pytest.mark.parametrize("name", ["RMSNorm", "layer norm", "RMSNorm, dropout"])
@pytest.mark.parametrize("how", ["subclass", "instance", "class"])
def test_a_norm_with_a_forward_of_its_own_is_called(name, part, how, monkeypatch):
    model, params = NORMED[name]
    layer = build(params, **model).get_submodule("3")
    norm, calls = find(layer, part), []
    original = type(norm).forward

    def forward(self, x):
        calls.append(x.shape)
        return original(self, x)
    if how == "subclass":
        norm.__class__ = type("Other", (type(norm),), {"forward": forward})
    elif how == "class":
        monkeypatch.setattr(type(norm), "forward", forward)
    else:
        monkeypatch.setattr(norm, "forward", lambda x: forward(norm, x))
    run(layer)
    assert calls == [(40, 2, 256)] * (2 if how == "class" else 1)
