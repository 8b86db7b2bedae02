"""Hooks on a layer's projections, and projections that stand in for them, are not passed by.

Tolerance, before any run: without a hook the two differ by a few roundings to bf16 in what is stored between the products, 2^-9 of its size each: 1 % of the
result's norm is five times that and more."""
import pytest
import torch

pytestmark = pytest.mark.gpu

PLAIN = dict(glu_activation=None, mlp_bias=True)
STACKS = {"plain MLP, biases": (dict(PLAIN), "up_proj"), "plain MLP, tanh": (dict(glu_activation=None, use_openai_gelu=True), "up_proj"),
          "gated MLP, gate": ({}, "gate_proj"), "gated MLP, up": ({}, "up_proj"), "attention, q": ({}, "q_proj"), "attention, v": ({}, "v_proj"),
          "attention, k with a bias": (dict(attention_qkv_bias=True), "k_proj"), "packed projections": (dict(qkv_pack=True), "wqkv")}


def build(layer):
    from easyllm_amd import runner
    torch.manual_seed(5)
    cfg = dict(num_layers=1, hidden_size=256, num_attention_heads=4, intermediate_size=712, vocab_size=520, seq_length=96, bf16=True,
               checkpoint_activations=False, fp32_logits=False, transformer_layer_params=dict(layer))
    model = runner.build_model({"type": "llama_custom", "kwargs": cfg}).cuda()
    with torch.no_grad():
        for p in model.parameters():
            if p.dim() == 1:
                p.add_(0.2 * torch.randn_like(p))
    return model


def find(layer, name):
    return getattr(layer.mlp if hasattr(layer.mlp, name) else layer.self_attn, name)


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


def test_a_residual_does_not_pass_a_hooked_down_projection_by():
    mlp = build(PLAIN).get_submodule("3").mlp
    x, r = (torch.randn(40, 256, device="cuda").bfloat16() for _ in range(2))
    want, bias = mlp(x, residual=r)
    seen = []
    hook = mlp.down_proj.register_forward_hook(lambda m, i, o: seen.append(o))
    got, bias2 = mlp(x, residual=r)
    hook.remove()
    assert len(seen) == 1 and bias is None and bias2 is None and close(got, want)
