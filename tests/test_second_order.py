"""Differentiating twice: the backward kernels have no derivative of their own, which is an error where it is asked for and nothing where it is not."""
import pytest
import torch

from easyllm_amd import functional as F
from easyllm_amd.checkpointing import checkpoint


def test_a_recomputed_chunk_is_differentiated_once():
    x = torch.ones(3, requires_grad=True)
    y = checkpoint(lambda v: v * v * v, x)
    (g,) = torch.autograd.grad(y.sum(), x, create_graph=True)
    assert torch.equal(g.detach(), torch.full((3,), 3.0))
    with pytest.raises(RuntimeError, match="twice"):
        torch.autograd.grad((g * g + x).sum(), x)  # (not what is left without g's part)


def test_a_sum_is_differentiated_as_often_as_one_likes(monkeypatch):
    monkeypatch.setattr(F.K, "add", lambda a, b: a + b)
    x = torch.full((3,), 2.0, requires_grad=True)
    (g,) = torch.autograd.grad((F.add(x, x) ** 3).sum(), x, create_graph=True)
    (h,) = torch.autograd.grad(g.sum(), x)
    assert torch.equal(h, torch.full((3,), 8 * 6 * 2.0))


def rnd(*shape, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").bfloat16()


def calls():
    ids = lambda: torch.arange(6, device="cuda").view(2, 3)  # noqa: E731

    def rotary(q, k):
        from easyllm_amd.positional_embeddings import RotaryEmbedding
        cos, sin = RotaryEmbedding(64, precision=torch.bfloat16).cuda().tables(5, q.device)
        return F.apply_rotary_pair(q, k, cos, sin)
    head, mat, vec = (5, 1, 2, 64), (10, 64), (64,)
    return {
        "linear": (lambda x, w: F.linear(x, w), (mat, (72, 64))), "fan_out_linear": (lambda x, w, v: F.fan_out_linear(x, w, v), (mat, (72, 64), (72, 64))),
        "linear_fp32_output": (lambda x, w: F.linear_fp32_output(x, w), (mat, (72, 64))), "bias_add": (lambda x, b: F.bias_add(x, b), (mat, vec)),
        "linear_act": (lambda x, w, b, r: F.linear_act(x, w, b, "gelu", r), (mat, (72, 64), (72,), (10, 72))),
        "linear_act, no activation": (lambda x, w: F.linear_act(x, w), (mat, (72, 64))),
        "rmsnorm": (lambda x, w: F.rmsnorm(x, w, 1e-6), (mat, vec)), "rmsnorm_pass": (lambda x, w: F.rmsnorm_pass(x, w, 1e-6), (mat, vec)),
        "add_rmsnorm": (lambda x, r, w: F.add_rmsnorm(x, r, w, 1e-6), (mat, mat, vec)), "layer_norm": (lambda x, w, b: F.layer_norm(x, w, b), (mat, vec, vec)),
        "layer_norm_pass": (lambda x, w: F.layer_norm_pass(x, w), (mat, vec)), "add_layer_norm": (lambda x, r, w: F.add_layer_norm(x, r, w), (mat, mat, vec)),
        "dropout_add_layer_norm": (lambda x, r, w, b: F.dropout_add_layer_norm(x, r, w, None, bias=b, p=0.5, rng=(1, 2)), (mat, mat, vec, vec)),
        "dropout_add_rmsnorm": (lambda x, r, w: F.dropout_add_rmsnorm(x, r, w, p=0.5, rng=(1, 2)), (mat, mat, vec)),
        "dropout_add": (lambda x, r, b: F.dropout_add(x, r, b, p=0.5, rng=(1, 2)), (mat, mat, vec)), "swiglu": (lambda g, u: F.swiglu(g, u), (mat, mat)),
        "rotary": (rotary, (head, head)), "flash_attention": (lambda q, k, v: F.flash_attention(q, k, v), (head, head, head)),
        "embedding": (lambda w: F.embedding(ids(), w), ((8, 64),)), "transpose01": (lambda x: F.transpose01(x), ((3, 2, 64),)),
        "to_fp32": (lambda x: F.to_fp32(x), (mat,)), "loss": (lambda x: F.vocab_parallel_cross_entropy(x, torch.arange(10, device="cuda")), (mat,)),
        "fused loss": (lambda x: F.fused_cross_entropy_loss(x, torch.arange(10, device="cuda")), (mat,)),
    }


NAMES = ["linear", "fan_out_linear", "linear_fp32_output", "bias_add", "linear_act", "linear_act, no activation", "rmsnorm", "rmsnorm_pass", "add_rmsnorm", "layer_norm",
         "layer_norm_pass", "add_layer_norm", "dropout_add_layer_norm", "dropout_add_rmsnorm", "dropout_add", "swiglu", "rotary", "flash_attention", "embedding", "transpose01",
         "to_fp32", "loss", "fused loss"]


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_an_operator_is_differentiated_once(name):
    call, shapes = calls()[name]
    assert sorted(calls()) == sorted(NAMES)
    leaves = [rnd(*s, seed=i).requires_grad_(True) for i, s in enumerate(shapes)]

    def total():
        outs = call(*leaves)
        return sum((o.float() ** 2).sum() for o in (outs if isinstance(outs, tuple) else (outs,)))
    once = torch.autograd.grad(total(), leaves)
    twice = torch.autograd.grad(total(), leaves, create_graph=True)
    for a, b in zip(once, twice):
        assert torch.equal(a, b.detach())
    passed_on = {"linear_act": 3, "dropout_add": 1, "bias_add": 0}.get(name)  # that input's gradient is the one that arrived
    for i, g in enumerate(twice):
        if i == passed_on:  # 2 y, whose square's derivative is four times that of y's square
            (h,) = torch.autograd.grad((g.float() ** 2).sum(), leaves[0])
            assert ((h.double() - 4 * once[0].double()).norm() / (4 * once[0].double()).norm()).item() <= 2e-2  # (a few roundings to bf16)
            continue
        with pytest.raises(RuntimeError, match="twice"):  # (alone, and where the rest of a sum could be differentiated)
            torch.autograd.grad((g.float() ** 2).sum() + (leaves[0].float() ** 2).sum(), leaves[0])
