"""Frequencies of rotary positions under captured graphs."""
import pytest
import torch

pytestmark = pytest.mark.gpu

SCALINGS = {"dynamic": {"type": "dynamic", "factor": 2.0, "original_length": 16}, "linear": {"type": "linear", "factor": 3.0}, "yarn": {"type": "yarn", "factor": 4.0, "original_length": 32}, "none": None}


def rnd(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").bfloat16()


def small_tensors():
    """What a freed block of frequencies would be used for next."""
    return [torch.full((n,), 7.0, dtype=torch.float64, device="cuda") for n in (8, 16, 24, 32, 64) for _ in range(200)]


@pytest.mark.parametrize("name", SCALINGS)
def test_a_captured_call_outlives_whatever_the_module_does(name):
    from easyllm_amd.positional_embeddings import RotaryEmbedding
    rope = RotaryEmbedding(64, rotary_dim=48, interleaved=True, scaling=SCALINGS[name]).cuda()
    q, k, dq, dk = rnd(40, 2, 4, 64, seed=1).requires_grad_(), rnd(40, 2, 2, 64, seed=2).requires_grad_(), rnd(40, 2, 4, 64, seed=3), rnd(40, 2, 2, 64, seed=4)

    def step():
        outs = rope.rotate(q, k)
        return [*(y.detach() for y in outs), *torch.autograd.grad(outs, (q, k), (dq, dk))]

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    other = {"inv_freq": rope.inv_freq.clone() * 0.75}
    for between in (lambda: rope.rotate(rnd(300, 2, 4, 64), None), lambda: rope.load_state_dict(dict(rope.state_dict())), lambda: rope.load_state_dict(other), rope.cuda):
        between()
        torch.cuda.synchronize()
        keep = small_tensors()
        with torch.no_grad():
            q.copy_(rnd(40, 2, 4, 64, seed=5))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, step())), between
        del keep


@pytest.mark.parametrize("name", SCALINGS)
def test_a_captured_training_step_does_too(name):
    from easyllm_amd import runner
    torch.manual_seed(5)
    cfg = dict(num_layers=2, hidden_size=128, num_attention_heads=2, intermediate_size=136, vocab_size=72, seq_length=64, bf16=True, fp32_logits=False, checkpoint_activations=False,
               position_embedding_kwargs=dict(interleaved=True, scaling=SCALINGS[name]))
    model = runner.build_model({"type": "llama_custom", "kwargs": cfg}).cuda()
    runner.attach_main_grads(model)

    def batch(seed, s=64):
        ids = torch.randint(0, 72, (2, s), device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))
        return (ids, torch.arange(s, device="cuda").expand(2, s).contiguous(), None), (ids.roll(-1, 1), torch.ones(2, s, device="cuda"))

    step = runner.GraphedStep(model, *batch(1))
    for seed in (2, 3, 4):
        with torch.no_grad():
            model(batch(seed, 200)[0])
        model.load_state_dict({n: v.clone() for n, v in model.state_dict().items()})
        torch.cuda.synchronize()
        keep = small_tensors()
        loss = step(*batch(seed))
        torch.cuda.synchronize()
        step.flush()
        captured = loss.item(), {n: p.main_grad.clone() for n, p in model.named_parameters()}
        runner.zero_main_grads(model)
        eager = runner.forward_step(model, *batch(seed))
        assert eager.item() == captured[0] and all(torch.equal(p.main_grad, captured[1][n]) for n, p in model.named_parameters())
        del eager, keep


def test_lengths_that_change_stop_nothing(monkeypatch):
    """Ten lengths in turn, forward and backward: no call waits for the device."""
    from easyllm_amd.positional_embeddings import RotaryEmbedding
    rope = RotaryEmbedding(64, scaling=SCALINGS["dynamic"]).cuda()
    inputs = [(rnd(s, 2, 4, 64, seed=s).requires_grad_(), rnd(s, 2, 2, 64, seed=s + 1)) for s in range(8, 58, 5)]

    def waits(*_):
        raise AssertionError("a call waited for the device")
    monkeypatch.setattr(torch.cuda, "synchronize", waits)
    torch.cuda.set_sync_debug_mode("error")
    try:
        for q, k in inputs:
            y, z = rope.rotate(q, k)
            torch.autograd.grad(y, q, torch.ones_like(y))
    finally:
        torch.cuda.set_sync_debug_mode("default")


def test_an_evaluation_under_inference_mode_and_a_training_step_behind_it():
    from easyllm_amd.positional_embeddings import RotaryEmbedding
    for scaling in SCALINGS.values():
        rope = RotaryEmbedding(64, rotary_dim=32, scaling=scaling).cuda()
        q = rnd(40, 2, 4, 64)
        with torch.inference_mode():
            seen = rope.rotate(q, None)[0]
        leaf = q.clone().requires_grad_()
        y = rope.rotate(leaf, None)[0]
        assert torch.equal(seen, y) and torch.autograd.grad(y, leaf, torch.ones_like(y))[0].shape == q.shape


def test_a_cast_that_leaves_the_weights_leaves_a_captured_call():
    """bf16 weights stay where they are under .bfloat16(), and a graph of them may be replayed; inv_freq does not."""
    from easyllm_amd.positional_embeddings import RotaryEmbedding
    rope = RotaryEmbedding(64, scaling=SCALINGS["yarn"]).cuda()
    q = rnd(40, 2, 4, 64)
    want = rope.rotate(q, None)[0]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = rope.rotate(q, None)[0]
    rope.bfloat16()
    torch.cuda.synchronize()
    keep = small_tensors()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(captured, want)
    del keep


def test_a_document_is_turned_alone_as_it_is_packed():
    """With a length in the scaling, whatever lies in the row beside it."""
    from easyllm_amd.positional_embeddings import RotaryEmbedding
    rope = RotaryEmbedding(64, scaling=dict(SCALINGS["dynamic"], length=90)).cuda()
    lengths = (12, 40, 7, 31)
    q, k = rnd(sum(lengths), 1, 4, 64, seed=1), rnd(sum(lengths), 1, 2, 64, seed=2)
    ids, cu = torch.cat([torch.arange(n) for n in lengths])[None].cuda(), torch.tensor([0, 12, 52, 59, 90]).cuda()
    packed = rope.rotate(q, k, ids, cu)
    for first, n in zip((0, 12, 52, 59), lengths):
        alone = rope.rotate(q[first:first + n], k[first:first + n])
        assert all(torch.equal(a, b[first:first + n]) for a, b in zip(alone, packed))


@pytest.mark.parametrize("packed", [False, True])
def test_a_stack_with_a_dynamic_scaling_of_a_length(monkeypatch, packed):
    """Loss and gradients against 64 bits, of frequencies by the rule: inv_freq (2 length / 48 - 1)^(-j / (n - 1)), here of 512 tokens and 24 frequencies.  (A power and a product in 64 bits: a few
    times 2^-53.)"""
    import test_long_context_training_gpu as T
    name = "a larger base for 512 tokens"
    monkeypatch.setitem(T.STACKS, name, (dict(rotary_dim=48, scaling={"type": "dynamic", "factor": 2.0, "original_length": 48, "length": 512}), "silu"))
    rope = T.build(name).get_submodule("3").self_attn.rotary_emb
    want = rope.inv_freq.double() * (2 * 512 / 48 - 1) ** -(torch.arange(24, dtype=torch.float64, device="cuda") / 23)
    assert bool(((rope.frequencies(T.S, torch.device("cuda", 0))[0] - want).abs() <= want * 2.0 ** -48).all())
    T.test_loss_and_gradients(name, packed)
