"""Rotary tables under captured steps and behind evaluations."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def build(**kw):
    from easyllm_amd import runner
    torch.manual_seed(5)
    cfg = dict(num_layers=2, hidden_size=128, num_attention_heads=2, intermediate_size=136, vocab_size=72, seq_length=64, bf16=True, fp32_logits=False, checkpoint_activations=False, **kw)
    model = runner.build_model({"type": "llama_custom", "kwargs": cfg}).cuda()
    runner.attach_main_grads(model)
    return model


def batch(seed, s=64):
    ids = torch.randint(0, 72, (2, s), device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))
    return (ids, torch.arange(s, device="cuda").expand(2, s).contiguous(), None), (ids.roll(-1, 1), torch.ones(2, s, device="cuda"))


def results(model, loss):
    return loss.item(), {n: p.main_grad.clone() for n, p in model.named_parameters()}


@pytest.mark.parametrize("warmup", [2, 1])
def test_a_captured_step_outlives_longer_tables(warmup):
    from easyllm_amd import runner
    model = build()
    step = runner.GraphedStep(model, *batch(1), warmup=warmup)
    for seed in (2, 3, 4):
        with torch.no_grad():
            model(batch(seed, 200 * seed)[0])
        torch.cuda.synchronize()
        keep = [torch.full((64, 32), 7.0, device="cuda") for _ in range(100)]  # (where tables were)
        loss = step(*batch(seed))
        torch.cuda.synchronize()
        step.flush()
        captured = results(model, loss)
        runner.zero_main_grads(model)
        loss, grads = results(model, runner.forward_step(model, *batch(seed)))
        assert loss == captured[0] and all(torch.equal(grads[n], captured[1][n]) for n in grads)
        del keep


def test_tables_made_in_a_graph_are_no_one_elses():
    from easyllm_amd.positional_embeddings import RotaryEmbedding
    rope = RotaryEmbedding(64).cuda()
    device = torch.device("cuda", 0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = rope.tables(40, device)
    own = rope.tables(40, device)
    assert own[0] is not captured[0]
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(captured[0], own[0]) and torch.equal(captured[1], rope.tables(30, device)[1])


def test_a_step_behind_an_evaluation_under_inference_mode():
    from easyllm_amd import runner
    for native in (True, False):
        model, fresh = build(), build()
        for m in (model, fresh):
            for layer in (m.get_submodule("3"), m.get_submodule("4")):
                layer.native_call_flops = 1e12 if native else 0
        with torch.inference_mode():
            model(batch(1)[0])
        (loss, grads), (want, expected) = (results(m, runner.forward_step(m, *batch(2))) for m in (model, fresh))
        assert loss == want and all(torch.equal(grads[n], expected[n]) for n in grads)
