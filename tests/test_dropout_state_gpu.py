"""Captured steps with dropout over the end of a process: what they keep, what goes on, and what is refused."""
import json

import pytest
import torch

pytestmark = pytest.mark.gpu


def build(p=0.2, **kw):
    from easyllm_amd import runner
    torch.manual_seed(5)
    cfg = dict(num_layers=2, hidden_size=256, num_attention_heads=4, intermediate_size=712, vocab_size=520, seq_length=96, bf16=True, checkpoint_activations=False,
               fp32_logits=False, hidden_dropout=p)
    cfg.update(kw)
    model = runner.build_model({"type": "llama_custom", "kwargs": cfg}).cuda()
    runner.attach_main_grads(model)
    return model


def batch(seed=1, b=2, s=96):
    g = torch.Generator().manual_seed(seed)
    tokens, labels = torch.randint(0, 520, (b, s), generator=g).cuda(), torch.randint(0, 520, (b, s), generator=g).cuda()
    return (tokens, torch.arange(s).expand(b, s).contiguous().cuda(), None), (labels, torch.ones(b, s, device="cuda"))


@pytest.fixture(autouse=True)
def draws_of_their_own():
    from easyllm_amd import dropout
    kept = dropout.get_state()
    yield
    dropout.set_state(kept)


def replayed(step, n):
    out = []
    for i in range(n):
        loss = step(*batch(seed=i)).item()
        out.append((loss, {k: w.main_grad.clone() for k, w in step.model.named_parameters()}))
    return out


@pytest.mark.parametrize("recompute", [False, True])
def test_a_resumed_run_draws_what_the_uninterrupted_one_does(recompute):
    from easyllm_amd import dropout, runner
    dropout.manual_seed(41)
    dropout.next_draw()
    step = runner.GraphedStep(build(checkpoint_activations=recompute), *batch())
    before = replayed(step, 3)
    kept = json.loads(json.dumps({"eager": dropout.get_state(), "step": step.dropout_state()}))
    want, eager = replayed(step, 3), [dropout.next_draw() for _ in range(3)]
    assert len({loss for loss, _ in before + want}) == 6
    del step
    dropout.manual_seed(12345)  # another process, which has drawn numbers already
    dropout.next_draw()
    dropout.set_state(kept["eager"])
    again = runner.GraphedStep(build(checkpoint_activations=recompute), *batch(seed=3), dropout_state=kept["step"])
    assert [dropout.next_draw() for _ in range(3)] == eager
    for (a, ga), (b, gb) in zip(replayed(again, 3), want):
        assert a == b
        for n in ga:
            assert torch.equal(ga[n], gb[n]), n
    assert again.dropout_state() == {"step": 6, "draws": [tuple(d) for d in kept["step"]["draws"]]}


def test_a_run_that_kept_no_step_draws_numbers_of_its_own():
    """Captured behind set_state, its calls come after all that the first run's were given."""
    from easyllm_amd import dropout, runner
    dropout.manual_seed(41)
    step = runner.GraphedStep(build(), *batch())
    first = step.dropout_state()["draws"]
    kept = dropout.get_state()
    dropout.manual_seed(0)
    dropout.set_state(kept)
    second = runner.GraphedStep(build(), *batch()).dropout_state()
    assert second["step"] == 0 and not set(first) & set(second["draws"])


def test_a_step_captured_before_the_draws_were_restored_is_refused():
    """It would repeat, from its first replay on, the masks that the interrupted run began with."""
    from easyllm_amd import dropout, runner
    dropout.manual_seed(41)
    step = runner.GraphedStep(build(), *batch())
    step(*batch())
    for again in (lambda: dropout.set_state(dropout.get_state()), lambda: dropout.manual_seed(41)):
        again()
        with pytest.raises(RuntimeError, match="capture again"):
            step(*batch())
    assert step.dropout_state()["step"] == 1
    plain = runner.GraphedStep(build(p=0), *batch())  # (nothing to draw, nothing to mind)
    dropout.manual_seed(1)
    plain(*batch())
    assert plain.dropout_state() == {"step": 0, "draws": []}


def test_the_state_of_another_model_is_refused():
    from easyllm_amd import runner
    state = runner.GraphedStep(build(), *batch()).dropout_state()
    assert len(state["draws"]) == 5
    for layers, text in ((1, "3 of 5 dropout calls"), (3, "more dropout calls")):
        with pytest.raises(RuntimeError, match=text):
            runner.GraphedStep(build(num_layers=layers), *batch(), dropout_state=state)
