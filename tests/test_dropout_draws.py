"""Dropout's numbers where a forward pass is repeated (CPU)."""
import pytest
import torch

from easyllm_amd import dropout
from easyllm_amd.checkpointing import checkpoint


@pytest.fixture(autouse=True)
def draws_of_their_own():
    kept = dropout.get_state()
    dropout.manual_seed(7)
    yield
    dropout.set_state(kept)


def test_a_repetition_that_draws_less_than_the_forward_did_is_refused():
    with dropout.recording() as draws:
        dropout.next_draw()
        dropout.next_draw()
    with pytest.raises(RuntimeError, match="1 of 2"):
        with dropout.replaying(draws):
            dropout.next_draw()
    with pytest.raises(KeyError):  # (what went wrong inside is what is raised)
        with dropout.replaying(draws):
            raise KeyError
    with dropout.replaying(draws):
        assert [dropout.next_draw(), dropout.next_draw()] == draws
    assert dropout.next_draw() == (7, 2, None)  # (nothing is being replayed any more)


def test_a_chunk_that_is_put_into_evaluation_before_its_backward_is_refused():
    layer = torch.nn.Module()

    def forward(x):
        return x * dropout.next_draw().offset if layer.training else x
    x = torch.ones(3, requires_grad=True)
    y = checkpoint(forward, x)
    layer.eval()
    with pytest.raises(RuntimeError, match="0 of 1"):
        y.sum().backward()


def drawing(x):
    scale = 1 + dropout.next_draw().offset
    return x * x * scale  # (x is kept, so a recomputation happens, and gets this far)


@pytest.mark.parametrize("reentrant", [True, False])
def test_a_recomputation_that_does_not_replay_is_refused(reentrant):
    """Another library's checkpointing: its second forward would draw a mask of its own."""
    from torch.utils.checkpoint import checkpoint as other
    x = torch.ones(3, requires_grad=True)
    y = other(drawing, x, use_reentrant=reentrant)
    with pytest.raises(RuntimeError, match="inside a backward pass"):
        y.sum().backward()


def test_a_recomputation_that_replays_goes_on():
    from torch.utils.checkpoint import checkpoint as other
    x = torch.ones(3, requires_grad=True)
    draws = []

    def chunk(v):
        if draws:
            with dropout.replaying(draws):
                return drawing(v)
        with dropout.recording() as made:
            v = drawing(v)
        draws.extend(made)
        return v
    dropout.next_draw()
    other(chunk, x, use_reentrant=False).sum().backward()
    assert torch.equal(x.grad, torch.full((3,), 4.0))
    assert dropout.next_draw().offset == 2
