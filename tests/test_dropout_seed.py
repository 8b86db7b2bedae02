"""Which seed the draws of a process take (CPU)."""
import pytest
import torch

from easyllm_amd import dropout


@pytest.fixture
def unseeded(monkeypatch):
    """As a process starts: nobody has seeded dropout."""
    state = torch.get_rng_state()
    for name, value in (("_seed", None), ("_calls", 0), ("_given", False)):
        monkeypatch.setattr(dropout, name, value, raising=False)
    yield
    torch.set_rng_state(state)


def numbers(n):
    return [dropout.next_draw()[:2] for _ in range(n)]


def test_without_a_seed_of_its_own_torchs_counts(unseeded):
    torch.manual_seed(11)
    assert numbers(2) == [(11, 0), (11, 1)] and dropout.get_state() == (11, 2)
    torch.manual_seed(12)
    assert dropout.get_state() == (12, 0) and numbers(2) == [(12, 0), (12, 1)]
    torch.manual_seed(11)
    assert numbers(1) == [(11, 0)]
    torch.manual_seed(11)  # (not to be told from none)
    assert numbers(1) == [(11, 1)]


@pytest.mark.parametrize("seed", [lambda: dropout.manual_seed(5), lambda: dropout.set_state((5, 0))])
def test_one_of_its_own_stays(unseeded, seed):
    torch.manual_seed(11)
    numbers(1)
    seed()
    torch.manual_seed(12)
    assert numbers(2) == [(5, 0), (5, 1)]
