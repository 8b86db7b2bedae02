"""Whom a module's rotary tables are for (CPU; tables of the host's in place of the kernel's)."""
import pytest
import torch

from easyllm_amd import positional_embeddings as P
from easyllm_amd.positional_embeddings import RotaryEmbedding

CPU = torch.device("cpu")


@pytest.fixture
def rope(monkeypatch):
    def table(inv_freq, n, factor):
        angle = torch.arange(n)[:, None] / factor * inv_freq
        return torch.cos(angle), torch.sin(angle)
    monkeypatch.setattr(P.K, "rope_table", table)
    return RotaryEmbedding(32)


def test_tables_that_a_capture_was_given_stay(rope, monkeypatch):
    """A graph holds no reference to them: longer ones may take their place, not their memory."""
    rope.tables(10, CPU)
    monkeypatch.setattr(P, "_capturing", lambda device: True)
    given = rope.tables(8, CPU)
    assert rope.tables(10, CPU)[0] is given[0]
    monkeypatch.undo()
    monkeypatch.setattr(P.K, "rope_table", lambda inv_freq, n, factor: (torch.zeros(n, 16), torch.zeros(n, 16)))
    assert rope.tables(20, CPU)[0] is not given[0]
    held = [t for pair in rope._captured for t in pair]
    assert len(held) == 2 and all(a is b for a, b in zip(held, given))


def test_tables_that_a_capture_makes_are_the_graphs(rope, monkeypatch):
    """They hold nothing before its first replay, and may be overwritten behind any."""
    monkeypatch.setattr(P, "_capturing", lambda device: True)
    given = rope.tables(10, CPU)
    monkeypatch.setattr(P, "_capturing", lambda device: False)
    assert rope.tables(10, CPU)[0] is not given[0] and torch.equal(rope.tables(10, CPU)[0], given[0])


def test_tables_of_an_evaluation_train(rope):
    with torch.inference_mode():
        rope.tables(10, CPU)
    assert not any(t.is_inference() for t in rope.tables(10, CPU))
