"""What a module of rotary positions keeps of its frequencies, and for whom (CPU)."""
import pytest
import torch

from easyllm_amd import positional_embeddings as P
from easyllm_amd.positional_embeddings import RotaryEmbedding

CPU = torch.device("cpu")
SCALINGS = [None, {"type": "linear", "factor": 3.0}, {"type": "dynamic", "factor": 2.0, "original_length": 16}, {"type": "yarn", "factor": 4.0, "original_length": 32}]


@pytest.mark.parametrize("scaling", SCALINGS)
def test_a_captured_call_has_frequencies_of_its_own(monkeypatch, scaling):
    """A graph holds no reference to a tensor that was there before it: whatever replaces that one, the replays would read freed memory."""
    rope = RotaryEmbedding(64, rotary_dim=32, scaling=scaling)
    eager = rope.frequencies(40, CPU)
    assert rope.frequencies(40, CPU)[0] is eager[0]
    monkeypatch.setattr(P, "_capturing", lambda device: True)
    first, second = rope.frequencies(40, CPU), rope.frequencies(40, CPU)
    assert len({t.data_ptr() for t in (rope.inv_freq, eager[0], first[0], second[0])}) == 4
    assert torch.equal(first[0], eager[0]) and torch.equal(second[0], eager[0]) and first[1] == second[1] == eager[1]
    monkeypatch.undo()
    assert rope.frequencies(40, CPU)[0] is eager[0]  # (nor does anybody else read the graph's)


@pytest.mark.parametrize("scaling", SCALINGS)
def test_a_scale_factor_divides_in_64_bits(scaling):
    """The quotient is off by a few roundings of 2^-53 (the division's, or a reciprocal's and two products'), where a division in 32 bits is off by up to 2^-24: at position 10^6 0.03 of a radian."""
    rope, whole = (RotaryEmbedding(64, scale_factor=f, scaling=scaling) for f in (3.0, 1.0))
    got, want = rope.frequencies(40, CPU)[0], whole.frequencies(40, CPU)[0] / 3.0
    assert got.dtype is torch.float64 and bool(((got - want).abs() <= want * 2.0 ** -50).all())
