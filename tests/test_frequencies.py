"""What a module of rotary positions keeps of its frequencies, and for whom (CPU)."""
import copy
import pickle
import sys
import threading

import pytest
import torch

from easyllm_amd import positional_embeddings as P
from easyllm_amd.positional_embeddings import RotaryEmbedding

CPU = torch.device("cpu")
SCALINGS = [None, {"type": "linear", "factor": 3.0}, {"type": "dynamic", "factor": 2.0, "original_length": 16}, {"type": "yarn", "factor": 4.0, "original_length": 32}]


@pytest.mark.parametrize("scaling", SCALINGS)
def test_nothing_of_a_call_is_kept_for_the_next(scaling):
    """A captured graph holds no reference to a tensor that was there before it, and another stream or thread does not wait for one: a call's frequencies are its own."""
    rope = RotaryEmbedding(64, rotary_dim=32, scaling=scaling)
    held = lambda: {t.data_ptr() for t in vars(rope).values() if torch.is_tensor(t)} | {rope.inv_freq.data_ptr()}  # noqa: E731
    before = held()
    first, second = rope.frequencies(40, CPU), rope.frequencies(40, CPU)
    assert torch.equal(first[0], second[0]) and first[0].data_ptr() != second[0].data_ptr() and held() == before and not {first[0].data_ptr(), second[0].data_ptr()} & before
    want = rope.frequencies(7, CPU)[0].clone()
    rope.load_state_dict({"inv_freq": rope.inv_freq * 2})
    assert torch.equal(rope.frequencies(7, CPU)[0], 2 * want) and held() == before


@pytest.mark.parametrize("scaling", SCALINGS)
def test_an_evaluation_leaves_nothing_that_training_cannot_use(scaling):
    """Tensors made under inference_mode cannot be saved for a backward pass."""
    rope = RotaryEmbedding(64, rotary_dim=32, scaling=scaling)
    with torch.inference_mode():
        rope.frequencies(40, CPU)
    assert not rope.frequencies(40, CPU)[0].is_inference()


def test_threads_of_different_lengths_get_their_own():
    rope = RotaryEmbedding(64, scaling={"type": "dynamic", "factor": 2.0, "original_length": 16})
    lengths = range(20, 420, 100)
    want = {n: rope.frequencies(n, CPU)[0].clone() for n in lengths}
    wrong = []

    def ask(n):
        for _ in range(300):
            if not torch.equal(rope.frequencies(n, CPU)[0], want[n]):
                wrong.append(n)
    interval = sys.getswitchinterval()
    sys.setswitchinterval(1e-6)
    try:
        threads = [threading.Thread(target=ask, args=(n,)) for n in lengths]
        [t.start() for t in threads]
        [t.join() for t in threads]
    finally:
        sys.setswitchinterval(interval)
    assert not wrong


@pytest.mark.parametrize("scaling", SCALINGS)
def test_a_module_that_is_cast_or_copied(scaling):
    """The factors stay in 64 bits whatever inv_freq is held in; a module on no device at all goes on to a real one."""
    rope = RotaryEmbedding(64, rotary_dim=32, scaling=scaling)
    want = rope.frequencies(40, CPU)[0]
    low = copy.deepcopy(rope).bfloat16()
    off = (low.frequencies(40, CPU)[0] - want).abs() / want
    assert low.frequencies(40, CPU)[0].dtype is torch.float64 and bool((off <= 2.0 ** -8).all())
    assert torch.equal(pickle.loads(pickle.dumps(rope)).frequencies(40, CPU)[0], want)
    with torch.device("meta"):
        empty = RotaryEmbedding(64, rotary_dim=32, scaling=scaling)
    empty = empty.to_empty(device="cpu")
    empty.load_state_dict(rope.state_dict())
    assert torch.equal(empty.frequencies(40, CPU)[0], want)


@pytest.mark.parametrize("scaling", SCALINGS)
def test_a_scale_factor_divides_in_64_bits(scaling):
    """The quotient is off by a few roundings of 2^-53 (the division's, or a reciprocal's and two products'), where a division in 32 bits is off by up to 2^-24: at position 10^6 0.03 of a radian."""
    rope, whole = (RotaryEmbedding(64, scale_factor=f, scaling=scaling) for f in (3.0, 1.0))
    got, want = rope.frequencies(40, CPU)[0], whole.frequencies(40, CPU)[0] / 3.0
    assert got.dtype is torch.float64 and bool(((got - want).abs() <= want * 2.0 ** -50).all())


DYNAMIC = {"type": "dynamic", "factor": 2.0, "original_length": 16}


def test_a_row_of_several_texts_has_no_length_of_its_own():
    """A document of 12 tokens is not stretched when it is alone; in a row of 40 it was turned as one of 40, and one at position 1000 of a longer text as if it began there."""
    q = torch.zeros(40, 1, 2, 64, dtype=torch.bfloat16)
    ids = torch.cat((torch.arange(12), torch.arange(28)))[None]
    rope = RotaryEmbedding(64, scaling=DYNAMIC)
    assert torch.equal(rope.frequencies(12, CPU)[0], rope.inv_freq.double()) and not torch.equal(rope.frequencies(40, CPU)[0], rope.inv_freq.double())
    for kw in (dict(position_ids=ids), dict(cu_seqlens=torch.tensor([0, 12, 40])), dict(position_ids=ids, cu_seqlens=torch.tensor([0, 12, 40]))):
        with pytest.raises(ValueError, match='needs a "length"'):
            rope.rotate(q, q, **kw)


def test_texts_that_have_a_length_are_turned(monkeypatch):
    """Whole rows go by their length; packed ones by the scaling's own, whatever they hold."""
    seen = []
    monkeypatch.setattr(P.F_, "rotary_embed", lambda q, k, inv_freq, ids, **kw: seen.append(inv_freq) or (q, k))
    q, ids, cu = torch.zeros(40, 1, 2, 64), torch.arange(40)[None], torch.tensor([0, 12, 40])
    RotaryEmbedding(64, scaling=DYNAMIC).rotate(q, q)
    fixed = RotaryEmbedding(64, scaling=dict(DYNAMIC, length=100))
    fixed.rotate(q, q, ids, cu)
    fixed.rotate(q[:12], q[:12], ids[:, :12])
    j = torch.arange(32, dtype=torch.float64)
    for got, length in zip(seen, (40, 100, 100)):
        want = fixed.inv_freq.double() * (2 * length / 16 - 1) ** (-j / 31)
        assert bool(((got - want).abs() <= want * 2.0 ** -48).all())
    for scaling in (None, {"type": "linear", "factor": 3.0}, {"type": "yarn", "factor": 4.0, "original_length": 32}):
        RotaryEmbedding(64, rotary_dim=32, scaling=scaling).rotate(q, q, ids, cu)


def test_an_attention_tells_its_positions_of_documents(monkeypatch):
    from easyllm_amd import runner, transformer
    cfg = dict(num_layers=1, hidden_size=64, num_attention_heads=1, intermediate_size=72, vocab_size=64, seq_length=16, bf16=True, position_embedding_kwargs={"scaling": DYNAMIC})
    attn = runner.build_model({"type": "llama_custom", "kwargs": cfg}).get_submodule("3").self_attn
    monkeypatch.setattr(transformer.F_, "fan_out_linear", lambda x, *weights: tuple(x @ w.t() for w in weights))
    with pytest.raises(ValueError, match='needs a "length"'):
        attn(torch.zeros(40, 1, 64, dtype=torch.bfloat16), None, torch.tensor([0, 12, 40]))
