"""Traces of evaluations, replayed on other inputs."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def rnd(*shape, seed=0, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda") * scale).bfloat16()


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("op", ["rotary", "rotary alone", "gated mlp", "gated linear"])
def test_a_traced_evaluation_is_the_call(op):
    from easyllm_amd import functional as F
    inv_freq = 10000.0 ** -(torch.arange(32, device="cuda", dtype=torch.float64) / 32)
    call, *shapes = {"rotary": (lambda q, k: F.rotary_embed(q, k, inv_freq), (30, 2, 4, 64), (30, 2, 2, 64)),
                     "rotary alone": (lambda q: F.rotary_embed(q, None, inv_freq)[0], (30, 2, 4, 64)),
                     "gated mlp": (F.gated_mlp, (40, 64), (72, 64), (72, 64), (64, 72)), "gated linear": (F.gated_linear, (40, 64), (72, 64), (72, 64))}[op]
    values = lambda seed: [rnd(*s, seed=seed + i) for i, s in enumerate(shapes)]  # noqa: E731
    with torch.no_grad():
        traced = torch.jit.trace(call, values(1), check_trace=False)
        for seed in (2, 3):
            got, want = traced(*values(seed)), call(*values(seed))
            got, want = ((t,) if torch.is_tensor(t) else t for t in (got, want))
            assert all(torch.equal(a, b) for a, b in zip(got, want))
