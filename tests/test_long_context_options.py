"""Options of rotary positions, gated MLPs and the optimizer's state, on the host (CPU)."""
import ctypes
import math

import pytest
import torch

from easyllm_amd import _lib, kernels as K, optimizer
from easyllm_amd.positional_embeddings import RotaryEmbedding, scaled_frequencies


def theirs(kind, n, base, length, **scaling):
    """transformers' frequencies for a head of 2 n"""
    from transformers import LlamaConfig
    from transformers.modeling_rope_utils import ROPE_INIT_FUNCTIONS
    params = dict(rope_type=kind, rope_theta=base, **scaling)
    cfg = LlamaConfig(hidden_size=8 * n, num_attention_heads=4, max_position_embeddings=int(scaling.get("original_max_position_embeddings", 2048)), rope_theta=base)
    cfg.rope_scaling = params
    cfg.rope_parameters = params
    return ROPE_INIT_FUNCTIONS[kind](cfg, torch.device("cpu"), seq_len=length)


@pytest.mark.parametrize("n", [16, 32, 64])
@pytest.mark.parametrize("base", [10000.0, 500000.0])
@pytest.mark.parametrize("kind,length", [("linear", None), ("dynamic", 1000), ("dynamic", 5000), ("dynamic", 16384), ("yarn", None)])
def test_scaled_frequencies_are_the_librarys(kind, length, n, base):
    """(in fp32 there: a few roundings, of exponents of up to 13 in powers of the base)"""
    inv_freq = base ** -(torch.arange(n, dtype=torch.float64) / n)
    scaling = {"type": kind, "factor": 4.0, "original_length": 2048} if kind != "linear" else {"type": kind, "factor": 4.0}
    got, factor = scaled_frequencies(inv_freq, base, scaling, length)
    want, want_factor = theirs(kind, n, base, length, factor=4.0, **({"original_max_position_embeddings": 2048} if kind == "yarn" else {}))
    assert got.dtype is torch.float64 and torch.allclose(got, want.double(), rtol=1e-5, atol=0)
    assert abs(factor - want_factor) <= 1e-6


def test_frequencies_of_a_module():
    rope = RotaryEmbedding(64, base=10000, rotary_dim=32, scale_factor=2.0)
    assert rope.general and list(rope.state_dict()) == ["inv_freq"] and rope.inv_freq.shape == (16,)
    cpu = torch.device("cpu")
    got, factor = rope.frequencies(100, cpu)
    assert factor == 1.0 and torch.allclose(got, rope.inv_freq.double() / 2, rtol=1e-7)
    rope.load_state_dict({"inv_freq": torch.full((16,), 0.5)})
    assert torch.equal(rope.frequencies(100, cpu)[0], torch.full((16,), 0.25, dtype=torch.float64))
    longer = RotaryEmbedding(64, scaling={"type": "dynamic", "factor": 2.0, "original_length": 128})
    assert torch.equal(longer.frequencies(64, cpu)[0], longer.inv_freq.double())
    a, b = longer.frequencies(256, cpu)[0], longer.frequencies(512, cpu)[0]
    assert bool((a[1:] < longer.inv_freq.double()[1:]).all()) and bool((b[1:] < a[1:]).all())
    fixed = RotaryEmbedding(64, scaling={"type": "dynamic", "factor": 2.0, "original_length": 128, "length": 512})
    assert torch.equal(fixed.frequencies(7, cpu)[0], b)
    with pytest.raises(NotImplementedError):
        rope.tables(10, cpu)
    plain = RotaryEmbedding(64, rotary_dim=64)
    assert not plain.general and list(plain.state_dict()) == ["inv_freq"]


@pytest.mark.parametrize("kw,error", [(dict(rotary_dim=0), ValueError), (dict(rotary_dim=33), ValueError), (dict(rotary_dim=66), ValueError), (dict(scaling={"type": "ntk"}), NotImplementedError),
                                      (dict(scaling={"type": "linear"}), ValueError), (dict(scaling={"type": "linear", "factor": 0.5}), ValueError),
                                      (dict(scaling={"type": "yarn", "factor": 2.0}), ValueError), (dict(scaling={"type": "linear", "factor": 2.0, "original_length": 5}), ValueError),
                                      (dict(scaling={"type": "dynamic", "factor": 2.0, "original_length": 0}), ValueError),
                                      (dict(scaling={"type": "yarn", "factor": float("nan"), "original_length": 10}), ValueError)])
def test_positions_that_are_refused(kw, error):
    with pytest.raises(error):
        RotaryEmbedding(64, **kw)


def build(**kw):
    from easyllm_amd import runner
    cfg = dict(num_layers=1, hidden_size=64, num_attention_heads=1, intermediate_size=72, vocab_size=64, seq_length=16, bf16=True)
    cfg.update(kw)
    return runner.build_model({"type": "llama_custom", "kwargs": cfg})


def test_a_model_takes_the_options():
    model = build(position_embedding_kwargs={"rotary_dim": 32, "interleaved": True}, transformer_layer_params={"glu_activation": "relu", "glu_fusion": True})
    layer = model.get_submodule("3")
    assert layer.self_attn.rotary_emb.general and layer.mlp.fused_gate == "relu" and not model.get_submodule("1").positions_in_tables
    assert {"3.mlp.gate_proj.weight", "3.mlp.up_proj.weight", "3.mlp.down_proj.weight"} <= set(model.state_dict())
    plain = build()
    assert not plain.get_submodule("3").self_attn.rotary_emb.general and plain.get_submodule("1").positions_in_tables and plain.get_submodule("3").mlp.fused_gate is None


@pytest.mark.parametrize("layer", [dict(glu_activation="tanh", glu_fusion=True), dict(glu_activation=None, glu_fusion=True), dict(glu_activation="gelu")])
def test_gates_that_are_refused(layer):
    with pytest.raises(NotImplementedError):
        build(transformer_layer_params=layer)


def test_optimizer_state_by_group_and_size():
    def param(n):
        p = torch.nn.Parameter(torch.zeros(n, dtype=torch.bfloat16))
        p.main_grad = torch.zeros(n)
        return p
    a, b, c, d = param(5000), param(100), param(5000), param(300)
    opt = optimizer.FusedAdam([{"params": [a, b]}, {"params": [c, d], "state_bits": 32}], state_bits=8, min_8bit_size=200)
    assert opt.state[a]["exp_avg"].dtype is torch.uint8 and opt.state[a]["exp_avg_scale"].numel() == 20 and opt.state[a]["number"] == 0
    assert all(opt.state[p]["exp_avg"].dtype is torch.float32 and "number" not in opt.state[p] for p in (b, c, d))
    opt = optimizer.FusedAdam([a, b, c, d], state_bits=8, min_8bit_size=200)
    assert [opt.state[p].get("number") for p in (a, b, c, d)] == [0, None, 2, 3]
    assert optimizer.FusedAdam([a]).state[a]["exp_avg"].dtype is torch.float32
    with pytest.raises(ValueError, match="state_bits"):
        optimizer.FusedAdam([a], state_bits=16)
    model = build()
    for p in model.parameters():
        p.main_grad = torch.zeros(p.shape)
    opt = optimizer.build_optimizer({"type": "AdamW8bit", "kwargs": {"lr": 1e-3, "min_8bit_size": 0}}, model)
    assert all("number" in st for st in opt.state.values()) and len({st["number"] for st in opt.state.values()}) == len(opt.state)


def test_the_library_refuses_before_it_launches():
    lib = _lib.load()
    side = _lib.RotarySide(16, 16, 2, 128, 128, 64)

    def rotary(q=side, k=None, inv=16, s=4, b=1, d=64, turned=64, pos=None, interleaved=0):
        return lib.ezl_rotary(q, k, inv, 0, pos, 1, 1, s, b, d, turned, interleaved, 1.0, 0, None)
    for kw in (dict(q=None), dict(inv=None), dict(inv=18), dict(s=-1), dict(s=1 << 31), dict(d=60), dict(d=2056, turned=64), dict(turned=0), dict(turned=33), dict(turned=66), dict(pos=20),
               dict(q=_lib.RotarySide(None, 16, 2, 128, 128, 64)), dict(q=_lib.RotarySide(16, 24, 2, 128, 128, 64)), dict(q=_lib.RotarySide(16, 16, 2, 124, 128, 64)),
               dict(q=_lib.RotarySide(16, 16, -1, 128, 128, 64)), dict(q=_lib.RotarySide(16, 16, 2, 128, 128, -64)), dict(k=_lib.RotarySide(16, None, 2, 128, 128, 64))):
        assert rotary(**kw) in (-1, -2), kw
    for turned, interleaved in ((2, 0), (6, 0), (2, 1), (1026, 1)):  # (257 pieces of 8 elements, one more than a workgroup has threads)
        assert rotary(d=2048, turned=turned, interleaved=interleaved) == -2, (turned, interleaved)
    assert rotary(s=0) == 0 and rotary(q=_lib.RotarySide(None, None, 0, 0, 0, 0)) == 0

    def tensor(n=10, number=0, **kw):
        t = _lib.Adam8Tensor(16, 16, 16, 16, 16, 16, 16, n, number)
        for name, v in kw.items():
            setattr(t, name, v)
        return (_lib.Adam8Tensor * 1)(t)
    how = lambda **kw: _lib.Adam8(**dict(dict(lr=1e-3, beta1=0.9, beta2=0.99, eps=1e-8, weight_decay=0, step=1, seed=0, bias_correction=1), **kw))  # noqa: E731
    null = (ctypes.c_void_p * 1)(None)
    for kw in (dict(master=None), dict(exp_avg=None), dict(exp_avg_sq_scale=None), dict(grad=None), dict(n=-1), dict(n=1 << 35), dict(master=24), dict(exp_avg=24), dict(exp_avg_scale=20), dict(grad=8),
               dict(param_bf16=20)):
        assert lib.ezl_adamw8_list(1, tensor(**kw), how(), None, None) == -1, kw
    for step in (0, -1, 1 << 32):
        assert lib.ezl_adamw8_list(1, tensor(), how(step=step), None, None) == -1
    assert lib.ezl_adamw8_list(-1, tensor(), how(), None, None) == -1 and lib.ezl_adamw8_list(1, None, how(), None, None) == -1 and lib.ezl_adamw8_list(1, tensor(), None, None, None) == -1
    assert lib.ezl_adamw8_list(0, None, how(), None, None) == 0 and lib.ezl_adamw8_list(1, tensor(n=0), how(), None, None) == 0
    assert lib.ezl_moments8_list(1, tensor(), null, null, None) == -1 and lib.ezl_moments8_list(0, None, None, None, None) == 0

    def gated(act=0, x=16, wg=16, wu=16, out=16, kept=None, M=4, f=16, K=16, ldx=16, ldw=16, ws=None):
        return lib.ezl_gated_fwd(act, x, wg, wu, out, kept, M, f, K, ldx, ldw, ws, 0, None)
    for kw in (dict(act=-1), dict(act=4), dict(x=None), dict(wg=None), dict(wu=None), dict(out=None), dict(kept=24), dict(M=-1), dict(f=12), dict(K=0), dict(K=12, ldx=16), dict(ldx=8),
               dict(ldw=12), dict(x=24), dict(wu=24), dict(out=24), dict(f=1 << 21, ldw=16), dict(ws=24)):
        assert gated(**kw) in (-1, -2), kw
    assert gated(M=0) == 0 and gated(f=0) == 0

    def gated_bwd(act=0, dy=16, wd=16, kept=16, dg=16, du=16, mid=None, M=4, f=16, K=16, lddy=16, ldw=16):
        return lib.ezl_gated_bwd(act, dy, wd, kept, dg, du, mid, M, f, K, lddy, ldw, None, 0, None)
    for kw in (dict(act=9), dict(dy=None), dict(wd=None), dict(kept=None), dict(kept=24), dict(dg=None), dict(du=None), dict(mid=24), dict(M=-1), dict(f=12), dict(K=0), dict(lddy=8), dict(ldw=8)):
        assert gated_bwd(**kw) in (-1, -2), kw
    for kw in (dict(act=4), dict(f=12), dict(f=-8), dict(M=-1), dict(f=1 << 21), dict(d=None), dict(d=24), dict(kept=None), dict(kept=24), dict(dg=8), dict(du=None)):
        c = dict(dict(act=0, d=16, kept=16, dg=16, du=16, M=3, f=16), **kw)
        assert lib.ezl_gate_bwd(*c.values(), None) in (-1, -2), kw
    assert lib.ezl_gate_bwd(0, None, None, None, None, 0, 16, None) == 0 and lib.ezl_gate_bwd(0, None, None, None, None, 5, 0, None) == 0
    for M, f in ((1, 8), (16, 32), (17, 40), (100, 688), (0, 64), (1 << 20, 13696)):
        assert lib.ezl_gated_kept_bytes(M, f) == K._kept_bytes(M, f) >= 5 * M * f
    mlp = lambda **kw: _lib.GatedMLP(**dict(dict(M=4, h=16, f=16, n=16, gate=16, up=16, down=16, ldw=16, ldd=16, act=0), **kw))  # noqa: E731
    nbytes = lib.ezl_gated_mlp_bytes(mlp(), 0)
    assert nbytes > 0 and lib.ezl_gated_mlp_bytes(mlp(), 1) > nbytes and lib.ezl_gated_mlp_bytes(mlp(h=0), 0) == -1 and lib.ezl_gated_mlp_bytes(None, 0) == -1
    for m, kw in ((mlp(h=12), {}), (mlp(f=12), {}), (mlp(n=12), {}), (mlp(M=-1), {}), (mlp(gate=None), {}), (mlp(down=None), {}), (mlp(act=7), {}), (None, {}), (mlp(), dict(x=None)), (mlp(), dict(y=None)),
                  (mlp(), dict(temp=None)), (mlp(), dict(temp=24)), (mlp(), dict(nbytes=nbytes - 1)), (mlp(), dict(kept=24))):
        c = dict(dict(x=16, y=16, kept=None, temp=16, nbytes=1 << 40), **kw)
        assert lib.ezl_gated_mlp_fwd(m, c["x"], 16, c["y"], c["kept"], c["temp"], c["nbytes"], None) in (-1, -2), (m, kw)
    for kw in (dict(x=None), dict(dy=None), dict(kept=None), dict(kept=24), dict(temp=None), dict(nbytes=8), dict(dx=24)):
        c = dict(dict(x=16, dy=16, kept=16, dx=16, temp=16, nbytes=1 << 40), **kw)
        assert lib.ezl_gated_mlp_bwd(mlp(), c["x"], 16, c["dy"], c["kept"], c["dx"], None, None, None, c["temp"], c["nbytes"], None) in (-1, -2), kw


def test_yarn_leaves_fast_waves_and_divides_slow_ones():
    inv_freq = 10000.0 ** -(torch.arange(64, dtype=torch.float64) / 64)
    got, factor = scaled_frequencies(inv_freq, 10000.0, {"type": "yarn", "factor": 8.0, "original_length": 4096}, 0)
    turns = 4096 * inv_freq / (2 * math.pi)
    assert torch.equal(got[turns > 40], inv_freq[turns > 40]) and torch.allclose(got[turns < 0.8], inv_freq[turns < 0.8] / 8, rtol=1e-12)
    assert abs(factor - (0.1 * math.log(8) + 1)) < 1e-12 and scaled_frequencies(inv_freq, 10000.0, {"type": "yarn", "factor": 8.0, "original_length": 4096, "attention_factor": 1.0}, 0)[1] == 1.0
