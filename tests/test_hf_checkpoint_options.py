"""Checkpoint names of stacks with layer norm, biases and a plain MLP: nothing is lost or written over on the way out and back (CPU)."""
import os

import pytest
import torch

from easyllm_amd import hf_checkpoint as H
from easyllm_amd import runner

LN = dict(layer_norm_params={"type": "mixed_fused_norm"})
PLAIN = dict(glu_activation=None, mlp_bias=True, attention_qkv_bias=True, attention_o_bias=True)
STACKS = {"layer norm, plain MLP, biases": dict(LN, transformer_layer_params=PLAIN), "layer norm, gated MLP": LN,
          "RMSNorm, plain MLP": dict(transformer_layer_params=dict(glu_activation=None)), "llama": {}}


def build(seed, **kw):
    kwargs = dict(num_layers=2, hidden_size=64, num_attention_heads=4, intermediate_size=96, vocab_size=128, seq_length=32, bf16=True, fp32_logits=False)
    kwargs.update(kw)
    kwargs = {k: dict(v) if isinstance(v, dict) else v for k, v in kwargs.items()}
    model = runner.build_model({"type": "llama_custom", "kwargs": kwargs})
    g = torch.Generator().manual_seed(seed)
    with torch.no_grad():
        for p in model.parameters():  # (no two tensors alike, a norm's weight and bias among them)
            p.copy_(torch.randn(p.shape, generator=g))
    return model


@pytest.mark.parametrize("name", STACKS)
def test_a_stack_comes_back_as_it_was(name, tmp_path):
    from safetensors.torch import save_file
    model, other = build(1, **STACKS[name]), build(2, **STACKS[name])
    out = H.megatron_to_hf_llama(model.state_dict(), 2)
    params = dict(model.named_parameters())
    assert len(out) == len(params) and len({t.data_ptr() for t in out.values()}) == len(params)
    assert out["model.norm.weight"].data_ptr() == params["6.weight"].data_ptr()
    assert ("model.norm.bias" in out) == ("layer norm" in name)
    save_file({k: v.contiguous() for k, v in out.items()}, os.path.join(tmp_path, "model.safetensors"))
    assert H.load_llama_from_hf_format(str(tmp_path), other) is True
    for n, p in other.named_parameters():
        assert torch.equal(p, params[n]), n


@pytest.mark.parametrize("saved,target,what", [("layer norm, gated MLP", "llama", "bias"), ("layer norm, plain MLP, biases", "RMSNorm, plain MLP", "bias"),
                                               ("llama", "RMSNorm, plain MLP", "gate_proj")])
def test_a_tensor_that_the_stack_has_no_place_for_is_refused(saved, target, what):
    """And by name, not by a shape that happens to differ: a norm's bias has the shape of its weight."""
    model = build(2, **STACKS[target])
    dt = H.hf_to_megatron_llama(H.megatron_to_hf_llama(build(1, **STACKS[saved]).state_dict(), 2), model)
    with pytest.raises(ValueError, match=what):
        H.copy_into_model(dt, model)


def test_tensors_of_layers_that_live_elsewhere_are_passed_by():
    """Layers of a deeper checkpoint, whose numbers may be those of the final norm and the head, and biases of the attention's projections."""
    model = build(1)
    dt = {"%d.%s" % (i, n): torch.zeros(64) for i in (5, 6, 7, 9) for n in ("mlp.up_proj.weight", "input_layernorm.weight", "input_layernorm.bias")}
    assert H.copy_into_model(dict(dt, **{"3.self_attn.q_proj.bias": torch.zeros(64)}), model) == set()
