"""The device block with scaled, interleaved and partial rotary embeddings:
forward against transformers' Llama layer, forward and gradients against the
block's autograd form (K3 linears, torch for the rest).

Bounds: the fused forward carries float32 through 2**-16 hi/lo products; a
block of a handful of such steps is held to 2e-5 of its largest output, as the
unscaled block is, and its gradients (bf16x3) to 1e-4 of the largest."""

from __future__ import annotations

import dataclasses

import pytest
import torch

from mround_b200.pipeline.arch import RopeScaling, get_arch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


LLAMA3 = RopeScaling("llama3", 8.0, 16, 1.0, 4.0)
YARN = RopeScaling("yarn", 4.0, 32)


def off(got, ref):
    return ((got.double().cpu() - ref.double().cpu()).abs().max() / ref.double().abs().max().cpu()).item()


@pytest.mark.parametrize("scaling", [LLAMA3, YARN, RopeScaling("linear", 3.0)])
def test_scaled_block_matches_transformers(scaling):
    from transformers.models.llama import modeling_llama as mod
    from transformers.models.llama.configuration_llama import LlamaConfig

    from mround_b200.pipeline.block import DeviceBlock, Precision
    from mround_b200.pipeline.model import SyntheticModel, rope_scaling_config

    arch = dataclasses.replace(get_arch("tiny-llama"), rope_scaling=scaling)
    params = SyntheticModel(arch, seed=5).block(0)
    cfg = LlamaConfig(
        hidden_size=arch.hidden, num_attention_heads=arch.heads, num_key_value_heads=arch.kv_heads,
        head_dim=arch.head_dim, intermediate_size=arch.intermediate, rms_norm_eps=arch.rms_eps,
        max_position_embeddings=256, attn_implementation="eager",
        rope_parameters={**rope_scaling_config(scaling), "rope_theta": arch.rope_theta})
    layer = mod.LlamaDecoderLayer(cfg, 0).float().eval()
    state = {f"{k}.weight": v.float() for k, v in params.linears.items()}
    state["input_layernorm.weight"] = params.input_norm.float()
    state["post_attention_layernorm.weight"] = params.post_norm.float()
    layer.load_state_dict(state)
    g = torch.Generator().manual_seed(1)
    x = torch.randn(2, 72, arch.hidden, generator=g)
    cos_sin = mod.LlamaRotaryEmbedding(cfg)(x, torch.arange(72)[None])
    mask = torch.full((72, 72), float("-inf")).triu(1)[None, None]
    with torch.no_grad():
        want = layer(x, attention_mask=mask, position_embeddings=cos_sin)
    want = want[0] if isinstance(want, tuple) else want
    got, _ = DeviceBlock(arch, params, "cuda").forward_fused(x.cuda(), Precision(), False)
    assert off(got, want) <= 2e-5


@pytest.mark.parametrize("scaling,interleaved,rotary_dim", [
    (None, True, None), (None, False, 16), (LLAMA3, True, 24), (YARN, False, 8)])
@pytest.mark.parametrize("s", [40, 128])
def test_layouts_match_the_autograd_form(scaling, interleaved, rotary_dim, s):
    from mround_b200.pipeline.block import DeviceBlock, Precision
    from mround_b200.pipeline.model import SyntheticModel

    arch = dataclasses.replace(get_arch("tiny-qwen2"), rope_scaling=scaling,
                               rope_interleaved=interleaved, rotary_dim=rotary_dim)
    blk = DeviceBlock(arch, SyntheticModel(arch, seed=6).block(0), "cuda")
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(2, s, arch.hidden, device="cuda", generator=g)
    dout = torch.randn(2, s, arch.hidden, device="cuda", generator=g)
    grads = {}
    for layer in blk.layers.values():
        layer.grad = torch.empty(layer.w.shape, dtype=torch.float32, device="cuda")
    leaf = x.clone().requires_grad_()
    want = blk.forward(leaf, Precision(), train=True)
    want.backward(dout)
    for name, layer in blk.layers.items():
        grads[name] = layer.grad.clone()
        layer.grad.fill_(float("nan"))
    got, saved = blk.forward_fused(x, Precision(), True)
    assert off(got, want.detach()) <= 2e-5
    dx = blk.backward_fused(saved, dout, Precision(), want_dx=True)
    assert off(dx, leaf.grad) <= 1e-4
    for name, layer in blk.layers.items():
        assert off(layer.grad, grads[name]) <= 1e-4, name
