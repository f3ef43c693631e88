"""Scaled, interleaved and partial rotary embeddings on the host: the tables
against transformers' rotary modules, the loader's reading of configurations,
and the fields that carry them."""

from __future__ import annotations

import dataclasses

import pytest
import torch

from mround_b200.exceptions import ArchitectureError, CalibrationError
from mround_b200.pipeline.arch import RopeScaling, get_arch
from mround_b200.pipeline.block import apply_rope, rope_tables
from mround_b200.pipeline.loader import CheckpointModel
from mround_b200.pipeline.model import SyntheticModel
from mround_b200.pipeline.resume import run_fingerprint
from mround_b200.schemes import QuantScheme, TuningConfig
from tests.test_loader import write_checkpoint

LLAMA3 = RopeScaling("llama3", 8.0, 256, low_freq_factor=1.0, high_freq_factor=4.0)
YARN = RopeScaling("yarn", 4.0, 512)
SCALINGS = [RopeScaling("linear", 4.0), LLAMA3, RopeScaling("llama3", 32.0, 128, 1.5, 3.0), YARN,
            RopeScaling("yarn", 16.0, 64, beta_fast=8.0, beta_slow=2.0, attention_factor=1.25)]


def settings(s: RopeScaling, theta: float) -> dict:
    from mround_b200.pipeline.model import rope_scaling_config

    return {**rope_scaling_config(s), "rope_theta": theta}


@pytest.mark.parametrize("scaling", SCALINGS)
@pytest.mark.parametrize("head_dim,theta", [(32, 1e4), (64, 5e5), (128, 1e6)])
def test_tables_match_transformers(scaling, head_dim, theta):
    """transformers computes frequencies and angles in float32: an angle p f is
    off by a few 2**-24 of itself (three roundings of f, one of the product),
    and so are cosine and sine, times the attention factor."""
    from transformers.models.llama import modeling_llama as mod
    from transformers.models.llama.configuration_llama import LlamaConfig

    original = scaling.original_max_position or 1024
    cfg = LlamaConfig(hidden_size=4 * head_dim, num_attention_heads=4, head_dim=head_dim,
                      max_position_embeddings=int(original * scaling.factor),
                      rope_parameters=settings(scaling, theta))
    positions = torch.arange(700)[None]
    cos, sin = mod.LlamaRotaryEmbedding(cfg)(torch.zeros(1, 700, 4), positions)
    got = rope_tables(700, head_dim, theta, "cpu", scaling)
    half = head_dim // 2
    for mine, theirs in zip(got, (cos[0, :, :half], sin[0, :, :half])):
        bound = 2.0 * (16 * 2.0 ** -24 * 700 + 2.0 ** -22)
        assert (mine - theirs).abs().max() <= bound


def test_unscaled_tables_are_as_before():
    inv = 1e4 ** (-torch.arange(0, 16, dtype=torch.float64) * 2.0 / 32)
    ang = torch.arange(50, dtype=torch.float64)[:, None] * inv[None, :]
    cos, sin = rope_tables(50, 32, 1e4, "cpu")
    assert torch.equal(cos, torch.cos(ang).float()) and torch.equal(sin, torch.sin(ang).float())


def test_layouts_are_permutations_of_each_other():
    """Interleaved columns (2j, 2j + 1) turned are half columns (j, j + r/2)
    turned, in the other order; the rest of the head is untouched."""
    x = torch.randn(2, 3, 9, 20)
    cos, sin = rope_tables(9, 12, 1e4, "cpu")
    order = torch.cat((torch.arange(0, 12, 2), torch.arange(1, 12, 2), torch.arange(12, 20)))
    half = apply_rope(x[..., order], cos, sin)
    assert torch.equal(apply_rope(x, cos, sin, "interleaved")[..., order], half)
    assert torch.equal(half[..., 12:], x[..., 12:])


@pytest.mark.parametrize("scaling", [LLAMA3, YARN, RopeScaling("linear", 2.0)])
@pytest.mark.parametrize("new_style", [False, True])
def test_loader_reads_scalings(tmp_path, scaling, new_style):
    def edit(c):
        entry = settings(scaling, 12345.0)
        if new_style:
            c.pop("rope_theta", None)
            c["rope_parameters"] = entry
        else:
            c["rope_theta"] = entry.pop("rope_theta")
            c["rope_scaling"] = entry

    write_checkpoint(tmp_path, edit_config=edit)
    arch = CheckpointModel(tmp_path).arch
    assert arch.rope_scaling == scaling and arch.rope_theta == 12345.0
    assert not arch.rope_interleaved and arch.rotary_dim is None


def test_loader_reads_the_interleaved_layout(tmp_path):
    write_checkpoint(tmp_path, edit_config=lambda c: c.update(rope_traditional=True))
    assert CheckpointModel(tmp_path).arch.rope_layout == "interleaved"


@pytest.mark.parametrize("entry", [
    {"rope_type": "dynamic", "factor": 2.0},
    {"rope_type": "longrope", "factor": 2.0},
    {"rope_type": "linear"},
    {"rope_type": "linear", "factor": 0.5},
    {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 512, "mscale": 0.7},
    {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 512,
     "truncate": False},
    {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 4.0, "high_freq_factor": 1.0,
     "original_max_position_embeddings": 512},
])
def test_loader_refuses(tmp_path, entry):
    write_checkpoint(tmp_path, edit_config=lambda c: c.update(rope_scaling=entry))
    with pytest.raises(ArchitectureError):
        CheckpointModel(tmp_path)


def test_refusals_of_the_fields():
    for kw in (dict(kind="ntk", factor=2.0), dict(kind="linear", factor=0.0),
               dict(kind="yarn", factor=2.0), dict(kind="llama3", factor=2.0),
               dict(kind="yarn", factor=2.0, original_max_position=64, beta_fast=1.0)):
        with pytest.raises(ArchitectureError):
            RopeScaling(**kw)
    arch = get_arch("tiny-llama")
    for r in (0, 3, arch.head_dim + 2):
        with pytest.raises(ArchitectureError):
            dataclasses.replace(arch, rotary_dim=r)


def test_written_configuration_reads_back(tmp_path):
    arch = dataclasses.replace(get_arch("tiny-llama"), rope_scaling=YARN, rope_interleaved=True)
    config = SyntheticModel(arch).config()
    assert config["rope_traditional"] is True
    write_checkpoint(tmp_path, "tiny-llama", edit_config=lambda c: c.update(
        {k: config[k] for k in ("rope_scaling", "rope_traditional")}))
    read = CheckpointModel(tmp_path).arch
    assert read.rope_scaling == YARN and read.rope_interleaved
    assert "rope_scaling" not in SyntheticModel(get_arch("tiny-llama")).config()


def test_fingerprint_of_an_unscaled_run_is_unchanged():
    """A resume directory written before the rotary fields existed stays valid;
    a scaled run has a fingerprint of its own."""
    def of(arch):
        return run_fingerprint(model="m", arch=arch, scheme=QuantScheme(bits=4),
                               tuning=TuningConfig(), scheme_by_layer=None, batches=[[1, 2]],
                               world=1)["arch"]

    arch = get_arch("tiny-llama")
    assert set(of(arch)) == {"name", "family", "hidden", "layers", "heads", "kv_heads", "head_dim",
                             "intermediate", "vocab", "rms_eps", "rope_theta", "qkv_bias", "tied"}
    assert of(dataclasses.replace(arch, rope_scaling=LLAMA3))["rope_scaling"]["factor"] == 8.0


@pytest.mark.parametrize("kw", [
    dict(sensitivity_objective="kl", average_bits=3.0),
    dict(sensitivity_objective="teacher"),
    dict(sensitivity_objective="teacher", average_bits=3.0, sensitivity_top_logits=0),
    dict(sensitivity_objective="teacher", average_bits=3.0, sensitivity_top_logits=257),
    dict(sensitivity_objective="teacher", average_bits=3.0, sensitivity_temperature=0.0),
])
def test_objective_refusals(tmp_path, kw):
    from mround_b200.api import quantize

    with pytest.raises(CalibrationError, match="sensitivity"):
        quantize("synthetic:tiny-llama", output_dir=tmp_path, **kw)


def test_scoring_refusals():
    from mround_b200.pipeline.scoring import score_widths

    model = SyntheticModel(get_arch("tiny-llama"))
    other = SyntheticModel(dataclasses.replace(get_arch("tiny-llama"), vocab=256))
    scheme = QuantScheme(bits=4, group_size=32)
    for kw in (dict(objective="kl"), dict(teacher=model), dict(objective="teacher", teacher=other),
               dict(objective="teacher", top_logits=0), dict(objective="teacher", top_logits=257)):
        with pytest.raises(ValueError):
            score_widths(model, [], (2, 4), scheme, **kw)
