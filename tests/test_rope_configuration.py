"""Where a checkpoint's configuration may state its rotary settings: each is read
wherever it stands, and what the block would ignore, or what contradicts itself,
is refused."""

from __future__ import annotations

import dataclasses

import pytest

from mround_b200.exceptions import ArchitectureError
from mround_b200.pipeline.arch import RopeScaling, get_arch
from mround_b200.pipeline.loader import CheckpointModel
from mround_b200.pipeline.model import SyntheticModel
from test_loader import write_checkpoint

LINEAR = {"rope_type": "linear", "factor": 2.0}


def read(tmp_path, name="tiny-qwen2", top_theta=None, **keys):
    def edit(c):
        c.pop("rope_theta", None)
        if top_theta is not None:
            c["rope_theta"] = top_theta
        c.update(keys)

    write_checkpoint(tmp_path, name, edit_config=edit)
    return CheckpointModel(tmp_path).arch


@pytest.mark.parametrize("keys", [
    dict(rope_scaling={**LINEAR, "rope_theta": 5e5}),
    dict(rope_parameters={**LINEAR, "rope_theta": 5e5}),
    dict(top_theta=5e5, rope_scaling={**LINEAR, "rope_theta": 5e5}),
    dict(rope_scaling=LINEAR, rope_parameters={"rope_theta": 5e5}),
    dict(rope_scaling={**LINEAR, "rope_theta": 5e5}, rope_parameters={**LINEAR, "rope_theta": 5e5}),
])
def test_theta_wherever_it_stands(tmp_path, keys):
    arch = read(tmp_path, **keys)
    assert arch.rope_theta == 5e5 and arch.rope_scaling == RopeScaling("linear", 2.0)


def test_theta_by_default(tmp_path):
    assert read(tmp_path, rope_scaling=LINEAR).rope_theta == 10000.0


@pytest.mark.parametrize("keys", [
    dict(top_theta=1e4, rope_scaling={**LINEAR, "rope_theta": 5e5}),
    dict(top_theta=1e4, rope_parameters={"rope_type": "default", "rope_theta": 5e5}),
    dict(rope_scaling={**LINEAR, "rope_theta": 1e4}, rope_parameters={"rope_theta": 5e5}),
    dict(rope_scaling=LINEAR, rope_parameters={"rope_type": "default"}),
    dict(rope_scaling=LINEAR, rope_parameters={"rope_type": "linear", "factor": 4.0}),
])
def test_contradictions_are_refused(tmp_path, keys):
    with pytest.raises(ArchitectureError, match="differently"):
        read(tmp_path, **keys)


@pytest.mark.parametrize("entry", ["linear", [2.0], 4])
def test_entries_of_another_form_are_refused(tmp_path, entry):
    with pytest.raises(ArchitectureError, match="rope_scaling"):
        read(tmp_path, rope_scaling=entry)


@pytest.mark.parametrize("keys", [
    dict(partial_rotary_factor=0.5),
    dict(rope_parameters={"rope_type": "default", "partial_rotary_factor": 0.5}),
    dict(rope_parameters={"partial_rotary_factor": 0.5}),
    dict(rope_scaling={**LINEAR, "partial_rotary_factor": 0.5}),
    dict(partial_rotary_factor=0.5, rope_scaling={**LINEAR, "partial_rotary_factor": 0.5}),
])
def test_part_of_a_head_wherever_it_is_stated(tmp_path, keys):
    arch = read(tmp_path, **keys)
    assert arch.rotary_dim == arch.head_dim // 2
    assert (arch.rope_scaling is None) == ("rope_scaling" not in keys)


@pytest.mark.parametrize("keys", [
    dict(), dict(partial_rotary_factor=1.0), dict(partial_rotary_factor=None),
    dict(rope_parameters={"rope_type": "default", "rope_theta": 1e4, "factor": 1.0}),
    dict(rope_scaling={**LINEAR, "partial_rotary_factor": 1.0}),
])
def test_the_whole_head_by_default(tmp_path, keys):
    assert read(tmp_path, **keys).rotary_dim is None


@pytest.mark.parametrize("keys", [
    dict(partial_rotary_factor=0.0), dict(partial_rotary_factor=1.5),
    dict(partial_rotary_factor=-0.5), dict(partial_rotary_factor=0.02),
    dict(partial_rotary_factor=0.5, rope_parameters={"partial_rotary_factor": 0.25}),
    dict(rope_parameters={"rope_type": "default", "mrope_section": [2, 3, 3]}),
    dict(rope_scaling={"rope_type": "default", "factor": 4.0}),
    dict(rope_scaling={"type": "default", "mscale": 0.7}),
    dict(rope_scaling={"factor": 4.0}), dict(rope_parameters={"rope_theta": 1e4, "factor": 2.0}),
])
def test_what_the_block_would_ignore_is_refused(tmp_path, keys):
    with pytest.raises(ArchitectureError):
        read(tmp_path, **keys)


@pytest.mark.parametrize("fields", [
    dict(rotary_dim=4), dict(rotary_dim=6, rope_interleaved=True),
    dict(rotary_dim=8, rope_scaling=RopeScaling("linear", 4.0), rope_theta=5e5),
    dict(rope_scaling=RopeScaling("yarn", 4.0, 512, attention_factor=1.25)), dict(),
])
def test_written_configuration_reads_back_whole(tmp_path, fields):
    """All of the rotary fields, through the configuration that the model writes."""
    arch = dataclasses.replace(get_arch("tiny-llama"), **fields)
    config = SyntheticModel(arch).config()
    write_checkpoint(tmp_path, "tiny-llama", edit_config=lambda c: (c.clear(), c.update(config)))
    got = CheckpointModel(tmp_path).arch
    assert dataclasses.replace(got, name=arch.name) == arch


def test_every_rotated_part_survives_its_factor():
    """rotary_dim / head_dim, written as a float, gives back rotary_dim."""
    from mround_b200.pipeline.loader import _rotary_dim

    for head_dim in range(4, 513, 2):
        for columns in range(2, head_dim, 2):
            assert _rotary_dim({"partial_rotary_factor": columns / head_dim}, {}, head_dim) == columns
