"""Where a checkpoint's configuration may state its rotary settings: each is read
wherever it stands, and what the block would ignore, or what contradicts itself,
is refused."""

from __future__ import annotations

import pytest

from mround_b200.exceptions import ArchitectureError
from mround_b200.pipeline.arch import RopeScaling
from mround_b200.pipeline.loader import CheckpointModel
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
