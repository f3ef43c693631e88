"""A bounded wait of a matrix product that gave up is reported by the device's
status word alone; what keeps the products' results reads it and stops.  The
failure is made on the host: the status call is replaced."""

from __future__ import annotations

import contextlib
import types

import pytest
import torch

from mround_b200 import kernels
from mround_b200._native import lib
from mround_b200.exceptions import DeviceError
from mround_b200.pipeline.arch import get_arch
from mround_b200.pipeline.model import SyntheticModel, zipf_tokens
from mround_b200.pipeline.runner import QuantizationRunner
from mround_b200.schemes import QuantScheme, TuningConfig


class Status:
    """The library, but for the status word: 0 until the given read, then -5."""

    def __init__(self, at: int = 0) -> None:
        self.at, self.reads, self.resets = at, 0, []

    def __getattr__(self, name):
        return getattr(lib(), name)

    def mr_gemm_status(self, reset):
        self.reads += 1
        self.resets.append(reset)
        return -5 if self.reads > self.at else 0


@pytest.fixture
def failing(monkeypatch):
    def install(at=0):
        status = Status(at)
        monkeypatch.setattr(kernels, "lib", lambda: status)
        return status

    return install


@pytest.fixture
def no_device(monkeypatch):
    monkeypatch.setattr(torch.cuda, "device", lambda device: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "synchronize", lambda device=None: None)


def test_a_report_is_raised_and_cleared(failing, no_device):
    status = failing(at=1)
    kernels.check_products()
    with pytest.raises(DeviceError, match="gave up"):
        kernels.check_products("cuda:0")
    assert status.resets == [1, 1]


@pytest.mark.parametrize("fails", [False, True])
def test_a_block_is_checked_before_it_is_handed_on(failing, no_device, monkeypatch, fails):
    status = failing(at=0 if fails else 9)
    closed = []
    tuner = types.SimpleNamespace(tunables=[types.SimpleNamespace(members=[])], skipped=[],
                                  search=lambda inputs: 0.0, commit=lambda keep: {"mlp": "layer"},
                                  close=lambda: closed.append(1))
    runner = QuantizationRunner.__new__(QuantizationRunner)
    runner.device, runner.keep_codes = "cuda:0", False
    runner.tuning = types.SimpleNamespace(iters=1)
    monkeypatch.setattr(runner, "tuner_for", lambda *a: tuner)
    monkeypatch.setattr(runner, "_tune", lambda *a: dict(initial=1.0, final=0.5, reverted=False,
                                                         gap=None, step_seconds=0.0))
    meter = types.SimpleNamespace(stage=lambda name: contextlib.nullcontext(), peak=0, stages={})
    block = types.SimpleNamespace(index=0)
    if fails:
        with pytest.raises(DeviceError):
            runner.quantize_block(block, "b", [], [], meter=meter)
    else:
        assert runner.quantize_block(block, "b", [], [], meter=meter)[1] == {"b.mlp": "layer"}
    assert status.reads == 1 and closed == [1]


@pytest.mark.gpu
def test_runs_stop_at_a_report(failing, tmp_path):
    """Capturing, scoring, tuning (which records no block) and the whole call."""
    from mround_b200.api import quantize
    from mround_b200.pipeline.scoring import capture_top_logits, score_widths

    model = SyntheticModel(get_arch("tiny-llama"), seed=1)
    batches = [zipf_tokens(model.arch.vocab, 2, 16, seed=3)]
    scheme = QuantScheme(4, 32)
    tuning = TuningConfig(iters=1, n_samples=2, seq_len=16, batch_size=2)
    failing()
    with pytest.raises(DeviceError):
        capture_top_logits(model, batches, 8)
    for objective in ("labels", "teacher"):
        failing(at=int(objective == "teacher"))  # not the capture's own check
        with pytest.raises(DeviceError):
            score_widths(model, batches, [4], scheme, objective=objective, top_logits=8)
    failing()
    with pytest.raises(DeviceError):
        QuantizationRunner(scheme, tuning, device="cuda").run(model, batches)
    failing(at=1)  # the first block is recorded, the second is not
    store = tmp_path / "resume"
    with pytest.raises(DeviceError):
        quantize(model, output_dir=tmp_path / "out", bits=4, group_size=32, tuning=tuning,
                 resume_dir=store)
    assert not (tmp_path / "out" / "config.json").exists()
    assert [f.name for f in sorted(store.glob("block_*"))] == ["block_0000.pt"]
