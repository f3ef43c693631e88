"""Scoring by distillation, end to end: the teacher's top logits, the loss at
each width's anchors and every layer's score against a CPU float32 autograd
oracle, with a scaled, interleaved rotary embedding (rel 1e-3, as the
cross-entropy scores are held)."""

from __future__ import annotations

import dataclasses
import json

import numpy as np
import pytest
import torch

from mround_b200.pipeline.arch import RopeScaling, get_arch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


ARCH = dataclasses.replace(get_arch("tiny-qwen2"), rope_interleaved=True,
                           rope_scaling=RopeScaling("llama3", 8.0, 16, 1.0, 4.0))


def oracle(model, batches, widths, group, targets, temperature, monkeypatch):
    from mround_b200.pipeline.block import apply_rope, rope_tables
    from oracle import block_tuner
    from oracle.deltaloss import delta_loss, rtn

    arch = model.arch

    def rope(x, theta):
        cos, sin = rope_tables(x.shape[-2], arch.head_dim, theta, "cpu", arch.rope_scaling)
        return apply_rope(x, cos, sin, arch.rope_layout)

    monkeypatch.setattr(block_tuner, "rope", rope)
    linears = block_tuner.LINEARS
    blocks = [block_tuner.OracleBlock(arch, model.block(i), {p: 2 for p in linears}, group)
              for i in range(arch.layers)]
    embed = model.embed_tokens().float()

    def logits_of(batch):
        x = embed[torch.as_tensor(batch, dtype=torch.long)[:, :-1]]
        for blk in blocks:
            x = blk.forward(x)
        h = block_tuner.rms_norm(x, model.final_norm().float(), arch.rms_eps)
        return (h @ embed.t()).flatten(0, 1)

    dense, scores, losses = [], {}, {}
    for blk in blocks:
        blk.committed = {p: blk.w[p] for p in linears}
    with torch.no_grad():
        dense = [logits_of(b) for b in batches]
    for bits in widths:
        for blk in blocks:
            blk.committed = {p: torch.from_numpy(rtn(blk.w[p].numpy(), bits, group))
                             .requires_grad_(True) for p in linears}
        total = 0.0
        for batch, (v, i) in zip(batches, targets):
            for blk in blocks:
                for t in blk.committed.values():
                    t.grad = None
            log_q = torch.log_softmax(logits_of(batch).double() / temperature, 1).gather(1, i.cpu())
            log_p = torch.log_softmax(v.cpu().double() / temperature, 1)
            loss = temperature ** 2 * (log_p.exp() * (log_p - log_q)).sum(1).mean()
            loss.backward()
            total += loss.item()
            for n, blk in enumerate(blocks):
                for p in linears:
                    at = scores.setdefault(f"model.layers.{n}.{p}", {})
                    at[bits] = at.get(bits, 0.0) + delta_loss(
                        blk.w[p].numpy(), blk.committed[p].grad.numpy(), bits, group)
        losses[bits] = total / len(batches)
    return dense, scores, losses


@pytest.mark.parametrize("seq,temperature", [(33, 1.0), (30, 2.0)])
def test_distillation_scores_match_oracle(seq, temperature, monkeypatch):
    from mround_b200.pipeline.model import SyntheticModel, zipf_tokens
    from mround_b200.pipeline.scoring import capture_top_logits, score_widths
    from mround_b200.schemes import QuantScheme

    model = SyntheticModel(ARCH, seed=4)
    tokens = zipf_tokens(ARCH.vocab, 3, seq, seed=1)
    batches = [tokens[0:1], tokens[1:3]]
    widths = (2, 3, 4)
    targets = capture_top_logits(model, batches, 40)
    scheme = QuantScheme(bits=4, group_size=32, symmetry="asym")
    got = score_widths(model, batches, widths, scheme, objective="teacher", top_logits=40,
                       temperature=temperature)
    dense, want, losses = oracle(model, batches, widths, 32, targets, temperature, monkeypatch)
    for (v, i), full in zip(targets, dense):
        scale = full.abs().max()
        assert (v.cpu() - full.gather(1, i.cpu())).abs().max() <= 2e-5 * scale
        # nothing left out is above what was kept, by more than both are off
        rest = full.scatter(1, i.cpu(), float("-inf")).amax(1)
        assert (rest <= v[:, -1].cpu() + 4e-5 * scale).all()
    assert set(got.scores) == set(want)
    for bits in widths:
        assert got.losses[bits] == pytest.approx(losses[bits], rel=1e-3)
        for key in want:
            assert got.scores[key][bits] == pytest.approx(want[key][bits], rel=1e-3), (key, bits)
    assert got.losses[2] > got.losses[3] > got.losses[4] > 0
    widest = score_widths(model, batches, widths, scheme, objective="teacher", top_logits=40,
                          temperature=temperature, gradient_source="widest", teacher=model)
    for key in want:
        assert widest.scores[key][4] == pytest.approx(got.scores[key][4], rel=1e-6)
    assert set(widest.losses) == {4}


def test_label_scores_do_not_carry_losses():
    from mround_b200.pipeline.model import SyntheticModel, zipf_tokens
    from mround_b200.pipeline.scoring import score_widths
    from mround_b200.schemes import QuantScheme

    model = SyntheticModel(get_arch("tiny-llama"), seed=2)
    got = score_widths(model, [zipf_tokens(model.arch.vocab, 1, 17, seed=1)], (2, 4),
                       QuantScheme(bits=4, group_size=32, symmetry="asym"))
    assert got.losses is None


def test_mixed_run_planned_by_distillation(tmp_path):
    from mround_b200.api import quantize
    from mround_b200.pipeline.model import SyntheticModel
    from mround_b200.schemes import TuningConfig

    result = quantize(SyntheticModel(ARCH, seed=1), output_dir=tmp_path, group_size=32,
                      symmetry="asym", average_bits=3.0, candidate_bits=(2, 3, 4),
                      scoring_samples=2, scoring_seq_len=32, progress=None,
                      tuning=TuningConfig(iters=2, n_samples=2, seq_len=32, batch_size=2),
                      sensitivity_objective="teacher", sensitivity_top_logits=16,
                      sensitivity_temperature=1.5)
    record = json.loads((tmp_path / "mround_run.json").read_text())["mixed"]
    assert record["objective"]["name"] == "teacher" and record["objective"]["top_logits"] == 16
    assert record["assignments"] and np.isfinite(result.mixed["predicted_loss"])
    config = json.loads((tmp_path / "config.json").read_text())
    assert config["rope_scaling"]["rope_type"] == "llama3" and config["rope_traditional"] is True
