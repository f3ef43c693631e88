"""The fused block's linears with their epilogues (K13) against the same block
composed of K3 GEMMs, residual copies and the SwiGLU kernel: bit for bit, since
both add the same products in the same order."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def mm(a, layer, out, prec, accumulate=False):
    from mround_b200 import kernels

    t, n, k = a[0].shape[0], layer.out_features, layer.in_features
    kernels.gemm(a[0], a[1] if prec >= 2 else None, layer.wq_hi, layer.wq_lo if prec == 3 else None,
                 out, m=t, n=n, k=k, a_kmajor=True, b_kmajor=True, lda=k, ldb=k, ldc=n,
                 precision=prec, accumulate=accumulate)
    return out


@pytest.mark.parametrize("arch,b,s", [("tiny-llama", 1, 8), ("tiny-qwen2", 2, 40),
                                      ("smollm2-135m", 2, 512), ("qwen2.5-0.5b", 1, 1000)])
@pytest.mark.parametrize("forward,tuned", [(3, True), (3, False), (2, False), (1, False)])
def test_block_equals_its_composition(arch, b, s, forward, tuned):
    from mround_b200 import kernels
    from mround_b200.pipeline.arch import get_arch
    from mround_b200.pipeline.block import TF32, DeviceBlock, Precision
    from mround_b200.pipeline.model import SyntheticModel

    ar = get_arch(arch)
    blk = DeviceBlock(ar, SyntheticModel(ar, seed=3).block(0), "cuda")
    if tuned:  # a weight that bf16 does not hold: two parts
        g = torch.Generator(device="cuda").manual_seed(1)
        for layer in blk.layers.values():
            w = layer.w.float() * (1 + 0.01 * torch.randn(layer.w.shape, device="cuda", generator=g))
            layer.wq_hi, layer.wq_lo = kernels.split_bf16(w)
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(b, s, ar.hidden, device="cuda", generator=g)
    prec = Precision(forward, TF32, TF32)
    out, saved = blk.forward_fused(x, prec, True)
    plain, none = blk.forward_fused(x, prec, False)
    assert none is None and torch.equal(out, plain)
    p = forward if tuned else min(forward, 2)
    t = b * s
    x2 = x.view(t, ar.hidden)
    hres = mm(saved["att"], blk.layers["o"], x2.clone(), p, accumulate=True)
    assert torch.equal(hres, saved["hres"])
    gu = mm(saved["h2"], blk.layers["gate_up"], torch.empty(t, 2 * ar.intermediate, device="cuda"), p)
    assert torch.equal(gu, saved["gu"])
    act = kernels.swiglu_split(gu, t, ar.intermediate, t32=True)
    assert all(torch.equal(e, f) for e, f in zip(act, saved["act"]))
    want = mm(act, blk.layers["down"], hres.clone(), p, accumulate=True)
    assert torch.equal(want.view_as(out), out)
    assert math.isfinite(out.abs().max().item())
