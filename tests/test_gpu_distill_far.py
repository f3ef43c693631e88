"""K12 on rows whose logits are large beside the temperature, against float64.

Whatever the size of a row, q depends on differences alone.  A term's exponent
(x - max) c takes at most three roundings of 2**-24 of itself (the difference, c
and the product, or c and one fused step); terms with (max - x) / T above 128
are below 2**-126 and count as nothing.  Sums are float32 within a thread, of
which a row of up to 16 KB has 96 and any other at least 224, and 2**-22 per
exponential.  So q is within
    e = (n / 96 + 16) * 2**-24 + 2**-21 + 3 * 128 * 2**-24
of its value, and log q within e + 2**-23 (max - x) / T.  The teacher's logits
stay within 16 T of one another: p is within 3 * 24 * 2**-24 + 2**-22 < 2**-17
of its value, which moves the loss by that part of sum p |log p - log q|.
"""

from __future__ import annotations

import pytest
import torch


@pytest.fixture(scope="module")
def K():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from mround_b200 import kernels

    return kernels


def rows_of(n, v, temperature, dtype):
    """Uniform rows at v and -v, rows of two neighbouring values there, and rows
    of ordinary logits that are masked with -v for the most part."""
    g = torch.Generator(device="cuda").manual_seed(n)
    x = torch.empty(8, n, device="cuda", dtype=dtype)
    x[0], x[1] = v, -v
    for r, at in ((2, v), (3, -v)):
        x[r] = at
        bits = x[r].view(torch.int32 if dtype == torch.float32 else torch.int16)
        bits[::3] -= 1
    for r in (4, 5, 6, 7):
        x[r] = torch.randn(n, device="cuda", generator=g) * 3 * temperature
    x[4, 40:] = -v
    x[5, :-40] = -v
    x[6, n // 2:] = -v
    x[7, 40:] = -v
    x[7, 50:60] = v
    return x


def reference(x, t, i, temperature):
    d = x.double() - x.double().max(1, keepdim=True).values
    log_q = torch.log_softmax(d / temperature, 1)
    log_p = torch.log_softmax(t.double() / temperature, 1)
    p = log_p.exp()
    each = log_p - log_q.gather(1, i)
    mass = torch.zeros_like(log_q).scatter_add_(1, i, p)
    size = (p * each.abs()).sum(1)
    far = (p * d.gather(1, i).abs() / temperature).sum(1)
    return temperature ** 2 * (p * each).sum(1), size, far, log_q.exp(), mass


@pytest.mark.gpu
@pytest.mark.parametrize("temperature", [1e-3, 0.1, 1.0, 4.0])
@pytest.mark.parametrize("v,dtype", [
    (v, torch.float32) for v in (3e4, 1e7, 1.162e7, 1e8, 1e9, 1e10, 1e12, 1e20, 3e37)] + [
    (1e9, torch.bfloat16), (1e10, torch.bfloat16), (1e20, torch.bfloat16), (6e4, torch.float16)])
def test_rows_far_from_zero(K, v, dtype, temperature):
    """The loss, the gradient, in place and as a pair; whole rows (many) and rows
    divided among CTAs (8 of 40000 columns)."""
    for n, copies in ((1000, 1), (1000, 25), (40000, 1)):
        x = rows_of(n, v, temperature, dtype).repeat(copies, 1)
        rows = x.shape[0]
        g = torch.Generator(device="cuda").manual_seed(1)
        i = torch.randint(0, n, (rows, 5), device="cuda", generator=g)
        i[:, 0], i[:, 1] = 7, n - 7
        t = torch.randn(rows, 5, device="cuda", generator=g).clamp(-4, 4) * (2 * temperature)
        loss, size, far, q, mass = reference(x, t, i, temperature)
        grad = temperature * (q - mass)
        e = (n / 96 + 16) * 2.0 ** -24 + 2.0 ** -21 + 3 * 128 * 2.0 ** -24
        off = temperature ** 2 * (e + 2.0 ** -23 * far + 2.0 ** -17 * size) + 2.0 ** -24 * loss.abs()
        goff = temperature * (q * e + mass * 2.0 ** -17)
        step = torch.finfo(dtype).eps / 2
        tiny = torch.finfo(dtype).smallest_normal * step
        only = K.distill_topk(x, t, i, temperature=temperature)
        both, got = K.distill_topk_grad(x, t, i, temperature=temperature)
        pair_loss, (hi, lo) = K.distill_topk_grad(x, t, i, temperature=temperature, split=True)
        y = x.clone()
        in_loss, same = K.distill_topk_grad(y, t, i, temperature=temperature, out=y)
        for value in (only, both):
            assert ((value.double() - loss).abs() <= off).all()
        assert torch.equal(pair_loss, both) and torch.equal(in_loss, both)
        assert ((got.double() - grad).abs() <= goff + step * (grad.abs() + goff) + tiny).all()
        assert torch.equal(same, got)
        pair = hi.double() + lo.double()
        assert ((pair - grad).abs() <= goff + 2.0 ** -16 * (grad.abs() + goff) + 2.0 ** -126).all()
