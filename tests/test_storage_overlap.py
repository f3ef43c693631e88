"""Outputs that share storage with what a call reads, or with one another, are
refused; columns of one buffer beside each other are not.  The rule itself on the
CPU, against the sets of elements; the calls on the device."""

from __future__ import annotations

import random

import pytest
import torch

from mround_b200.exceptions import SchemeError


def shares(a, b):
    from mround_b200.kernels import _check_apart

    try:
        _check_apart("a", a, "b", b)
    except SchemeError:
        return True
    return False


def test_neighbours_in_one_buffer():
    a = torch.zeros(8, 64)
    rows = torch.zeros(2, 5, 48)  # [q | k | v] of two sequences
    q, k = rows[..., :24].view(2, 5, 4, 6), rows[..., 24:36].view(2, 5, 2, 6)
    for x, y in ((a[:, :32], a[:, 32:]), (a[:4], a[4:]), (a[::2], a[1::2]), (q, k),
                 (a[:, ::2], a[:, 1::2]), (a[:0], a), (q[:1], k[1:])):
        assert not shares(x, y) and not shares(y, x)
    for x, y in ((a, a), (a[:, :33], a[:, 32:]), (a[:5], a[4:]), (a[::2], a[2::2]),
                 (a[:4, :8], a.view(-1)[:32].view(4, 8)), (q, rows[..., 18:30].view(2, 5, 2, 6)),
                 (a[3], a[:, 5]), (a, a.view(torch.bfloat16)[2:3, :4])):
        assert shares(x, y) and shares(y, x)


def test_no_shared_element_is_missed():
    """Random views of one buffer: a common element is always found, and a view's
    rows beside another's, of one stride, are never taken for one."""
    rng = random.Random(0)
    met = 0
    for _ in range(4000):
        base, index = torch.zeros(400, dtype=rng.choice([torch.float32, torch.bfloat16])), torch.arange(400)
        views, sets = [], []
        for _ in range(2):
            shape = [rng.randint(1, 4) for _ in range(rng.randint(1, 3))]
            stride = [rng.choice([0, 1, 2, 3, 4, 8, 12, 16, 24, 30]) for _ in shape]
            at = rng.randint(0, 100)
            views.append(torch.as_strided(base, shape, stride, at))
            sets.append(set(torch.as_strided(index, shape, stride, at).flatten().tolist()))
        if sets[0] & sets[1]:
            met += 1
            assert shares(*views)
    assert met > 300
    for _ in range(500):
        pitch = rng.randint(8, 40)
        a0, b0 = rng.randint(0, pitch - 1), rng.randint(0, pitch - 1)
        wa, wb = rng.randint(1, pitch - a0), rng.randint(1, pitch - b0)
        base = torch.zeros(9, pitch)
        a, b = base[rng.randint(0, 3):, a0:a0 + wa], base[rng.randint(0, 3):, b0:b0 + wb]
        assert shares(a, b) == (a0 < b0 + wb and b0 < a0 + wa)


@pytest.fixture(scope="module")
def K():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from mround_b200 import kernels

    return kernels


@pytest.mark.gpu
def test_linear_refuses_shared_outputs(K):
    z = lambda *s, **k: torch.zeros(*s, device="cuda", **k)  # noqa: E731
    bf = dict(dtype=torch.bfloat16)
    x, w = (z(32, 64, **bf), z(32, 64, **bf)), (z(64, 64, **bf), z(64, 64, **bf))
    buf, wide = z(32, 256), z(64, 64)
    for bad in (dict(out=x[0]), dict(out=x[1]), dict(out=w[0][:32]), dict(out=w[1][8:40]),
                dict(out=buf[:, :64], pre=buf[:, 32:96]), dict(out=buf[:, :64], pre=buf[:, :64]),
                dict(out=buf[:, :64], t32=buf[:, 8:72]), dict(out=buf[:, 64:128],
                                                               t32=buf[:, 128:192],
                                                               pre=buf[:, 160:224]),
                dict(out=wide[:32], residual=wide[16:48]), dict(pre=wide[:32], residual=wide[:32]),
                dict(t32=wide[:32], residual=wide[8:40]), dict(out=wide[:32], bias=wide[3]),
                dict(pre=wide[:32], bias=wide[31])):
        with pytest.raises(SchemeError, match="storage"):
            K.linear(x, w, **bad)
    # what may be shared, and neighbours
    r = torch.randn(32, 64, device="cuda")
    want = K.linear(x, w, residual=r)
    buf[:, 64:128] = r
    assert torch.equal(K.linear(x, w, residual=buf[:, 64:128], out=buf[:, 64:128],
                                pre=buf[:, 128:192]), want)
    t = r.clone()
    assert torch.equal(K.linear(x, w, residual=t, t32=t), want)
    K.linear(x[0], w[0], out=buf.view(torch.bfloat16)[:, :64], pre=buf[:, 32:96])


@pytest.mark.gpu
def test_rotary_refuses_shared_outputs(K):
    from mround_b200.pipeline.block import rope_tables

    cos, sin = rope_tables(6, 8, 1e4, "cuda")
    rows = torch.randn(2, 6, 64, device="cuda")
    heads = lambda first, n: rows[..., first:first + 8 * n].view(2, 6, n, 8)  # noqa: E731
    q, k = heads(0, 4), heads(32, 2)
    fresh = torch.empty(2, 6, 4, 8, device="cuda")
    flat = torch.zeros(2 * 6 * 4 * 8 + 8, device="cuda")
    shifted = flat[:-8].view(2, 6, 4, 8), flat[8:].view(2, 6, 4, 8)
    bad = [(q, k, (q, heads(24, 2))), (q, k, (heads(8, 4), k)), (q, k, (heads(16, 4), None)),
           (q, k, (fresh, fresh[:, :, :2])), (q, None, (heads(8, 4), None)),
           (shifted[0], None, (shifted[1], None)),
           (q, q, (q, torch.empty_like(fresh)))]
    for a, b, out in bad:
        for turn in (K.rotary, K.rotary_bwd):
            with pytest.raises(SchemeError, match="storage|None"):
                turn(a, b, cos, sin, out=out)
    table = torch.zeros(2 * 6 * 4 * 8, device="cuda")
    table[:24].copy_(cos.flatten())
    with pytest.raises(SchemeError, match="cos"):
        K.rotary(q, None, table[:24].view(6, 4), sin, out=(table.view(2, 6, 4, 8), None))
    want = K.rotary(q, k, cos, sin)
    K.rotary(q, k, cos, sin, out=(q, heads(48, 2)))
    assert torch.equal(q, want[0]) and torch.equal(heads(48, 2), want[1])
    K.rotary(heads(48, 2), k, cos, sin, out=(heads(48, 2), k))
    assert torch.equal(k, want[1])


@pytest.mark.gpu
def test_distillation_refuses_shared_outputs(K):
    buf = torch.randn(6, 64, device="cuda")
    t, i = torch.randn(6, 3, device="cuda"), torch.zeros(6, 3, dtype=torch.int64, device="cuda")
    flat = torch.randn(6 * 32 + 4, device="cuda")
    for x, out, teacher, weight in (
            (buf[:, :32], buf[:, 16:48], t, None), (buf[:5, :32], buf[1:, :32], t[:5], None),
            (flat[:-4].view(6, 32), flat[4:].view(6, 32), t, None),
            (buf[:, :32], buf[:, 32:], buf[2, 32:50].view(6, 3), None),
            (buf[:, :32], buf[:, 32:], t, buf[3, 40:46])):
        with pytest.raises(SchemeError, match="storage"):
            K.distill_topk_grad(x, teacher, i[:x.shape[0]], out=out, weight=weight)
    _, want = K.distill_topk_grad(buf[:, :32], t, i)
    _, got = K.distill_topk_grad(buf[:, :32], t, i, out=buf[:, 32:])
    assert torch.equal(got, want)
