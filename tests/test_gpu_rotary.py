"""K10 (rotary positions) against the rotation in float64.

Error bound per value: one rounding to the type (half a step, eps / 2 of the
value; half the smallest subnormal where that is larger) on a float32
expression x1 c -+ x2 s whose three roundings are each at most 2**-24 of
|x1 c| + |x2 s|.
"""

from __future__ import annotations

import pytest
import torch

from mround_b200.exceptions import PlatformError, SchemeError
from mround_b200.pipeline.block import rope_tables

TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


@pytest.fixture(scope="module")
def K():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from mround_b200 import kernels

    return kernels


def turned(x, cos, sin, layout, transposed):
    """(result, sum of the terms' magnitudes) in float64; cos, sin (B, S, r/2)."""
    r = 2 * cos.shape[-1]
    x = x.double()
    c, s = cos.double()[:, :, None], sin.double()[:, :, None]
    if transposed:
        s = -s
    y, size = x.clone(), x.abs()
    i1 = torch.arange(r // 2) if layout == "half" else torch.arange(0, r, 2)
    i2 = i1 + (r // 2 if layout == "half" else 1)
    x1, x2 = x[..., i1], x[..., i2]
    y[..., i1], y[..., i2] = x1 * c - x2 * s, x1 * s + x2 * c
    size[..., i1] = (x1 * c).abs() + (x2 * s).abs()
    size[..., i2] = (x1 * s).abs() + (x2 * c).abs()
    return y, size


def check(got, x, cos, sin, layout, transposed):
    ref, size = turned(x, cos, sin, layout, transposed)
    r = 2 * cos.shape[-1]
    half_step = torch.finfo(got.dtype).eps / 2
    f32 = 3 * 2.0 ** -24 * size
    bound = (ref.abs() + f32) * half_step + f32 + TINY[got.dtype] / 2
    assert ((got.double() - ref).abs() <= bound).all()
    assert torch.equal(got[..., r:], x[..., r:])  # copied


CASES = [
    # batch, positions, q heads, k heads, head dim, rotated columns
    (1, 1, 28, 4, 128, 128),
    (1, 1, 1, 1, 2, 2),
    (2, 33, 3, 1, 64, 32),
    (3, 7, 9, 3, 80, 16),
    (1, 130, 5, 5, 34, 10),
    (2, 5, 2, 1, 7, 6),
    (1, 3, 40, 8, 256, 192),
    (1, 2, 2, 2, 1024, 1024),
    (2, 9, 3, 2, 36, 20),
    (1, 5, 7, 1, 106, 16),
    (1, 2, 1, 1, 1022, 500),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("b,s,hq,hkv,d,r", CASES)
def test_rotation_and_gradient(K, dtype, layout, b, s, hq, hkv, d, r):
    g = torch.Generator(device="cuda").manual_seed(d)
    rows = torch.randn(b, s, (hq + 2 * hkv) * d, device="cuda", generator=g).to(dtype)
    q = rows[..., :hq * d].view(b, s, hq, d)
    k = rows[..., hq * d:(hq + hkv) * d].view(b, s, hkv, d)
    cos, sin = rope_tables(4096, r, 1e4, "cuda")
    pos = torch.randint(0, 4096, (b, s), device="cuda", generator=g)
    for turn, transposed in ((K.rotary, False), (K.rotary_bwd, True)):
        yq, yk = turn(q, k, cos, sin, positions=pos, layout=layout)
        check(yq, q, cos[pos], sin[pos], layout, transposed)
        check(yk, k, cos[pos], sin[pos], layout, transposed)
    only, none = K.rotary(q, None, cos, sin, positions=pos, layout=layout)
    assert none is None and torch.equal(only, K.rotary(q, k, cos, sin, positions=pos,
                                                       layout=layout)[0])


@pytest.mark.gpu
@pytest.mark.parametrize("shift", [0, 1])
def test_strides_positions_and_in_place(K, shift):
    """(B, H, S, D) storage seen as (B, S, H, D), data off the 16-byte grid,
    1-D and int32 positions, results written over the inputs."""
    b, s, h, d = 2, 19, 3, 64
    g = torch.Generator(device="cuda").manual_seed(1)
    store = torch.randn(b * h * s * d + shift, device="cuda", generator=g).to(torch.bfloat16)
    q = store[shift:].view(b, h, s, d).transpose(1, 2)
    k = torch.randn(b, s, 1, d + 3, device="cuda", generator=g).to(torch.bfloat16)[..., 1:d + 1]
    cos, sin = rope_tables(64, d, 1e6, "cuda")
    q0, k0 = q.clone(), k.clone()
    first = torch.arange(s, device="cuda").expand(b, s)
    yq, yk = K.rotary(q, k, cos, sin)
    check(yq, q0, cos[first], sin[first], "half", False)
    check(yk, k0, cos[first], sin[first], "half", False)
    pos = torch.arange(s, device="cuda", dtype=torch.int32).flip(0).contiguous()
    at = pos.long().expand(b, s)
    yq, yk = K.rotary(q, k, cos, sin, positions=pos, out=(q, k))
    assert yq.data_ptr() == q.data_ptr() and yk.data_ptr() == k.data_ptr()
    check(q, q0, cos[at], sin[at], "half", False)
    check(k, k0, cos[at], sin[at], "half", False)


@pytest.mark.gpu
def test_position_outside_the_tables_is_nan(K):
    cos, sin = rope_tables(8, 32, 1e4, "cuda")
    q = torch.ones(1, 4, 2, 48, device="cuda")
    pos = torch.tensor([0, -1, 8, 2 ** 40], device="cuda")
    y, _ = K.rotary(q, None, cos, sin, positions=pos)
    assert torch.isfinite(y[:, 0]).all()
    assert torch.isnan(y[:, 1:, :, :32]).all() and (y[..., 32:] == 1).all()


@pytest.mark.gpu
def test_offsets_beyond_32_bits(K):
    far = 2 ** 32 + 64
    store = torch.empty(far + 64, dtype=torch.bfloat16, device="cuda")
    q = store.as_strided((2, 1, 1, 64), (far, 64, 64, 1))
    q.copy_(torch.randn(2, 1, 1, 64, device="cuda"))
    cos, sin = rope_tables(4, 64, 1e4, "cuda")
    q0 = q.clone()
    pos = torch.tensor([[3], [2]], device="cuda")
    K.rotary(q, None, cos, sin, positions=pos, out=(q, None))
    check(q, q0, cos[pos], sin[pos], "half", False)


@pytest.mark.gpu
def test_graph_and_side_stream(K):
    cos, sin = rope_tables(32, 64, 1e4, "cuda")
    q = torch.randn(1, 5, 2, 64, device="cuda")
    pos = torch.arange(5, device="cuda")
    want = K.rotary(q, None, cos, sin, positions=pos + 3)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    out = torch.zeros_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            K.rotary(q, None, cos, sin, positions=pos, out=(out, None))
    pos.add_(3)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    assert K.rotary(q[:0], None, cos, sin)[0].shape == (0, 5, 2, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("layout,d,r", [("half", 64, 32), ("interleaved", 64, 64),
                                        ("interleaved", 32, 8), ("half", 20, 6),
                                        ("interleaved", 18, 10)])
def test_block_operand_forms(K, layout, d, r):
    """The decoder block's forms: float32 rows to bf16 hi/lo head tensors and
    back.  bf16 rounds by at most 2**-8 of the value: hi leaves 2**-8 |y|, of
    which lo leaves 2**-8, so hi + lo is within 2**-16 |y|."""
    b, s, hq, hkv = 2, 21, 4, 2
    g = torch.Generator(device="cuda").manual_seed(r)
    qkv = torch.randn(b * s, (hq + 2 * hkv) * d, device="cuda", generator=g)
    cos, sin = rope_tables(s, r, 1e4, "cuda")
    heads = qkv.view(b, s, hq + 2 * hkv, d)
    at = torch.arange(s, device="cuda").expand(b, s)
    ref, size = turned(heads, cos[at], sin[at], layout, False)
    ref[:, :, hq + hkv:] = heads[:, :, hq + hkv:].double()
    got = K.rope_split(qkv, cos, sin, b, s, hq, hkv, d, layout=layout, rotary_dim=r)
    got = torch.cat([p[0].double() + p[1].double() for p in got], 1).transpose(1, 2)
    bound = 2.0 ** -16 * ref.abs() + 3 * 2.0 ** -24 * size + 2.0 ** -133
    assert ((got - ref).abs() <= bound * 1.01).all()

    back, size = turned(heads, cos[at], sin[at], layout, True)
    back[:, :, hq + hkv:] = heads[:, :, hq + hkv:].double()
    parts = [heads[:, :, a:e].transpose(1, 2).contiguous()
             for a, e in ((0, hq), (hq, hq + hkv), (hq + hkv, hq + 2 * hkv))]
    hi, lo, t32 = K.rope_bwd_split(*parts, cos, sin, b, s, hq, hkv, d, t32=True, layout=layout,
                                   rotary_dim=r)
    got = (hi.double() + lo.double()).view_as(back)
    bound = 2.0 ** -16 * back.abs() + 3 * 2.0 ** -24 * size + 2.0 ** -133
    assert ((got - back).abs() <= bound * 1.01).all()
    # tf32 keeps 11 significant bits
    off = (t32.double().view_as(back) - back).abs()
    assert (off <= (2.0 ** -11 * back.abs() + 3 * 2.0 ** -24 * size) * 1.01).all()


def test_refusals():
    from mround_b200 import kernels as K

    cos = torch.zeros(8, 16)
    with pytest.raises(PlatformError, match="CUDA"):
        K.rotary(torch.zeros(1, 1, 1, 32), None, cos, cos)
    with pytest.raises(SchemeError, match="layout"):
        K.rotary(torch.zeros(1, 1, 1, 32), None, cos, cos, layout="neox")
    with pytest.raises(SchemeError, match="batch, positions"):
        K.rotary(torch.zeros(1, 1, 32), None, cos, cos)
    lib = K.lib()
    p = 1 << 12
    from mround_b200._native import RotaryHeads
    import ctypes

    h = RotaryHeads(p, p, 32, 32, 32, 32, 32, 32, 1)
    at = ctypes.addressof(h)
    for d, r, rows, dtype in ((32, 3, 8, 0), (32, 34, 8, 0), (2048, 32, 8, 0), (32, 32, 0, 0),
                              (32, 32, 8, 3)):
        assert lib.mr_rotary(at, None, p, p, rows, None, 0, 0, 1, 1, d, r, 0, 0, dtype, None) == -1
    assert lib.mr_rotary_split(p, p, p, 1, 4, 2, 1, 32, 34, 0, p, p, p, p, p, p, None) == -1
    assert lib.mr_rotary_bwd_split(p, p, p, p, p, 1, 4, 2, 1, 32, 16, 0, p, None, None, None) == -1


@pytest.mark.gpu
def test_refusals_on_the_device(K):
    cos, sin = rope_tables(8, 32, 1e4, "cuda")
    q = torch.zeros(1, 4, 2, 32, device="cuda")
    bad = [dict(positions=torch.zeros(3, dtype=torch.int64, device="cuda")),
           dict(positions=torch.zeros(4, device="cuda")),
           dict(out=(q, q)), dict(out=(q.bfloat16(), None)), dict(layout="x")]
    for kw in bad:
        with pytest.raises(SchemeError):
            K.rotary(q, None, cos, sin, **kw)
    with pytest.raises(SchemeError):
        K.rotary(q, q[..., :16], cos, sin)
    with pytest.raises(SchemeError):
        K.rotary(q.expand(1, 4, 2, 32).double(), None, cos, sin)
    with pytest.raises(SchemeError, match="8 rows"):
        K.rotary(torch.zeros(1, 9, 2, 32, device="cuda"), None, cos, sin)
    with pytest.raises(SchemeError, match="contiguous"):
        K.rotary(torch.zeros(1, 4, 2, 64, device="cuda")[..., ::2], None, cos, sin)
    with pytest.raises(SchemeError, match="fit head dim"):
        K.rotary(q[..., :16], None, cos, sin)
    with pytest.raises(PlatformError):
        K.rotary(q, None, cos.cpu(), sin)


@pytest.mark.gpu
def test_refuses_shared_outputs(K):
    """Outputs whose elements share storage, or overlay the input differently."""
    cos, sin = rope_tables(8, 32, 1e4, "cuda")
    q = torch.zeros(2, 4, 2, 32, device="cuda")
    with pytest.raises(SchemeError, match="share storage"):
        K.rotary(q, None, cos, sin, out=(q[:1].expand(2, 4, 2, 32), None))
    with pytest.raises(SchemeError, match="strides"):
        K.rotary(q, None, cos, sin, out=(q.view(2, 2, 4, 32).transpose(1, 2), None))
    one = torch.ones(1, 1, 2, 32, device="cuda")  # strides of single positions do not count
    again = one.as_strided((1, 1, 2, 32), (7, 5, 32, 1))
    want = K.rotary(one, None, cos, sin)[0]
    assert torch.equal(K.rotary(one, None, cos, sin, out=(again, None))[0], want)


def test_packed_arguments():
    """The bytes passed for a structure are the structure's."""
    from mround_b200 import _native as n

    heads = (1 << 40, 3 << 33, 5, 1 << 35, 7, 0, 11, 1 << 41, 13)
    assert n.pack_rotary_heads(*heads) == bytes(n.RotaryHeads(*heads))
    for operand in ((1 << 40, 3 << 33, 1 << 35, 1), (1 << 40, None, 8, 0)):
        packed = n.pack_linear_operand(*(v or 0 for v in operand))
        assert packed == bytes(n.LinearOperand(*operand))
        assert n.unpack_linear_operand(packed) == tuple(v or 0 for v in operand)
