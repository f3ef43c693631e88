"""K13 (matrix product with an epilogue, and its gradients) against float64.

Bounds: the tensor cores multiply bf16 exactly and add in float32, one
rounding (or truncation) of at most 2**-23 of a partial sum per 16 k and
product, and per CTA that shares k; with S = sum |x||w| every partial sum is at
most S, so z is within dz = (products * (k / 16 + 1) + 16) * 2**-23 * S (16
covers the join, the bias and 8 shares).  Activations have slopes of at most
1.13 and are evaluated to 2**-20 of |z| (where bf16 alone is written, to 2**-13
of the value: test_activation_over_its_range).  bf16 rounds by at most 2**-8 of the
value, a hi/lo pair leaves 2**-16, tf32 2**-11, float32 2**-24.
"""

from __future__ import annotations

import math

import pytest
import torch

from mround_b200.exceptions import PlatformError, SchemeError


@pytest.fixture(scope="module")
def K():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from mround_b200 import kernels

    return kernels


def parts(t):
    return t if isinstance(t, tuple) else (t, None)


def product(x, w):
    """(sum of the kernel's products, sum of magnitudes, their number), float64."""
    (xh, xl), (wh, wl) = parts(x), parts(w)
    xh, wh = xh.double(), wh.double()
    z, size, count = xh @ wh.t(), xh.abs() @ wh.abs().t(), 1
    for a, b in ((xl, wh), (xh, wl)):
        if a is None or b is None:
            continue
        z = z + a.double() @ b.double().t()
        size, count = size + a.double().abs() @ b.double().abs().t(), count + 1
    return z, size, count


def acted(z, act):
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "gelu":
        return torch.nn.functional.gelu(z)
    if act == "gelu_tanh":
        return torch.nn.functional.gelu(z, approximate="tanh")
    if act == "swiglu":
        g, u = z.chunk(2, 1)
        return g * torch.sigmoid(g) * u
    return z


def bounds(x, w, bias, act, residual):
    """(z, its bound, out, its bound before the output's rounding)."""
    z, size, count = product(x, w)
    k = parts(x)[0].shape[1]
    if bias is not None:
        z, size = z + bias.double(), size + bias.double().abs()
    off = (count * (k / 16 + 1) + 16) * 2.0 ** -23 * size
    y = acted(z, act)
    if act == "swiglu":
        (g, u), (dg, du) = z.chunk(2, 1), off.chunk(2, 1)
        dy = 1.13 * dg * (u.abs() + du) + g.abs() * du + 2.0 ** -20 * (g * u).abs()
    else:
        dy = off if act == "none" else 1.13 * off + 2.0 ** -20 * z.abs()
    if residual is not None:
        y = y + residual.double()
        dy = dy + 2.0 ** -24 * y.abs()
    return z, off, y, dy


def close(got, ref, off, step):
    assert ((got.double() - ref).abs() <= off + step * (ref.abs() + off) + 2.0 ** -126).all()


STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def make(T, F, k, act, kind, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows = 2 * F if act == "swiglu" else F
    ld = -(-k // 8) * 8
    pad = lambda n, s: (torch.randn(n, ld, device="cuda", generator=g) * s)[:, :k]  # noqa: E731
    x, w = pad(T, 1.0), pad(rows, 1.5 / math.sqrt(k))

    def split(t):
        # the row stride of t, so that an odd k keeps a stride of 8
        wide = torch.zeros(t.shape[0], ld, device="cuda")
        wide[:, :k] = t
        hi = wide.bfloat16()
        lo = (wide - hi.float()).bfloat16()
        return hi[:, :k], lo[:, :k]

    xs, ws = split(x), split(w)
    return (xs if kind >= 2 else xs[0]), (ws if kind == 3 else ws[0]), g


def run(K, T, F, k, act, kind, *, bias, residual, splits=None, seed=0):
    x, w, g = make(T, F, k, act, kind, seed)
    rows = parts(w)[0].shape[0]
    b = torch.randn(rows, device="cuda", generator=g) if bias else None
    r = None if residual is None else torch.randn(T, F, device="cuda", generator=g).to(residual)
    z, dz, y, dy = bounds(x, w, b, act, r)
    pre = torch.full((T, rows), math.nan, device="cuda")
    t32 = torch.full((T, F), math.nan, device="cuda")
    for dtype in (torch.float32, torch.bfloat16):
        got = K.linear(x, w, bias=b, act=act, residual=r, dtype=dtype, pre=pre, t32=t32,
                       splits=splits)
        assert got.dtype == dtype
        close(got, y, dy, STEP[dtype])
        close(pre, z, dz, 0.0)
        close(t32, y, dy, 2.0 ** -11)
    hi, lo = K.linear(x, w, bias=b, act=act, residual=r, split=True, splits=splits)
    close(hi.double() + lo.double(), y, dy, 2.0 ** -16)
    assert K.lib().mr_gemm_status(0) == 0


SHAPES = [(1, 1, 1), (1, 130, 72), (2, 64, 64), (7, 200, 1000), (16, 128, 512), (17, 127, 65),
          (33, 300, 200), (64, 129, 2048), (65, 63, 8), (127, 256, 333), (130, 96, 1024),
          (300, 520, 136), (513, 1000, 704)]


@pytest.mark.gpu
@pytest.mark.parametrize("T,F,k", SHAPES)
@pytest.mark.parametrize("kind", [1, 2, 3])
def test_products(K, T, F, k, kind):
    run(K, T, F, k, "none", kind, bias=True, residual=torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh", "swiglu"])
@pytest.mark.parametrize("T,F,k", [(1, 1, 8), (3, 70, 256), (33, 65, 100), (129, 320, 512),
                                   (520, 257, 192)])
@pytest.mark.parametrize("kind", [1, 3])
def test_activations(K, act, T, F, k, kind):
    run(K, T, F, k, act, kind, bias=T % 2 == 1, residual=torch.bfloat16 if T > 3 else None)


@pytest.mark.gpu
@pytest.mark.parametrize("splits", [1, 2, 4, 8])
@pytest.mark.parametrize("T,F,k", [(1, 100, 64), (5, 300, 1100), (40, 129, 520), (200, 140, 4096)])
def test_shared_k(K, splits, T, F, k):
    """Every divisor of k, more CTAs than K slices among them."""
    run(K, T, F, k, "swiglu", 2, bias=True, residual=None, splits=splits)
    run(K, T, F, k, "none", 1, bias=False, residual=torch.float32, splits=splits)


@pytest.mark.gpu
@pytest.mark.parametrize("T,F,k", [(1000, 1500, 640), (2048, 640, 1024), (4100, 4000, 264),
                                   (777, 5000, 72), (256, 20000, 64)])
@pytest.mark.parametrize("act,kind", [("none", 1), ("swiglu", 1), ("swiglu", 3), ("gelu", 2)])
def test_many_tokens(K, T, F, k, act, kind):
    run(K, T, F, k, act, kind, bias=True, residual=torch.bfloat16)


@pytest.mark.gpu
def test_results_of_a_token_do_not_depend_on_the_others(K):
    """splits = 1 fixes the order of the sums across tile shapes and kernels."""
    for act, kind in (("none", 1), ("swiglu", 3), ("silu", 2)):
        x, w, g = make(1200, 700, 1032, act, kind, 3)
        whole = K.linear(x, w, act=act, dtype=torch.float32, splits=1)
        for n in (1, 5, 20, 40, 100, 300, 700):
            some = tuple(p[:n] for p in x) if isinstance(x, tuple) else x[:n]
            assert torch.equal(K.linear(some, w, act=act, dtype=torch.float32, splits=1), whole[:n])


@pytest.mark.gpu
def test_strides_and_results_in_place(K):
    """Column ranges of wider tensors as operands, residual and output; the
    output over the residual; nothing outside is written."""
    g = torch.Generator(device="cuda").manual_seed(4)
    for T, F, k in ((3, 50, 96), (150, 333, 320), (600, 601, 128)):
        x = torch.randn(T, k + 24, device="cuda", generator=g).bfloat16()[:, 8:8 + k]
        w = torch.randn(F, k + 8, device="cuda", generator=g).bfloat16()[:, :k]
        wide = torch.randn(T, F + 13, device="cuda", generator=g)
        before = wide.clone()
        r = wide[:, 5:5 + F]
        _, _, y, dy = bounds(x, w, None, "none", r.clone())
        got = K.linear(x, w, residual=r, out=r)
        assert got.data_ptr() == r.data_ptr()
        close(r, y, dy, 2.0 ** -24)
        assert torch.equal(wide[:, :5], before[:, :5])
        assert torch.equal(wide[:, 5 + F:], before[:, 5 + F:])


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["none", "silu", "gelu", "gelu_tanh", "swiglu"])
@pytest.mark.parametrize("T,F,k", [(1, 3, 8), (5, 66, 40), (70, 200, 136), (333, 130, 512),
                                   (1030, 515, 264)])
def test_gradients(K, act, T, F, k):
    for kind, dy_type in ((1, torch.bfloat16), (3, torch.float32)):
        x, w, g = make(T, F, -(-k // 8) * 8, act, kind, T)
        rows = parts(w)[0].shape[0]
        pre = torch.randn(T, rows, device="cuda", generator=g) * 2
        dy = torch.randn(T, F, device="cuda", generator=g).to(dy_type)
        z = pre.double().requires_grad_()
        dz, = torch.autograd.grad(acted(z, act), z, dy.double())
        # dz in float32: slopes evaluated to 2**-19 of their terms (at most
        # 1 + |z|), then carried as a pair
        size = dy.double().abs()
        if act == "swiglu":
            gate, up = pre.double().chunk(2, 1)
            size = torch.cat([size * up.abs() * (1 + gate.abs()), size * (1 + gate.abs())], 1)
        elif act != "none":
            size = size * (1 + pre.double().abs())
        edz = 2.0 ** -19 * size + 2.0 ** -16 * dz.abs()
        dx, dw, db = K.linear_bwd(dy, x, w, act=act, pre=None if act == "none" else pre,
                                  bias_grad=True, dtype=torch.float32)
        dx16, dw16, none = K.linear_bwd(dy, x, w, act=act, pre=pre, dtype=torch.bfloat16)
        assert none is None
        (xh, xl), (wh, wl) = parts(x), parts(w)
        xd = xh.double() + (0 if xl is None else xl.double())
        wd = wh.double() + (0 if wl is None else wl.double())
        products = 2 if kind == 1 else 3
        for got, got16, a, b, ea in ((dx, dx16, dz, wd, edz), (dw, dw16, dz.t(), xd, edz.t())):
            ref, mass = a @ b, a.abs() @ b.abs()
            n = a.shape[1]
            # lo * lo, which three products leave out: 2**-8 of each factor
            lost = 2.0 ** -16 if kind == 3 else 0.0
            off = (ea @ b.abs() + ((products * (n / 16 + 1) + 16) * 2.0 ** -23 + lost) * 1.01 * mass)
            close(got, ref, off, 2.0 ** -24)
            # bf16 gradients of single operands: dz is rounded to bf16 first, by at
            # most 2**-8 |dz|, hence by 2**-8 sum |dz| |b| in the product
            rounded = 2.0 ** -8 if kind == 1 else 0.0
            # and act' is evaluated for that rounding: an exponential of
            # |v| <= 128 errs by (2 + 1.2 |v|) 2**-23 < 2**-15 of its value, the
            # normal tail by 5.5e-5 < 2**-14, each in a term of size
            rough = 2.0 ** -14 * (size if got16 is dx16 else size.t()) if kind == 1 else 0 * ea
            close(got16, ref, off + rounded * mass + rough @ b.abs(), 2.0 ** -8)
        ref = dz.sum(0)
        off = 2.0 ** -19 * size.sum(0) + (T / 4 + 8) * 2.0 ** -24 * dz.abs().sum(0)
        close(db, ref, off, 2.0 ** -24)


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh", "swiglu"])
def test_gradients_against_differences(K, act):
    """The bias gradient against central differences of sum(dy * out) in each
    bias value: h = 1/64, third derivatives of at most 2 |dy| (1 + |up|)."""
    T, F, k, h = 6, 20, 32, 1.0 / 64
    x, w, g = make(T, F, k, act, 3, 1)
    rows = parts(w)[0].shape[0]
    b = torch.randn(rows, device="cuda", generator=g)
    dy = torch.randn(T, F, device="cuda", generator=g)
    pre = torch.empty(T, rows, device="cuda")
    K.linear(x, w, bias=b, act=act, pre=pre)
    _, _, db = K.linear_bwd(dy, x, w, act=act, pre=pre, bias_grad=True)
    size = pre.double().abs().max() + 1
    for j in range(rows):
        e = torch.zeros(rows, device="cuda")
        e[j] = h
        up, down = (K.linear(x, w, bias=b + s * e, act=act).double() for s in (1, -1))
        diff = (dy.double() * (up - down)).sum() / (2 * h)
        mass = dy.double().abs()[:, j % F].sum()
        bound = mass * size * (2 * h * h / 6 + 2.0 ** -18 * size / h)
        assert abs(diff - db[j].double()) <= bound


@pytest.mark.gpu
def test_outputs_beyond_32_bits(K):
    T, F, k = 70000, 33000, 8
    g = torch.Generator(device="cuda").manual_seed(6)
    x = torch.randn(T, k, device="cuda", generator=g).bfloat16()
    w = torch.randn(F, k, device="cuda", generator=g).bfloat16()
    out = K.linear(x, w)
    for t in (0, 1, 65073, 65074, 65075, T - 1):
        _, _, y, dy = bounds(x[t:t + 1], w, None, "none", None)
        close(out[t:t + 1], y, dy, 2.0 ** -8)


@pytest.mark.gpu
def test_captured_training_step(K):
    """Forward and gradients in two graphs that share nothing, replayed in turn."""
    x, w, g = make(70, 96, 128, "swiglu", 1, 2)
    dy = torch.randn(70, 96, device="cuda", generator=g).bfloat16()
    b = torch.randn(192, device="cuda", generator=g)

    def step():
        pre = torch.empty(70, 192, device="cuda")
        out = K.linear(x, w, bias=b, act="swiglu", pre=pre)
        return (out, *K.linear_bwd(dy, x, w, act="swiglu", pre=pre, bias_grad=True))

    step()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    x.copy_(torch.randn(70, 128, device="cuda", generator=g))
    want = step()
    for graph, _ in graphs * 2:
        graph.replay()
    for _, out in graphs:
        assert all(torch.equal(a, e) for a, e in zip(out, want))


@pytest.mark.gpu
def test_no_tokens(K):
    x, w, _ = make(4, 16, 32, "none", 1)
    assert K.linear(x[:0], w).shape == (0, 16)
    dx, dw, db = K.linear_bwd(torch.empty(0, 16, device="cuda"), x[:0], w, bias_grad=True)
    assert dx.shape == (0, 32) and not dw.any() and not db.any()


def test_refusals():
    from mround_b200 import kernels as K
    from mround_b200._native import LinearOperand
    import ctypes

    x, w = torch.zeros(2, 8, dtype=torch.bfloat16), torch.zeros(4, 8, dtype=torch.bfloat16)
    with pytest.raises(PlatformError, match="CUDA"):
        K.linear(x, w)
    with pytest.raises(SchemeError, match="act"):
        K.linear(x, w, act="relu6")
    with pytest.raises(SchemeError, match="bfloat16"):
        K.linear(x.float(), w)
    lib = K.lib()
    p = 1 << 12

    def call(x=(p, None, 64, 1), w=(p, None, 64, 1), T=4, F=8, k=64, act=0, res=None, rdt=0, ldr=8,
             out=p, odt=0, lo=None, ldo=8, pre=None, ldp=16, splits=0):
        a, b = LinearOperand(*x), LinearOperand(*w)
        return lib.mr_linear(ctypes.addressof(a), ctypes.addressof(b), T, F, k, act, None, res, rdt,
                             ldr, out, odt, lo, None, ldo, pre, ldp, splits, None)

    for bad in (dict(x=(None, None, 64, 1)), dict(x=(p, None, 56, 1)), dict(w=(p, p, 64, 1)),
                dict(T=0), dict(k=0), dict(act=5), dict(splits=3), dict(splits=16), dict(odt=2),
                dict(lo=p), dict(ldo=7), dict(res=p, rdt=2), dict(res=p, ldr=7),
                dict(act=4, w=(p, None, 64, 0)), dict(act=4, pre=p, ldp=15), dict(out=None)):
        assert call(**bad) == -1, bad
    for bad in (dict(x=(p + 2, None, 64, 1)), dict(x=(p, None, 68, 1)), dict(w=(p, None, 66, 1)),
                dict(x=(p, p + 8, 64, 1))):
        assert call(**bad) == -2, bad
    assert lib.mr_act_grad(p, 0, 8, None, 8, 4, 8, 1, p, p, 8, None, None, None) == -1
    assert lib.mr_act_grad(p, 2, 8, p, 8, 4, 8, 1, p, p, 8, None, None, None) == -1
    assert lib.mr_act_grad(p, 0, 8, p, 8, 65535 * 64 + 1, 8, 1, p, p, 8, None, None, None) == -1
    assert lib.mr_act_grad_workspace_bytes(64, 8, 1) == 0  # one strip: none needed
    assert lib.mr_act_grad(p, 0, 8, p, 8, 65, 8, 1, p, p, 8, p, None, None) == -6
    assert lib.mr_act_grad(p, 0, 8, p, 8, 4, 8, 1, None, p, 8, None, None, None) == -1
    assert lib.mr_act_grad(p, 0, 8, p, 8, 4, 8, 1, None, None, 8, None, None, None) == -1


@pytest.mark.gpu
def test_refusals_on_the_device(K):
    x, w, _ = make(4, 16, 32, "none", 1)
    z = lambda *s, **k: torch.zeros(*s, device="cuda", **k)  # noqa: E731
    for bad in (dict(bias=z(15)), dict(bias=z(16).half()), dict(residual=z(4, 15)),
                dict(residual=z(4, 16).half()), dict(out=z(4, 16).half()), dict(dtype=torch.float16),
                dict(pre=z(4, 15)), dict(splits=3), dict(out=z(4, 16), dtype=torch.bfloat16),
                dict(out=z(4, 16), split=True), dict(t32=z(4, 20)[:, :16]),
                dict(out=z(1, 16).expand(4, 16))):
        with pytest.raises(SchemeError):
            K.linear(x, w, **bad)
    for a, b in ((x[:, ::2], w[:, ::2]), (x, w[:, :31]), (x, (w, w)), (x.t(), w), (x[0], w),
                 ((x, x[:2]), w)):
        with pytest.raises(SchemeError):
            K.linear(a, b)
    with pytest.raises(SchemeError, match="gate"):
        K.linear(x, w[:15], act="swiglu")
    odd = z(4, 33, dtype=torch.bfloat16)
    with pytest.raises(SchemeError, match="multiple"):
        K.linear(odd, z(16, 33, dtype=torch.bfloat16))
    with pytest.raises(SchemeError):  # data off the 16-byte grid
        K.linear(z(4, 40, dtype=torch.bfloat16)[:, 1:33], w)
    with pytest.raises(SchemeError, match="pre-activation"):
        K.linear_bwd(z(4, 16), x, w, act="silu")
    with pytest.raises(SchemeError):
        K.linear_bwd(z(4, 15), x, w)
    for dy in (z(4, 16), z(4, 16, dtype=torch.bfloat16)):
        with pytest.raises(SchemeError, match="pair"):
            K.linear_bwd(dy, x, (w, w))
    with pytest.raises(PlatformError):
        K.linear(x, w.cpu())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh", "swiglu"])
def test_activation_over_its_range(K, act, dtype):
    """Each activation alone (one column, weight 1) from far below to far above
    zero, where the tails lose their size first.

    bf16 results hold their own size: half a step, 2^-8 of the value, and the
    activation's 2^-13, down to 2^-100 (smaller ones may be zero).  float32 ones
    hold the size of z: each form is z times a factor of at most 1 that a few
    rounded steps compute, less than 2^-20 with what the exponent's argument,
    at most 128 where the factor is above 2^-126, has lost (2^-24 of it)."""
    z = torch.linspace(-14, 14, 4093, device="cuda").to(torch.bfloat16)
    w = torch.zeros(16 if act == "swiglu" else 8, 8, dtype=torch.bfloat16, device="cuda")
    w[:, 0] = 1
    x = torch.zeros(z.numel(), 8, dtype=torch.bfloat16, device="cuda")
    x[:, 0] = z
    if act == "swiglu":  # silu(z) times 1
        w[8:, 0], w[8:, 1], x[:, 1] = 0, 1, 1
    out = K.linear(x, w, act=act, dtype=dtype).double()
    d = z.double()
    if act == "gelu":
        want = 0.5 * d * torch.special.erfc(-d / math.sqrt(2))
    elif act == "gelu_tanh":
        want = d * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (d + 0.044715 * d ** 3))
    else:
        want = d * torch.sigmoid(d)
    err = (out - want[:, None]).abs()
    if dtype == torch.bfloat16:
        bound = want.abs() * (2.0 ** -8 + 2.0 ** -13) + 2.0 ** -100
    else:
        bound = d.abs() * (2.0 ** -20 + 128 * 2.0 ** -24)
    assert (err <= bound[:, None]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("T,F,k", [(1, 8, 8), (1, 13, 40), (5, 24, 72), (129, 520, 136), (66, 33, 64)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_gradients_of_a_plain_linear(K, T, F, k, dtype):
    """A bf16 dy without an activation, which is itself the products' operand
    where its rows allow; a column slice of a wider one, whose neighbours must
    not be read as its own; and one at an odd offset, which takes the copy."""
    x, w, g = make(T, F, k, "none", 1, 5)
    wide = torch.full((T, F + 24), math.nan, device="cuda", dtype=torch.bfloat16)
    for first in (0, 8, 3):
        dy = wide[:, first:first + F]
        dy.copy_(torch.randn(T, F, device="cuda", generator=g))
        dx, dw, db = K.linear_bwd(dy, x, w, bias_grad=True, dtype=dtype)
        dx1, dw1, none = K.linear_bwd(dy, x, w, dtype=dtype)
        assert none is None and torch.equal(dx, dx1) and torch.equal(dw, dw1)
        for got, a, b in ((dx, dy.double(), w.double()), (dw, dy.double().t(), x.double())):
            mass = a.abs() @ b.abs()
            off = (2 * (a.shape[1] / 16 + 1) + 16) * 2.0 ** -23 * mass
            close(got, a @ b, off, STEP[dtype])
        off = (T / 4 + 8) * 2.0 ** -24 * dy.double().abs().sum(0)
        close(db, dy.double().sum(0), off, 2.0 ** -24)
        wide.fill_(math.nan)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh", "swiglu"])
def test_activation_of_large_values(K, act, dtype):
    """Far from zero an activation is z or nothing, without overflow on the way."""
    z = torch.tensor([1e2, 1e4, 1e20, 3e38, math.inf], device="cuda").to(torch.bfloat16)
    z = torch.cat([z, -z[:-1], torch.tensor([math.nan], device="cuda").to(torch.bfloat16)])
    w = torch.zeros(16 if act == "swiglu" else 8, 8, dtype=torch.bfloat16, device="cuda")
    x = torch.zeros(z.numel(), 8, dtype=torch.bfloat16, device="cuda")
    x[:, 0], x[:, 1] = z, 1
    w[0, 0] = 1
    if act == "swiglu":
        w[8, 1] = 1
    out = K.linear(x, w, act=act, dtype=dtype)[:, 0]
    # swiglu's up row multiplies the infinity by its zero weight: 0 * inf is NaN
    finite = 4 if act == "swiglu" else 5
    assert torch.equal(out[:finite], z[:finite].to(dtype))
    assert (out[5:9].float().abs() <= 2.0 ** -100).all() and out[9].isnan()


@pytest.mark.gpu
def test_refuses_outputs_in_operands(K):
    x, w, g = make(32, 32, 32, "none", 1, 3)
    buf = torch.zeros(32, 64, device="cuda")
    for bad in (dict(out=x), dict(out=w),
                dict(out=buf[:, :32], residual=buf.view(-1)[:1024].view(32, 32)),
                dict(out=buf[:, :32], residual=buf.view(torch.bfloat16)[:, :32])):
        with pytest.raises(SchemeError, match="storage"):
            K.linear(x, w, **bad)


@pytest.mark.gpu
def test_two_streams_at_once(K):
    """Calls that overlap share nothing: the same results as one after another."""
    cases = [make(T, F, 512, act, 1, i) + (act,)
             for i, (T, F, act) in enumerate([(1, 4096, "silu"), (300, 700, "gelu"),
                                              (2000, 1000, "swiglu")])]
    def step(x, w, act):
        pre = torch.empty(x.shape[0], w.shape[0], device="cuda")
        y = K.linear(x, w, act=act, pre=pre)
        return (y, *K.linear_bwd(y, x, w, act=act, pre=pre, bias_grad=True))

    want = [step(x, w, act) for x, w, _, act in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    got = []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                got.append([step(x, w, act) for x, w, _, act in cases])
    torch.cuda.synchronize()
    for run_ in got:
        for a, b in zip(run_, want):
            assert all(torch.equal(p, q) for p, q in zip(a, b))
