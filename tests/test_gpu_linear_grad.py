"""The gradients of K13 where its activations are far out, and what they may not
depend on."""

from __future__ import annotations

import pytest
import torch


@pytest.fixture(scope="module")
def K():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from mround_b200 import kernels

    return kernels


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh", "swiglu"])
def test_slopes_of_large_values(K, act, dtype):
    """Far from zero a slope is 1 or nothing, without overflow on the way; with
    and without the bias gradient, which is that of each token alone here."""
    z = torch.tensor([1e2, 1e4, 1e9, 1e13, 2e13, 1e18, 1e19, 1e20, 3e38], device="cuda")
    z = torch.cat([z, -z])
    n = z.numel()
    up = z > 0
    x = torch.ones(n, 8, device="cuda", dtype=torch.bfloat16)
    dy = torch.ones(n, 1, device="cuda")
    if act == "swiglu":  # silu(z) times 1: the gate's slope, and silu(z) for the up row
        w = torch.zeros(2, 8, device="cuda", dtype=torch.bfloat16)
        w[0, 0] = w[1, 1] = 1
        pre = torch.stack([z, torch.ones_like(z)], 1).contiguous()
    else:
        w = torch.ones(1, 8, device="cuda", dtype=torch.bfloat16)
        pre = z[:, None].contiguous()
    for bias_grad in (True, False):
        dx, _, _ = K.linear_bwd(dy, x, w, act=act, pre=pre, bias_grad=bias_grad, dtype=dtype)
        assert torch.equal(dx[up, 0], torch.ones(n // 2, device="cuda", dtype=dtype))
        assert (dx[~up, 0].float().abs() <= 2.0 ** -100).all()
    for i in range(n):
        _, _, db = K.linear_bwd(dy[i:i + 1], x[i:i + 1], w, act=act, pre=pre[i:i + 1],
                                bias_grad=True, dtype=dtype)
        assert db[0] == 1 if up[i] else abs(db[0]) <= 2.0 ** -100


def operands(T, F, k, act, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows = 2 * F if act == "swiglu" else F
    x = torch.randn(T, k, device="cuda", generator=g).bfloat16()
    w = (torch.randn(rows, k, device="cuda", generator=g) / k ** 0.5).bfloat16()
    dy = torch.randn(T, F, device="cuda", generator=g).bfloat16()
    pre = torch.randn(T, rows, device="cuda", generator=g) * 2
    return x, w, dy, pre


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh", "swiglu"])
@pytest.mark.parametrize("T,F,k", [(5, 66, 40), (200, 515, 264)])
def test_bias_gradient_changes_no_other(K, T, F, k, act, dtype):
    """dx and dw are the same whether the bias gradient is asked for or not."""
    x, w, dy, pre = operands(T, F, k, act, T)
    dx, dw, _ = K.linear_bwd(dy, x, w, act=act, pre=pre, bias_grad=True, dtype=dtype)
    dx1, dw1, none = K.linear_bwd(dy, x, w, act=act, pre=pre, dtype=dtype)
    assert none is None and torch.equal(dx, dx1) and torch.equal(dw, dw1)


@pytest.mark.gpu
@pytest.mark.parametrize("T,F,k", [(128, 200, 136), (129, 200, 136), (300, 520, 264),
                                   (100, 4104, 2056)])
@pytest.mark.parametrize("act", ["none", "silu", "gelu_tanh", "swiglu"])
def test_bf16_gradients_err_by_one_rounding(K, T, F, k, act):
    """Gradients in bf16 are those in float32 rounded: dz is carried as a pair,
    so that both come from the same sums.  float32 against 64 bits is tested
    elsewhere."""
    x, w, dy, pre = operands(T, F, k, act, T)
    for d in (dy, dy.float() + 2.0 ** -10):  # of a float32 dy too
        args = dict(act=act, pre=None if act == "none" else pre)
        dx, dw, _ = K.linear_bwd(d, x, w, dtype=torch.float32, **args)
        dx16, dw16, _ = K.linear_bwd(d, x, w, dtype=torch.bfloat16, **args)
        assert torch.equal(dx16, dx.bfloat16()) and torch.equal(dw16, dw.bfloat16())


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["none", "gelu_tanh", "swiglu"])
def test_gradient_of_a_token_does_not_depend_on_the_others(K, act):
    """splits = 1 fixes the order of the sums, and the tokens' number no precision."""
    x, w, dy, pre = operands(600, 330, 520, act, 7)
    whole, _, _ = K.linear_bwd(dy, x, w, act=act, pre=pre, splits=1)
    for n in (1, 16, 128, 129, 300):
        some, _, _ = K.linear_bwd(dy[:n], x[:n], w, act=act, pre=pre[:n], splits=1)
        assert torch.equal(some, whole[:n])


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["none", "silu", "gelu", "gelu_tanh", "swiglu"])
@pytest.mark.parametrize("T,F,k", [(3, 70, 256), (300, 257, 192), (2100, 640, 520)])
def test_tf32_copy_changes_no_other(K, T, F, k, act):
    """out is the same whether its tf32 copy, or z, is asked for or not."""
    x, w, _, pre = operands(T, F, k, act, T)
    t32 = torch.empty(T, F, device="cuda")
    for dtype in (torch.bfloat16, torch.float32):
        out = K.linear(x, w, act=act, dtype=dtype)
        assert torch.equal(K.linear(x, w, act=act, dtype=dtype, t32=t32), out)
        assert torch.equal(K.linear(x, w, act=act, dtype=dtype, pre=pre), out)
        # the copy is the value before its rounding to bf16, kept to 2^-11 of it
        off = 2.0 ** -11 + (2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24)
        assert ((t32 - out.float()).abs() <= off * (1 + off) * t32.abs() + 2.0 ** -126).all()
