"""K11 (top logits) exactly, and K12 (distillation from them) against float64.

K12's bounds: the sum of exponentials is float32 within a thread (at most
n / 512 + 16 terms of 2**-22 relative error each, each addition 2**-24) and
float64 beyond, so log q and q / q_ref - 1 are within
    e = (n / 512 + 16) * 2**-24 + 2**-21 + 3 * 2**-23 * max|x| / T
(the last: the exponent (x - max) c takes three roundings, of the difference,
of c = log2(e) / T and of the product, and the distance is at most 2 max|x|).
The loss is then within w T^2 e (sum p = 1), plus its own rounding; a gradient within w T (q e + 2**-24 p) plus half a step of its type.
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


def top_ref(x, k):
    v, i = x.float().sort(dim=1, descending=True, stable=True)
    return v[:, :k], i[:, :k]


def check_top(K, x, k):
    v, i = K.topk_logits(x, k)
    rv, ri = top_ref(x, k)
    assert torch.equal(i, ri)
    assert torch.equal(v.nan_to_num(nan=7e37), rv.nan_to_num(nan=7e37))


TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n,k", [(1, 1, 1), (3, 7, 7), (2, 50, 1), (5, 513, 64),
                                      (4, 4097, 100), (3, 50257, 20), (2, 152064, 256),
                                      (300, 2048, 33), (1, 151936, 128)])
def test_top_logits_of_random_rows(K, dtype, rows, n, k):
    g = torch.Generator(device="cuda").manual_seed(n + k)
    check_top(K, torch.randn(rows, n, device="cuda", generator=g).mul_(3).to(dtype), k)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [40, 9001, 70000])
@pytest.mark.parametrize("k", [1, 37, 256])
def test_top_logits_of_awkward_rows(K, n, k):
    """Ties, equal and masked rows, rising and falling rows, NaN, infinities,
    both zeros: the list overflows in most of them."""
    k = min(k, n)
    g = torch.Generator(device="cuda").manual_seed(n)
    ramp = torch.arange(n, device="cuda").float()
    x = torch.stack([
        torch.zeros(n, device="cuda"),
        torch.full((n,), -math.inf, device="cuda"),
        ramp, -ramp, ramp % 3,
        torch.randint(-2, 2, (n,), device="cuda", generator=g).float() * 0.0,
        torch.full((n,), math.nan, device="cuda"),
        torch.randn(n, device="cuda", generator=g),
        torch.randn(n, device="cuda", generator=g),
        torch.full((n,), torch.finfo(torch.float32).min, device="cuda"),
    ])
    x[7, ::5] = math.nan
    x[8, ::7] = math.inf
    x[8, 1::2] = -math.inf
    x[9, n // 2] = -math.inf
    x[1, n - 1] = 0.5
    check_top(K, x, k)
    check_top(K, x.bfloat16(), k)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n,k", [(3, 40000, 64), (3, 40000, 200), (200, 9001, 40),
                                      (160, 50257, 256), (2, 152064, 1)])
def test_top_logits_of_few_levels(K, dtype, rows, n, k):
    """Rows of few distinct values, the largest common or rare, early or late;
    values of one type's smallest size, where the others are zero."""
    g = torch.Generator(device="cuda").manual_seed(n + rows)
    levels = torch.randint(0, 50, (rows, n), device="cuda", generator=g).float()
    check_top(K, levels.to(dtype), k)
    check_top(K, torch.randn(rows, n, device="cuda", generator=g).round().to(dtype), k)
    rising = levels + torch.arange(n, device="cuda") // 1000
    check_top(K, rising.to(dtype), k)
    check_top(K, (-rising).to(dtype), k)
    tiny = levels.to(dtype).mul_(torch.finfo(dtype).smallest_normal).div_(64)
    assert (tiny > 0).any()
    check_top(K, tiny, k)


@pytest.mark.gpu
def test_top_logits_of_strided_rows(K):
    """A column range of wider rows, off the 16-byte grid; the rest is not read."""
    g = torch.Generator(device="cuda").manual_seed(3)
    for dtype in TYPES:
        wide = torch.full((6, 1031), math.inf, device="cuda", dtype=dtype)
        for first in (0, 1, 5):
            x = wide[:, first:first + 1001]
            x.copy_(torch.randn(6, 1001, device="cuda", generator=g))
            check_top(K, x, 50)
            x.fill_(math.inf)
    assert K.topk_logits(wide[:0], 3)[0].shape == (0, 3)


def reference(x, t, i, temperature, w):
    """(loss, gradient, p scattered, q) in float64."""
    log_q = torch.log_softmax(x.double() / temperature, 1)
    kept = i >= 0
    log_p = torch.log_softmax((t.double() / temperature).masked_fill(~kept, -math.inf), 1)
    p = log_p.exp().nan_to_num(nan=0.0)
    at = i.clamp(min=0)
    each = torch.where(p > 0, p * (log_p - log_q.gather(1, at)), torch.zeros_like(p))
    mass = torch.zeros_like(log_q).scatter_add_(1, at, p)
    w = w.double()
    live = ((w != 0) & (p.sum(1) > 0))[:, None]
    q = log_q.exp()
    grad = torch.where(live, (w * temperature)[:, None] * (q - mass), torch.zeros_like(q))
    loss = torch.where(live[:, 0], w * temperature ** 2 * each.sum(1), torch.zeros_like(w))
    return loss, grad, mass, q


def error_of_q(x, temperature):
    n = x.shape[1]
    big = x.float().abs()
    big = big[torch.isfinite(big)].max().item() if torch.isfinite(big).any() else 0.0
    return (n / 512 + 16) * 2.0 ** -24 + 2.0 ** -21 + 3 * 2.0 ** -23 * big / temperature


def check_distill(K, x, t, i, temperature, w):
    loss, grad, mass, q = reference(x, t, i, temperature, w)
    e = error_of_q(x, temperature)
    wt = (w.double().abs() * temperature)[:, None]
    only = K.distill_topk(x, t, i, temperature=temperature, weight=w)
    both, g = K.distill_topk_grad(x, t, i, temperature=temperature, weight=w)
    # the loss alone and the loss beside a gradient add in different orders
    # (blocks of other sizes): each is within the bound, not equal to the other
    for got in (only, both):
        off = wt[:, 0] * temperature * e + 2.0 ** -24 * loss.abs()
        assert ((got.double() - loss).abs() <= off).all()
    step = torch.finfo(x.dtype).eps / 2
    f32 = wt * (q * e + 2.0 ** -23 * mass)
    bound = f32 + (grad.abs() + f32) * step + torch.finfo(x.dtype).smallest_normal * step
    assert ((g.double() - grad).abs() <= bound).all()
    l2, (hi, lo) = K.distill_topk_grad(x, t, i, temperature=temperature, weight=w, split=True)
    assert torch.equal(l2, both)
    pair = hi.double() + lo.double()
    # hi leaves at most 2**-8 |g|, of which lo leaves at most 2**-8
    assert ((pair - grad).abs() <= f32 + 2.0 ** -16 * (grad.abs() + f32) + 2.0 ** -133).all()
    return both, g


def teacher(x, k, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    noisy = x.float() + torch.randn(x.shape, device="cuda", generator=g)
    v, i = noisy.topk(k, dim=1)
    return v.contiguous(), i.contiguous()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n,k,temperature", [
    (1, 1, 1, 1.0), (3, 9, 9, 2.0), (5, 1001, 16, 1.0), (4, 4096, 100, 4.0), (2, 50257, 256, 0.7),
    (3, 152064, 64, 1.0), (170, 515, 3, 1.5)])
def test_distillation(K, dtype, rows, n, k, temperature):
    g = torch.Generator(device="cuda").manual_seed(n)
    x = torch.randn(rows, n, device="cuda", generator=g).mul_(3).to(dtype)
    t, i = teacher(x, k, n + 1)
    w = torch.rand(rows, device="cuda", generator=g) + 0.1
    check_distill(K, x, t, i, temperature, w)


@pytest.mark.gpu
def test_absent_repeated_and_masked_entries(K):
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn(8, 777, device="cuda", generator=g) * 2
    t, i = teacher(x, 6, 8)
    x[2, 700:] = -math.inf                       # masked vocabulary
    x[5] = torch.finfo(torch.float32).min        # a uniform row at the type's lowest value
    i[0, 3:] = -1                                # absent entries
    i[1, 1] = i[1, 0]
    i[1, 4] = i[1, 0]                            # one column three times
    t[2, 1] = -math.inf                          # an entry without mass
    i[2] = torch.arange(6, device="cuda")
    i[3] = -1                                    # no entry at all
    x[4] = math.nan                              # a row without weight
    i[6, 2:] = -1
    t[7, :] = 1e4
    w = torch.ones(8, device="cuda")
    w[4] = 0
    x4, x5 = x[4].clone(), x[5].clone()
    keep = [0, 1, 2, 6, 7]
    check_distill(K, x[keep].contiguous(), t[keep].contiguous(), i[keep].contiguous(), 1.0, w[keep])
    loss, grad = K.distill_topk_grad(x, t, i, weight=w)
    assert loss[3] == 0 and loss[4] == 0 and not grad[3].any() and not grad[4].any()
    # equal logits: q = 1 / 777 everywhere, and KL = sum p log p + log 777
    p = torch.softmax(t[5].double(), 0)
    want = (p * p.log()).sum() + math.log(777)
    off = (777 / 512 + 16) * 2.0 ** -24 + 2.0 ** -21 + 2.0 ** -24 * want.item()
    assert abs(loss[5].item() - want.item()) <= off
    assert torch.equal(x[5], x5) and torch.isnan(x4).all()
    i[6, 0] = 777                                # beyond the vocabulary: that row alone is NaN
    loss2, grad2 = K.distill_topk_grad(x, t, i, weight=w)
    assert torch.isnan(loss2[6]) and torch.isnan(grad2[6]).all()
    assert torch.equal(loss2[:6], loss[:6]) and torch.equal(grad2[:6], grad[:6])


@pytest.mark.gpu
def test_kept_column_the_student_masks(K):
    x = torch.zeros(2, 64, device="cuda")
    x[0, 3] = -math.inf
    x[1] = math.nan
    t, i = torch.zeros(2, 2, device="cuda"), torch.tensor([[3, 4], [3, 4]], device="cuda")
    loss, grad = K.distill_topk_grad(x, t, i)
    assert loss[0] == math.inf and torch.isnan(loss[1]) and torch.isnan(grad[1]).all()
    want = torch.full((64,), 1 / 63, dtype=torch.float64, device="cuda")
    want[3], want[4] = -0.5, 1 / 63 - 0.5
    assert ((grad[0].double() - want).abs() <= 2.0 ** -20).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_strided_and_in_place(K, dtype):
    g = torch.Generator(device="cuda").manual_seed(9)
    wide = torch.randn(7, 1031, device="cuda", generator=g).to(dtype)
    before = wide.clone()
    x = wide[:, 3:1004]
    t, i = teacher(x, 12, 10)
    w = torch.rand(7, device="cuda", generator=g)
    loss, grad = check_distill(K, x, t, i, 2.0, w)
    l2, same = K.distill_topk_grad(x, t, i, temperature=2.0, weight=w, out=x)
    assert same.data_ptr() == x.data_ptr()
    assert torch.equal(l2, loss) and torch.equal(x, grad)
    assert torch.equal(wide[:, :3], before[:, :3]) and torch.equal(wide[:, 1004:], before[:, 1004:])


@pytest.mark.gpu
def test_gradient_against_differences(K):
    """Central differences with h = 0.05: the third derivative of w T^2 KL in
    one logit is at most 0.1 w / T, so they are within h^2 / 60 of the
    gradient, plus the loss's own error over h."""
    g = torch.Generator(device="cuda").manual_seed(2)
    n, h, temperature = 40, 0.05, 1.5
    x = torch.randn(1, n, device="cuda", generator=g)
    t, i = teacher(x, 5, 3)
    _, grad = K.distill_topk_grad(x, t, i, temperature=temperature)
    step = torch.eye(n, device="cuda") * h
    many = lambda s: K.distill_topk(x + s, t.expand(n, -1).contiguous(),  # noqa: E731
                                    i.expand(n, -1).contiguous(), temperature=temperature)
    diff = (many(step) - many(-step)) / (2 * h)
    e = temperature ** 2 * error_of_q(x + step, temperature) + 2.0 ** -24 * 4
    # x + h and x - h are rounded: their distance is off by up to 2**-23 |x|
    assert ((diff - grad[0]).abs() <= h * h / 60 + e / h + 2.0 ** -22 * 4 / h).all()


@pytest.mark.gpu
def test_captured_pass_of_teacher_and_student(K):
    """Teacher's top logits and the student's loss and gradient in one graph,
    replayed on new logits; a second graph of the same calls in between."""
    teach, stud = torch.randn(9, 3001, device="cuda"), torch.randn(9, 3001, device="cuda")

    def step():
        v, i = K.topk_logits(teach, 32)
        return K.distill_topk_grad(stud, v, i, temperature=2.0)

    step()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    for seed in range(2):
        teach.copy_(torch.randn(9, 3001, device="cuda"))
        stud.copy_(torch.randn(9, 3001, device="cuda"))
        want = step()
        for graph, _ in graphs:
            graph.replay()
        for _, out in graphs:
            assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_refusals():
    from mround_b200 import kernels as K

    x, t, i = torch.zeros(2, 8), torch.zeros(2, 3), torch.zeros(2, 3, dtype=torch.int64)
    with pytest.raises(PlatformError, match="CUDA"):
        K.topk_logits(x, 2)
    with pytest.raises(PlatformError, match="CUDA"):
        K.distill_topk_grad(x, t, i)
    lib = K.lib()
    p = 1 << 12
    for n, ld, k, dtype in ((8, 7, 2, 0), (8, 8, 9, 0), (8, 8, 0, 0), (1000, 1000, 257, 0),
                            (8, 8, 2, 3)):
        assert lib.mr_topk_logits(p, 2, n, ld, k, dtype, p, p, None) == -1
    assert lib.mr_topk_logits(p + 2, 2, 8, 8, 2, 0, p, p, None) == -2
    for temperature in (0.0, -1.0, math.nan, math.inf):
        assert lib.mr_distill_topk(p, 2, 8, 8, 0, p, p, 3, temperature, None, p, None, None, None,
                                   0, None) == -1
    for loss, grad, hi, lo, ldg in ((None, None, None, None, 8), (p, p, p, p, 8),
                                    (p, None, p, None, 8), (p, p, None, None, 7)):
        assert lib.mr_distill_topk(p, 2, 8, 8, 0, p, p, 3, 1.0, None, loss, grad, hi, lo, ldg,
                                   None) == -1


@pytest.mark.gpu
def test_refusals_on_the_device(K):
    x = torch.zeros(2, 8, device="cuda")
    t, i = torch.zeros(2, 3, device="cuda"), torch.zeros(2, 3, dtype=torch.int64, device="cuda")
    for bad in (lambda: K.topk_logits(x, 9), lambda: K.topk_logits(x, 0),
                lambda: K.topk_logits(x[0], 2), lambda: K.topk_logits(x.double(), 2),
                lambda: K.topk_logits(x.t(), 1), lambda: K.topk_logits(x[:1].expand(2, 8), 1),
                lambda: K.distill_topk(x, t, i, temperature=0.0),
                lambda: K.distill_topk(x, t[:1], i[:1]), lambda: K.distill_topk(x, t, i.int()),
                lambda: K.distill_topk(x, t.double(), i),
                lambda: K.distill_topk(x, t, i, weight=torch.ones(3, device="cuda")),
                lambda: K.distill_topk_grad(x, t, i, out=torch.zeros(2, 7, device="cuda")),
                lambda: K.distill_topk_grad(x, t, i, out=x, split=True),
                lambda: K.distill_topk_grad(x, t, i, out=x.half())):
        with pytest.raises(SchemeError):
            bad()
    with pytest.raises(PlatformError):
        K.distill_topk(x, t.cpu(), i)


@pytest.mark.gpu
def test_refuses_a_gradient_that_overlays_the_logits_differently(K):
    buf = torch.zeros(4, 16, device="cuda")
    t, i = torch.zeros(2, 3, device="cuda"), torch.zeros(2, 3, dtype=torch.int64, device="cuda")
    with pytest.raises(SchemeError, match="storage"):
        K.distill_topk_grad(buf[:2, :8], t, i, out=buf.view(-1)[:16].view(2, 8))
