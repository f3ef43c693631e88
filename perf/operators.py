"""Measured cases of the operators a scoring pass by self-distillation runs.

Four operators of ``mround_b200.kernels``: rotary positions (``rotary``,
``rotary_bwd``), the largest logits of each row (``topk_logits``), the
distillation loss against a teacher's top logits with its gradient
(``distill_topk``, ``distill_topk_grad``), and the matrix product with bias,
activation and residual in its epilogue with its gradients (``linear``,
``linear_bwd``).  With ``own`` false, ``run`` computes the same results with
elementary torch operations in float32, rounded once at the end.
"""

from __future__ import annotations

import math

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_BYTES = {"f32": 4, "bf16": 2, "f16": 2}

_MOST_FLOPS = 2 * 8192 * 37888 * 3584  # of the largest product below


def listed():
    return [
        # one new token of one sequence, 100k tokens into its context
        dict(name="rotary one token", op="rotary", dtype="bf16", batch=1, seq=1, hq=28, hkv=4,
             dim=128, rdim=128, layout="half", backward=False, start=100000, table=131072),
        # the calibration batch of the tuning step: 8 sequences of 2048 tokens
        dict(name="rotary batch", op="rotary", dtype="f32", batch=8, seq=2048, hq=28, hkv=4,
             dim=128, rdim=128, layout="half", backward=False, start=0, table=2048),
        # gradient of interleaved pairs over part of a head, odd length, packed positions
        dict(name="rotary gradient", op="rotary", dtype="bf16", batch=3, seq=1021, hq=14, hkv=2,
             dim=80, rdim=32, layout="interleaved", backward=True, start=7, table=8192),
        # the candidates of one decoded token
        dict(name="top logits of one row", op="topk", dtype="f32", rows=1, vocab=151936, k=20,
             masked=0),
        # teacher capture over a scoring batch, vocabulary padded with masked columns
        dict(name="top logits of a batch", op="topk", dtype="bf16", rows=1024, vocab=152064, k=64,
             masked=128),
        # a short scoring sequence of the smallest model
        dict(name="distill few rows", op="distill", dtype="bf16", rows=37, vocab=49152, k=16,
             temperature=2.0, gradient=True),
        # evaluation only: the loss of a scoring batch, odd vocabulary
        dict(name="distill loss", op="distill", dtype="f32", rows=511, vocab=50257, k=100,
             temperature=1.0, gradient=False),
        # loss and gradient of a 2048-token sequence (2047 shifted positions)
        dict(name="distill gradient", op="distill", dtype="f32", rows=2047, vocab=152064, k=64,
             temperature=1.0, gradient=True),
        # gate|up of the MLP for one new token: the weights are read once
        dict(name="linear one token", op="linear", tokens=1, n=18944, k=3584, act="swiglu",
             bias=False, residual=False, backward=False),
        # an output projection with its residual for a short ragged prompt
        dict(name="linear short prompt", op="linear", tokens=333, n=896, k=4864, act="none",
             bias=True, residual=True, backward=False),
        # gate|up of the MLP over four calibration sequences
        dict(name="linear batch", op="linear", tokens=8192, n=18944, k=3584, act="swiglu",
             bias=False, residual=False, backward=False),
        # a training step's linear with its gradients, ragged token count
        dict(name="linear training", op="linear", tokens=2047, n=11008, k=2048, act="gelu_tanh",
             bias=True, residual=False, backward=True),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["rotary", "topk", "distill", "linear"])
    if op == "rotary":
        dim = 2 * _spread(rng, 16, 128)
        hkv = rng.choice([1, 2, 3, 4, 8])
        seq = _spread(rng, 1, 4096)
        start = rng.randrange(0, 100000) if seq < 64 else rng.randrange(0, 64)
        return dict(op=op, dtype=rng.choice(["f32", "bf16", "f16"]),
                    batch=max(1, min(_spread(rng, 1, 32), 16384 // seq)), seq=seq,
                    hq=hkv * rng.randrange(1, 8), hkv=hkv, dim=dim,
                    rdim=dim if rng.random() < 0.6 else 2 * rng.randrange(1, dim // 2 + 1),
                    layout=rng.choice(["half", "interleaved"]), backward=rng.random() < 0.5,
                    start=start, table=start + seq + rng.randrange(0, 500))
    if op == "topk":
        vocab = _spread(rng, 2000, 152064)
        return dict(op=op, dtype=rng.choice(["f32", "bf16", "f16"]), rows=_spread(rng, 1, 1024),
                    vocab=vocab, k=_spread(rng, 1, 128),
                    masked=rng.choice([0, 0, rng.randrange(1, 200)]))
    if op == "distill":
        return dict(op=op, dtype=rng.choice(["f32", "bf16", "f16"]), rows=_spread(rng, 1, 2047),
                    vocab=_spread(rng, 2000, 152064), k=_spread(rng, 1, 128),
                    temperature=rng.choice([1.0, 1.5, 2.0, 4.0]), gradient=rng.random() < 0.6)
    tokens, n, k = _spread(rng, 1, 8192), _spread(rng, 64, 18944), 8 * _spread(rng, 8, 1024)
    backward = rng.random() < 0.4
    act = rng.choice(["none", "silu", "gelu", "gelu_tanh", "swiglu"])
    if backward or tokens > 512:  # no dearer than the largest listed one
        while 2 * tokens * n * k * (2 if act == "swiglu" else 1) * (3 if backward else 1) > _MOST_FLOPS:
            tokens = max(1, tokens // 2)
    return dict(op=op, tokens=tokens, n=n, k=k, act=act, bias=rng.random() < 0.5,
                residual=rng.random() < 0.5, backward=backward)


def _features(case):
    return case["n"] * (2 if case["act"] == "swiglu" else 1)


def work(case):
    op = case["op"]
    if op == "rotary":
        tokens = case["batch"] * case["seq"]
        moved = tokens * (case["hq"] + case["hkv"]) * case["dim"] * 2 * _BYTES[case["dtype"]]
        return {"bytes": moved + case["seq"] * case["rdim"] * 4,
                "flops": tokens * (case["hq"] + case["hkv"]) * case["rdim"] * 3}
    if op == "topk":
        cells = case["rows"] * case["vocab"]
        return {"bytes": cells * _BYTES[case["dtype"]] + case["rows"] * case["k"] * 12,
                "flops": cells}
    if op == "distill":
        cells = case["rows"] * case["vocab"]
        return {"bytes": cells * _BYTES[case["dtype"]] * (2 if case["gradient"] else 1)
                + case["rows"] * (case["k"] * 12 + 8), "flops": cells * 5}
    t, f, k, n = case["tokens"], _features(case), case["k"], case["n"]
    product = 2 * t * f * k
    moved = 2 * (t * k + f * k + t * n * (2 if case["residual"] else 1)) + 4 * f * case["bias"]
    if case["backward"]:  # dy in; dx, dw and the bias gradient out
        return {"bytes": moved + 2 * (t * n + t * k + f * k) + 4 * f * case["bias"],
                "flops": 3 * product}
    return {"bytes": moved, "flops": product}


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def prepare(case, seed):
    g = _generator(seed)
    op = case["op"]
    state = dict(case=case)
    if op == "rotary":
        dt = _TYPES[case["dtype"]]
        b, s, hq, hkv, d = (case[x] for x in ("batch", "seq", "hq", "hkv", "dim"))
        rows = torch.randn(b, s, (hq + 2 * hkv) * d, device="cuda", generator=g).to(dt)
        # q and k as views of the fused projection's rows
        state["q"] = rows[..., :hq * d].view(b, s, hq, d)
        state["k"] = rows[..., hq * d:(hq + hkv) * d].view(b, s, hkv, d)
        half = case["rdim"] // 2
        inv = 1e6 ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half)
        angle = torch.arange(case["table"], dtype=torch.float64, device="cuda")[:, None] * inv
        state["cos"], state["sin"] = angle.cos().float(), angle.sin().float()
        first = case["start"] + torch.randint(0, case["table"] - case["start"] - s + 1, (b, 1),
                                              device="cuda", generator=g)
        state["positions"] = first + torch.arange(s, device="cuda")
        return state
    if op in ("topk", "distill"):
        rows, vocab = case["rows"], case["vocab"]
        # a few likely tokens over a long tail, as a language model's rows have
        x = torch.randn(rows, vocab, device="cuda", generator=g)
        rank = torch.randperm(vocab, device="cuda", generator=g) + 1
        x = (x * 1.8 - 1.1 * rank.float().log()).to(_TYPES[case["dtype"]])
        if op == "topk":
            if case["masked"]:
                x[:, -case["masked"]:] = -math.inf
            state["logits"] = x
            return state
        state["logits"] = x
        k = case["k"]
        noisy = x.float() + 0.5 * torch.randn(rows, vocab, device="cuda", generator=g)
        value, index = noisy.topk(k, dim=1)
        if k > 4:  # some rows kept fewer logits
            short = torch.rand(rows, device="cuda", generator=g) < 0.2
            index[short, -2:] = -1
        state["t_logits"], state["t_index"] = value.contiguous(), index.contiguous()
        # padded positions carry no weight
        state["weight"] = (torch.rand(rows, device="cuda", generator=g) < 0.95).float() / rows
        return state
    t, n, k, f = case["tokens"], case["n"], case["k"], _features(case)
    state["x"] = torch.randn(t, k, device="cuda", generator=g).to(torch.bfloat16)
    state["w"] = (torch.randn(f, k, device="cuda", generator=g) / math.sqrt(k)).to(torch.bfloat16)
    state["bias"] = 0.1 * torch.randn(f, device="cuda", generator=g) if case["bias"] else None
    state["residual"] = (torch.randn(t, n, device="cuda", generator=g).to(torch.bfloat16)
                         if case["residual"] else None)
    if case["backward"]:
        state["dy"] = torch.randn(t, n, device="cuda", generator=g).to(torch.bfloat16)
    return state


# ------------------------------------------------------------------ plain forms
def _rotate(x, cos, sin, layout, backward):
    r = 2 * cos.shape[-1]
    a = x[..., :r].float()
    a1, a2 = (a[..., :r // 2], a[..., r // 2:]) if layout == "half" else (a[..., ::2], a[..., 1::2])
    cos, sin = cos[:, :, None], (-sin if backward else sin)[:, :, None]
    b1, b2 = a1 * cos - a2 * sin, a1 * sin + a2 * cos
    turned = (torch.cat((b1, b2), -1) if layout == "half"
              else torch.stack((b1, b2), -1).reshape(a.shape))
    return torch.cat((turned.to(x.dtype), x[..., r:]), -1)


def _distill(x, t_logits, t_index, weight, temperature, gradient):
    dtype = x.dtype
    x = x.float() / temperature
    top = x.max(1, keepdim=True).values
    e = (x - top).exp()
    total = e.sum(1, keepdim=True)
    kept = t_index >= 0
    at = t_index.clamp(min=0)
    t = torch.where(kept, t_logits.double() / temperature, -math.inf)
    t = t - t.max(1, keepdim=True).values
    p = t.exp()
    p = p / p.sum(1, keepdim=True)
    log_p = t - t.exp().sum(1, keepdim=True).log()
    log_q = (x.gather(1, at) - top).double() - total.double().log()
    term = torch.where(p > 0, p * (log_p - log_q), 0.0)
    loss = (weight.double() * temperature ** 2 * term.sum(1)).float()
    if not gradient:
        return loss
    grad = e / total
    grad.scatter_add_(1, at, -p.float())
    return loss, (grad * (weight * temperature)[:, None]).to(dtype)


def _act(z, act):
    if act == "silu":
        return z / (1 + (-z).exp())
    if act == "gelu":
        return 0.5 * z * (1 + (z * math.sqrt(0.5)).erf())
    if act == "gelu_tanh":
        return 0.5 * z * (1 + (math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)).tanh())
    if act == "swiglu":
        gate, up = z.chunk(2, dim=1)
        return gate / (1 + (-gate).exp()) * up
    return z


def _act_grad(dy, z, act):
    if act == "silu":
        s = 1 / (1 + (-z).exp())
        return dy * s * (1 + z * (1 - s))
    if act == "gelu":
        return dy * (0.5 * (1 + (z * math.sqrt(0.5)).erf())
                     + z * (-0.5 * z * z).exp() / math.sqrt(2 * math.pi))
    if act == "gelu_tanh":
        h = (math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)).tanh()
        return dy * (0.5 * (1 + h) + 0.5 * z * (1 - h * h) * math.sqrt(2 / math.pi)
                     * (1 + 3 * 0.044715 * z * z))
    if act == "swiglu":
        gate, up = z.chunk(2, dim=1)
        s = 1 / (1 + (-gate).exp())
        return torch.cat((dy * up * s * (1 + gate * (1 - s)), dy * gate * s), 1)
    return dy


def _linear(state, case):
    x, w = state["x"].float(), state["w"].float()
    z = x @ w.t()
    if state["bias"] is not None:
        z = z + state["bias"]
    out = _act(z, case["act"])
    if state["residual"] is not None:
        out = out + state["residual"].float()
    out = out.to(torch.bfloat16)
    if not case["backward"]:
        return out
    dz = _act_grad(state["dy"].float(), z, case["act"])
    found = [out, (dz @ w).to(torch.bfloat16), (dz.t() @ x).to(torch.bfloat16)]
    return found + [dz.sum(0)] if case["bias"] else found


def run(state):
    case = state["case"]
    op = case["op"]
    if own:
        return _run_own(state, case, op)
    if op == "rotary":
        cos, sin = state["cos"][state["positions"]], state["sin"][state["positions"]]
        return [_rotate(x, cos, sin, case["layout"], case["backward"])
                for x in (state["q"], state["k"])]
    if op == "topk":
        value, index = state["logits"].float().sort(dim=1, descending=True, stable=True)
        return value[:, :case["k"]].contiguous(), index[:, :case["k"]].contiguous()
    if op == "distill":
        return _distill(state["logits"], state["t_logits"], state["t_index"], state["weight"],
                        case["temperature"], case["gradient"])
    return _linear(state, case)


# ------------------------------------------------------------------ the framework's calls
def _run_own(state, case, op):
    from mround_b200 import kernels

    if op == "rotary":
        turn = kernels.rotary_bwd if case["backward"] else kernels.rotary
        return list(turn(state["q"], state["k"], state["cos"], state["sin"],
                         positions=state["positions"], layout=case["layout"]))
    if op == "topk":
        return kernels.topk_logits(state["logits"], case["k"])
    if op == "distill":
        of = kernels.distill_topk_grad if case["gradient"] else kernels.distill_topk
        return of(state["logits"], state["t_logits"], state["t_index"], weight=state["weight"],
                  temperature=case["temperature"])
    if not case["backward"]:
        return kernels.linear(state["x"], state["w"], bias=state["bias"], act=case["act"],
                              residual=state["residual"])
    pre = torch.empty((case["tokens"], _features(case)), dtype=torch.float32, device="cuda")
    out = kernels.linear(state["x"], state["w"], bias=state["bias"], act=case["act"],
                         residual=state["residual"], pre=pre)
    found = [out, *kernels.linear_bwd(state["dy"], state["x"], state["w"], act=case["act"],
                                      pre=pre, bias_grad=case["bias"])]
    return found if case["bias"] else found[:3]


# ------------------------------------------------------------------ definitions in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op == "rotary":
        r = case["rdim"]
        at = state["positions"].cpu()
        turn = torch.complex(state["cos"].cpu()[at].double(), state["sin"].cpu()[at].double())
        turn = (turn.conj() if case["backward"] else turn)[:, :, None, :]
        found = []
        for x in (state["q"], state["k"]):
            y = x.cpu().double()
            if case["layout"] == "half":
                z = torch.complex(y[..., :r // 2].clone(), y[..., r // 2:r].clone()) * turn
                y[..., :r // 2], y[..., r // 2:r] = z.real, z.imag
            else:
                z = torch.complex(y[..., 0:r:2].clone(), y[..., 1:r:2].clone()) * turn
                y[..., 0:r:2], y[..., 1:r:2] = z.real, z.imag
            found.append(y)
        return found
    if op == "topk":
        value, index = state["logits"].double().sort(dim=1, descending=True, stable=True)
        return value[:, :case["k"]].contiguous(), index[:, :case["k"]].contiguous()
    if op == "distill":
        log_q = torch.log_softmax(state["logits"].double() / case["temperature"], 1)
        t = state["t_logits"].double() / case["temperature"]
        t = t.masked_fill(state["t_index"] < 0, -math.inf)
        log_p = torch.log_softmax(t, 1)
        at = state["t_index"].clamp(min=0)
        p = log_p.exp()
        each = p * (log_p.masked_fill(p == 0, 0.0) - log_q.gather(1, at))
        weight = state["weight"].double()
        loss = each.sum(1) * weight * case["temperature"] ** 2
        if not case["gradient"]:
            return loss
        grad = log_q.exp_().scatter_add_(1, at, -p)
        return loss, grad.mul_((weight * case["temperature"])[:, None])
    x, w = state["x"].double(), state["w"].double()
    z = torch.mm(x, w.t())
    if case["bias"]:
        z += state["bias"].double()
    act = {"none": lambda v: v, "silu": torch.nn.functional.silu,
           "gelu": torch.nn.functional.gelu,
           "gelu_tanh": lambda v: torch.nn.functional.gelu(v, approximate="tanh"),
           "swiglu": lambda v: (torch.nn.functional.silu(v[:, :case["n"]]) * v[:, case["n"]:])}
    z.requires_grad_(case["backward"])
    y = act[case["act"]](z)
    out = y.detach() + (state["residual"].double() if case["residual"] else 0.0)
    if not case["backward"]:
        return out
    (dz,) = torch.autograd.grad(y, z, state["dy"].double())
    found = [out, torch.mm(dz, w), torch.mm(dz.t(), x)]
    return found + [dz.sum(0)] if case["bias"] else found
