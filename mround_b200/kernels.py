"""Torch-tensor front end of the native kernels (the ``mround/kernels`` slot).

Each function validates the tensors it is handed (device, dtype, contiguity,
shape), passes raw pointers and the current CUDA stream to one C entry point
of ``libmround_b200.so``, and returns without synchronizing.  Every function
runs only on the GPU: a CPU tensor is refused with ``PlatformError``.
"""

from __future__ import annotations

import functools

import torch

from mround_b200._native import (
    check,
    lib,
    pack_linear_operand,
    pack_rotary_heads,
    unpack_linear_operand,
)
from mround_b200.exceptions import DeviceError, PlatformError, SchemeError

__all__ = [
    "LossWorkspace",
    "check_products",
    "colsumsq_split",
    "deltaloss",
    "distill_topk",
    "distill_topk_grad",
    "fq_forward",
    "gemm",
    "gemm_batched",
    "gemm_tf32",
    "linear",
    "linear_bwd",
    "loss_apply",
    "loss_hist_pass",
    "loss_outlier",
    "loss_select_digit",
    "pack_mlx",
    "rotary",
    "rotary_bwd",
    "round_tf32",
    "scale_search",
    "split_bf16",
    "ste_signsgd",
    "topk_logits",
]

DEVICE_GROUPS = (8, 16, 32, 64, 128, 256)

# Kernel launches issued through this module (bench.py reports them), and an
# optional timing hook for GEMM launches: when ``GEMM_EVENTS`` is a list, each
# K3 launch appends ``(start_event, end_event, algorithmic_flops, cost)``, cost
# being the launch's tensor work in bf16 products per algorithmic product
# (1-3 for the bf16 splits, TF32_PRODUCT_COST for one tf32 product).
LAUNCHES = [0]
GEMM_EVENTS: list | None = None


def _count(n: int = 1) -> None:
    LAUNCHES[0] += n


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _ptr(t: torch.Tensor | None, dtype: torch.dtype, name: str, numel: int | None = None) -> int | None:
    if t is None:
        return None
    if not t.is_cuda:
        raise PlatformError(f"{name} must be a CUDA tensor (the tuning path has no CPU fallback)")
    if t.dtype != dtype:
        raise SchemeError(f"{name} must be {dtype}, got {t.dtype}")
    if not t.is_contiguous():
        raise SchemeError(f"{name} must be contiguous")
    if numel is not None and t.numel() != numel:
        raise SchemeError(f"{name} has {t.numel()} elements, expected {numel}")
    return t.data_ptr()


def _weight_args(w, v, alpha, beta, group):
    if w.dim() != 2:
        raise SchemeError(f"expected a 2-D weight, got shape {tuple(w.shape)}")
    rows, cols = w.shape
    if group not in DEVICE_GROUPS or cols % group:
        raise SchemeError(f"group {group} is not supported on the device for {cols} columns")
    ng = rows * (cols // group)
    return (
        rows,
        cols,
        _ptr(w, torch.bfloat16, "w", rows * cols),
        _ptr(v, torch.float32, "v", rows * cols),
        _ptr(alpha, torch.float32, "alpha", ng),
        _ptr(beta, torch.float32, "beta", ng),
    )


def _scheme_args(symmetric: bool, init_scale, ng: int):
    if init_scale is not None and not symmetric:
        raise SchemeError("a searched scale belongs to a symmetric scheme")
    return int(bool(symmetric)), _ptr(init_scale, torch.float32, "init_scale", ng)


def fq_forward(w, v, alpha, beta, *, bits: int, group: int, eps: float, wq_hi=None, wq_lo=None,
               wq_f32=None, wq_t32=None, scale=None, zp=None, symmetric: bool = False,
               init_scale=None) -> None:
    """K1: write the fake-quantized weight (bf16 hi/lo split, float32 and/or
    its tf32 rounding -- the backward GEMMs' operand).

    ``symmetric`` selects the symmetric code range; ``init_scale`` (float32,
    one per group) the searched scale.
    """
    rows, cols, pw, pv, pa, pb = _weight_args(w, v, alpha, beta, group)
    n, ng = rows * cols, rows * (cols // group)
    sym, pinit = _scheme_args(symmetric, init_scale, ng)
    status = lib().mr_fq_forward(
        pw, pv, pa, pb, rows, cols, group, bits, sym, pinit, eps,
        _ptr(wq_hi, torch.bfloat16, "wq_hi", n), _ptr(wq_lo, torch.bfloat16, "wq_lo", n),
        _ptr(wq_f32, torch.float32, "wq_f32", n), _ptr(wq_t32, torch.float32, "wq_t32", n),
        _ptr(scale, torch.float32, "scale", ng),
        _ptr(zp, torch.float32, "zp", ng), _stream())
    check(status, "mr_fq_forward")
    _count()


def ste_signsgd(gq, w, v, alpha, beta, *, bits: int, group: int, eps: float, lr: float,
                lo: float, hi: float, update: bool = True, gv=None, galpha=None, gbeta=None,
                wq_hi=None, wq_lo=None, wq_t32=None, symmetric: bool = False,
                init_scale=None) -> None:
    """K2: straight-through gradients, then (if ``update``) the signed step in
    place and the next step's operands (bf16 hi/lo, tf32)."""
    rows, cols, pw, pv, pa, pb = _weight_args(w, v, alpha, beta, group)
    n, ng = rows * cols, rows * (cols // group)
    sym, pinit = _scheme_args(symmetric, init_scale, ng)
    status = lib().mr_ste_signsgd(
        _ptr(gq, torch.float32, "gq", n), pw, pv, pa, pb, rows, cols, group, bits, sym, pinit,
        eps, lr, lo,
        hi, int(bool(update)), _ptr(gv, torch.float32, "gv", n),
        _ptr(galpha, torch.float32, "galpha", ng), _ptr(gbeta, torch.float32, "gbeta", ng),
        _ptr(wq_hi, torch.bfloat16, "wq_hi", n), _ptr(wq_lo, torch.bfloat16, "wq_lo", n),
        _ptr(wq_t32, torch.float32, "wq_t32", n), _stream())
    check(status, "mr_ste_signsgd")
    _count()


def ste_signsgd_codes(gq, w, v, alpha, beta, *, bits: int, group: int, eps: float, lr: float,
                      lo: float, hi: float, codes, qscale, qzp=None, symmetric: bool = False,
                      init_scale=None) -> None:
    """K2's signed step, writing the next step's codes (uint8, one per weight)
    and per-group scale / zero point instead of the operands."""
    rows, cols, pw, pv, pa, pb = _weight_args(w, v, alpha, beta, group)
    n, ng = rows * cols, rows * (cols // group)
    sym, pinit = _scheme_args(symmetric, init_scale, ng)
    status = lib().mr_ste_signsgd_codes(
        _ptr(gq, torch.float32, "gq", n), pw, pv, pa, pb, rows, cols, group, bits, sym, pinit,
        eps, lr, lo, hi, _ptr(codes, torch.uint8, "codes", n),
        _ptr(qscale, torch.float32, "qscale", ng), _ptr(qzp, torch.float32, "qzp", ng), _stream())
    check(status, "mr_ste_signsgd_codes")
    _count()


MAX_K2_SEGMENTS = 8


def ste_signsgd_segments(segments: list[dict], *, group: int, eps: float,
                         symmetric: bool = False) -> None:
    """K2's signed step over up to ``MAX_K2_SEGMENTS`` matrices in one launch.

    Each segment is a dict with ``gq, w, v, alpha, beta`` (tensors), ``bits``,
    ``lr``, ``lo``, ``hi`` and optional ``init_scale``, and either the next
    operands (``wq_hi``, ``wq_lo``, ``wq_t32``) or the next codes (``codes``,
    ``qscale``, ``qzp``).  Bit for bit one ``ste_signsgd(update=True)`` /
    ``ste_signsgd_codes`` per segment."""
    from mround_b200._native import K2Segment

    if not 1 <= len(segments) <= MAX_K2_SEGMENTS:
        raise SchemeError(f"1 to {MAX_K2_SEGMENTS} segments per launch, got {len(segments)}")
    table = (K2Segment * len(segments))()
    for i, sg in enumerate(segments):
        rows, cols, pw, pv, pa, pb = _weight_args(sg["w"], sg["v"], sg["alpha"], sg["beta"], group)
        n, ng = rows * cols, rows * (cols // group)
        init = sg.get("init_scale")
        _, pinit = _scheme_args(symmetric, init, ng)
        table[i] = K2Segment(
            _ptr(sg["gq"], torch.float32, "gq", n), pw, pv, pa, pb, pinit, rows, cols, sg["bits"],
            sg["lr"], sg["lo"], sg["hi"],
            _ptr(sg.get("wq_hi"), torch.bfloat16, "wq_hi", n),
            _ptr(sg.get("wq_lo"), torch.bfloat16, "wq_lo", n),
            _ptr(sg.get("wq_t32"), torch.float32, "wq_t32", n),
            _ptr(sg.get("codes"), torch.uint8, "codes", n),
            _ptr(sg.get("qscale"), torch.float32, "qscale", ng),
            _ptr(sg.get("qzp"), torch.float32, "qzp", ng))
    status = lib().mr_ste_signsgd_segments(table, len(segments), group, int(bool(symmetric)), eps,
                                           _stream())
    check(status, "mr_ste_signsgd_segments")
    _count()


def dequant_split(codes, qscale, qzp, *, group: int, symmetric: bool, wq_hi=None, wq_lo=None,
                  wq_t32=None) -> None:
    """Operands (bf16 hi/lo, tf32) from codes and per-group scale / zero point."""
    rows, cols = codes.shape
    n, ng = rows * cols, rows * (cols // group)
    status = lib().mr_dequant_split(
        _ptr(codes, torch.uint8, "codes", n), _ptr(qscale, torch.float32, "qscale", ng),
        _ptr(qzp, torch.float32, "qzp", ng), rows, cols, group, int(bool(symmetric)),
        _ptr(wq_hi, torch.bfloat16, "wq_hi", n), _ptr(wq_lo, torch.bfloat16, "wq_lo", n),
        _ptr(wq_t32, torch.float32, "wq_t32", n), _stream())
    check(status, "mr_dequant_split")
    _count()


def pack_mlx(w, v, alpha, beta, *, bits: int, group: int, eps: float, want_codes: bool = False,
             symmetric: bool = False, init_scale=None):
    """K5: ``(packed uint32 as int32, scales bf16, biases bf16, codes or None)``.

    Codes are uint8, or int8 under a symmetric scheme.
    """
    rows, cols, pw, pv, pa, pb = _weight_args(w, v, alpha, beta, group)
    sym, pinit = _scheme_args(symmetric, init_scale, rows * (cols // group))
    if 32 % bits == 0:
        if cols % (32 // bits):
            raise SchemeError(f"cols={cols} does not tile {bits}-bit words")
        words = cols // (32 // bits)
    else:
        if cols % 32:
            raise SchemeError(f"cols={cols} is not a multiple of 32 at {bits} bits")
        words = cols // 32 * bits
    dev = w.device
    packed = torch.empty((rows, words), dtype=torch.int32, device=dev)
    scales = torch.empty((rows, cols // group), dtype=torch.bfloat16, device=dev)
    biases = torch.empty_like(scales)
    code_dtype = torch.int8 if sym else torch.uint8
    codes = torch.empty((rows, cols), dtype=code_dtype, device=dev) if want_codes else None
    status = lib().mr_pack_mlx(
        pw, pv, pa, pb, rows, cols, group, bits, sym, pinit, eps, packed.data_ptr(), scales.data_ptr(),
        biases.data_ptr(), None if codes is None else codes.data_ptr(), _stream())
    check(status, "mr_pack_mlx")
    _count()
    return packed, scales, biases, codes


class LossWorkspace:
    """Device scratch of the loss kernels (selection state, histogram, partial sums)."""

    def __init__(self, device: torch.device | str = "cuda") -> None:
        nbytes = int(lib().mr_loss_workspace_bytes())
        self.buffer = torch.zeros(nbytes, dtype=torch.uint8, device=device)
        self.loss = torch.zeros((), dtype=torch.float64, device=device)
        self.thr = torch.zeros((), dtype=torch.float32, device=device)
        self.hist = torch.zeros(2048, dtype=torch.int32, device=device)

    @property
    def ptr(self) -> int:
        return self.buffer.data_ptr()


def loss_outlier(pred, target, ws: LossWorkspace, *, suppress: bool, denom: float, k: int,
                 grad=None, threshold: float | None = None) -> None:
    """K4 single-device: loss into ``ws.loss``, threshold into ``ws.thr``, grad optional."""
    n = pred.numel()
    pp = _ptr(pred, torch.float32, "pred")
    pt = _ptr(target, torch.float32, "target", n)
    status = lib().mr_loss_outlier(
        pp, pt, n, int(k), int(bool(suppress)), float(denom),
        -1.0 if threshold is None else float(threshold), _ptr(grad, torch.float32, "grad", n),
        ws.loss.data_ptr(), ws.thr.data_ptr(), ws.ptr, _stream())
    check(status, "mr_loss_outlier")
    _count(8 if (suppress and threshold is None) else 2)


def loss_hist_pass(pred, target, ws: LossWorkspace, pass_index: int) -> torch.Tensor:
    """One radix pass of the threshold selection; returns this rank's histogram."""
    n = pred.numel()
    status = lib().mr_loss_hist_pass(
        _ptr(pred, torch.float32, "pred"), _ptr(target, torch.float32, "target", n), n,
        int(pass_index), ws.ptr, ws.hist.data_ptr(), _stream())
    check(status, "mr_loss_hist_pass")
    _count()
    return ws.hist


def loss_select_digit(ws: LossWorkspace, k: int, pass_index: int) -> None:
    """Narrow the selection with the (possibly all-reduced) histogram in ``ws.hist``."""
    status = lib().mr_loss_select_digit(ws.hist.data_ptr(), int(k), int(pass_index), ws.ptr,
                                        ws.thr.data_ptr(), _stream())
    check(status, "mr_loss_select_digit")
    _count()


def loss_apply(pred, target, ws: LossWorkspace, *, suppress: bool, denom: float, grad=None) -> None:
    """Loss and gradient with the threshold already in ``ws.thr``."""
    n = pred.numel()
    status = lib().mr_loss_apply(
        _ptr(pred, torch.float32, "pred"), _ptr(target, torch.float32, "target", n), n,
        float(denom), ws.thr.data_ptr(), int(bool(suppress)), _ptr(grad, torch.float32, "grad", n),
        ws.loss.data_ptr(), ws.ptr, _stream())
    check(status, "mr_loss_apply")
    _count(2)


def deltaloss(g, w, *, bits: list[int] | tuple[int, ...], group: int, eps: float, out,
              symmetric: bool = False, grids=None) -> None:
    """K6: ``out[j] += sum |g * (RTN_bits[j](w) - w)|`` (``out`` float64, on device).

    ``grids``: one searched scale tensor per width (float32, one per group) for
    a searched scheme, else None.
    """
    import ctypes

    if w.dim() != 2:
        raise SchemeError("expected a 2-D weight")
    rows, cols = w.shape
    if grids is not None and not symmetric:
        raise SchemeError("searched grids belong to a symmetric scheme")
    widths = (ctypes.c_int * len(bits))(*[int(b) for b in bits])
    grid_arr = None
    if grids is not None:
        if len(grids) != len(bits):
            raise SchemeError("one searched grid per width")
        ptrs = [_ptr(gr, torch.float32, "grid", rows * (cols // group)) for gr in grids]
        grid_arr = ctypes.cast((ctypes.c_void_p * len(ptrs))(*ptrs), ctypes.c_void_p)
    status = lib().mr_deltaloss(
        _ptr(g, torch.float32, "g", rows * cols), _ptr(w, torch.bfloat16, "w", rows * cols),
        rows, cols, group, ctypes.cast(widths, ctypes.c_void_p), len(bits), int(bool(symmetric)),
        grid_arr, eps, _ptr(out, torch.float64, "out", len(bits)), _stream())
    check(status, "mr_deltaloss")
    _count()


def scale_search(w, *, bits: int, group: int, candidates, importance=None, out=None):
    """K8: the searched scale of every group of ``w`` (bf16 (rows, cols)).

    ``candidates``: effective ranges in evaluation order (anchor first), any
    sequence of floats, converted to float32.  ``importance``: float32 (cols,)
    or None.  Returns float32 (rows, cols // group).
    """
    import ctypes

    if w.dim() != 2:
        raise SchemeError("expected a 2-D weight")
    rows, cols = w.shape
    if group not in DEVICE_GROUPS or cols % group:
        raise SchemeError(f"group {group} is not supported on the device for {cols} columns")
    cands = [float(c) for c in candidates]
    if not 1 <= len(cands) <= 256:
        raise SchemeError("1 to 256 candidates")
    arr = (ctypes.c_float * len(cands))(*cands)
    if out is None:
        out = torch.empty((rows, cols // group), dtype=torch.float32, device=w.device)
    status = lib().mr_scale_search(
        _ptr(w, torch.bfloat16, "w", rows * cols), rows, cols, group, bits,
        ctypes.cast(arr, ctypes.c_void_p), len(cands),
        _ptr(importance, torch.float32, "importance", cols),
        _ptr(out, torch.float32, "out", rows * (cols // group)), _stream())
    check(status, "mr_scale_search")
    _count()
    return out


def colsumsq_split(hi, lo, out) -> None:
    """``out[c] += sum_r (hi + lo)[r, c]^2`` for a float32 activation in bf16 parts."""
    if hi.dim() != 2:
        raise SchemeError("expected a 2-D activation")
    rows, cols = hi.shape
    status = lib().mr_colsumsq_split(
        _ptr(hi, torch.bfloat16, "hi", rows * cols),
        _ptr(lo, torch.bfloat16, "lo", rows * cols) if lo is not None else None, rows, cols,
        _ptr(out, torch.float32, "out", cols), _stream())
    check(status, "mr_colsumsq_split")
    _count()


def split_bf16(x, hi=None, lo=None, *, want_lo: bool = True):
    """float32 -> (bf16 hi, bf16 lo); ``hi + lo`` carries 16 significant bits."""
    n = x.numel()
    if hi is None:
        hi = torch.empty(x.shape, dtype=torch.bfloat16, device=x.device)
    if lo is None and want_lo:
        lo = torch.empty(x.shape, dtype=torch.bfloat16, device=x.device)
    status = lib().mr_split_bf16(_ptr(x, torch.float32, "x"), n, _ptr(hi, torch.bfloat16, "hi", n),
                                 _ptr(lo, torch.bfloat16, "lo", n) if lo is not None else None,
                                 _stream())
    check(status, "mr_split_bf16")
    _count()
    return hi, lo


def gemm(a_hi, a_lo, b_hi, b_lo, c, *, m: int, n: int, k: int, a_kmajor: bool, b_kmajor: bool,
         lda: int, ldb: int, ldc: int, precision: int, bias=None, accumulate: bool = False) -> None:
    """K3: ``C[m, n] (+)= sum_k A[m, k] B[n, k]`` on the tcgen05 tensor cores."""
    timing = GEMM_EVENTS is not None
    if timing:
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
    status = lib().mr_gemm(
        _ptr(a_hi, torch.bfloat16, "a_hi"), _ptr(a_lo, torch.bfloat16, "a_lo"), lda, int(a_kmajor),
        _ptr(b_hi, torch.bfloat16, "b_hi"), _ptr(b_lo, torch.bfloat16, "b_lo"), ldb, int(b_kmajor),
        _ptr(c, torch.float32, "c"), ldc, _ptr(bias, torch.float32, "bias"), int(bool(accumulate)),
        m, n, k, precision, _stream())
    check(status, "mr_gemm")
    _count()
    if timing:
        end.record()
        GEMM_EVENTS.append((start, end, 2.0 * m * n * k, precision))


def check_products(device=None) -> None:
    """Raise :class:`DeviceError` if a matrix product of ``device`` (the current one
    when None) gave up a wait, and clear the report.  Synchronizes the device.

    The products (:func:`gemm` and its relatives, :func:`linear`,
    :func:`linear_bwd`) wait for at most 2 s at a time inside the kernel.  One that
    gives up writes nothing, nor do later ones of its kind, and no launch reports
    it: whoever keeps their results calls this first, as tuning does before a block
    is handed on and scoring before its scores are."""
    with torch.cuda.device(device):
        status = int(lib().mr_gemm_status(1))
    if status:
        raise DeviceError("a matrix product gave up waiting on the device; results since the last "
                          f"check are not valid (status {status})")


def gemm_rs(a_hi, a_lo, b_hi, b_lo, *, m: int, n: int, k: int, a_kmajor: bool, b_kmajor: bool,
            lda: int, ldb: int, precision: int, dst_ptrs, ldd: int, rows_per_rank: int,
            flag_ptrs, done, epoch: int) -> None:
    """K3 whose rows go to their owner ranks over NVLink (fused reduce-scatter).

    ``dst_ptrs[o]`` / ``flag_ptrs[o]``: device addresses (ints) of rank o's
    slot and flag for this source rank; ``done``: this rank's zeroed int32
    counter; ``epoch``: the exchange's step number (> 0, increasing).
    """
    import ctypes

    world = len(dst_ptrs)
    if len(flag_ptrs) != world:
        raise SchemeError("one flag per destination rank")
    timing = GEMM_EVENTS is not None
    if timing:
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
    dsts = (ctypes.c_void_p * world)(*dst_ptrs)
    flags = (ctypes.c_void_p * world)(*flag_ptrs)
    status = lib().mr_gemm_rs(
        _ptr(a_hi, torch.bfloat16, "a_hi"), _ptr(a_lo, torch.bfloat16, "a_lo"), lda, int(a_kmajor),
        _ptr(b_hi, torch.bfloat16, "b_hi"), _ptr(b_lo, torch.bfloat16, "b_lo"), ldb, int(b_kmajor),
        m, n, k, precision, ctypes.cast(dsts, ctypes.c_void_p), ldd, rows_per_rank,
        ctypes.cast(flags, ctypes.c_void_p), world, _ptr(done, torch.int32, "done", 1), int(epoch),
        _stream())
    check(status, "mr_gemm_rs")
    _count()
    if timing:
        end.record()
        GEMM_EVENTS.append((start, end, 2.0 * m * n * k, precision))


# tensor time of one tf32 product, in bf16 products (tf32 runs at half the rate)
TF32_PRODUCT_COST = 2


def gemm_tile(*, m: int, n: int, k: int, precision: int, a_kmajor: bool, b_kmajor: bool,
              batch: int = 1, causal: int = 0) -> tuple[int, int]:
    """The output tile (rows, columns) K3 uses for this shape."""
    args = (m, n, k, batch, precision, int(a_kmajor), int(b_kmajor), causal)
    rows, width = int(lib().mr_gemm_tile_m(*args)), int(lib().mr_gemm_tile_n(*args))
    check(min(rows, width, 0), "mr_gemm_tile")
    return rows, width


def gemm_tile_n(*, m: int, n: int, k: int, precision: int, a_kmajor: bool, b_kmajor: bool,
                batch: int = 1, causal: int = 0) -> int:
    """The output tile width (128, 224 or 256) K3 uses for this shape."""
    return gemm_tile(m=m, n=n, k=k, precision=precision, a_kmajor=a_kmajor, b_kmajor=b_kmajor,
                     batch=batch, causal=causal)[1]


def gemm_tf32(a, b, c, *, m: int, n: int, k: int, a_kmajor: bool, b_kmajor: bool, lda: int,
              ldb: int, ldc: int, bias=None, accumulate: bool = False) -> None:
    """K3, one tf32 product: ``C[m, n] (+)= sum_k A[m, k] B[n, k]`` with float32
    operands already rounded to tf32 (``round_tf32`` or a kernel's t32 output)."""
    timing = GEMM_EVENTS is not None
    if timing:
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
    status = lib().mr_gemm_tf32(
        _ptr(a, torch.float32, "a"), lda, int(a_kmajor), _ptr(b, torch.float32, "b"), ldb,
        int(b_kmajor), _ptr(c, torch.float32, "c"), ldc, _ptr(bias, torch.float32, "bias"),
        int(bool(accumulate)), m, n, k, _stream())
    check(status, "mr_gemm_tf32")
    _count()
    if timing:
        end.record()
        GEMM_EVENTS.append((start, end, 2.0 * m * n * k, TF32_PRODUCT_COST))


def gemm_rs_tf32(a, b, *, m: int, n: int, k: int, a_kmajor: bool, b_kmajor: bool, lda: int,
                 ldb: int, dst_ptrs, ldd: int, rows_per_rank: int, flag_ptrs, done,
                 epoch: int) -> None:
    """``gemm_rs`` with one tf32 product of float32 operands."""
    import ctypes

    world = len(dst_ptrs)
    if len(flag_ptrs) != world:
        raise SchemeError("one flag per destination rank")
    timing = GEMM_EVENTS is not None
    if timing:
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
    dsts = (ctypes.c_void_p * world)(*dst_ptrs)
    flags = (ctypes.c_void_p * world)(*flag_ptrs)
    status = lib().mr_gemm_rs_tf32(
        _ptr(a, torch.float32, "a"), lda, int(a_kmajor), _ptr(b, torch.float32, "b"), ldb,
        int(b_kmajor), m, n, k, ctypes.cast(dsts, ctypes.c_void_p), ldd, rows_per_rank,
        ctypes.cast(flags, ctypes.c_void_p), world, _ptr(done, torch.int32, "done", 1), int(epoch),
        _stream())
    check(status, "mr_gemm_rs_tf32")
    _count()
    if timing:
        end.record()
        GEMM_EVENTS.append((start, end, 2.0 * m * n * k, TF32_PRODUCT_COST))


def reduce_slots(slots, flags, epoch: int, out) -> None:
    """Wait for every source's flag to reach ``epoch``, then out = sum of the
    ``slots`` (world, ...) in rank order."""
    world = slots.shape[0]
    n = out.numel()
    status = lib().mr_reduce_slots(
        _ptr(slots, torch.float32, "slots"), slots[0].numel(), n, world,
        _ptr(flags, torch.int64, "flags", world), int(epoch), _ptr(out, torch.float32, "out", n),
        _stream())
    check(status, "mr_reduce_slots")
    _count()


def peer_send(dst_ptr: int, src, flag_ptr: int, epoch: int) -> None:
    """Copy ``src`` (contiguous float32 rows) to ``dst_ptr`` with the copy
    engine, then release ``epoch`` into the flag at ``flag_ptr`` -- both on the
    current stream."""
    if not src.is_contiguous():
        raise SchemeError("peer_send needs contiguous rows")
    status = lib().mr_peer_send(dst_ptr, _ptr(src, torch.float32, "src"), src.numel() * 4,
                                flag_ptr, int(epoch), _stream())
    check(status, "mr_peer_send")
    _count()


def causal_fraction(causal: int, m: int, n: int, k: int, seq: int, bk: int = 64) -> float:
    """Share of the dense tile work a causal mode of K3 actually computes
    (mirrors the kernel's tile and K-tile predicates; BM = 128, K slices of
    ``bk``: 64 when both operands are MN-major, else 32)."""
    if not causal:
        return 1.0
    bm = 128
    bn = 128 if n <= 128 else 256
    m_tiles = -(-m // bm)
    k_tiles = -(-k // bk)
    n_tiles = -(-n // bn)
    done = 0
    for tm in range(m_tiles):
        m0 = tm * bm
        if causal == 1:
            done += min(n_tiles, (m0 % seq + bm - 1) // bn + 1) * k_tiles
        elif causal == 2:
            done += min(k_tiles, (m0 % seq + bm + bk - 1) // bk) * n_tiles
        else:
            done += sum(1 for kt in range(k_tiles) if (kt * bk) % seq + bk - 1 >= m0) * n_tiles
    return done / (m_tiles * n_tiles * k_tiles)


def gemm_batched(a_hi, a_lo, b_hi, b_lo, c, *, m: int, n: int, k: int, batch: int, a_kmajor: bool,
                 b_kmajor: bool, lda: int, ldb: int, ldc: int, stride_a: int, stride_b: int,
                 stride_c: int, precision: int, accumulate: bool = False, causal: int = 0,
                 seq: int = 0) -> None:
    """K3 over ``batch`` equally shaped problems in one launch (``causal``: see the header)."""
    timing = GEMM_EVENTS is not None
    if timing:
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
    status = lib().mr_gemm_batched(
        _ptr(a_hi, torch.bfloat16, "a_hi"), _ptr(a_lo, torch.bfloat16, "a_lo"), lda, stride_a,
        int(a_kmajor), _ptr(b_hi, torch.bfloat16, "b_hi"), _ptr(b_lo, torch.bfloat16, "b_lo"), ldb,
        stride_b, int(b_kmajor), _ptr(c, torch.float32, "c"), ldc, stride_c, None,
        int(bool(accumulate)), m, n, k, batch, precision, int(causal), int(seq), _stream())
    check(status, "mr_gemm_batched")
    _count()
    if timing:
        end.record()
        frac = causal_fraction(causal, m, n, k, seq, 64 if not (a_kmajor or b_kmajor) else 32)
        GEMM_EVENTS.append((start, end, 2.0 * m * n * k * batch * frac, precision))


# ---------------------------------------------------------------- block ops
def _pair(shape, device):
    return (torch.empty(shape, dtype=torch.bfloat16, device=device),
            torch.empty(shape, dtype=torch.bfloat16, device=device))


def _t32(shape, device, want: bool):
    return torch.empty(shape, dtype=torch.float32, device=device) if want else None


def rmsnorm_split(x, w, eps: float, *, t32: bool = False):
    """x (T, h) float32, w (h,) bf16 -> (hi, lo, rstd, tf32 copy or None)."""
    t, h = x.shape
    hi, lo = _pair((t, h), x.device)
    tt = _t32((t, h), x.device, t32)
    rstd = torch.empty(t, dtype=torch.float32, device=x.device)
    st = lib().mr_rmsnorm_split(_ptr(x, torch.float32, "x"), _ptr(w, torch.bfloat16, "w", h), t, h,
                                eps, hi.data_ptr(), lo.data_ptr(),
                                _ptr(tt, torch.float32, "t32", t * h), rstd.data_ptr(), _stream())
    check(st, "mr_rmsnorm_split")
    _count()
    return hi, lo, rstd, tt


def rmsnorm_bwd_split(dy, x, w, rstd, resid, *, split: bool = True, t32: bool = False, out=None):
    """RMSNorm backward plus ``resid`` (or None): ``(hi, lo)`` when ``split``,
    the tf32-rounded copy when ``t32``, and the float32 gradient written to
    ``out`` when given.  Returns (hi, lo, t32) with None for what was not asked."""
    t, h = x.shape
    hi, lo = _pair((t, h), x.device) if split else (None, None)
    tt = _t32((t, h), x.device, t32)
    st = lib().mr_rmsnorm_bwd_split(
        _ptr(dy, torch.float32, "dy", t * h), _ptr(x, torch.float32, "x"),
        _ptr(w, torch.bfloat16, "w", h), _ptr(rstd, torch.float32, "rstd", t),
        _ptr(resid, torch.float32, "resid", t * h), t, h, None if hi is None else hi.data_ptr(),
        None if lo is None else lo.data_ptr(), _ptr(tt, torch.float32, "t32", t * h),
        _ptr(out, torch.float32, "out", t * h), _stream())
    check(st, "mr_rmsnorm_bwd_split")
    _count()
    return hi, lo, tt


def _whole_half(layout: str, rotary_dim, d: int) -> bool:
    """Whether the rotation is the half layout over the whole head."""
    _interleaved(layout)
    return layout == "half" and rotary_dim in (None, d)


def rope_split(qkv, cos, sin, b: int, s: int, hq: int, hkv: int, d: int, *, layout: str = "half",
               rotary_dim: int | None = None):
    """qkv rows -> rope(q), rope(k), v as (B, H, S, D) hi/lo pairs.  ``rotary_dim``: the
    head's rotated columns (tables (s, rotary_dim / 2)), the whole head by default."""
    dev = qkv.device
    q = _pair((b, hq, s, d), dev)
    k = _pair((b, hkv, s, d), dev)
    v = _pair((b, hkv, s, d), dev)
    if not _whole_half(layout, rotary_dim, d):
        r = d if rotary_dim is None else rotary_dim
        st = lib().mr_rotary_split(_ptr(qkv, torch.float32, "qkv", b * s * (hq + 2 * hkv) * d),
                                   _ptr(cos, torch.float32, "cos", s * r // 2),
                                   _ptr(sin, torch.float32, "sin", s * r // 2), b, s, hq, hkv, d,
                                   r, _interleaved(layout), q[0].data_ptr(), q[1].data_ptr(),
                                   k[0].data_ptr(), k[1].data_ptr(), v[0].data_ptr(),
                                   v[1].data_ptr(), _stream())
        check(st, "mr_rotary_split")
        _count()
        return q, k, v
    st = lib().mr_rope_split(_ptr(qkv, torch.float32, "qkv", b * s * (hq + 2 * hkv) * d),
                             _ptr(cos, torch.float32, "cos", s * d // 2),
                             _ptr(sin, torch.float32, "sin", s * d // 2), b, s, hq, hkv, d,
                             q[0].data_ptr(), q[1].data_ptr(), k[0].data_ptr(), k[1].data_ptr(),
                             v[0].data_ptr(), v[1].data_ptr(), _stream())
    check(st, "mr_rope_split")
    _count()
    return q, k, v


def rope_bwd_split(dq, dk, dv, cos, sin, b: int, s: int, hq: int, hkv: int, d: int, *,
                   split: bool = True, t32: bool = False, layout: str = "half",
                   rotary_dim: int | None = None):
    """The qkv-row gradient as (hi, lo, tf32 copy), None for what was not asked."""
    shape = (b * s, (hq + 2 * hkv) * d)
    hi, lo = _pair(shape, dq.device) if split else (None, None)
    tt = _t32(shape, dq.device, t32)
    if not _whole_half(layout, rotary_dim, d):
        r = d if rotary_dim is None else rotary_dim
        nq, nkv = b * s * hq * d, b * s * hkv * d
        st = lib().mr_rotary_bwd_split(
            _ptr(dq, torch.float32, "dq", nq), _ptr(dk, torch.float32, "dk", nkv),
            _ptr(dv, torch.float32, "dv", nkv), _ptr(cos, torch.float32, "cos", s * r // 2),
            _ptr(sin, torch.float32, "sin", s * r // 2), b, s, hq, hkv, d, r, _interleaved(layout),
            None if hi is None else hi.data_ptr(), None if lo is None else lo.data_ptr(),
            _ptr(tt, torch.float32, "t32", shape[0] * shape[1]), _stream())
        check(st, "mr_rotary_bwd_split")
        _count()
        return hi, lo, tt
    st = lib().mr_rope_bwd_split(_ptr(dq, torch.float32, "dq"), _ptr(dk, torch.float32, "dk"),
                                 _ptr(dv, torch.float32, "dv"), _ptr(cos, torch.float32, "cos"),
                                 _ptr(sin, torch.float32, "sin"), b, s, hq, hkv, d,
                                 None if hi is None else hi.data_ptr(),
                                 None if lo is None else lo.data_ptr(),
                                 _ptr(tt, torch.float32, "t32", shape[0] * shape[1]), _stream())
    check(st, "mr_rope_bwd_split")
    _count()
    return hi, lo, tt


def heads_split(src, b: int, s: int, h: int, d: int, *, merge: bool, t32: bool = False):
    """Head layout change as (hi, lo, tf32 copy or None)."""
    shape = (b * s, h * d) if merge else (b, h, s, d)
    hi, lo = _pair(shape, src.device)
    tt = _t32(shape, src.device, t32)
    st = lib().mr_heads_split(_ptr(src, torch.float32, "src", b * s * h * d), b, s, h, d, int(merge),
                              hi.data_ptr(), lo.data_ptr(),
                              _ptr(tt, torch.float32, "t32", b * s * h * d), _stream())
    check(st, "mr_heads_split")
    _count()
    return hi, lo, tt


def swiglu_split(gu, t: int, i: int, *, t32: bool = False):
    """silu(g) * u as (hi, lo, tf32 copy or None), from a gate|up that is at hand;
    the block's forward has it from the epilogue of :func:`linear`, bit for bit."""
    hi, lo = _pair((t, i), gu.device)
    tt = _t32((t, i), gu.device, t32)
    st = lib().mr_swiglu_split(_ptr(gu, torch.float32, "gu", t * 2 * i), t, i, hi.data_ptr(),
                               lo.data_ptr(), _ptr(tt, torch.float32, "t32", t * i), _stream())
    check(st, "mr_swiglu_split")
    _count()
    return hi, lo, tt


def swiglu_bwd_split(dact, gu, t: int, i: int, *, split: bool = True, t32: bool = False):
    """The gate|up gradient as (hi, lo, tf32 copy), None for what was not asked."""
    hi, lo = _pair((t, 2 * i), gu.device) if split else (None, None)
    tt = _t32((t, 2 * i), gu.device, t32)
    st = lib().mr_swiglu_bwd_split(_ptr(dact, torch.float32, "dact", t * i),
                                   _ptr(gu, torch.float32, "gu", t * 2 * i), t, i,
                                   None if hi is None else hi.data_ptr(),
                                   None if lo is None else lo.data_ptr(),
                                   _ptr(tt, torch.float32, "t32", t * 2 * i), _stream())
    check(st, "mr_swiglu_bwd_split")
    _count()
    return hi, lo, tt


def ce_grad_split(logits, labels, scale: float):
    """(softmax(logits) - onehot(labels)) * scale per row, as bf16 (hi, lo)."""
    rows, vocab = logits.shape
    hi, lo = _pair((rows, vocab), logits.device)
    if labels.dtype != torch.int64 or not labels.is_contiguous() or labels.numel() != rows:
        raise SchemeError("labels must be a contiguous int64 tensor of one label per row")
    st = lib().mr_ce_grad_split(_ptr(logits, torch.float32, "logits"), labels.data_ptr(), rows,
                                vocab, float(scale), hi.data_ptr(), lo.data_ptr(), _stream())
    check(st, "mr_ce_grad_split")
    _count()
    return hi, lo


def round_tf32(x, out=None):
    """float32 -> its tf32 rounding (round to nearest, ties away), float32."""
    n = x.numel()
    if out is None:
        out = torch.empty_like(x)
    st = lib().mr_round_tf32(_ptr(x, torch.float32, "x"), n, _ptr(out, torch.float32, "out", n),
                             _stream())
    check(st, "mr_round_tf32")
    _count()
    return out


def softmax_causal_split(scores, rows: int, s: int, scale: float, band: bool = False):
    """Causal softmax (row r at position r % s) as bf16 hi/lo parts; ``scores``
    is left unchanged."""
    hi, lo = _pair(scores.shape, scores.device)
    st = lib().mr_softmax_causal_split(_ptr(scores, torch.float32, "scores", rows * s), rows, s,
                                       float(scale), int(band), hi.data_ptr(), lo.data_ptr(),
                                       _stream())
    check(st, "mr_softmax_causal_split")
    _count()
    return hi, lo


def softmax_bwd_split(dp, p, rows: int, s: int, scale: float, band: bool = False):
    """Softmax backward from dP (float32) and P as its (hi, lo) parts."""
    hi, lo = _pair(dp.shape, dp.device)
    st = lib().mr_softmax_bwd_split(_ptr(dp, torch.float32, "dp", rows * s),
                                    _ptr(p[0], torch.bfloat16, "p_hi", rows * s),
                                    _ptr(p[1], torch.bfloat16, "p_lo", rows * s), rows, s,
                                    float(scale), int(band), hi.data_ptr(), lo.data_ptr(),
                                    _stream())
    check(st, "mr_softmax_bwd_split")
    _count()
    return hi, lo


# ------------------------------------------------- rotary, logits and linear operators
# Unlike the functions above, these take tensors of any CUDA device and launch
# on that device's current stream.  Like them they are not recorded by autograd: an
# input that requires a gradient gives an output that does not, and the gradients
# are what the *_bwd and *_grad functions return.
DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _interleaved(layout: str) -> int:
    if layout not in ("half", "interleaved"):
        raise SchemeError(f"layout must be 'half' or 'interleaved', got {layout!r}")
    return int(layout == "interleaved")


def _device_of(names: str, *tensors) -> int:
    """The index of the CUDA device all given tensors (None apart) share."""
    dev = None
    for t in tensors:
        if t is not None:
            index = t.get_device()
            if index != dev or index < 0:
                if index < 0 or dev is not None:
                    name = next(n for n, u in zip(names.split(), tensors) if u is t)
                    if index < 0:
                        raise PlatformError(f"{name} must be a CUDA tensor (there is no CPU "
                                            "fallback)")
                    raise SchemeError(f"{name} is on cuda:{index}, expected cuda:{dev}")
                dev = index
    return dev


# the stream's handle alone: torch.cuda.current_stream() builds an object (3 us).
# Device and stream are asked for once a CUDA tensor is at hand, so the lazy
# initialization that torch.cuda.current_device() checks for (1 us) has been.
_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _launch(name: str, dev: int, *args) -> None:
    """One C entry point on device ``dev``'s current stream (appended to ``args``)."""
    fn = getattr(lib(), name)
    if dev == _current_device():
        status = fn(*args, _raw_stream(dev))
    else:
        with torch.cuda.device(dev):
            status = fn(*args, _raw_stream(dev))
    if status:
        check(status, name)
    LAUNCHES[0] += 1


def _strides(t: torch.Tensor) -> list[int]:
    """The strides that count: of dimensions with more than one element."""
    return [stride for size, stride in zip(t.shape, t.stride()) if size > 1]


@functools.lru_cache(maxsize=1024)
def _extent(shape, stride, size: int) -> int:
    """Bytes from a layout's first element to behind its last."""
    return (sum((n - 1) * s for n, s in zip(shape, stride)) + 1) * size if 0 not in shape else 0


def _meet(a, b, size_a: int, size_b: int, shift: int) -> bool:
    """Whether two layouts, the second's first byte ``shift`` after the first's, may
    share a byte.  Dimensions are (stride in bytes, extent), largest stride first.
    A stride that both step by is taken out, and what is left of both compared
    within one period; False is certain, True is not where the strides differ."""
    span_a = sum(s * (n - 1) for s, n in a) + size_a
    span_b = sum(s * (n - 1) for s, n in b) + size_b
    if shift >= span_a or -shift >= span_b:
        return False
    period = max(a[0][0] if a else 0, b[0][0] if b else 0)
    if period == 0:
        return True
    rest_a = a[1:] if a and a[0][0] == period else a
    rest_b = b[1:] if b and b[0][0] == period else b
    if (sum(s * (n - 1) for s, n in rest_a) + size_a > period
            or sum(s * (n - 1) for s, n in rest_b) + size_b > period):
        return True
    shift %= period
    return (_meet(rest_a, rest_b, size_a, size_b, shift)
            or _meet(rest_a, rest_b, size_a, size_b, shift - period))


@functools.lru_cache(maxsize=1024)
def _layouts_meet(shape_a, stride_a, size_a: int, shape_b, stride_b, size_b: int,
                  shift: int) -> bool:
    dims = [sorted(((s * size, n) for n, s in zip(shape, stride) if n > 1 and s), reverse=True)
            for shape, stride, size in ((shape_a, stride_a, size_a), (shape_b, stride_b, size_b))]
    return _meet(*dims, size_a, size_b, shift)


def _span(t: torch.Tensor) -> tuple[int, int]:
    """The addresses of a tensor's first byte and of the one behind its last."""
    at = t.data_ptr()
    return at, at + (t.nbytes if t.is_contiguous() else
                     _extent(t.shape, t.stride(), t.element_size()))


def _same(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two tensors are the same elements in the same order."""
    return (a is b or (a.data_ptr() == b.data_ptr() and a.dtype == b.dtype
                       and _strides(a) == _strides(b)))


def _check_apart(name: str, written: torch.Tensor, names: str, *read) -> None:
    """Refuse a tensor to write that may share bytes with one that is read (None
    apart).  Columns of one buffer beside each other share none, though their
    address ranges interleave."""
    first, end = _span(written)
    for i, t in enumerate(read):
        if t is None:
            continue
        at, behind = _span(t)
        if (first < behind and at < end and first < end and at < behind and
                _layouts_meet(written.shape, written.stride(), written.element_size(), t.shape,
                              t.stride(), t.element_size(), at - first)):
            raise SchemeError(f"{name} shares storage with {names.split()[i]}")


def _dtype_code(t: torch.Tensor, name: str) -> int:
    code = DTYPES.get(t.dtype)
    if code is None:
        raise SchemeError(f"{name} must be float32, bfloat16 or float16, got {t.dtype}")
    return code


def _rotary_heads(name: str, x, y, b: int, s: int, d: int, dtype) -> bytes:
    """``mr_rotary_heads`` of the heads ``x``, turned into ``y`` (of x's shape)."""
    bx, px, heads, dx = x.shape
    if bx != b or px != s or dx != d or x.dtype != dtype or heads == 0:
        raise SchemeError(f"{name} is {tuple(x.shape)} {x.dtype}, expected ({b}, {s}, at least one "
                          f"head, {d}) {dtype}")
    xb, xs, xh, xd = x.stride()
    yb, ys, yh, yd = y.stride()
    if (xd != 1 or yd != 1) and d > 1:
        raise SchemeError(f"{name}'s last dimension must be contiguous")
    return pack_rotary_heads(x.data_ptr(), y.data_ptr(), xb, xs, xh, yb, ys, yh, heads)


def _rotary(q, k, cos, sin, positions, layout, out, transposed):
    inter = _interleaved(layout)
    if q.dim() != 4 or (k is not None and k.dim() != 4):
        raise SchemeError("q and k are (batch, positions, heads, head dim)")
    b, s, _, d = q.shape
    dtype = q.dtype
    given = ()
    if out is None:
        out = (torch.empty_like(q), None if k is None else torch.empty_like(k))
    else:
        given = out
        for x, y in ((q, out[0]), (k, out[1])):
            if (x is None) != (y is None):
                raise SchemeError("out is a (q, k) pair with k None exactly where k is")
            if x is not None and (y.shape != x.shape or y.dtype != dtype):
                raise SchemeError(f"an output is {tuple(y.shape)} {y.dtype}, expected "
                                  f"{tuple(x.shape)} {dtype}")
            if x is not None and 0 in _strides(y):
                raise SchemeError(f"an output's elements share storage, strides {y.stride()}")
            if x is not None and y.data_ptr() == x.data_ptr() and _strides(y) != _strides(x):
                raise SchemeError("an output in its input's storage must have its strides")
    yq, yk = out
    dev = _device_of("q k cos sin positions out_q out_k", q, k, cos, sin, positions, *given)
    code = _dtype_code(q, "q")
    if cos.dim() != 2 or cos.shape != sin.shape:
        raise SchemeError(f"cos and sin are (positions, rotated columns / 2) tables, got "
                          f"{tuple(cos.shape)} and {tuple(sin.shape)}")
    rows, half = cos.shape
    if not 1 <= half <= d // 2 or d > 1024:
        raise SchemeError(f"tables of {half} pairs do not fit head dim {d} (at most 1024)")
    pos_ptr, pos64, pos_stride = None, 0, 0
    if positions is not None:
        pos64 = positions.dtype == torch.int64
        if not pos64 and positions.dtype != torch.int32:
            raise SchemeError(f"positions must be int64 or int32, got {positions.dtype}")
        shape = tuple(positions.shape)
        if shape == (b, s):
            pos_stride = s
        elif shape != (s,):
            raise SchemeError(f"positions must be ({s},) or ({b}, {s}), got {shape}")
        if not positions.is_contiguous():
            raise SchemeError("positions must be contiguous")
        pos_ptr = positions.data_ptr()
    elif s > rows:
        raise SchemeError(f"{s} positions but tables of {rows} rows")
    hq = _rotary_heads("q", q, yq, b, s, d, dtype)
    hk = None if k is None else _rotary_heads("k", k, yk, b, s, d, dtype)
    if given and b * s:
        # in place, each output is exactly its own input
        q_in, k_in = _same(yq, q), k is not None and _same(yk, k)
        _check_apart("out's q", yq, "q k cos sin positions", None if q_in else q, k, cos, sin,
                     positions)
        if k is not None:
            _check_apart("out's k", yk, "k q cos sin positions out's-q", None if k_in else k,
                         None if q_in and k_in else q, cos, sin, positions, None if q_in else yq)
    if b * s:
        _launch("mr_rotary", dev, hq, hk,
                _ptr(cos, torch.float32, "cos"), _ptr(sin, torch.float32, "sin"), rows, pos_ptr,
                pos64, pos_stride, b, s, d, 2 * half, inter, transposed, code)
    return out


def rotary(q, k, cos, sin, *, positions=None, layout: str = "half", out=None):
    """K10: rotary positions on ``q`` (B, S, Hq, D) and ``k`` (B, S, Hkv, D) or None.

    float32, bfloat16 or float16 (computed in float32, rounded once); any
    strides with contiguous columns, so views of a fused projection or of
    (B, H, S, D) storage need no copy.  ``cos`` / ``sin``: float32 (rows,
    r / 2) tables as :func:`mround_b200.pipeline.block.rope_tables` makes them;
    the head's first r columns turn, the rest are copied.  ``layout``: pairs
    (j, j + r/2) for "half", (2j, 2j + 1) for "interleaved".  ``positions``:
    int32 or int64 (S,) or (B, S) table rows, 0..S-1 by default; a position
    outside the tables gives NaN.  ``out``: a (q, k) pair of tensors to write,
    which may be ``q`` and ``k`` themselves, and share no other storage with what
    is read.  Returns (q, k) turned."""
    return _rotary(q, k, cos, sin, positions, layout, out, 0)


def rotary_bwd(dq, dk, cos, sin, *, positions=None, layout: str = "half", out=None):
    """Gradients of :func:`rotary`'s inputs from those of its outputs (the
    transposed rotation; same arguments)."""
    return _rotary(dq, dk, cos, sin, positions, layout, out, 1)


MAX_TOPK = 256


def _logit_rows(logits):
    """(rows, columns, row stride) of a 2-D tensor with contiguous columns."""
    if logits.dim() != 2:
        raise SchemeError(f"logits are (rows, vocabulary), got shape {tuple(logits.shape)}")
    rows, n = logits.shape
    ld, inner = logits.stride()
    if n == 0 or (n > 1 and inner != 1) or n > 0x7FFFFFFF:
        raise SchemeError("the logits' columns must be contiguous, at least one")
    if rows <= 1:
        ld = n
    if ld < n:
        raise SchemeError("the logits' rows overlap")
    return rows, n, ld


def topk_logits(logits, k: int):
    """K11: the ``k`` largest logits of each row and their columns, in descending
    order with equal values by lowest column (NaN counts as the largest).

    ``logits``: (rows, vocabulary) float32, bfloat16 or float16, contiguous
    columns.  1 <= k <= min(vocabulary, 256).  Returns float32 values and int64
    columns, (rows, k) each -- what :func:`distill_topk` takes."""
    dev = _device_of("logits", logits)
    rows, n, ld = _logit_rows(logits)
    code = _dtype_code(logits, "logits")
    if not 1 <= k <= min(n, MAX_TOPK):
        raise SchemeError(f"k must be 1 to {min(n, MAX_TOPK)}, got {k}")
    values = logits.new_empty((rows, k), dtype=torch.float32)
    index = logits.new_empty((rows, k), dtype=torch.int64)
    if rows:
        _launch("mr_topk_logits", dev, logits.data_ptr(), rows, n, ld, k, code, values.data_ptr(),
                index.data_ptr())
    return values, index


def _distill(logits, t_logits, t_index, temperature, weight, loss, grad, pair, ldg):
    dev = _device_of("logits t_logits t_index weight out", logits, t_logits, t_index, weight, grad)
    rows, n, ld = _logit_rows(logits)
    code = _dtype_code(logits, "logits")
    shape = tuple(t_logits.shape)
    if len(shape) != 2 or shape[0] != rows or tuple(t_index.shape) != shape:
        raise SchemeError(f"t_logits and t_index are ({rows}, k), got {shape} and "
                          f"{tuple(t_index.shape)}")
    k = shape[1]
    if not 1 <= k <= MAX_TOPK:
        raise SchemeError(f"1 to {MAX_TOPK} teacher logits per row, got {k}")
    if not 1e-3 <= float(temperature) <= 1e3:
        raise SchemeError(f"temperature must be 0.001 to 1000, got {temperature}")
    args = (_ptr(t_logits, torch.float32, "t_logits"), _ptr(t_index, torch.int64, "t_index"), k,
            float(temperature), _ptr(weight, torch.float32, "weight", rows))
    if rows:
        _launch("mr_distill_topk", dev, logits.data_ptr(), rows, n, ld, code, *args,
                None if loss is None else loss.data_ptr(),
                None if grad is None else grad.data_ptr(),
                None if pair[0] is None else pair[0].data_ptr(),
                None if pair[1] is None else pair[1].data_ptr(), ldg)


def distill_topk(logits, t_logits, t_index, *, temperature: float = 1.0, weight=None):
    """K12, the loss alone: per row, ``weight * T^2 * KL(p || q)`` with
    ``p = softmax(t_logits / T)`` over the teacher's kept logits and
    ``q = softmax(logits / T)`` over the whole vocabulary.

    ``logits``: (rows, vocabulary) float32, bfloat16 or float16, contiguous
    columns.  ``t_logits`` float32 and ``t_index`` int64, (rows, k), k <= 256: a
    negative column is an absent entry, a repeated one counts as often as it
    occurs, one beyond the vocabulary makes its row NaN.  ``weight``: float32
    (rows,); a row of weight 0, or without an entry, gives 0 whatever it holds.
    Returns float32 (rows,)."""
    loss = logits.new_empty(logits.shape[:1], dtype=torch.float32)
    _distill(logits, t_logits, t_index, temperature, weight, loss, None, (None, None), 0)
    return loss


def distill_topk_grad(logits, t_logits, t_index, *, temperature: float = 1.0, weight=None,
                      out=None, split: bool = False):
    """K12, the loss and its gradient in one launch: arguments of
    :func:`distill_topk`; the gradient is that of the losses' sum with respect
    to ``logits`` (an upstream gradient per row goes into ``weight``).

    The gradient has the logits' type, in ``out`` when given (contiguous
    columns; ``logits`` itself may be given), or with ``split`` is the bf16
    (hi, lo) pair that :func:`gemm` takes.  Returns (loss, gradient)."""
    loss = logits.new_empty(logits.shape[:1], dtype=torch.float32)
    if split:
        if out is not None:
            raise SchemeError("a split gradient is allocated by the call")
        pair = _pair(logits.shape, logits.device)
        _distill(logits, t_logits, t_index, temperature, weight, loss, None, pair,
                 logits.shape[-1])
        return loss, pair
    if out is None:
        out = torch.empty_like(logits, memory_format=torch.contiguous_format)
        ldg = logits.shape[-1]
    else:
        if out.shape != logits.shape or out.dtype != logits.dtype:
            raise SchemeError(f"out must be {tuple(logits.shape)} {logits.dtype}")
        _, _, ldg = _logit_rows(out)
        if logits.shape[0]:
            _check_apart("out", out, "logits t_logits t_index weight",
                         None if _same(out, logits) else logits, t_logits, t_index, weight)
    _distill(logits, t_logits, t_index, temperature, weight, loss, out, (None, None), ldg)
    return loss, out


ACTIVATIONS = {"none": 0, "silu": 1, "gelu": 2, "gelu_tanh": 3, "swiglu": 4}
LINEAR_SPLITS = (1, 2, 4, 8)


def _act_code(act: str) -> int:
    code = ACTIVATIONS.get(act)
    if code is None:
        raise SchemeError(f"act must be one of {', '.join(ACTIVATIONS)}, got {act!r}")
    return code


def _parts(t, name: str):
    """(hi, lo or None) of a bf16 operand given as a tensor or as a pair."""
    if isinstance(t, torch.Tensor):
        if t.dim() == 2 and t.dtype == torch.bfloat16:
            return t, None
    elif len(t) == 2 and all(p.dim() == 2 and p.dtype == torch.bfloat16 for p in t):
        hi, lo = t
        if lo.shape != hi.shape or lo.stride() != hi.stride():
            raise SchemeError(f"{name}'s parts must have one shape and layout")
        return hi, lo
    raise SchemeError(f"{name} must be a 2-D bfloat16 tensor or a (hi, lo) pair of them")


def _operand(parts, name: str, kmajor: bool):
    """``mr_linear_operand`` of parts whose columns (K-major) or rows are k."""
    hi, lo = parts
    rows, cols = hi.shape
    ld, inner = hi.stride()
    if rows == 1:
        ld = -(-cols // 8) * 8
    if (inner != 1 and cols > 1) or ld < cols or ld % 8:
        raise SchemeError(f"{name} needs contiguous columns and a row stride that is a multiple "
                          f"of 8, got strides {hi.stride()}")
    return pack_linear_operand(hi.data_ptr(), 0 if lo is None else lo.data_ptr(), ld, kmajor)


def _row_stride(t, rows: int, cols: int, dtypes, name: str) -> int:
    ld, inner = t.stride() if t.dim() == 2 else (0, 0)
    if t.dtype not in dtypes or tuple(t.shape) != (rows, cols):
        raise SchemeError(f"{name} must be ({rows}, {cols}) of {dtypes}, got {tuple(t.shape)} "
                          f"{t.dtype}")
    if rows == 1:
        ld = cols
    if (inner != 1 and cols > 1) or ld < cols:
        raise SchemeError(f"{name} needs contiguous columns in rows that do not overlap")
    return ld


_LINEAR_OUT = (torch.float32, torch.bfloat16)


def _linear_call(dev, x, w, toks, feats, k, act, bias, residual, ldr, out, lo, t32, ldo, pre, ldp,
                 splits):
    timing = GEMM_EVENTS is not None
    if timing:
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
    _launch("mr_linear", dev, x, w, toks, feats, k, act,
            None if bias is None else bias.data_ptr(),
            None if residual is None else residual.data_ptr(),
            0 if residual is None else DTYPES[residual.dtype], ldr, out.data_ptr(),
            DTYPES[out.dtype], None if lo is None else lo.data_ptr(),
            None if t32 is None else t32.data_ptr(), ldo, None if pre is None else pre.data_ptr(),
            ldp, splits)
    if timing:
        end.record()
        products = 1 + sum(unpack_linear_operand(p)[1] != 0 for p in (x, w))
        GEMM_EVENTS.append((start, end, 2.0 * toks * feats * (2 if act == 4 else 1) * k, products))


def linear(x, w, *, bias=None, act: str = "none", residual=None, out=None, dtype=None,
           split: bool = False, t32=None, pre=None, splits: int | None = None):
    """K13: ``act(x @ w.T + bias) + residual`` in one kernel, float32 accumulation.

    ``x`` (T, k) and ``w`` (features, k): bfloat16 tensors with contiguous
    columns and a row stride that is a multiple of 8, or (hi, lo) pairs of them
    as :func:`split_bf16` makes (``w`` a pair only with ``x`` a pair).
    ``act``: "none", "silu", "gelu" (erf), "gelu_tanh" or "swiglu", where ``w``
    holds [gate | up] rows and the output has half as many columns.  ``bias``
    float32 (features,); ``residual`` float32 or bfloat16 of the output's shape.

    The output is ``dtype`` (float32 or bfloat16; by default bfloat16, float32
    when ``x`` is a pair), in ``out`` when given (which may be ``residual``),
    or with ``split`` a bf16 (hi, lo) pair.  ``t32``: a contiguous float32
    tensor that also receives the output rounded to tf32.  ``pre``: a float32
    (T, features) tensor that receives ``x @ w.T + bias``, for
    :func:`linear_bwd`.  ``out`` or ``t32`` may be ``residual``; what is written
    shares no other storage with what is read, or with one another.

    ``splits``: how many CTAs share the k of one output tile (1, 2, 4 or 8),
    chosen by size when None.  It fixes the order of the sums: with 1 a token's
    result is the same whatever other tokens are in the call.

    A wait inside the kernel that gives up leaves the output unwritten;
    :func:`check_products` raises for it."""
    code = _act_code(act)
    xp, wp = _parts(x, "x"), _parts(w, "w")
    dev = _device_of("x x_lo w w_lo bias residual out t32 pre", *xp, *wp, bias, residual, out, t32,
                     pre)
    toks, k = xp[0].shape
    rows = wp[0].shape[0]
    if wp[0].shape[1] != k or k == 0 or rows == 0:
        raise SchemeError(f"x {tuple(xp[0].shape)} and w {tuple(wp[0].shape)} do not share a k")
    if wp[1] is not None and xp[1] is None:
        raise SchemeError("w is a (hi, lo) pair but x is not")
    if act == "swiglu" and rows % 2:
        raise SchemeError(f"a swiglu weight has as many gate as up rows, got {rows} rows")
    if splits is not None and splits not in LINEAR_SPLITS:
        raise SchemeError(f"splits must be one of {LINEAR_SPLITS}, got {splits}")
    feats = rows // 2 if act == "swiglu" else rows
    lo, ldo = None, feats
    given = out is not None
    if split:
        if out is not None or dtype is not None:
            raise SchemeError("a split output is allocated by the call")
        out, lo = _pair((toks, feats), xp[0].device)
    elif out is None:
        dtype = dtype or (torch.bfloat16 if xp[1] is None else torch.float32)
        if dtype not in _LINEAR_OUT:
            raise SchemeError(f"dtype must be float32 or bfloat16, got {dtype}")
        out = xp[0].new_empty((toks, feats), dtype=dtype)
    else:
        if dtype is not None and out.dtype != dtype:
            raise SchemeError(f"out is {out.dtype}, not {dtype}")
        ldo = _row_stride(out, toks, feats, _LINEAR_OUT, "out")
    if t32 is not None:
        if _row_stride(t32, toks, feats, (torch.float32,), "t32") != ldo:
            raise SchemeError("t32 must have the output's row stride")
    ldr = 0 if residual is None else _row_stride(residual, toks, feats, _LINEAR_OUT, "residual")
    ldp = 0 if pre is None else _row_stride(pre, toks, rows, (torch.float32,), "pre")
    if bias is not None:
        _ptr(bias, torch.float32, "bias", rows)
    if toks:
        for name, written in (("out", out if given else None), ("t32", t32), ("pre", pre)):
            if written is not None:
                # of what is read, out or t32 may be the residual
                _check_apart(name, written, "x x_lo w w_lo bias residual out t32", *xp, *wp, bias,
                             None if residual is None or (written is not pre
                                                          and _same(written, residual))
                             else residual,
                             out if given and written is not out else None,
                             t32 if written is pre else None)
        _linear_call(dev, _operand(xp, "x", True), _operand(wp, "w", True), toks, feats, k, code,
                     bias, residual, ldr, out, lo, t32, ldo, pre, ldp, splits or 0)
    return (out, lo) if split else out


def linear_bwd(dy, x, w, *, act: str = "none", pre=None, bias_grad: bool = False, dtype=None,
               splits: int | None = None):
    """Gradients of :func:`linear`: ``(dx, dw, dbias or None)`` from ``dy``
    (float32 or bfloat16), the operands and the ``pre`` that the forward wrote
    (not needed where ``act`` is "none").  The residual's gradient is ``dy``.

    ``dx = dz @ w`` and ``dw = dz.T @ x``, ``dz = dy * act'(pre)``, are ``dtype``
    (float32 or bfloat16; by default as the output of :func:`linear`), the bias
    gradient float32.  ``dz`` is formed in float32 and carried into both products
    as a bf16 pair (2^-16 of it is lost), whatever the gradients' type; a
    bfloat16 ``dy`` without an activation is taken as it is."""
    code = _act_code(act)
    xp, wp = _parts(x, "x"), _parts(w, "w")
    dev = _device_of("dy x x_lo w w_lo pre", dy, *xp, *wp, pre)
    empty = dy.new_empty
    toks, k = xp[0].shape
    rows = wp[0].shape[0]
    if wp[0].shape[1] != k or k == 0 or rows == 0 or (act == "swiglu" and rows % 2):
        raise SchemeError(f"x {tuple(xp[0].shape)} and w {tuple(wp[0].shape)} are not the operands "
                          "of a linear")
    if wp[1] is not None and xp[1] is None:
        raise SchemeError("w is a (hi, lo) pair but x is not")
    feats = rows // 2 if act == "swiglu" else rows
    ldy = _row_stride(dy, toks, feats, _LINEAR_OUT, "dy")
    if pre is None and act != "none":
        raise SchemeError(f"the gradient of {act} needs the pre-activation")
    ldp = 0 if pre is None else _row_stride(pre, toks, rows, (torch.float32,), "pre")
    if splits is not None and splits not in LINEAR_SPLITS:
        raise SchemeError(f"splits must be one of {LINEAR_SPLITS}, got {splits}")
    out_dtype = dtype or (torch.bfloat16 if xp[1] is None else torch.float32)
    if out_dtype not in _LINEAR_OUT:
        raise SchemeError(f"dtype must be float32 or bfloat16, got {out_dtype}")
    x_op, w_op = _operand(xp, "x", False), _operand(wp, "w", False)
    dx = empty((toks, k), dtype=out_dtype)
    dw = empty((rows, k), dtype=out_dtype)
    db = empty(rows, dtype=torch.float32) if bias_grad else None
    if toks == 0:
        dw.zero_()
        if db is not None:
            db.zero_()
        return dx, dw, db
    # without an activation a bf16 dy is dz
    as_is = (act == "none" and dy.dtype == torch.bfloat16 and xp[1] is None and
             (toks == 1 or ldy % 8 == 0) and dy.data_ptr() % 16 == 0)
    hi, lo, ldz = None, None, 0
    if not as_is:
        ldz = -(-rows // 8) * 8
        hi = empty((toks, ldz), dtype=torch.bfloat16)
        # one bf16 alone would halve both products' work (2047 x 11008 by 2048, tanh
        # GELU: 176 us instead of 330), but err by 1.41 times the rounding of a bf16
        # gradient itself
        lo = torch.empty_like(hi)
    scratch = None
    if bias_grad:
        nbytes = int(lib().mr_act_grad_workspace_bytes(toks, feats, code))
        if nbytes:
            scratch = empty(nbytes, dtype=torch.uint8)
    if bias_grad or not as_is:
        z = None if act == "none" else pre.data_ptr()
        _launch("mr_act_grad", dev, dy.data_ptr(), DTYPES[dy.dtype], ldy, z, ldp, toks, feats, code,
                None if hi is None else hi.data_ptr(), None if lo is None else lo.data_ptr(), ldz,
                None if db is None else db.data_ptr(),
                None if scratch is None else scratch.data_ptr())
    n = splits or 0
    if as_is:
        hi, ldz = dy, ldy if toks > 1 else -(-rows // 8) * 8
    dz = (hi.data_ptr(), 0 if lo is None else lo.data_ptr(), ldz)
    _linear_call(dev, pack_linear_operand(*dz, True), w_op, toks, k, rows, 0, None, None, 0, dx,
                 None, None, k, None, 0, n)
    _linear_call(dev, pack_linear_operand(*dz, False), x_op, rows, k, toks, 0, None, None, 0, dw,
                 None, None, k, None, 0, n)
    return dx, dw, db
