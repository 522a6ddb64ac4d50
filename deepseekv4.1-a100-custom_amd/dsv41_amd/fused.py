"""Fused element-wise ops of the expert path with the call surface of the reference's dsv41/fused.py:
fake_quant_fp8 (fused.py:47-83) and swiglu_quant (fused.py:283-345), on HIP kernels; and the residual + RMSNorm whose output is a
product's FP8 or FP4 operand (add_rmsnorm_quant)."""
from __future__ import annotations

import torch

from . import _lib
from .quant import _TYPE, _rows16, attach_codes, fake_quant_fp8 as _fq8


def fake_quant_fp8(x: torch.Tensor, block: int = 32) -> torch.Tensor:
    """Per-32 FP8 fake quantisation in x's dtype (fused.py:82-83; identical to quant.fake_quant_fp8)."""
    return _fq8(x, block)


def swiglu_quant(gu: torch.Tensor, weights: torch.Tensor | None, inter: int, limit: float, permute: bool = False) -> torch.Tensor:
    """SwiGLU of each row's gate half (columns [0, inter)) and up half (columns [inter, 2 inter)) of gu (fp32 or bf16),
    times the row's routing weight when `weights` is given, rounded to bf16 and then to FP8 per 32 columns; returns the
    bf16 [rows, inter] values, h = fq8(bf16(w * silu(min(g, L)) * clamp(u, +-L))) (fused.py:334-345). `permute` stores
    each 8 columns in the 8-k permuted order.

    The same launch also writes the FP8 codes and E8M0 bytes those values are made from and records them on the
    result (quant.attach_codes): the FP4 GEMM surfaces (fp4_gemm_tc, fp4_gemv_pairs, grouped_fp4_gemm) take them as
    their activation operand instead of quantising the result again (a launch less per call; the values are
    identical, so the GEMM result is too)."""
    dev = _lib.require_cuda(gu, weights)
    if gu.dtype not in (torch.float32, torch.bfloat16):
        gu = gu.float()
    if gu.stride(-1) != 1:
        gu = gu.contiguous()
    rows = gu.shape[0]
    y = torch.empty(rows, inter, device=dev, dtype=torch.bfloat16)
    codes = torch.empty(rows, inter, device=dev, dtype=torch.uint8)
    scales = torch.empty(rows, inter // 32, device=dev, dtype=torch.uint8)
    w = None if weights is None else weights.reshape(-1).to(torch.float32).contiguous()
    _lib.call("dsv41_swiglu_quant", _lib.ptr(gu), 1 if gu.dtype == torch.bfloat16 else 0, gu.stride(0), _lib.ptr(w), rows, inter,
              float(limit), _lib.ptr(codes), _lib.ptr(scales), _lib.ptr(y),
              1 if permute else 0, _lib.stream(dev))
    return attach_codes(y, codes, scales, permute)


def swiglu_quant_codes(gu: torch.Tensor, weights: torch.Tensor | None, inter: int, limit: float, codes: torch.Tensor | None = None,
                       scales: torch.Tensor | None = None):
    """The same SwiGLU epilogue returning the down projection's MFMA operand directly:
    (E4M3 codes uint8 [rows, inter], E8M0 bytes uint8 [rows, inter/32])."""
    dev = _lib.require_cuda(gu, weights)
    rows = gu.shape[0]
    if codes is None:
        codes = torch.empty(rows, inter, device=dev, dtype=torch.uint8)
    if scales is None:
        scales = torch.empty(rows, inter // 32, device=dev, dtype=torch.uint8)
    w = None if weights is None else weights.reshape(-1)
    _lib.call("dsv41_swiglu_quant", _lib.ptr(gu), 1 if gu.dtype == torch.bfloat16 else 0, gu.stride(0), _lib.ptr(w), rows, inter,
              float(limit), _lib.ptr(codes), _lib.ptr(scales),
              None, 0, _lib.stream(dev))
    return codes, scales


NORM_MAX = 32768   # longest row of add_rmsnorm_quant (csrc/mx.h)
_BITS = {"fp8": 8, "fp4": 4}


def _apart(out: torch.Tensor, t: torch.Tensor, same: bool = True) -> bool:
    """Whether the rows of out share no byte with those of t, or are the same rows exactly where `same` allows it (matrices of one type, as
    the kernel walks them)."""
    es, n = out.element_size(), out.shape[1] * out.element_size()
    so, st = _lib.row_stride(out) * es, _lib.row_stride(t) * es
    a, b = out.data_ptr(), t.data_ptr()
    if a == b and so == st and out.shape == t.shape:
        return same
    if a + (out.shape[0] - 1) * so + n <= b or b + (t.shape[0] - 1) * st + n <= a:
        return True
    return so == st and n <= (a - b) % so <= so - n   # other columns of the same wider rows


def add_rmsnorm_quant(x: torch.Tensor, residual: torch.Tensor | None, w: torch.Tensor, eps: float, fmt: str = "fp8", y: bool = False,
                      out: torch.Tensor | None = None):
    """Residual addition, RMSNorm and quantisation of rows in one launch: r = x + residual, rounded to x's dtype (the residual stream that
    the next layer reads; x itself where residual is None); v = r / sqrt(mean(r^2) + eps) * w in fp32; v per 32 values as `fmt` "fp8"
    (E4M3, the rounding of quant_fp8_e8m0) or "fp4" (E2M1, quant_fp4), with no rounding in between.
    x, residual [..., K], w [K]: bf16, fp16 or fp32, all of one dtype; K % 32 == 0, K <= 32768. Returns (codes uint8 [..., K] or [..., K / 2],
    E8M0 bytes uint8 [..., K / 32], r), the first two being the operand of w4.linear_fp4 (FP8: of the expert GEMMs too); with `y` also
    v rounded to x's dtype (a router's input). `out` receives r: a tensor like x, which may be x or residual itself; its version counter moves
    as with torch's own in-place operations.
    A group with a NaN or an infinity in it gets the byte 255 and codes 0x7F (FP8) or 0 (FP4), NaN in every product; a row whose mean
    square is NaN or overflows fp32 is such a row or rounds to zeros, as the formula has it.
    Inference only: inputs (and an out) with a gradient to follow (reverse or forward mode) are refused, and so is a tracer."""
    bits, dt, shape = _BITS.get(fmt), x.dtype, x.shape
    if bits is None:
        raise ValueError(f"fmt is 'fp8' or 'fp4', got {fmt!r}")
    if dt not in _TYPE or w.dtype != dt or (residual is not None and residual.dtype != dt) or (out is not None and out.dtype != dt):
        raise TypeError("add_rmsnorm_quant takes x, residual, w and out of one dtype (bf16, fp16 or fp32), got "
                        + ", ".join(str(t.dtype) for t in (x, residual, w, out) if t is not None))
    K = shape[-1] if shape else 0
    if K == 0 or K % 32 or K > NORM_MAX or w.shape != (K,):
        raise ValueError(f"add_rmsnorm_quant: rows of a multiple of 32, at most {NORM_MAX}, and w of a row's length; got {tuple(shape)} and {tuple(w.shape)}")
    if not eps >= 0:
        raise ValueError(f"eps is not negative, got {eps}")
    if (residual is not None and residual.shape != shape) or (out is not None and out.shape != shape):
        raise ValueError(f"residual and out are shaped like x {tuple(shape)}, got {[tuple(t.shape) for t in (residual, out) if t is not None]}")
    if out is not None and residual is None:
        raise ValueError("without a residual r is x itself: there is nothing to write into out")
    _lib.inference_only("add_rmsnorm_quant", x, residual, w, out)
    dev = x.device
    if not x.is_cuda or w.device != dev or (residual is not None and residual.device != dev) or (out is not None and out.device != dev):
        _lib.require_cuda(x, residual, w, out)
    lead, rows, given = shape[:-1], x.numel() // K, out is not None
    px, pw, pr, po, sx, sr, so = x.data_ptr(), w.data_ptr(), None, None, K, K, K
    if residual is not None and out is None and x.is_contiguous() and residual.is_contiguous() and w.is_contiguous() and not (
            (px | pw | (pr := residual.data_ptr())) & 15):
        out = torch.empty_like(x)
        po = out.data_ptr()
    else:
        keep, px, pw, pr, po, sx, sr, so, out = _norm_rows(x, residual, w, out, K)   # `keep`: copies live until the launch
    codes = torch.empty((*lead, K * bits // 8), dtype=torch.uint8, device=dev)
    scales = torch.empty((*lead, K // 32), dtype=torch.uint8, device=dev)
    yt = torch.empty(shape, dtype=dt, device=dev) if y else None
    if rows:
        _lib.launch(dev, "dsv41_add_rmsnorm_mx", px, sx, pr, sr, pw, eps, _TYPE[dt], rows, K, bits, po, so, yt.data_ptr() if y else None,
                    codes.data_ptr(), scales.data_ptr())
        if given:
            torch.autograd.graph.increment_version(out)   # the launch wrote past torch: autograd and an FP8 record on out have to see it
    r = x if residual is None else out
    return (codes, scales, r, yt) if y else (codes, scales, r)


def _norm_rows(x, residual, w, out, K: int):
    """add_rmsnorm_quant's rows where they are not all plain: (tensors to keep, pointers of x, w, residual, out, their row strides, out)."""
    es = x.element_size()
    x2 = _rows16(x.reshape(-1, K), es)
    if w.stride(0) != 1 or w.data_ptr() % 16:
        w = w.clone(memory_format=torch.contiguous_format)
    if residual is None:
        return (x2, w), x2.data_ptr(), w.data_ptr(), None, None, _lib.row_stride(x2), K, K, None
    r2 = _rows16(residual.reshape(-1, K), es)
    if out is None:
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        o2 = out.view(-1, K)
    else:
        try:
            o2 = out.view(-1, K)
        except RuntimeError:
            o2 = None
        if o2 is None or (o2.shape[0] and _rows16(o2, es) is not o2):
            raise ValueError("out needs rows of 16-byte pieces in one regular layout (unit stride within a row, aligned rows)")
        # each value of x and the residual is read by the thread that writes r there; w is read by every row, after r is written
        if not (_apart(o2, x2) and _apart(o2, r2) and _apart(o2, w.view(1, K), same=False)):
            raise ValueError("out overlaps an input without being it")
    return ((x2, r2, w), x2.data_ptr(), w.data_ptr(), r2.data_ptr(), o2.data_ptr(), _lib.row_stride(x2), _lib.row_stride(r2), _lib.row_stride(o2), out)
