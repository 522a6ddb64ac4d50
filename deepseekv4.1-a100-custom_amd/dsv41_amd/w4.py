"""Dense weights kept as FP4 on the device (E2M1 codes, one E8M0 byte per 32 values along k: the experts' format), and their product
with activations in FP4 or FP8. Beside w8 (FP8 dense weights, half of bf16's bytes) these take a quarter.

The product is y = x . w^T with x rounded per 32 values along k to E2M1 (quant.quant_fp4) or E4M3 (quant.quant_fp8_e8m0) and both
operands' E8M0 scales applied inside the block-scaled MFMA; sums are fp32 and y is rounded once. FP4 activations run at twice the
matrix rate of FP8 ones. Activations that are codes already (fused.add_rmsnorm_quant, swiglu_quant's record) are taken as they are.

Stored order of W4: tiles of 16 rows x 128 k, the k blocks of 32 in the order in which one MFMA step takes them (csrc/mx.h), zero
padded to whole tiles, so any N and any K that is a multiple of 32 runs.
"""
from __future__ import annotations

import torch
import torch.nn.functional as F

from . import _lib, hipkern
from .quant import _TYPE, _rows16, attached_codes, dequant_fp4, quant_fp4


class W4:
    """FP4 dense weights in the stored order: `w4` uint8 [N / 16, K / 128, 1024] and `s4` uint8 [N / 16, K / 128, 64] (both rounded up),
    `shape` (N, K)."""
    __slots__ = ("w4", "s4", "shape", "device")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor):
        """codes: uint8 [N, K / 2], two E2M1 codes per byte, the even k in the low nibble; scales: E8M0 bytes [N, K / 32], as quant_fp4
        and a checkpoint give them (any one-byte type, read as bytes). K % 32 == 0. Laid out once, here."""
        if scales.element_size() != 1:   # codes in wider words either hold the same bytes or do not fit the scales
            raise TypeError(f"W4: scales are E8M0 bytes, got {scales.dtype}")
        codes, scales = codes.view(torch.uint8), scales.view(torch.uint8)
        if codes.dim() != 2 or scales.dim() != 2 or codes.shape[1] % 16 or codes.shape[1] == 0 or codes.shape[0] == 0:
            raise ValueError(f"W4: codes [N, K / 2] with K % 32 == 0 and scales [N, K / 32], got {tuple(codes.shape)} and {tuple(scales.shape)}")
        N, K = codes.shape[0], codes.shape[1] * 2
        if tuple(scales.shape) != (N, K // 32):
            raise ValueError(f"W4: scales {tuple(scales.shape)} do not fit codes of {N} x {K}, which need {(N, K // 32)}")
        if codes.device != scales.device:
            raise RuntimeError(f"tensors on different devices: {codes.device} and {scales.device}")
        nb, kb = -(-N // 16), -(-K // 128)
        if nb * 16 != N or kb * 128 != K:
            codes = F.pad(codes, (0, kb * 64 - K // 2, 0, nb * 16 - N))
            scales = F.pad(scales, (0, kb * 4 - K // 32, 0, nb * 16 - N))
        # block b = 2 g + s of a tile: codes [rows, tiles, g, s, 16 B] -> [tiles, s, g, rows, 16 B], scales [rows, tiles, g, s] -> [tiles, g, rows, s]
        self.w4 = codes.reshape(nb, 16, kb, 2, 2, 16).permute(0, 2, 4, 3, 1, 5).reshape(nb, kb, 1024).contiguous()
        self.s4 = scales.reshape(nb, 16, kb, 2, 2).permute(0, 2, 3, 1, 4).reshape(nb, kb, 64).contiguous()
        self.shape = (N, K)
        self.device = codes.device

    @classmethod
    def from_dense(cls, w: torch.Tensor) -> "W4":
        """From dense weights [N, K] (bf16, fp16 or fp32, on the GPU), rounded by quant_fp4."""
        if w.dim() != 2:
            raise ValueError(f"W4.from_dense takes a matrix, got {tuple(w.shape)}")
        return cls(*quant_fp4(w.detach()))

    @property
    def dtype(self):
        return torch.bfloat16

    def natural(self):
        """(codes [N, K / 2], scales [N, K / 32]) in row-major order."""
        (N, K), (nb, kb, _) = self.shape, self.w4.shape
        codes = self.w4.view(nb, kb, 2, 2, 16, 16).permute(0, 4, 1, 3, 2, 5).reshape(nb * 16, kb * 64)
        scales = self.s4.view(nb, kb, 2, 16, 2).permute(0, 3, 1, 2, 4).reshape(nb * 16, kb * 4)
        return codes[:N, :K // 2].contiguous(), scales[:N, :K // 32].contiguous()

    def bf16(self) -> torch.Tensor:
        """The dequantised weights, bf16 [N, K]."""
        return dequant_fp4(*self.natural())

    @staticmethod
    def cat(ws: list) -> "W4":
        """One W4 whose rows are the given weights' rows in order. Every part but the last needs a row count that is a multiple of 16:
        a tile never straddles two parts."""
        if not ws or len({w.shape[1] for w in ws}) != 1 or any(w.shape[0] % 16 for w in ws[:-1]):
            raise ValueError(f"W4.cat: equal K and whole 16-row tiles, got {[w.shape for w in ws]}")
        out = W4.__new__(W4)
        out.w4, out.s4 = torch.cat([w.w4 for w in ws]), torch.cat([w.s4 for w in ws])
        out.shape, out.device = (sum(w.shape[0] for w in ws), ws[0].shape[1]), ws[0].device
        return out


def _operand(x, K: int):
    """(codes 2-d, scales 2-d, bits per code, leading shape) of an operand pair for K values per row."""
    if len(x) != 2:
        raise ValueError(f"operand: a pair (codes, scales), got {len(x)} tensors")
    codes, scales = x
    if codes.dtype not in (torch.uint8, torch.float8_e4m3fn) or scales.dtype not in (torch.uint8, torch.float8_e8m0fnu):
        raise TypeError(f"operand: uint8 (or float8) codes and E8M0 scale bytes, got {codes.dtype} and {scales.dtype}")
    if codes.dtype != torch.uint8:
        codes = codes.view(torch.uint8)
    if scales.dtype != torch.uint8:
        scales = scales.view(torch.uint8)
    shape = codes.shape
    lead, n = shape[:-1], shape[-1] if shape else 0
    if n not in (K, K // 2) or scales.shape != (*lead, K // 32):
        raise ValueError(f"operand: codes [..., {K}] (FP8) or [..., {K // 2}] (FP4) and scales [..., {K // 32}] for K = {K}, got "
                         f"{tuple(shape)} and {tuple(scales.shape)}")
    fmt = 8 if n == K else 4
    if len(shape) != 2:
        codes, scales = codes.reshape(-1, n), scales.reshape(-1, K // 32)
    return _rows16(codes, 1, most=1 << 21), _rows16(scales, 1, 1, 1 << 21), fmt, lead


_ACTS = (None, "fp4", "fp8")


def linear_fp4(x, w: W4, act: str | None = None, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """y [..., N] = x . w^T for FP4 weights w (a W4 of N x K), accumulated in fp32 and rounded once to out_dtype (bf16, fp16 or fp32).

    x: bf16, fp16 or fp32 [..., K], rounded per 32 values to `act` = "fp4" (the default) or "fp8" first; out_dtype defaults to x's.
    Or an operand pair (codes, scales) as quant_fp4, quant_fp8_e8m0 and add_rmsnorm_quant give it: [..., K / 2] E2M1 or [..., K] E4M3
    codes with [..., K / 32] E8M0 bytes; out_dtype then defaults to bf16. Any number of rows, none included.
    Sums of FP8 codes carry about 17 bits whatever out_dtype is: the matrix unit adds their products with FP4 codes eight at a time and
    drops what is below 2^-13 of the largest (1.3e-5 of y for normal activations); sums of FP4 codes carry fp32's 24.
    An E8M0 byte 255 (the mark of a group with a NaN or an infinity in it) makes the row's, or the weight row's, outputs NaN.
    Inference only: an x with a gradient to follow (reverse or forward mode) is refused, and so is a tracer."""
    if not isinstance(w, W4):
        raise TypeError(f"linear_fp4 takes W4 weights, got {type(w).__name__}")
    if act not in _ACTS:
        raise ValueError(f"act is 'fp4' or 'fp8', got {act!r}")
    N, K = w.shape
    if isinstance(x, (tuple, list)):
        codes, scales, fmt, lead = _operand(x, K)
        if act is not None and act != f"fp{fmt}":
            raise ValueError(f"the operand holds FP{fmt} codes and act is {act!r}")
        dtype = out_dtype or torch.bfloat16
        if dtype not in _TYPE:
            raise TypeError(f"linear_fp4 gives bf16, fp16 or fp32, got {dtype}")
        _lib.inference_only("linear_fp4")
        if not codes.is_cuda or codes.device != w.device or scales.device != w.device:
            _lib.require_cuda(codes, scales, w.w4)
        y = hipkern.mx_gemm(codes, scales, fmt, w, dtype)
        return y if len(lead) == 1 else y.view(*lead, N)
    shape, dtype = x.shape, out_dtype or x.dtype
    if x.dtype not in _TYPE or dtype not in _TYPE:
        raise TypeError(f"linear_fp4 takes and gives bf16, fp16 or fp32, got {x.dtype} for {dtype}")
    if not shape or shape[-1] != K:
        raise ValueError(f"x {tuple(shape)} does not fit weights of {N} x {K}")
    _lib.inference_only("linear_fp4", x)
    if not x.is_cuda or x.device != w.device:
        _lib.require_cuda(x, w.w4)
    fmt = 8 if act == "fp8" else 4
    if fmt == 8:
        known = attached_codes(x, False)
        if known is not None:
            return linear_fp4(known, w, out_dtype=dtype)
    y = hipkern.mx_linear(_rows16(x if len(shape) == 2 else x.reshape(-1, K), x.element_size(), 16, 1 << 24), fmt, w, dtype)
    return y if len(shape) == 2 else y.view(*shape[:-1], N)
