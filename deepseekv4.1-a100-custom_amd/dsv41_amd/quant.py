"""Numeric formats of the FP4 expert path, with the call surface of the reference's dsv41/quant.py.

- E8M0 scales: one byte b, value 2^(b-127) (quant.py:27-31).
- FP4 expert weights: two E2M1 codes per byte, the even k in the low nibble, and one E8M0 byte for every 32 k of a row
  (quant.py:6, 98-110).
- FP8 activations: per-32 power-of-two scale, E4M3 round-to-nearest-even (quant.py:45-64).

- FP4 quantisation: per-32 power-of-two scale, E2M1 round-to-nearest-even (quant_fp4).

dequant_fp4 / quant_fp4 / fake_quant_fp8 / quant_fp8 run HIP kernels (GPU tensors only). The tiled-layout helpers are
pure layout permutations done with torch views at load time, as in the reference (quant.py:113-139).
"""
from __future__ import annotations

import torch

from . import _lib

FP8_MAX = 448.0
FP4_MAX = 6.0
FP4_TABLE = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0])


def e8m0_to_float(b: torch.Tensor) -> torch.Tensor:
    """E8M0 scale bytes (any 1-byte dtype, e.g. the raw F8_E8M0 checkpoint bytes) -> their values 2^(b - 127) as
    float32 (quant.py:27-31): built from the exponent bits, so byte 0 is the subnormal 2^-127 and 255 is +inf."""
    u = b.view(torch.uint8).to(torch.int32)
    bits = torch.where(u == 0, torch.full_like(u, 0x00400000), u << 23)
    return bits.view(torch.float32)


def dequant_fp4(packed: torch.Tensor, scale: torch.Tensor, block: int = 32, tiled: bool = False) -> torch.Tensor:
    """uint8 [..., N, K/2] + uint8 [..., N, K/32] -> bf16 [..., N, K], bit-exact with quant.dequant_fp4
    (quant.py:106-110). `tiled`: inputs in the tile_fp4 / tile_fp4_scales layout."""
    assert block == 32
    dev = _lib.require_cuda(packed, scale)
    p = packed.contiguous().view(torch.uint8)
    s = scale.contiguous().view(torch.uint8)
    K = p.shape[-1] * 2
    rows = p.numel() // (K // 2)
    assert s.numel() == rows * (K // 32), "scale shape does not match the packed weights"
    out = torch.empty(*p.shape[:-1], K, dtype=torch.bfloat16, device=dev)
    _lib.call("dsv41_dequant_fp4", _lib.ptr(p), _lib.ptr(s), rows, K, 1 if tiled else 0, _lib.ptr(out), _lib.stream(dev))
    return out


_TYPE = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}   # tensor types of the dsv41_mx_* entries


def _rows16(x2: torch.Tensor, es: int, align: int = 16, most: int = 1 << 62) -> torch.Tensor:
    """x2 [rows, n] of es-byte elements with unit column stride, rows that do not overlap, `align`-byte aligned and at most `most` elements
    apart: itself, or a copy."""
    rows, n = x2.shape
    s0, s1 = x2.stride()
    if (s1 == 1 or n == 1) and not x2.data_ptr() % align and (rows <= 1 or (n <= s0 <= most and not s0 * es % align)):
        return x2
    return x2.clone(memory_format=torch.contiguous_format)


def quant_fp4(x: torch.Tensor, block: int = 32, values: bool = False):
    """Per-32 FP4 quantisation of bf16, fp16 or fp32 x [..., K], K % 32 == 0: (E2M1 codes uint8 [..., K / 2], two per byte, the even k in
    the low nibble; E8M0 bytes uint8 [..., K / 32]), what dequant_fp4, w4.W4 and w4.linear_fp4 take. The scale is the smallest power of
    two, from 2^-126 on, with amax <= 6 * scale, so nothing saturates; codes are rounded to nearest even and keep the sign of zero.
    `values`: also the bf16 values that the codes stand for (dequant_fp4 of the two), from the same launch; an amax above 1.75 * 2^127
    rounds up to 2^128, infinity in bf16.
    A group with a NaN or an infinity in it gets the byte 255 and zero codes: dequant_fp4 and the product give NaN for all of it.
    Inference only: an x with a gradient to follow (reverse or forward mode) is refused, and so is a tracer."""
    if block != 32:
        raise ValueError(f"quant_fp4 has groups of 32, got {block}")
    dt, shape = x.dtype, x.shape
    if dt not in _TYPE:
        raise TypeError(f"quant_fp4 takes bf16, fp16 or fp32, got {dt}")
    K = shape[-1] if shape else 0
    if K % 32 or K == 0:
        raise ValueError(f"quant_fp4: the last dimension is a multiple of 32, got {tuple(shape)}")
    _lib.inference_only("quant_fp4", x)
    if not x.is_cuda:
        _lib.require_cuda(x)
    dev, lead, rows, ld = x.device, shape[:-1], x.numel() // K, K
    vals = torch.empty_like(x, dtype=torch.bfloat16, memory_format=torch.contiguous_format) if values else None
    if not x.is_contiguous() or x.data_ptr() & 15:
        x = _rows16(x.reshape(-1, K), x.element_size())
        ld = _lib.row_stride(x)
    codes = torch.empty((*lead, K // 2), dtype=torch.uint8, device=dev)
    scales = torch.empty((*lead, K // 32), dtype=torch.uint8, device=dev)
    if rows:
        _lib.launch(dev, "dsv41_mx_quant", x.data_ptr(), _TYPE[dt], rows, K, ld, 4, K, codes.data_ptr(), scales.data_ptr(),
                    vals.data_ptr() if values else None)
    return (codes, scales, vals) if values else (codes, scales)


def quant_fp8_e8m0(x: torch.Tensor, block: int = 32, permuted: bool = False, codes: torch.Tensor | None = None,
                   scales: torch.Tensor | None = None):
    """Per-32 FP8 quantisation in the MFMA operand format: (E4M3 codes uint8 [..., K], E8M0 bytes uint8
    [..., K/32]), codes in natural k order. `permuted`: x is in the 8-k permuted order of permute_x."""
    assert block == 32
    dev = _lib.require_cuda(x)
    K = x.shape[-1]
    x2 = x.reshape(-1, K)
    if x2.stride(-1) != 1:
        x2 = x2.contiguous()
    assert x2.dtype in (torch.bfloat16, torch.float32)
    rows = x2.shape[0]
    if codes is None:
        codes = torch.empty(*x.shape, dtype=torch.uint8, device=dev)
    if scales is None:
        scales = torch.empty(*x.shape[:-1], K // 32, dtype=torch.uint8, device=dev)
    _lib.call("dsv41_quant_fp8", _lib.ptr(x2), 1 if x2.dtype == torch.float32 else 0, rows, K, x2.stride(0), 1 if permuted else 0,
              _lib.ptr(codes), _lib.ptr(scales), None, _lib.stream(dev))
    return codes, scales


def quant_fp8_split(x: torch.Tensor, permuted: bool = False, flag: bool = True):
    """bf16 x [..., K] as two FP8 operand terms, x = hi + lo per 32-group (dsv41_quant_fp8_split): returns (hi codes,
    hi scales, lo codes, lo scales, lo flag). hi is exactly quant_fp8_e8m0(x); lo is the residual rounded to E4M3 with
    its own E8M0 byte, so hi + lo reproduces the bf16 values (exactly, except residuals below the lo term's normal
    range, which stay within 2^-21 of the group's amax). The flag (device int32 [1]; None when flag=False, which saves
    the launch that clears it) is 1 when some lo code is not zero: the GEMMs that would read the weights a second time
    for the lo term skip that pass when it is 0."""
    dev = _lib.require_cuda(x)
    K = x.shape[-1]
    if x.dtype != torch.bfloat16:
        raise TypeError(f"quant_fp8_split takes bf16 activations (the reference's kernels take bf16), got {x.dtype}")
    x2 = x.reshape(-1, K)
    if x2.stride(-1) != 1 or x2.stride(0) % 8 or x2.data_ptr() % 16:
        x2 = x2.clone(memory_format=torch.contiguous_format)   # a fresh allocation: aligned, row stride K
    rows = x2.shape[0]
    hc = torch.empty(*x.shape, dtype=torch.uint8, device=dev)
    lc = torch.empty(*x.shape, dtype=torch.uint8, device=dev)
    hs = torch.empty(*x.shape[:-1], K // 32, dtype=torch.uint8, device=dev)
    ls = torch.empty(*x.shape[:-1], K // 32, dtype=torch.uint8, device=dev)
    f = torch.empty(1, dtype=torch.int32, device=dev) if flag else None
    _lib.call("dsv41_quant_fp8_split", _lib.ptr(x2), rows, K, x2.stride(0), 1 if permuted else 0, _lib.ptr(hc), _lib.ptr(hs), _lib.ptr(lc),
              _lib.ptr(ls), _lib.ptr(f), _lib.stream(dev))
    return hc, hs, lc, ls, f


def attach_codes(x: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, permuted: bool = False) -> torch.Tensor:
    """Record on the bf16 tensor x that its values are exactly the FP8 operand (E4M3 codes, E8M0 bytes) in natural k
    order, as the kernel that wrote x also wrote them (swiglu_quant: the fq8 rounding produces the codes first and the
    bf16 values from them). `permuted`: x holds the values in the 8-k permuted order of permute_x. The record is
    tied to x's version counter, storage address, shape and strides, so an in-place change of x (through x or any view
    of it), a resize or a set_ drops it; views and copies of x carry none. Library entry points that write into a
    caller's tensor (`out=` arguments) bump no version counter, except add_rmsnorm_quant: a tensor passed to the others must not be
    read as an operand afterwards on the strength of an earlier record. Inference-mode tensors keep no version counter, so they get no record (an in-place change could
    not be seen) and are quantised again where used. Returns x."""
    assert codes.shape == x.shape and scales.shape == (*x.shape[:-1], x.shape[-1] // 32)
    if not x.is_inference():
        x._dsv41_fp8 = (codes, scales, bool(permuted), x._version, x.data_ptr(), tuple(x.shape), tuple(x.stride()))
    return x


def attached_codes(x: torch.Tensor, permuted: bool):
    """(codes, scales) recorded on x by attach_codes for the same k order, if x is unchanged since; else None."""
    t = getattr(x, "_dsv41_fp8", None)
    if (t is None or x.is_inference() or t[2] != bool(permuted) or t[3] != x._version or t[4] != x.data_ptr()
            or t[5] != tuple(x.shape) or t[6] != tuple(x.stride())):
        return None
    return t[0], t[1]


def fake_quant_fp8(x: torch.Tensor, block: int = 32) -> torch.Tensor:
    """act_quant(..., inplace=True) of the reference: per-32 power-of-two scale, E4M3 RNE, dequantised, in
    x's dtype (quant.py:45-54)."""
    assert block == 32
    dev = _lib.require_cuda(x)
    K = x.shape[-1]
    x2 = x.reshape(-1, K)
    if x2.stride(-1) != 1:
        x2 = x2.contiguous()
    assert x2.dtype in (torch.bfloat16, torch.float32)
    out = torch.empty(x.shape, dtype=x.dtype, device=dev)
    _lib.call("dsv41_quant_fp8", _lib.ptr(x2), 1 if x2.dtype == torch.float32 else 0, x2.shape[0], K, x2.stride(0), 0,
              None, None, _lib.ptr(out), _lib.stream(dev))
    return out


def fake_quant_codes(x: torch.Tensor):
    """fake_quant_fp8 of a bf16 [rows, K] tensor and, from the same launch, its FP8 operand: (values, E4M3 codes, E8M0 bytes)."""
    dev = _lib.require_cuda(x)
    rows, K = x.shape
    assert x.dtype == torch.bfloat16 and x.stride(1) == 1
    out = torch.empty(rows, K, dtype=torch.bfloat16, device=dev)
    codes = torch.empty(rows, K, dtype=torch.uint8, device=dev)
    scales = torch.empty(rows, K // 32, dtype=torch.uint8, device=dev)
    _lib.call("dsv41_quant_fp8", _lib.ptr(x), 0, rows, K, x.stride(0), 0, _lib.ptr(codes), _lib.ptr(scales), _lib.ptr(out), _lib.stream(dev))
    return out, codes, scales


def quant_fp8(x: torch.Tensor, block: int = 32):
    """The FP8 rounding without the dequantisation (quant.py:57-64): the float8_e4m3fn codes and one float32 power of two
    per 32 values."""
    codes, e8 = quant_fp8_e8m0(x, block)
    return codes.view(torch.float8_e4m3fn), e8m0_to_float(e8)


# ------------------------------------------------------------------ the tile_fp4 layout of the expert weights
# quant.py:113-139: [E, N, K/2] -> [E][N/16][K/128][16 rows][64 B] (scales [N/16][K/128][16][4]). Each 1 KiB
# block is exactly the 16-row x 128-k weight tile one block-scaled MFMA consumes, so the kernels read the
# tiled layout with one contiguous 1 KiB load per wave.
def tile_fp4(w: torch.Tensor) -> torch.Tensor:
    E, N, Kh = w.shape
    assert N % 16 == 0 and Kh % 64 == 0
    return w.view(E, N // 16, 16, Kh // 64, 64).permute(0, 1, 3, 2, 4).reshape(E, N, Kh).contiguous()


def untile_fp4(w: torch.Tensor) -> torch.Tensor:
    E, N, Kh = w.shape
    return w.view(E, N // 16, Kh // 64, 16, 64).permute(0, 1, 3, 2, 4).reshape(E, N, Kh).contiguous()


def tile_fp4_scales(s: torch.Tensor) -> torch.Tensor:
    E, N, Ks = s.shape
    assert N % 16 == 0 and Ks % 4 == 0
    return s.view(E, N // 16, 16, Ks // 4, 4).permute(0, 1, 3, 2, 4).reshape(E, N, Ks).contiguous()


def untile_fp4_scales(s: torch.Tensor) -> torch.Tensor:
    E, N, Ks = s.shape
    return s.view(E, N // 16, Ks // 4, 16, 4).permute(0, 1, 3, 2, 4).reshape(E, N, Ks).contiguous()


def tile_bf16(w: torch.Tensor) -> torch.Tensor:
    """bf16 [N, K] row-major -> [N/16][K/32][16 rows][32 k]: one 16 x 32 tile (the A operand of one bf16 16x16x32 MFMA)
    is one contiguous 1 KiB block, as tile_fp4 does for the FP4 experts (quant.py:118-122), so a wave streams whole
    blocks. This build's layout for the bf16 shared expert in the fused decode launches (applied once at load)."""
    N, K = w.shape
    assert N % 16 == 0 and K % 32 == 0 and w.dtype == torch.bfloat16
    return w.reshape(N // 16, 16, K // 32, 32).permute(0, 2, 1, 3).reshape(N, K).contiguous()


def untile_bf16(w: torch.Tensor) -> torch.Tensor:
    N, K = w.shape
    return w.reshape(N // 16, K // 32, 16, 32).permute(0, 2, 1, 3).reshape(N, K).contiguous()


def dequant_fp8_block(w: torch.Tensor, scale: torch.Tensor, block: int = 32, tiled: bool = False) -> torch.Tensor:
    """float8_e4m3fn (or uint8 E4M3 bytes) [N, K] with E8M0 scales [ceil(N/32), ceil(K/32)] -> bf16 [N, K]: the fp32
    product rounded to bf16, bit-exact with quant.dequant_fp8_block (quant.py:90-95). `tiled`: w in the layout of
    w8.tile (the result is row-major either way)."""
    assert block == 32
    dev = _lib.require_cuda(w, scale)
    wb = w.view(torch.uint8)
    s = scale.view(torch.uint8)
    N, K = wb.shape
    assert wb.stride(1) == 1 and s.stride(1) == 1 and K % 16 == 0
    assert s.shape[0] * 32 >= N and s.shape[1] * 32 >= K, "scale shape does not cover the weights"
    out = torch.empty(N, K, dtype=torch.bfloat16, device=dev)
    _lib.call("dsv41_dequant_fp8", _lib.ptr(wb), wb.stride(0), 1 if tiled else 0, _lib.ptr(s), s.stride(0), N, K, _lib.ptr(out),
              out.stride(0), _lib.stream(dev))
    return out
