"""Performance cases of the microscaled dense operators: quantisation to FP4 (E2M1 codes with one E8M0 byte per 32 values), the
dense product with FP4 weights, and the residual + RMSNorm that writes the product's operand.

A case is a dict of plain values; `kind` names the operator:
  quant   quant.quant_fp4: `rows` x `k` values to codes and scale bytes, and the values that they stand for.
  norm    fused.add_rmsnorm_quant with FP8 (E4M3) codes: `rows` x `k`, the residual stream and the operand.
  linear  w4.linear_fp4: `rows` activations of `k` values, rounded to `act`, times FP4 weights n x k.
  block   the two in a row as a layer runs them: norm to an `act` operand, then the product that reads it.

With `own` false a pass computes the operators' definitions with elementary torch operations in 32 bits.
"""
import math
import os
import sys

import torch

own = False

EPS = 1e-6
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
# (n, k) of a layer's dense projections, of shared experts (gate and up together, down), and of larger generic layers
DENSE = ((5120, 8192), (4608, 5120), (32768, 1280), (1280, 5120), (5120, 2304), (3328, 7168), (7168, 1664), (8192, 8192))


def _ops():
    """The framework's modules (where `own` is true)."""
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "deepseekv4.1-a100-custom_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from dsv41_amd import fused, quant, w4
    return fused, quant, w4


def _case(name, kind, rows, k, dtype="bf16", n=0, act="fp8"):
    c = {"kind": kind, "rows": rows, "k": k, "dtype": dtype}
    if kind in ("linear", "block"):
        c.update(n=n, act=act)
    return dict(c, name=name) if name else c


def listed():
    return [
        _case("quantise 16 x 5120", "quant", 16, 5120),                                # a decode batch's activations
        _case("quantise 32768 x 5120", "quant", 32768, 5120),                          # a weight matrix at load
        _case("norm 1 x 5120", "norm", 1, 5120),                                       # one token being decoded
        _case("norm 333 x 7168", "norm", 333, 7168, "fp16"),                           # a short prompt
        _case("norm 16384 x 5120", "norm", 16384, 5120),                               # a long prompt
        _case("W4A4 1 row 5120 x 8192", "linear", 1, 8192, n=5120, act="fp4"),         # an output projection, one token
        _case("W4A8 16 rows 4608 x 5120", "linear", 16, 5120, n=4608, act="fp8"),      # a decode batch
        _case("W4A4 97 rows 5120 x 8192", "linear", 97, 8192, n=5120, act="fp4"),      # a large decode batch
        _case("W4A8 700 rows 3999 x 2336", "linear", 700, 2336, "fp32", n=3999, act="fp8"),   # odd sizes, fp32 activations
        _case("W4A4 8192 rows 8192 x 8192", "linear", 8192, 8192, n=8192, act="fp4"),  # a long prompt, compute-bound
        _case("block W4A4 1 row", "block", 1, 5120, n=4608, act="fp4"),                # norm and projection, one token
        _case("block W4A8 2048 rows", "block", 2048, 7168, n=3328, act="fp8"),         # norm and a shared expert's gate and up, a prompt
    ]


def _log(rng, lo, hi):
    return min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49))))))


def draw(rng):
    kind = rng.choice(("quant", "norm", "linear", "linear", "linear", "block"))
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    if kind in ("quant", "norm"):
        return _case("", kind, _log(rng, 1, 16384), 32 * _log(rng, 8, 256), dtype)
    n, k = rng.choice(DENSE) if rng.random() < 0.5 else (_log(rng, 200, 8192), 32 * _log(rng, 8, 256))
    return _case("", kind, _log(rng, 1, 8192), k, dtype, n, rng.choice(("fp4", "fp8")))


# --------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _out(c):
    """The type of a product's result: the activations', but bf16 for fp32 activations rounded to FP8. The matrix unit adds the products of FP8
    and FP4 codes eight at a time with bits below 2^-13 of the largest dropped (1e-5 of the result), so their fp32 digits say nothing."""
    return torch.bfloat16 if c["dtype"] == "fp32" and c["act"] == "fp8" else DTYPES[c["dtype"]]


def _acts(g, c):
    """Normal activations with a few channels that are an order of magnitude larger."""
    x = torch.randn(c["rows"], c["k"], generator=g, device="cuda")
    hot = torch.randint(0, c["k"], (max(1, c["k"] // 256),), generator=g, device="cuda")
    x[:, hot] *= 15.0
    return x.to(DTYPES[c["dtype"]])


def _weights(g, c):
    """Packed E2M1 codes [n, k / 2] and E8M0 bytes [n, k / 32] of normal weights, as a checkpoint holds them."""
    w = torch.randn(c["n"], c["k"], generator=g, device="cuda") / math.sqrt(c["k"])
    codes, scales, _ = _plain_fp4(w)
    return codes, scales


def _norm_inputs(g, c):
    w = (1 + 0.2 * torch.randn(c["k"], generator=g, device="cuda")).to(DTYPES[c["dtype"]])
    return {"x": _acts(g, c), "res": 2 * _acts(g, c), "g": w}


def _inputs(case, seed):
    c, g = case, _gen(seed)
    s = _norm_inputs(g, c) if c["kind"] in ("norm", "block") else {"x": _acts(g, c)}
    if c["kind"] in ("linear", "block"):
        s["codes"], s["scales"] = _weights(g, c)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if own and "codes" in s:
        s["w"] = _ops()[2].W4(s["codes"], s["scales"])   # the weights as a program loads them, once
    return s


# --------------------------------------------------------------------------- the plain forms
def _groups(v):
    return v.reshape(*v.shape[:-1], -1, 32)


def _pow2f(e):
    """2^e in 32 bits, -126 <= e <= 127, from its exponent bits."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _plain_fp4(x):
    """(packed codes, E8M0 bytes, values) of x by 32-bit operations: scale 2^e, e the smallest with amax <= 6 * 2^e (at least -126)."""
    v = _groups(x.to(torch.float32))
    amax = v.abs().amax(-1, keepdim=True)
    m, p = torch.frexp(amax)                                    # amax = m 2^p, 0.5 <= m < 1
    e = torch.where(m <= 0.75, p - 3, p - 2).clamp_min(-126)
    e = torch.where(amax > 0, e, -126)
    q = v * _pow2f(-e)
    a = q.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    a = torch.round(a / step) * step                            # half to even on every step, as E2M1's even codes are
    values = torch.copysign(a, q) * _pow2f(e)
    code = torch.where(a < 2, 2 * a, torch.where(a < 4, a + 2, 4 + a / 2)).to(torch.uint8) | (torch.signbit(q).to(torch.uint8) << 3)
    code = code.reshape(*x.shape[:-1], -1, 2)
    packed = code[..., 0] | (code[..., 1] << 4)
    return packed, (e + 127).to(torch.uint8).reshape(*x.shape[:-1], -1), values.reshape(x.shape)


def _plain_fp8(x):
    """(E4M3 codes, E8M0 bytes, values) of fp32 x: scale 2^e, e the smallest with max(amax, 1e-4) <= 448 * 2^e."""
    v = _groups(x)
    m, p = torch.frexp(v.abs().amax(-1, keepdim=True).clamp_min(1e-4) / 448.0)
    e = torch.where(m == 0.5, p - 1, p)
    codes = (v * _pow2f(-e)).to(torch.float8_e4m3fn)
    values = codes.to(torch.float32) * _pow2f(e)
    return codes.reshape(x.shape), (e + 127).to(torch.uint8).reshape(*x.shape[:-1], -1), values.reshape(x.shape)


def _plain_weights(codes, scales):
    table = torch.tensor((0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0), device=codes.device)
    v = table[torch.stack((codes & 15, codes >> 4), -1).reshape(codes.shape[0], -1).to(torch.int32)]
    return (_groups(v) * _pow2f(scales.to(torch.int32) - 127)[..., None]).reshape(v.shape)


def _plain_norm(s):
    r = (s["x"].to(torch.float32) + s["res"].to(torch.float32)).to(s["x"].dtype)
    v = r.to(torch.float32)
    return v * torch.rsqrt(v.square().mean(-1, keepdim=True) + EPS) * s["g"].to(torch.float32), r


def _plain_round(x, act):
    return (_plain_fp4(x) if act == "fp4" else _plain_fp8(x.to(torch.float32)))[2].to(torch.float32)


def _plain(s):
    c = s["case"]
    if c["kind"] == "quant":
        codes, scales, values = _plain_fp4(s["x"])
        return values.to(torch.bfloat16), codes, scales
    if c["kind"] == "norm":
        v, r = _plain_norm(s)
        codes, scales, _ = _plain_fp8(v)
        return codes, scales.view(torch.float8_e8m0fnu), r
    w = _plain_weights(s["codes"], s["scales"])
    if c["kind"] == "linear":
        return (_plain_round(s["x"], c["act"]) @ w.t()).to(_out(c))
    v, r = _plain_norm(s)
    return (_plain_round(v, c["act"]) @ w.t()).to(_out(c)), r


def run(state):
    if not own:
        return _plain(state)
    fused, quant, w4 = _ops()
    c = state["case"]
    if c["kind"] == "quant":
        codes, scales, values = quant.quant_fp4(state["x"], values=True)
        return values, codes, scales
    if c["kind"] == "norm":
        codes, scales, r = fused.add_rmsnorm_quant(state["x"], state["res"], state["g"], EPS)
        return codes.view(torch.float8_e4m3fn), scales.view(torch.float8_e8m0fnu), r
    if c["kind"] == "linear":
        return w4.linear_fp4(state["x"], state["w"], act=c["act"], out_dtype=_out(c))
    codes, scales, r = fused.add_rmsnorm_quant(state["x"], state["res"], state["g"], EPS, fmt=c["act"])
    return w4.linear_fp4((codes, scales), state["w"], out_dtype=_out(c)), r


# --------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    c = case
    M, K, es = c["rows"], c["k"], 4 if c["dtype"] == "fp32" else 2
    if c["kind"] == "quant":
        return {"bytes": M * K * (es + 2) + M * K // 2 + M * K // 32, "flops": 4 * M * K}
    if c["kind"] == "norm":
        return {"bytes": M * K * (3 * es + 1) + M * K // 32 + K * es, "flops": 8 * M * K}
    N = c["n"]
    b, f = N * K // 2 + N * K // 32 + M * N * (4 if _out(c) == torch.float32 else 2), 2 * M * N * K
    if c["kind"] == "linear":
        return {"bytes": b + M * K * es, "flops": f}
    return {"bytes": b + 3 * M * K * es + K * es, "flops": f + 8 * M * K}   # the operand between the two need not reach memory


# --------------------------------------------------------------------------- 64-bit results
def _pow2(e):
    """2^e in 64 bits, from its exponent bits."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _exact_fp4(v):
    """(values, exponents, code numbers) by counting the midpoints between E2M1 neighbours below each magnitude; ties to even codes."""
    v = _groups(v)
    a = v.abs()
    e = torch.ceil(torch.log2(a.amax(-1, keepdim=True).clamp_min(2.0 ** -200) / 6.0)).to(torch.int32).clamp_min(-126)
    top = a.amax(-1, keepdim=True)                              # log2 may round across an integer: settle it by comparison
    e = torch.where(top > 6.0 * _pow2(e), e + 1, torch.where((top <= 6.0 * _pow2(e - 1)) & (e > -126), e - 1, e))
    a = a / _pow2(e)
    idx = torch.zeros_like(a, dtype=torch.uint8)
    for i, mid in enumerate((0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)):
        idx += (a > mid) if i % 2 == 0 else (a >= mid)
    mag = torch.where(idx < 4, idx / 2.0, torch.where(idx < 6, idx - 2.0, 2.0 * idx - 8.0)).double()
    return torch.where(torch.signbit(v), -mag, mag) * _pow2(e), e, idx | (torch.signbit(v).to(torch.uint8) << 3)


def _exact_fp8(v):
    """(values over the scale, exponents): E4M3 by its definition, three mantissa bits above 2^-6, steps of 2^-9 below."""
    v = _groups(v)
    top = v.abs().amax(-1, keepdim=True).clamp_min(1e-4)
    e = torch.ceil(torch.log2(top / 448.0)).to(torch.int32)
    e = torch.where(top > 448.0 * _pow2(e), e + 1, torch.where(top <= 448.0 * _pow2(e - 1), e - 1, e))
    q = v / _pow2(e)
    step = _pow2((torch.frexp(q)[1] - 1).clamp_min(-6) - 3)
    return torch.round(q / step) * step, e


def _exact_round(v, act):
    if act == "fp4":
        return _exact_fp4(v)[0].reshape(v.shape)
    q, e = _exact_fp8(v)
    return (q * _pow2(e)).reshape(v.shape)


def _exact_product(a, codes, scales):
    mag = torch.tensor((0, 1, 2, 3, 4, 6, 8, 12), dtype=torch.float64, device=codes.device) / 2
    out = []
    for c, s in zip(codes.split(2048), scales.split(2048)):
        two = [torch.where(h >= 8, -1.0, 1.0).double() * mag[(h & 7).long()] for h in (c & 15, c >> 4)]
        w = _groups(torch.stack(two, -1).reshape(c.shape[0], -1)) * _pow2(s.to(torch.int32) - 127)[..., None]
        out.append(a @ w.reshape(c.shape[0], -1).t())
    return torch.cat(out, -1)


def exact(case, seed):
    c, s = case, _inputs(case, seed)
    if c["kind"] == "quant":
        values, e, code = _exact_fp4(s["x"].double())
        code = code.reshape(c["rows"], -1, 2)
        return values.reshape(c["rows"], -1), code[..., 0] | (code[..., 1] << 4), (e + 127).to(torch.uint8).reshape(c["rows"], -1)
    if c["kind"] == "linear":
        return _exact_product(_exact_round(s["x"].double(), c["act"]), s["codes"], s["scales"])
    # the stream is stored in its own type, so that rounding is part of the definition
    r = (s["x"].double() + s["res"].double()).to(s["x"].dtype).double()
    v = r / torch.sqrt(r.square().mean(-1, keepdim=True) + EPS) * s["g"].double()
    if c["kind"] == "norm":
        q, e = _exact_fp8(v)
        return q.reshape(v.shape), _pow2(e).reshape(c["rows"], -1), s["x"].double() + s["res"].double()
    return _exact_product(_exact_round(v, c["act"]), s["codes"], s["scales"]), s["x"].double() + s["res"].double()
