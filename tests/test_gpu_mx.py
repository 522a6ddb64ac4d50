"""The microscaled dense operators on the GPU (quant_fp4, add_rmsnorm_quant, W4 / linear_fp4) against plain implementations in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
MID = (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)                    # between E2M1 neighbours; ties go to the even code
MAG = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def pow2(e):
    """2^e in 64 bits."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def ceil_log2_ratio(top, m):
    """The smallest integer e with top <= m * 2^e (64 bits, top > 0)."""
    e = torch.ceil(torch.log2(top / m)).to(torch.int32)
    return torch.where(top > m * pow2(e), e + 1, torch.where(top <= m * pow2(e - 1), e - 1, e))


def ref_fp4(x):
    """(code numbers [.., K], E8M0 bytes [.., K/32], values fp64) of x by the definition, on the CPU."""
    v = x.double().cpu().reshape(*x.shape[:-1], -1, 32)
    a = v.abs()
    top = a.amax(-1, keepdim=True)                               # NaN if one is in the group
    bad = ~torch.isfinite(top)
    e = ceil_log2_ratio(torch.where(bad | (top == 0), torch.ones_like(top), top), 6.0).clamp_min(-126)
    e = torch.where(top == 0, torch.full_like(e, -126), e)
    q = a / pow2(e)
    idx = torch.zeros(q.shape, dtype=torch.uint8)
    for i, mid in enumerate(MID):
        idx += (q > mid) if i % 2 == 0 else (q >= mid)
    code = idx | (torch.signbit(v).to(torch.uint8) << 3)
    val = torch.tensor(MAG, dtype=torch.float64)[idx.long()] * pow2(e)
    val = torch.where(torch.signbit(v), -val, val)
    code = torch.where(bad, torch.zeros_like(code), code)
    val = torch.where(bad, torch.full_like(val, math.nan), val)
    byte = torch.where(bad, torch.full_like(e, 255), e + 127).to(torch.uint8)
    return code.reshape(x.shape), byte.reshape(*x.shape[:-1], -1), val.reshape(x.shape)


def ref_fp8(v):
    """(values over the scale, E8M0 bytes, values) of fp64 v by E4M3's definition and the framework's scale rule."""
    v = v.reshape(*v.shape[:-1], -1, 32)
    e = ceil_log2_ratio(v.abs().amax(-1, keepdim=True).clamp_min(float(torch.tensor(1e-4))), 448.0)
    q = v / pow2(e)
    step = pow2((torch.frexp(q)[1] - 1).clamp_min(-6) - 3)
    q = torch.round(q / step) * step
    shape = (*v.shape[:-2], -1)
    return q.reshape(shape), (e + 127).to(torch.uint8).reshape(*v.shape[:-2], -1), (q * pow2(e)).reshape(shape)


def pack(code):
    c = code.reshape(*code.shape[:-1], -1, 2)
    return c[..., 0] | (c[..., 1] << 4)


def gen(seed):
    return torch.Generator().manual_seed(seed)


def randn(g, *shape, dtype=torch.float32, spread=0.0):
    x = torch.randn(*shape, generator=g)
    if spread:
        x = x * torch.exp(spread * torch.randn(*shape[:-1], 1, generator=g))
    return x.to(dtype)


# --------------------------------------------------------------------------- quant_fp4
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("shape", [(1, 32), (3, 96), (5, 7, 160), (33, 5120), (257, 1184), (0, 64)])
def test_quant_fp4_matches_the_definition(dtype, shape):
    from dsv41_amd import quant
    x = randn(gen(1), *shape, dtype=DT[dtype], spread=3.0)
    codes, scales, values = quant.quant_fp4(x.cuda(), values=True)
    assert codes.shape == (*shape[:-1], shape[-1] // 2) and scales.shape == (*shape[:-1], shape[-1] // 32) and values.shape == shape
    if not x.numel():
        return
    code, byte, val = ref_fp4(x)
    assert torch.equal(codes.cpu(), pack(code)) and torch.equal(scales.cpu(), byte)
    assert values.dtype == torch.bfloat16 and torch.equal(values.cpu().double(), val)
    c2, s2 = quant.quant_fp4(x.cuda())
    assert torch.equal(c2, codes) and torch.equal(s2, scales)
    assert torch.equal(quant.dequant_fp4(codes, scales).view(torch.int16), values.view(torch.int16))


@pytest.mark.parametrize("dtype", DT)
def test_quant_fp4_borders(dtype):
    """Every tie and its neighbours, scale borders, signed zeros, the smallest and largest magnitudes."""
    from dsv41_amd import quant
    t = DT[dtype]
    eps = torch.finfo(t).eps
    mids = torch.tensor(MID + MAG)
    near = torch.cat([mids, mids * (1 + eps), mids * (1 - eps)])
    near = torch.cat([near, -near])
    rows = []
    for e in (-14, -3, 0, 1, 9, 13):
        for top in (6.0, 4.0, 6.0 * (1 + eps), 3.1):
            r = torch.zeros(64)
            r[0], r[32] = top, -top
            r[1:32], r[33:64] = near[:31], near[31:62] if near.numel() >= 62 else near[-31:]
            rows.append((r.clamp(-top, top) * 2.0 ** e).to(t))
    big, tiny = torch.finfo(t).max, torch.finfo(t).tiny
    rows.append(torch.full((64,), big).to(t))
    rows.append(torch.full((64,), tiny).to(t))
    rows.append((torch.arange(64) * (tiny / 16)).to(t))             # subnormals of the type
    rows.append(torch.tensor([0.0, -0.0] * 32).to(t))
    x = torch.stack(rows)
    codes, scales, values = quant.quant_fp4(x.cuda(), values=True)
    code, byte, val = ref_fp4(x)
    assert torch.equal(scales.cpu(), byte)
    assert torch.equal(codes.cpu(), pack(code))
    # the largest bf16 and fp32 values round to 4 * 2^126 = 2^128, which bf16 holds as infinity; every other value is a bf16 value
    assert torch.equal(values.cpu(), val.to(torch.bfloat16))


@pytest.mark.parametrize("dtype", DT)
def test_quant_fp4_marks_groups_that_are_not_finite(dtype):
    from dsv41_amd import quant
    x = randn(gen(2), 6, 128, dtype=DT[dtype])
    x[0, 5], x[1, 40], x[2, 127], x[3, 0] = math.nan, math.inf, -math.inf, -math.nan
    codes, scales, values = quant.quant_fp4(x.cuda(), values=True)
    code, byte, val = ref_fp4(x)
    assert torch.equal(scales.cpu(), byte) and torch.equal(codes.cpu(), pack(code))
    assert (byte == 255).sum() == 4
    assert torch.equal(torch.isnan(values.cpu()), torch.isnan(val))
    assert torch.equal(torch.nan_to_num(values.cpu().double()), torch.nan_to_num(val))


def test_quant_fp4_strides():
    """Rows of a wider matrix, a transposed view, a base that is not aligned, expanded rows, a last dimension with a stride."""
    from dsv41_amd import quant
    base = randn(gen(3), 40, 320, dtype=torch.bfloat16).cuda()
    for x in (base[:, 64:224], base[::2, :64], base.t()[:, :32], base.reshape(-1)[3:3 + 64 * 5].view(5, 64), base[:1, :96].expand(7, 96),
              base[:, ::5], base.view(8, 5, 320).transpose(0, 1)[..., :64]):
        want = quant.quant_fp4(x.clone(memory_format=torch.contiguous_format))
        got = quant.quant_fp4(x)
        assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])


# --------------------------------------------------------------------------- add_rmsnorm_quant
def ref_norm(x, res, w, eps):
    """(r in x's dtype, v fp64) from the formula: r is rounded to the stream's type, everything behind it is 64-bit."""
    r = x if res is None else (x.float() + res.float()).to(x.dtype)
    d = r.double()
    return r, d / torch.sqrt(d.square().mean(-1, keepdim=True) + eps) * w.double()


def check_operand(codes, scales, v, fmt):
    """codes / scales against v quantised exactly. The kernel's fp32 v is off by few 2^-24 relative: where v lies that near a rounding
    border the neighbouring code is as right, and where a group's amax lies that near a scale border the neighbouring scale is. Every other
    code has to be equal; the borders may not be met by more than one value in 2000 (an interval of 16 * 2^-24 around borders that are
    at least 2^-5 apart relative to the value holds about 2^-15 of them)."""
    from dsv41_amd import quant
    if fmt == "fp8":
        q, byte, val = ref_fp8(v)
        got = codes.cpu().view(torch.float8_e4m3fn).double()
    else:
        code, byte, val = ref_fp4(v)
        got = None
    gs = scales.cpu().repeat_interleave(32, -1).to(torch.int32) - 127
    if got is None:
        c = codes.cpu()
        c = torch.stack((c & 15, c >> 4), -1).reshape(v.shape)
        mag = torch.tensor(MAG, dtype=torch.float64)[(c & 7).long()]
        got = torch.where(c >= 8, -mag, mag)
    gv = got * pow2(gs)
    differ = gv != val
    assert differ.double().mean().item() <= 1 / 2000
    assert (scales.cpu() != byte).sum().item() <= max(1, byte.numel() // 2000)
    # where it differs, the code that was taken is a nearest one up to 16 * 2^-24 of the value: its error is not larger than the exact one's by more
    err, best = (gv - v).abs()[differ], (val - v).abs()[differ]
    same_scale = (gs == byte.repeat_interleave(32, -1).to(torch.int32) - 127)[differ]
    assert (err <= best + 32 * 2.0 ** -24 * v.abs()[differ])[same_scale].all()


@pytest.mark.parametrize("fmt", ["fp8", "fp4"])
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("rows,K", [(1, 32), (1, 5120), (3, 2048), (5, 2080), (7, 8192), (2, 8224), (333, 7168), (2, 32768), (0, 64)])
def test_add_rmsnorm_quant(rows, K, dtype, fmt):
    from dsv41_amd import fused
    g, t = gen(rows * 131 + K), DT[dtype]
    x, res = randn(g, rows, K, dtype=t, spread=1.0), randn(g, rows, K, dtype=t, spread=1.0)
    w = (1 + 0.3 * torch.randn(K, generator=g)).to(t)
    codes, scales, r, y = fused.add_rmsnorm_quant(x.cuda(), res.cuda(), w.cuda(), 1e-6, fmt=fmt, y=True)
    assert codes.shape == (rows, K if fmt == "fp8" else K // 2) and scales.shape == (rows, K // 32) and r.dtype == t and y.dtype == t
    if rows == 0:
        return
    want_r, v = ref_norm(x, res, w, 1e-6)
    assert torch.equal(r.cpu(), want_r)
    check_operand(codes, scales, v, fmt)
    # y: one rounding to t (half a step: eps / 2) of a value that is off by at most 16 * 2^-24 (sum of K squares in a tree of lanes and
    # waves, square root, two products); below t's normal range half a step of its smallest value
    tol = (torch.finfo(t).eps / 2 + 16 * 2.0 ** -24) * v.abs() + torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2
    assert ((y.cpu().double() - v).abs() <= tol).all()
    c0, s0, r0 = fused.add_rmsnorm_quant(want_r.cuda(), None, w.cuda(), 1e-6, fmt=fmt)
    assert torch.equal(c0, codes) and torch.equal(s0, scales) and torch.equal(r0.cpu(), want_r)


def test_add_rmsnorm_quant_in_place_and_strides():
    from dsv41_amd import fused
    g = gen(5)
    buf = randn(g, 3, 9, 4 * 640, dtype=torch.bfloat16).cuda()
    x, res = buf[..., 640:1280], buf[..., 1280:1920]
    w = randn(g, 640, dtype=torch.bfloat16).cuda()
    want = fused.add_rmsnorm_quant(x.contiguous(), res.contiguous(), w, 1e-5)
    keep = buf.clone()
    got = fused.add_rmsnorm_quant(x, res, w, 1e-5, out=res)          # into the residual's own place
    assert got[2] is res and all(torch.equal(a, b) for a, b in zip(want, got))
    assert torch.equal(buf[..., :1280], keep[..., :1280]) and torch.equal(buf[..., 1920:], keep[..., 1920:])   # nothing beside it
    buf.copy_(keep)
    got = fused.add_rmsnorm_quant(x, res, w, 1e-5, out=x)
    assert all(torch.equal(a, b) for a, b in zip(want, got)) and torch.equal(buf[..., 1280:], keep[..., 1280:])
    buf.copy_(keep)
    got = fused.add_rmsnorm_quant(x, res, w, 1e-5, out=buf[..., 1920:])
    assert all(torch.equal(a, b) for a, b in zip(want, got)) and torch.equal(buf[..., :1920], keep[..., :1920])
    odd = torch.empty(640 * 4 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(4, 640).copy_(x.reshape(-1, 640)[:4])   # rows off 16 bytes
    wodd = torch.empty(641, dtype=torch.bfloat16, device="cuda")[1:].copy_(w)
    assert torch.equal(fused.add_rmsnorm_quant(odd, odd, wodd, 1e-5)[0], fused.add_rmsnorm_quant(odd.clone(), odd.clone(), w, 1e-5)[0])


@pytest.mark.parametrize("fmt", ["fp8", "fp4"])
def test_add_rmsnorm_quant_edges(fmt):
    """A zero row, a row with a NaN, one with an infinity, one whose mean square overflows fp32, eps = 0."""
    from dsv41_amd import fused, w4
    x = randn(gen(6), 5, 128)
    x[1, 3], x[2, 70] = math.nan, math.inf
    x[0] = 0
    x[3] *= 1e30
    w = torch.ones(128)
    codes, scales, r = fused.add_rmsnorm_quant(x.cuda(), torch.zeros_like(x).cuda(), w.cuda(), 1e-6, fmt=fmt)
    assert torch.equal(torch.nan_to_num(r.cpu()), torch.nan_to_num(x)) and (scales[1] == 255).all() and scales[2].eq(255).sum() >= 1
    sign_free = 0x7F if fmt == "fp8" else 0x77
    assert not codes[0].any() and not (codes[3] & sign_free).any()   # zeros, which keep their signs
    W = w4.W4.from_dense(torch.eye(128).cuda())
    y = w4.linear_fp4((codes, scales), W)
    assert torch.isnan(y[1]).all() and torch.isnan(y[2]).all() and torch.isfinite(y[[0, 3, 4]]).all()
    c0, s0, _ = fused.add_rmsnorm_quant(x[4:].cuda(), None, w.cuda(), 0.0, fmt=fmt)
    check_operand(c0, s0, ref_norm(x[4:], None, w, 0.0)[1], fmt)


def test_add_rmsnorm_quant_many_rows():
    """More rows than one launch holds threads for (2^32 of them): rows of every launch as alone."""
    from dsv41_amd import fused
    rows = (1 << 24) + 7
    x = torch.empty(rows, 32, dtype=torch.bfloat16, device="cuda").normal_(generator=torch.Generator("cuda").manual_seed(31))
    w = randn(gen(31), 32, dtype=torch.bfloat16).cuda()
    got = fused.add_rmsnorm_quant(x, x, w, 1e-6, fmt="fp4")
    for at in (0, (1 << 21) - 3, (1 << 21) * 5 - 3, (1 << 24) - 4, rows - 6):
        want = fused.add_rmsnorm_quant(x[at:at + 6], x[at:at + 6], w, 1e-6, fmt="fp4")
        assert all(torch.equal(a[at:at + 6], b) for a, b in zip(got, want))


def test_offsets_past_32_bits():
    """Inputs, codes and outputs of more than 2^32 bytes or 2^31 values: the last rows as alone, or against 64 bits."""
    from dsv41_amd import fused, quant, w4
    M, K = 70000, 32768
    x = torch.empty(M, K, dtype=torch.bfloat16, device="cuda").normal_(generator=torch.Generator("cuda").manual_seed(32))
    tail = x[-9:].clone()
    for got, want in ((quant.quant_fp4(x), quant.quant_fp4(tail)), (fused.add_rmsnorm_quant(x, x, x[0], 1e-6), fused.add_rmsnorm_quant(tail, tail, x[0], 1e-6))):
        assert all(torch.equal(a[-9:], b) for a, b in zip(got, want))
    del got
    codes, scales = rand_w4(gen(32), 40, K, 118, 126)
    W, wv = w4.W4(codes.cuda(), scales.cuda()), deq4(codes, scales)
    for act in ("fp4", "fp8"):
        check_product(w4.linear_fp4(x, W, act=act)[-9:], ref_round(tail, act), wv, "bf16", act)
        op = quant.quant_fp4(x) if act == "fp4" else quant.quant_fp8_e8m0(x)
        check_product(w4.linear_fp4(op, W)[-9:], ref_round(tail, act), wv, "bf16", act)
        del op
    del x
    codes, scales = rand_w4(gen(33), 34000, 64, 118, 126)              # y of 2.2 * 2^31 values
    x = randn(gen(33), 140000, 64, dtype=torch.bfloat16)
    y = w4.linear_fp4(x.cuda(), w4.W4(codes.cuda(), scales.cuda()))
    check_product(y[-9:], ref_fp4(x[-9:])[2], deq4(codes, scales), "bf16", "fp4")


def test_norm_operand_equals_the_quantisers():
    """The codes are the quantisers' of the fp32 rows: with fp32 rows and y the two are bit for bit the same."""
    from dsv41_amd import fused, quant
    x = randn(gen(7), 37, 1664, spread=1.0).cuda()
    w = randn(gen(8), 1664).cuda()
    c, s, _, y = fused.add_rmsnorm_quant(x, None, w, 1e-6, fmt="fp8", y=True)
    c2, s2 = quant.quant_fp8_e8m0(y)
    assert torch.equal(c, c2) and torch.equal(s, s2)
    c, s, _, y = fused.add_rmsnorm_quant(x, None, w, 1e-6, fmt="fp4", y=True)
    c2, s2 = quant.quant_fp4(y)
    assert torch.equal(c, c2) and torch.equal(s, s2)


# --------------------------------------------------------------------------- W4 / linear_fp4
def rand_w4(g, N, K, lo=115, hi=130):
    codes = torch.randint(0, 256, (N, K // 2), generator=g, dtype=torch.uint8)
    scales = torch.randint(lo, hi, (N, K // 32), generator=g, dtype=torch.uint8)
    return codes, scales


def deq4(codes, scales):
    c = torch.stack((codes & 15, codes >> 4), -1).reshape(codes.shape[0], -1)
    mag = torch.tensor(MAG, dtype=torch.float64)[(c & 7).long()]
    return torch.where(c >= 8, -mag, mag) * pow2(scales.to(torch.int32) - 127).repeat_interleave(32, -1)


def ref_round(x, act):
    return ref_fp4(x)[2] if act == "fp4" else ref_fp8(x.double().cpu())[2]


def check_product(y, xv, wv, dtype, act):
    """y against the 64-bit product of the rounded operands, with the error that the matrix unit's additions may make.

    FP4 x FP4: products are multiples of 2^-2 below 2^6 over their scales, exact; per block of 32 one fp32 addition, at worst truncated:
    2^-23 of the magnitudes' sum each. FP8 x FP4 in addition: eight products at a time (k = 8 i .. 8 i + 7) are aligned to the largest of
    them, and bits below 2^-13 of its power of two are dropped (test_fp8_products_are_added_eight_at_a_time); the largest one loses nothing, its
    significand has 4 + 2 bits, so seven products lose less than 2^-13 of the largest each. One rounding to dtype on top: half a step."""
    want, mag = xv @ wv.t(), xv.abs() @ wv.abs().t()
    t = DT[dtype]
    tol = torch.finfo(t).eps / 2 * want.abs() + 2.0 ** -23 * (2 + xv.shape[1] // 32) * mag + torch.finfo(t).smallest_normal * torch.finfo(t).eps
    if act == "fp8":
        eight = lambda v: v.abs().reshape(v.shape[0], -1, 8).amax(-1)
        tol = tol + 7 * 2.0 ** -13 * (eight(xv) @ eight(wv).t())
    d = (y.cpu().double() - want).abs()
    assert (d <= tol).all(), f"largest excess {(d / tol).max().item():.3g}"


def test_fp8_products_are_added_eight_at_a_time():
    """The premise of check_product: beside a product of 2^10, one of 2^(10 - j) among the same eight k counts down to j = 13 and is dropped
    below; among other eights it counts in full. The FP4 product drops nothing (down to 2^-5 of the largest, all that E2M1 has)."""
    from dsv41_amd import w4
    for at, other in ((0, 5), (40, 47), (0, 8), (70, 127), (31, 32)):
        small = [2.0 ** (10 - j) for j in range(1, 19)]
        x, w = torch.zeros(len(small), 128), torch.zeros(1, 128)
        w[0, at], w[0, other] = 4.0, 1.0
        # a group's scale is 1 (amax 448 in every group), its codes are exact; 448 sits at a k whose weight is zero
        free = [next(k for k in range(32 * g, 32 * g + 32) if k not in (at, other)) for g in range(4)]
        x[:, free] = 448.0
        x[:, at], x[:, other] = 256.0, torch.tensor(small).clamp_max(256.0)
        W = w4.W4.from_dense(w.cuda())
        assert torch.equal(W.bf16().float().cpu(), w)
        y = w4.linear_fp4(x.cuda(), W, act="fp8", out_dtype=torch.float32).cpu()[:, 0].double() - 1024.0
        got = x[:, other].double()
        for j, (d, s) in enumerate(zip(y.tolist(), got.tolist())):
            kept = at // 8 != other // 8 or s >= 2.0 ** -3
            if s >= 2.0 ** -9:
                assert d == (s if kept else 0.0), (at, other, j)


SHAPES = [(1, 16, 32), (1, 1, 64), (2, 33, 96), (5, 100, 128), (16, 4608, 5120), (17, 48, 160), (31, 65, 256), (64, 64, 384), (65, 130, 512),
          (97, 1280, 2304), (128, 256, 1664), (129, 257, 800), (300, 515, 1184), (700, 3999, 2336), (0, 64, 128)]


@pytest.mark.parametrize("act", ["fp4", "fp8"])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_linear_fp4(M, N, K, act):
    from dsv41_amd import w4
    g = gen(M + 7 * N + K)
    codes, scales = rand_w4(g, N, K)
    W = w4.W4(codes.cuda(), scales.cuda())
    assert W.shape == (N, K) and all(torch.equal(a.cpu(), b) for a, b in zip(W.natural(), (codes, scales)))
    dtype = list(DT)[(M + N) % 3]
    x = randn(g, M, K, dtype=DT[dtype], spread=1.0)
    y = w4.linear_fp4(x.cuda(), W, act=act)
    assert y.shape == (M, N) and y.dtype == DT[dtype]
    if M:
        wv = deq4(codes, scales)
        if dtype == "fp16":                                       # keep the outputs inside fp16
            scales = (scales.to(torch.int32) - 8).to(torch.uint8)
            y, wv = w4.linear_fp4(x.cuda(), w4.W4(codes.cuda(), scales.cuda()), act=act), deq4(codes, scales)
        check_product(y, ref_round(x, act), wv, dtype, act)


@pytest.mark.parametrize("act", ["fp4", "fp8"])
def test_linear_fp4_large_tiles(act):
    """The largest tile: whole and ragged in both directions, K with half a 256-k stage at the end."""
    from dsv41_amd import hipkern, w4
    for M, N, K in ((4096, 4096, 640), (4090, 4083, 896)):
        g = gen(M)
        codes, scales = rand_w4(g, N, K, 120, 126)
        assert hipkern.mx_plan(M, N, K, 4 if act == "fp4" else 8)[0] == 2
        x = randn(g, M, K, dtype=torch.bfloat16)
        y = w4.linear_fp4(x.cuda(), w4.W4(codes.cuda(), scales.cuda()), act=act)
        xv, wv = ref_round(x, act), deq4(codes, scales)
        rows = torch.cat([torch.arange(0, M, 97), torch.arange(M - 5, M)])
        check_product(y.cpu()[rows], xv[rows], wv, "bf16", act)


@pytest.mark.parametrize("act", ["fp4", "fp8"])
@pytest.mark.parametrize("dtype", DT)
def test_linear_fp4_few_rows(dtype, act):
    """The kernel for few rows rounds x itself: the same bits as from the quantisers' operand, at every workgroup shape, K shorter than a
    tile and longer than the streams' depth; and right against 64 bits."""
    from dsv41_amd import hipkern, quant, w4
    g = gen(21)
    bits = 4 if act == "fp4" else 8
    for M, N, K in ((1, 16, 32), (2, 31, 224), (3, 48, 288), (16, 33, 2016), (1, 640, 8192), (5, 8200, 1280), (16, 17000, 544), (1, 33000, 320), (16, 64, 8192),
                    (7, 100, 12800)):
        codes, scales = rand_w4(g, N, K, 112, 120)
        W = w4.W4(codes.cuda(), scales.cuda())
        assert hipkern.mx_plan(M, N, K, bits) == (3, 0)
        x = randn(g, M, K, dtype=DT[dtype], spread=0.5)
        y = w4.linear_fp4(x.cuda(), W, act=act)
        op = quant.quant_fp4(x.cuda()) if act == "fp4" else quant.quant_fp8_e8m0(x.cuda() if dtype != "fp16" else x.float().cuda())
        assert torch.equal(w4.linear_fp4(op, W, out_dtype=DT[dtype]), y), (M, N, K)
        at = torch.unique(torch.cat([torch.arange(0, N, 61), torch.arange(max(0, N - 20), N)]))
        check_product(y.cpu()[:, at], ref_round(x, act), deq4(codes[at], scales[at]), dtype, act)
    assert hipkern.mx_plan(16, 64, 16384, 8)[0] == 0              # rows that do not fit LDS: tiles
    codes, scales = rand_w4(g, 64, 16384, 112, 120)
    x = randn(g, 16, 16384, dtype=DT[dtype])
    check_product(w4.linear_fp4(x.cuda(), w4.W4(codes.cuda(), scales.cuda()), act="fp8"), ref_round(x, "fp8"), deq4(codes, scales), dtype, "fp8")


@pytest.mark.parametrize("fmt", ["fp4", "fp8"])
def test_linear_fp4_operands(fmt):
    """Operand pairs: the quantisers' own, strided, off alignment, 3-d; the result is that of the tensor they came from."""
    from dsv41_amd import quant, w4
    g = gen(11)
    for K in (1664, 1184, 96):
        W = w4.W4(*[t.cuda() for t in rand_w4(g, 200, K)])
        x = randn(g, 6, 5, K, dtype=torch.bfloat16).cuda()
        codes, scales = quant.quant_fp4(x) if fmt == "fp4" else quant.quant_fp8_e8m0(x)
        want = w4.linear_fp4(x, W, act=fmt)
        assert want.shape == (6, 5, 200)
        assert torch.equal(w4.linear_fp4((codes, scales), W), want)
        assert torch.equal(w4.linear_fp4((codes, scales), W, act=fmt, out_dtype=torch.float32).to(torch.bfloat16), want)
        n = codes.shape[-1]
        wide, ws = torch.full((6, 5, n + 48), 127, dtype=torch.uint8, device="cuda"), torch.full((6, 5, K // 32 + 3), 255, dtype=torch.uint8, device="cuda")   # NaN around them
        wide[..., 9:9 + n], ws[..., 1:1 + K // 32] = codes, scales
        assert torch.equal(w4.linear_fp4((wide[..., 9:9 + n], ws[..., 1:1 + K // 32]), W), want)
        wide[..., :16], wide[..., 16:16 + n], wide[..., 16 + n:] = 127, codes, 127
        assert torch.equal(w4.linear_fp4((wide[..., 16:16 + n], ws[..., 1:1 + K // 32]), W), want)
        few = w4.linear_fp4(x[:2], W, act=fmt)                        # ten rows: the other kernel
        assert torch.equal(w4.linear_fp4((wide[:2, :, 16:16 + n], ws[:2, :, 1:1 + K // 32]), W), few)
        assert torch.equal(w4.linear_fp4((codes[:2], scales[:2]), W), few)
        if fmt == "fp8":
            assert torch.equal(w4.linear_fp4((codes.view(torch.float8_e4m3fn), scales.view(torch.float8_e8m0fnu)), W), want)


@pytest.mark.parametrize("act", ["fp4", "fp8"])
def test_linear_fp4_nan_rows_stay_alone(act):
    """A NaN or an infinity in x reaches its own row only, one in a weight row its own column only; with half a stage of k at the end."""
    from dsv41_amd import w4
    g = gen(12)
    for M, N, K in ((3, 40, 128), (70, 130, 384), (5, 48, 1664)):
        codes, scales = rand_w4(g, N, K)
        scales[7, K // 32 - 1] = 255
        x = randn(g, M, K)
        x[1, K - 1] = math.inf
        x[M - 1, 0] = math.nan
        y = w4.linear_fp4(x.cuda(), w4.W4(codes.cuda(), scales.cuda()), act=act).cpu()
        bad = torch.zeros(M, N, dtype=torch.bool)
        bad[1], bad[M - 1], bad[:, 7] = True, True, True
        assert torch.equal(torch.isnan(y), bad)


def test_linear_fp4_every_tile_at_every_size():
    """The three tile kernels and both operand forms at sizes that the plan would give another one: fewer rows and columns than a tile, one
    tile and a row more, K of one tile, an odd number of tiles and more stages than a ring holds. FP4 products and sums are exact here."""
    from dsv41_amd import _lib, quant, w4
    L = _lib.lib()
    g = gen(22)
    for M, N, K in ((1, 1, 128), (17, 40, 256), (64, 64, 384), (65, 257, 1152), (129, 130, 640), (257, 256, 1280), (300, 515, 2176),
                    (20, 70, 32), (65, 66, 96), (70, 30, 160), (130, 257, 1184), (260, 300, 2144)):
        codes, scales = rand_w4(g, N, K, 120, 124)
        W = w4.W4(codes.cuda(), scales.cuda())
        x = randn(g, M, K, dtype=torch.bfloat16).cuda()
        for fmt in (4, 8):
            c, s = quant.quant_fp4(x) if fmt == 4 else quant.quant_fp8_e8m0(x)
            ws = torch.empty(M * (K + 128) * 2, dtype=torch.uint8, device="cuda")
            out = []
            for plan in (0, 1, 2):
                y, z = (torch.full((M + 1, N), -7.0, device="cuda") for _ in range(2))
                st = torch.cuda.current_stream().cuda_stream
                assert L.dsv41_mx_gemm(W.w4.data_ptr(), W.s4.data_ptr(), N, K, c.data_ptr(), c.stride(0), s.data_ptr(), K // 32, fmt, M, 2, y.data_ptr(), N,
                                       plan, ws.data_ptr(), ws.numel(), st) == 0
                assert L.dsv41_mx_linear(W.w4.data_ptr(), W.s4.data_ptr(), N, K, x.data_ptr(), 0, K, fmt, M, 2, z.data_ptr(), N, plan, ws.data_ptr(),
                                         ws.numel(), st) == 0
                assert torch.equal(y, z) and (y[M] == -7).all()
                out.append(y[:M])
            assert torch.equal(out[0], out[1]) and torch.equal(out[0], out[2])   # the same order of additions
            stages = -(-K // 256)
            ws = torch.full((M * (K + 128) * 2 + -(-M // 64) * -(-N // 64) * (16 + 16384 * stages) + 16,), 255, dtype=torch.uint8, device="cuda")
            for parts in {min(2, stages), stages // 2 + 1, stages}:             # K in parts: sums of another order
                y, z = (torch.full((M + 1, N), -7.0, device="cuda") for _ in range(2))
                assert L.dsv41_mx_gemm(W.w4.data_ptr(), W.s4.data_ptr(), N, K, c.data_ptr(), c.stride(0), s.data_ptr(), K // 32, fmt, M, 2, y.data_ptr(), N,
                                       parts << 4, ws.data_ptr(), ws.numel(), st) == 0
                assert L.dsv41_mx_linear(W.w4.data_ptr(), W.s4.data_ptr(), N, K, x.data_ptr(), 0, K, fmt, M, 2, z.data_ptr(), N, parts << 4, ws.data_ptr(),
                                         ws.numel(), st) == 0
                assert torch.equal(y, z) and (y[M] == -7).all()
                check_product(y[:M], ref_round(x.cpu(), f"fp{fmt}"), deq4(codes, scales), "fp32", f"fp{fmt}")
            check_product(out[0], ref_round(x.cpu(), f"fp{fmt}"), deq4(codes, scales), "fp32", f"fp{fmt}")


@pytest.mark.parametrize("act", ["fp4", "fp8"])
def test_linear_fp4_k_in_parts(act):
    """Few tiles of a long K: the parts' sums are added in one order, whichever of them ends last, in calls one behind the other, on two
    streams at once and in a replayed graph."""
    from dsv41_amd import hipkern, quant, w4
    g = gen(25)
    for M, N, K in ((17, 70, 8192), (100, 1000, 8160), (33, 5120, 7168)):
        assert hipkern.mx_plan(M, N, K, int(act[2]))[0] == 0 and hipkern.mx_parts(M, N, K, int(act[2])) > 1
        codes, scales = rand_w4(g, N, K, 112, 120)
        W = w4.W4(codes.cuda(), scales.cuda())
        x = randn(g, M, K, dtype=torch.bfloat16).cuda()
        op = quant.quant_fp4(x) if act == "fp4" else quant.quant_fp8_e8m0(x)
        want = w4.linear_fp4(x, W, act=act)
        at = torch.unique(torch.cat([torch.arange(0, N, 61), torch.arange(N - 20, N)]))
        check_product(want.cpu()[:, at], ref_round(x.cpu(), act), deq4(codes[at], scales[at]), "bf16", act)
        assert all(torch.equal(w4.linear_fp4(op if i % 2 else x, W, act=act), want) for i in range(20))
        x2 = randn(g, M, K, dtype=torch.bfloat16).cuda()
        want2 = w4.linear_fp4(x2, W, act=act)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        a, b = [], []
        for _ in range(10):
            a.append(w4.linear_fp4(x, W, act=act))
            with torch.cuda.stream(side):
                b.append(w4.linear_fp4(x2, W, act=act))
        torch.cuda.synchronize()
        assert all(torch.equal(y, want) for y in a) and all(torch.equal(y, want2) for y in b)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = [w4.linear_fp4(x, W, act=act), w4.linear_fp4(x2, W, act=act)]
        for seed in range(4):
            x.copy_(randn(gen(200 + seed), M, K, dtype=torch.bfloat16))
            want = w4.linear_fp4(x, W, act=act)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out[0], want) and torch.equal(out[1], want2)


def test_linear_fp4_rows_in_chunks(monkeypatch):
    from dsv41_amd import hipkern, quant, w4
    monkeypatch.setattr(hipkern, "_mx_chunk", lambda nk: 30000)
    W = w4.W4(*[t.cuda() for t in rand_w4(gen(23), 32, 64)])
    x = randn(gen(24), 70001, 64, dtype=torch.bfloat16).cuda()
    y, z = w4.linear_fp4(x, W), w4.linear_fp4(quant.quant_fp4(x), W)
    monkeypatch.undo()
    want = w4.linear_fp4(x, W)
    assert torch.equal(y, want) and torch.equal(z, want)


def test_linear_fp4_x_strides():
    from dsv41_amd import w4
    g = gen(13)
    W = w4.W4(*[t.cuda() for t in rand_w4(g, 96, 256)])
    base = randn(g, 20, 1280, dtype=torch.bfloat16).cuda()
    for x in (base[:, 256:512], base[:, 3:259], base[::3, :256], base[:1, :256].expand(9, 256), base[:, ::5], base.view(4, 5, 1280)[..., 512:768].transpose(0, 1)):
        assert torch.equal(w4.linear_fp4(x, W), w4.linear_fp4(x.clone(memory_format=torch.contiguous_format), W))


def test_w4_layout_and_cat():
    from dsv41_amd import quant, w4
    g = gen(14)
    w = randn(g, 100, 480).cuda()
    W = w4.W4.from_dense(w)
    codes, scales, vals = quant.quant_fp4(w, values=True)
    assert torch.equal(W.bf16().view(torch.int16), vals.view(torch.int16))
    a, b = w4.W4(codes[:48], scales[:48]), w4.W4(codes[48:], scales[48:])
    both = w4.W4.cat([a, b])
    assert both.shape == W.shape and torch.equal(both.w4, W.w4) and torch.equal(both.s4, W.s4)
    x = randn(g, 3, 480).cuda()
    assert torch.equal(w4.linear_fp4(x, both), w4.linear_fp4(x, W))


# --------------------------------------------------------------------------- together, and inside the layer
@pytest.mark.parametrize("act", ["fp4", "fp8"])
def test_block(act):
    """Norm to an operand, product, residual into the next norm: two layers, against 64 bits with the operand's rounding from the kernel."""
    from dsv41_amd import fused, w4
    g = gen(15)
    H, N, M = 1280, 1280, 19
    ws = [rand_w4(g, N, H, 118, 122) for _ in range(2)]
    Ws = [w4.W4(c.cuda(), s.cuda()) for c, s in ws]
    norms = [(1 + 0.2 * torch.randn(H, generator=g)).to(torch.bfloat16) for _ in range(2)]
    x, res = randn(g, M, H, dtype=torch.bfloat16), randn(g, M, H, dtype=torch.bfloat16)
    for (c, s), W, n in zip(ws, Ws, norms):
        codes, scales, r = fused.add_rmsnorm_quant(x.cuda(), res.cuda(), n.cuda(), 1e-6, fmt=act)
        y = w4.linear_fp4((codes, scales), W)
        want_r, v = ref_norm(x, res, n, 1e-6)
        assert torch.equal(r.cpu(), want_r)
        check_operand(codes, scales, v, act)
        e = pow2(scales.cpu().to(torch.int32) - 127).repeat_interleave(32, -1)
        xv = deq4(codes.cpu(), scales.cpu()) if act == "fp4" else codes.cpu().view(torch.float8_e4m3fn).double() * e
        check_product(y, xv, deq4(c, s), "bf16", act)
        x, res = y.cpu(), r.cpu()


def test_linear_w_and_shared_expert_take_w4():
    """w8.linear_w rounds to FP8; a MoE layer with an FP4 shared expert equals the same layer with the dequantised one as bf16, up to the
    rounding of its products (bf16 gate and up, whose FP8 codes may fall the other way; bf16 outputs)."""
    from dsv41_amd import fused, moe, quant, w4, w8
    g = gen(16)
    H, I, E, k = 1024, 384, 8, 2
    dev = "cuda"
    by = lambda *s: torch.randint(0, 256, s, generator=g, dtype=torch.uint8).to(dev)
    sc = lambda *s: torch.randint(118, 122, s, generator=g, dtype=torch.uint8).to(dev)
    ex = moe.ExpertWeights(quant.tile_fp4(by(E, 2 * I, H // 2)), quant.tile_fp4_scales(sc(E, 2 * I, H // 32)), quant.tile_fp4(by(E, H, I // 2)),
                           quant.tile_fp4_scales(sc(E, H, I // 32)), tiled=True)
    W13, W2 = w4.W4(by(2 * I, H // 2), sc(2 * I, H // 32)), w4.W4(by(H, I // 2), sc(H, I // 32))
    gate = torch.randn(E, H, generator=g).to(dev)
    four = moe.MoE(ex, gate, topk=k, swiglu_limit=10.0, sh_w13=W13, sh_w2=W2)
    dense = moe.MoE(ex, gate, topk=k, swiglu_limit=10.0, sh_w13=W13.bf16(), sh_w2=W2.bf16())
    for T in (1, 5, 16, 40):
        x = randn(g, T, H, dtype=torch.bfloat16).to(dev)
        xq = quant.fake_quant_fp8(x)
        assert torch.equal(w8.linear_w(x, W13), w4.linear_fp4(xq, W13, act="fp8"))
        h = fused.swiglu_quant(w8.linear_w(xq, W13), None, I, 10.0)
        assert torch.equal(w8.linear_w(h, W2), w4.linear_fp4(h.clone(), W2, act="fp8"))
        a, b = four(x), dense(x)
        d = (a.double() - b.double()).norm() / b.double().norm()
        assert d <= 2.0 ** -7, d
        eid, wt = four.last_routing
        via = moe.moe_experts(xq, eid, wt, ex, 10.0, out=torch.empty_like(x), shared=(W13, W2)) if T <= 16 else a
        assert (via.double() - a.double()).norm() <= 2.0 ** -8 * a.double().norm()


def test_offload_layers_take_an_fp4_shared_expert():
    """OffloadMoE at decode and prefill sizes against the same layer with the dequantised shared expert; its runtime's captured graphs against
    its eager form."""
    from dsv41_amd import moe, offload, quant, w4
    g = gen(18)
    H, I, E, k = 1024, 384, 8, 2
    by = lambda *s: torch.randint(0, 256, s, generator=g, dtype=torch.uint8).cuda()
    sc = lambda *s: torch.randint(118, 122, s, generator=g, dtype=torch.uint8).cuda()
    host = offload.HostExpertWeights.of(moe.ExpertWeights(quant.tile_fp4(by(E, 2 * I, H // 2)), quant.tile_fp4_scales(sc(E, 2 * I, H // 32)),
                                                          quant.tile_fp4(by(E, H, I // 2)), quant.tile_fp4_scales(sc(E, H, I // 32)), tiled=True))
    W13, W2 = w4.W4(by(2 * I, H // 2), sc(2 * I, H // 32)), w4.W4(by(H, I // 2), sc(H, I // 32))
    gate = torch.randn(E, H, generator=g).cuda()
    make = lambda a, b, i=0: offload.OffloadMoE(host, gate, topk=k, swiglu_limit=10.0, sh_w13=a, sh_w2=b, device="cuda", layer_id=i)
    four, dense = make(W13, W2), make(W13.bf16(), W2.bf16())
    for T in (1, 33):
        x = randn(g, T, H, dtype=torch.bfloat16).cuda()
        a, b = four(x).double(), dense(x).double()
        assert (a - b).norm() <= 2.0 ** -7 * b.norm()
    layers = [four, make(W13, W2, 1)]
    eager, graphs = (offload.OffloadDecodeRuntime(layers, use_graphs=u) for u in (False, True))
    graphs.capture()
    for t in range(3):
        x = randn(g, 1, H, dtype=torch.bfloat16).cuda()
        assert torch.equal(eager.step(x).clone(), graphs.step(x).clone())


def test_streams_and_graph():
    """On another stream than the inputs' own, and captured and replayed with new inputs: equal to the eager calls."""
    from dsv41_amd import fused, w4
    g = gen(17)
    W = w4.W4(*[t.cuda() for t in rand_w4(g, 640, 1280)])
    n = randn(g, 1280, dtype=torch.bfloat16).cuda()
    x, res = randn(g, 24, 1280, dtype=torch.bfloat16).cuda(), randn(g, 24, 1280, dtype=torch.bfloat16).cuda()

    def step():
        c, s, r = fused.add_rmsnorm_quant(x, res, n, 1e-6, fmt="fp4")
        return w4.linear_fp4((c, s), W), w4.linear_fp4(x, W, act="fp8"), w4.linear_fp4(x[:1], W), r

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(4):
        x.copy_(randn(gen(100 + seed), 24, 1280, dtype=torch.bfloat16))
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, out))


def test_add_rmsnorm_quant_refuses_the_weight_as_output():
    """One row: `out` of the weight's shape may be x or the residual, not the weight, which is left as it was."""
    from dsv41_amd import fused
    g = gen(41)
    x, res, w = (randn(g, *s, dtype=torch.bfloat16).cuda() for s in ((1, 5120), (1, 5120), (5120,)))
    keep, want = w.clone(), fused.add_rmsnorm_quant(x, res, w, 1e-6)
    with pytest.raises(ValueError, match="overlaps"):
        fused.add_rmsnorm_quant(x, res, w, 1e-6, out=w.view(1, 5120))
    assert torch.equal(w, keep)
    assert all(torch.equal(a, b) for a, b in zip(want, fused.add_rmsnorm_quant(x, res, w, 1e-6, out=x)))


def test_add_rmsnorm_quant_output_drops_an_fp8_record():
    """swiglu_quant's result carries its FP8 codes; a norm that writes r over it drops them, so that a product of r is r's."""
    from dsv41_amd import fused, quant, w4, w8
    g = gen(42)
    W = w4.W4(*[t.cuda() for t in rand_w4(g, 96, 256)])
    res, n = randn(g, 9, 256, dtype=torch.bfloat16).cuda(), randn(g, 256, dtype=torch.bfloat16).cuda()
    h = fused.swiglu_quant(randn(g, 9, 512).cuda(), None, 256, 10.0)
    old = w4.linear_fp4(h, W, act="fp8")
    assert quant.attached_codes(h, False) is not None
    want = fused.add_rmsnorm_quant(h.clone(), res, n, 1e-6)
    got = fused.add_rmsnorm_quant(h, res, n, 1e-6, out=h)
    assert got[2] is h and all(torch.equal(a, b) for a, b in zip(want, got)) and quant.attached_codes(h, False) is None
    y = w4.linear_fp4(want[2], W, act="fp8")
    assert torch.equal(w4.linear_fp4(h, W, act="fp8"), y) and torch.equal(w8.linear_w(h, W), y) and not torch.equal(y, old)


@pytest.mark.parametrize("fmt", [4, 8])
@pytest.mark.parametrize("dtype", DT)
def test_c_quantiser_both_formats_and_padding(dtype, fmt):
    """dsv41_mx_quant as a C caller has it: E2M1 and E4M3 codes of strided rows, columns K .. Kp - 1 as zero codes under a zero group's scale
    byte, groups that are not finite marked, scale borders, and nothing written behind the last row."""
    from dsv41_amd import _lib, quant
    t = DT[dtype]
    for rows, K, Kp in ((1, 32, 32), (5, 96, 128), (33, 1184, 1280), (300, 160, 160), (7, 64, 512)):
        x = randn(gen(51 + rows), rows, K, dtype=t, spread=2.0)
        if rows > 4:
            x[0, 3], x[1, K - 1], x[2, 0], x[3, :32] = math.nan, math.inf, -math.inf, 0
            top = torch.tensor(448.0 if fmt == 8 else 6.0, dtype=t)
            x[4, :64] = 0
            x[4, 5], x[4, 40] = top, -torch.nextafter(top, 2 * top)          # the largest code, and a step above: the next scale
        wide = torch.empty(rows, K + 16, dtype=t, device="cuda").normal_()
        wide[:, 8:8 + K] = x.cuda()
        codes = torch.full((rows + 1, Kp * fmt // 8), 0xA5, dtype=torch.uint8, device="cuda")
        scales = torch.full((rows + 1, Kp // 32), 0xA5, dtype=torch.uint8, device="cuda")
        assert wide[:, 8:].data_ptr() % 16 == 0
        assert _lib.lib().dsv41_mx_quant(wide[:, 8:].data_ptr(), list(DT).index(dtype), rows, K, K + 16, fmt, Kp, codes.data_ptr(), scales.data_ptr(), None,
                                         torch.cuda.current_stream().cuda_stream) == 0
        assert (codes[rows] == 0xA5).all() and (scales[rows] == 0xA5).all()
        codes, scales = codes[:rows].cpu(), scales[:rows].cpu()
        bad = ~torch.isfinite(x.float()).reshape(rows, -1, 32).all(-1)
        if fmt == 4:
            code, byte, _ = ref_fp4(x)                                       # groups that are not finite: code 0, byte 255
            want, zero = pack(code), 1
        else:
            ok = torch.where(bad.repeat_interleave(32, -1), torch.zeros((), dtype=t), x)
            want, byte = (a.cpu() for a in quant.quant_fp8_e8m0(ok.float().cuda()))
            q = ref_fp8(ok.double())
            assert torch.equal(want.view(torch.float8_e4m3fn).double(), q[0]) and torch.equal(byte, q[1])
            want[bad.repeat_interleave(32, -1)], byte[bad], zero = 0x7F, 255, 105   # 105: e of the floor, 1e-4 <= 448 * 2^-22
        assert bad.sum() == (0 if rows <= 4 else 3)
        n = K * fmt // 8
        assert torch.equal(codes[:, :n], want) and not codes[:, n:].any()
        assert torch.equal(scales[:, :K // 32], byte) and (scales[:, K // 32:] == zero).all()
