"""The microscaled dense operators without a GPU: the stored order of W4, what the Python entry points refuse, and what the C entries
refuse before any launch."""
import ctypes
import os

import pytest
import torch


def rand_w4(N, K, seed=0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randint(0, 256, (N, K // 2), generator=g, dtype=torch.uint8), torch.randint(0, 256, (N, K // 32), generator=g, dtype=torch.uint8))


@pytest.mark.parametrize("N,K", [(1, 32), (16, 256), (17, 288), (100, 1184), (48, 5120)])
def test_w4_stored_order(N, K):
    """Every code and scale byte is where the kernels look for it, the padding is zero, and natural() gives the bytes back."""
    from dsv41_amd import w4
    codes, scales = rand_w4(N, K)
    W = w4.W4(codes, scales)
    nb, kb = -(-N // 16), -(-K // 128)
    assert W.shape == (N, K) and W.w4.shape == (nb, kb, 1024) and W.s4.shape == (nb, kb, 64)
    for n in {0, N - 1, N // 2, min(N - 1, 15)}:
        for block in range(K // 32):                              # 32 k: 16 bytes of codes, one scale
            t, b = divmod(block, 4)
            g, s = divmod(b, 2)
            at = s * 512 + g * 256 + (n % 16) * 16
            assert torch.equal(W.w4[n // 16, t, at:at + 16], codes[n, block * 16:block * 16 + 16])
            assert W.s4[n // 16, t, g * 32 + (n % 16) * 2 + s] == scales[n, block]
    assert W.w4.long().sum() == codes.long().sum() and W.s4.long().sum() == scales.long().sum()
    got = W.natural()
    assert torch.equal(got[0], codes) and torch.equal(got[1], scales)


def test_w4_cat_and_refusals():
    from dsv41_amd import w4
    codes, scales = rand_w4(50, 320)
    both = w4.W4.cat([w4.W4(codes[:32], scales[:32]), w4.W4(codes[32:], scales[32:])])
    assert both.shape == (50, 320) and all(torch.equal(a, b) for a, b in zip(both.natural(), (codes, scales)))
    with pytest.raises(ValueError):
        w4.W4.cat([w4.W4(codes[:30], scales[:30]), w4.W4(codes[30:], scales[30:])])   # a tile across two parts
    with pytest.raises(ValueError):
        w4.W4.cat([])
    with pytest.raises(ValueError):
        w4.W4.cat([w4.W4(codes[:32], scales[:32]), w4.W4(*rand_w4(16, 64))])
    with pytest.raises(ValueError):
        w4.W4(codes, scales[:, :-1])
    with pytest.raises(ValueError):
        w4.W4(codes[:, :-8], scales)                              # K % 32
    with pytest.raises(ValueError):
        w4.W4(codes[0], scales[0])
    with pytest.raises(ValueError):
        w4.W4(codes[:0], scales[:0])
    with pytest.raises(ValueError):
        w4.W4.from_dense(torch.zeros(2, 3, 64))


def test_linear_fp4_refusals():
    """Everything wrong is named before a device is asked for; correct calls without a GPU are refused as everywhere in the package."""
    from dsv41_amd import w4
    W = w4.W4(*rand_w4(20, 256))
    x = torch.zeros(3, 256, dtype=torch.bfloat16)
    for bad in (torch.zeros(3, 255, dtype=torch.bfloat16), torch.zeros(3, 128, dtype=torch.bfloat16), torch.tensor(1.0)):
        with pytest.raises(ValueError):
            w4.linear_fp4(bad, W)
    with pytest.raises(TypeError):
        w4.linear_fp4(x.double(), W)
    with pytest.raises(TypeError):
        w4.linear_fp4(x, torch.zeros(20, 256))
    with pytest.raises(TypeError):
        w4.linear_fp4(x, W, out_dtype=torch.float64)
    with pytest.raises(ValueError):
        w4.linear_fp4(x, W, act="int8")
    with pytest.raises(RuntimeError, match="gradient"):
        w4.linear_fp4(x.clone().requires_grad_(), W)
    c8, c4, s = torch.zeros(3, 256, dtype=torch.uint8), torch.zeros(3, 128, dtype=torch.uint8), torch.zeros(3, 8, dtype=torch.uint8)
    for pair in ((c8, s[:, :7]), (c8[:2], s), (c8[:, :200], s), (c8, s, s), (c4, s[:, :4])):
        with pytest.raises(ValueError):
            w4.linear_fp4(pair, W)
    with pytest.raises(ValueError):
        w4.linear_fp4((c8, s), W, act="fp4")
    with pytest.raises(TypeError):
        w4.linear_fp4((c8.int(), s), W)
    with pytest.raises(TypeError):
        w4.linear_fp4((c8, s.float()), W)
    with pytest.raises(TypeError):
        w4.linear_fp4((c8, s), W, out_dtype=torch.int32)
    for call in (lambda: w4.linear_fp4(x, W), lambda: w4.linear_fp4((c8, s), W), lambda: w4.linear_fp4((c4, s), W)):
        with pytest.raises(RuntimeError, match="GPU only"):
            call()


def test_quant_and_norm_refusals():
    from dsv41_amd import fused, quant
    x = torch.zeros(4, 64)
    for bad in (torch.zeros(4, 63), torch.zeros(4, 0), torch.tensor(2.0)):
        with pytest.raises(ValueError):
            quant.quant_fp4(bad)
    with pytest.raises(ValueError):
        quant.quant_fp4(x, block=16)
    for dt in (torch.float64, torch.int8):
        with pytest.raises(TypeError):
            quant.quant_fp4(x.to(dt))
    with pytest.raises(RuntimeError, match="GPU only"):
        quant.quant_fp4(x)
    w = torch.ones(64)
    norm = fused.add_rmsnorm_quant
    with pytest.raises(TypeError):
        norm(x, x.half(), w, 1e-6)
    with pytest.raises(TypeError):
        norm(x, x, w.bfloat16(), 1e-6)
    with pytest.raises(TypeError):
        norm(x.double(), x.double(), w.double(), 1e-6)
    with pytest.raises(TypeError):
        norm(x, x, w, 1e-6, out=torch.zeros(4, 64, dtype=torch.bfloat16))
    for a in ((x[:, :50], x[:, :50], w[:50]), (x, x[:3], w), (x, x, w[:32]), (torch.zeros(1, 32800), None, torch.ones(32800))):
        with pytest.raises(ValueError):
            norm(*a, 1e-6)
    with pytest.raises(ValueError):
        norm(x, x, w, -1.0)
    with pytest.raises(ValueError):
        norm(x, x, w, float("nan"))
    with pytest.raises(ValueError):
        norm(x, x, w, 1e-6, fmt="int8")
    with pytest.raises(ValueError):
        norm(x, None, w, 1e-6, out=torch.zeros(4, 64))
    with pytest.raises(ValueError):
        norm(x, x, w, 1e-6, out=torch.zeros(5, 64))
    for a in ((x.clone().requires_grad_(), x, w), (x, x.clone().requires_grad_(), w), (x, x, w.clone().requires_grad_())):
        with pytest.raises(RuntimeError, match="gradient"):
            norm(*a, 1e-6)
    with pytest.raises(RuntimeError, match="GPU only"):
        norm(x, x, w, 1e-6)


def test_norm_output_overlap():
    """Which outputs count as apart from an input: the same rows, other memory, other columns of the same wider rows."""
    from dsv41_amd.fused import _apart
    buf = torch.zeros(8, 256)
    a = buf[:, :64]
    assert _apart(a, a) and _apart(a, torch.zeros(8, 64)) and _apart(a, buf[:, 64:128]) and _apart(buf[:, 192:], a) and _apart(a[:4], a[4:])
    assert not _apart(a, buf[:, 32:96]) and not _apart(buf[:, 32:96], a) and not _apart(a[1:], a[:-1]) and not _apart(a[:4], a[::2])
    flat = buf.view(-1)[:512].view(8, 64)
    assert not _apart(a, flat) and not _apart(flat, a)


def test_c_entries_refuse_without_launch():
    from dsv41_amd import _lib
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("library not built")
    L = _lib.lib()
    p, q = ctypes.c_void_p(4096), ctypes.c_void_p(4104)

    def quant(x=p, dtype=0, rows=4, K=64, ldx=64, fmt=4, Kp=64, codes=p, scales=p, values=None):
        return L.dsv41_mx_quant(x, dtype, rows, K, ldx, fmt, Kp, codes, scales, values, None)
    assert quant(rows=0) == 0
    for bad in (dict(x=None), dict(codes=None), dict(scales=None), dict(dtype=3), dict(dtype=-1), dict(rows=-1), dict(K=48), dict(K=0), dict(ldx=32),
                dict(fmt=5), dict(Kp=32), dict(Kp=80), dict(ldx=68), dict(x=q), dict(codes=q), dict(values=q), dict(fmt=8, values=p),
                dict(Kp=128, values=p), dict(dtype=2, ldx=66), dict(rows=1 << 50)):
        assert quant(**bad) == -1, bad

    def norm(x=p, ldx=64, res=p, ldr=64, w=p, eps=1e-6, dtype=0, rows=4, K=64, fmt=8, out=p, ldo=64, y=None, codes=p, scales=p):
        return L.dsv41_add_rmsnorm_mx(x, ldx, res, ldr, w, eps, dtype, rows, K, fmt, out, ldo, y, codes, scales, None)
    assert norm(rows=0) == 0
    for bad in (dict(x=None), dict(w=None), dict(codes=None), dict(scales=None), dict(out=None), dict(dtype=3), dict(rows=-1), dict(rows=1 << 32),
                dict(K=48), dict(K=32800, ldx=32800, ldr=32800, ldo=32800), dict(fmt=0), dict(eps=-1.0), dict(eps=float("nan")), dict(ldx=32), dict(ldr=32),
                dict(ldo=32), dict(ldx=68), dict(ldr=68), dict(ldo=68), dict(x=q), dict(res=q), dict(out=q), dict(w=q), dict(y=q)):
        assert norm(**bad) == -1, bad

    def gemm(w=p, s=p, N=64, K=256, xc=p, ldx=256, xs=p, ldxs=8, fmt=8, M=4, out_type=0, y=p, ldy=64, plan=0, ws=p, ws_bytes=1 << 20):
        return L.dsv41_mx_gemm(w, s, N, K, xc, ldx, xs, ldxs, fmt, M, out_type, y, ldy, plan, ws, ws_bytes, None)
    assert gemm(M=0) == 0
    for bad in (dict(w=None), dict(s=None), dict(xc=None), dict(xs=None), dict(y=None), dict(N=0), dict(K=0), dict(K=240), dict(M=-1), dict(fmt=6),
                dict(out_type=3), dict(out_type=-1), dict(ldx=128), dict(ldx=264), dict(ldxs=4), dict(ldxs=7), dict(ldy=63), dict(w=q), dict(xc=q),
                dict(s=q), dict(y=q), dict(plan=99), dict(plan=-1), dict(plan=2 << 4), dict(plan=(2 << 4) + 1, K=512, ldx=512, ldxs=16),
                dict(plan=2 << 4, K=512, ldx=512, ldxs=16, ws_bytes=16 + 32768), dict(plan=2 << 4, N=1 << 30, ldy=1 << 30, K=512, ldx=512, ldxs=16, M=1 << 18), dict(ldx=1 << 22), dict(ldxs=1 << 22),
                dict(plan=3, M=17), dict(plan=3, M=16, K=16384, ldx=16384, ldxs=512), dict(ws=None), dict(ws=q), dict(ws_bytes=31)):
        assert gemm(**bad) == -1, bad

    def linear(w=p, s=p, N=64, K=96, x=p, dtype=0, ldx=96, fmt=8, M=4, out_type=0, y=p, ldy=64, plan=0, ws=p, ws_bytes=1 << 20):
        return L.dsv41_mx_linear(w, s, N, K, x, dtype, ldx, fmt, M, out_type, y, ldy, plan, ws, ws_bytes, None)
    assert linear(M=0) == 0
    for bad in (dict(w=None), dict(s=None), dict(x=None), dict(y=None), dict(ws=None), dict(ws_bytes=4 * 128 + 4 * 4 - 1), dict(ws=q), dict(N=0), dict(K=0),
                dict(K=80), dict(M=-1), dict(fmt=0), dict(dtype=3), dict(out_type=3), dict(ldx=64), dict(ldx=100), dict(ldy=63), dict(x=q), dict(plan=4),
                dict(plan=3, M=17), dict(plan=3, M=16, K=16384, ldx=16384)):
        assert linear(**bad) == -1, bad


@pytest.mark.parametrize("rows", [1, 2])
def test_norm_output_is_never_the_weight(rows):
    """`out` may be x or the residual, not the weight: the kernel reads it after r is written. One row has the weight's own shape."""
    from dsv41_amd import fused
    x, res, w = torch.zeros(rows, 64), torch.zeros(rows, 64), torch.ones(64)
    for out in (x, res):
        assert fused._norm_rows(x, res, w, out, 64)[-1] is out
    buf = torch.ones(4 * 64)
    for w, out in ((w, w.view(1, 64).expand(rows, 64)), (buf[:64], buf[:rows * 64].view(rows, 64)), (buf[32:96], buf[:rows * 64].view(rows, 64))):
        with pytest.raises(ValueError):
            fused._norm_rows(x, res, w, out, 64)


def test_norm_output_counts_as_changed(monkeypatch):
    """`out` is written past torch: its version counter moves, so an FP8 record on it (or on a tensor that it is a view of) is dropped and
    autograd sees the change. Inputs and outputs of the call's own stay as they are."""
    from dsv41_amd import _lib, fused, quant
    monkeypatch.setattr(_lib, "require_cuda", lambda *t: None)
    monkeypatch.setattr(_lib, "launch", lambda *a: None)
    recorded = lambda *s: quant.attach_codes(torch.zeros(*s, dtype=torch.bfloat16), torch.zeros(*s, dtype=torch.uint8),
                                             torch.zeros(*s[:-1], s[-1] // 32, dtype=torch.uint8))
    w = torch.ones(64, dtype=torch.bfloat16)
    for pick in (lambda x, r: x, lambda x, r: r, lambda x, r: x.view(4, 64), lambda x, r: recorded(4, 64)):
        x, res = recorded(4, 64), recorded(4, 64)
        out = pick(x, res)
        base = x if out._base is x else out
        before = {id(t): t._version for t in (x, res, w)}
        assert fused.add_rmsnorm_quant(x, res, w, 1e-6, out=out)[2] is out
        assert quant.attached_codes(base, False) is None
        for t in (x, res, w):
            assert t is base or t._version == before[id(t)] and (t is w or quant.attached_codes(t, False) is not None)
    x, res = recorded(4, 64), recorded(4, 64)
    fused.add_rmsnorm_quant(x, res, w, 1e-6)
    assert quant.attached_codes(x, False) is not None and quant.attached_codes(res, False) is not None
    a = torch.ones(4, 64, dtype=torch.bfloat16, requires_grad=True)
    h = a * 2
    loss = (h * h).sum()
    with torch.no_grad():
        fused.add_rmsnorm_quant(torch.zeros_like(h), h, w, 1e-6, out=h)
    with pytest.raises(RuntimeError, match="inplace operation"):
        loss.backward()
    with torch.inference_mode():
        h = torch.zeros(4, 64, dtype=torch.bfloat16)
        assert fused.add_rmsnorm_quant(h, h, w, 1e-6, out=h)[2] is h


@pytest.mark.parametrize("K", [32, 128, 1024, 131072, (1 << 20) - 32, 1 << 20])
def test_rows_of_a_launch_fit_its_offsets(monkeypatch, K):
    """Every launch of mx_linear and mx_gemm has rows x tiles of 128 k below 2^29 and at most 65535 x 16 rows, at row counts around the
    limits; the launches together are all rows, once."""
    from dsv41_amd import _lib, hipkern
    seen = []
    monkeypatch.setattr(_lib, "launch", lambda dev, name, *a: seen.append((name, a[3], a[8] if name.endswith("linear") else a[9])))
    nk = -(-K // 128)
    limit = min(65535 * 16, ((1 << 29) - 1) // nk)

    class W:
        shape, w4, s4 = (1, K), torch.empty(0), torch.empty(0)
    for M in sorted({1, 17, 65535, 65536, 65537, limit, limit + 1, 2 * limit + 3}):
        for call in (lambda: hipkern.mx_linear(torch.empty(M, K, dtype=torch.bfloat16, device="meta"), 8, W, torch.bfloat16),
                     lambda: hipkern.mx_gemm(torch.empty(M, K, dtype=torch.uint8, device="meta"), torch.empty(M, K // 32, dtype=torch.uint8, device="meta"),
                                             8, W, torch.bfloat16)):
            seen.clear()
            assert call().shape == (M, 1)
            assert sum(rows for _, _, rows in seen) == M and all(k == K and 0 < rows <= limit for _, k, rows in seen), (M, seen)


def test_c_entries_refuse_before_the_operand():
    """Sizes that the product's launch cannot take are refused before the launch that makes its operand. Addresses are never read: a call that
    is let through ends with the runtime's error where there is no GPU, and is not made where there is one."""
    from dsv41_amd import _lib
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("library not built")
    if torch.cuda.is_available():
        pytest.skip("a call that is not refused would launch")
    L = _lib.lib()
    p, big = ctypes.c_void_p(4096), (1 << 62)

    def gemm(N=64, K=256, fmt=8, M=64, plan=0):
        return L.dsv41_mx_gemm(p, p, N, K, p, K * fmt // 8, p, K // 32, fmt, M, 0, p, N, plan, p, big, None)

    def linear(N=64, K=256, fmt=8, M=64, plan=0):
        return L.dsv41_mx_linear(p, p, N, K, p, 0, K, fmt, M, 0, p, N, plan, p, big, None)
    for call in (gemm, linear):
        assert call() > 0                                         # no device
        for fmt in (4, 8):
            for plan in (0, 1, 2):
                assert call(fmt=fmt, plan=plan, M=65536, K=1 << 20) == -1            # rows x tiles of 128 k: 2^29
                assert call(fmt=fmt, plan=plan, M=65535, K=1 << 20) > 0
                assert call(fmt=fmt, plan=plan, M=1 << 19, N=1 << 29, K=32) == -1    # tiles
    assert linear(M=1048561, K=32) == -1 and linear(M=1048560, K=32) > 0             # rows of the rounding's launch


def test_c_entries_refuse_more_weight_rows_than_a_launch_holds():
    """2^29 weight rows: the kernel for few rows would need 2^32 threads, and row counts next to 2^31 would wrap while tiles are counted."""
    from dsv41_amd import _lib
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("library not built")
    if torch.cuda.is_available():
        pytest.skip("a call that is not refused would launch")
    L = _lib.lib()
    p, big = ctypes.c_void_p(4096), (1 << 62)

    def gemm(N, fmt, plan):
        return L.dsv41_mx_gemm(p, p, N, 32, p, 2 * fmt * 4, p, 1, fmt, 1, 0, p, N, plan, p, big, None)

    def linear(N, fmt, plan):
        return L.dsv41_mx_linear(p, p, N, 32, p, 0, 32, fmt, 1, 0, p, N, plan, p, big, None)
    for call in (gemm, linear):
        for fmt in (4, 8):
            assert call((1 << 29) - 128, fmt, 3) > 0              # no device
            assert call(1 << 29, fmt, 3) == -1
            for plan in (0, 1, 2, 3):
                assert call((1 << 31) - 1, fmt, plan) == -1
                assert call((1 << 31) - 64, fmt, plan) == -1


def test_quant_fp4_refuses_a_gradient():
    """Its values would take x's place without a graph. Without grad mode, and for detached weights, there is nothing to lose."""
    from dsv41_amd import quant, w4
    x = torch.zeros(4, 64, requires_grad=True)
    for values in (False, True):
        with pytest.raises(RuntimeError, match="gradient"):
            quant.quant_fp4(x, values=values)
        with torch.no_grad(), pytest.raises(RuntimeError, match="GPU only"):
            quant.quant_fp4(x, values=values)
    with pytest.raises(RuntimeError, match="GPU only"):
        w4.W4.from_dense(x)


def test_norm_refuses_an_output_that_needs_a_gradient():
    from dsv41_amd import fused
    x, w = torch.zeros(4, 64), torch.ones(64)
    for out in (torch.zeros(4, 64, requires_grad=True), torch.zeros(4, 64, requires_grad=True) * 1):
        with pytest.raises(RuntimeError, match="gradient"):
            fused.add_rmsnorm_quant(x, x, w, 1e-6, out=out)
        with torch.no_grad(), pytest.raises(RuntimeError, match="GPU only"):
            fused.add_rmsnorm_quant(x, x, w, 1e-6, out=out)


def _entries():
    """The three entry points as functions of one float matrix [4, 64]."""
    from dsv41_amd import fused, quant, w4, w8
    W, n = w4.W4(*rand_w4(20, 64)), torch.ones(64)
    pair = torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8)
    return {"quant_fp4": lambda x: quant.quant_fp4(x, values=True)[2], "linear_fp4": lambda x: w4.linear_fp4(x, W), "linear_w": lambda x: w8.linear_w(x, W),
            "pair": lambda x: w4.linear_fp4(pair, W) + x[:, :20], "norm": lambda x: fused.add_rmsnorm_quant(x, x, n, 1e-6)[2],
            "norm residual": lambda x: fused.add_rmsnorm_quant(torch.zeros(4, 64), x, n, 1e-6)[2],
            "norm weight": lambda x: fused.add_rmsnorm_quant(torch.zeros(4, 64), None, x[0], 1e-6, y=True)[3],
            "norm out": lambda x: fused.add_rmsnorm_quant(torch.zeros(4, 64), torch.zeros(4, 64), n, 1e-6, out=x)[2]}


@pytest.mark.parametrize("name", ["quant_fp4", "linear_fp4", "linear_w", "norm", "norm residual", "norm weight", "norm out"])
def test_forward_mode_tangents_are_refused(name):
    """A launch would drop an input's tangent; without one, a dual level around the call is nothing to it."""
    import torch.autograd.forward_ad as fwd
    call = _entries()[name]
    with fwd.dual_level():
        x = fwd.make_dual(torch.zeros(4, 64), torch.ones(4, 64))
        with pytest.raises(RuntimeError, match="gradient"):
            call(x)
        with torch.no_grad(), pytest.raises(RuntimeError, match="gradient"):
            call(x)
        with torch.inference_mode(), pytest.raises(RuntimeError, match="GPU only"):
            call(x)
        with pytest.raises(RuntimeError, match="GPU only"):
            call(torch.zeros(4, 64))


@pytest.mark.parametrize("name", ["quant_fp4", "linear_fp4", "linear_w", "pair", "norm"])
def test_traces_are_refused(name):
    """torch's tracers would record the empty outputs and not the launch."""
    from torch.fx.experimental.proxy_tensor import make_fx
    call = _entries()[name]
    for trace in (lambda: torch.jit.trace(call, torch.zeros(4, 64)), lambda: make_fx(call)(torch.zeros(4, 64))):
        with pytest.raises(RuntimeError, match="trace"):
            trace()


def test_w4_pairs_are_no_shared_expert_of_the_decode_launches():
    """The two decode launches read bf16 or FP8 shared experts; moe_experts runs an FP4 pair as launches of its own. Where the launches are
    asked for directly, and in the layers that only know them, a W4 is named instead of failing inside."""
    from dsv41_amd import moe, w4
    W = w4.W4(*rand_w4(32, 64))
    for pair in ((W, W), [W, W], (W, torch.zeros(64, 16)), (torch.zeros(32, 64), W)):
        with pytest.raises(TypeError, match="W4"):
            moe.SharedExpert.of(pair)
    with pytest.raises(TypeError, match="W4"):
        moe.SharedExpert.prepare(W, W)
    bf = moe.SharedExpert.of((torch.zeros(32, 64), torch.zeros(64, 16)))
    assert not bf.tiled and moe.SharedExpert.of(bf) is bf and moe.SharedExpert.of(None) is None


def test_oproj_a_names_w4():
    """The grouped output projection has no FP4 form: the dequantised weights are the caller's choice."""
    from dsv41_amd import w4, w8
    with pytest.raises(TypeError, match="W4"):
        w8.oproj_a(torch.zeros(1, 2, 2, 64, dtype=torch.bfloat16), w4.W4(*rand_w4(32, 64)), 2, 16)


def test_w4_scales_are_bytes():
    """Wider elements would be read as several scale bytes each (fp32 scales of blocks of 128 have just the bytes of E8M0's 32); wider codes
    either hold the same bytes or do not fit the scales."""
    from dsv41_amd import w4
    codes, scales = rand_w4(16, 256)
    for c, s in ((codes, torch.ones(16, 2)), (codes.long(), scales.long()), (codes.to(torch.bfloat16), scales.to(torch.bfloat16)),
                 (codes, scales.view(torch.int32))):
        with pytest.raises(TypeError, match="byte"):
            w4.W4(c, s)
    for c in (codes.long(), torch.zeros(16, 128), torch.zeros(16, 256, dtype=torch.bfloat16)):
        with pytest.raises(ValueError):
            w4.W4(c, scales)
    want = w4.W4(codes, scales)
    for c, s in ((codes.view(torch.int8), scales.view(torch.float8_e8m0fnu)), (codes.view(torch.float4_e2m1fn_x2), scales), (codes.view(torch.int32), scales),
                 (codes, scales.view(torch.int8))):
        W = w4.W4(c, s)
        assert torch.equal(W.w4, want.w4) and torch.equal(W.s4, want.s4)
