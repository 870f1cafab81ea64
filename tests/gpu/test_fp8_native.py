"""Native 8-bit quantisation (bit for bit) and products (bounds from the arithmetic)."""

from __future__ import annotations

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover - collected on CPU, skipped there
    pytest.skip("needs CUDA", allow_module_level=True)

from mia_train_b200.ops import _native  # noqa: E402
from mia_train_b200.ops.fp8 import (  # noqa: E402
    BLOCK, Fp8Matrix, _empty, _quantize, fp8_gemm, fp8_linear, quantize_fp8, quantize_reference,
)
from mia_train_b200.ops.linear import ACT_GELU, gelu_grad_reference  # noqa: E402

DEV = torch.device("cuda", 0)
E4M3, E5M2 = torch.float8_e4m3fn, torch.float8_e5m2
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(params=[0, 1], ids=["128x128", "256x256"])
def tile(request):
    previous = _native.native().set_fp8_tile(request.param)
    yield request.param
    _native.native().set_fp8_tile(previous)


def _no_errors():
    torch.cuda.synchronize()
    assert _native.native().check_errors(0) == 0


def _loud(r, c, dtype=F32, seed=0):
    torch.manual_seed(seed)
    x = torch.randn(r, c, device=DEV) * torch.exp(torch.randn(r, 1, device=DEV)) * torch.exp(torch.randn(c, device=DEV))
    return x.to(dtype)


def _same(q: Fp8Matrix, ref: Fp8Matrix):
    assert (q.rows, q.cols, q.block_rows) == (ref.rows, ref.cols, ref.block_rows)
    assert torch.equal(q.scale.nan_to_num(-1.0), ref.scale.nan_to_num(-1.0))
    a, b = q.data[:, :q.cols].view(torch.uint8), ref.data[:, :q.cols].view(torch.uint8)
    nan = ref.data[:, :q.cols].float().isnan()
    assert torch.equal(a.masked_fill(nan, 0), b.masked_fill(nan, 0))
    assert torch.equal(q.data[:, :q.cols].float().isnan(), nan)


SHAPES = [(1, 1), (1, 16), (7, 128), (128, 7), (129, 136), (200, 300), (513, 384), (33, 1029)]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("block", [1, BLOCK])
def test_quantise_both_ways(shape, block, dtype):
    x = _loud(*shape, dtype)
    for fmt in (E4M3, E5M2):
        q, qt = _quantize(x, block, fmt, True, True)
        _same(q, quantize_reference(x, block, fmt))
        _same(qt, quantize_reference(x.t(), block, fmt))
        _same(_quantize(x, block, fmt, True, False)[0], quantize_reference(x, block, fmt))
        if block == 1:
            _same(_quantize(x, block, fmt, False, True)[1], quantize_reference(x.t(), block, fmt))


def test_quantise_strides_and_alignment():
    base = _loud(64, 400, BF16)
    for x in (base[:, 8:208], base[:, 3:150], base[1:33:2, :], base.t().contiguous().t()):
        _same(quantize_fp8(x), quantize_reference(x.contiguous(), 1, E4M3))
    flat = torch.randn(64 * 72 + 1, device=DEV)[1:].view(64, 72)  # 4-byte aligned
    _same(quantize_fp8(flat, block_rows=BLOCK), quantize_reference(flat, BLOCK, E4M3))


def test_quantise_borders_and_non_finite():
    x = torch.zeros(6, 260, device=DEV)
    x[0, 0], x[1, 0], x[2, 0], x[3, 0], x[4, 130], x[5, 259] = 448.0, 448.00006, 2.0**-140, 3e38, float("nan"), float("inf")
    x[0, 1:5] = torch.tensor([17.0, 19.0, 2.0**-10, 1.5 * 2.0**-9])  # ties and subnormals
    q, qt = _quantize(x, 1, E4M3, True, True)
    _same(q, quantize_reference(x, 1, E4M3))
    _same(qt, quantize_reference(x.t(), 1, E4M3))


@pytest.mark.parametrize("shape", [(1, 8), (130, 136), (257, 40), (300, 33)])
def test_quantise_gradient_with_factors_and_sums(shape):
    r, c = shape
    dy, pre, gamma = _loud(r, c, BF16), torch.randn(r, c, device=DEV).bfloat16(), torch.rand(c, device=DEV)
    sums = torch.ones(c, device=DEV)
    _quantize(dy, 1, E4M3, False, False, sums=sums)
    exact = dy.double().sum(0)
    bound = (128 + 8 + r / 128) * 2.0**-24 * dy.double().abs().sum(0)  # adds along the longest chain
    assert ((sums.double() - exact).abs() <= bound).all()
    before = sums.clone()
    q, qt = _quantize(dy, 1, E4M3, True, True, aux=pre, gamma=gamma, sums=sums, accumulate=True)
    v = dy.double() * gelu_grad_reference(pre).double() * gamma.double()
    # the kernel's GELU derivative is off by 3e-6 absolute at most; then half a step of e4m3
    slack = 2.0**-4 * v.abs() + (1 + 2.0**-4) * 4e-6 * dy.double().abs() * gamma.double()
    for got, want, s in ((q.dequantize(), v, q.scale), (qt.dequantize().t(), v, qt.scale)):
        full = s.repeat_interleave(BLOCK, 0)
        full = full[:c].t() if got.shape == (r, c) and s is q.scale else full[:r]
        assert ((got.double() - want).abs() <= slack + full.double() * 2.0**-10 + 2.0**-126).all()
    total = (dy.double().abs() * gamma.double()).sum(0)
    assert ((sums.double() - before.double() - v.sum(0)).abs() <= (4e-6 + (140 + r / 128) * 2.0**-24 * 1.2) * total
            + 2.0**-23 * (before.double().abs() + v.sum(0).abs())).all()


def test_quantise_writes_only_its_outputs():
    x = _loud(70, 90, BF16)
    big = torch.full((72, 96), 0x55, device=DEV, dtype=torch.uint8)
    scale = torch.full((2, 72), 7.0, device=DEV)
    q = big[1:71].view(E4M3)
    _native.native().fp8_quantize(x, None, None, False, False, q, scale[:1, :70], None, None, None, False)
    assert (big[0] == 0x55).all() and (big[71] == 0x55).all() and (scale[1] == 7).all() and (scale[0, 70:] == 7).all()


def _product_bound(a: torch.Tensor, b: torch.Tensor, k: int) -> torch.Tensor:
    """Products of 8-bit values are exact; sums of 128 may be truncated to fp32 at every add (one step,
    2^-23), the blocks are added with one rounding each, and two scales are powers of two."""
    return (BLOCK + -(-k // BLOCK)) * 2.0**-23 * (a.double().abs() @ b.double().abs().t())


def _operands(m, n, k, b_block, fa=E4M3, fb=E4M3):
    a = _quantize(_loud(m, k, BF16, 1), 1, fa, True, False)[0]
    b = _quantize(_loud(n, k, BF16, 2), BLOCK if b_block else 1, fb, True, False)[0]
    return a, b


# the last has several tiles per SM and many K blocks
GEMMS = [(1, 1, 1), (1, 8, 16), (5, 33, 130), (128, 128, 128), (129, 257, 384), (300, 520, 1000), (64, 1024, 2048),
         (1029, 640, 1712), (2048, 512, 256), (31, 4096, 512), (700, 1283, 77), (512, 768, 4100), (5120, 1280, 16384)]


@pytest.mark.parametrize("b_block", [True, False])
@pytest.mark.parametrize("m,n,k", GEMMS)
def test_products(m, n, k, b_block, tile):
    a, b = _operands(m, n, k, b_block)
    da, db = a.dequantize(), b.dequantize()
    exact = da.double() @ db.double().t()
    y = fp8_gemm(a, b, out_dtype=F32)
    assert ((y.double() - exact).abs() <= _product_bound(da, db, k)).all()
    z = fp8_gemm(a, b)
    assert ((z.double() - exact).abs() <= _product_bound(da, db, k) * 1.01 + exact.abs() * 2.0**-8 * 1.01).all()
    _no_errors()


@pytest.mark.parametrize("fa,fb", [(E4M3, E5M2), (E5M2, E4M3), (E5M2, E5M2)])
@pytest.mark.parametrize("b_block", [True, False])
def test_product_formats(fa, fb, b_block, tile):
    a, b = _operands(200, 264, 400, b_block, fa, fb)
    da, db = a.dequantize(), b.dequantize()
    y = fp8_gemm(a, b, out_dtype=F32)
    assert ((y.double() - da.double() @ db.double().t()).abs() <= _product_bound(da, db, 400)).all()
    _no_errors()


def test_block_scales_of_the_left_operand(tile):
    a = quantize_fp8(_loud(300, 256, BF16, 1), block_rows=BLOCK)
    b = quantize_fp8(_loud(200, 256, BF16, 2))
    da, db = a.dequantize(), b.dequantize()
    for left, right, x, y in ((a, b, da, db), (a, a, da, da)):
        got = fp8_gemm(left, right, out_dtype=F32)
        assert ((got.double() - x.double() @ y.double().t()).abs() <= _product_bound(x, y, 256)).all()


@pytest.mark.parametrize("m,n,k", [(130, 264, 300), (70, 77, 200), (1030, 1544, 640)])
@pytest.mark.parametrize("b_block", [True, False])
def test_epilogue(m, n, k, b_block, tile):
    a, b = _operands(m, n, k, b_block)
    torch.manual_seed(3)
    bias, gamma = torch.randn(n, device=DEV), torch.rand(n, device=DEV)
    res = torch.randn(m, n, device=DEV).bfloat16()
    da, db = a.dequantize(), b.dequantize()
    acc = da.double() @ db.double().t() + bias.double()
    slack = _product_bound(da, db, k) * 1.2 + acc.abs() * 2.0**-22  # |gelu'| < 1.13
    pre = torch.empty(m, n, device=DEV, dtype=BF16)
    y = fp8_gemm(a, b, bias=bias, act=ACT_GELU, gamma=gamma, residual=res, aux_out=pre)
    assert ((pre.double() - acc).abs() <= slack + acc.abs() * 2.0**-8 * 1.01).all()
    want = res.double() + gamma.double() * F.gelu(acc)
    assert ((y.double() - want).abs() <= slack + 4e-6 * (1 + acc.abs()) + want.abs() * 2.0**-8 * 1.01).all()
    out = torch.randn(m, n, device=DEV)
    base = out.clone()
    fp8_gemm(a, b, out=out, accumulate=True)
    want = base.double() + acc - bias.double()
    assert ((out.double() - want).abs() <= slack + (want.abs() + base.double().abs() + acc.abs() + bias.double().abs()) * 2.0**-23).all()
    _no_errors()


@pytest.mark.parametrize("b_block", [True, False])
def test_epilogue_over_many_tiles(b_block, tile):
    """Several tiles an SM through each form of the epilogue: the staging buffers are used again and again."""
    m, n, k = 4096, 2568, 256
    a, b = _operands(m, n, k, b_block)
    torch.manual_seed(5)
    bias, gamma, res = torch.randn(n, device=DEV), torch.rand(n, device=DEV), torch.randn(m, n, device=DEV).bfloat16()
    da, db = a.dequantize(), b.dequantize()
    acc = da.double() @ db.double().t() + bias.double()
    slack = _product_bound(da, db, k) * 1.2 + acc.abs() * 2.0**-22
    pre = torch.empty(m, n, device=DEV, dtype=BF16)
    y = fp8_gemm(a, b, bias=bias, act=ACT_GELU, aux_out=pre)
    assert ((pre.double() - acc).abs() <= slack + acc.abs() * 2.0**-8 * 1.01).all()
    assert ((y.double() - F.gelu(acc)).abs() <= slack + 4e-6 * (1 + acc.abs()) + F.gelu(acc).abs() * 2.0**-8 * 1.01).all()
    y = fp8_gemm(a, b, bias=bias, gamma=gamma, residual=res)
    want = res.double() + gamma.double() * acc
    assert ((y.double() - want).abs() <= slack + want.abs() * 2.0**-8 * 1.01 + (res.double().abs() + acc.abs()) * 2.0**-23).all()
    out = torch.ones(m, n, device=DEV)
    fp8_gemm(a, b, out=out, accumulate=True)
    want = 1 + acc - bias.double()
    assert ((out.double() - want).abs() <= slack + (want.abs() + acc.abs() + bias.double().abs() + 1) * 2.0**-23).all()
    _no_errors()


def test_long_sum_into_few_tiles(tile):
    """The two halves of K that fill the SMs: same numbers on every run, and no halves when adding to a gradient."""
    a, b = _operands(640, 520, 8200, False)
    da, db = a.dequantize(), b.dequantize()
    exact = da.double() @ db.double().t()
    first = fp8_gemm(a, b, out_dtype=F32)
    assert ((first.double() - exact).abs() <= _product_bound(da, db, 8200)).all()
    assert all(torch.equal(fp8_gemm(a, b, out_dtype=F32), first) for _ in range(4))
    sums = [fp8_gemm(a, b, out=torch.ones(640, 520, device=DEV), accumulate=True) for _ in range(4)]
    assert all(torch.equal(s, sums[0]) for s in sums)
    assert ((sums[0].double() - 1 - exact).abs() <= _product_bound(da, db, 8200) + (1 + exact.abs()) * 2.0**-23).all()
    _no_errors()


def test_extreme_scales_and_non_finite_blocks(tile):
    x = torch.ones(130, 300, device=DEV)
    x[1] *= 2.0**100
    x[2] *= 2.0**-120
    x[3, 140] = float("nan")
    w = torch.ones(140, 300, device=DEV)
    w[:, 128:256] = 0
    for block in (1, BLOCK):
        y = fp8_gemm(quantize_fp8(x), quantize_fp8(w, block_rows=block), out_dtype=F32)
        assert (y[0] == 172).all() and (y[1] == 172 * 2.0**100).all() and (y[2] == 172 * 2.0**-120).all()
        assert y[3].isnan().all() and y[4:].isfinite().all()
    huge = torch.full((8, 128), 2.0**125, device=DEV)
    z = fp8_gemm(quantize_fp8(huge), quantize_fp8(torch.zeros(8, 128, device=DEV)), out_dtype=F32)
    assert (z == 0).all()
    pair = torch.zeros(8, 128, device=DEV)
    pair[:, 0], pair[:, 1] = 2.0**125, 0
    other = torch.zeros(8, 128, device=DEV)
    other[:, 1] = 2.0**125
    for block in (1, BLOCK):
        assert (fp8_gemm(quantize_fp8(pair), quantize_fp8(other, block_rows=block), out_dtype=F32) == 0).all()


def test_writes_only_its_output(tile):
    a, b = _operands(130, 72, 200, True)
    out = torch.full((134, 72), 7.0, device=DEV, dtype=BF16)
    fp8_gemm(a, b, out=out[2:132])
    assert (out[:2] == 7).all() and (out[132:] == 7).all()
    _no_errors()


def test_strided_scales_are_taken():
    a, b = _operands(40, 77, 300, False)
    wide = torch.full((3, 90), float("nan"), device=DEV)
    wide[:, :77] = b.scale
    assert torch.equal(fp8_gemm(a, b), fp8_gemm(a, Fp8Matrix(b.data, wide[:, :77], b.cols, 1)))


def test_repeats_are_identical(tile):
    # the last size gives every SM several tiles
    for m, n, k in ((1000, 776, 1536), (8192, 1280, 5120)):
        for b_block in (False, True):
            a, b = _operands(m, n, k, b_block)
            first = fp8_gemm(a, b, out_dtype=F32)
            assert all(torch.equal(fp8_gemm(a, b, out_dtype=F32), first) for _ in range(5))


@pytest.mark.parametrize("m,k,n", [(1, 384, 384), (9, 40, 33), (257, 384, 1536), (2048, 1024, 512), (1541, 392, 77)])
def test_linear_and_gradients(m, k, n):
    x, w = _loud(m, k, BF16, 3).requires_grad_(True), (_loud(n, k, F32, 4) / k**0.5).requires_grad_(True)
    b = torch.randn(n, device=DEV, requires_grad=True)
    dy = _loud(m, n, BF16, 5)
    y = fp8_linear(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    q = lambda t, rows: quantize_reference(t.detach(), rows, E4M3).dequantize().double()  # noqa: E731
    xq, wq, xt, dyq, dyt = q(x, 1), q(w, BLOCK), q(x.t(), 1), q(dy, 1), q(dy.t(), 1)
    for got, l, r, extra, kk in ((y, xq, wq, b.detach().double(), k), (dx, dyq, wq.t(), 0.0, n), (dw, dyt, xt, 0.0, m)):
        exact = l @ r.t() + extra
        unit = 2.0**-8 * 1.01 if got.dtype == BF16 else 2.0**-23
        assert ((got.detach().double() - exact).abs() <= 1.01 * _product_bound(l, r, kk) + exact.abs() * unit).all()
    assert ((db.double() - dy.double().sum(0)).abs() <= (140 + m / 128) * 2.0**-24 * dy.double().abs().sum(0)).all()
    _no_errors()


def test_linear_matches_the_cpu():
    torch.manual_seed(7)
    x, w, b = torch.randn(2, 65, 200).bfloat16(), torch.randn(136, 200) / 14, torch.randn(136)
    res, g, dy = torch.randn(2, 65, 136).bfloat16(), torch.rand(136), torch.randn(2, 65, 136).bfloat16()

    def run(dev):
        leaves = [t.to(dev).requires_grad_(True) for t in (x, w, b, res, g)]
        y = fp8_linear(leaves[0], leaves[1], leaves[2], activation="gelu", residual=leaves[3], gamma=leaves[4])
        return [y, *torch.autograd.grad(y, leaves, dy.to(dev))]

    for got, want in zip(run(DEV), run("cpu"), strict=True):
        # GELU' differs by 3e-6, which can move a quantised gradient by one e4m3 step (2^-3) now and then
        assert (got.cpu().double() - want.double()).norm() <= 2.0**-8 * want.double().norm()


def test_autocast_and_fp32():
    x, w = torch.randn(40, 64, device=DEV), torch.randn(48, 64, device=DEV)
    assert fp8_linear(x, w).dtype == F32
    y = fp8_linear(x, w, activation="gelu", residual=torch.ones(40, 48, device=DEV), gamma=torch.ones(48, device=DEV))
    h = quantize_reference(x, 1, E4M3).dequantize() @ quantize_reference(w, BLOCK, E4M3).dequantize().t()
    torch.testing.assert_close(y, 1 + F.gelu(h), rtol=1e-4, atol=1e-4)
    with torch.autocast("cuda", dtype=BF16):
        assert fp8_linear(x, w).dtype == BF16


def test_shadow_is_read_and_main_grad_written():
    torch.manual_seed(8)
    x, dy = torch.randn(300, 64, device=DEV).bfloat16(), torch.randn(300, 72, device=DEV).bfloat16()
    w = torch.nn.Parameter(torch.randn(72, 64, device=DEV))
    b = torch.nn.Parameter(torch.randn(72, device=DEV))
    dw, db = torch.autograd.grad(fp8_linear(x, w, b), (w, b), dy)
    w.main_grad, b.main_grad = torch.ones_like(w), torch.ones_like(b)
    shadow = torch.randn(72, 64, device=DEV).bfloat16()
    w._mia_shadow = shadow
    y = fp8_linear(x, w, b)
    y.backward(dy)
    assert torch.equal(y, fp8_linear(x, shadow, b.detach()))
    torch.testing.assert_close(w.main_grad, dw + 1, rtol=2.0**-22, atol=2.0**-22)
    torch.testing.assert_close(b.main_grad, db + 1, rtol=2.0**-22, atol=2.0**-22)


def test_captured_and_replayed_with_new_inputs():
    x, w = torch.randn(200, 256, device=DEV).bfloat16().requires_grad_(True), torch.randn(136, 256, device=DEV, requires_grad=True)
    dy = torch.randn(200, 136, device=DEV).bfloat16()

    def step():
        y = fp8_linear(x, w)
        return y.detach(), *torch.autograd.grad(y, (x, w), dy)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    g, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    with torch.cuda.graph(g2):
        out2 = step()
    with torch.no_grad():
        x.copy_(torch.randn(200, 256, device=DEV))
    g.replay()
    g2.replay()
    torch.cuda.synchronize()
    for a, b, e in zip(out, out2, step(), strict=True):
        assert torch.equal(a, e) and torch.equal(b, e)
    _no_errors()


def test_side_streams_run_apart():
    a, b = _operands(700, 512, 1024, True)
    want = fp8_gemm(a, b)
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs.append(fp8_gemm(a, b))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_native_refusals():
    a, b = _operands(16, 24, 128, True)
    out = torch.empty(16, 24, device=DEV, dtype=BF16)
    n = _native.native()
    ok = [a.data, a.scale, False, b.data, b.scale, True, 128, out, None, None, None, None, 0, False]
    n.fp8_gemm(*ok)
    bads = [(0, a.data.float()), (0, a.data.cpu()), (1, a.scale[:, :8]), (1, a.scale.double()), (2, True), (3, b.data[:, :64]),
            (4, b.scale[:0]), (6, 0), (6, 129), (7, out[:8]), (7, out.half()), (8, torch.zeros(23, device=DEV)),
            (9, out.float()), (10, torch.zeros(24, device=DEV).half()), (12, 2)]
    for i, bad in bads:
        args = list(ok)
        args[i] = bad
        with pytest.raises(RuntimeError):
            n.fp8_gemm(*args)
    q = _empty(16, 128, 1, E4M3, DEV)
    x = torch.zeros(16, 128, device=DEV)
    n.fp8_quantize(x, None, None, False, False, q.data, q.scale, None, None, None, False)
    for args in ((x.double(), None, None, False, False, q.data, q.scale), (x, None, None, True, False, q.data, q.scale),
                 (x, None, None, False, True, q.data, q.scale), (x, None, None, False, False, q.data[:8], q.scale),
                 (x, x, None, False, False, q.data, q.scale), (x, None, x[0, :5], False, False, q.data, q.scale),
                 (x[:, :100], None, None, False, False, q.data, q.scale), (x, None, x[0], False, False, q.data, q.scale)):
        with pytest.raises(RuntimeError):
            n.fp8_quantize(*args, None, None, None, False)
