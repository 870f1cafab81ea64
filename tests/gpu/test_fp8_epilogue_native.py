"""Epilogues of the native 8-bit product that read what TMA and the tensor core left for a whole warp."""

from __future__ import annotations

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover - collected on CPU, skipped there
    pytest.skip("needs CUDA", allow_module_level=True)

from mia_train_b200.ops import _native  # noqa: E402
from mia_train_b200.ops.fp8 import BLOCK, Fp8Matrix, fp8_gemm, fp8_linear, quantize_fp8  # noqa: E402

DEV = torch.device("cuda", 0)
BF16, F32 = torch.bfloat16, torch.float32
E4M3, E5M2 = torch.float8_e4m3fn, torch.float8_e5m2


@pytest.fixture(params=[0, 1], ids=["128x128", "256x256"])
def tile(request):
    previous = _native.native().set_fp8_tile(request.param)
    yield request.param
    _native.native().set_fp8_tile(previous)


def _no_errors():
    torch.cuda.synchronize()
    assert _native.native().check_errors(0) == 0


@pytest.mark.parametrize("b_block", [True, False])
@pytest.mark.parametrize("m,n,k", [(4096, 2568, 256), (8192, 1280, 1280)])
def test_residual_repeats_are_identical(m, n, k, b_block, tile):
    """Products and residual are integers that every sum holds exactly, so each repeat has one right answer."""
    torch.manual_seed(0)
    a = quantize_fp8(torch.randint(-4, 5, (m, k), device=DEV).float())
    b = quantize_fp8(torch.randint(-4, 5, (n, k), device=DEV).float(), block_rows=BLOCK if b_block else 1)
    res = torch.randint(-128, 129, (m, n), device=DEV).bfloat16()
    want = (a.dequantize().double() @ b.dequantize().double().t() + res.double()).to(BF16)
    for _ in range(8):
        assert torch.equal(fp8_gemm(a, b, residual=res), want)
    _no_errors()


def _product_bound(a, b, k):
    """Products of 8-bit values are exact; sums of 128 may be truncated to fp32 at every add (one step, 2^-23), and
    the blocks are added with one rounding each."""
    return (BLOCK + -(-k // BLOCK)) * 2.0**-23 * (a.double().abs() @ b.double().abs().t())


@pytest.mark.parametrize("fmt", [E4M3, E5M2])
@pytest.mark.parametrize("block", [1, BLOCK])
# one row; ragged K; an odd width (stored by the lanes); several tiles an SM
@pytest.mark.parametrize("m,k,n", [(1, 384, 384), (1, 200, 77), (130, 200, 264), (300, 1712, 77), (4096, 256, 2568)])
def test_weight_quantised_once(m, k, n, block, fmt, tile):
    torch.manual_seed(m + k + n)
    x = (torch.randn(m, k, device=DEV) * torch.exp(torch.randn(k, device=DEV))).to(BF16)
    w = quantize_fp8(torch.randn(n, k, device=DEV) / k**0.5, block_rows=block, dtype=fmt)
    bias, gamma = torch.randn(n, device=DEV), torch.rand(n, device=DEV)
    res = torch.randn(m, n, device=DEV).to(BF16)
    xq, wq = quantize_fp8(x).dequantize(), w.dequantize()
    acc = xq.double() @ wq.double().t() + bias.double()
    base = _product_bound(xq, wq, k) * 1.2 + acc.abs() * 2.0**-22  # |gelu'| < 1.13
    with torch.no_grad():
        for act, g, r in ((None, None, None), (None, gamma, res), ("gelu", None, None), ("gelu", gamma, None),
                          ("gelu", None, res), ("gelu", gamma, res)):
            h = F.gelu(acc) if act else acc
            want = (h if g is None else g.double() * h) + (0 if r is None else r.double())
            # the kernel's GELU is off by 4e-6 absolute at most; one rounding each of product and sum; then bf16's half step
            slack = base + 4e-6 * (1 + acc.abs()) * (act is not None) + (h.abs() + want.abs()) * 2.0**-23
            y = fp8_linear(x, w, bias, activation=act, gamma=g, residual=r)
            assert y.dtype == BF16 and y.shape == (m, n)
            assert ((y.double() - want).abs() <= slack + want.abs() * 2.0**-8 * 1.01).all(), (act, g is None, r is None)
            y = fp8_linear(x.float(), w, bias, activation=act, gamma=g, residual=None if r is None else r.float())
            assert y.dtype == F32 and ((y.double() - want).abs() <= slack).all(), (act, g is None, r is None)
    _no_errors()


def test_weight_quantised_once_under_autocast_and_with_batches():
    torch.manual_seed(4)
    x, w = torch.randn(2, 3, 5, 64, device=DEV), torch.randn(48, 64, device=DEV)
    q = quantize_fp8(w, block_rows=BLOCK)
    res = torch.randn(2, 3, 5, 48, device=DEV)
    with torch.no_grad(), torch.autocast("cuda", dtype=BF16):
        y = fp8_linear(x, q, activation="gelu", residual=res)
        assert y.shape == res.shape and y.dtype == BF16
        assert torch.equal(y, fp8_linear(x, w, activation="gelu", residual=res))
    with pytest.raises(ValueError, match="no backward"):
        fp8_linear(x.requires_grad_(True), q)


def _powers(exponents, cols=128):
    return torch.tensor([2.0**e for e in exponents], device=DEV)[:, None].expand(-1, cols).contiguous()


@pytest.mark.parametrize("block", [1, BLOCK])
def test_row_scales_at_both_ends_of_the_range(block, tile):
    """128 equal products of powers of two are exact whenever they are fp32 numbers, whatever their factors' sizes."""
    rows = [120, 100, 60, 0, -60, -100, -120, -140]
    a = quantize_fp8(_powers(rows))
    for other in rows:
        b = quantize_fp8(_powers([other] * 9 if block == BLOCK else [other, 0, -other if abs(other) < 127 else 0] * 3), block_rows=block)
        want = a.dequantize().double() @ b.dequantize().double().t()
        got = fp8_gemm(a, b, out_dtype=F32).double()
        normal = (want >= 2.0**-126) & (want < 2.0**128)
        assert torch.equal(got[normal], want[normal])
        assert (got[want >= 2.0**128] == float("inf")).all()
        # below the normal numbers: at most half a step of fp32's subnormals for each of the 128 products
        assert ((got - want).abs()[want < 2.0**-126] <= 128 * 2.0**-150).all()
    _no_errors()


@pytest.mark.parametrize("block", [1, BLOCK])
def test_small_sums_under_huge_scales(block, tile):
    """Both blocks' largest values meet zeros; what is left is 2^-18 of a product of scales beyond fp32."""
    a, b = torch.zeros(8, 256, device=DEV), torch.zeros(9, 256, device=DEV)
    a[:, 0], a[:, 1] = 2.0**126, 2.0**109
    b[:, 2], b[:, 1] = 2.0**30, 2.0**13
    a[:, 128:], b[:, 128:] = 2.0**60, 2.0**50  # an ordinary block next to it
    qa, qb = quantize_fp8(a), quantize_fp8(b, block_rows=block)
    assert (qa.scale[0] == 2.0**118).all() and (qb.scale[0] == 2.0**22).all()
    assert (fp8_gemm(qa, qb, out_dtype=F32) == 2.0**122 + 2.0**117).all()
    _no_errors()


@pytest.mark.parametrize("scale_a,scale_b", [(3e38, 1e-30), (1e-30, 3e38), (3e38, 2e-38), (1e-37, 1e30), (-2.5, 1e-3), (0.0, 3e38),
                                              (3e38, 3e38), (1e-44, 1e38)])
@pytest.mark.parametrize("fmt", [E4M3, E5M2])
@pytest.mark.parametrize("block", [1, BLOCK])
def test_any_fp32_scales(block, fmt, scale_a, scale_b, tile):
    """Scales that a caller brings need not be powers of two, nor of one sign."""
    torch.manual_seed(5)
    one = quantize_fp8(torch.ones(140, 300, device=DEV), block_rows=block, dtype=fmt)
    a0 = quantize_fp8(torch.randint(-3, 4, (130, 300), device=DEV).float())
    a = Fp8Matrix(a0.data, torch.full_like(a0.scale, scale_a), 300)
    b = Fp8Matrix(one.data, torch.full_like(one.scale, scale_b), 300, block)
    sums = [(a0.data[:, c:min(c + 128, 300)].double()).sum(1, keepdim=True) * one.data[:, 0].double() for c in (0, 128, 256)]
    fa, fb = (torch.tensor(v, dtype=F32).double().item() for v in (scale_a, scale_b))
    terms = [s * fa * fb for s in sums]
    want, size = sum(terms), sum(t.abs() for t in terms)
    got = fp8_gemm(a, b, out_dtype=F32).double()
    safe = size < 2.0**127
    # two roundings of a term's scales, one of each of three sums
    assert ((got - want).abs()[safe] <= 5 * 2.0**-24 * size[safe] + 2.0**-149).all()
    big = torch.stack([t.abs() for t in terms]).amin(0) >= 2.0**128
    assert not got[big].isfinite().any()
    assert (got[size == 0] == 0).all()
    _no_errors()


@pytest.mark.parametrize("where", [0, 1, 2])
@pytest.mark.parametrize("block", [1, BLOCK])
def test_rows_next_to_a_huge_one_stay_exact(block, where, tile):
    """Row 37 alone meets scales past the range, in one of three blocks; integers elsewhere are summed exactly."""
    torch.manual_seed(6)
    a, b = torch.randint(-4, 5, (300, 384), device=DEV).float(), torch.zeros(72, 384, device=DEV)
    b[:] = torch.randint(-4, 5, (72, 384), device=DEV)
    at = slice(128 * where, 128 * where + 128)
    a[:, at], b[:, at] = 0, 0
    a[37, 128 * where], a[37, 128 * where + 1] = 2.0**126, 2.0**109  # scale 2^118
    b[:, 128 * where + 2], b[:, 128 * where + 1] = 2.0**30, 2.0**13  # scale 2^22
    qa, qb = quantize_fp8(a), quantize_fp8(b, block_rows=block)
    got = fp8_gemm(qa, qb, out_dtype=F32).double()
    want = a.double() @ b.double().t()
    want[37] = 2.0**122  # the integers are below half a step of it
    assert torch.equal(got, want)
    _no_errors()


@pytest.mark.parametrize("first", [True, False])
@pytest.mark.parametrize("fmt", [E4M3, E5M2])
@pytest.mark.parametrize("block", [1, BLOCK])
def test_tiny_blocks_of_a_row_with_huge_ones_count(block, fmt, first, tile):
    """One block's scales multiply beyond fp32 over a zero sum; another's are at the ends of the range and give 32."""
    a, b = torch.zeros(40, 256, device=DEV), torch.zeros(9, 256, device=DEV)
    huge, tiny = (slice(0, 128), slice(128, 256)) if first else (slice(128, 256), slice(0, 128))
    a[:, huge.start], b[:, huge.start + 1] = 2.0**126, 2.0**100
    a[:, tiny], b[:, tiny] = 2.0**-120, 2.0**118
    qa, qb = quantize_fp8(a, dtype=fmt), quantize_fp8(b, block_rows=block, dtype=fmt)
    assert qa.scale.max() * qb.scale.max() == float("inf") and qa.scale.min() == 2.0**-126
    assert (fp8_gemm(qa, qb, out_dtype=F32) == 32).all()
    _no_errors()
