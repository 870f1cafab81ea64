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
