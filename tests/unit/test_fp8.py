"""8-bit quantisation and linear layers on the CPU: scales, rounding, products, gradients, refusals."""

from __future__ import annotations

import math

import pytest
import torch
import torch.nn.functional as F

from mia_train_b200.ops.fp8 import BLOCK, LIMITS, Fp8Matrix, fp8_gemm, fp8_linear, quantize_fp8
from mia_train_b200.ops.linear import ACT_GELU

E4M3, E5M2 = torch.float8_e4m3fn, torch.float8_e5m2


def round_exact(x: torch.Tensor, rows: int, dtype=E4M3) -> torch.Tensor:
    """x on its scaled 8-bit grid, in 64 bits, block by block from the definition."""
    mant, low = (3, -6) if dtype == E4M3 else (2, -14)
    x, out = x.double(), torch.zeros_like(x, dtype=torch.float64)
    for r in range(0, x.shape[0], rows):
        for c in range(0, x.shape[1], BLOCK):
            part = x[r:r + rows, c:c + BLOCK]
            top = part.abs().max().item()
            s = 2.0 ** max(-126, math.ceil(math.log2(top / LIMITS[dtype]))) if top > 0 else 1.0
            while top / s > LIMITS[dtype]:  # guard log2's own rounding
                s *= 2
            v = part / s
            step = torch.exp2((torch.frexp(v)[1].double() - 1).clamp(min=low) - mant)
            out[r:r + rows, c:c + BLOCK] = torch.round(v / step) * step * s
    return out


def _loud(r, c, seed=0):
    torch.manual_seed(seed)
    return torch.randn(r, c) * torch.exp(2 * torch.randn(r, 1)) * torch.exp(torch.randn(c))


@pytest.mark.parametrize("dtype", [E4M3, E5M2])
@pytest.mark.parametrize("rows", [1, BLOCK])
@pytest.mark.parametrize("shape", [(1, 1), (3, 16), (5, 129), (130, 257), (128, 128)])
def test_quantise_is_the_nearest_scaled_value(shape, rows, dtype):
    x = _loud(*shape)
    q = quantize_fp8(x, block_rows=rows, dtype=dtype)
    assert (q.rows, q.cols) == shape and q.data.shape[1] % 16 == 0
    assert torch.equal(q.dequantize().double(), round_exact(x, rows, dtype))
    assert (q.scale.log2() == q.scale.log2().round()).all()


def test_scales_at_the_borders():
    edge = torch.tensor([[448.0], [448.0000305], [224.0], [0.0], [2.0**-140], [3e38]])
    q = quantize_fp8(edge)
    assert q.scale[0].tolist() == [1.0, 2.0, 0.5, 2.0**-126, 2.0**-126, 2.0**120]
    assert (q.dequantize()[[0, 2, 3], 0] == edge[[0, 2, 3], 0]).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_non_finite_block_poisons_its_products_only(bad):
    x = torch.ones(3, 300)
    x[1, 130] = bad
    q = quantize_fp8(x)
    assert q.scale.isnan().nonzero().tolist() == [[1, 1]]
    y = fp8_gemm(q, quantize_fp8(torch.ones(4, 300), block_rows=BLOCK), out_dtype=torch.float32)
    assert y[1].isnan().all() and torch.equal(y[[0, 2]], torch.full((2, 4), 300.0))


def test_weight_transpose_is_the_same_numbers():
    w = _loud(200, 300)
    assert torch.equal(quantize_fp8(w, block_rows=BLOCK).dequantize().t(), quantize_fp8(w.t(), block_rows=BLOCK).dequantize())


def test_gemm_epilogue():
    torch.manual_seed(0)
    a, b = quantize_fp8(torch.randn(5, 200)), quantize_fp8(torch.randn(7, 200), block_rows=BLOCK)
    bias, gamma, res = torch.randn(7), torch.rand(7), torch.randn(5, 7)
    acc = a.dequantize().double() @ b.dequantize().double().t() + bias.double()
    pre = torch.empty(5, 7)
    y = fp8_gemm(a, b, out_dtype=torch.float32, bias=bias, act=ACT_GELU, gamma=gamma, residual=res, aux_out=pre)
    torch.testing.assert_close(pre.double(), acc, rtol=1e-5, atol=1e-5)
    torch.testing.assert_close(y.double(), res.double() + gamma.double() * F.gelu(acc), rtol=1e-5, atol=1e-5)
    out = torch.ones(5, 7)
    fp8_gemm(a, b, out=out, accumulate=True)
    torch.testing.assert_close(out.double(), acc - bias.double() + 1, rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize("m,k,n", [(1, 8, 8), (5, 130, 33), (130, 64, 140)])
def test_linear_and_gradients_follow_the_definition(m, k, n):
    x, w, b, dy = _loud(m, k), torch.randn(n, k) / k**0.5, torch.randn(n), _loud(m, n, 1)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    y = fp8_linear(*leaves)
    xq, wq = round_exact(x, 1), round_exact(w, BLOCK)
    torch.testing.assert_close(y.double(), xq @ wq.t() + b.double(), rtol=1e-5, atol=1e-5)
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    tol = dict(rtol=1e-5, atol=1e-5 * dy.abs().max().item() * x.abs().max().item() * m)
    torch.testing.assert_close(dx.double(), round_exact(dy, 1) @ wq, **tol)
    torch.testing.assert_close(dw.double(), round_exact(dy.t(), 1) @ round_exact(x.t(), 1).t(), **tol)
    torch.testing.assert_close(db.double(), dy.double().sum(0), **tol)


def test_gradient_approximates_differences():
    """The gradients are those of the unquantised layer up to 8-bit rounding: every product is off by at
    most 2 * 2^-4 relative (two roundings of half a step of 2^-3), so each entry by that share of sum |.||.|."""
    torch.manual_seed(3)
    x, w = torch.randn(9, 40, requires_grad=True), torch.randn(12, 40, requires_grad=True)
    dy = torch.randn(9, 12)
    dx, dw = torch.autograd.grad(fp8_linear(x, w), (x, w), dy)
    rel = (1 + 2.0**-4) ** 2 - 1
    # below its block's normals a value is off by half a step of 2^-9 scales, a scale being at most max / 224;
    # twice that covers the products of two such errors
    slack = 2 * 2.0**-10 / 224
    for got, a, b in ((dx, dy, w), (dw, dy.t(), x)):
        bound = rel * (a.abs() @ b.abs()) + slack * (a.abs().max() * b.abs().sum(0) + (a.abs().sum(1, keepdim=True) * b.abs().max()))
        assert ((got - a @ b).abs() <= bound).all()


def test_fused_options_and_shapes():
    torch.manual_seed(4)
    x, w, b = torch.randn(2, 3, 24).bfloat16(), torch.randn(16, 24), torch.randn(16)
    res, g = torch.randn(2, 3, 16).bfloat16(), torch.rand(16)
    leaves = [t.requires_grad_(True) for t in (x, w, b, res, g)]
    y = fp8_linear(x, w, b, activation="gelu", residual=res, gamma=g)
    assert y.shape == (2, 3, 16) and y.dtype == torch.bfloat16
    h = round_exact(x.detach().reshape(-1, 24), 1) @ round_exact(w.detach(), BLOCK).t() + b.detach().double()
    want = (res.detach().double().view(-1, 16) + g.detach().double() * F.gelu(h)).view(2, 3, 16)
    torch.testing.assert_close(y.double(), want, rtol=2**-8, atol=1e-4)
    grads = torch.autograd.grad(y, leaves, torch.randn_like(y))
    for leaf, grad in zip(leaves, grads, strict=True):
        assert grad.shape == leaf.shape and grad.dtype == leaf.dtype and grad.isfinite().all()


def test_weight_quantised_once():
    torch.manual_seed(5)
    x, w, b = torch.randn(4, 40), torch.randn(10, 40), torch.randn(10)
    q = quantize_fp8(w, block_rows=BLOCK)
    with torch.no_grad():
        assert torch.equal(fp8_linear(x, q, b), fp8_linear(x, w, b))
    with pytest.raises(ValueError, match="no backward"):
        fp8_linear(x.requires_grad_(True), q, b)


def test_main_grad_receives_the_weight_gradients():
    torch.manual_seed(6)
    x, dy = torch.randn(6, 32), torch.randn(6, 8)
    w, b = torch.nn.Parameter(torch.randn(8, 32)), torch.nn.Parameter(torch.randn(8))
    dw, db = torch.autograd.grad(fp8_linear(x, w, b), (w, b), dy)
    w.main_grad, b.main_grad = torch.ones(8, 32), torch.ones(8)
    fp8_linear(x, w, b).backward(dy)
    assert w.grad is None and b.grad is None
    torch.testing.assert_close(w.main_grad, dw + 1)
    torch.testing.assert_close(b.main_grad, db + 1)


def test_refusals():
    x, w = torch.randn(3, 16), torch.randn(4, 16)
    for bad in (dict(x=torch.randn(3, 8)), dict(x=torch.randn(0, 16)), dict(bias=torch.zeros(3)), dict(gamma=torch.zeros(4, 1)),
                dict(residual=torch.zeros(4, 4)), dict(x=x.half()), dict(x=x.double())):
        with pytest.raises(ValueError):
            fp8_linear(**{"x": x, "weight": w, **bad})
    for args, kw in (((x.double(),), {}), ((x[0],), {}), ((x,), dict(block_rows=2)), ((x,), dict(dtype=torch.float16)),
                     ((x[:0],), {})):
        with pytest.raises(ValueError):
            quantize_fp8(*args, **kw)
    q = quantize_fp8(x)
    for kw in (dict(data=q.data.float()), dict(scale=q.scale.double()), dict(cols=17), dict(cols=0), dict(block_rows=3),
               dict(block_rows=BLOCK), dict(data=q.data[:, :8])):
        with pytest.raises(ValueError):
            Fp8Matrix(**{"data": q.data, "scale": q.scale, "cols": 16, "block_rows": 1, **kw})
    with pytest.raises(ValueError):
        fp8_gemm(q, quantize_fp8(torch.randn(4, 17)))
