"""Linear layers whose matrix products run on 8-bit floating point with block scales.

A matrix is held as 8-bit values (e4m3, or e5m2 where range matters more than precision) and one
scale per block of 128 along the summed axis: `Fp8Matrix`. The scale s of a block is the smallest power
of two >= 2^-126 with max|x| / s <= 448 (57344 for e5m2), so x / s is exact and the only rounding is
the one to 8 bits; a block with an infinity or a NaN has the scale NaN. Activations and gradients use
1 x 128 blocks, weights 128 x 128 blocks (`block_rows = 128`), which makes a weight's transpose the
same numbers.

`fp8_linear(x, weight, bias, activation, residual, gamma)` is `ops.linear.linear` on such products:

    y  = residual + gamma * act(Q(x) Q(W)^T + bias)      Q(x) 1 x 128 along K
    dX = Q(dZ) Q(W)                                      Q(dZ) 1 x 128 along N
    dW = Q(dZ^T) Q(x^T)^T                                both 1 x 128 along the rows (tokens) of x
    db = sum of dZ over the tokens                       from the unquantised gradient

One kernel reads a tensor once and writes both quantisations of it (rows and transposed columns); in
backward it also multiplies by the GELU derivative and `gamma` and sums the bias gradient. What
backward keeps is 8-bit: half of what `linear` keeps. Products are accumulated in fp32; scales are
applied in fp32. A weight that is an `Fp8Matrix` (quantised once, for inference) has no backward.

The native kernels take bf16, fp16 or fp32 inputs on CUDA and write bf16 or fp32; on the CPU the
same quantisation runs in PyTorch.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from ._autograd import differentiable_once
from ._native import native, use_native
from ._params import grad_sink
from .linear import _ACTS, ACT_GELU, compute_dtype, gelu_grad_reference, gelu_reference

BLOCK = 128
LIMITS = {torch.float8_e4m3fn: 448.0, torch.float8_e5m2: 57344.0}
_EXPONENT = {torch.float8_e4m3fn: 8, torch.float8_e5m2: 15}  # both limits are 1.75 * 2^exponent
_DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def _ceil(n: int, unit: int) -> int:
    return -(-n // unit)


@dataclass(frozen=True)
class Fp8Matrix:
    """(rows, cols) 8-bit values and their block scales.

    `data` (rows, cols rounded up to 16) holds the values, `scale` (ceil(cols / 128), rows) fp32 the
    scales, or (ceil(cols / 128), ceil(rows / 128)) with `block_rows = 128`.
    """

    data: torch.Tensor
    scale: torch.Tensor
    cols: int
    block_rows: int = 1

    def __post_init__(self) -> None:
        d, s = self.data, self.scale
        if d.dtype not in LIMITS or d.dim() != 2 or d.stride(1) != 1 or d.shape[1] % 16 or d.stride(0) % 16:
            raise ValueError(f"data must be a row-major e4m3fn or e5m2 matrix padded to 16 columns, got {d.dtype} "
                             f"{tuple(d.shape)} with strides {d.stride()}")
        if self.block_rows not in (1, BLOCK):
            raise ValueError(f"block_rows must be 1 or {BLOCK}, got {self.block_rows}")
        if not 0 < self.cols <= d.shape[1]:
            raise ValueError(f"cols must be within 1..{d.shape[1]}, got {self.cols}")
        want = (_ceil(self.cols, BLOCK), _ceil(d.shape[0], self.block_rows))
        if s.dtype != torch.float32 or tuple(s.shape) != want or s.device != d.device:
            raise ValueError(f"scale must be fp32 {want} on {d.device}, got {s.dtype} {tuple(s.shape)} on {s.device}")
        if s.shape[1] > 1 and s.stride(1) != 1:
            raise ValueError(f"scale must be row-major, got strides {s.stride()}")

    @property
    def rows(self) -> int:
        return self.data.shape[0]

    def dequantize(self) -> torch.Tensor:
        """fp32 (rows, cols)."""
        s = self.scale.repeat_interleave(BLOCK, 0)[: self.cols].t()
        if self.block_rows != 1:
            s = s.repeat_interleave(self.block_rows, 0)[: self.rows]
        return self.data[:, : self.cols].float() * s


def block_scales_reference(x: torch.Tensor, block_rows: int, dtype: torch.dtype) -> torch.Tensor:
    """(ceil(rows / block_rows), ceil(cols / 128)) scales of fp32 x, from the bits of each block's maximum."""
    r, c = x.shape
    rb, cb = _ceil(r, block_rows), _ceil(c, BLOCK)
    padded = torch.nn.functional.pad(x, (0, cb * BLOCK - c, 0, rb * block_rows - r))
    bits = padded.abs().view(torch.int32).view(rb, block_rows, cb, BLOCK).amax(dim=(1, 3))
    up = (bits & 0x7FFFFF) > 0x600000
    exponent = ((bits >> 23) - _EXPONENT[dtype] + up).clamp(min=1)
    scale = (exponent << 23).view(torch.float32)
    return torch.where(bits >= 0x7F800000, torch.full_like(scale, float("nan")), scale)


def quantize_reference(x: torch.Tensor, block_rows: int, dtype: torch.dtype) -> Fp8Matrix:
    x = x.float()
    r, c = x.shape
    scale = block_scales_reference(x, block_rows, dtype)
    full = scale.repeat_interleave(block_rows, 0)[:r].repeat_interleave(BLOCK, 1)[:, :c]
    data = torch.zeros((r, _ceil(c, 16) * 16), device=x.device, dtype=dtype)
    data[:, :c] = (x / full).to(dtype)
    return Fp8Matrix(data, scale.t().contiguous(), c, block_rows)


def _empty(rows: int, cols: int, block_rows: int, dtype: torch.dtype, device: torch.device) -> Fp8Matrix:
    data = torch.empty((rows, _ceil(cols, 16) * 16), device=device, dtype=dtype)
    scale = torch.empty((_ceil(cols, BLOCK), _ceil(rows, block_rows)), device=device, dtype=torch.float32)
    return Fp8Matrix(data, scale, cols, block_rows)


def _quantize(
    x: torch.Tensor,
    block_rows: int,
    dtype: torch.dtype,
    rows: bool,
    cols: bool,
    aux: torch.Tensor | None = None,
    gamma: torch.Tensor | None = None,
    sums: torch.Tensor | None = None,
    accumulate: bool = False,
) -> tuple[Fp8Matrix | None, Fp8Matrix | None]:
    """Q(v) and Q(v^T) of v = x * gelu'(aux) * gamma (each factor optional), and v's column sums."""
    r, c = x.shape
    if use_native(x):
        q = _empty(r, c, block_rows, dtype, x.device) if rows else None
        qt = _empty(c, r, block_rows, dtype, x.device) if cols else None
        native().fp8_quantize(
            x, aux, gamma, block_rows == BLOCK, dtype == torch.float8_e5m2,
            q.data if q is not None else None, q.scale if q is not None else None,
            qt.data if qt is not None else None, qt.scale if qt is not None else None, sums, accumulate,
        )
        return q, qt
    v = x.float()
    if aux is not None:
        v = v * gelu_grad_reference(aux)
    if gamma is not None:
        v = v * gamma
    if sums is not None:
        sums.copy_(sums + v.sum(0) if accumulate else v.sum(0))
    return (quantize_reference(v, block_rows, dtype) if rows else None,
            quantize_reference(v.t(), block_rows, dtype) if cols else None)


def quantize_fp8(x: torch.Tensor, *, block_rows: int = 1, dtype: torch.dtype = torch.float8_e4m3fn) -> Fp8Matrix:
    """x (rows, cols) with 1 x 128 scales (activations) or, with `block_rows = 128`, 128 x 128 (weights)."""
    if x.dim() != 2 or x.shape[0] == 0 or x.shape[1] == 0 or x.dtype not in _DTYPES:
        raise ValueError(f"quantize_fp8 needs a non-empty bf16, fp16 or fp32 matrix, got {x.dtype} {tuple(x.shape)}")
    if dtype not in LIMITS:
        raise ValueError(f"dtype must be one of {tuple(LIMITS)}, got {dtype}")
    if block_rows not in (1, BLOCK):
        raise ValueError(f"block_rows must be 1 or {BLOCK}, got {block_rows}")
    x = x.detach()
    q, _ = _quantize(x if x.stride(1) == 1 else x.contiguous(), block_rows, dtype, True, False)
    return q


def fp8_gemm(
    a: Fp8Matrix,
    b: Fp8Matrix,
    *,
    out: torch.Tensor | None = None,
    out_dtype: torch.dtype = torch.bfloat16,
    bias: torch.Tensor | None = None,
    residual: torch.Tensor | None = None,
    gamma: torch.Tensor | None = None,
    act: int = 0,
    accumulate: bool = False,
    aux_out: torch.Tensor | None = None,
) -> torch.Tensor:
    """D[m, n] = sum_k a[m, k] b[n, k] with `ops.linear.gemm`'s epilogue (`act` none or GELU); no autograd."""
    if a.cols != b.cols or a.data.device != b.data.device:
        raise ValueError(f"operands must share K and a device, got {a.cols} on {a.data.device} and {b.cols} on {b.data.device}")
    if out is None:
        out = torch.empty((a.rows, b.rows), device=a.data.device, dtype=out_dtype)
    if use_native(a.data):
        native().fp8_gemm(a.data, a.scale, a.block_rows != 1, b.data, b.scale, b.block_rows != 1, a.cols, out,
                          bias, residual, gamma, aux_out, act, accumulate)
        return out
    with torch.autocast(out.device.type, enabled=False):
        acc = a.dequantize() @ b.dequantize().t()
    if bias is not None:
        acc = acc + bias.float()
    if act == ACT_GELU:
        if aux_out is not None:
            aux_out.copy_(acc)
        acc = gelu_reference(acc)
    if gamma is not None:
        acc = acc * gamma.float()
    if residual is not None:
        acc = acc + residual.float()
    out.copy_(acc + out.float() if accumulate else acc)
    return out


class _Fp8Linear(torch.autograd.Function):
    """The PyTorch path; on CUDA `csrc/block_ops.cpp` holds the same node."""

    @staticmethod
    def forward(ctx, x2, weight, bias, residual, gamma, act, cdtype, grad):  # type: ignore[override]
        e4m3 = torch.float8_e4m3fn
        need_x, need_w, need_b, _, need_g = (grad and n for n in ctx.needs_input_grad[:5])
        product = need_x or need_w or need_b  # some gradient goes through the activation
        n = weight.shape[0]
        shadow = getattr(weight, "_mia_shadow", None)  # under a sharded optimizer only the bf16 copy is current
        w = (shadow if shadow is not None else weight).detach().reshape(n, -1)
        xq, xt = _quantize(x2, 1, e4m3, True, need_w)
        wq, wt = _quantize(w, BLOCK, e4m3, True, need_x)
        g, bf = (t.detach().float() if t is not None else None for t in (gamma, bias))
        pre = torch.empty((x2.shape[0], n), device=x2.device, dtype=cdtype) if act == ACT_GELU and product else None
        y = fp8_gemm(xq, wq, out_dtype=cdtype, bias=bf, residual=residual, gamma=g, act=act, aux_out=pre)
        keep = {"xt": xt, "wt": wt, "xq": xq if need_g else None, "wq": wq if need_g else None}
        ctx.held = {k: (m.cols, m.block_rows) for k, m in keep.items() if m is not None}
        flat = [t for m in keep.values() if m is not None for t in (m.data, m.scale)]
        # gamma scales the gradient of the product; the bias is in the activation that gamma's own gradient recomputes
        ctx.save_for_backward(pre, g if product else None, bf if need_g else None, *flat)
        ctx.meta = (act, weight.dtype, weight.shape, gamma.dtype if gamma is not None else None,
                    bias.dtype if bias is not None else None)
        ctx.sinks = (grad_sink(weight), grad_sink(bias))
        # y is linear in x, weight, bias and gamma alone, but not in two that are multiplied, nor behind an activation
        ctx.open = (need_x and need_w) or ((act != 0 or need_g) and product)
        return y

    @staticmethod
    @differentiable_once("fp8_linear")
    def backward(ctx, dy):  # type: ignore[override]
        pre, g, bf, *flat = ctx.saved_tensors
        held = {k: Fp8Matrix(flat[2 * i], flat[2 * i + 1], cols, block)
                for i, (k, (cols, block)) in enumerate(ctx.held.items())}
        act, wdtype, wshape, gdtype, bdtype = ctx.meta
        need_x, need_w, need_b, need_r, need_g = ctx.needs_input_grad[:5]
        n = dy.shape[1]
        dgamma = None
        if need_g:
            # d(gamma * h) / d gamma needs h = act(x W^T + b): recomputed once, from the saved operands
            h = fp8_gemm(held["xq"], held["wq"], out_dtype=torch.float32, bias=bf, act=act)
            dgamma = (dy.float() * h).sum(0).to(gdtype)
        w_sink, b_sink = ctx.sinks
        sums = None
        if need_b:
            sums = b_sink if b_sink is not None else torch.empty(n, device=dy.device, dtype=torch.float32)
        dzq, dzt = _quantize(dy, 1, torch.float8_e4m3fn, need_x, need_w, aux=pre, gamma=g, sums=sums,
                             accumulate=b_sink is not None)
        dx = fp8_gemm(dzq, held["wt"], out_dtype=dy.dtype) if need_x else None
        dw = None
        if need_w:
            if w_sink is not None:
                fp8_gemm(dzt, held["xt"], out=w_sink.view(n, -1), accumulate=True)
            else:
                dw = fp8_gemm(dzt, held["xt"], out_dtype=torch.float32).to(wdtype).view(wshape)
        db = sums.to(bdtype) if need_b and b_sink is None else None
        return dx, dw, db, (dy if need_r else None), dgamma, None, None, None


def fp8_linear(
    x: torch.Tensor,
    weight: torch.Tensor | Fp8Matrix,
    bias: torch.Tensor | None = None,
    activation: str | None = None,
    residual: torch.Tensor | None = None,
    gamma: torch.Tensor | None = None,
) -> torch.Tensor:
    """`residual + gamma * act(x @ weight.T + bias)` on 8-bit products; see the module docstring.

    Computes in the autocast dtype (else x's): bf16, or fp32 without activation, residual or gamma
    fused (they are then applied by PyTorch).
    """
    act = _ACTS[activation]
    quantised = isinstance(weight, Fp8Matrix)
    n, k = (weight.rows, weight.cols) if quantised else (weight.shape[0], weight[0].numel())
    device = weight.data.device if quantised else weight.device
    if x.shape[-1] != k or x.device != device or x.numel() == 0 or n == 0:
        raise ValueError(f"x must be non-empty with {k} channels on {device}, got {tuple(x.shape)} on {x.device}")
    if bias is not None and (bias.shape != (n,) or bias.device != device):
        raise ValueError(f"bias must be a vector of length {n} on {device}, got {tuple(bias.shape)} on {bias.device}")
    if gamma is not None and (gamma.shape != (n,) or gamma.device != device):
        raise ValueError(f"gamma must be a vector of length {n} on {device}, got {tuple(gamma.shape)} on {gamma.device}")
    if residual is not None and (residual.shape != (*x.shape[:-1], n) or residual.device != device):
        raise ValueError(f"residual must be {(*x.shape[:-1], n)} on {device}, got {tuple(residual.shape)}")
    cdtype = compute_dtype(x)
    if cdtype not in (torch.bfloat16, torch.float32):
        raise ValueError(f"fp8_linear computes in bf16 or fp32, got {cdtype}")
    if torch.is_grad_enabled() and quantised and any(
        t is not None and t.requires_grad for t in (x, bias, residual, gamma)
    ):
        raise ValueError("a weight quantised once has no backward; pass the weight tensor to train")
    fused = cdtype == torch.bfloat16
    f_act, f_gamma, f_res = (act, gamma, residual) if fused else (0, None, None)
    if x.dtype not in _DTYPES:
        x = x.to(cdtype)
    if use_native(x):
        if quantised:
            y = native().fp8_linear_quantized(x, weight.data, weight.scale, weight.block_rows != 1, k, bias, f_res, f_gamma,
                                              f_act, fused)
        else:
            # under a sharded optimizer only the bf16 copy of a weight is current
            y = native().fp8_linear(x, weight, bias, f_res, f_gamma, f_act, fused, getattr(weight, "_mia_shadow", None),
                                    grad_sink(weight), grad_sink(bias))
    else:
        x2 = x.reshape(-1, k)
        res2 = f_res.reshape(-1, n).to(cdtype) if f_res is not None else None
        if quantised:
            y = fp8_gemm(_quantize(x2.detach(), 1, torch.float8_e4m3fn, True, False)[0], weight, out_dtype=cdtype,
                         bias=bias, residual=res2, gamma=f_gamma, act=f_act)
        else:
            y = _Fp8Linear.apply(x2, weight, bias, res2, f_gamma, f_act, cdtype, torch.is_grad_enabled())
        y = y.reshape(*x.shape[:-1], n)
    if fused:
        return y
    if act == ACT_GELU:
        y = gelu_reference(y)
    if gamma is not None:
        y = y * gamma
    return y if residual is None else residual + y
