"""RMS norm of query and key heads with the position rotation in the same pass.

`qk_norm_rope(q, k, q_weight, k_weight, angles, pairs, eps)` normalises every head of q (B, T, Hq, D)
and k (B, T, Hk, D) over its channels, multiplies by the learned weight (D) of q or k, and rotates
the channel pairs by the token's angles (`ops/attention.py` states that form):

    n = x * rsqrt(mean(x^2) + eps) * weight,   y = rotate_pairs(n, angles, pairs)

in fp32, rounded once. The inputs may be strided views of a packed projection; the outputs share one
contiguous buffer. `angles` (1 or B, T, P), read in fp32, and `pairs` (P, 2) may be None: norm only. Each channel is
in one pair at most; a pair that names a channel outside the head is skipped on CUDA. The backward pass
recomputes the norm from q and k (nothing else is kept) and returns the gradients of q, k, both
weights and the angles.

`qk_norm_rope_attention(qkv, ...)` is `ops.attention.rope_attention` on normalised heads: norm and
rotation read q and k out of the packed (B, N, 3, H, D) projection, attention reads v in place, and the
backward pass leaves dq, dk and dv in one packed gradient.
"""

from __future__ import annotations

import torch

from ._autograd import differentiable_once
from ._native import native, use_native
from ._params import grad_sink
from .attention import _native_ok as _attention_native_ok
from .attention import attention_reference, rotate_pairs_reference

MAX_HEAD_DIM = 256
_DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def head_norm_rope_reference(
    x: torch.Tensor,
    weight: torch.Tensor | None,
    angles: torch.Tensor | None,
    pairs: torch.Tensor | None,
    eps: float,
) -> torch.Tensor:
    acc = torch.promote_types(x.dtype, torch.float32)
    xf = x.to(acc)
    n = xf * torch.rsqrt(xf.square().mean(-1, keepdim=True) + eps)
    if weight is not None:
        n = n * weight.to(acc)
    if angles is not None and pairs is not None and pairs.numel():
        n = rotate_pairs_reference(n, angles, pairs.long())
    return n.to(x.dtype)


def _native_norm_ok(q: torch.Tensor, k: torch.Tensor) -> bool:
    d = q.shape[-1]
    return q.dtype in _DTYPES and k.dtype == q.dtype and d % 8 == 0 and 8 <= d <= MAX_HEAD_DIM and use_native(q, k)


def _prepared(angles: torch.Tensor | None, pairs: torch.Tensor | None, device: torch.device):
    if angles is None or pairs is None or pairs.numel() == 0:
        return None, torch.zeros((0, 2), dtype=torch.int32, device=device)
    return angles.float().contiguous(), pairs.to(device=device, dtype=torch.int32).contiguous()


class _Norms:
    """Weight and angle gradients of the attention node."""

    @staticmethod
    def sinks(qw: torch.Tensor | None, kw: torch.Tensor | None):
        """Both weights' `main_grad`. The kernel writes both gradients at once, so one parameter used as both weights
        gets them through autograd, which adds them."""
        if qw is not None and qw is kw:
            return None, None
        return grad_sink(qw), grad_sink(kw)

    @staticmethod
    def weight(w: torch.Tensor | None) -> torch.Tensor | None:
        return w.float().contiguous() if w is not None else None

    @staticmethod
    def grads(ctx, d: int, device: torch.device):
        """(dqw, dkw, accumulate bits): a parameter's `main_grad` where it has one."""
        outs, bits = [], 0
        for s, (sink, wanted) in enumerate(zip(ctx.sinks, ctx.want_w, strict=True)):
            if not wanted:
                outs.append(None)
            elif sink is not None:
                outs.append(sink.view(d))
                bits |= 1 << s
            else:
                outs.append(torch.empty(d, device=device, dtype=torch.float32))
        return outs, bits

    @staticmethod
    def returned(ctx, outs):
        return [
            None if o is None or sink is not None else o.to(dtype)
            for o, sink, dtype in zip(outs, ctx.sinks, ctx.w_dtypes, strict=True)
        ]

    @staticmethod
    def angle_grad(dangles: torch.Tensor | None, shape, dtype) -> torch.Tensor | None:
        if dangles is None:
            return None
        if shape[0] == 1 and dangles.shape[0] != 1:
            dangles = dangles.sum(0, keepdim=True)
        return dangles.to(dtype)


def _check(q, k, q_weight, k_weight, angles, pairs) -> None:
    qs, ks = q.shape, k.shape
    if len(qs) != 4 or len(ks) != 4 or (qs[0], qs[1], qs[3]) != (ks[0], ks[1], ks[3]) or not qs[2] or not ks[2]:
        raise ValueError(f"q and k must be (B, T, H, D) of one batch, length and head size, got {tuple(qs)} and "
                         f"{tuple(ks)}")
    if q.dtype != k.dtype or q.device != k.device or not q.is_floating_point():
        raise ValueError(f"q and k must share a floating-point dtype and a device, got {q.dtype} on {q.device} and "
                         f"{k.dtype} on {k.device}")
    b, t, _, d = qs
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is not None and (w.shape != (d,) or w.device != q.device):
            raise ValueError(f"{name} must be a vector of the head size {d} on {q.device}, got {tuple(w.shape)} on {w.device}")
    if (angles is None) != (pairs is None):
        raise ValueError("angles and pairs come together")
    if angles is None:
        return
    if pairs.dim() != 2 or pairs.shape[1] != 2 or pairs.shape[0] > d // 2 or pairs.is_floating_point():
        raise ValueError(f"pairs must be integer (P, 2) with P <= {d // 2}, got {pairs.dtype} {tuple(pairs.shape)}")
    if angles.dim() != 3 or angles.shape[0] not in (1, b) or angles.shape[1:] != (t, pairs.shape[0]) or angles.device != q.device:
        raise ValueError(f"angles must be (1 or {b}, {t}, {pairs.shape[0]}) on {q.device}, got {tuple(angles.shape)} on "
                         f"{angles.device}")


def qk_norm_rope(
    q: torch.Tensor,
    k: torch.Tensor,
    q_weight: torch.Tensor | None,
    k_weight: torch.Tensor | None,
    angles: torch.Tensor | None = None,
    pairs: torch.Tensor | None = None,
    eps: float = 1e-6,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Normalised and rotated (q, k); see the module docstring."""
    _check(q, k, q_weight, k_weight, angles, pairs)
    if _native_norm_ok(q, k):
        q_sink, k_sink = _Norms.sinks(q_weight, k_weight)
        return native().qk_norm_rope(q, k, q_weight, k_weight, angles, pairs, float(eps), q_sink, k_sink)
    pairs = pairs.to(q.device) if pairs is not None else None
    return (head_norm_rope_reference(q, q_weight, angles, pairs, eps),
            head_norm_rope_reference(k, k_weight, angles, pairs, eps))


class _NativeNormRopeAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, qkv, qw, kw, angles, pairs, scale, eps):  # type: ignore[override]
        b, n, _, h, d = qkv.shape
        qkv = qkv.contiguous()
        ang, pr = _prepared(angles, pairs, qkv.device)
        qwf, kwf = _Norms.weight(qw), _Norms.weight(kw)
        qk = torch.empty((b, n, 2, h, d), device=qkv.device, dtype=qkv.dtype)
        q, k, v = qk[:, :, 0], qk[:, :, 1], qkv[:, :, 2]
        native().qk_norm_fwd(qkv[:, :, 0], qkv[:, :, 1], qwf, kwf, ang, pr, q, k, float(eps))
        o = torch.empty((b, n, h, d), device=qkv.device, dtype=qkv.dtype)
        lse = torch.empty((b, h, n), device=qkv.device, dtype=torch.float32)
        native().attention_fwd_strided(q, k, v, o, lse, float(scale))
        ctx.save_for_backward(qkv, qk, o, lse, qwf, kwf, ang, pr)
        ctx.scale, ctx.eps = float(scale), float(eps)
        ctx.sinks = _Norms.sinks(qw, kw)
        ctx.w_dtypes = tuple(w.dtype if w is not None else None for w in (qw, kw))
        ctx.angles_meta = (angles.shape, angles.dtype) if angles is not None else None
        ctx.open = True  # the softmax makes every gradient depend on every operand
        return o

    @staticmethod
    @differentiable_once("qk_norm_rope_attention")
    def backward(ctx, do):  # type: ignore[override]
        qkv, qk, o, lse, qw, kw, ang, pairs = ctx.saved_tensors
        b, n, _, h, d = qkv.shape
        do = do.to(qkv.dtype).contiguous()
        dqkv = torch.empty_like(qkv)
        none = torch.zeros((0, 2), dtype=torch.int32, device=qkv.device)
        native().rope_attention_bwd_packed(qk[:, :, 0], qk[:, :, 1], qkv[:, :, 2], o, do, lse, None, none, dqkv, None,
                                           ctx.scale)
        ctx.want_w = ctx.needs_input_grad[1:3]
        dws, bits = _Norms.grads(ctx, d, qkv.device)
        dangles = None
        if ang is not None and ctx.needs_input_grad[3]:
            dangles = torch.empty((b, n, pairs.shape[0]), device=qkv.device, dtype=torch.float32)
        dq, dk = dqkv[:, :, 0], dqkv[:, :, 1]  # the rotated-space gradients, replaced in place
        native().qk_norm_bwd(dq, dk, qkv[:, :, 0], qkv[:, :, 1], qw, kw, ang, pairs, dq, dk, dws[0], dws[1], bits,
                             dangles, ctx.eps)
        if ctx.angles_meta is not None:
            dangles = _Norms.angle_grad(dangles, *ctx.angles_meta)
        return dqkv, *_Norms.returned(ctx, dws), dangles, None, None, None


def qk_norm_rope_attention(
    qkv: torch.Tensor,
    q_weight: torch.Tensor | None,
    k_weight: torch.Tensor | None,
    angles: torch.Tensor | None,
    pairs: torch.Tensor | None,
    scale: float,
    eps: float = 1e-6,
) -> torch.Tensor:
    """Packed (B, N, 3, H, D) projections -> attention over normalised, rotated heads, (B, N, H, D)."""
    if qkv.dim() != 5 or qkv.shape[2] != 3:
        raise ValueError(f"qkv must be (B, N, 3, H, D), got {tuple(qkv.shape)}")
    q, k, v = qkv.unbind(dim=2)
    _check(q, k, q_weight, k_weight, angles, pairs)
    if qkv.numel() and _attention_native_ok(qkv, qkv.shape[-1]):
        return _NativeNormRopeAttention.apply(qkv, q_weight, k_weight, angles, pairs, scale, eps)
    q, k = qk_norm_rope(q, k, q_weight, k_weight, angles, pairs, eps)
    return attention_reference(q, k, v, scale)
