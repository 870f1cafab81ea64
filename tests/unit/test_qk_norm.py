"""Query/key head norm with rotation on the CPU: formula, gradients, refusals."""

from __future__ import annotations

import pytest
import torch

from mia_train_b200.layers.common.rope import axial_pairs, split_rope_dims
from mia_train_b200.ops.qk_norm import qk_norm_rope, qk_norm_rope_attention


def _oracle(x, w, angles, pairs, eps):
    """Norm and rotation as the complex product (n_i + i n_j) e^{i angle}, in 64 bits."""
    x = x.double()
    n = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    if w is not None:
        n = n * w.double()
    if pairs is None:
        return n
    i, j = pairs[:, 0].long(), pairs[:, 1].long()
    z = torch.complex(n[..., i], n[..., j]) * torch.polar(torch.ones_like(angles).double(), angles.double())[:, :, None]
    out = n.clone()
    out[..., i], out[..., j] = z.real, z.imag
    return out


@pytest.mark.parametrize("hq,hk,d", [(2, 2, 16), (4, 1, 24), (1, 3, 6)])
@pytest.mark.parametrize("shared", [True, False])
def test_forward_and_gradients(hq, hk, d, shared):
    torch.manual_seed(0)
    b, t = 2, 5
    pairs = axial_pairs(split_rope_dims(d, 3))
    q, k = torch.randn(b, t, hq, d, requires_grad=True), torch.randn(b, t, hk, d, requires_grad=True)
    qw, kw = torch.rand(d, requires_grad=True), torch.rand(d, requires_grad=True)
    ang = torch.randn(1 if shared else b, t, pairs.shape[0], requires_grad=True)
    leaves = (q, k, qw, kw, ang)
    yq, yk = qk_norm_rope(q, k, qw, kw, ang, pairs, eps=1e-5)
    d64 = [v.detach().double().requires_grad_(True) for v in leaves]
    oq, ok = _oracle(d64[0], d64[2], d64[4], pairs, 1e-5), _oracle(d64[1], d64[3], d64[4], pairs, 1e-5)
    torch.testing.assert_close(yq.double(), oq, rtol=1e-5, atol=1e-6)
    torch.testing.assert_close(yk.double(), ok, rtol=1e-5, atol=1e-6)
    gq, gk = torch.randn_like(yq), torch.randn_like(yk)
    got = torch.autograd.grad((yq, yk), leaves, (gq, gk))
    want = torch.autograd.grad((oq, ok), d64, (gq.double(), gk.double()))
    for a, e in zip(got, want, strict=True):
        torch.testing.assert_close(a.double(), e, rtol=1e-4, atol=1e-5)


def test_norm_only_and_no_weights():
    q, k = torch.randn(1, 3, 2, 8), torch.randn(1, 3, 1, 8)
    yq, yk = qk_norm_rope(q, k, None, None)
    torch.testing.assert_close(yq.double(), _oracle(q, None, None, None, 1e-6), rtol=1e-5, atol=1e-6)
    torch.testing.assert_close(yk.double(), _oracle(k, None, None, None, 1e-6), rtol=1e-5, atol=1e-6)


def test_attention_is_norm_then_rotation_then_attention():
    torch.manual_seed(1)
    b, n, h, d = 2, 7, 2, 12
    pairs = axial_pairs(split_rope_dims(d, 3))
    qkv = torch.randn(b, n, 3, h, d, requires_grad=True)
    qw, kw = torch.rand(d, requires_grad=True), torch.rand(d, requires_grad=True)
    ang = torch.randn(1, n, pairs.shape[0])
    out = qk_norm_rope_attention(qkv, qw, kw, ang, pairs, d**-0.5)
    q, k = _oracle(qkv[:, :, 0], qw, ang, pairs, 1e-6), _oracle(qkv[:, :, 1], kw, ang, pairs, 1e-6)
    p = torch.softmax(torch.einsum("bqhd,bkhd->bhqk", q, k) * d**-0.5, -1)
    want = torch.einsum("bhqk,bkhd->bqhd", p, qkv[:, :, 2].double())
    torch.testing.assert_close(out.double(), want, rtol=1e-4, atol=1e-5)
    assert all(g is not None for g in torch.autograd.grad(out.sum(), (qkv, qw, kw)))


@pytest.mark.parametrize("change", [
    dict(k=torch.zeros(2, 4, 1, 8)), dict(k=torch.zeros(2, 3, 1, 16)), dict(k=torch.zeros(2, 3, 1, 8).bfloat16()),
    dict(q_weight=torch.ones(4)), dict(k_weight=torch.ones(8, 1)), dict(angles=None), dict(pairs=None),
    dict(pairs=torch.zeros(5, 2, dtype=torch.int32), angles=torch.zeros(2, 3, 5)),
    dict(pairs=torch.zeros(2, 2)), dict(angles=torch.zeros(3, 3, 2)), dict(angles=torch.zeros(2, 4, 2)),
])
def test_refusals(change):
    args = dict(q=torch.zeros(2, 3, 2, 8), k=torch.zeros(2, 3, 1, 8), q_weight=torch.ones(8), k_weight=torch.ones(8),
                angles=torch.zeros(2, 3, 2), pairs=torch.tensor([[0, 4], [1, 5]], dtype=torch.int32))
    qk_norm_rope(**args)
    with pytest.raises(ValueError):
        qk_norm_rope(**{**args, **change})
    with pytest.raises(ValueError):
        qk_norm_rope_attention(torch.zeros(2, 3, 2, 2, 8), None, None, None, None, 1.0)
