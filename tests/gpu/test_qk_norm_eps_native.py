"""Native query/key norm without an eps: steps of a warp that reach past the last head add nothing."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover - collected on CPU, skipped there
    pytest.skip("needs CUDA", allow_module_level=True)

from mia_train_b200.ops.qk_norm import qk_norm_rope  # noqa: E402

DEV = torch.device("cuda", 0)
F32, BF16 = torch.float32, torch.bfloat16
U = 2.0**-24


def _exact(x, w, ang, i, j, eps):
    n = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w
    c, s = ang.cos()[:, :, None], ang.sin()[:, :, None]
    out = n.index_copy(-1, i, n[..., i] * c - n[..., j] * s)
    return out.index_copy(-1, j, n[..., j] * c + n[..., i] * s)


# 1e-50 is no fp32 number: it becomes zero
@pytest.mark.parametrize("eps", [0.0, 1e-50, 1e-38])
@pytest.mark.parametrize("dtype", [F32, BF16])
# 256 / D' heads to a step: none of these counts is a multiple of it
@pytest.mark.parametrize("hq,hk,d", [(3, 1, 64), (5, 3, 32), (9, 2, 40), (1, 1, 128), (3, 5, 96), (7, 6, 64), (1, 2, 256)])
def test_gradients_without_eps(hq, hk, d, dtype, eps):
    torch.manual_seed(hq * 100 + d)
    b, t, p = 2, 11, d // 2
    i = torch.arange(p, device=DEV)
    pairs = torch.stack([i, i + p], 1).int()
    make = lambda *s: torch.randn(*s, device=DEV)  # noqa: E731
    q, k = make(b, t, hq, d).to(dtype), make(b, t, hk, d).to(dtype)
    leaves = [q, k, 1 + 0.3 * make(d), 1 + 0.3 * make(d), make(1, t, p)]
    dq, dk = make(b, t, hq, d).to(dtype), make(b, t, hk, d).to(dtype)

    def grads(f, leaves, dq, dk):
        leaves = [v.detach().requires_grad_(True) for v in leaves]
        return torch.autograd.grad(f(leaves), leaves, (dq, dk))

    got = grads(lambda v: qk_norm_rope(*v, pairs, eps=eps), leaves, dq, dk)
    j = i + p
    want = grads(lambda v: (_exact(v[0], v[2], v[4], i, j, eps), _exact(v[1], v[3], v[4], i, j, eps)),
                 [v.double() for v in leaves], dq.double(), dk.double())
    # per value: d adds of squares, root, sine, cosine and a dozen products; sums of b t h values of at most `top`
    steps = (d / 2 + 32) * U
    for g, w in zip(got, want, strict=True):
        assert g.isfinite().all()
        count = b * t * (hq + hk) if g.dim() < 4 else 1
        top = 8 * max(w.abs().max().item(), 1.0)
        unit = torch.finfo(g.dtype).eps / 2 if g.dtype == BF16 else 0.0
        assert ((g.double() - w).abs() <= w.abs() * unit * 1.01 + (steps + count * U) * top * 4).all()


def test_a_zero_head_without_eps_is_not_a_number_in_its_own_gradients_only():
    """x / 0 has no value, in the formula as in the kernel; the other token's gradients keep theirs."""
    torch.manual_seed(7)
    q = torch.randn(1, 2, 3, 64, device=DEV)
    q[0, 0, 1] = 0
    q.requires_grad_(True)
    k = torch.randn(1, 2, 3, 64, device=DEV)
    y = qk_norm_rope(q, k, None, None, eps=0.0)[0]
    (g,) = torch.autograd.grad(y, q, torch.ones_like(y))
    bad = torch.zeros(1, 2, 3, dtype=torch.bool, device=DEV)
    bad[0, 0, 1] = True
    assert torch.equal(y.isnan().any(-1), bad) and torch.equal(g.isnan().any(-1), bad)
