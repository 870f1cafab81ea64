"""Native query/key norm with rotation against the formula in 64 bits, with error bounds from the arithmetic."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover - collected on CPU, skipped there
    pytest.skip("needs CUDA", allow_module_level=True)

from mia_train_b200.layers.common.rope import axial_pairs, split_rope_dims  # noqa: E402
from mia_train_b200.ops.qk_norm import qk_norm_rope, qk_norm_rope_attention  # noqa: E402

DEV = torch.device("cuda", 0)
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
EPS = 1e-6
U = 2.0**-24  # half a step of fp32


def _pairs(kind, d):
    if kind == "none":
        return None
    if kind == "half":
        i = torch.arange(d // 2)
        return torch.stack([i, i + d // 2], 1).int().to(DEV)
    if kind == "one":  # a single pair, second channel first
        return torch.tensor([[d - 1, 0]], dtype=torch.int32, device=DEV)
    return axial_pairs(split_rope_dims(d, 3)).to(DEV)


def _forward(x, w, ang, pairs):
    n = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)
    if w is not None:
        n = n * w
    if pairs is None:
        return n
    i, j = pairs[:, 0].long(), pairs[:, 1].long()
    c, s = ang.cos()[:, :, None], ang.sin()[:, :, None]
    out = n.clone()
    out = out.index_copy(-1, i, n[..., i] * c - n[..., j] * s)
    return out.index_copy(-1, j, n[..., j] * c + n[..., i] * s)


def _within(got, want, dtype, slack):
    """One rounding to dtype plus fp32 arithmetic of at most `slack` (a tensor or number, absolute)."""
    unit = torch.finfo(dtype).eps / 2 if dtype != F32 else 0.0
    tiny = 2.0**-25 if dtype == F16 else 0.0  # half a step of the fp16 subnormals
    err = (got.double() - want).abs()
    bound = want.abs() * unit * (1 + 2.0**-10) + slack + tiny
    assert (err <= bound).all(), f"{(err / bound.clamp(min=1e-300)).max().item():.3g} times the bound"


def _case(b, t, hq, hk, d, kind, shared, dtype, weights=True, grad_scale=1.0):
    torch.manual_seed(b * 1000 + t * 10 + d)
    packed = torch.randn(b, t, hq + 2 * hk, d, device=DEV).to(dtype)
    q, k = packed[:, :, :hq], packed[:, :, hq:hq + hk]
    pairs = _pairs(kind, d)
    ang = None if pairs is None else 20 * torch.randn(1 if shared else b, t, pairs.shape[0], device=DEV)
    qw = 1 + 0.3 * torch.randn(d, device=DEV) if weights else None
    kw = 1 + 0.3 * torch.randn(d, device=DEV) if weights else None
    dq = (grad_scale * torch.randn(b, t, hq, d, device=DEV)).to(dtype)
    dk = (grad_scale * torch.randn(b, t, hk, d, device=DEV)).to(dtype)
    return q, k, qw, kw, ang, pairs, dq, dk


def _run(q, k, qw, kw, ang, pairs, dq, dk):
    leaves = [t.detach().requires_grad_(True) if t is not None else None for t in (q, k, qw, kw, ang)]
    yq, yk = qk_norm_rope(*leaves, pairs, eps=EPS)
    some = [t for t in leaves if t is not None]
    grads = iter(torch.autograd.grad((yq, yk), some, (dq, dk)))
    return yq, yk, [next(grads) if t is not None else None for t in leaves]


def _compare(q, k, qw, kw, ang, pairs, dq, dk):
    dtype = q.dtype
    yq, yk, got = _run(q, k, qw, kw, ang, pairs, dq, dk)
    d64 = [t.detach().double().requires_grad_(True) if t is not None else None for t in (q, k, qw, kw, ang)]
    oq, ok = _forward(d64[0], d64[2], d64[4], pairs), _forward(d64[1], d64[3], d64[4], pairs)
    some = [t for t in d64 if t is not None]
    it = iter(torch.autograd.grad((oq, ok), some, (dq.double(), dk.double())))
    want = [next(it) if t is not None else None for t in d64]
    d, heads = q.shape[-1], q.shape[2] + k.shape[2]
    with torch.no_grad():
        # The rounding chain of one output: the sum of squares (d adds), the root and its reciprocal, three
        # products, sine and cosine (2 steps each), the rotation: under d / 2 + 16 half steps of |n_i| + |n_j|.
        steps = (d / 2 + 16) * U
        dangle_abs = 0.0
        for y, o, x, w, g, dx, wx in ((yq, oq, d64[0], d64[2], dq, got[0], want[0]), (yk, ok, d64[1], d64[3], dk, got[1], want[1])):
            n = _forward(x, w, None, None)
            size = n.abs().amax(-1, keepdim=True) * 2
            _within(y, o, dtype, steps * size)
            # dx = r (g - xhat mean(g xhat)), |g| <= 2 max|dy| max|w|, |mean(g xhat)| <= max|g| (mean |xhat| <= 1)
            r = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)
            top = g.double().abs().amax(-1, keepdim=True) * 2 * (w.abs().max() if w is not None else 1.0)
            _within(dx, wx, dtype, 2 * steps * r * top * (1 + (x * r).abs().amax(-1, keepdim=True)))
            dangle_abs = dangle_abs + 2 * (n.abs().amax(-1) * g.double().abs().amax(-1)).sum(2)
        rows = q.shape[0] * q.shape[1]
        for s, (x, g) in enumerate(((q, dq), (k, dk))):
            if want[2 + s] is None:
                continue
            # a sum of rows * heads terms of at most 2 max|dy| |xhat|, each with the chain's error; summing in
            # fp32 adds at most half a step of the partial sums per add along the longest chain
            h = x.shape[2]
            xhat = x.double() / torch.sqrt((x.double() ** 2).mean(-1, keepdim=True) + EPS)
            total = (2 * g.double().abs().amax(-1, keepdim=True) * xhat.abs()).sum((0, 1, 2))
            chain = min(rows * h, -(-rows // 4) * -(-h // 1)) + 700
            _within(got[2 + s], want[2 + s], F32, (steps + min(chain, 20000) * U) * total)
        if want[4] is not None:
            slack = ((heads + 8) * U + 2 * steps) * dangle_abs[:, :, None]
            _within(got[4], want[4], F32, slack.sum(0, keepdim=True) if want[4].shape[0] == 1 else slack)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("kind", ["half", "axial", "one", "none"])
@pytest.mark.parametrize("d", [8, 32, 40, 64, 80, 128, 256])
def test_head_sizes_and_pairs(d, kind, dtype):
    _compare(*_case(2, 13, 3, 2, d, kind, True, dtype))


@pytest.mark.parametrize("b,t,hq,hk", [(1, 1, 1, 1), (1, 3, 16, 16), (3, 7, 5, 1), (2, 129, 16, 4), (4, 1000, 6, 6), (1, 1, 40, 8)])
@pytest.mark.parametrize("shared", [True, False])
def test_shapes(b, t, hq, hk, shared):
    _compare(*_case(b, t, hq, hk, 64, "axial", shared, BF16))


def test_without_weights():
    _compare(*_case(2, 9, 4, 4, 64, "half", False, BF16, weights=False))


def test_long_sequence():
    _compare(*_case(1, 20011, 2, 2, 32, "axial", True, F32))


def test_zero_and_huge_heads():
    q, k, qw, kw, ang, pairs, dq, dk = _case(1, 4, 2, 2, 64, "half", True, F32)
    q = q.clone()
    q[0, 0, 0] = 0.0  # all-zero head: n = 0, dx = g / sqrt(eps)
    q[0, 1] *= 1e15
    q[0, 2] *= 1e-12
    _compare(q, k, qw, kw, ang, pairs, dq, dk)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_non_finite_head_stays_in_its_head(bad):
    q, k, qw, kw, ang, pairs, *_ = _case(1, 4, 4, 4, 64, "half", True, BF16)
    clean, _ = qk_norm_rope(q, k, qw, kw, ang, pairs)
    q = q.clone()
    q[0, 2, 1, 5] = bad
    y, _ = qk_norm_rope(q, k, qw, kw, ang, pairs)
    assert y[0, 2, 1].isnan().any()
    keep = torch.ones(4, 4, dtype=torch.bool, device=DEV)
    keep[2, 1] = False
    assert torch.equal(y[0][keep], clean[0][keep])


def test_strides_alignment_and_layouts():
    q, k, qw, kw, ang, pairs, dq, dk = _case(2, 6, 4, 4, 64, "axial", False, BF16)
    want = _run(q, k, qw, kw, ang, pairs, dq, dk)
    odd = torch.empty(q.numel() + 1, device=DEV, dtype=BF16)[1:].view(q.shape).copy_(q)  # 2-byte aligned
    heads_first = k.transpose(1, 2).contiguous().transpose(1, 2)
    expanded = dq[:, :1].expand(-1, 6, -1, -1)
    for a, b2, g in ((odd, heads_first, dq), (q[:, :, :, :], k, dq)):
        got = _run(a, b2, qw, kw, ang, pairs, g, dk)
        for x, y in zip((*want[:2], *want[2]), (*got[:2], *got[2]), strict=True):
            assert torch.equal(x, y)
    a = _run(q, k, qw, kw, ang, pairs, expanded, dk)
    b = _run(q, k, qw, kw, ang, pairs, expanded.contiguous(), dk)
    assert all(torch.equal(x, y) for x, y in zip(a[2], b[2], strict=True))


def test_pairs_outside_the_head_are_skipped():
    q, k, qw, kw, *_ = _case(1, 5, 2, 2, 32, "none", True, F32)
    pairs = torch.tensor([[0, 16], [99, 3], [-1, 4], [5, 5]], dtype=torch.int32, device=DEV)
    ang = torch.randn(1, 5, 4, device=DEV)
    got = _run(q, k, qw, kw, ang, pairs, torch.ones_like(q), torch.ones_like(k))
    want = _run(q, k, qw, kw, ang[:, :, :1].contiguous(), pairs[:1], torch.ones_like(q), torch.ones_like(k))
    assert torch.equal(got[0], want[0]) and torch.equal(got[2][0], want[2][0])
    assert torch.equal(got[2][4][:, :, :1], want[2][4]) and (got[2][4][:, :, 1:] == 0).all()


def test_repeats_are_identical():
    args = _case(2, 500, 8, 8, 64, "axial", True, BF16)
    a, b = _run(*args), _run(*args)
    assert all(torch.equal(x, y) for x, y in zip((*a[:2], *a[2]), (*b[:2], *b[2]), strict=True))


def test_partial_gradients():
    q, k, qw, kw, ang, pairs, dq, dk = _case(2, 6, 4, 4, 64, "axial", False, BF16)
    full = _run(q, k, qw, kw, ang, pairs, dq, dk)[2]
    kwr = kw.clone().requires_grad_(True)
    qr = q.detach().requires_grad_(True)
    yq, yk = qk_norm_rope(qr, k, qw, kwr, ang, pairs, eps=EPS)
    a, b = torch.autograd.grad((yq, yk), (qr, kwr), (dq, dk))
    assert torch.equal(a, full[0]) and torch.equal(b, full[3])
    # only one of the outputs is used
    yq, yk = qk_norm_rope(qr, k, qw, kwr, ang, pairs, eps=EPS)
    (c,) = torch.autograd.grad(yq, (qr,), dq)
    assert torch.equal(c, full[0])


def test_main_grad_accumulates():
    q, k, qw, kw, ang, pairs, dq, dk = _case(1, 6, 4, 4, 64, "half", True, BF16)
    full = _run(q, k, qw, kw, ang, pairs, dq, dk)[2]
    p = torch.nn.Parameter(qw.clone())
    p.main_grad = torch.ones_like(qw)
    yq, yk = qk_norm_rope(q, k, p, kw, ang, pairs, eps=EPS)
    torch.autograd.backward((yq,), (dq,))
    assert p.grad is None
    torch.testing.assert_close(p.main_grad, full[2] + 1, rtol=2 * U, atol=2 * U)


def test_one_parameter_as_both_weights():
    q, k, qw, kw, ang, pairs, dq, dk = _case(1, 300, 4, 4, 64, "half", True, BF16)
    full = _run(q, k, qw, qw.clone(), ang, pairs, dq, dk)[2]
    for sink in (False, True):
        p = torch.nn.Parameter(qw.clone())
        if sink:
            p.main_grad = torch.zeros_like(qw)
        yq, yk = qk_norm_rope(q, k, p, p, ang, pairs, eps=EPS)
        torch.autograd.backward((yq, yk), (dq, dk))
        torch.testing.assert_close(p.grad, full[2] + full[3], rtol=2 * U, atol=2 * U)
        assert not sink or (p.main_grad == 0).all()


def test_attention_on_normed_heads_matches_the_separate_calls():
    from mia_train_b200.ops.attention import rope_attention

    torch.manual_seed(0)
    b, n, h, d = 2, 130, 4, 64
    pairs = _pairs("axial", d)
    qkv = torch.randn(b, n, 3, h, d, device=DEV).bfloat16().requires_grad_(True)
    qw, kw = torch.rand(d, device=DEV).requires_grad_(True), torch.rand(d, device=DEV).requires_grad_(True)
    ang = torch.randn(b, n, pairs.shape[0], device=DEV, requires_grad=True)
    out = qk_norm_rope_attention(qkv, qw, kw, ang, pairs, d**-0.5)
    q, k = qk_norm_rope(qkv[:, :, 0], qkv[:, :, 1], qw, kw, ang, pairs)
    ref = rope_attention(torch.stack([q, k, qkv[:, :, 2]], 2), None, None, d**-0.5)
    assert torch.equal(out, ref)
    do = torch.randn_like(out)
    got = torch.autograd.grad(out, (qkv, qw, kw, ang), do)
    want = torch.autograd.grad(ref, (qkv, qw, kw, ang), do)
    for a, e in zip(got, want, strict=True):
        # dq is summed by atomics in both: equal up to the order of fp32 sums and one bf16 rounding of dq
        torch.testing.assert_close(a.float(), e.float(), rtol=2**-6, atol=2**-7 * e.abs().max().item())


def test_captured_and_replayed():
    q, k, qw, kw, ang, pairs, dq, dk = _case(2, 40, 4, 4, 64, "axial", True, BF16)
    want = _run(q, k, qw, kw, ang, pairs, dq, dk)
    want = [t.detach().clone() for t in (*want[:2], *want[2])]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        _run(q, k, qw, kw, ang, pairs, dq, dk)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = _run(q, k, qw, kw, ang, pairs, dq, dk)
    for _ in range(2):
        g.replay()
    torch.cuda.synchronize()
    for a, e in zip((*out[:2], *out[2]), want, strict=True):
        assert torch.equal(a, e)


def test_native_refusals():
    from mia_train_b200.ops._native import native

    q = torch.zeros(1, 2, 2, 64, device=DEV, dtype=BF16)
    pairs, ang, w = _pairs("half", 64), torch.zeros(1, 2, 32, device=DEV), torch.ones(64, device=DEV)
    ok = [q, q, w, w, ang, pairs, torch.empty_like(q), torch.empty_like(q), EPS]
    native().qk_norm_fwd(*ok)
    for i, bad in ((0, q[..., :60]), (1, q.float()), (1, q[:, :1]), (2, w[:32]), (2, w.half()), (4, ang[:, :1]), (4, ang.half()),
                   (5, pairs.long()), (6, torch.empty(1, 2, 3, 64, device=DEV, dtype=BF16)), (7, q.cpu()),
                   (0, torch.zeros(257, device=DEV, dtype=BF16)[1:].view(1, 2, 2, 64))):
        args = list(ok)
        args[i] = bad
        with pytest.raises(RuntimeError):
            native().qk_norm_fwd(*args)
    assert qk_norm_rope(q[:, :0], q[:, :0], w, w, ang[:, :0], pairs)[0].shape == (1, 0, 2, 64)
