"""Native rotation by positions against the complex product in 64 bits."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover - collected on CPU, skipped there
    pytest.skip("needs CUDA", allow_module_level=True)

from mia_train_b200.ops.rotary import rotary, rotary_frequencies  # noqa: E402

DEV = torch.device("cuda", 0)
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
U = 2.0**-24


def _turn(x, positions, freq, layout, amplitude):
    p = freq.shape[-1]
    angle = positions.double() @ freq.double()
    c, s = amplitude * angle.cos()[..., None, :], amplitude * angle.sin()[..., None, :]
    if layout == "half":
        x1, x2 = x[..., :p], x[..., p:2 * p]
        y = torch.cat([x1 * c - x2 * s, x2 * c + x1 * s], -1)
    else:
        x1, x2 = x[..., 0:2 * p:2], x[..., 1:2 * p:2]
        y = torch.stack([x1 * c - x2 * s, x2 * c + x1 * s], -1).flatten(-2)
    return torch.cat([y, x[..., 2 * p:]], -1)


def _case(b, t, hq, hk, d, p, axes, dtype, seed=0, far=1000):
    gen = torch.Generator(device=DEV).manual_seed(seed + 100 * d + t)
    normal = lambda *s: torch.randn(*s, device=DEV, generator=gen)  # noqa: E731
    proj = normal(b, t, hq + 2 * hk, d).to(dtype)
    q, k = proj[:, :, :hq], proj[:, :, hq:hq + hk]
    if axes == 1:
        positions = torch.randint(0, far, (b, t, 1), device=DEV, generator=gen)
    else:
        positions = normal(b, t, axes) * 8
    freq = torch.rand(axes, p, device=DEV, generator=gen) ** 4
    return q, k, positions, freq, normal(b, t, hq, d).to(dtype), normal(b, t, hk, d).to(dtype)


def _within(got, want, bound, dtype):
    unit = torch.finfo(dtype).eps / 2 if dtype != F32 else 0.0
    err = (got.double() - want).abs()
    total = want.abs() * unit * (1 + 2.0**-10) + bound + (2.0**-25 if dtype == F16 else 0.0)
    assert (err <= total).all(), f"{(err / total.clamp(min=1e-300)).max().item():.3g} times the bound"


def _compare(q, k, positions, freq, dq, dk, layout, amplitude, learn):
    dtype, one = q.dtype, freq.shape[0] == 1
    leaves = [q.detach().requires_grad_(True), k.detach().requires_grad_(True), freq.detach().requires_grad_(learn)]
    got_q, got_k = rotary(leaves[0], leaves[1], positions.squeeze(-1) if one else positions,
                          leaves[2].squeeze(0) if one else leaves[2], layout=layout, amplitude=amplitude)
    grads = torch.autograd.grad((got_q, got_k), leaves if learn else leaves[:2], (dq, dk))
    wide = [x.detach().double().requires_grad_(True) for x in (q, k, freq)]
    want_q, want_k = (_turn(x, positions, wide[2], layout, amplitude) for x in wide[:2])
    expected = torch.autograd.grad((want_q, want_k), wide, (dq.double(), dk.double()))
    with torch.no_grad():
        # the angle's fraction of a turn, sine and cosine (2 steps each), the amplitude, two products and a sum: under
        # 16 half steps of both channels of the pair
        for got, want, x in ((got_q, want_q, q), (got_k, want_k, k), (grads[0], expected[0], dq), (grads[1], expected[1], dk)):
            size = abs(amplitude) * 2 * x.double().abs().amax(-1, keepdim=True)
            _within(got, want, 16 * U * size, dtype)
        if learn:
            # sums over tokens and heads: the rotation's error in every term, and an add per term in fp32
            terms = 2 * abs(amplitude) * sum((x.double().abs().amax(-1) * g.double().abs().amax(-1)).sum(2) for x, g in
                                             ((q, dq), (k, dk)))
            total = (positions.double().abs() * terms[..., None]).sum((0, 1))[:, None]
            _within(grads[2], expected[2], (16 + 400) * U * total, F32)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("d,p", [(64, 32), (64, 16), (128, 32), (40, 20), (40, 8), (8, 1), (96, 45), (256, 128), (64, 0)])
def test_head_sizes(d, p, dtype, layout):
    _compare(*_case(2, 13, 3, 2, d, p, 1, dtype), layout, 1.0, p > 0)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("axes", [2, 3, 4])
@pytest.mark.parametrize("b,t,hq,hk", [(1, 1, 1, 1), (3, 257, 4, 4), (1, 4101, 8, 2)])
def test_axes_and_learned_frequencies(b, t, hq, hk, axes, layout):
    _compare(*_case(b, t, hq, hk, 64, 32, axes, BF16), layout, 1.3, True)


@pytest.mark.parametrize("kind", [torch.int32, torch.int64, torch.float32, torch.float64])
def test_far_positions_keep_their_accuracy(kind):
    """A position of 2^20 at frequency 1: its angle in fp32 would be off by 2^-4."""
    q, k, positions, freq, dq, dk = _case(1, 64, 2, 1, 64, 32, 1, F32, far=1 << 20)
    _compare(q, k, positions.to(kind), freq, dq, dk, "half", 1.0, False)


@pytest.mark.parametrize("scaling", [None, "linear", "ntk", "yarn"])
def test_stretched_frequencies(scaling):
    freq, amplitude = rotary_frequencies(64, scaling=scaling, factor=8.0, original_length=4096, device=DEV)
    q, k, positions, _, dq, dk = _case(2, 50, 2, 2, 128, 32, 1, BF16, far=32768)
    _compare(q, k, positions, freq[None], dq, dk, "interleaved", amplitude, False)


def test_shapes_of_tokens_and_positions():
    q, k, _, freq, _, _ = _case(2, 30, 2, 2, 32, 16, 1, BF16)
    positions = torch.arange(30, device=DEV)
    yq, yk = rotary(q, k, positions, freq[0])
    for want, got in ((yq, rotary(q, k, positions.expand(2, 30), freq[0])[0]), (yq, rotary(q, None, positions, freq[0])[0]),
                      (yk[1], rotary(q[1], k[1], positions, freq[0])[1]), (yq, rotary(q, k, positions[None], freq[0])[0])):
        assert torch.equal(want, got)
    assert rotary(q, None, positions, freq[0])[1] is None
    assert rotary(q[:, :0], k[:, :0], positions[:0], freq[0])[0].shape == (2, 0, 2, 32)
    odd = torch.zeros(2, 30, 2, 33, device=DEV, dtype=BF16)
    odd[..., 1:] = q
    assert torch.equal(rotary(odd[..., 1:], None, positions, freq[0])[0], yq)


def test_one_of_two_gradients_and_the_same_bits_every_time():
    q, k, positions, freq, dq, dk = _case(2, 300, 4, 2, 64, 32, 3, BF16)
    leaves = [x.detach().requires_grad_(True) for x in (q, k, freq)]
    first = None
    for _ in range(3):
        yq, yk = rotary(*leaves[:2], positions, leaves[2])
        got = torch.autograd.grad(yq, leaves, dq, allow_unused=True)
        assert (got[1] == 0).all()
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(got, first, strict=True))


def test_captured_graph():
    q, k, positions, freq, dq, dk = _case(2, 64, 2, 2, 64, 32, 3, BF16)
    leaves = [x.detach().clone().requires_grad_(True) for x in (q, k, freq)]

    def run():
        y = rotary(*leaves[:2], positions, leaves[2])
        return [*(x.detach() for x in y), *torch.autograd.grad(y, leaves, (dq, dk))]

    want = run()
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        got = run()
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want, strict=True))


def test_changed_operands_and_second_derivatives_are_refused():
    q, k, positions, freq, dq, dk = _case(1, 20, 1, 1, 32, 16, 2, BF16)
    leaf, learned = q.detach().clone().requires_grad_(True), freq.detach().requires_grad_(True)
    x = leaf * 1
    y, _ = rotary(x, None, positions, learned)
    x.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward(dq)
    y, _ = rotary(leaf, None, positions, learned)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(y, leaf, dq, create_graph=True)
    y, _ = rotary(leaf, None, positions, freq)  # linear in q: a constant gradient is returned
    torch.autograd.grad(y, leaf, dq, create_graph=True)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("far", [1.0, 300.0, 1e5])
def test_given_angles(far, dtype, layout):
    """Angles in radians, reduced from their fp32 value: 2^-48 of it is lost."""
    q, k, _, _, dq, dk = _case(2, 40, 3, 1, 64, 16, 1, dtype)
    angles = far * torch.randn(1, 40, 16, device=DEV)
    leaves = [x.detach().requires_grad_(True) for x in (q, k)]
    y = rotary(*leaves, angles, None, layout=layout)
    grads = torch.autograd.grad(y, leaves, (dq, dk))
    eye = torch.eye(16, device=DEV)
    for got, x, turned in ((y[0], q, angles), (y[1], k, angles), (grads[0], dq, -angles), (grads[1], dk, -angles)):
        want = _turn(x.double(), turned, eye, layout, 1.0)
        _within(got, want, 16 * U * 2 * x.double().abs().amax(-1, keepdim=True), dtype)


def test_heads_without_channels():
    q = torch.zeros(2, 3, 2, 0, device=DEV, dtype=BF16)
    assert rotary(q, q, torch.arange(3, device=DEV), torch.zeros(0, device=DEV))[0].shape == q.shape


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("table", [torch.float32, torch.float64])
@pytest.mark.parametrize("kind", [torch.int32, torch.int64, torch.float32, torch.float64])
def test_frequencies_that_are_not_finite_give_nan(kind, table, layout):
    """In their own pairs, at every position (0 too), in outputs and in gradients."""
    q, k, positions, freq, dq, dk = _case(1, 40, 2, 1, 64, 32, 1, F32)
    positions[0, 7] = 0
    bad = {3: torch.nan, 9: torch.inf, 30: -torch.inf}
    freq = freq.to(table)
    for at, x in bad.items():
        freq[0, at] = x
    leaves = [q.detach().requires_grad_(True), k.detach().requires_grad_(True), freq[0].detach().requires_grad_(True)]
    y = rotary(*leaves[:2], positions.squeeze(-1).to(kind), leaves[2], layout=layout)
    grads = torch.autograd.grad(y, leaves, (dq, dk))
    pair = torch.zeros(32, dtype=torch.bool, device=DEV)
    pair[list(bad)] = True
    channel = pair.repeat(2) if layout == "half" else pair.repeat_interleave(2)
    for x in (*y, *grads[:2]):
        assert x[..., channel].isnan().all() and x[..., ~channel].isfinite().all()
    assert torch.equal(grads[2].isnan(), pair)


@pytest.mark.parametrize("f", [-1e-20, -2.0**-60, 1e300, -3.25, 6.283185307179586])
def test_frequencies_at_the_ends_of_a_turn(f):
    q, k, positions, freq, dq, dk = _case(1, 40, 2, 1, 64, 32, 1, F32)
    freq = torch.full((1, 32), f, device=DEV, dtype=torch.float64)
    if abs(f) < 100:
        _compare(q, k, positions, freq, dq, dk, "half", 1.0, False)
    else:  # far beyond what 64 bits resolve: any angle, but a rotation
        y, _ = rotary(q, k, positions.squeeze(-1), freq[0])
        assert torch.allclose(y[..., :32] ** 2 + y[..., 32:] ** 2, q[..., :32] ** 2 + q[..., 32:] ** 2, rtol=1e-5)


@pytest.mark.parametrize("far", [1.0, 1e5])
def test_angles_that_are_not_finite_give_nan(far):
    q = torch.randn(1, 5, 1, 8, device=DEV)
    angles = far * torch.randn(5, 4, device=DEV)
    angles[2, 1], angles[3, 2] = torch.nan, torch.inf
    y, _ = rotary(q, None, angles, None)
    bad = ~angles.isfinite().repeat(1, 2)
    assert torch.equal(y[0, :, 0].isnan(), bad)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("axes", [1, 3])
@pytest.mark.parametrize("d", [64, 33])
def test_a_learned_table_without_pairs(d, axes, layout):
    """Nothing turns: the heads are copied, and the table's gradient has no element."""
    _compare(*_case(2, 13, 3, 2, d, 0, axes, BF16), layout, 1.0, True)
