"""Native dropout against the generator's definition, bit for bit."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover - collected on CPU, skipped there
    pytest.skip("needs CUDA", allow_module_level=True)

from mia_train_b200.ops.dropout import STEPS, dropout, dropout_reference, random_halves_reference  # noqa: E402

DEV = torch.device("cuda", 0)
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _rng(seed=11, offset=8):
    return torch.tensor([seed, offset], device=DEV)


def _words(c, k):
    """Philox4x32-10 on Python integers."""
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(b >> 32) ^ c[1] ^ k[0], b & 0xFFFFFFFF, (a >> 32) ^ c[3] ^ k[1], a & 0xFFFFFFFF]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (9,), (3, 5), (2, 3, 128), (257, 1283), (4096, 1024)])
def test_equals_the_definition(shape, residual, dtype):
    # one fp32 product (and sum) per element, rounded once, in kernel and oracle: equal to the bit,
    # unless the kernel contracts product and sum into one rounding, which then is nearer the exact value
    torch.manual_seed(0)
    x = torch.randn(shape, device=DEV).to(dtype).requires_grad_(True)
    r = torch.randn(shape, device=DEV).to(dtype).requires_grad_(True) if residual else None
    y = dropout(x, 0.3, residual=r, rng=_rng())
    dropped = round(0.3 * STEPS)
    if residual:
        exact = dropout_reference(x.detach().double(), dropped, _rng(), r.detach().double())
        # the scale is an fp32 number (2^-24), as are product and sum; then the rounding to dtype
        unit = torch.finfo(dtype).eps / 2 * (dtype != F32) + 3 * 2.0**-24
        bound = exact.abs() * unit + (x.detach().double().abs() * 1.5) * 3 * 2.0**-24
        assert ((y.detach().double() - exact).abs() <= bound * (1 + 1e-6) + 2.0**-25).all()
    else:
        assert torch.equal(y, dropout_reference(x.detach(), dropped, _rng()))
    dy = torch.randn(shape, device=DEV).to(dtype)
    grads = torch.autograd.grad(y, (x, r) if residual else (x,), dy)
    assert torch.equal(grads[0], dropout_reference(dy, dropped, _rng()))
    if residual:
        assert torch.equal(grads[1], dy)


def test_matches_the_cpu_mask():
    x = torch.randn(1000)
    a = dropout(x, 0.6, rng=torch.tensor([5, 4]))
    assert torch.equal(dropout(x.to(DEV), 0.6, rng=torch.tensor([5, 4], device=DEV)).cpu(), a)


@pytest.mark.parametrize("shift", [1, 3])
def test_unaligned_and_strided(shift):
    base = torch.randn(4099, device=DEV).bfloat16()
    x = base[shift:shift + 4001]  # 2-byte aligned only
    want = dropout_reference(x.clone(), round(0.5 * STEPS), _rng())
    assert torch.equal(dropout(x, 0.5, rng=_rng()), want)
    m = torch.randn(64, 80, device=DEV).bfloat16()
    assert torch.equal(dropout(m.t(), 0.5, rng=_rng()), dropout_reference(m.t().contiguous(), round(0.5 * STEPS), _rng()))
    # a gradient with zero strides
    leaf = m.clone().requires_grad_(True)
    (g,) = torch.autograd.grad(dropout(leaf, 0.5, rng=_rng()).sum(), leaf)
    assert torch.equal(g, dropout_reference(torch.ones_like(m), round(0.5 * STEPS), _rng()))


def test_writes_nothing_behind_its_output():
    from mia_train_b200.ops._native import native

    buf = torch.full((1032,), 7.0, device=DEV, dtype=BF16)
    x = torch.randn(1001, device=DEV).bfloat16()
    native().dropout_apply(x, None, buf[:1001], 32768, _rng(), None)
    assert (buf[1001:] == 7.0).all()


def test_indices_beyond_31_bits():
    n = 2**31 + 13
    if torch.cuda.mem_get_info()[0] < 12 * 2**30:
        pytest.skip("needs 12 GB")
    x = torch.ones(n, device=DEV, dtype=BF16)
    y = dropout(x, 0.5, rng=_rng(2, 4))
    del x
    tail = y[n - 13:].float()
    want = []
    for g in (2**28, 2**28 + 1):  # the last two groups
        want += [h for w in _words([g, 0, 4, 0x80000000], [2, 0]) for h in (w & 0xFFFF, w >> 16)]
    assert (tail != 0).tolist() == [h >= STEPS // 2 for h in want[:13]]


def test_generator_draws_and_graph_replays():
    x = torch.ones(1 << 14, device=DEV, requires_grad=True)
    torch.manual_seed(1)
    a, b = dropout(x, 0.5), dropout(x, 0.5)
    torch.manual_seed(1)
    assert torch.equal(dropout(x, 0.5), a) and not torch.equal(a, b)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    ones = torch.ones_like(x)
    with torch.cuda.stream(s):  # warm-up on the capturing stream
        torch.autograd.grad(dropout(x, 0.5), x, ones)
    torch.cuda.current_stream().wait_stream(s)
    del a, b
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = dropout(x, 0.5)
        (dx,) = torch.autograd.grad(y, x, ones)
    seen = []
    for _ in range(3):
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, dx)  # x and dy are ones: forward and backward drew the same mask
        seen.append(y.detach().clone())
    assert not torch.equal(seen[0], seen[1]) and not torch.equal(seen[1], seen[2])


def test_activation_checkpointing_replays_the_mask():
    from torch.utils.checkpoint import checkpoint

    x = torch.randn(512, 64, device=DEV, requires_grad=True)
    torch.manual_seed(4)
    f = lambda t: dropout(t, 0.4) * 2  # noqa: E731
    (a,) = torch.autograd.grad(f(x).square().sum(), x)
    torch.manual_seed(4)
    (b,) = torch.autograd.grad(checkpoint(f, x, use_reentrant=False).square().sum(), x)
    assert torch.equal(a, b)


def test_side_stream():
    x = torch.randn(1 << 20, device=DEV)
    want = dropout(x, 0.2, rng=_rng())
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = dropout(x, 0.2, rng=_rng())
    s.synchronize()
    assert torch.equal(got, want)


def test_native_refusals():
    from mia_train_b200.ops._native import native

    x, y = torch.zeros(16, device=DEV), torch.empty(16, device=DEV)
    ok = (x, None, y, 100, _rng(), None)
    native().dropout_apply(*ok)
    for i, bad in ((0, x.double()), (0, x.cpu()), (1, x[:8]), (2, y.bfloat16()), (3, 65537), (4, _rng().float()),
                   (4, _rng().cpu()), (5, _rng()[:1])):
        args = list(ok)
        args[i] = bad
        with pytest.raises(RuntimeError):
            native().dropout_apply(*args)
    assert random_halves_reference(0, _rng()).numel() == 0
    assert dropout(torch.empty(0, 3, device=DEV), 0.5).shape == (0, 3)
