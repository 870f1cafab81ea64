"""Counter-based dropout on the CPU: generator vectors, statistics, gradients, refusals."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from mia_train_b200.ops.dropout import STEPS, dropout, dropout_reference, random_halves_reference


def _philox_words(counter, key, rounds=10):
    """Philox4x32 on Python integers, from the definition (Salmon et al., SC 2011)."""
    c, k = list(counter), list(key)
    for _ in range(rounds):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(b >> 32) ^ c[1] ^ k[0], b & 0xFFFFFFFF, (a >> 32) ^ c[3] ^ k[1], a & 0xFFFFFFFF]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def test_oracle_matches_the_published_vector():
    # known-answer test of Philox4x32-10 published with the paper: zero counter, zero key
    assert _philox_words([0] * 4, [0] * 2) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]


@pytest.mark.parametrize("seed,offset", [(0, 0), (1, 4), (-5, 12), (2**62 + 12345, 2**40 + 8)])
def test_halves_follow_the_counter(seed, offset):
    got = random_halves_reference(8 * 37 + 3, torch.tensor([seed, offset])).tolist()
    assert len(got) == 8 * 37 + 3
    key = [seed & 0xFFFFFFFF, seed >> 32 & 0xFFFFFFFF]
    for g in (0, 1, 36, 37):
        words = _philox_words([g, 0, offset & 0xFFFFFFFF, (offset >> 32 & 0xFFFFFFFF) | 0x80000000], key)
        want = [h for w in words for h in (w & 0xFFFF, w >> 16)]
        assert got[8 * g:8 * g + 8] == want[:len(got[8 * g:8 * g + 8])]


def test_large_counts_use_the_high_counter_word():
    # a group index beyond 32 bits reaches the second counter word (checked through the arithmetic alone)
    word = 0xFFFFFFFF
    group = torch.tensor([2**32 + 5])
    assert (group & word).item() == 5 and (group >> 32).item() == 1


@pytest.mark.parametrize("p", [0.1, 0.5, 0.9])
def test_keep_rate_and_mean(p):
    n = 1 << 17
    x = torch.ones(n, dtype=torch.float32)
    y = dropout(x, p, rng=torch.tensor([17, 0]))
    kept = (y != 0).double().mean().item()
    # binomial: six standard deviations
    assert abs(kept - (1 - p)) < 6 * (p * (1 - p) / n) ** 0.5 + 1 / STEPS
    dropped = round(p * STEPS)
    scale = torch.tensor(STEPS / (STEPS - dropped), dtype=torch.float32)
    assert torch.equal(y[y != 0], scale.expand(int((y != 0).sum())))


def test_neighbouring_offsets_and_seeds_are_unrelated():
    n = 1 << 15
    a, b, c = (random_halves_reference(n, torch.tensor(r)) for r in ([3, 0], [3, 4], [4, 0]))
    for other in (b, c):
        agree = ((a >= STEPS // 2) == (other >= STEPS // 2)).double().mean().item()
        assert abs(agree - 0.5) < 6 * 0.5 / n**0.5


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (3, 5), (2, 3, 17)])
def test_gradient_is_the_scaled_mask(shape, residual):
    torch.manual_seed(0)
    rng = torch.tensor([9, 16])
    x = torch.randn(shape, dtype=torch.float64, requires_grad=True)
    r = torch.randn(shape, dtype=torch.float64, requires_grad=True) if residual else None
    inputs = (x, r) if residual else (x,)
    # linear in its inputs: differences are exact up to rounding
    assert torch.autograd.gradcheck(lambda *a: dropout(a[0], 0.3, residual=a[1] if residual else None, rng=rng), inputs)
    y = dropout(x, 0.3, residual=r, rng=rng)
    dy = torch.randn(shape, dtype=torch.float64)
    grads = torch.autograd.grad(y, inputs, dy)
    dropped = round(0.3 * STEPS)
    keep = (random_halves_reference(x.numel(), rng) >= dropped).view(shape)
    torch.testing.assert_close(grads[0], torch.where(keep, dy * (STEPS / (STEPS - dropped)), 0.0), rtol=1e-15, atol=0)
    if residual:
        assert torch.equal(grads[1], dy)


def test_mask_follows_row_major_order_of_any_strides():
    x = torch.randn(6, 10)
    rng = torch.tensor([1, 0])
    t = x.t().contiguous().t()  # same values, other strides
    assert not t.is_contiguous() and torch.equal(dropout(t, 0.4, rng=rng), dropout(x, 0.4, rng=rng))


def test_pair_may_advance_before_backward():
    x = torch.randn(64, requires_grad=True)
    rng = torch.tensor([5, 0])
    y = dropout(x, 0.5, rng=rng)
    rng[1] += 4
    (dx,) = torch.autograd.grad(y, x, torch.ones(64))
    assert torch.equal(dx != 0, y != 0)


def test_generator_seed_reproduces_and_calls_differ():
    x = torch.ones(512)
    torch.manual_seed(3)
    a, b = dropout(x, 0.5), dropout(x, 0.5)
    torch.manual_seed(3)
    assert torch.equal(dropout(x, 0.5), a) and not torch.equal(a, b)


def test_identity_and_extremes():
    x, r = torch.randn(5, 3), torch.randn(5, 3)
    assert dropout(x, 0.0) is x and dropout(x, 0.7, training=False) is x
    assert torch.equal(dropout(x, 0.7, residual=r, training=False), r + x)
    assert torch.equal(dropout(x, 1.0, rng=torch.tensor([0, 0])), torch.zeros_like(x))
    assert torch.equal(dropout(x, 1.0, residual=r, rng=torch.tensor([0, 0])), r)
    assert dropout(torch.empty(0, 4), 0.5).shape == (0, 4)


def test_dropped_infinities_leave_nothing():
    x = torch.full((4096,), float("inf"))
    y = dropout(x, 0.5, rng=torch.tensor([2, 0]))
    assert not y.isnan().any() and y.isinf().any() and (y == 0).any()


def test_rounded_once():
    torch.manual_seed(1)
    x, r = torch.randn(333).bfloat16(), torch.randn(333).bfloat16()
    rng = torch.tensor([8, 4])
    y = dropout(x, 0.25, residual=r, rng=rng)
    exact = dropout_reference(x.double(), round(0.25 * STEPS), rng, r.double())
    err = (y.double() - exact).abs()
    assert (err <= exact.abs() * torch.finfo(torch.bfloat16).eps / 2 * (1 + 1e-6)).all()


@pytest.mark.parametrize("bad", [
    dict(p=-0.1), dict(p=1.5), dict(p=float("nan")),
    dict(residual=torch.zeros(4, 3)), dict(residual=torch.zeros(4, 4, dtype=torch.float64)),
    dict(residual=torch.zeros(4)),  # a broadcast residual is the caller's to expand
    dict(rng=torch.zeros(2)), dict(rng=torch.zeros(3, dtype=torch.int64)),
])
def test_refusals(bad):
    args = {"p": 0.5, **bad}
    with pytest.raises(ValueError):
        dropout(torch.zeros(4, 4), args.pop("p"), **args)
    with pytest.raises(ValueError):
        dropout(torch.zeros(4, dtype=torch.int64), 0.5)


def test_counter_fits_numpy_check():
    # the 16-bit split product against numpy's 64-bit unsigned product
    from mia_train_b200.ops.dropout import _mul_hi_lo

    a = np.random.default_rng(0).integers(0, 2**32, 1000, dtype=np.uint64)
    hi, lo = _mul_hi_lo(torch.from_numpy(a.astype(np.int64)), 0xD2511F53)
    prod = a * np.uint64(0xD2511F53)
    assert np.array_equal(hi.numpy().astype(np.uint64), prod >> np.uint64(32))
    assert np.array_equal(lo.numpy().astype(np.uint64), prod & np.uint64(0xFFFFFFFF))
