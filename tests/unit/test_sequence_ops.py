"""Packed attention, rotation by positions and distillation from top logits on the CPU, and what they refuse."""

from __future__ import annotations

import math

import pytest
import torch

from mia_train_b200.ops.attention import rotate_pairs_reference
from mia_train_b200.ops.distill import top_logit_distillation, top_logits
from mia_train_b200.ops.packed_attention import PackedSequences, packed_attention
from mia_train_b200.ops.rotary import rotary, rotary_frequencies


# -------------------------------------------------------------------------------- packed attention


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lq,lk", [([3, 0, 5, 1], None), ([2, 4, 0, 3], [5, 1, 2, 0]), ([], None), ([0], [4])])
def test_bounds_say_which_pairs_see_each_other(lq, lk, causal):
    seq = PackedSequences(lq, lk, causal=causal, device="cpu")
    keys = lq if lk is None else lk
    seen = torch.zeros(sum(lq), sum(keys), dtype=torch.bool)
    a = c = 0
    for m, n in zip(lq, keys, strict=True):
        block = torch.ones(m, n, dtype=torch.bool)
        seen[a:a + m, c:c + n] = block.tril(n - m) if causal else block
        a, c = a + m, c + n
    assert (seq.num_queries, seq.num_keys, len(seq)) == (sum(lq), sum(keys), len(lq))
    j, i = torch.arange(seq.num_keys), torch.arange(seq.num_queries)
    q, k = seq.q_bounds, seq.k_bounds
    assert q.shape == (sum(lq), 2) and k.shape == (sum(keys), 2) and q.dtype == k.dtype == torch.int32
    assert torch.equal((j >= q[:, :1]) & (j < q[:, 1:]), seen)
    assert torch.equal((i >= k[:, :1]) & (i < k[:, 1:]), seen.t())
    for table in (q, k):  # the kernels take the range of many rows from the first and the last
        assert (table.diff(dim=0) >= 0).all()


def test_lengths_come_in_several_forms():
    for lengths in ((2, 3), torch.tensor([2, 3]), torch.tensor([2, 3], dtype=torch.int32)):
        assert PackedSequences(lengths, device="cpu").lengths == (2, 3)
    for bad in ([1, -1], [2**31], [1.5], [[1]]):
        with pytest.raises((ValueError, TypeError)):
            PackedSequences(bad, device="cpu")
    with pytest.raises(ValueError):
        PackedSequences([1, 2], [3], device="cpu")
    with pytest.raises(TypeError):
        PackedSequences(torch.tensor([1.0]), device="cpu")


@pytest.mark.parametrize("causal", [False, True])
def test_packed_attention_is_attention_of_every_sequence(causal):
    torch.manual_seed(0)
    lq, lk = [3, 1, 6, 0], [5, 2, 4, 3]
    q, k, v = (torch.randn(n, h, 8, dtype=torch.float64, requires_grad=True) for n, h in ((12, 4), (16, 2), (16, 2)))
    out = packed_attention(q, k, v, PackedSequences(lq, lk, causal=causal, device="cpu"), 0.3)
    a = c = 0
    for m, n in zip(lq, lk, strict=True):
        for h in range(4):
            s = q[a:a + m, h] @ k[c:c + n, h // 2].t() * 0.3
            if causal:
                s = s.masked_fill(~torch.ones(m, n, dtype=torch.bool).tril(n - m), -math.inf)
            want = torch.softmax(s, -1).nan_to_num(0.0) @ v[c:c + n, h // 2]
            assert torch.allclose(out[a:a + m, h], want, atol=1e-12)
        a, c = a + m, c + n
    assert (out[10:] == 0).all()
    out.sum().backward()
    assert (q.grad[10:] == 0).all() and (k.grad[14:] == 0).all() and q.grad.isfinite().all()
    assert torch.autograd.gradcheck(
        lambda *x: packed_attention(*x, PackedSequences([2, 3], causal=causal, device="cpu")),
        [torch.randn(5, h, 8, dtype=torch.float64, requires_grad=True) for h in (2, 1, 1)])


def test_packed_attention_refusals():
    q, k = torch.randn(5, 4, 8), torch.randn(5, 2, 8)
    seq = PackedSequences([2, 3], device="cpu")
    packed_attention(q, k, k, seq)
    for bad in (lambda: packed_attention(q[:4], k, k, seq), lambda: packed_attention(q, k[:4], k[:4], seq),
                lambda: packed_attention(q, k, k[:, :1], seq), lambda: packed_attention(q[:, :3], k, k, seq),
                lambda: packed_attention(q, k.double(), k.double(), seq), lambda: packed_attention(q[0], k, k, seq),
                lambda: packed_attention(q, k[..., :4], k[..., :4], seq),
                lambda: packed_attention(q, k[:, :0], k[:, :0], seq),
                lambda: packed_attention(q, k, k, seq, math.inf)):
        with pytest.raises(ValueError):
            bad()


# -------------------------------------------------------------------------------------- rotation


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("p", [0, 3, 4])
def test_rotation_is_that_of_the_angle_table(layout, p):
    torch.manual_seed(0)
    q, k = torch.randn(2, 5, 3, 8), torch.randn(2, 5, 1, 8)
    freq, positions = torch.rand(2, p), torch.randn(2, 5, 2)
    pair = torch.arange(p)
    pairs = torch.stack([pair, pair + p] if layout == "half" else [2 * pair, 2 * pair + 1], 1)
    for got, x in zip(rotary(q, k, positions, freq, layout=layout), (q, k), strict=True):
        assert torch.allclose(got, rotate_pairs_reference(x, positions @ freq, pairs), atol=1e-5)


def test_rotation_gradients_and_shapes():
    torch.manual_seed(0)
    q, k = (torch.randn(3, h, 6, dtype=torch.float64, requires_grad=True) for h in (2, 1))
    freq = torch.rand(2, 2, dtype=torch.float64, requires_grad=True)
    positions = torch.randn(3, 2, dtype=torch.float64)
    assert torch.autograd.gradcheck(lambda *x: rotary(x[0], x[1], positions, x[2], layout="interleaved", amplitude=1.5),
                                    (q, k, freq))
    y, none = rotary(q, None, torch.arange(3), freq[0])
    assert none is None and y.shape == q.shape


def test_frequencies():
    freq, amplitude = rotary_frequencies(8, 100.0)
    assert torch.allclose(freq, 100.0 ** -(torch.arange(4).double() / 4)) and amplitude == 1.0
    linear, _ = rotary_frequencies(8, 100.0, scaling="linear", factor=4.0)
    assert torch.allclose(linear, freq / 4)
    ntk, _ = rotary_frequencies(8, 100.0, scaling="ntk", factor=4.0)
    assert torch.allclose(ntk[[0, 3]], freq[[0, 3]] / torch.tensor([1.0, 4.0], dtype=torch.float64))
    plain, _ = rotary_frequencies(128)
    yarn, amplitude = rotary_frequencies(128, scaling="yarn", factor=8.0, original_length=4096)
    turns = 4096 * plain / (2 * math.pi)
    assert amplitude == pytest.approx(0.1 * math.log(8) + 1)
    # the ramp's ends are whole pairs: one pair of slack on either side
    fast, slow = int((turns > 32).sum()) - 1, int((turns >= 1).sum()) + 1
    assert torch.equal(yarn[:fast], plain[:fast]) and torch.allclose(yarn[slow:], plain[slow:] / 8)
    assert ((yarn <= plain) & (yarn >= plain / 8 * (1 - 1e-12))).all()
    for bad in (dict(rotary_dim=7), dict(rotary_dim=8, base=1.0), dict(rotary_dim=8, scaling="other"),
                dict(rotary_dim=8, factor=0.5), dict(rotary_dim=8, scaling="yarn", factor=2.0)):
        with pytest.raises(ValueError):
            rotary_frequencies(**bad)


def test_rotary_refusals():
    q, k, positions, freq = torch.randn(2, 5, 3, 8), torch.randn(2, 5, 1, 8), torch.arange(5), torch.rand(4)
    rotary(q, k, positions, freq)
    for bad in (lambda: rotary(q, k, positions, freq, layout="other"), lambda: rotary(q, k[:1], positions, freq),
                lambda: rotary(q, k.double(), positions, freq), lambda: rotary(q, k, positions[:4], freq),
                lambda: rotary(q, k, positions, torch.rand(5)), lambda: rotary(q, k, positions, freq.half()),
                lambda: rotary(q, k, positions.to(torch.int16), freq), lambda: rotary(q, k, positions, torch.rand(2, 4)),
                lambda: rotary(q, k, torch.randn(5, 5), torch.rand(5, 4)),
                lambda: rotary(q, k, torch.randn(5, requires_grad=True), freq),
                lambda: rotary(q, k, positions, freq, amplitude=math.nan)):
        with pytest.raises(ValueError):
            bad()


# ----------------------------------------------------------------------------------- distillation


def test_top_logits_order():
    x = torch.tensor([[1.0, 3.0, 3.0, -math.inf, 0.0], [-0.0, 0.0, -0.0, 0.0, 0.0]])
    values, indices, lse = top_logits(x, 3, tau=0.5)
    assert indices.tolist() == [[1, 2, 0], [0, 1, 2]]
    assert torch.allclose(lse, torch.logsumexp(x / 0.5, 1)) and torch.equal(values, x.gather(1, indices))
    for bad in (lambda: top_logits(x, 6), lambda: top_logits(x, 0), lambda: top_logits(x[0], 1),
                lambda: top_logits(x, 1, tau=-1.0), lambda: top_logits(x.long(), 1)):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("tail", [False, True])
def test_distillation_is_the_divergence(tail):
    torch.manual_seed(0)
    s = torch.randn(4, 9, dtype=torch.float64, requires_grad=True)
    teacher = torch.randn(4, 9, dtype=torch.float64)
    values, indices, _ = top_logits(teacher, 3)
    lse = torch.logsumexp(teacher / 0.7, 1) if tail else None
    w = torch.tensor([1.0, 0.5, 0.0, 2.0])
    got = top_logit_distillation(s, values, indices, tau=0.5, teacher_tau=0.7, teacher_lse=lse, weights=w, norm=3.0)
    q = torch.softmax(s / 0.5, 1)
    p = torch.softmax(teacher / 0.7, 1).gather(1, indices)
    qk = q.gather(1, indices)
    if tail:
        rows = (p * (p / qk).log()).sum(1)
        p_t, q_t = 1 - p.sum(1), 1 - qk.sum(1)
        rows = rows + p_t * (p_t / q_t).log()
    else:
        p = p / p.sum(1, keepdim=True)
        rows = (p * (p / qk).log()).sum(1)
    assert got.item() == pytest.approx((rows * w).sum().item() / 3.0, rel=1e-5)
    grad, = torch.autograd.grad(got, s)
    want, = torch.autograd.grad((rows * w).sum() / 3.0, s)
    assert torch.allclose(grad, want, atol=1e-6)


@pytest.mark.parametrize("tail", [False, True])
def test_entries_left_out_and_rows_without_weight(tail):
    s = torch.randn(3, 6, requires_grad=True)
    with torch.no_grad():
        s[2] = math.nan
    values = torch.tensor([[1.0, 0.0], [2.0, math.nan], [0.0, 0.0]])
    indices = torch.tensor([[4, 9], [-1, -1], [0, 1]])
    lse = torch.tensor([1.5, 0.0, 0.0]) if tail else None
    loss = top_logit_distillation(s, values, indices, teacher_lse=lse, weights=torch.tensor([1.0, 0.0 if tail else 1.0, 0.0]))
    grad, = torch.autograd.grad(loss, s)
    assert loss.isfinite() and grad.isfinite().all() and (grad[1:] == 0).all() and (grad[0] != 0).all()


def test_distillation_refusals():
    s, values, indices = torch.randn(3, 6), torch.randn(3, 2), torch.zeros(3, 2, dtype=torch.int64)
    top_logit_distillation(s, values, indices)
    for bad in (lambda: top_logit_distillation(s[0], values, indices), lambda: top_logit_distillation(s, values[:2], indices[:2]),
                lambda: top_logit_distillation(s, values, indices[:, :1]), lambda: top_logit_distillation(s, values, values),
                lambda: top_logit_distillation(s, values[:, :0], indices[:, :0]),
                lambda: top_logit_distillation(s, values, indices, tau=0.0),
                lambda: top_logit_distillation(s, values, indices, teacher_tau=math.inf),
                lambda: top_logit_distillation(s, values, indices, norm=0.0),
                lambda: top_logit_distillation(s, values, indices, weights=torch.ones(2)),
                lambda: top_logit_distillation(s, values, indices, teacher_lse=torch.ones(3, 1)),
                lambda: top_logit_distillation(s[:, :0], values, indices),
                lambda: top_logit_distillation(s, values.repeat(1, 600), indices.repeat(1, 600))):
        with pytest.raises(ValueError):
            bad()


def test_rotation_by_given_angles():
    torch.manual_seed(0)
    q, k, angles = torch.randn(2, 5, 3, 8), torch.randn(2, 5, 1, 8), 30 * torch.randn(5, 4)
    pair = torch.arange(4)
    pairs = torch.stack([pair, pair + 4], 1)
    for got, x in zip(rotary(q, k, angles, None), (q, k), strict=True):
        assert torch.allclose(got, rotate_pairs_reference(x, angles, pairs), atol=1e-5)
    for bad in (lambda: rotary(q, k, angles.double(), None), lambda: rotary(q, k, angles[0], None),
                lambda: rotary(q, k, torch.randn(5, 5), None), lambda: rotary(q, k, angles.requires_grad_(True), None)):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("dim,base,length", [(64, 100.0, 4096), (128, 10000.0, 131072), (64, 100.0, 200), (128, 10000.0, 4096),
                                             (6, 10000.0, 131072), (32, 10000.0, 20)])
def test_yarn_divides_only_pairs_that_turn_seldom(dim, base, length):
    """A pair's share of the division by the number of its turns, pair by pair. Where the ramp ends past the last pair (a small
    base, a long trained length) the last pairs turn often and are not divided in full."""
    factor, fast, slow = 8.0, 32.0, 1.0
    plain, _ = rotary_frequencies(dim, base)
    yarn, _ = rotary_frequencies(dim, base, scaling="yarn", factor=factor, original_length=length)

    def pair_of(turns):  # the pair that turns so often, not a whole number
        return dim * math.log(length / (turns * 2 * math.pi)) / (2 * math.log(base))

    low, high = max(math.floor(pair_of(fast)), 0), min(math.ceil(pair_of(slow)), dim - 1)
    for n, (a, b) in enumerate(zip(plain.tolist(), yarn.tolist(), strict=True)):
        share = min(max((n - low) / (high - low), 0.0), 1.0)  # of the division
        assert b == pytest.approx(a * (1 - share) + a / factor * share, rel=1e-12)
        if length * a / (2 * math.pi) >= fast:
            assert share <= 1 / (high - low)  # the lower end is a whole pair


def test_yarn_values_known_in_advance():
    """By hand: base 100, 64 channels, length 4096: the ramp is from pair 20 to 46, the last pair (31) 11 / 26 along it."""
    plain, _ = rotary_frequencies(64, 100.0)
    yarn, _ = rotary_frequencies(64, 100.0, scaling="yarn", factor=8.0, original_length=4096)
    assert (yarn[31] / plain[31]).item() == pytest.approx(1 - 11 / 26 * 7 / 8, rel=1e-12)
    assert torch.equal(yarn[:21], plain[:21])


def test_a_query_whose_scores_are_all_minus_infinity_gives_nan():
    q, k = torch.randn(5, 2, 8), torch.rand(5, 1, 8) + 0.1
    q[1, :, 0] = -math.inf
    out = packed_attention(q, k, k, PackedSequences([2, 3], device="cpu"))
    assert out[1].isnan().all() and out[[0, 2, 3, 4]].isfinite().all()


def test_plans_made_in_inference_mode_serve_training():
    """Autograd does not save tensors that were made in inference mode."""
    with torch.inference_mode():
        own = PackedSequences([5, 0, 3], [700, 2, 9], device="cpu")
    assert own.items is not None
    assert not any(t.is_inference() for t in (own.q_bounds, own.k_bounds, own.items, own.pieces))


@pytest.mark.parametrize("where", ["value", "inf", "lse"])
@pytest.mark.parametrize("tail", [False, True])
def test_a_teacher_that_is_not_finite_shows_in_the_loss(where, tail):
    values, lse = torch.tensor([[0.5, 0.0], [0.0, -1.0]]), torch.tensor([1.0, 1.0]) if tail else None
    if where == "lse" and not tail:
        return
    if where == "lse":
        lse[0] = math.nan
    else:
        values[0, 1] = math.nan if where == "value" else math.inf
    s = torch.randn(2, 5, requires_grad=True)
    loss = top_logit_distillation(s, values, torch.tensor([[0, 1], [2, 3]]), teacher_lse=lse)
    grad, = torch.autograd.grad(loss, s)
    assert not loss.isfinite() and not grad[0].isfinite().any() and grad[1].isfinite().all()


@pytest.mark.parametrize("tail", [False, True])
def test_a_class_named_twice(tail):
    """The gradient of one entry with both shares; the loss of two, less by sum p_j log(P / p_j)."""
    torch.manual_seed(0)
    s = torch.randn(1, 6, requires_grad=True)
    values, indices = torch.tensor([[0.3, 0.3, -0.2]]), torch.tensor([[4, 4, 1]])
    lse = torch.tensor([1.6]) if tail else None
    twice = top_logit_distillation(s, values, indices, teacher_lse=lse)
    once = top_logit_distillation(s, torch.tensor([[0.3 + math.log(2), -0.2]]), indices[:, 1:], teacher_lse=lse)
    base = 1.6 if tail else math.log(2 * math.exp(0.3) + math.exp(-0.2))
    assert twice.item() == pytest.approx(once.item() - 2 * math.exp(0.3 - base) * math.log(2), abs=1e-6)
    grads = [torch.autograd.grad(x, s)[0] for x in (twice, once)]
    assert torch.allclose(*grads, atol=1e-7)
    sure = top_logit_distillation(torch.tensor([[50.0, 0.0, 0.0]]), torch.zeros(1, 2), torch.zeros(1, 2, dtype=torch.int64))
    assert sure.item() == pytest.approx(-math.log(2))


@pytest.mark.parametrize("tau", [0.0, -1.0, math.nan, math.inf, 9e-29, 1.1e28])
def test_temperatures_that_are_refused(tau):
    s, values, indices = torch.randn(3, 6), torch.randn(3, 2), torch.zeros(3, 2, dtype=torch.int64)
    for bad in (lambda: top_logits(s, 2, tau=tau), lambda: top_logit_distillation(s, values, indices, tau=tau),
                lambda: top_logit_distillation(s, values, indices, teacher_tau=tau)):
        with pytest.raises(ValueError, match="tau must be within"):
            bad()


def test_more_tokens_or_rows_than_a_kernel_counts_are_refused():
    many = 2**31
    q, one = torch.zeros(1, 1, 8).expand(many, 1, 8), torch.zeros(1, 1).expand(many, 1)
    with pytest.raises(ValueError, match="tokens"):
        rotary(q, None, torch.zeros(1, dtype=torch.int32).expand(many), torch.ones(4))
    with pytest.raises(ValueError, match="rows"):
        top_logit_distillation(one, one, torch.zeros(1, 1, dtype=torch.int32).expand(many, 1))
