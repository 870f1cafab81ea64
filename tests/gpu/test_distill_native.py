"""Native top logits and distillation from them against the definitions in 64 bits."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover - collected on CPU, skipped there
    pytest.skip("needs CUDA", allow_module_level=True)

from mia_train_b200.ops.distill import top_logit_distillation, top_logits  # noqa: E402

DEV = torch.device("cuda", 0)
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
TYPES = [BF16, F16, F32]


def _logits(r, v, dtype, seed=0, size=1.0):
    gen = torch.Generator(device=DEV).manual_seed(seed + v)
    return (size * torch.randn(r, v, device=DEV, generator=gen)).to(dtype)


# ------------------------------------------------------------------------------------- top logits


def _check_top(x, k, tau=1.0):
    values, indices, lse = top_logits(x, k, tau=tau)
    order = torch.sort(x.double(), dim=1, descending=True, stable=True)
    assert values.dtype == x.dtype and indices.dtype == torch.int64
    assert torch.equal(indices, order.indices[:, :k])
    assert torch.equal(values, x.gather(1, order.indices[:, :k])) or values.isnan().any()
    z = x.double() / tau
    want = torch.logsumexp(z, 1)
    # differences to the maximum (a step each), exp2 of the multi-function unit, a thread's some 300 adds at most
    assert ((lse.double() - want).abs() <= 2.0**-17 + 2.0**-22 * z.abs().amax(1))[want.isfinite()].all()
    assert torch.equal(lse[~want.isfinite()].double().nan_to_num(7.0), want[~want.isfinite()].nan_to_num(7.0))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("r,v,k", [(1, 1, 1), (3, 7, 7), (2, 255, 255), (2, 256, 256), (5, 1000, 8), (4, 4097, 100),
                                   (3, 65536, 64), (2, 131071, 256), (1, 20000, 1)])
def test_top_sizes(r, v, k, dtype):
    _check_top(_logits(r, v, dtype), k, 0.3)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("levels", [1, 2, 3, 40])
def test_equal_logits_go_by_the_lower_index(levels, dtype):
    gen = torch.Generator(device=DEV).manual_seed(levels)
    x = torch.randint(0, levels, (4, 30011), device=DEV, generator=gen).to(dtype)
    for k in (1, 33, 256):
        _check_top(x, k)


def test_special_values():
    x = _logits(6, 5000, F32)
    x[0] = -math.inf
    x[1, :] = torch.where(torch.arange(5000, device=DEV) % 2 == 0, 0.0, -0.0)
    x[2, 77] = math.inf
    x[3, 5:4000] = -math.inf
    x[4, :] = torch.finfo(F32).min
    x[5, 100::7] = x[5, 100]
    _check_top(x, 64)
    x = _logits(2, 5000, F32)
    x[0, 4000] = x[0, 17] = math.nan
    values, indices, lse = top_logits(x, 3)
    assert indices[0, :2].tolist() == [17, 4000] and values[0, :2].isnan().all() and lse[0].isnan()
    assert torch.equal(indices[1], x[1].topk(3).indices)
    x[0] = math.nan
    assert top_logits(x, 3)[1][0].tolist() == [0, 1, 2]


def test_top_strides_streams_and_graphs():
    wide = _logits(6, 3001, BF16)
    view = wide[::2, 1:2999]
    _check_top(view, 17)
    _check_top(wide.t(), 5)
    want = top_logits(view, 17)
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        got = top_logits(view, 17)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want, strict=True))
    assert [tuple(t.shape) for t in top_logits(wide[:0], 3)] == [(0, 3), (0, 3), (0,)]


# ----------------------------------------------------------------------------------- distillation


def _definition(s, values, indices, tau, teacher_tau, lse, w, norm):
    """Loss, gradient and bounds in 64 bits, entry by entry of the teacher's list."""
    r, v = s.shape
    x = s.double()
    at = indices.long()
    given = (at >= 0) & (at < v)
    safe = torch.where(given, at, 0)
    t = torch.where(given, values.double(), -math.inf) / teacher_tau
    base = torch.logsumexp(t, 1, keepdim=True) if lse is None else lse.double()[:, None]
    p = torch.where(t > -math.inf, (t - base).exp(), 0.0)
    log_q = torch.log_softmax(x / tau, 1)
    q = log_q.exp()
    per = torch.where(p > 0, p * ((t - base).nan_to_num(0.0) - log_q.gather(1, safe)), 0.0)
    rows = per.sum(1)
    mass = p.sum(1, keepdim=True)
    dense = torch.zeros_like(x).scatter_add(1, safe, p)
    named = torch.zeros_like(x).scatter_add(1, safe, given.double()) > 0
    noise = q * mass + dense
    grad = q * mass - dense
    if lse is not None:
        rest = torch.where(named.all(1, keepdim=True), 0.0, (1 - mass).clamp(min=0))
        other = torch.logsumexp(torch.where(named, -math.inf, log_q), 1, keepdim=True)
        rows = rows + torch.where(rest > 0, rest * (rest.clamp(min=1e-300).log() - other), 0.0)[:, 0]
        share = torch.where(named, 0.0, (log_q - other).exp().nan_to_num(0.0))
        grad = q * (mass + rest) - dense - rest * share
        noise = noise + rest * (q + share)
        mass = mass + rest
    w = torch.ones(r, device=s.device, dtype=torch.float64) if w is None else w.double()
    span = (x.amax(1) - x.amin(1)) / tau
    # a logit's difference to the maximum and its product with 1 / tau (a step each of the exponent's size), exp2, sums
    rho = 2.0**-17 + 2.0**-21 * span
    f = w[:, None] / (norm * tau)
    unit = torch.finfo(s.dtype).eps / 2
    # exp2 of the multi-function unit gives 0 for results below 2^-126, which f and at most twice the mass then multiply
    bound = f * noise * rho[:, None] + unit * (f * grad).abs() + (2.0**-25 if s.dtype == F16 else 1e-38) + 2.0**-125 * f * mass
    loss_bound = (w * mass[:, 0] * rho).sum() / norm + 2.0**-23 * ((w * rows).sum() / norm).abs()
    return (w * rows).sum() / norm, f * grad, loss_bound, bound


def _distill(r, v, k, dtype, tail, weights, tau=0.5, teacher_tau=0.7, seed=0, index=torch.int64, kind=F32, upstream=1.0):
    gen = torch.Generator(device=DEV).manual_seed(seed + v + k)
    s = _logits(r, v, dtype, seed)
    teacher = s.float() * 0.5 + _logits(r, v, F32, seed + 1)
    values, indices = teacher.topk(k, dim=1)
    values = values.to(kind)
    lse = torch.logsumexp(teacher.double() / teacher_tau, 1).float() if tail else None
    w = torch.rand(r, device=DEV, generator=gen) * (torch.arange(r, device=DEV) % 3 != 1) if weights else None
    return _check_distill(s, values, indices.to(index), tau, teacher_tau, lse, w, upstream)


def _check_distill(s, values, indices, tau, teacher_tau, lse, w, upstream=1.0, norm=None):
    leaf = s.detach().requires_grad_(True)
    loss = top_logit_distillation(leaf, values, indices, tau=tau, teacher_tau=teacher_tau, teacher_lse=lse, weights=w,
                                  norm=norm)
    grad, = torch.autograd.grad(loss * upstream, leaf)
    want, want_grad, loss_bound, bound = _definition(s, values, indices, tau, teacher_tau, lse, w, norm or s.shape[0])
    assert loss.dtype == F32 and grad.dtype == s.dtype
    assert (loss.double() - want).abs() <= loss_bound, f"loss {loss.item()} for {want.item()}"
    err = (grad.double() - upstream * want_grad).abs()
    bound = abs(upstream) * bound + (2.0**-25 if s.dtype == F16 else 0.0)
    assert (err <= bound).all(), f"{(err / bound).max().item():.3g} times the bound"
    return loss, grad


@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("r,v,k", [(1, 2, 1), (4, 9, 3), (5, 1000, 8), (3, 4097, 64), (7, 65536, 64), (2, 20001, 1024)])
def test_distill_sizes(r, v, k, dtype, tail, weights):
    _distill(r, v, k, dtype, tail, weights)


@pytest.mark.parametrize("kind", [BF16, F16, F32, torch.float64])
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_distill_types_of_the_teacher(kind, index):
    _distill(3, 500, 5, BF16, False, False, kind=kind, index=index)


@pytest.mark.parametrize("tau,teacher_tau", [(0.04, 0.04), (1.0, 0.07), (8.0, 3.0)])
@pytest.mark.parametrize("tail", [False, True])
def test_distill_temperatures_and_upstream_gradients(tau, teacher_tau, tail):
    _distill(4, 3001, 20, F32, tail, True, tau, teacher_tau, upstream=-3.7)


@pytest.mark.parametrize("tail", [False, True])
def test_every_class_given(tail):
    """No class is left: the teacher's lse may leave some rounding of 1, which has nowhere to go."""
    _distill(3, 64, 64, F32, tail, False)


@pytest.mark.parametrize("tail", [False, True])
def test_a_sure_student(tail):
    """A mass outside the teacher's classes that is far below a step of 1 still has its logarithm."""
    s = _logits(2, 4000, F32)
    s[:, 3] += 150.0
    indices = torch.tensor([[3, 9], [3, 11]], device=DEV)
    values = torch.tensor([[5.0, 1.0], [3.0, 2.5]], device=DEV)
    lse = torch.tensor([5.2, 4.1], device=DEV) if tail else None
    _check_distill(s, values, indices, 1.0, 1.0, lse, None)


@pytest.mark.parametrize("tail", [False, True])
def test_indices_that_repeat_or_name_no_class(tail):
    s = _logits(4, 777, F32)
    indices = torch.tensor([[5, 5, 700, 5], [-1, 3, -1, 8], [900, 776, 0, 1], [2, 3, 4, 4]], device=DEV)
    values = torch.tensor([[1.0, 2.0, 0.5, -1.0], [9.0, 1.0, math.nan, 0.0], [3.0, 2.0, 1.0, 0.0],
                           [-math.inf, 1.0, 2.0, -math.inf]], device=DEV)
    values[1, 2] = 4.0
    lse = torch.tensor([4.0, 2.0, 4.5, 3.0], device=DEV) if tail else None
    _check_distill(s, values, indices, 0.8, 1.0, lse, None)


def test_rows_without_a_teacher_or_a_weight():
    s = _logits(4, 1001, BF16)
    values, indices = s.float().topk(6, dim=1)
    indices[2] = -1  # nothing given: no loss and no gradient
    w = torch.tensor([1.0, 0.0, 1.0, 0.5], device=DEV)
    clean_loss, clean = _check_distill(s, values, indices, 0.5, 0.5, None, w)
    assert (clean[1] == 0).all() and (clean[2] == 0).all()
    s[1] = math.nan  # a row of weight 0 is not read
    leaf = s.detach().requires_grad_(True)
    loss = top_logit_distillation(leaf, values, indices, tau=0.5, teacher_tau=0.5, weights=w)
    grad, = torch.autograd.grad(loss, leaf)
    assert torch.equal(loss, clean_loss) and torch.equal(grad, clean)


@pytest.mark.parametrize("tail", [False, True])
def test_masked_classes(tail):
    """Student logits of -inf or the type's lowest value have no share and no gradient."""
    for low in (-math.inf, torch.finfo(BF16).min):
        s = _logits(3, 1500, BF16)
        s[:, 1000:] = low
        values, indices = s[:, :1000].float().topk(5, dim=1)
        lse = torch.logsumexp(s[:, :1000].float(), 1) if tail else None
        leaf = s.detach().requires_grad_(True)
        loss = top_logit_distillation(leaf, values, indices, teacher_lse=lse)
        grad, = torch.autograd.grad(loss, leaf)
        assert loss.isfinite() and (grad[:, 1000:] == 0).all()
        short = s[:, :1000].contiguous().requires_grad_(True)
        want = top_logit_distillation(short, values, indices, teacher_lse=lse)
        want_grad, = torch.autograd.grad(want, short)
        # the sums of another length are added up in another order
        assert (loss - want).abs() <= 2.0**-16
        assert ((grad[:, :1000].float() - want_grad.float()).abs() <= 2.0**-7 * want_grad.float().abs() + 2.0**-17).all()


def test_distill_strides_graph_and_the_same_bits():
    wide = _logits(8, 2049, BF16)
    s = wide[::2, 1:2048]
    values, indices = s.float().topk(9, dim=1)
    first = _check_distill(s, values, indices, 0.5, 0.5, None, None)
    again = _check_distill(s, values, indices, 0.5, 0.5, None, None)
    assert all(torch.equal(a, b) for a, b in zip(first, again, strict=True))
    _check_distill(wide.t(), *wide.t().float().topk(3, dim=1), 1.0, 1.0, None, None)
    leaf = s.detach().clone().requires_grad_(True)

    def run():
        loss = top_logit_distillation(leaf, values, indices, tau=0.5, teacher_tau=0.5)
        return [loss.detach(), *torch.autograd.grad(loss, leaf)]

    want = run()
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        got = run()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want, strict=True))


def test_no_rows():
    s = torch.zeros(0, 50, device=DEV, requires_grad=True)
    loss = top_logit_distillation(s, torch.zeros(0, 3, device=DEV), torch.zeros(0, 3, device=DEV, dtype=torch.int64))
    assert loss.item() == 0 and torch.autograd.grad(loss, s)[0].shape == (0, 50)


def test_a_teacher_and_its_student_together():
    """Top logits of one network are what the other learns from; the divergence from itself is 0."""
    teacher = _logits(16, 8192, F32, size=0.3)
    values, indices, lse = top_logits(teacher, 64, tau=0.07)
    for tail in (None, lse):
        loss, grad = _check_distill(teacher, values, indices, 0.07, 0.07, tail, None)
        if tail is not None:  # with all classes in play the student is at the optimum
            assert loss.abs() <= 2.0**-14 and (grad.abs() <= 2.0**-14).all()
    _check_distill(_logits(16, 8192, BF16, 5, 0.3), values, indices, 0.1, 0.07, lse, None)


def test_second_derivatives_and_refusals():
    s = _logits(3, 100, F32).requires_grad_(True)
    values, indices = s.detach().topk(4, dim=1)
    loss = top_logit_distillation(s, values, indices)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(loss, s, create_graph=True)
    for bad in (
        lambda: top_logit_distillation(s.double(), values, indices),
        lambda: top_logit_distillation(s, values.cpu(), indices),
        lambda: top_logits(s.double(), 3),
        lambda: top_logits(s, 257),
        lambda: top_logits(s, 101),
        lambda: top_logits(s, 0),
        lambda: top_logits(s, 3, tau=0.0),
    ):
        with pytest.raises(ValueError):
            bad()


def test_offsets_beyond_32_bits():
    """The last of more than 2^31 logits give the same bits as in a tensor of their own (of 300 rows: fewer are summed by
    more threads, in another order)."""
    s = torch.zeros(33000, 65536, device=DEV, dtype=BF16)
    s[-3:] = _logits(3, 65536, BF16)
    near = s[-300:].clone()
    for got, want in zip(top_logits(s, 5), top_logits(near, 5), strict=True):
        assert torch.equal(got[-300:], want)
    values, indices, _ = top_logits(s, 4)
    w = torch.zeros(33000, device=DEV)
    w[-3:] = 1.0
    leaves = [s.requires_grad_(True), near.requires_grad_(True)]
    losses = [top_logit_distillation(x, values[-len(x):], indices[-len(x):], weights=w[-len(x):], norm=3.0) for x in leaves]
    assert torch.equal(*losses)
    grads = [torch.autograd.grad(loss, x)[0] for loss, x in zip(losses, leaves, strict=True)]
    assert torch.equal(grads[0][-300:], grads[1]) and not grads[0][:300].any() and grads[1][-3:].any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("weights", [None, F32, torch.float64])
def test_a_rest_of_the_teacher_far_below_one(dtype, weights):
    """The shares given sum to 1 - 3e-8 and the student is as sure: with teacher_lse in fp64 the others' gradient, which is
    all rest, has the bound's digits. (In fp32 an lse near 30 is off by 1e-6, thirty times the rest.)"""
    v = 3000
    s = torch.zeros(3, v, device=DEV)
    s[:, 0] = 40.0
    teacher = _logits(3, v, F32).double()
    teacher[:, 0] = 26.0
    values, indices = teacher.topk(2, dim=1)
    lse = torch.logsumexp(teacher, 1)
    assert ((1 - (values - lse[:, None]).exp().sum(1)) < 1e-7).all()
    w = torch.tensor([1.0, 0.0, 0.3], device=DEV, dtype=weights) if weights else None
    _, grad = _check_distill(s.to(dtype), values, indices, 1.0, 1.0, lse, w)
    if dtype != F16:  # the others' share of the rest: its bound says something
        assert (grad[0, 1:] < 0).any()


@pytest.mark.parametrize("kind", [BF16, F16, F32, torch.float64])
def test_distill_types_of_lse_and_weights(kind):
    s = _logits(3, 500, BF16)
    values, indices = s.float().topk(5, dim=1)
    lse, w = torch.logsumexp(s.double(), 1).to(kind) + 0.125, torch.tensor([0.5, 0.0, 2.0], device=DEV, dtype=kind)
    _check_distill(s, values, indices, 1.0, 1.0, lse, w)
    both = torch.stack([lse, w], 1)  # strided
    _check_distill(s, values, indices, 1.0, 1.0, both[:, 0], both[:, 1])


@pytest.mark.parametrize("where", ["value", "inf", "lse"])
@pytest.mark.parametrize("tail", [False, True])
def test_a_teacher_that_is_not_finite_shows_in_the_loss(where, tail):
    values = torch.tensor([[0.5, 0.0], [0.0, -1.0]], device=DEV)
    lse = torch.tensor([1.0, 1.0], device=DEV) if tail else None
    if where == "lse" and not tail:
        return
    if where == "lse":
        lse[0] = math.nan
    else:
        values[0, 1] = math.nan if where == "value" else math.inf
    s = _logits(2, 5, F32).requires_grad_(True)
    loss = top_logit_distillation(s, values, torch.tensor([[0, 1], [2, 3]], device=DEV), teacher_lse=lse)
    grad, = torch.autograd.grad(loss, s)
    assert not loss.isfinite() and not grad[0].isfinite().any() and grad[1].isfinite().all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tau", [1e-28, 1e-10, 1e10, 1e28])
def test_temperatures_at_the_ends_of_their_range(tau, dtype):
    """Where one logit stands for all, and where all are the same; logits of -inf have no share in either."""
    x = _logits(3, 1001, dtype)
    x[1, 5:900] = -math.inf
    x[2] = -math.inf
    x[2, 77] = 0.5
    values, indices, lse = top_logits(x, 3, tau=tau)
    want = torch.logsumexp(x.double() / tau, 1)
    top = (x.double() / tau).amax(1).abs()
    # as in _check_top; the sum itself is rounded to fp32
    assert ((lse.double() - want).abs() <= 2.0**-17 + 2.0**-22 * top).all()
    leaf = x.requires_grad_(True)
    loss = top_logit_distillation(leaf, values[:, :1], indices[:, :1], tau=tau)
    grad, = torch.autograd.grad(loss, leaf)
    # -log of the largest logit's probability: 0 where it stands for all, log of the number of others where all are the same
    count = torch.isfinite(x.detach()).sum(1).double()
    rows = torch.log(count) if tau > 1 else torch.zeros_like(count)
    assert (loss.double() - rows.mean()).abs() <= 2.0**-16
    assert grad.isfinite().all() and (grad[2] == 0).all()
