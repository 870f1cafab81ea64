"""What the native nodes keep between forward and backward: seen by autograd's checks, and no more than is read."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover - collected on CPU, skipped there
    pytest.skip("needs CUDA", allow_module_level=True)

from mia_train_b200.ops.fp8 import fp8_linear  # noqa: E402
from mia_train_b200.ops.qk_norm import qk_norm_rope, qk_norm_rope_attention  # noqa: E402

DEV = torch.device("cuda", 0)
BF16 = torch.bfloat16
CHANGED = "modified by an inplace operation"


def _half_pairs(d):
    i = torch.arange(d // 2)
    return torch.stack([i, i + d // 2], 1).int().to(DEV)


def _heads():
    torch.manual_seed(0)
    pairs = _half_pairs(64)
    t = {"q": torch.randn(2, 5, 3, 64, device=DEV).bfloat16(), "k": torch.randn(2, 5, 3, 64, device=DEV).bfloat16(),
         "qw": torch.rand(64, device=DEV), "kw": torch.rand(64, device=DEV),
         "angles": torch.randn(1, 5, 32, device=DEV), "pairs": pairs}
    for key in ("q", "k", "qw", "kw", "angles"):
        t[key].requires_grad_(True)
    return t


@pytest.mark.parametrize("name", ["q", "k", "qw", "kw", "angles", "pairs"])
@pytest.mark.parametrize("entry", ["norm", "attention"])
def test_head_norm_refuses_operands_changed_before_backward(name, entry):
    t = _heads()
    if entry == "norm":
        y = qk_norm_rope(t["q"], t["k"], t["qw"], t["kw"], t["angles"], t["pairs"])[0]
    else:
        packed = torch.stack([t["q"], t["k"], t["k"]], 2).detach().requires_grad_(True)
        t["q"] = t["k"] = packed
        y = qk_norm_rope_attention(packed, t["qw"], t["kw"], t["angles"], t["pairs"], 0.125)
    with torch.no_grad():
        t[name].add_(1)
    with pytest.raises(RuntimeError, match=CHANGED):
        y.float().sum().backward()


@pytest.mark.parametrize("dtype", [torch.float32, BF16])
def test_head_norm_takes_converted_weights_as_they_were(dtype):
    """A weight in another type is converted in the forward pass; the copy is what backward differentiates with."""
    t = _heads()
    qw = t["qw"].detach().to(dtype)
    dy = torch.randn_like(t["q"])

    def grads(change):
        w = qw.clone().requires_grad_(True)
        y = qk_norm_rope(t["q"], t["k"], w, None, t["angles"], t["pairs"])[0]
        if change:
            with torch.no_grad():
                w.mul_(3)
        return torch.autograd.grad(y, (t["q"], w, t["angles"]), dy)

    if dtype == torch.float32:
        with pytest.raises(RuntimeError, match=CHANGED):
            grads(True)
        return
    for a, b in zip(grads(False), grads(True), strict=True):
        assert torch.equal(a, b)


def _linear(act=None, gamma=True, n=64):
    torch.manual_seed(1)
    t = {"x": torch.randn(40, 32, device=DEV).bfloat16(), "weight": torch.randn(n, 32, device=DEV),
         "bias": torch.randn(n, device=DEV), "gamma": torch.rand(n, device=DEV) if gamma else None}
    t = {k: v.requires_grad_(True) for k, v in t.items() if v is not None}
    return t, lambda: fp8_linear(t["x"], t["weight"], t["bias"], activation=act, gamma=t.get("gamma"))


@pytest.mark.parametrize("act", [None, "gelu"])
@pytest.mark.parametrize("name", ["gamma", "bias"])
def test_linear_refuses_vectors_changed_before_backward(name, act):
    """gamma scales the gradient of the product, bias is in the recomputed activation behind gamma's own gradient."""
    t, run = _linear(act)
    y = run()
    with torch.no_grad():
        t[name].add_(1)
    with pytest.raises(RuntimeError, match=CHANGED):
        y.float().sum().backward()


@pytest.mark.parametrize("name", ["x", "weight", "bias"])
def test_linear_allows_changes_of_what_backward_does_not_read(name):
    """x and weight are kept as 8-bit copies, and without gamma nothing in the backward pass depends on the bias."""
    t, run = _linear("gelu", gamma=False)
    dy = torch.randn(40, 64, device=DEV).bfloat16()
    leaves = list(t.values())
    want = torch.autograd.grad(run(), leaves, dy)
    y = run()
    with torch.no_grad():
        t[name].mul_(3)
    for a, b in zip(torch.autograd.grad(y, leaves, dy), want, strict=True):
        assert torch.equal(a, b)


M, K, N = 512, 1024, 1024
# 8-bit x and weight with their scales (the allocator hands out multiples of 512 bytes), and y
OPERANDS = M * K + 4 * M * K // 128 + N * K + 512
OUTPUT = 2 * M * N


@pytest.mark.parametrize("mode", ["no_grad", "inference_mode", "constants", "residual_only"])
def test_gelu_without_a_backward_writes_no_preactivation(mode):
    torch.manual_seed(2)
    x, w = torch.randn(M, K, device=DEV).bfloat16(), torch.randn(N, K, device=DEV)
    b, res = torch.randn(N, device=DEV), torch.randn(M, N, device=DEV).bfloat16()
    train = mode in ("no_grad", "inference_mode")
    for t in (x, w, b):
        t.requires_grad_(train)
    res.requires_grad_(mode == "residual_only")
    grad = {"no_grad": torch.no_grad(), "inference_mode": torch.inference_mode()}.get(mode, torch.enable_grad())

    def run():
        with grad:
            return fp8_linear(x, w, b, activation="gelu", residual=res)

    first = run()
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    y = run()
    assert torch.cuda.max_memory_allocated() - before == OPERANDS + OUTPUT
    assert torch.equal(y, first) and y.requires_grad == (mode == "residual_only")


def test_gelu_output_does_not_depend_on_grad_mode():
    """With its pre-activation the residual takes another form of the epilogue: the numbers stay the same."""
    torch.manual_seed(3)
    x, w = torch.randn(300, 256, device=DEV).bfloat16(), torch.randn(264, 256, device=DEV, requires_grad=True)
    b, g = torch.randn(264, device=DEV), torch.rand(264, device=DEV)
    res = torch.randn(300, 264, device=DEV).bfloat16()
    for kw in (dict(), dict(gamma=g), dict(residual=res), dict(gamma=g, residual=res)):
        y = fp8_linear(x, w, b, activation="gelu", **kw)
        with torch.no_grad():
            z = fp8_linear(x, w, b, activation="gelu", **kw)
        # the same fp32 terms, but product and sum may be one rounding or two (half a step, 2^-24, of either term):
        # that moves a rounding to bf16 by a step (at most 2^-7) where it falls between two, one time in 2^14 or so
        gap = (y.detach().double() - z.double()).abs()
        term = res.double().abs() if "residual" in kw else torch.zeros_like(gap)
        assert (gap <= z.double().abs() * 2.0**-7 + (2 * term + z.double().abs()) * 2.0**-23).all()
        assert (gap > 0).double().mean() < 2.0**-8


def test_gamma_alone_needs_no_preactivation():
    t, run = _linear("gelu")
    dy = torch.randn(40, 64, device=DEV).bfloat16()
    want = torch.autograd.grad(run(), t["gamma"], dy)[0]
    for k, v in t.items():
        v.requires_grad_(k == "gamma")
    assert torch.equal(torch.autograd.grad(run(), t["gamma"], dy)[0], want)


@pytest.mark.parametrize("second", [("x", "weight"), ("gamma", "bias"), ("gamma", "x"), ("gamma", "weight")])
def test_second_derivative_of_a_linear_layer_is_refused_for_a_constant_gradient(second):
    t, run = _linear()
    for k, v in t.items():
        v.requires_grad_(k in second)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(run().float().sum(), t[second[0]], create_graph=True)


@pytest.mark.parametrize("leaf", ["x", "weight", "bias"])
def test_second_derivative_behind_an_activation_is_refused(leaf):
    t, run = _linear("gelu", gamma=False)
    for k, v in t.items():
        v.requires_grad_(k == leaf)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(run().float().sum(), t[leaf], create_graph=True)


@pytest.mark.parametrize("wanted", ["x", "weight", "gamma", "bias"])
def test_linear_layers_have_no_second_derivative_in_one_operand(wanted):
    """The layer is linear in each operand alone: the gradient is a constant, and is returned as one."""
    t, run = _linear()
    for k, v in t.items():
        v.requires_grad_(k == wanted)
    want = torch.autograd.grad(run().float().sum(), t[wanted])[0]
    got = torch.autograd.grad(run().float().sum(), t[wanted], create_graph=True)[0]
    assert torch.equal(got, want) and not got.requires_grad


@pytest.mark.parametrize("leaf", ["q", "k", "angles"])
@pytest.mark.parametrize("entry", ["norm", "attention"])
def test_second_derivative_of_head_norms_is_refused_for_a_constant_gradient(leaf, entry):
    t = _heads()
    packed = torch.stack([t["q"], t["k"], t["k"]], 2).detach().requires_grad_(leaf != "angles")
    for k, v in t.items():
        if k != "pairs":
            v.requires_grad_(k == leaf)
    if entry == "norm":
        y = sum(o.float().sum() for o in qk_norm_rope(t["q"], t["k"], t["qw"], t["kw"], t["angles"], t["pairs"]))
    else:
        y = qk_norm_rope_attention(packed, t["qw"], t["kw"], t["angles"], t["pairs"], 0.125).float().sum()
    wrt = t[leaf] if entry == "norm" or leaf == "angles" else packed
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(y, wrt, create_graph=True)


def test_dropout_of_a_constant_gradient_needs_no_second_derivative():
    from mia_train_b200.ops.dropout import dropout

    x = torch.randn(40, 64, device=DEV, requires_grad=True)
    rng = torch.tensor([3, 4], device=DEV)
    got = torch.autograd.grad(dropout(x, 0.5, rng=rng).sum(), x, create_graph=True)[0]
    assert torch.equal(got, torch.autograd.grad(dropout(x, 0.5, rng=rng).sum(), x)[0])
