"""What the CPU path of the 8-bit linear layer keeps between forward and backward."""

from __future__ import annotations

import pytest
import torch

from mia_train_b200.ops.fp8 import fp8_linear


def _linear(act=None, gamma=True):
    torch.manual_seed(1)
    t = {"x": torch.randn(5, 32).bfloat16(), "weight": torch.randn(8, 32), "bias": torch.randn(8)}
    if gamma:
        t["gamma"] = torch.rand(8)
    t = {k: v.requires_grad_(True) for k, v in t.items()}
    return t, lambda: fp8_linear(t["x"], t["weight"], t["bias"], activation=act, gamma=t.get("gamma"))


@pytest.mark.parametrize("act", [None, "gelu"])
@pytest.mark.parametrize("name", ["gamma", "bias"])
def test_vectors_changed_before_backward_are_refused(name, act):
    t, run = _linear(act)
    y = run()
    with torch.no_grad():
        t[name].add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.float().sum().backward()


@pytest.mark.parametrize("name", ["x", "weight", "bias"])
def test_changes_of_what_backward_does_not_read_are_allowed(name):
    t, run = _linear("gelu", gamma=False)
    dy = torch.randn(5, 8).bfloat16()
    leaves = list(t.values())
    want = torch.autograd.grad(run(), leaves, dy)
    y = run()
    with torch.no_grad():
        t[name].mul_(3)
    for a, b in zip(torch.autograd.grad(y, leaves, dy), want, strict=True):
        assert torch.equal(a, b)


@pytest.mark.parametrize("mode", ["no_grad", "constants", "gamma_only"])
def test_gelu_without_a_product_gradient_keeps_no_preactivation(mode, monkeypatch):
    import mia_train_b200.ops.fp8 as fp8

    asked = []
    real = fp8.fp8_gemm
    monkeypatch.setattr(fp8, "fp8_gemm", lambda *a, **kw: asked.append(kw.get("aux_out")) or real(*a, **kw))
    quantised = []
    both = fp8._quantize
    monkeypatch.setattr(fp8, "_quantize", lambda *a, **kw: quantised.append(a[4]) or both(*a, **kw))
    t, run = _linear("gelu")
    for k, v in t.items():
        v.requires_grad_(mode == "no_grad" or (mode == "gamma_only" and k == "gamma"))
    with torch.set_grad_enabled(mode != "no_grad"):
        y = run()
    assert asked == [None] and quantised == [False, False]
    if mode == "gamma_only":
        (g,) = torch.autograd.grad(y.float().sum(), t["gamma"])
        for v in t.values():
            v.requires_grad_(True)
        assert torch.equal(g, torch.autograd.grad(run().float().sum(), t["gamma"])[0])


@pytest.mark.parametrize("act,wanted", [(None, ("x", "weight")), (None, ("gamma", "bias")), (None, ("gamma", "x")),
                                        ("gelu", ("x",)), ("gelu", ("weight",)), ("gelu", ("bias",))])
def test_second_derivative_is_refused_for_a_constant_gradient(act, wanted):
    t, run = _linear(act, gamma="gamma" in wanted)
    for k, v in t.items():
        v.requires_grad_(k in wanted)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(run().float().sum(), t[wanted[0]], create_graph=True)


@pytest.mark.parametrize("wanted", ["x", "weight", "gamma", "bias"])
def test_a_linear_layer_has_no_second_derivative_in_one_operand(wanted):
    t, run = _linear()
    for k, v in t.items():
        v.requires_grad_(k == wanted)
    want = torch.autograd.grad(run().float().sum(), t[wanted])[0]
    got = torch.autograd.grad(run().float().sum(), t[wanted], create_graph=True)[0]
    assert torch.equal(got, want) and not got.requires_grad
