"""Distillation from a teacher of which only every row's top logits are kept.

`top_logits(logits, k, tau)` gives the k largest logits of every row (largest first, equal ones by the lower index;
a NaN counts as larger than every number), their classes (int64) and logsumexp(logits / tau) in fp32, in one
kernel that sorts no row. `top_logit_distillation(student, values, indices, ...)` is the Kullback-Leibler divergence

    sum_r weights_r * sum_j p_rj (log p_rj - log q_rj) / norm,    q = softmax(student / tau)

of a student (R, V) from the teacher's shares p of the classes `indices` (R, K), K <= 1024:

* without `teacher_lse`, p = softmax(values / teacher_tau) over the given classes;
* with `teacher_lse` (R) = logsumexp(all of the teacher's logits / teacher_tau), p = exp(values / teacher_tau -
  teacher_lse), and the classes that are not given count as one more, with the rest of 1 for p and the student's
  mass outside the given classes for q.

An index outside 0 .. V - 1 is left out (lists of different lengths are filled up with -1), and a row of weight 0 is not
read and gives zeros, whatever it holds. `norm` defaults to R. A class that a row names twice has the sum of its shares in
the gradient; the loss adds p_j log p_j entry by entry, as the formula has it, which is less than with both entries in
one by a number that does not depend on the student (such a loss can be negative).
The teacher and the weights get no gradient. A teacher logit of -inf has no share. Shares, their rest of 1 and the loss are
computed in 64 bits; `values` and `teacher_lse` are taken as precise as they come, so a rest that is far below 1 needs them
in fp64 (an fp32 lse of 20 moves it by 1e-6).
"""

from __future__ import annotations

import math

import torch

from ._native import native, use_native

MAX_TOP = 256
MAX_GIVEN = 1024
MAX_CLASSES = 1 << 20  # a bit for every class fits the shared memory of a block
TAUS = 1e-28, 1e28  # log2(e) / tau and what fp32 leaves of it are fp32 numbers
_DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def _positive(value: float, name: str) -> float:
    if not (math.isfinite(value) and value > 0):
        raise ValueError(f"{name} must be positive and finite, got {value}")
    return float(value)


def _temperature(value: float, name: str) -> float:
    if not TAUS[0] <= value <= TAUS[1]:
        raise ValueError(f"{name} must be within {TAUS[0]} .. {TAUS[1]}, got {value}")
    return float(value)


def top_logits_reference(logits: torch.Tensor, k: int, tau: float):
    acc = torch.promote_types(logits.dtype, torch.float32)
    values, indices = torch.sort(logits, dim=1, descending=True, stable=True)
    return values[:, :k].contiguous(), indices[:, :k].contiguous(), torch.logsumexp(logits.to(acc) / tau, 1).float()


@torch.no_grad()
def top_logits(logits: torch.Tensor, k: int, *, tau: float = 1.0) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(values (R, k), indices (R, k) int64, log-sum-exp (R) fp32) of logits (R, V); see the module docstring."""
    if logits.dim() != 2 or not logits.is_floating_point():
        raise ValueError(f"logits must be a floating-point (R, V), got {logits.dtype} {tuple(logits.shape)}")
    if not 1 <= k <= min(MAX_TOP, logits.shape[1]):
        raise ValueError(f"k must be in 1 .. {min(MAX_TOP, logits.shape[1])}, got {k}")
    _temperature(tau, "tau")
    if use_native(logits):
        if logits.dtype not in _DTYPES or logits.shape[1] >= 2**31 - 1024 or logits.shape[0] >= 2**31:
            raise ValueError(f"on CUDA, top_logits takes bf16, fp16 and fp32, got {logits.dtype} {tuple(logits.shape)}")
        return native().top_logits(logits, int(k), float(tau))
    return top_logits_reference(logits, k, tau)


def top_logit_distillation_reference(student, values, indices, tau, teacher_tau, teacher_lse, weights, norm):
    acc = torch.promote_types(student.dtype, torch.float32)
    r, v = student.shape
    w = torch.ones(r, device=student.device) if weights is None else weights
    read = (w != 0).unsqueeze(1)
    given = (indices >= 0) & (indices < v) & read
    at = torch.where(given, indices, 0).long()
    log_q = torch.log_softmax(torch.where(read, student.to(acc), 0.0) / tau, 1)
    t = torch.where(given, values.double(), -math.inf) / teacher_tau
    lse = torch.logsumexp(t, 1, keepdim=True) if teacher_lse is None else teacher_lse.double().unsqueeze(1)
    p = torch.where(given & (t != -math.inf), (t - lse).exp(), 0.0)
    some = p != 0  # a NaN among them stays one
    log_p = torch.where(some, t - lse, 0.0)
    rows = torch.where(some, p * (log_p - log_q.gather(1, at).double()), 0.0).sum(1)
    if teacher_lse is not None:
        outside = torch.ones_like(log_q, dtype=torch.int32).scatter_reduce(1, at, (~given).int(), "amin") > 0
        rest = torch.where(outside.any(1), (1 - p.sum(1)).clamp(min=0), 0.0)
        others = torch.logsumexp(torch.where(outside, log_q, -math.inf), 1).double()
        has = rest != 0
        rows = rows + torch.where(has, rest * (torch.where(has, rest, 1.0).log() - torch.where(has, others, 0.0)), 0.0)
    return (torch.where(read[:, 0], rows * w.double(), 0.0).sum() / norm).float()


def top_logit_distillation(
    student: torch.Tensor,
    values: torch.Tensor,
    indices: torch.Tensor,
    *,
    tau: float = 1.0,
    teacher_tau: float = 1.0,
    teacher_lse: torch.Tensor | None = None,
    weights: torch.Tensor | None = None,
    norm: float | None = None,
) -> torch.Tensor:
    """The divergence (a scalar, fp32) of student (R, V) from a teacher's top logits; see the module docstring."""
    if student.dim() != 2 or student.shape[1] == 0 or not student.is_floating_point():
        raise ValueError(f"student must be a floating-point (R, V), got {student.dtype} {tuple(student.shape)}")
    r, v = student.shape
    if r >= 2**31:
        raise ValueError(f"at most {2**31 - 1} rows, got {r}")
    if values.dim() != 2 or values.shape != indices.shape or values.shape[0] != r or not 1 <= values.shape[1] <= MAX_GIVEN:
        raise ValueError(f"values and indices must be ({r}, 1 .. {MAX_GIVEN}), got {tuple(values.shape)} and "
                         f"{tuple(indices.shape)}")
    if not values.is_floating_point() or indices.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"values must be floating-point, indices int32 or int64, got {values.dtype} and {indices.dtype}")
    for name, x in (("teacher_lse", teacher_lse), ("weights", weights)):
        if x is not None and (x.shape != (r,) or not x.is_floating_point()):
            raise ValueError(f"{name} must be a floating-point vector of {r}, got {x.dtype} {tuple(x.shape)}")
    for name, x in (("values", values), ("indices", indices), ("teacher_lse", teacher_lse), ("weights", weights)):
        if x is not None and x.device != student.device:
            raise ValueError(f"student is on {student.device}, {name} on {x.device}")
    tau, teacher_tau = _temperature(tau, "tau"), _temperature(teacher_tau, "teacher_tau")
    norm = _positive(float(max(r, 1)) if norm is None else float(norm), "norm")
    values, teacher_lse, weights = (x.detach() if x is not None else None for x in (values, teacher_lse, weights))
    if use_native(student):
        if student.dtype not in _DTYPES or values.dtype not in (*_DTYPES, torch.float64) or v > MAX_CLASSES:
            raise ValueError(f"on CUDA, top_logit_distillation takes bf16, fp16 and fp32 students of at most {MAX_CLASSES} "
                             f"classes, got {student.dtype} {tuple(student.shape)} and {values.dtype} values")
        return native().top_logit_distillation(student, values, indices, teacher_lse, weights, tau, teacher_tau, norm)
    return top_logit_distillation_reference(student, values, indices, tau, teacher_tau, teacher_lse, weights, norm)
