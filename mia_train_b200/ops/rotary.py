"""Rotation of query and key heads by their tokens' positions, and frequencies for contexts longer than trained on.

`rotary(q, k, positions, frequencies, layout=, amplitude=)` turns the first 2 P channels of every head of q
(B, T, Hq, D) and k (B, T, Hk, D), or of (T, H, D) without a batch, as P pairs:

    angle[t, p] = sum_a positions[t, a] * frequencies[a, p]
    y1 = amplitude * (x1 cos - x2 sin),   y2 = amplitude * (x2 cos + x1 sin)

with the pairs (p, p + P) for `layout="half"` and (2 p, 2 p + 1) for `"interleaved"`; the other channels are copied.
`positions` are integers or floats, one per token, (T) or (B, T), with `frequencies` (P), or one coordinate per axis,
(T, A) or (B, T, A), with `frequencies` (A, P) and A <= 4. Without frequencies `positions` holds the angles themselves,
fp32 (T, P) or (B, T, P). Angles are reduced to a turn with at least 48 bits, of integer positions with 53, so that
those of far positions are as good as of near ones; the rest is fp32, rounded once. q and k may be strided views of a packed projection;
the outputs share one contiguous buffer. `k` may be None. Gradients go to q, k and the frequencies, not to positions or angles.
A frequency that is not finite makes its pairs NaN. On CUDA bf16, fp16 and fp32 heads of up to 256 channels are rotated by
the native kernel, other types and wider heads by PyTorch math, as everything on the CPU.

`rotary_frequencies(rotary_dim, base, scaling=...)` gives the frequencies base^(-p / P) in fp64 and the amplitude:

* "linear": positions are divided by `factor`.
* "ntk": the base grows so that the last pair's frequency is divided by `factor` and the first pair's kept.
* "yarn": pairs that turn more than `beta_fast` times over `original_length` are kept, those that turn less than
  `beta_slow` times are divided by `factor`, with a linear ramp over the pairs between, whose ends are whole pairs (below
  and above) within 0 .. rotary_dim - 1; the upper end may lie past the last pair, which then is not divided in full. The
  amplitude is 0.1 ln(factor) + 1.
"""

from __future__ import annotations

import math

import torch

from ._native import native, use_native

MAX_HEAD_DIM = 256
MAX_AXES = 4
LAYOUTS = ("half", "interleaved")
SCALINGS = (None, "linear", "ntk", "yarn")
_DTYPES = (torch.bfloat16, torch.float16, torch.float32)
_POSITIONS = (torch.int64, torch.int32, torch.float32, torch.float64)


def rotary_frequencies(
    rotary_dim: int,
    base: float = 10000.0,
    *,
    scaling: str | None = None,
    factor: float = 1.0,
    original_length: int | None = None,
    beta_fast: float = 32.0,
    beta_slow: float = 1.0,
    device: torch.device | str | None = None,
) -> tuple[torch.Tensor, float]:
    """(frequencies (rotary_dim // 2) fp64, amplitude); see the module docstring."""
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even and at least 2, got {rotary_dim}")
    if base <= 1.0:
        raise ValueError(f"rotary base must be greater than 1, got {base}")
    if scaling not in SCALINGS:
        raise ValueError(f"scaling must be one of {SCALINGS}, got {scaling!r}")
    if not factor >= 1.0:
        raise ValueError(f"factor must be at least 1, got {factor}")
    p = rotary_dim // 2
    pair = torch.arange(p, dtype=torch.float64)
    if scaling == "ntk" and p > 1:
        base = base * factor ** (p / (p - 1))
    freq = base ** -(pair / p)
    amplitude = 1.0
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "yarn":
        if original_length is None or original_length < 1 or not 0 < beta_slow < beta_fast:
            raise ValueError("yarn needs original_length >= 1 and 0 < beta_slow < beta_fast, got "
                             f"{original_length}, {beta_slow} and {beta_fast}")
        # a pair turns original_length * freq / (2 pi) times: solved for the pair's number
        low, high = (p * math.log(original_length / (turns * 2 * math.pi)) / math.log(base) for turns in (beta_fast, beta_slow))
        low, high = max(math.floor(low), 0), min(math.ceil(high), rotary_dim - 1)
        ramp = ((pair - low) / max(high - low, 1e-3)).clamp(0, 1)
        freq = freq * (1 - ramp) + freq / factor * ramp
        amplitude = 0.1 * math.log(factor) + 1.0
    return freq.to(device), amplitude


def _rotate_reference(x: torch.Tensor, angles: torch.Tensor, layout: str, amplitude: float) -> torch.Tensor:
    acc = torch.promote_types(x.dtype, torch.float32)
    p = angles.shape[-1]
    cos, sin = ((amplitude * f(angles)).to(acc).unsqueeze(-2) for f in (torch.cos, torch.sin))
    head, rest = x[..., :2 * p].to(acc), x[..., 2 * p:].to(acc)
    if layout == "half":
        x1, x2 = head[..., :p], head[..., p:]
        y = torch.cat([x1 * cos - x2 * sin, x2 * cos + x1 * sin], -1)
    else:
        x1, x2 = head[..., 0::2], head[..., 1::2]
        y = torch.stack([x1 * cos - x2 * sin, x2 * cos + x1 * sin], -1).flatten(-2)
    return torch.cat([y, rest], -1).to(x.dtype)


def rotary(
    q: torch.Tensor,
    k: torch.Tensor | None,
    positions: torch.Tensor,
    frequencies: torch.Tensor | None,
    *,
    layout: str = "half",
    amplitude: float = 1.0,
) -> tuple[torch.Tensor, torch.Tensor | None]:
    """Rotated (q, k); see the module docstring."""
    if layout not in LAYOUTS:
        raise ValueError(f"layout must be one of {LAYOUTS}, got {layout!r}")
    if not math.isfinite(amplitude):
        raise ValueError(f"amplitude must be finite, got {amplitude}")
    if q.dim() not in (3, 4) or not q.is_floating_point():
        raise ValueError(f"q must be a floating-point (T, H, D) or (B, T, H, D), got {q.dtype} {tuple(q.shape)}")
    if k is not None and (k.dim() != q.dim() or k.shape[:-2] != q.shape[:-2] or k.shape[-1] != q.shape[-1]
                          or k.dtype != q.dtype or k.device != q.device):
        raise ValueError(f"q and k must share tokens, head size, dtype and device, got {q.dtype} {tuple(q.shape)} on "
                         f"{q.device} and {k.dtype} {tuple(k.shape)} on {k.device}")
    batched = q.dim() == 4
    b, t, hq, d = q.shape if batched else (1, *q.shape)
    if t >= 2**31:
        raise ValueError(f"at most {2**31 - 1} tokens in a row of the batch, got {t}")
    if frequencies is None:
        if positions.dim() not in (2, 3) or positions.dtype != torch.float32:
            raise ValueError(f"angles must be fp32 (T, P) or (B, T, P), got {positions.dtype} {tuple(positions.shape)}")
        multi, table, axes, p = True, None, positions.shape[-1], positions.shape[-1]
    elif frequencies.dim() not in (1, 2) or frequencies.dtype not in (torch.float32, torch.float64):
        raise ValueError(f"frequencies must be fp32 or fp64 (P) or (A, P), got {frequencies.dtype} {tuple(frequencies.shape)}")
    else:
        multi = frequencies.dim() == 2
        table = frequencies if multi else frequencies.unsqueeze(0)
        axes, p = table.shape
    if 2 * p > d or (table is not None and not 1 <= axes <= MAX_AXES):
        raise ValueError(f"{axes} axes and {p} pairs: at most {MAX_AXES} axes and {d // 2} pairs of a head of {d}")
    where = positions if multi else positions.unsqueeze(-1)
    if positions.dtype not in _POSITIONS or tuple(where.shape) not in {(t, axes), (1, t, axes), (b, t, axes)}:
        raise ValueError(f"positions must be int32, int64, fp32 or fp64 for {t} tokens of {b} rows and {axes} axes, got "
                         f"{positions.dtype} {tuple(positions.shape)}")
    if positions.device != q.device or (table is not None and table.device != q.device):
        raise ValueError(f"q is on {q.device}, positions on {positions.device}, frequencies on "
                         f"{table.device if table is not None else None}")
    if positions.requires_grad:
        raise ValueError("rotary gives no gradient for positions")
    if where.dim() == 2:
        where = where.unsqueeze(0)
    if q.dtype in _DTYPES and d <= MAX_HEAD_DIM and use_native(q):
        q4 = q if batched else q.unsqueeze(0)
        k4 = q4[:, :, :0].detach() if k is None else (k if batched else k.unsqueeze(0))
        yq, yk = native().rotary(q4, k4, where, table, layout == "interleaved", float(amplitude))
        if not batched:
            yq, yk = yq.squeeze(0), yk.squeeze(0)
        return yq, (None if k is None else yk)
    angles = where.double() if table is None else (where.double().unsqueeze(-1) * table.double()).sum(-2)
    if not batched:
        angles = angles.squeeze(0)
    return (_rotate_reference(q, angles, layout, amplitude),
            None if k is None else _rotate_reference(k, angles, layout, amplitude))
