"""Attention over sequences of different lengths laid end to end, without padding them to one length.

`PackedSequences(lengths, key_lengths, causal=)` says which rows belong together; it is made once for a batch and
used by every layer. `packed_attention(q, k, v, sequences, scale)` takes q (Tq, Hq, D) and k, v (Tk, Hk, D), Hk a
divisor of Hq (query head h reads key head h // (Hq // Hk)), and returns (Tq, Hq, D): every query attends to the
keys of its own sequence. With `causal`, the last query of a sequence sees its last key, the one before it one key
less: query i of Lq sees the keys j <= i + Lk - Lq of Lk. A query that sees no key gives zeros and takes no part in
the gradients, and so do rows behind the last sequence, which are not read. A query whose scores are all -inf is 0 / 0: NaN.

On CUDA in bf16 and fp16 with D % 8 == 0 and D <= 128 this is the native kernel, in fp32 a native kernel without
tensor cores, a warp per row, for checks and small problems (2 x 1029 tokens, 16 heads of 64: 3.2 ms forward, 10.3 ms
backward); statistics and sums are held in fp32. The probabilities and their gradients are rounded to the inputs'
type on their way into the second matrix products; what rounding takes from the output is kept for the backward pass (a
second tensor of its size). Sums have a fixed order: the same inputs give the same bits. What a
sequence holds reaches no other sequence's results, not even an infinity or NaN. On the CPU it is PyTorch math,
sequence by sequence.
"""

from __future__ import annotations

import math
from collections.abc import Sequence

import numpy as np
import torch

from ._native import native, use_native

MAX_HEAD_DIM = 128
MAX_FEW = 16  # queries of a sequence that the kernel for few queries takes
PIECE = 512  # keys of a sequence that it takes at a time
_DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def _host_lengths(lengths: Sequence[int] | torch.Tensor, name: str) -> np.ndarray:
    if isinstance(lengths, torch.Tensor):
        if lengths.is_floating_point() or lengths.dtype == torch.bool:
            raise TypeError(f"{name} must be whole numbers, got {lengths.dtype}")
        lengths = lengths.detach().cpu().numpy()
    out = np.asarray(lengths)
    if out.size == 0:
        out = out.astype(np.int64)
    if out.ndim != 1 or not np.issubdtype(out.dtype, np.integer):
        raise TypeError(f"{name} must be a flat list of whole numbers, got {out.dtype} of shape {out.shape}")
    out = out.astype(np.int64)
    if (out < 0).any():
        raise ValueError(f"{name} must not be negative, got {out.min()}")
    if out.sum() >= 2**31 - 256:
        raise ValueError(f"{name} add up to {out.sum()} rows; at most {2**31 - 257}")
    return out


def capturing(device: torch.device) -> bool:
    """Whether what this thread launches on `device` now goes into a CUDA graph."""
    if device.type != "cuda":
        return False
    with torch.cuda.device(device):
        return torch.cuda.is_current_stream_capturing()


class PackedSequences:
    """Lengths of sequences laid end to end, and with them which query sees which key.

    `lengths` are the query rows of every sequence, `key_lengths` its key rows (the same where None). Built on the
    host: lengths on a CUDA device are read back first. The tables go to `device` before the constructor returns, which
    waits for that: it cannot be called while a graph is captured. A graph that was captured with a plan reads its tables in
    every replay, so the plan has to stay as long as the graph. Made in inference mode, a plan serves training too.
    """

    @torch.inference_mode(False)
    def __init__(
        self,
        lengths: Sequence[int] | torch.Tensor,
        key_lengths: Sequence[int] | torch.Tensor | None = None,
        *,
        causal: bool = False,
        device: torch.device | str | None = None,
    ) -> None:
        lq = _host_lengths(lengths, "lengths")
        lk = lq if key_lengths is None else _host_lengths(key_lengths, "key_lengths")
        if len(lq) != len(lk):
            raise ValueError(f"{len(lq)} lengths but {len(lk)} key_lengths")
        self.lengths = tuple(int(n) for n in lq)
        self.key_lengths = tuple(int(n) for n in lk)
        self.causal = bool(causal)
        self.num_queries, self.num_keys = int(lq.sum()), int(lk.sum())
        self.device = torch.device(device if device is not None else ("cuda" if torch.cuda.is_available() else "cpu"))
        if self.device.type == "cuda" and self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        if capturing(self.device):
            raise RuntimeError("PackedSequences are copied from the host: make them before a graph is captured")
        q0, k0 = np.concatenate([[0], np.cumsum(lq)[:-1]]), np.concatenate([[0], np.cumsum(lk)[:-1]])
        if len(lq) == 0:
            q0 = k0 = lq
        # keys [lo, hi) of every query and queries [lo, hi) of every key; neither end falls from row to row
        i, j = np.arange(self.num_queries) - np.repeat(q0, lq), np.arange(self.num_keys) - np.repeat(k0, lk)
        k_lo, k_hi = np.repeat(k0, lq), np.repeat(k0 + lk, lq)
        q_lo, q_hi = np.repeat(q0, lk), np.repeat(q0 + lq, lk)
        if self.causal:
            k_hi = k_lo + np.clip(i + 1 + np.repeat(lk - lq, lq), 0, np.repeat(lk, lq))
            q_lo = q_lo + np.clip(j - np.repeat(lk - lq, lk), 0, np.repeat(lq, lk))
        self.q_bounds = self._table(k_lo, k_hi)
        self.k_bounds = self._table(q_lo, q_hi)
        self.max_queries = int(lq.max(initial=0))
        self.pairs = int((k_hi - k_lo).sum())
        # scores that 128-row tiles compute: every tile all keys from its first row's first to its last row's last
        tiles = k_hi[np.minimum(np.arange(127, self.num_queries + 127, 128), self.num_queries - 1)] - k_lo[::128]
        self.tile_pairs = int((-(-np.maximum(tiles, 0) // 128)).sum()) * 128 * 128
        self.items = self.pieces = None
        if self.tile_pairs > 16 * self.pairs and self.max_queries <= MAX_FEW:
            self._make_items(q0, lq, k0, lk)

    def _make_items(self, q0: np.ndarray, lq: np.ndarray, k0: np.ndarray, lk: np.ndarray) -> None:
        """Pieces of at most `PIECE` keys of every sequence that has queries."""
        some = lq > 0
        q0, lq, k0, lk = q0[some], lq[some], k0[some], lk[some]
        count = np.maximum(-(-lk // PIECE), 1)
        first = np.cumsum(count) - count
        seq = np.repeat(np.arange(len(lq)), count)
        lo = k0[seq] + (np.arange(len(seq)) - first[seq]) * PIECE
        hi = np.minimum(lo + PIECE, (k0 + lk)[seq])
        self.items = torch.from_numpy(np.stack([q0[seq], lq[seq], lo, hi], 1).astype(np.int32)).to(self.device)
        self.pieces = self._table(first, count)

    def _table(self, lo: np.ndarray, hi: np.ndarray) -> torch.Tensor:
        # a copy from pageable memory: it is there when the call returns, for any stream
        return torch.from_numpy(np.stack([lo, hi], 1).astype(np.int32)).to(self.device)

    def __len__(self) -> int:
        return len(self.lengths)


def packed_attention_reference(
    q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, sequences: PackedSequences, scale: float
) -> torch.Tensor:
    acc = torch.promote_types(q.dtype, torch.float32)
    group = q.shape[1] // k.shape[1]
    outs, a, c = [], 0, 0
    for m, n in zip(sequences.lengths, sequences.key_lengths, strict=True):
        qs, ks, vs = q[a:a + m].to(acc), k[c:c + n].to(acc), v[c:c + n].to(acc)
        a, c = a + m, c + n
        blind = min(m, max(0, m - n)) if sequences.causal else (m if n == 0 else 0)
        if n == 0:
            blind = m
        outs.append(qs.new_zeros(blind, *qs.shape[1:]))
        if blind == m:
            continue
        ks, vs = ks.repeat_interleave(group, 1), vs.repeat_interleave(group, 1)
        score = torch.einsum("ihd,jhd->hij", qs[blind:], ks) * scale
        if sequences.causal:
            late = torch.ones(m - blind, n, dtype=torch.bool, device=q.device).triu(1 + n - (m - blind))
            score = score.masked_fill(late, -math.inf)
        outs.append(torch.einsum("hij,jhd->ihd", torch.softmax(score, -1), vs))
    outs.append(q.new_zeros(q.shape[0] - a, *q.shape[1:], dtype=acc))
    return torch.cat(outs).to(q.dtype)


def _check(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, sequences: PackedSequences) -> None:
    if q.dim() != 3 or k.dim() != 3 or k.shape != v.shape or q.shape[2] != k.shape[2]:
        raise ValueError(f"q must be (Tq, Hq, D), k and v (Tk, Hk, D) of one head size, got {tuple(q.shape)}, "
                         f"{tuple(k.shape)} and {tuple(v.shape)}")
    if not (q.dtype == k.dtype == v.dtype) or not q.is_floating_point() or not (q.device == k.device == v.device):
        raise ValueError(f"q, k and v must share a floating-point dtype and a device, got {q.dtype} on {q.device}, "
                         f"{k.dtype} on {k.device} and {v.dtype} on {v.device}")
    if k.shape[1] == 0 or q.shape[1] == 0 or q.shape[1] % k.shape[1] or q.shape[2] == 0:
        raise ValueError(f"{q.shape[1]} query heads of {q.shape[2]} channels cannot share {k.shape[1]} key heads")
    if q.shape[0] < sequences.num_queries or k.shape[0] < sequences.num_keys:
        raise ValueError(f"the sequences have {sequences.num_queries} queries and {sequences.num_keys} keys, q and k "
                         f"{q.shape[0]} and {k.shape[0]} rows")
    if sequences.device != q.device:
        raise ValueError(f"the sequences are on {sequences.device}, q on {q.device}")


def packed_attention(
    q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, sequences: PackedSequences, scale: float | None = None
) -> torch.Tensor:
    """Softmax attention within every sequence; see the module docstring. `scale` defaults to D ** -0.5."""
    _check(q, k, v, sequences)
    scale = q.shape[2] ** -0.5 if scale is None else float(scale)
    if not math.isfinite(scale):
        raise ValueError(f"scale must be finite, got {scale}")
    if use_native(q):
        d = q.shape[2]
        if q.dtype not in _DTYPES or d % 8 or d > MAX_HEAD_DIM:
            raise ValueError(f"on CUDA, packed_attention takes bf16, fp16 and fp32 heads of a multiple of 8 and at most "
                             f"{MAX_HEAD_DIM} channels, got {q.dtype} heads of {d}")
        if q.shape[1] > 65535:
            raise ValueError(f"at most 65535 query heads, got {q.shape[1]}")
        return native().packed_attention(q, k, v, sequences.q_bounds, sequences.k_bounds, scale, sequences.items,
                                         sequences.pieces, sequences.max_queries, sequences.tile_pairs, sequences.pairs)
    return packed_attention_reference(q, k, v, sequences, scale)
