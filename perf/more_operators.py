"""Cases that measure the operators of packed sequences and of distillation from stored teacher logits.

Four families, in the order a step runs them:

* ``rot``: rotation of query and key heads by angles computed from the tokens' positions (one number or a
  coordinate per axis) and a table of frequencies; half or interleaved channel pairs, the whole head or
  part of it: forward, or forward with the gradients of q, k and the frequencies.
* ``attn``: softmax attention over sequences of different lengths laid end to end, with fewer key than
  query heads and an optional causal mask (the last query of a sequence sees its last key): forward, or
  forward with the gradients of q, k and v. Rows behind the last sequence give zeros.
* ``top``: the k largest logits of every row with their indices, largest first and ties by the lowest
  index, and the row's log-sum-exp at a temperature.
* ``distill``: the Kullback-Leibler divergence of a student's classes from a teacher's top logits, over
  those classes alone or with one more class for all others: loss and gradient.

``own`` is set from outside: False computes the plain forms with elementary torch operations, True
calls ``mia_train_b200.ops``.
"""

from __future__ import annotations

import math

import torch

own = False


# ------------------------------------------------------------------------------------------ cases


def listed() -> list[dict]:
    return [
        # One crop of eight patches with its class token through a small encoder, evaluation: the
        # smallest call.
        {"name": "rot_small_crop", "op": "rot", "train": False, "b": 1, "t": 9, "hq": 6, "hk": 6, "d": 64, "rotary": 64,
         "layout": "half", "axes": 1, "scaling": "none", "dtype": "bf16"},
        # A packed batch of long token sequences with grouped heads, half of each head rotated, frequencies
        # stretched for a longer context.
        {"name": "rot_long_grouped_train", "op": "rot", "train": True, "b": 1, "t": 16384, "hq": 32, "hk": 8, "d": 128,
         "rotary": 64, "layout": "interleaved", "axes": 1, "scaling": "yarn", "dtype": "bf16"},
        # Volumes of 4096 patches with a class token and four registers, three coordinates a token,
        # learned frequencies.
        {"name": "rot_volume_learned_train", "op": "rot", "train": True, "b": 4, "t": 4101, "hq": 16, "hk": 16, "d": 64,
         "rotary": 64, "layout": "half", "axes": 3, "scaling": "none", "dtype": "bf16"},
        # Eight small crops of nine tokens in one call, evaluation: launch latency.
        {"name": "attn_small_crops", "op": "attn", "train": False, "lq": "8x9", "lk": "", "causal": False, "hq": 6, "hk": 6,
         "d": 64, "pad": 0, "dtype": "bf16"},
        # The multi-crop batch of a ViT-H-class encoder: 16 crops of 512 patches and 64 of 64, each with a
        # class token and four registers.
        {"name": "attn_multicrop_train", "op": "attn", "train": True, "lq": "16x517,64x69", "lk": "", "causal": False,
         "hq": 20, "hk": 20, "d": 64, "pad": 0, "dtype": "bf16"},
        # Four volumes of 4096 patches, a class token and four registers.
        {"name": "attn_volumes_train", "op": "attn", "train": True, "lq": "4x4101", "lk": "", "causal": False, "hq": 16,
         "hk": 16, "d": 64, "pad": 0, "dtype": "bf16"},
        # Token sequences of every length in one padded batch, causal, four query heads to a key head.
        {"name": "attn_causal_ragged_train", "op": "attn", "train": True, "lq": "8192,1,5003,131,2048,777,0,2999,64", "lk": "",
         "causal": True, "hq": 16, "hk": 4, "d": 128, "pad": 41, "dtype": "bf16"},
        # Attention pooling: one query per volume over all of its tokens, evaluation.
        {"name": "attn_pool_single_queries", "op": "attn", "train": False, "lq": "16x1", "lk": "8x4101,4x4096,4x1029",
         "causal": False, "hq": 16, "hk": 16, "d": 64, "pad": 0, "dtype": "fp16"},
        # The class tokens of eight samples' two global crops over a head of 65536 prototypes.
        {"name": "top_class_tokens", "op": "top", "r": 16, "v": 65536, "k": 32, "tau": 0.07, "dtype": "fp32"},
        # The masked patches of the same batch.
        {"name": "top_masked_patches", "op": "top", "r": 1229, "v": 65536, "k": 64, "tau": 0.07, "dtype": "bf16"},
        # A few rows of a small head, in 32 bits: launch latency.
        {"name": "distill_few_rows", "op": "distill", "r": 4, "v": 1000, "k": 8, "tail": False, "weights": False,
         "tau": 0.1, "teacher_tau": 0.07, "dtype": "fp32"},
        # The masked patches of a batch against a stored teacher, the other prototypes as one class.
        {"name": "distill_masked_patches", "op": "distill", "r": 1229, "v": 65536, "k": 64, "tail": True, "weights": True,
         "tau": 0.1, "teacher_tau": 0.07, "dtype": "bf16"},
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    op = rng.choice(("rot", "attn", "attn", "top", "distill"))
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    if op == "rot":
        d = rng.choice((32, 40, 64, 64, 80, 96, 128))
        rotary = rng.choice((d, d, d // 2, d // 4 * 2))
        hk = rng.randint(1, 16)
        hq = hk * rng.choice((1, 1, 2, 4)) if hk <= 8 else hk
        b = _log_int(rng, 1, 8)
        t = _log_int(rng, 1, max(1, 16384 * 40 * 128 // (2 * b * (hq + hk) * d)))
        return {"op": "rot", "train": rng.random() < 0.6, "b": b, "t": min(t, 32768), "hq": hq, "hk": hk, "d": d,
                "rotary": rotary, "layout": rng.choice(("half", "interleaved")), "axes": rng.choice((1, 1, 2, 3)),
                "scaling": rng.choice(("none", "linear", "ntk", "yarn")), "dtype": dtype}
    if op == "attn":
        d = rng.choice((32, 40, 64, 64, 80, 96, 128))
        hk = rng.choice((1, 2, 4, 5, 8))
        hq = hk * rng.choice((1, 1, 2, 3, 4))
        causal = rng.random() < 0.5
        cross = rng.random() < 0.3
        kinds = rng.choice((1, 1, 2, 3, 5))
        lq, lk, budget = [], [], 4.0e10 / (hq * d)
        for _ in range(kinds):
            a = rng.choice((0, 1, _log_int(rng, 2, 128), _log_int(rng, 2, 4096), _log_int(rng, 128, 8192)))
            c = rng.choice((0, 1, _log_int(rng, 2, 4096), _log_int(rng, 128, 8192))) if cross else a
            n = min(_log_int(rng, 1, 64), int(budget / kinds / max(1, a * c)), 40000 // kinds // max(1, a, c))
            lq.append(f"{max(1, n)}x{a}" if n >= 1 else "1x1")
            lk.append(f"{max(1, n)}x{c}" if n >= 1 else "1x1")
        lq.append("2x7")  # never without a query
        lk.append("2x7")
        return {"op": "attn", "train": rng.random() < 0.6, "lq": ",".join(lq), "lk": ",".join(lk) if cross else "",
                "causal": causal, "hq": hq, "hk": hk, "d": d, "pad": rng.choice((0, 0, 3, 200)),
                "dtype": rng.choice(("bf16", "bf16", "fp16"))}
    v = rng.choice((_log_int(rng, 64, 131072), _log_int(rng, 64, 131072) // 8 * 8, 65536))
    r = _log_int(rng, 1, max(1, min(8192, 30_000_000 // v)))
    k = min(_log_int(rng, 1, 256), v)
    if op == "top":
        return {"op": "top", "r": r, "v": v, "k": k, "tau": round(rng.uniform(0.04, 2.0), 3), "dtype": dtype}
    return {"op": "distill", "r": r, "v": v, "k": k, "tail": rng.random() < 0.5 and k < v, "weights": rng.random() < 0.5,
            "tau": round(rng.uniform(0.05, 2.0), 3), "teacher_tau": round(rng.uniform(0.04, 2.0), 3), "dtype": dtype}


def _lengths(text: str) -> list[int]:
    """"2x7,5" -> [7, 7, 5]"""
    out = []
    for part in filter(None, text.split(",")):
        n, _, length = part.rpartition("x")
        out += [int(length)] * int(n or 1)
    return out


def _visible(lq: int, lk: int, causal: bool) -> int:
    """Query-key pairs that a sequence's mask leaves: query i sees the keys j <= i + lk - lq."""
    if not causal:
        return lq * lk
    first = lk - lq + 1  # keys that the first query sees
    skipped = min(lq, max(0, 1 - first))  # queries that see none
    n = lq - skipped
    return n * (max(first, 1) + lk) // 2 if n > 0 else 0


SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


def work(case: dict) -> dict:
    op = case["op"]
    if op == "rot":
        rows = case["b"] * case["t"] * (case["hq"] + case["hk"])
        e, f = SIZE[case["dtype"]], 8 * case["axes"] * case["rotary"] // 2
        pos = 4 * case["b"] * case["t"] * case["axes"]
        data = rows * case["d"] * e
        if not case["train"]:  # q, k, positions and frequencies in; q', k' out
            return {"bytes": 2 * data + pos + f, "flops": 3 * rows * case["rotary"]}
        learned = case["axes"] > 1
        # q, k, dq', dk' in; q', k', dq, dk (and the frequencies' gradient) out
        return {"bytes": 4 * data + pos + (2 if learned else 1) * f, "flops": (10 if learned else 6) * rows * case["rotary"]}
    if op == "attn":
        lq, lk = _lengths(case["lq"]), _lengths(case["lk"] or case["lq"])
        e, d = SIZE[case["dtype"]], case["d"]
        q = (sum(lq) + case["pad"]) * case["hq"] * d * e
        kv = (sum(lk) + case["pad"]) * case["hk"] * d * e
        pairs = sum(_visible(a, c, case["causal"]) for a, c in zip(lq, lk, strict=True)) * case["hq"]
        if not case["train"]:  # q, k, v in; o out
            return {"bytes": 2 * q + 2 * kv, "flops": 4 * pairs * d}
        # q, k, v, do in; o, dq, dk, dv out; two products forward, five backward
        return {"bytes": 4 * q + 4 * kv, "flops": 14 * pairs * d}
    e = SIZE[case["dtype"]]
    logits = case["r"] * case["v"]
    if op == "top":  # logits in; values, indices and log-sum-exp out
        return {"bytes": logits * e + case["r"] * (case["k"] * (e + 8) + 4), "flops": 3 * logits}
    # logits and the teacher's values and indices in; the gradient out
    return {"bytes": 2 * logits * e + case["r"] * case["k"] * 12, "flops": 6 * logits}


# ------------------------------------------------------------------------------------------ inputs

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _frequencies(rotary: int, scaling: str) -> tuple[torch.Tensor, float]:
    """Frequencies of base 10000 in 64 bits and the amplitude, for a context 8 times the 4096 trained on."""
    p = rotary // 2
    base, factor, length = 10000.0, 8.0, 4096
    exponent = torch.arange(p, dtype=torch.float64) / max(p, 1)
    if scaling == "ntk":  # the last frequency is divided by the factor, the first kept
        base = base * factor ** (p / (p - 1)) if p > 1 else base
    freq = base**-exponent
    if scaling == "linear":
        return freq / factor, 1.0
    if scaling == "yarn":
        # pairs that turn at least 32 times over the trained length are kept, those that turn less than
        # once are divided by the factor, linear in the pair's number in between
        low, high = (p * math.log(length / (turns * 2 * math.pi)) / math.log(base) for turns in (32.0, 1.0))
        low, high = max(math.floor(low), 0), min(math.ceil(high), p - 1)
        ramp = ((torch.arange(p, dtype=torch.float64) - low) / max(high - low, 1e-3)).clamp(0, 1)
        return freq * (1 - ramp) + freq / factor * ramp, 0.1 * math.log(factor) + 1.0
    return freq, 1.0


def prepare(case: dict, seed: int) -> dict:
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, device=dev, generator=gen)

    def uniform(*shape):
        return torch.rand(*shape, device=dev, generator=gen)

    if case["op"] == "rot":
        b, t, hq, hk, d, axes = (case[key] for key in ("b", "t", "hq", "hk", "d", "axes"))
        # q, k and v share the projection's output; q and k are views of it
        proj = normal(b, t, hq + 2 * hk, d).to(dtype)
        freq, amplitude = _frequencies(case["rotary"], case["scaling"])
        freq = freq.to(dev)
        token = torch.arange(t, device=dev)
        if axes == 1:
            # sequences that begin somewhere in a context of 131072 tokens
            start = torch.randint(0, 131072, (b, 1), device=dev, generator=gen)
            positions = start + token
        else:
            # patch coordinates of a 16-wide grid; every pair follows one axis
            coords = torch.stack([token // 16 ** (axes - 1 - a) % 16 for a in range(axes)], -1).float()
            positions = coords.expand(b, t, axes) + uniform(b, 1, axes)
            pair = torch.arange(freq.shape[0], device=dev)
            freq = torch.where(pair % axes == torch.arange(axes, device=dev)[:, None], freq, 0.0).float()
        out = {"case": case, "q": proj[:, :, :hq], "k": proj[:, :, hq:hq + hk], "positions": positions.contiguous(),
               "freq": freq, "amplitude": amplitude}
        if case["train"]:
            out["q"], out["k"] = (out[key].detach().requires_grad_(True) for key in ("q", "k"))
            if axes > 1:
                out["freq"].requires_grad_(True)
            out["dq"] = (0.01 * normal(b, t, hq, d)).to(dtype)
            out["dk"] = (0.01 * normal(b, t, hk, d)).to(dtype)
        return out
    if case["op"] == "attn":
        lq, lk = _lengths(case["lq"]), _lengths(case["lk"])
        hq, hk, d, pad = (case[key] for key in ("hq", "hk", "d", "pad"))
        tq = sum(lq) + pad
        if lk:
            q = normal(tq, hq, d).to(dtype)
            kv = normal(sum(lk) + pad, 2 * hk, d).to(dtype)
            k, v = kv[:, :hk], kv[:, hk:]
        else:  # views of one projection
            proj = normal(tq, hq + 2 * hk, d).to(dtype)
            q, k, v = proj[:, :hq], proj[:, hq:hq + hk], proj[:, hq + hk:]
        out = {"case": case, "q": q, "k": k, "v": v, "lq": lq, "lk": lk or lq}
        if case["train"]:
            out.update({key: out[key].detach().requires_grad_(True) for key in ("q", "k", "v")})
            out["do"] = (0.01 * normal(tq, hq, d)).to(dtype)
        if own:
            from mia_train_b200.ops.packed_attention import PackedSequences

            out["sequences"] = PackedSequences(lq, lk or None, causal=case["causal"], device=dev)
        return out
    r, v, k = case["r"], case["v"], case["k"]
    if case["op"] == "top":
        return {"case": case, "logits": (0.3 * normal(r, v) + 0.3 * normal(r, 1) * normal(v)).to(dtype)}
    # a student on its way to its teacher, at the size that cosine prototypes give
    teacher = 0.2 * normal(r, v)
    student = (0.5 * teacher + 0.15 * normal(r, v)).to(dtype)
    values, indices = torch.topk(teacher, k, dim=1)
    out = {"case": case, "s": student.requires_grad_(True), "values": values, "indices": indices,
           "lse": torch.logsumexp(teacher.double() / case["teacher_tau"], 1).float() if case["tail"] else None,
           "weights": uniform(r) * (uniform(r) > 0.1) if case["weights"] else None}
    return out


# ------------------------------------------------------------------------------------ plain forms


def _rot_plain(s: dict):
    case = s["case"]
    p, axes = case["rotary"] // 2, case["axes"]
    pos = s["positions"].double()
    freq = s["freq"].detach().double()
    # far positions need their angles in 64 bits
    angle = pos[..., None] * freq if axes == 1 else (pos[..., :, None] * freq).sum(-2)
    cos, sin = (s["amplitude"] * f(angle) for f in (torch.cos, torch.sin))
    cos, sin = cos.float()[:, :, None], sin.float()[:, :, None]
    channel = torch.arange(p, device=pos.device)
    first, second = (channel, channel + p) if case["layout"] == "half" else (2 * channel, 2 * channel + 1)

    def turn(x, sin):
        out = x.float().clone()
        a, b = x.float()[..., first], x.float()[..., second]
        out[..., first] = a * cos - b * sin
        out[..., second] = b * cos + a * sin
        return out

    dtype = s["q"].dtype
    q, k = s["q"].detach(), s["k"].detach()
    yq, yk = turn(q, sin), turn(k, sin)
    if not case["train"]:
        return yq.to(dtype), yk.to(dtype)
    dq, dk = turn(s["dq"], -sin), turn(s["dk"], -sin)
    out = [yq.to(dtype), yk.to(dtype), dq.to(dtype), dk.to(dtype)]
    if axes > 1:
        d_angle = sum((g.float()[..., second] * y[..., first] - g.float()[..., first] * y[..., second]).sum(2)
                      for g, y in ((s["dq"], yq), (s["dk"], yk)))
        out.append((pos[..., :, None] * d_angle[..., None, :].double()).sum((0, 1)).float())
    return tuple(out)


def _groups(lq: list[int], lk: list[int]):
    """Sequences of equal lengths together: (query length, key length, query starts, key starts)."""
    found: dict[tuple[int, int], tuple[list[int], list[int]]] = {}
    a = c = 0
    for m, n in zip(lq, lk, strict=True):
        starts = found.setdefault((m, n), ([], []))
        starts[0].append(a)
        starts[1].append(c)
        a, c = a + m, c + n
    return [(m, n, qs, ks) for (m, n), (qs, ks) in found.items()]


def _attn_plain(s: dict):
    case = s["case"]
    q, k, v = (s[key].detach() for key in ("q", "k", "v"))
    hq, hk, d = case["hq"], case["hk"], case["d"]
    g, scale = hq // hk, d**-0.5
    train = case["train"]
    out = torch.zeros_like(q, dtype=torch.float32)
    grads = [torch.zeros_like(x, dtype=torch.float32) for x in (q, k, v)] if train else []
    for m, n, q_starts, k_starts in _groups(s["lq"], s["lk"]):
        if m == 0 or n == 0:
            continue
        i, j = torch.arange(m, device=q.device), torch.arange(n, device=q.device)
        seen = (j <= i[:, None] + n - m) if case["causal"] else None
        most = max(1, (1 << 28) // (m * n * g))  # key heads of sequences at a time
        heads = min(hk, most)
        count = max(1, most // hk)
        for at in range(0, len(q_starts), count):
            rows = torch.tensor(q_starts[at:at + count], device=q.device)[:, None] + i
            cols = torch.tensor(k_starts[at:at + count], device=q.device)[:, None] + j
            for h in range(0, hk, heads):
                w = min(heads, hk - h)
                kh, qh = slice(h, h + w), slice(h * g, (h + w) * g)
                # (sequences, key heads, query heads of each, tokens, channels)
                qx = q[rows, qh].float().unflatten(2, (w, g)).permute(0, 2, 3, 1, 4)
                kx, vx = (x[cols, kh].float().permute(0, 2, 1, 3)[:, :, None] for x in (k, v))
                score = qx @ kx.transpose(-1, -2) * scale
                if seen is not None:
                    score = score.masked_fill(~seen, -math.inf)
                top = score.amax(-1, keepdim=True).clamp(min=-3e38)
                prob = (score - top).exp()
                total = prob.sum(-1, keepdim=True)
                prob = prob / total.clamp(min=1e-30)
                o = prob @ vx
                out[rows, qh] = o.permute(0, 3, 1, 2, 4).flatten(2, 3)
                if not train:
                    continue
                do = s["do"][rows, qh].float().unflatten(2, (w, g)).permute(0, 2, 3, 1, 4)
                d_prob = do @ vx.transpose(-1, -2)
                d_score = prob * (d_prob - (do * o).sum(-1, keepdim=True)) * scale
                grads[0][rows, qh] = (d_score @ kx).permute(0, 3, 1, 2, 4).flatten(2, 3)
                grads[1][cols, kh] = (d_score.transpose(-1, -2) @ qx).sum(2).permute(0, 2, 1, 3)
                grads[2][cols, kh] = (prob.transpose(-1, -2) @ do).sum(2).permute(0, 2, 1, 3)
    if not train:
        return out.to(q.dtype)
    return tuple(x.to(q.dtype) for x in (out, *grads))


def _top_plain(s: dict):
    case, x = s["case"], s["logits"]
    values, indices = torch.sort(x, dim=1, descending=True, stable=True)
    z = x.float() / case["tau"]
    top = z.amax(1, keepdim=True)
    lse = (z - top).exp().sum(1).log() + top[:, 0]
    return values[:, :case["k"]].contiguous(), indices[:, :case["k"]].contiguous(), lse


def _distill_plain(s: dict):
    case, x, at = s["case"], s["s"].detach(), s["indices"]
    z = x.float() / case["tau"]
    top = z.amax(1, keepdim=True)
    e = (z - top).exp()
    total = e.sum(1, keepdim=True)
    t = s["values"].double() / case["teacher_tau"]
    # the teacher's shares in 64 bits: what is left of 1 is a difference
    p = (t - s["lse"].double()[:, None]).exp() if case["tail"] else (t - torch.logsumexp(t, 1, keepdim=True)).exp()
    log_q = z.gather(1, at) - top - total.log()
    plogp = torch.where(p > 0, p * p.log(), 0.0)
    loss = (plogp - p * log_q).sum(1)
    q = e / total
    if case["tail"]:
        rest = (1 - p.sum(1, keepdim=True)).clamp(min=0)
        others = e.scatter(1, at, 0.0).sum(1, keepdim=True)
        loss = loss + (torch.where(rest > 0, rest * (rest.log() - (others / total).double().log()), 0.0))[:, 0]
        grad = q * (1 - (rest * total / others).float())
        grad.scatter_(1, at, q.gather(1, at) - p.float())
    else:
        grad = q.scatter_add(1, at, -p.float())
    w = s["weights"] if s["weights"] is not None else torch.ones_like(total[:, 0])
    loss = (loss * w).sum() / x.shape[0]
    return loss.float(), (grad * (w / (x.shape[0] * case["tau"]))[:, None]).to(x.dtype)


# -------------------------------------------------------------------------------------------- run


def run(state: dict):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return {"rot": _rot_plain, "attn": _attn_plain, "top": _top_plain, "distill": _distill_plain}[state["case"]["op"]](
            state)


def _run_own(s: dict):
    case = s["case"]
    if case["op"] == "rot":
        from mia_train_b200.ops.rotary import rotary

        args = (s["q"], s["k"], s["positions"], s["freq"])
        if not case["train"]:
            with torch.no_grad():
                return rotary(*args, layout=case["layout"], amplitude=s["amplitude"])
        yq, yk = rotary(*args, layout=case["layout"], amplitude=s["amplitude"])
        leaves = (s["q"], s["k"], s["freq"]) if case["axes"] > 1 else (s["q"], s["k"])
        return yq.detach(), yk.detach(), *torch.autograd.grad((yq, yk), leaves, (s["dq"], s["dk"]))
    if case["op"] == "attn":
        from mia_train_b200.ops.packed_attention import packed_attention

        if not case["train"]:
            with torch.no_grad():
                return packed_attention(s["q"], s["k"], s["v"], s["sequences"])
        o = packed_attention(s["q"], s["k"], s["v"], s["sequences"])
        return o.detach(), *torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["do"])
    if case["op"] == "top":
        from mia_train_b200.ops.distill import top_logits

        return top_logits(s["logits"], case["k"], tau=case["tau"])
    from mia_train_b200.ops.distill import top_logit_distillation

    loss = top_logit_distillation(s["s"], s["values"], s["indices"], tau=case["tau"], teacher_tau=case["teacher_tau"],
                                  teacher_lse=s["lse"], weights=s["weights"])
    return loss.detach(), *torch.autograd.grad(loss, s["s"])


# ------------------------------------------------------------------------------------------ exact


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    return {"rot": _rot_exact, "attn": _attn_exact, "top": _top_exact, "distill": _distill_exact}[case["op"]](s)


def _rot_exact(s: dict):
    """Rotation as the complex product (x1 + i x2) a e^{i angle}; gradients by autograd, in 64 bits."""
    case = s["case"]
    p = case["rotary"] // 2
    leaves = [s[key].detach().double().requires_grad_(True) for key in ("q", "k", "freq")]
    pos = s["positions"].double()
    if case["axes"] == 1:
        pos = pos[..., None]

    def one(x):
        head, rest = x[..., :2 * p], x[..., 2 * p:]
        pairs = head.unflatten(-1, (2, p)).transpose(-1, -2) if case["layout"] == "half" else head.unflatten(-1, (p, 2))
        angle = pos @ leaves[2].view(case["axes"], p)
        turn = torch.polar(torch.full_like(angle, s["amplitude"]), angle)[:, :, None]
        y = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        y = y.transpose(-1, -2).flatten(-2) if case["layout"] == "half" else y.flatten(-2)
        return torch.cat([y, rest], -1)

    with torch.enable_grad():
        yq, yk = one(leaves[0]), one(leaves[1])
        if not case["train"]:
            return yq.detach(), yk.detach()
        wanted = leaves if case["axes"] > 1 else leaves[:2]
        grads = torch.autograd.grad((yq, yk), wanted, (s["dq"].double(), s["dk"].double()))
    return yq.detach(), yk.detach(), *grads


def _attn_exact(s: dict):
    """Sequence by sequence and key head by key head, with autograd, in 64 bits."""
    case = s["case"]
    q, k, v = (s[key].detach() for key in ("q", "k", "v"))
    g = case["hq"] // case["hk"]
    if sum(m * n for m, n in zip(s["lq"], s["lk"], strict=True)) * case["hq"] * case["d"] > 4e11:
        return None
    outs = [torch.zeros_like(x, dtype=torch.float64) for x in (q, q, k, v)]
    a = c = 0
    for m, n in zip(s["lq"], s["lk"], strict=True):
        rows, cols = slice(a, a + m), slice(c, c + n)
        a, c = a + m, c + n
        if m == 0 or n == 0:
            continue
        blind = max(0, m - n) if case["causal"] else 0  # queries that see nothing
        rows = slice(rows.start + blind, rows.stop)
        step = case["hk"] if m * n * case["hq"] < 1 << 26 else 1
        for h in range(0, case["hk"], step):
            kh, qh = slice(h, h + step), slice(h * g, (h + step) * g)
            leaves = [x.double().requires_grad_(True) for x in (q[rows, qh], k[cols, kh], v[cols, kh])]
            with torch.enable_grad():
                kx, vx = (x.repeat_interleave(g, dim=1) for x in leaves[1:])
                score = torch.einsum("ihd,jhd->hij", leaves[0], kx) / math.sqrt(case["d"])
                if case["causal"]:
                    late = torch.ones(m - blind, n, dtype=torch.bool, device=q.device).triu(1 + n - (m - blind))
                    score = torch.where(late, -math.inf, score)
                o = torch.einsum("hij,jhd->ihd", torch.softmax(score, -1), vx)
                del score
                outs[0][rows, qh] = o.detach()
                if case["train"]:
                    got = torch.autograd.grad(o, leaves, s["do"][rows, qh].double())
                    for out, where, heads, x in zip(outs[1:], (rows, cols, cols), (qh, kh, kh), got, strict=True):
                        out[where, heads] = x
    return tuple(outs) if case["train"] else outs[0]


def _top_exact(s: dict):
    """By repeated selection order: the sort key is (value, -index), both whole in 64 bits."""
    case = s["case"]
    x = s["logits"].double()
    order = torch.argsort(-x, dim=1, stable=True)[:, :case["k"]]
    return x.gather(1, order), order, torch.logsumexp(x / case["tau"], 1)


def _distill_exact(s: dict):
    """The divergence of two log-distributions, classes outside the teacher's folded into one, with autograd."""
    case, at = s["case"], s["indices"]
    x = s["s"].detach().double().requires_grad_(True)
    t = s["values"].double() / case["teacher_tau"]
    with torch.enable_grad():
        log_q = torch.log_softmax(x / case["tau"], 1)
        picked = log_q.gather(1, at)
        log_p = t - s["lse"].double()[:, None] if case["tail"] else torch.log_softmax(t, 1)
        if case["tail"]:
            left = torch.ones_like(log_q, dtype=torch.bool).scatter(1, at, False)
            other = torch.logsumexp(torch.where(left, log_q, -math.inf), 1, keepdim=True)
            rest = -torch.expm1(torch.logsumexp(log_p, 1, keepdim=True))
            rest = rest.clamp(min=0)
            log_p = torch.cat([log_p, torch.where(rest > 0, rest, 1.0).log() + torch.where(rest > 0, 0.0, -math.inf)], 1)
            picked = torch.cat([picked, other], 1)
        p = log_p.exp()
        rows = torch.where(p > 0, p * (torch.where(p > 0, log_p, 0.0) - picked), 0.0).sum(1)
        w = s["weights"].double() if s["weights"] is not None else torch.ones_like(rows)
        loss = (rows * w).sum() / x.shape[0]
        grad, = torch.autograd.grad(loss, x)
    return loss.detach(), grad
