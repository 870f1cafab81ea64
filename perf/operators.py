"""Cases that measure the operators of an 8-bit, query/key-normalised, regularised transformer block.

Three families, in the order a block runs them:

* ``fp8``: a linear layer whose matrix products run on 8-bit floating point (e4m3) with one
  power-of-two scale per block of 128 along the summed axis (1 x 128 for activations and gradients,
  128 x 128 for weights): forward on weights that were quantised once, or forward with the gradients
  of input, weight and bias.
* ``qk``: RMS norm of every query and key head with its learned weight, followed by the position
  rotation: forward, or forward with the gradients of q, k, both weights and the angles.
* ``drop``: dropout from a counter-based generator (Philox4x32-10) added to an optional residual;
  the mask is a function of (seed, offset, element index) and never stored: forward and gradient.

``own`` is set from outside: False computes the plain forms with elementary torch operations, True
calls ``mia_train_b200.ops``.
"""

from __future__ import annotations

import math

import torch

own = False

FP8_BLOCK = 128


# ------------------------------------------------------------------------------------------ cases


def listed() -> list[dict]:
    return [
        # One pooled feature vector of a small encoder through a projection quantised once: the
        # smallest call, launch latency is all that counts.
        {"name": "fp8_pooled_row", "op": "fp8", "train": False, "m": 1, "k": 384, "n": 384},
        # A SwiGLU block's last projection in evaluation: hidden width rounded up to 8, ragged rows.
        {"name": "fp8_eval_ragged", "op": "fp8", "train": False, "m": 1029, "k": 1712, "n": 640},
        # The first MLP layer of a ViT-L masked autoencoder's encoder: 16 volumes x 128 visible tokens.
        {"name": "fp8_train_encoder", "op": "fp8", "train": True, "m": 2048, "k": 1024, "n": 4096},
        # The first MLP layer of the ViT-H-class encoder on four 4096-token volumes.
        {"name": "fp8_train_large", "op": "fp8", "train": True, "m": 16384, "k": 1280, "n": 5120},
        # Eight patch tokens and a class token of one small crop, evaluation.
        {"name": "qk_small_crop", "op": "qk", "train": False, "b": 1, "t": 9, "hq": 6, "hk": 6, "d": 64,
         "pairs": "half", "shared": True, "dtype": "bf16"},
        # The masked autoencoder's decoder: 16 volumes of 512 tokens, 16 heads of 32, axial angles.
        {"name": "qk_train_decoder", "op": "qk", "train": True, "b": 16, "t": 512, "hq": 16, "hk": 16, "d": 32,
         "pairs": "axial", "shared": False, "dtype": "bf16"},
        # Volumes of 4096 patch tokens with a class token and four registers, 16 heads of 64.
        {"name": "qk_train_volume", "op": "qk", "train": True, "b": 4, "t": 4101, "hq": 16, "hk": 16, "d": 64,
         "pairs": "half", "shared": True, "dtype": "bf16"},
        # Wide heads in 32 bits with fewer key than query heads, odd token count, evaluation.
        {"name": "qk_eval_wide_fp32", "op": "qk", "train": False, "b": 2, "t": 1025, "hq": 10, "hk": 5, "d": 128,
         "pairs": "axial", "shared": False, "dtype": "fp32"},
        # The branch output of one small crop (nine tokens, 384 channels) added to its residual.
        {"name": "drop_small_crop", "op": "drop", "rows": 9, "cols": 384, "p": 0.1, "residual": True, "dtype": "bf16"},
        # The MLP's hidden activations of the ViT-L encoder, no residual.
        {"name": "drop_hidden", "op": "drop", "rows": 2048, "cols": 4096, "p": 0.1, "residual": False, "dtype": "bf16"},
        # The hidden-width activations of four 4096-token ViT-H volumes with a residual.
        {"name": "drop_large", "op": "drop", "rows": 16384, "cols": 5120, "p": 0.2, "residual": True, "dtype": "bf16"},
        # 32-bit activations with odd extents.
        {"name": "drop_odd_fp32", "op": "drop", "rows": 1541, "cols": 1283, "p": 0.5, "residual": True, "dtype": "fp32"},
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    op = rng.choice(("fp8", "qk", "drop"))
    if op == "fp8":
        train = rng.random() < 0.5
        k, n = _log_int(rng, 64, 5120), _log_int(rng, 64, 5120)
        if rng.random() < 0.7:  # most layers have widths in multiples of 8
            k, n = -(-k // 8) * 8, -(-n // 8) * 8
        m = _log_int(rng, 1, 16384)
        m = max(1, min(m, 16384 * 1280 * 5120 // (k * n)))
        return {"op": "fp8", "train": train, "m": m, "k": k, "n": n}
    if op == "qk":
        d = rng.choice((32, 40, 64, 64, 80, 96, 128))
        hk = rng.randint(1, 16)
        hq = hk * rng.choice((1, 1, 1, 2, 3)) if hk <= 8 else hk
        b = _log_int(rng, 1, 16)
        most = 4 * 4101 * 2 * 16 * 64 // (b * (hq + hk) * d)
        t = _log_int(rng, 1, max(1, min(8192, most)))
        return {"op": "qk", "train": rng.random() < 0.6, "b": b, "t": t, "hq": hq, "hk": hk, "d": d,
                "pairs": rng.choice(("half", "axial")), "shared": rng.random() < 0.5,
                "dtype": rng.choice(("bf16", "bf16", "fp16", "fp32"))}
    cols = _log_int(rng, 1, 5120)
    rows = _log_int(rng, 1, min(65536, 16384 * 5120 // (2 * cols)))
    return {"op": "drop", "rows": rows, "cols": cols, "p": round(rng.uniform(0.01, 0.9), 3),
            "residual": rng.random() < 0.6, "dtype": rng.choice(("bf16", "bf16", "fp16", "fp32"))}


def work(case: dict) -> dict:
    size = {"bf16": 2, "fp16": 2, "fp32": 4}
    if case["op"] == "fp8":
        m, k, n = case["m"], case["k"], case["n"]
        if not case["train"]:  # x, 8-bit weight, bias in; y out
            return {"bytes": 2 * m * k + n * k + 4 * n + 2 * m * n, "flops": 2 * m * n * k}
        # x, fp32 weight, bias, dy in; y, dx, dw, db out
        return {"bytes": 2 * m * k + 4 * n * k + 4 * n + 2 * m * n + 2 * m * n + 2 * m * k + 4 * n * k + 4 * n,
                "flops": 6 * m * n * k}
    if case["op"] == "qk":
        rows = case["b"] * case["t"] * (case["hq"] + case["hk"])
        e = size[case["dtype"]]
        p = _pairs(case["pairs"], case["d"]).shape[0]
        ang = 4 * (1 if case["shared"] else case["b"]) * case["t"] * p
        data = rows * case["d"] * e
        if not case["train"]:
            return {"bytes": 2 * data + ang, "flops": 8 * rows * case["d"]}
        # q, k, dq', dk' and the angles in; q', k', dq, dk, dangles out
        return {"bytes": 5 * data + 2 * ang, "flops": 28 * rows * case["d"]}
    data = case["rows"] * case["cols"] * size[case["dtype"]]
    # x, dy (and the residual) in; y and dx out
    return {"bytes": data * (5 if case["residual"] else 4), "flops": 4 * case["rows"] * case["cols"]}


# ------------------------------------------------------------------------------------------ inputs

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _pairs(kind: str, d: int) -> torch.Tensor:
    """(P, 2) rotated channel pairs: the two halves of the head, or of one chunk per volume axis."""
    if kind == "half":
        first = torch.arange(d // 2)
        return torch.stack([first, first + d // 2], 1).to(torch.int32)
    each = 2 * (d // 6)
    widths = [each + 2 * ((d - 3 * each) // 2), each, each]
    starts = [0, widths[0], widths[0] + each]
    first = torch.cat([torch.arange(w // 2) + s for w, s in zip(widths, starts, strict=True)])
    half = torch.cat([torch.full((w // 2,), w // 2) for w in widths])
    return torch.stack([first, first + half], 1).to(torch.int32)


def prepare(case: dict, seed: int) -> dict:
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device=dev, generator=gen)

    def uniform(*shape):
        return torch.rand(*shape, device=dev, generator=gen)

    if case["op"] == "fp8":
        m, k, n = case["m"], case["k"], case["n"]
        # normalised activations with a few loud channels, as the input of a projection has them
        x = (normal(m, k) * torch.exp(0.8 * normal(k))).bfloat16()
        w = normal(n, k) / math.sqrt(k)
        bias = 0.1 * normal(n)
        if not case["train"]:
            q, s = _quantise(w, FP8_BLOCK)
            data = torch.zeros(n, -(-k // 16) * 16, device=dev, dtype=torch.float8_e4m3fn)
            data[:, :k] = q
            return {"case": case, "x": x, "data": data, "scale": s.t().contiguous(), "bias": bias}
        # token gradients of very different size, as a masked loss gives them
        dy = (1e-3 * normal(m, n) * torch.exp(2.0 * normal(m, 1))).bfloat16()
        return {"case": case, "x": x.requires_grad_(True), "w": w.requires_grad_(True),
                "bias": bias.requires_grad_(True), "dy": dy}
    if case["op"] == "qk":
        b, t, hq, hk, d = (case[key] for key in ("b", "t", "hq", "hk", "d"))
        dtype = DTYPES[case["dtype"]]
        pairs = _pairs(case["pairs"], d).to(dev)
        p = pairs.shape[0]
        # q, k and v share the projection's output; q and k are views of it
        proj = (normal(b, t, hq + 2 * hk, d) * torch.exp(0.5 * normal(d))).to(dtype)
        q, k = proj[:, :, :hq], proj[:, :, hq:hq + hk]
        # positions of a 16^3 patch grid times the axis frequencies; a prefix token stays unrotated
        side = 16
        token = torch.arange(t, device=dev)
        coords = torch.stack([token // (side * side), token // side % side, token % side], 1).float()
        freq = 100.0 ** (-torch.arange(p, device=dev).float() / p)
        angles = coords[:, torch.arange(p, device=dev) % 3] * freq
        angles[0] = 0.0
        angles = angles[None] if case["shared"] else angles[None] + 0.1 * normal(b, t, p)
        out = {"case": case, "q": q, "k": k, "pairs": pairs, "angles": angles.contiguous(),
               "qw": 1.0 + 0.2 * normal(d), "kw": 1.0 + 0.2 * normal(d)}
        if case["train"]:
            out.update({key: out[key].detach().requires_grad_(True) for key in ("q", "k", "qw", "kw", "angles")})
            out["dq"] = (0.01 * normal(b, t, hq, d)).to(dtype)
            out["dk"] = (0.01 * normal(b, t, hk, d)).to(dtype)
        return out
    dtype = DTYPES[case["dtype"]]
    shape = (case["rows"], case["cols"])
    out = {"case": case, "x": normal(*shape).to(dtype).requires_grad_(True), "dy": normal(*shape).to(dtype),
           "rng": torch.tensor([seed * 0x9E3779B97F4A7C15 % (1 << 62), 4 * (seed % 1000)], device=dev)}
    if case["residual"]:
        out["residual"] = (3.0 * uniform(*shape) - 1.5).to(dtype).requires_grad_(True)
    return out


# ------------------------------------------------------------------------------------ plain forms


def _quantise(x: torch.Tensor, rows: int) -> tuple[torch.Tensor, torch.Tensor]:
    """e4m3 values of x / s and the scales s (ceil(R / rows), ceil(C / 128)): s is the smallest power
    of two with max|x| / s <= 448 over each block of `rows` x 128."""
    x = x.float()
    r, c = x.shape
    rb, cb = -(-r // rows), -(-c // FP8_BLOCK)
    padded = torch.nn.functional.pad(x, (0, cb * FP8_BLOCK - c, 0, rb * rows - r))
    blocks = padded.view(rb, rows, cb, FP8_BLOCK)
    bits = blocks.abs().amax(dim=(1, 3)).view(torch.int32)
    up = (bits & 0x7FFFFF) > 0x600000  # the largest e4m3 value is 1.75 * 2^8
    scale = (((bits >> 23) - 8 + up).clamp(min=1) << 23).view(torch.float32)
    q = (blocks / scale[:, None, :, None]).to(torch.float8_e4m3fn)
    return q.view(rb * rows, cb * FP8_BLOCK)[:r, :c], scale


def _dequantise(q: torch.Tensor, scale: torch.Tensor, rows: int) -> torch.Tensor:
    r, c = q.shape
    full = scale.repeat_interleave(rows, 0)[:r].repeat_interleave(FP8_BLOCK, 1)[:, :c]
    return q.float() * full


def _rounded(x: torch.Tensor, rows: int) -> torch.Tensor:
    return _dequantise(*_quantise(x, rows), rows)


def _fp8_plain(s: dict):
    x, bias = s["x"].detach(), s["bias"].detach()
    if not s["case"]["train"]:
        w = _dequantise(s["data"][:, :x.shape[1]], s["scale"].t(), FP8_BLOCK)
        return (_rounded(x, 1) @ w.t() + bias).to(x.dtype)
    dy, w = s["dy"], _rounded(s["w"].detach(), FP8_BLOCK)
    y = _rounded(x, 1) @ w.t() + bias
    dx = _rounded(dy, 1) @ w
    dw = _rounded(dy.t(), 1) @ _rounded(x.t(), 1).t()
    return y.to(x.dtype), dx.to(x.dtype), dw, dy.float().sum(0)


def _norm_rotate(x, weight, cos, sin, first, second, eps):
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + eps)
    n = x * r * weight
    out = n.clone()
    out[..., first] = n[..., first] * cos - n[..., second] * sin
    out[..., second] = n[..., second] * cos + n[..., first] * sin
    return out, n, r


def _norm_rotate_grad(x, dout, weight, cos, sin, first, second, n, r):
    dn = dout.clone()
    dn[..., first] = dout[..., first] * cos + dout[..., second] * sin
    dn[..., second] = dout[..., second] * cos - dout[..., first] * sin
    dangle = (dn[..., second] * n[..., first] - dn[..., first] * n[..., second]).sum(2)
    xhat = x * r
    g = dn * weight
    dx = r * (g - xhat * (g * xhat).mean(-1, keepdim=True))
    return dx, (dn * xhat).sum((0, 1, 2)), dangle


def _qk_plain(s: dict, dtype=torch.float32):
    first, second = s["pairs"][:, 0].long(), s["pairs"][:, 1].long()
    angles = s["angles"].detach().to(dtype)
    cos, sin = angles.cos()[:, :, None], angles.sin()[:, :, None]
    q, k, qw, kw = (s[key].detach().to(dtype) for key in ("q", "k", "qw", "kw"))
    qo, qn, qr = _norm_rotate(q, qw, cos, sin, first, second, 1e-6)
    ko, kn, kr = _norm_rotate(k, kw, cos, sin, first, second, 1e-6)
    if not s["case"]["train"]:
        return qo, ko
    dq, dqw, dqa = _norm_rotate_grad(q, s["dq"].to(dtype), qw, cos, sin, first, second, qn, qr)
    dk, dkw, dka = _norm_rotate_grad(k, s["dk"].to(dtype), kw, cos, sin, first, second, kn, kr)
    dangles = dqa + dka
    if angles.shape[0] == 1:
        dangles = dangles.sum(0, keepdim=True)
    return qo, ko, dq, dk, dqw, dkw, dangles


def _mul_hi_lo(a: torch.Tensor, m: int) -> tuple[torch.Tensor, torch.Tensor]:
    """High and low 32 bits of a * m for 32-bit values held in int64."""
    lo = (a & 0xFFFF) * m
    hi = (a >> 16) * m + (lo >> 16)
    return hi >> 16, ((hi & 0xFFFF) << 16) | (lo & 0xFFFF)


def _philox_halves(count: int, rng: torch.Tensor) -> torch.Tensor:
    """`count` 16-bit random values: the halves, low first, of the words Philox4x32-10 (Salmon et
    al., SC 2011) gives for the counters (group of 8, offset with its top bit set) under key `seed`."""
    group = torch.arange(-(-count // 8), device=rng.device)
    seed, offset = rng[0], rng[1]
    word = 0xFFFFFFFF
    c0, c1 = group & word, group >> 32
    c2, c3 = (offset & word).expand_as(group), ((offset >> 32 & word) | 0x80000000).expand_as(group)
    k0, k1 = seed & word, seed >> 32 & word
    for _ in range(10):
        h0, l0 = _mul_hi_lo(c0, 0xD2511F53)
        h1, l1 = _mul_hi_lo(c2, 0xCD9E8D57)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & word, (k1 + 0xBB67AE85) & word
    words = torch.stack([c0, c1, c2, c3], 1)
    return torch.stack([words & 0xFFFF, words >> 16], 2).view(-1)[:count]


def _drop_plain(s: dict):
    x, dy = s["x"].detach(), s["dy"]
    dropped = round(s["case"]["p"] * 65536)
    keep = (_philox_halves(x.numel(), s["rng"]) >= dropped).view(x.shape)
    scale = 65536.0 / (65536 - dropped)
    y = torch.where(keep, x.float() * scale, 0.0)
    dx = torch.where(keep, dy.float() * scale, 0.0).to(x.dtype)
    if not s["case"]["residual"]:
        return y.to(x.dtype), dx
    return (s["residual"].detach().float() + y).to(x.dtype), dx, dy


# -------------------------------------------------------------------------------------------- run


def run(state: dict):
    case = state["case"]
    if own:
        return _run_own(state)
    with torch.no_grad():
        if case["op"] == "fp8":
            return _fp8_plain(state)
        if case["op"] == "qk":
            outs = _qk_plain(state)
            tensors = DTYPES[case["dtype"]]
            return tuple(o.to(tensors) for o in outs[:4]) + tuple(outs[4:])
        return _drop_plain(state)


def _run_own(s: dict):
    from mia_train_b200.ops.dropout import dropout
    from mia_train_b200.ops.fp8 import Fp8Matrix, fp8_linear
    from mia_train_b200.ops.qk_norm import qk_norm_rope

    case = s["case"]
    if case["op"] == "fp8":
        if not case["train"]:
            with torch.no_grad():
                weight = Fp8Matrix(s["data"], s["scale"], cols=case["k"], block_rows=FP8_BLOCK)
                return fp8_linear(s["x"], weight, s["bias"])
        y = fp8_linear(s["x"], s["w"], s["bias"])
        return y.detach(), *torch.autograd.grad(y, (s["x"], s["w"], s["bias"]), s["dy"])
    if case["op"] == "qk":
        if not case["train"]:
            with torch.no_grad():
                return qk_norm_rope(s["q"], s["k"], s["qw"], s["kw"], s["angles"], s["pairs"], eps=1e-6)
        qo, ko = qk_norm_rope(s["q"], s["k"], s["qw"], s["kw"], s["angles"], s["pairs"], eps=1e-6)
        leaves = (s["q"], s["k"], s["qw"], s["kw"], s["angles"])
        return qo.detach(), ko.detach(), *torch.autograd.grad((qo, ko), leaves, (s["dq"], s["dk"]))
    residual = s.get("residual")
    y = dropout(s["x"], case["p"], residual=residual, rng=s["rng"])
    leaves = (s["x"],) if residual is None else (s["x"], residual)
    return y.detach(), *torch.autograd.grad(y, leaves, s["dy"])


# ------------------------------------------------------------------------------------------ exact


def _e4m3_exact(v: torch.Tensor) -> torch.Tensor:
    """Nearest e4m3 value, ties to even, of 64-bit values of magnitude at most 448."""
    exponent = torch.frexp(v)[1].double() - 1
    step = torch.exp2(exponent.clamp(min=-6) - 3)
    return torch.round(v / step) * step


def _blocks_exact(x: torch.Tensor, rows: int) -> torch.Tensor:
    """x with every block of `rows` x 128 rounded to its scaled e4m3 grid, in 64 bits."""
    x = x.double()
    out = torch.empty_like(x)
    for c in range(0, x.shape[1], FP8_BLOCK):
        part = x[:, c:c + FP8_BLOCK]
        if rows == 1:
            top = part.abs().amax(1, keepdim=True)
        else:
            chunks = part.abs().amax(1).split(rows)
            top = torch.cat([chunk.amax().expand(chunk.shape[0]) for chunk in chunks])[:, None]
        m, e = torch.frexp(top / 448.0)  # top / 448 = m 2^e with m in [0.5, 1)
        power = torch.where(m == 0.5, e - 1, e).clamp(min=-126)
        scale = torch.exp2(power.double())
        out[:, c:c + FP8_BLOCK] = _e4m3_exact(part / scale) * scale
    return out


def _philox_exact(count: int, seed: int, offset: int) -> torch.Tensor:
    """The same counters evaluated with numpy's unsigned 64-bit integers."""
    import numpy as np

    word = np.uint64(0xFFFFFFFF)
    shift = np.uint64(32)
    group = np.arange(-(-count // 8), dtype=np.uint64)
    c = [group & word, group >> shift, np.full_like(group, offset & 0xFFFFFFFF),
         np.full_like(group, (offset >> 32 & 0xFFFFFFFF) | 0x80000000)]
    key = [seed & 0xFFFFFFFF, seed >> 32 & 0xFFFFFFFF]
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> shift) ^ c[1] ^ np.uint64(key[0]), b & word, (a >> shift) ^ c[3] ^ np.uint64(key[1]), a & word]
        key = [(key[0] + 0x9E3779B9) & 0xFFFFFFFF, (key[1] + 0xBB67AE85) & 0xFFFFFFFF]
    halves = np.stack([np.stack([v & np.uint64(0xFFFF), v >> np.uint64(16)], 1) for v in c], 1).reshape(-1)
    return torch.from_numpy(halves[:count].astype(np.int64))


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "fp8":
            x, bias = s["x"].detach(), s["bias"].detach().double()
            xq = _blocks_exact(x, 1)
            if not case["train"]:
                scale = s["scale"].double()
                w = s["data"].float().double()[:, :case["k"]]
                cols = torch.arange(case["k"], device=w.device) // FP8_BLOCK
                rows = torch.arange(case["n"], device=w.device) // FP8_BLOCK
                return xq @ (w * scale[cols][:, rows].t()).t() + bias
            w = _blocks_exact(s["w"].detach(), FP8_BLOCK)
            dy = s["dy"]
            dw = _blocks_exact(dy.t(), 1) @ _blocks_exact(x.t(), 1).t()
            return xq @ w.t() + bias, _blocks_exact(dy, 1) @ w, dw, dy.double().sum(0)
        if case["op"] == "qk":
            return _qk_exact(s)
        if case["rows"] * case["cols"] > 1 << 25:  # the numpy generator would take too long
            return None
        x, dy = s["x"].detach().double(), s["dy"].double()
        seed_word, offset = (int(v) for v in s["rng"].tolist())
        dropped = round(case["p"] * 65536)
        keep = (_philox_exact(x.numel(), seed_word, offset) >= dropped).view(x.shape).to(x.device).double()
        keep = keep * (65536.0 / (65536 - dropped))
        if case["residual"]:
            return s["residual"].detach().double() + x * keep, dy * keep, dy
        return x * keep, dy * keep


def _qk_exact(s: dict):
    """Norm and rotation as the complex product (n1 + i n2) e^{i angle}; gradients by autograd, in 64 bits."""
    first, second = s["pairs"][:, 0].long(), s["pairs"][:, 1].long()
    leaves = [s[key].detach().double().requires_grad_(True) for key in ("q", "k", "qw", "kw", "angles")]
    q, k, qw, kw, angles = leaves

    def one(x, weight):
        n = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * weight
        z = torch.complex(n[..., first], n[..., second]) * torch.polar(torch.ones_like(angles), angles)[:, :, None]
        rest = torch.ones(x.shape[-1], dtype=torch.bool, device=x.device)
        rest[first] = rest[second] = False
        out = torch.zeros_like(n).index_copy(-1, first, z.real).index_copy(-1, second, z.imag)
        return out + n * rest

    with torch.enable_grad():
        qo, ko = one(q, qw), one(k, kw)
        if not s["case"]["train"]:
            return qo.detach(), ko.detach()
        grads = torch.autograd.grad((qo, ko), leaves, (s["dq"].double(), s["dk"].double()))
    return qo.detach(), ko.detach(), *grads
