"""The operators together, as a transformer block runs them: 8-bit projections, normalised and rotated heads,
attention, dropout with the residual; eager, checkpointed and in a captured training step."""

from __future__ import annotations

import copy

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover - collected on CPU, skipped there
    pytest.skip("needs CUDA", allow_module_level=True)

from mia_train_b200.engine.fp8 import apply_fp8_linears  # noqa: E402
from mia_train_b200.layers.common.blocks import TransformerBlock  # noqa: E402
from mia_train_b200.layers.dinov3.block import SelfAttentionBlock  # noqa: E402
from mia_train_b200.ops import _native  # noqa: E402
from mia_train_b200.ops.dropout import STEPS, random_halves_reference  # noqa: E402
from mia_train_b200.ops.fp8 import BLOCK, quantize_reference  # noqa: E402

DEV = torch.device("cuda", 0)
E4M3 = torch.float8_e4m3fn


def _no_errors():
    torch.cuda.synchronize()
    assert _native.native().check_errors(0) == 0


def _q(t, rows):
    return quantize_reference(t, rows, E4M3).dequantize()


def test_block_forward_is_the_composition(monkeypatch):
    """Step by step in fp32 with the block's own intermediate roundings (bf16 activations, 8-bit operands)."""
    torch.manual_seed(0)
    b, n, dim, heads, p = 3, 70, 128, 2, 0.25
    d = dim // heads
    holder = torch.nn.Module()
    holder.blk = blk = TransformerBlock(dim, heads, qk_norm=True, dropout=p).to(DEV)
    for w in blk.parameters():
        if w.dim() == 1 and w.shape[0] == d:
            torch.nn.init.uniform_(w, 0.5, 1.5)
    apply_fp8_linears(holder)
    x = torch.randn(b, n, dim, device=DEV).bfloat16()
    coords = torch.randint(0, 8, (b, n, 3), device=DEV).float()
    pairs = [torch.tensor([7, 4 * i], device=DEV) for i in range(3)]
    it = iter(pairs)
    import mia_train_b200.layers.common.blocks as blocks

    real = blocks.drop
    monkeypatch.setattr(blocks, "drop", lambda t, q, residual=None: real(t, q, residual=residual, rng=next(it)))
    with torch.autocast("cuda", dtype=torch.bfloat16):
        got = blk(x, coords)

    bf = lambda t: t.bfloat16().float()  # noqa: E731
    it = iter(pairs)

    def dropped(t, residual):
        keep = (random_halves_reference(t.numel(), next(it)) >= round(p * STEPS)).view(t.shape)
        y = torch.where(keep, t * (STEPS / (STEPS - round(p * STEPS))), 0.0)
        return bf(y if residual is None else residual + y)

    def lin(m, t, act=False):
        y = (_q(t.reshape(-1, t.shape[-1]), 1) @ _q(m.weight.float(), BLOCK).t() + m.bias.float()).view(*t.shape[:-1], -1)
        return bf(F.gelu(y) if act else y)

    def norm(t, w):
        return t * torch.rsqrt(t.square().mean(-1, keepdim=True) + 1e-6) * w

    xf = x.float()
    h = bf(F.layer_norm(xf, (dim,), blk.norm1.weight, blk.norm1.bias))
    q, k, v = lin(blk.attn.qkv, h).view(b, n, 3, heads, d).unbind(2)
    tables = blk.rotary(coords)
    q, k = bf(tables(norm(q, blk.attn.q_norm.weight))), bf(tables(norm(k, blk.attn.k_norm.weight)))
    o = bf(F.scaled_dot_product_attention(q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2), scale=d**-0.5).transpose(1, 2))
    y = dropped(lin(blk.attn.proj, o.reshape(b, n, dim)), xf)
    h = bf(F.layer_norm(y, (dim,), blk.norm2.weight, blk.norm2.bias))
    want = dropped(lin(blk.mlp[2], dropped(lin(blk.mlp[0], h, True), None)), y)
    # Each of some twelve bf16 roundings can fall the other way and move an 8-bit operand by a step of 2^-3 now
    # and then; such moves are unrelated, so the whole differs by a few roundings of bf16 in norm.
    assert ((got.float() - want).norm() / want.norm()).item() < 12 * 2.0**-8
    _no_errors()


@pytest.mark.parametrize("kind", ["vit", "dinov3"])
def test_block_gradients_follow_the_torch_path(kind):
    """Native block against the same block on PyTorch math: 8-bit operands differ only where a bf16 rounding before
    them fell the other way."""
    torch.manual_seed(1)
    holder = torch.nn.Module()
    if kind == "vit":
        holder.blk = TransformerBlock(128, 2, qk_norm=True)
    else:
        holder.blk = SelfAttentionBlock(128, 2, qk_norm=True, init_values=0.5, qkv_bias=True)
    holder.to(DEV)
    apply_fp8_linears(holder)
    other = copy.deepcopy(holder)
    x = torch.randn(2, 130, 128, device=DEV)
    coords = torch.randint(0, 8, (2, 130, 3), device=DEV).float()
    dy = torch.randn(2, 130, 128, device=DEV)

    def run(m):
        leaf = x.clone().requires_grad_(True)
        with torch.autocast("cuda", dtype=torch.bfloat16):
            y = m.blk(leaf.bfloat16(), coords) if kind == "vit" else m.blk(leaf.bfloat16())
        grads = torch.autograd.grad(y.float(), [leaf, *m.parameters()], dy, allow_unused=True)
        return [y, *grads], ["y", "x", *[n for n, _ in m.named_parameters()]]

    got, names = run(holder)
    with _native.reference_math():
        want, _ = run(other)
    for name, a, e in zip(names, got, want, strict=True):
        assert (a is None) == (e is None), name
        if a is None or e.float().norm() < 1e-6:
            continue
        cos = F.cosine_similarity(a.float().flatten(), e.float().flatten(), dim=0).item()
        assert cos > 0.99, (name, cos)
    _no_errors()


def test_checkpointed_block_replays_masks():
    from torch.utils.checkpoint import checkpoint

    torch.manual_seed(2)
    holder = torch.nn.Module()
    holder.blk = blk = TransformerBlock(128, 2, qk_norm=True, dropout=0.3).to(DEV)
    apply_fp8_linears(holder)
    x = torch.randn(2, 64, 128, device=DEV).bfloat16().requires_grad_(True)

    def grad(f):
        torch.manual_seed(3)
        with torch.autocast("cuda", dtype=torch.bfloat16):
            return torch.autograd.grad(f(x).float().square().sum(), x)[0]

    a, b = grad(blk), grad(lambda t: checkpoint(blk, t, use_reentrant=False))
    # attention's dq is summed by atomics, whose order changes its last bits from run to run
    assert ((a.float() - b.float()).norm() / a.float().norm()).item() < 2.0**-6
    _no_errors()


def test_captured_training_step_uses_all_three(tmp_path):
    from mia_train_b200.algorithms.mae import MAE
    from mia_train_b200.engine.config import TrainerConfig
    from mia_train_b200.engine.graph_step import CapturedStep
    from mia_train_b200.engine.optimizer import build_optimizer
    from mia_train_b200.models.vit import ViT3D

    torch.manual_seed(4)
    model = ViT3D((32, 32, 32), (8, 8, 8), 1, 128, 2, 2, qk_norm=True, dropout=0.1)
    alg = MAE(model, input_axes="lcxyz", decoder_embed_dim=64, decoder_depth=1, decoder_num_heads=2).to(DEV)
    assert apply_fp8_linears(alg) == 12
    config = TrainerConfig(max_steps=50, batch_size=2, lr=1e-3, precision="bf16", linear_precision="fp8",
                           fused_optimizer="on", step_mode="graph")
    opt = build_optimizer(alg, config)
    batch = {"img": torch.randn(2, 1, 1, 32, 32, 32, device=DEV)}
    step = CapturedStep(alg, opt, config, batch)
    before = {n: p.detach().clone() for n, p in alg.named_parameters()}
    losses = [float(step(batch)["loss"]) for _ in range(8)]
    assert step.graph is not None and all(torch.isfinite(torch.tensor(losses)))
    assert len(set(losses)) == 8  # masks (of tokens and of dropout) are drawn anew on every replay
    for n, p in alg.named_parameters():
        if "inv_freqs" not in n:
            assert not torch.equal(p, before[n]), n
    _no_errors()


def test_second_derivatives_are_refused():
    from mia_train_b200.ops.dropout import dropout
    from mia_train_b200.ops.fp8 import fp8_linear
    from mia_train_b200.ops.qk_norm import qk_norm_rope

    x = torch.randn(4, 64, device=DEV, requires_grad=True)
    heads = torch.randn(1, 4, 2, 64, device=DEV, requires_grad=True)
    w = torch.randn(32, 64, device=DEV)
    for leaf, f in ((x, lambda t: dropout(t, 0.5)), (x, lambda t: fp8_linear(t, w)),
                    (heads, lambda t: qk_norm_rope(t, t, None, None)[0])):
        y = f(leaf)
        dy = torch.ones_like(y).requires_grad_(True)
        with pytest.raises(RuntimeError, match="differentiable once"):
            torch.autograd.grad(y, leaf, dy, create_graph=True)


def test_no_grad_keeps_nothing():
    from mia_train_b200.ops.fp8 import fp8_linear

    x, w = torch.randn(512, 1024, device=DEV).bfloat16(), torch.randn(1024, 1024, device=DEV, requires_grad=True)
    with torch.no_grad():
        y = fp8_linear(x, w)
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        z = fp8_linear(x, w)
        assert torch.cuda.memory_allocated() - before == z.numel() * 2 and torch.equal(y, z)
    assert not z.requires_grad
