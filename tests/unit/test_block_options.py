"""`qk_norm`, `dropout` and `linear_precision = "fp8"` in blocks, models and the Trainer (CPU)."""

from __future__ import annotations

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

from mia_train_b200.engine.config import LoRAConfig, TrainerConfig
from mia_train_b200.engine.fp8 import apply_fp8_linears, fp8_targets
from mia_train_b200.engine.lora import apply_lora
from mia_train_b200.layers.common.blocks import TransformerBlock
from mia_train_b200.layers.common.lora import is_fp8, promote, use_fp8
from mia_train_b200.layers.dinov3.block import SelfAttentionBlock
from mia_train_b200.models.dinov3_vit3d import DinoVisionTransformer3D
from mia_train_b200.models.muvit import MuViT3D
from mia_train_b200.models.vit import ViT3D
from mia_train_b200.ops import dropout as dropout_module


def _norm(x, w, eps):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * w


def test_block_qk_norm_is_the_formula():
    torch.manual_seed(0)
    blk = TransformerBlock(24, 2, qk_norm=True, rotary=False)
    for p in blk.parameters():
        nn.init.normal_(p, std=0.5)
    x = torch.randn(2, 5, 24)
    a = blk.attn
    h = F.layer_norm(x, (24,), blk.norm1.weight, blk.norm1.bias)
    q, k, v = F.linear(h, a.qkv.weight, a.qkv.bias).reshape(2, 5, 3, 2, 12).unbind(2)
    q, k = _norm(q, a.q_norm.weight, 1e-6), _norm(k, a.k_norm.weight, 1e-6)
    o = torch.einsum("bhqk,bkhd->bqhd", torch.softmax(torch.einsum("bqhd,bkhd->bhqk", q, k) * 12**-0.5, -1), v)
    y = x + F.linear(o.reshape(2, 5, 24), a.proj.weight, a.proj.bias)
    want = y + blk.mlp(F.layer_norm(y, (24,), blk.norm2.weight, blk.norm2.bias))
    torch.testing.assert_close(blk(x), want, rtol=1e-4, atol=1e-4)


@pytest.mark.parametrize("make", [
    lambda **kw: ViT3D((16, 16, 16), (8, 8, 8), 1, 24, 2, 2, **kw),
    lambda **kw: MuViT3D((1, 2), (16, 16, 16), (8, 8, 8), 1, 24, 2, 2, **kw),
])
def test_models_train_with_norms_and_dropout(make):
    torch.manual_seed(0)
    model = make(qk_norm=True, dropout=0.2)
    names = {n for n, _ in model.named_parameters()}
    assert {"blocks.0.attn.q_norm.weight", "blocks.1.attn.k_norm.weight"} <= names
    tokens = torch.randn(2, 8, 24)
    coords = torch.randn(2, 8, 3)
    run = lambda: [b(tokens, coords) for b in model.blocks][-1]  # noqa: E731
    model.train()
    assert not torch.equal(run(), run())  # masks differ between calls
    model.eval()
    assert torch.equal(run(), run())
    model.train()
    run().square().mean().backward()
    g = model.blocks[1].attn.q_norm.weight.grad
    assert g is not None and g.abs().sum() > 0
    plain = {n for n, _ in make().named_parameters()}
    assert not any("q_norm" in n for n in plain)


@pytest.mark.parametrize("ffn", ["mlp", "swiglu"])
@pytest.mark.parametrize("window", [0, 2])
def test_dinov3_options(ffn, window):
    torch.manual_seed(0)
    kw = dict(img_size=32, patch_size=8, in_chans=1, embed_dim=24, depth=2, num_heads=2, n_storage_tokens=2, ffn_layer=ffn,
              layerscale_init=0.5, window_size=window)
    model = DinoVisionTransformer3D(qk_norm=True, drop_rate=0.1, **kw)
    x = torch.randn(2, 1, 32, 32, 32)
    model.eval()
    out = model.forward_features(x)["x_norm_patchtokens"]
    assert torch.equal(out, model.forward_features(x)["x_norm_patchtokens"])
    model.train()
    out = model.forward_features(x)["x_norm_patchtokens"]
    out.square().mean().backward()
    assert all(b.attn.k_norm.weight.grad.abs().sum() > 0 for b in model.blocks)
    with pytest.raises(ValueError, match="drop_rate"):
        DinoVisionTransformer3D(drop_rate=1.0, **kw)


def test_windowed_norm_equals_global_norm_in_one_window():
    torch.manual_seed(0)
    kw = dict(img_size=16, patch_size=8, in_chans=1, embed_dim=24, depth=2, num_heads=2, qk_norm=True)
    a, b = DinoVisionTransformer3D(window_size=2, **kw), DinoVisionTransformer3D(**kw)
    for p in a.parameters():
        nn.init.normal_(p, std=0.3)
    b.load_state_dict(a.state_dict())
    x = torch.randn(2, 1, 16, 16, 16)
    torch.testing.assert_close(a.eval()(x), b.eval()(x), rtol=1e-4, atol=1e-4)


def test_dinov3_dropout_places_and_scales(monkeypatch):
    """Branch output times LayerScale is dropped and added; the hidden activations are dropped as well."""
    torch.manual_seed(0)
    blk = SelfAttentionBlock(8, 2, drop=0.5, init_values=0.3)
    calls = []
    real = dropout_module.dropout

    def spy(x, p, *, residual=None, training=True, rng=None):
        calls.append((tuple(x.shape), p, residual is not None))
        return real(x, p, residual=residual, training=training, rng=rng)

    monkeypatch.setattr("mia_train_b200.layers.dinov3.attention.dropout", spy)
    monkeypatch.setattr("mia_train_b200.layers.dinov3.ffn.dropout", spy)
    blk.train()
    blk(torch.randn(2, 3, 8))
    # the list path flattens tokens: (6, 8) rows
    assert [(c[0][-1], c[1], c[2]) for c in calls] == [(8, 0.5, True), (32, 0.5, False), (8, 0.5, True)]
    blk.eval()
    calls.clear()
    blk(torch.randn(2, 3, 8))
    assert calls == []


def test_block_dropout_refusal():
    for p in (-0.1, 1.0):
        with pytest.raises(ValueError, match="dropout"):
            TransformerBlock(24, 2, dropout=p)


def _algorithm(**kw):
    from mia_train_b200.algorithms.mae import MAE

    model = ViT3D((16, 16, 16), (8, 8, 8), 1, 24, 2, 2, **kw)
    return MAE(model, input_axes="lcxyz", decoder_embed_dim=24, decoder_depth=1, decoder_num_heads=2)


def test_fp8_marks_every_block_projection():
    alg = _algorithm()
    targets = fp8_targets(alg)
    assert len(targets) == 3 * 4 and "model.blocks.0.attn.qkv" in targets and "decoder_blocks.0.mlp.2" in targets
    assert apply_fp8_linears(alg) == 12 and all(is_fp8(m) for m in targets.values())
    assert not is_fp8(alg.decoder_head) and not is_fp8(alg.decoder_embed)


def test_fp8_block_close_to_full_precision_and_trains():
    torch.manual_seed(0)
    alg = _algorithm(qk_norm=True)
    x = {"img": torch.randn(2, 1, 1, 16, 16, 16)}
    torch.manual_seed(1)
    ref = alg(x)["loss"]
    ref.backward()
    want = {n: p.grad.clone() for n, p in alg.named_parameters() if p.grad is not None}
    alg.zero_grad()
    apply_fp8_linears(alg)
    torch.manual_seed(1)
    got = alg(x)["loss"]
    got.backward()
    assert not torch.equal(got, ref)  # the 8-bit path ran
    # every product is off by at most (1 + 2^-4)^2 - 1 = 13 % of its size and the roundings are unrelated: the
    # gradients point the same way
    for n, p in alg.named_parameters():
        if p.grad is not None and want[n].norm() > 1e-6:
            assert F.cosine_similarity(p.grad.flatten(), want[n].flatten(), dim=0) > 0.9, n


def test_fp8_refusals():
    with pytest.raises(ValueError, match="transformer block"):
        apply_fp8_linears(nn.Linear(4, 4))
    with pytest.raises(ValueError, match="tensor parallelism"):
        apply_fp8_linears(_algorithm(), tp=2)
    alg = _algorithm()
    apply_lora(alg.encoder, LoRAConfig(rank=2, alpha=4.0, targets=("attn_qkv",)))
    with pytest.raises(ValueError, match="lora"):
        apply_fp8_linears(alg)
    lin = promote(nn.Linear(8, 8), rank=2, alpha=2.0)
    with pytest.raises(ValueError):
        use_fp8(lin)
    base = dict(max_steps=2, batch_size=1)
    assert TrainerConfig(**base).linear_precision == "bf16"
    TrainerConfig(**base, precision="bf16", linear_precision="fp8")
    for bad in (dict(linear_precision="fp8"), dict(linear_precision="int8", precision="bf16")):
        with pytest.raises(ValueError, match="linear_precision"):
            TrainerConfig(**base, **bad)


def test_trainer_option_trains(tmp_path):
    from pathlib import Path

    from mia_train_b200.engine.run import run
    from mia_train_b200.utils.config import load_run_config

    path = Path(__file__).resolve().parents[2] / "configs" / "mae_fp8_smoke_synthetic.toml"
    assert load_run_config(path).trainer.linear_precision == "fp8"
    text = path.read_text()
    for old, new in (("max_steps = 30", "max_steps = 2"), ("warmup_steps = 5", "warmup_steps = 1"), ("depth = 6", "depth = 1"),
                     ("embed_dim = 384", "embed_dim = 48"), ("num_heads = 6\nqk", "num_heads = 2\nqk"),
                     ("decoder_embed_dim = 192", "decoder_embed_dim = 48"), ("checkpoint_every = 15", "checkpoint_every = 2"),
                     ("batch_size = 4", "batch_size = 2")):
        assert old in text
        text = text.replace(old, new)
    cfg = tmp_path / "c.toml"
    cfg.write_text(text)
    out = run(cfg, output_root=tmp_path)
    assert (out / "checkpoints").is_dir()
