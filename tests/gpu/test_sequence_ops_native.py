"""Rotation, packed attention and distillation together, as a step on crops of several sizes runs them, on the GPU."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover - collected on CPU, skipped there
    pytest.skip("needs CUDA", allow_module_level=True)

from mia_train_b200.layers.dinov3.attention import SelfAttention  # noqa: E402
from mia_train_b200.models.dinov3_vit3d import DinoVisionTransformer3D  # noqa: E402
from mia_train_b200.ops._native import reference_math  # noqa: E402
from mia_train_b200.ops.distill import top_logit_distillation, top_logits  # noqa: E402
from mia_train_b200.ops.packed_attention import PackedSequences, packed_attention  # noqa: E402
from mia_train_b200.ops.rotary import rotary, rotary_frequencies  # noqa: E402

DEV = torch.device("cuda", 0)


@pytest.mark.parametrize("kw", [{}, {"qk_norm": True}], ids=str)
def test_model_with_packed_crops(kw):
    """bf16 crops of two sizes through two blocks, packed and crop by crop, both against the fp32 model: the two ways round
    the same quantities (P, the attention's output, dS) to bf16, each time by 2^-9 at most."""
    kw = dict(img_size=32, patch_size=8, in_chans=1, embed_dim=128, depth=2, num_heads=2, n_storage_tokens=4, **kw)
    torch.manual_seed(0)
    plain = DinoVisionTransformer3D(**kw).to(DEV)
    packed = DinoVisionTransformer3D(packed_crops=True, **kw).to(DEV)
    packed.load_state_dict(plain.state_dict())
    crops = [torch.randn(2, 1, 32, 32, 32, device=DEV), torch.randn(6, 1, 16, 16, 16, device=DEV)]
    outs = []
    for model, half in ((plain, False), (plain, True), (packed, True)):
        with torch.autocast("cuda", dtype=torch.bfloat16, enabled=half):
            out = model.forward_features(crops, [None, None])
            # not a function of the norm's mean square, which is 1 whatever the weights
            loss = sum(o["x_norm_patchtokens"].float().sin().mean() for o in out)
        # one weight of every kind behind and before the attention
        some = [model.blocks[0].attn.qkv.weight, model.blocks[0].attn.proj.weight, model.blocks[1].attn.qkv.weight]
        outs.append([o["x_norm_patchtokens"].detach().float() for o in out] + list(torch.autograd.grad(loss, some)))
    for i, (exact, a, b) in enumerate(zip(*outs, strict=True)):
        off = [(x - exact).norm() for x in (a, b)]
        assert off[1] <= 2 * off[0] + 2.0**-9 * exact.norm(), (i, off, exact.norm())


def test_distilling_a_small_encoder_from_stored_logits():
    """One step: tokens of three sequences rotated, attended to and projected to classes, against a teacher's top
    logits. The native step against the same operators as PyTorch math in fp32 on the same values."""
    torch.manual_seed(0)
    lengths, hq, hk, d, v = [33, 70, 1], 4, 2, 32, 5000
    t = sum(lengths)
    x = torch.randn(t, 64, device=DEV)
    wq = (torch.randn(64, (hq + 2 * hk) * d, device=DEV) / 8).requires_grad_(True)
    wo = (torch.randn(hq * d, v, device=DEV) / hq / d**0.5).requires_grad_(True)
    freq, amplitude = rotary_frequencies(d // 2, scaling="yarn", factor=4.0, original_length=64, device=DEV)
    positions = torch.cat([torch.arange(n, device=DEV) for n in lengths])
    values, indices, lse = top_logits(torch.randn(t, v, device=DEV), 32)

    def step():
        h = (x @ wq).view(t, hq + 2 * hk, d)
        q, k = rotary(h[:, :hq], h[:, hq:hq + hk], positions, freq, layout="interleaved", amplitude=amplitude)
        o = packed_attention(q, k, h[:, hq + hk:], PackedSequences(lengths, causal=True, device=DEV))
        loss = top_logit_distillation(o.reshape(t, -1) @ wo, values, indices, teacher_lse=lse, tau=0.5)
        return loss.detach(), *torch.autograd.grad(loss, (wq, wo))

    got = step()
    with reference_math():
        want = step()
    for a, b in zip(got, want, strict=True):
        # fp32 throughout: sums of at most 5000 terms, errors of 2^-24 a term growing like their root, few steps deep
        assert (a - b).norm() <= 2.0**-16 * b.norm()


def test_packed_crops_train_after_an_evaluation_in_inference_mode():
    kw = dict(img_size=32, patch_size=8, in_chans=1, embed_dim=128, depth=2, num_heads=2, n_storage_tokens=4)
    torch.manual_seed(0)
    model = DinoVisionTransformer3D(packed_crops=True, **kw).to(DEV)
    crops = [torch.randn(2, 1, 32, 32, 32, device=DEV), torch.randn(6, 1, 16, 16, 16, device=DEV)]
    with torch.autocast("cuda", dtype=torch.bfloat16):
        with torch.inference_mode():
            want = model.forward_features(crops, [None, None])
        out = model.forward_features(crops, [None, None])
        sum(o["x_norm_patchtokens"].float().sin().mean() for o in out).backward()
    assert all(torch.equal(a["x_prenorm"], b["x_prenorm"]) for a, b in zip(want, out, strict=True))
    assert model.blocks[0].attn.qkv.weight.grad.isfinite().all()


def test_a_captured_block_keeps_its_plan():
    """Replayed after more crop shapes than a model keeps plans for, with the memory that theirs may have left written to."""
    torch.manual_seed(0)
    attn = SelfAttention(128, num_heads=2).to(DEV, torch.bfloat16)
    attn.packed_crops = True
    crops = [torch.randn(2, 200, 128, device=DEV, dtype=torch.bfloat16), torch.randn(3, 90, 128, device=DEV, dtype=torch.bfloat16)]
    with torch.no_grad():
        want = attn.forward_list(crops, rope_list=[None, None])
        torch.cuda.synchronize()
        graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(graph, stream=side):
            got = attn.forward_list(crops, rope_list=[None, None])
            with pytest.raises(RuntimeError, match="before a graph is captured"):
                attn.forward_list([x[:, :7] for x in crops], rope_list=[None, None])
        for n in range(1, 81):
            attn.forward_list([crops[0][:, :n], crops[1][:, :n]], rope_list=[None, None])
        junk = [torch.zeros(n, device=DEV, dtype=torch.int32) for n in (512, 1024, 1340, 2048) for _ in range(200)]
        for x in got:
            x.zero_()
        graph.replay()
        torch.cuda.synchronize()
    assert len(junk) == 800 and all(torch.equal(a, b) for a, b in zip(got, want, strict=True))


@pytest.mark.parametrize("qk_norm", [False, True])
@pytest.mark.parametrize("packed", [False, True])
def test_blocks_train_after_an_evaluation_in_inference_mode(packed, qk_norm):
    """The channel pairs that blocks keep are saved for backward."""
    model = DinoVisionTransformer3D(img_size=32, patch_size=8, in_chans=1, embed_dim=128, depth=1, num_heads=2, qk_norm=qk_norm,
                                    packed_crops=packed).to(DEV)
    crops = [torch.randn(2, 1, 32, 32, 32, device=DEV), torch.randn(6, 1, 16, 16, 16, device=DEV)]
    with torch.autocast("cuda", dtype=torch.bfloat16):
        with torch.inference_mode():
            model.forward_features(crops, [None, None])
        out = model.forward_features(crops, [None, None])
        sum(o["x_norm_patchtokens"].float().sin().mean() for o in out).backward()
    assert model.blocks[0].attn.qkv.weight.grad.isfinite().all()


def test_saved_tensors_may_go_through_hooks():
    """Kept on the host between the passes (save_on_cpu), where strided views come back contiguous: the same bits."""
    torch.manual_seed(0)
    lengths, hq, hk, d = [130, 40, 1], 4, 2, 64
    t = sum(lengths)
    base = torch.randn(t, hq + 2 * hk, d, device=DEV).half()
    freq = torch.rand(3, 16, device=DEV)
    positions = torch.randn(t, 3, device=DEV)
    seq = PackedSequences(lengths, causal=True, device=DEV)
    wide = torch.randn(t, 2 * 300, device=DEV)
    values, indices, lse = top_logits(torch.randn(t, 300, device=DEV), 8)

    def step():
        x, f, s = (y.detach().clone().requires_grad_(True) for y in (base, freq, wide))
        q, k = rotary(x[:, :hq], x[:, hq:hq + hk], positions, f)
        o = packed_attention(q, k, x[:, hq + hk:], seq)
        loss = top_logit_distillation(s[:, ::2], values, indices, teacher_lse=lse)
        return torch.autograd.grad(o.float().sin().sum() + top_logit_distillation(s[:, 300:], values, indices) + loss, (x, f, s))

    want = step()
    with torch.autograd.graph.save_on_cpu():
        got = step()
    assert all(torch.equal(a, b) for a, b in zip(got, want, strict=True))
