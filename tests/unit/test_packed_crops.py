"""`packed_crops`: all crops of a step in one attention call, on the CPU and in 64 bits (in 32 the first norms, which divide
by the 0.02 of the initial class token, alone leave some gradients with three digits)."""

from __future__ import annotations

from copy import deepcopy

import pytest
import torch

from mia_train_b200.layers.dinov3.attention import SelfAttention
from mia_train_b200.layers.dinov3.rope import CropRopes, RopeTables
from mia_train_b200.models.dinov3_vit import DinoVisionTransformer
from mia_train_b200.models.dinov3_vit3d import DinoVisionTransformer3D
from mia_train_b200.ops.packed_attention import PackedSequences

KW = dict(patch_size=8, in_chans=1, embed_dim=48, depth=2, num_heads=2, n_storage_tokens=2, pos_embed_rope_dtype="fp32")


def _pair(cls=DinoVisionTransformer3D, **kw):
    torch.manual_seed(0)
    plain = cls(img_size=16, **KW, **kw)
    packed = cls(img_size=16, packed_crops=True, **KW, **kw)
    packed.load_state_dict(plain.state_dict())
    return plain.double(), packed.double()


def _same(a, b):
    """The crop-wise call rotates q and k in 32 bits: sine, cosine, two products and a sum, 4 half steps of 2^-24 of each,
    which move the scores (below 1 here) and with them the outputs by at most 2^-21 a block; a gradient has twice that
    from forward and backward pass, in both of the two blocks."""
    assert (a - b).abs().max() <= 2.0**-19 * a.abs().max()


def _crops(rank=3):
    torch.manual_seed(1)
    return [torch.randn(2, 1, *(16,) * rank).double(), torch.randn(5, 1, *(8,) * rank).double()]


def _features(model, crops, masks=None):
    out = model.forward_features(crops, masks or [None, None])
    loss = sum((o["x_norm_patchtokens"].sin().sum() + o["x_norm_clstoken"].square().sum()) for o in out)
    grads = torch.autograd.grad(loss, [p for p in model.parameters() if p.requires_grad], allow_unused=True)
    return [o[k] for o in out for k in ("x_norm_patchtokens", "x_norm_clstoken")], grads


@pytest.mark.parametrize("kw", [{}, {"qk_norm": True}, {"mask_k_bias": True, "layerscale_init": 0.1},
                                {"pos_embed_rope_type": "superposition"}], ids=str)
def test_packed_crops_give_what_separate_calls_give(kw):
    plain, packed = _pair(**kw)
    if "mask_k_bias" in kw:
        for m in (plain, packed):
            for blk in m.blocks:
                blk.attn.qkv.bias_mask.fill_(1.0)
    masks = [torch.tensor([[True, False, True] + [False] * 5] * 2), None]
    for want, got in zip(*(_features(m, _crops(), masks) for m in (plain, packed)), strict=True):
        for a, b in zip(want, got, strict=True):
            assert (a is None) == (b is None)
            if a is not None:
                _same(a, b)


def test_packed_crops_of_the_2d_model_and_one_crop_size():
    plain, packed = _pair(DinoVisionTransformer)
    for want, got in zip(_features(plain, _crops(2))[0], _features(packed, _crops(2))[0], strict=True):
        _same(want, got)
    x = _crops(2)[0]
    assert torch.equal(plain(x), packed(x))  # nothing to pack


def test_packed_crops_with_stochastic_depth():
    plain, packed = _pair(drop_path_rate=0.4)
    out = []
    for m in (plain, packed):
        m.train()
        torch.manual_seed(3)  # the blocks draw the same samples
        out.append(_features(m, _crops())[0])
    for a, b in zip(*out, strict=True):
        _same(a, b)


def test_the_packed_path_runs(monkeypatch):
    from mia_train_b200.layers.dinov3 import attention as module

    calls = []
    real = module.packed_attention
    monkeypatch.setattr(module, "packed_attention", lambda *a: calls.append(a[0].shape) or real(*a))
    _, packed = _pair()
    packed.forward_features(_crops(), [None, None])
    assert calls == [(2 * 11 + 5 * 4, 2, 24)] * 2  # 8 + 3 and 1 + 3 tokens, two blocks
    learned = _pair(pos_embed_rope_type="superposition")[1]
    calls.clear()
    learned.forward_features(_crops(), [None, None])
    assert not calls or not learned.rope_embed.depth_scale.requires_grad


def test_blocks_share_their_plans():
    model = DinoVisionTransformer3D(img_size=16, packed_crops=True, **KW)
    model.forward_features([x.float() for x in _crops()], [None, None])
    shapes = ((2, 11), (5, 4))
    plan = model.blocks[0].attn.crop_plans(shapes, torch.device("cpu"))
    assert plan is model.blocks[1].attn.crop_plans(shapes, torch.device("cpu")) and len(model.blocks[0].attn.crop_plans._recent) == 1


def test_plans_stay_as_long_as_a_captured_step_may_read_them(monkeypatch):
    from mia_train_b200.layers.dinov3 import attention as module

    cpu, plans = torch.device("cpu"), module.CropPlans(most=3)
    first = plans(((2, 5),), cpu)
    assert plans(((2, 5),), cpu) is first
    monkeypatch.setattr(module, "capturing", lambda device: True)
    assert plans(((2, 5),), cpu) is first
    monkeypatch.setattr(module, "capturing", lambda device: False)
    others = [plans(((1, n),), cpu) for n in range(1, 9)]
    assert plans(((2, 5),), cpu) is first and plans(((1, 8),), cpu) is others[-1]
    assert plans(((1, 1),), cpu) is not others[0]  # the others go, the longest unused first
    assert plans._recent.keys() == {(((1, n),), cpu) for n in (1, 7, 8)}


def test_plans_are_not_made_while_a_graph_is_captured(monkeypatch):
    from mia_train_b200.ops import packed_attention as module

    monkeypatch.setattr(module, "capturing", lambda device: True)
    with pytest.raises(RuntimeError, match="before a graph is captured"):
        PackedSequences([3], device="cpu")


def test_a_copied_model_has_plans_of_its_own():
    model = DinoVisionTransformer3D(img_size=16, packed_crops=True, **KW)
    model.forward_features([x.float() for x in _crops()], [None, None])
    copy = deepcopy(model)
    mine, its = model.blocks[0].attn.crop_plans, copy.blocks[0].attn.crop_plans
    assert its is not mine and its is copy.blocks[1].attn.crop_plans and its._recent.keys() == mine._recent.keys()
    for a, b in zip(model.forward_features([x.float() for x in _crops()], [None, None]),
                    copy.forward_features([x.float() for x in _crops()], [None, None]), strict=True):
        assert torch.equal(a["x_prenorm"], b["x_prenorm"])


def test_channel_pairs_made_in_inference_mode_serve_training():
    model = DinoVisionTransformer3D(img_size=16, **KW)
    with torch.inference_mode():
        model.forward_features([x.float() for x in _crops()], [None, None])
    assert not model.blocks[0].attn._pairs.is_inference()


def test_angles_are_those_of_the_call():
    """One rotation in several lists, or changed in place between two calls."""
    torch.manual_seed(0)
    attn = SelfAttention(48, num_heads=2).double()
    attn.packed_crops = True
    x = [torch.randn(2, 9, 48).double(), torch.randn(3, 5, 48).double()]
    first, *second = (RopeTables(3 * torch.randn(n, 12)) for n in (8, 4, 4))

    def check(ropes):
        packed = attn.forward_list(x, rope_list=ropes)
        for a, b in zip(packed, (attn(t, rope=r) for t, r in zip(x, ropes, strict=True)), strict=True):
            _same(a, b)
        return packed[1]

    outs = [check([first, r]) for r in second]
    second[1].angles.mul_(0.5)
    outs.append(check([first, second[1]]))
    outs.append(check(CropRopes([first, second[0]])))
    assert torch.equal(outs[0], outs[3]) and not any(torch.equal(outs[0], y) for y in outs[1:3])
    given = [RopeTables(torch.randn(b, n, 12)) for b, n in ((2, 9), (3, 5))]  # angles of every sample: crop by crop
    check(given)


@pytest.mark.parametrize("kw", [{}, {"drop_path_rate": 0.4}], ids=str)
def test_the_blocks_of_a_forward_pass_share_their_angles(kw, monkeypatch):
    from mia_train_b200.layers.dinov3 import rope as module

    calls = []
    real = module.angles_end_to_end
    monkeypatch.setattr(module, "angles_end_to_end", lambda *a: calls.append(a[1]) or real(*a))
    model = DinoVisionTransformer3D(img_size=16, packed_crops=True, **KW, **kw).train()
    for n in (1, 2):
        model.forward_features([x.float() for x in _crops()], [None, None])
        assert len(calls) == n
