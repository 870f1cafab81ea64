"""A block takes attention classes that were written before the query/key norm."""

from __future__ import annotations

import pytest
import torch

from mia_train_b200.layers.dinov3.attention import SelfAttention
from mia_train_b200.layers.dinov3.block import SelfAttentionBlock


class Plain(SelfAttention):
    def __init__(self, dim, num_heads=8, qkv_bias=False, proj_bias=True, attn_drop=0.0, proj_drop=0.0, mask_k_bias=False,
                 use_fa4=False, device=None):
        super().__init__(dim, num_heads, qkv_bias, proj_bias, attn_drop, proj_drop, mask_k_bias, use_fa4, device=device)


def test_attention_class_without_qk_norm():
    torch.manual_seed(0)
    ours = SelfAttentionBlock(32, 2)
    block = SelfAttentionBlock(32, 2, attn_class=Plain)
    block.load_state_dict(ours.state_dict())
    x = torch.randn(2, 5, 32)
    assert torch.equal(block(x), ours(x))
    with pytest.raises(TypeError, match="qk_norm"):
        SelfAttentionBlock(32, 2, attn_class=Plain, qk_norm=True)


def test_new_options_come_after_every_former_argument():
    """Calls with positional arguments mean what they meant."""
    import inspect

    from mia_train_b200.models.dinov3_vit import DinoVisionTransformer
    from mia_train_b200.models.dinov3_vit3d import DinoVisionTransformer3D

    for cls in (SelfAttention, SelfAttentionBlock, DinoVisionTransformer, DinoVisionTransformer3D):
        names = list(inspect.signature(cls.__init__).parameters)
        assert names.index("device") < names.index("qk_norm"), cls.__name__
    attn = SelfAttention(32, 2, False, True, 0.0, 0.0, False, False, torch.device("cpu"))
    assert attn.q_norm is None
