"""What tensor parallelism refuses of dropout: the framework's own blocks with it, nothing else (Gloo ranks)."""

from __future__ import annotations

import pytest
import torch
import torch.nn as nn

pytestmark = pytest.mark.cpu_dist


def _model(kind):
    from mia_train_b200.models.dinov3_vit3d import DinoVisionTransformer3D
    from mia_train_b200.models.vit import ViT3D

    torch.manual_seed(0)
    if kind.startswith("dinov3"):
        return DinoVisionTransformer3D(img_size=16, patch_size=4, embed_dim=32, depth=1, num_heads=4,
                                       ffn_layer="swiglu" if "swiglu" in kind else "mlp",
                                       drop_rate=0.1 if "drop" in kind else 0.0)
    model = ViT3D(img_size=(16, 16, 16), patch_size=(8, 8, 8), embed_dim=32, depth=1, num_heads=4,
                  dropout=0.1 if kind == "vit3d drop" else 0.0)
    if kind == "own":  # as a user's model has it: a module of that name, inactive, and one that is active, outside the blocks
        model.head = nn.TransformerEncoderLayer(32, 2, 32, dropout=0.0)
        model.dropout = nn.Dropout(0.0)
        model.input_dropout = nn.Dropout(0.1)
    return model


def _apply(rank, world, kind):
    import torch.distributed as dist
    from torch.distributed.device_mesh import init_device_mesh

    from mia_train_b200.parallel.parallel_dims import ParallelDims
    from mia_train_b200.parallel.parallelize import _apply_tensor_parallel

    mesh = init_device_mesh("cpu", (world,), mesh_dim_names=("tp",))
    try:
        _apply_tensor_parallel(_model(kind), mesh, ParallelDims(tp=world, tp_comm="allreduce"))
    except ValueError as error:
        dist.barrier()
        return str(error)
    dist.barrier()
    return "accepted"


@pytest.mark.parametrize("kind", ["vit3d", "own", "dinov3"])
def test_models_without_dropout_in_their_blocks_are_accepted(run_distributed, kind):
    assert set(run_distributed(_apply, 2, kind).values()) == {"accepted"}


@pytest.mark.parametrize("kind", ["vit3d drop", "dinov3 drop", "dinov3 swiglu drop"])
def test_blocks_with_dropout_are_refused(run_distributed, kind):
    for message in run_distributed(_apply, 2, kind).values():
        assert "dropout" in message and "tensor parallelism" in message
