"""Query/key norms under tensor parallelism, and the options that tensor parallelism refuses (Gloo ranks)."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.cpu_dist


def _build(kind: str, **kw):
    """`loud`: weights large enough for the attention to be far from uniform."""
    model = _build_quiet(kind.removesuffix("_loud"), **kw)
    if kind.endswith("_loud"):
        torch.manual_seed(2)
        for p in model.parameters():
            torch.nn.init.normal_(p, std=0.3)
    return model


def _build_quiet(kind: str, **kw):
    from mia_train_b200.models.dinov3_vit3d import DinoVisionTransformer3D
    from mia_train_b200.models.vit import ViT3D

    torch.manual_seed(0)
    if kind == "vit3d":
        return ViT3D(img_size=(16, 16, 16), patch_size=(8, 8, 8), embed_dim=32, depth=2, num_heads=4, qk_norm=True, **kw)
    return DinoVisionTransformer3D(img_size=16, patch_size=4, embed_dim=32, depth=2, num_heads=4, n_storage_tokens=1,
                                   window_size=2, global_every=2, qk_norm=True)


def _loss(model, x):
    if hasattr(model, "forward_features"):
        out = model.forward_features(x)
        return out["x_norm_patchtokens"].square().mean() + out["x_norm_clstoken"].sum() * 0.1
    return model(x).square().mean()


def _matches_dense(rank, world, kind):
    import torch.distributed as dist

    from mia_train_b200.parallel.tensor_parallel import apply_tensor_parallel

    # in 64 bits: untrained attention is almost uniform, and a norm's gradient, a sum of terms P (dP - sum P dP) that
    # cancel, lies below the 32-bit rounding of dP (2^-24 of it; measured gradients 2e-9)
    dense, tp = _build(kind).double(), _build(kind).double()
    torch.manual_seed(1)
    x = torch.randn(2, 1, 16, 16, 16).double()
    ref = _loss(dense, x)
    ref.backward()
    apply_tensor_parallel(tp.tensor_parallel_plan(), dist.group.WORLD)
    out = _loss(tp, x)
    out.backward()
    norms = {n: (p, q) for (n, p), (_, q) in zip(tp.named_parameters(), dense.named_parameters(), strict=True) if "_norm." in n}
    worst = max(float((p.grad - q.grad).abs().max() / q.grad.abs().max()) for n, (p, q) in norms.items()
                if "q_norm" in n or "k_norm" in n)
    return len(norms), float((out - ref).abs() / ref.abs().clamp(min=1.0)), worst


@pytest.mark.parametrize("kind", ["vit3d", "windowed", "vit3d_loud", "windowed_loud"])
def test_norm_gradients_cover_every_head(run_distributed, kind):
    for n, loss_diff, worst in run_distributed(_matches_dense, 2, kind).values():
        assert n >= 4 and loss_diff < 1e-5 and worst < 1e-3


def _refuses(rank, world):
    import torch.distributed as dist
    from torch.distributed.device_mesh import init_device_mesh

    from mia_train_b200.parallel.parallel_dims import ParallelDims
    from mia_train_b200.parallel.parallelize import _apply_tensor_parallel

    dims = ParallelDims(tp=world)
    mesh = init_device_mesh("cpu", (world,), mesh_dim_names=("tp",))
    try:
        _apply_tensor_parallel(_build("vit3d", dropout=0.1), mesh, dims)
    except ValueError as error:
        dist.barrier()
        return str(error)
    return "accepted"


def test_dropout_is_refused(run_distributed):
    for message in run_distributed(_refuses, 2).values():
        assert "dropout" in message and "tensor parallelism" in message
