"""`packed_crops` from a configuration, and under tensor and data parallelism on Gloo ranks."""

from __future__ import annotations

from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.cpu_dist

KW = dict(img_size=16, patch_size=4, embed_dim=48, depth=2, num_heads=4, n_storage_tokens=2)


def _crops():
    torch.manual_seed(1)
    return [torch.randn(2, 1, 16, 16, 16), torch.randn(3, 1, 8, 8, 8)]


def _loss(model):
    out = model.forward_features(_crops(), [None, None])
    return sum(o["x_norm_patchtokens"].sin().mean() + o["x_norm_clstoken"].sin().mean() for o in out)


def _sharded_against_whole(rank, world, kw):
    import torch.distributed as dist

    from mia_train_b200.models.dinov3_vit3d import DinoVisionTransformer3D
    from mia_train_b200.ops import packed_attention as ops
    from mia_train_b200.parallel.tensor_parallel import apply_tensor_parallel

    whole, sharded = (DinoVisionTransformer3D(packed_crops=packed, **KW, **kw) for packed in (False, True))
    sharded.load_state_dict(whole.state_dict())
    whole, sharded = whole.double(), sharded.double()
    assert apply_tensor_parallel(sharded.tensor_parallel_plan(), dist.group.WORLD) > 0
    crops = _crops
    globals()["_crops"] = lambda: [x.double() for x in crops()]
    made = []
    real = ops.PackedSequences.__init__
    ops.PackedSequences.__init__ = lambda self, *a, **k: made.append(1) or real(self, *a, **k)
    losses = [_loss(m) for m in (whole, sharded)]
    for x in losses:
        x.backward()
    worst = 0.0
    for p, q in zip(sharded.parameters(), whole.parameters(), strict=True):
        if p.shape == q.shape and p.grad is not None:
            worst = max(worst, float((p.grad - q.grad).abs().max() / q.grad.abs().max().clamp(min=1e-30)))
    return len(made), float((losses[0] - losses[1]).abs() / losses[0].abs()), worst


@pytest.mark.parametrize("kw", [{}, {"qk_norm": True}], ids=str)
def test_packed_crops_under_tensor_parallelism(run_distributed, kw):
    """Each rank packs its own heads. In 64 bits but for the rotation, which the crop-wise call makes in 32 (2^-21 a block of
    scores below 1, as for the whole model), behind norms that divide by the 0.02 of the initial class token."""
    for made, loss, worst in run_distributed(_sharded_against_whole, 2, kw).values():
        assert made == 1 and loss <= 2.0**-19 and worst <= 2.0**-19 / 0.02


CONFIG = """
experiment_name = "dino"

[model]
name = "dinov3_vit3d"
img_size = 16
patch_size = 4
embed_dim = 32
depth = 2
num_heads = 2
packed_crops = true

[algorithm]
name = "dinov3"
global_crop_size = 16
local_crop_size = 8
n_local_crops = 2
head_n_prototypes = 64
head_hidden_dim = 32
head_bottleneck_dim = 16
total_steps = 10
warmup_teacher_temp_steps = 4

[data]
name = "synthetic_volumes"
shape = [24, 24, 24]
samples_per_epoch = 16

[trainer]
max_steps = 2
batch_size = 2
lr = 1e-3
warmup_steps = 1
precision = "fp32"
log_every = 1
checkpoint_every = 2
seed = 0

[parallelism]
{parallelism}
"""


def _packs_in_training(rank, world, root, config_path):
    from mia_train_b200.engine.run import run
    from mia_train_b200.layers.dinov3.attention import SelfAttention

    calls = []
    real = SelfAttention._attend_packed

    def recording(self, *a):
        calls.append(1)
        return real(self, *a)

    SelfAttention._attend_packed = recording
    run(Path(config_path), output_root=Path(root))
    return len(calls)


@pytest.mark.parametrize("parallelism", ["dp_shard = 2", 'tp = 2\ntp_comm = "allreduce"', 'tp = 2\ntp_comm = "collective"'])
def test_packed_crops_train_from_a_configuration(run_distributed, tmp_path, parallelism):
    cfg = tmp_path / "dino.toml"
    cfg.write_text(CONFIG.format(parallelism=parallelism))
    for calls in run_distributed(_packs_in_training, 2, str(tmp_path / "runs"), str(cfg)).values():
        assert (calls > 0) == ("collective" not in parallelism)  # the sequence-parallel modes go crop by crop
