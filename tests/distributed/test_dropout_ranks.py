"""Data-parallel ranks draw different dropout masks, though the Trainer seeds them alike (Gloo ranks)."""

from __future__ import annotations

from pathlib import Path

import pytest

pytestmark = pytest.mark.cpu_dist

CONFIG = """
experiment_name = "drop"
[model]
name = "vit3d"
img_size = [16, 16, 16]
patch_size = [8, 8, 8]
embed_dim = 32
depth = 1
num_heads = 2
dropout = 0.5
[algorithm]
name = "mae"
decoder_embed_dim = 16
decoder_depth = 1
decoder_num_heads = 2
[data]
name = "synthetic_volumes"
generator = "blobs"
shape = [16, 16, 16]
samples_per_epoch = 16
[trainer]
max_steps = 2
batch_size = 2
warmup_steps = 0
precision = "fp32"
checkpoint_every = 100
num_workers = 0
[parallelism]
{parallelism}
"""


def _drawn(rank, world, root, config_path):
    """(seed, offset) pairs of a short training run."""
    import mia_train_b200.ops.dropout as dropout
    from mia_train_b200.engine.run import run

    pairs = []
    real = dropout._draw

    def recording(device):
        pair = real(device)
        pairs.append(tuple(pair.tolist()))
        return pair

    dropout._draw = recording
    run(Path(config_path), output_root=Path(root), resume=None)
    return pairs


@pytest.mark.parametrize("parallelism", ["dp_shard = 2", "dp_replicate = 2"])
def test_ranks_draw_their_own_masks(run_distributed, tmp_path, parallelism):
    cfg = tmp_path / "drop.toml"
    cfg.write_text(CONFIG.format(parallelism=parallelism))
    out = run_distributed(_drawn, 2, str(tmp_path / "runs"), str(cfg))
    assert len(out[0]) == len(out[1]) >= 6  # three masks a block and step
    assert not set(out[0]) & set(out[1])
    # seeded alike: only the rank tells the pairs apart
    word = (1 << 64) - 1
    assert {(a ^ b) & word for (a, _), (b, _) in zip(out[0], out[1], strict=True)} == {0x9E3779B97F4A7C15}


def test_tensor_parallel_ranks_share_the_rank_of_their_replica():
    """Dropout itself is refused under tensor parallelism; the rank would be the same for the whole group."""
    from mia_train_b200.parallel.parallel_dims import ParallelDims

    class Mesh:
        def get_local_rank(self, name):
            return {"dp_replicate": 1, "dp_shard": 2}[name]

    assert ParallelDims(dp_replicate=2, dp_shard=3, tp=2).dp_rank(Mesh()) == 1 * 3 + 2
