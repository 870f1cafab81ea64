"""`set_rank`: the masks of data-parallel ranks."""

from __future__ import annotations

import pytest
import torch

from mia_train_b200.ops.dropout import dropout, set_rank


@pytest.fixture(autouse=True)
def _rank_zero():
    yield
    set_rank(0)


def _mask(rank, rng=None):
    set_rank(rank)
    torch.manual_seed(3)
    return dropout(torch.ones(4096), 0.5, rng=rng) != 0


def test_ranks_draw_apart_and_rank_zero_as_one_process():
    torch.manual_seed(3)
    alone = dropout(torch.ones(4096), 0.5) != 0
    masks = [_mask(r) for r in (0, 1, 2, 7)]
    assert torch.equal(masks[0], alone) and torch.equal(_mask(1), masks[1])
    for i in range(4):
        for j in range(i):
            # 4096 pairs of fair draws: equal in half of them, within six standard deviations (32 each)
            assert abs((masks[i] == masks[j]).sum().item() - 2048) < 6 * 32


def test_a_given_pair_is_taken_as_it_is():
    rng = torch.tensor([5, 4])
    assert torch.equal(_mask(0, rng), _mask(3, rng))


def test_backward_replays_the_rank_s_mask():
    set_rank(5)
    x = torch.ones(1000, requires_grad=True)
    y = dropout(x, 0.5)
    set_rank(0)
    assert torch.equal(torch.autograd.grad(y.sum(), x)[0], y.detach())


def test_negative_ranks_are_refused():
    with pytest.raises(ValueError, match="rank"):
        set_rank(-1)
