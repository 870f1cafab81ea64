"""Masks of data-parallel ranks on the GPU: drawn apart, replayed in backward and in captured graphs."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover - collected on CPU, skipped there
    pytest.skip("needs CUDA", allow_module_level=True)

from mia_train_b200.ops.dropout import dropout, set_rank  # noqa: E402

DEV = torch.device("cuda", 0)


@pytest.fixture(autouse=True)
def _rank_zero():
    yield
    set_rank(0)


def _run(rank):
    set_rank(rank)
    torch.manual_seed(3)
    x = torch.ones(1 << 14, device=DEV, requires_grad=True)
    y = dropout(x, 0.5)
    set_rank(0)  # the recorded pair counts in backward, not the rank of that moment
    assert torch.equal(torch.autograd.grad(y.sum(), x)[0], y.detach())
    return y.detach() != 0


def test_ranks_draw_apart():
    torch.manual_seed(3)
    alone = dropout(torch.ones(1 << 14, device=DEV), 0.5) != 0
    masks = [_run(r) for r in (0, 1, 2, 7)]
    assert torch.equal(masks[0], alone) and torch.equal(_run(1), masks[1])
    for i in range(4):
        for j in range(i):
            # fair draws agree in half of the places, within six standard deviations of 64
            assert abs((masks[i] == masks[j]).sum().item() - (1 << 13)) < 6 * 64


def test_captured_masks_are_the_rank_s():
    x = torch.ones(1 << 14, device=DEV)
    drawn = {}
    for rank in (0, 1):
        set_rank(rank)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = dropout(x, 0.5)
        torch.manual_seed(9)
        graph.replay()
        torch.cuda.synchronize()
        drawn[rank] = y.clone()
        torch.manual_seed(9)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, drawn[rank])
    assert not torch.equal(drawn[0], drawn[1])
