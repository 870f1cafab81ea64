"""Epilogues of the native 8-bit product that read what TMA and the tensor core left for a whole warp."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover - collected on CPU, skipped there
    pytest.skip("needs CUDA", allow_module_level=True)

from mia_train_b200.ops import _native  # noqa: E402
from mia_train_b200.ops.fp8 import BLOCK, fp8_gemm, quantize_fp8  # noqa: E402

DEV = torch.device("cuda", 0)
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(params=[0, 1], ids=["128x128", "256x256"])
def tile(request):
    previous = _native.native().set_fp8_tile(request.param)
    yield request.param
    _native.native().set_fp8_tile(previous)


def _no_errors():
    torch.cuda.synchronize()
    assert _native.native().check_errors(0) == 0


@pytest.mark.parametrize("b_block", [True, False])
@pytest.mark.parametrize("m,n,k", [(4096, 2568, 256), (8192, 1280, 1280)])
def test_residual_repeats_are_identical(m, n, k, b_block, tile):
    """Products and residual are integers that every sum holds exactly, so each repeat has one right answer."""
    torch.manual_seed(0)
    a = quantize_fp8(torch.randint(-4, 5, (m, k), device=DEV).float())
    b = quantize_fp8(torch.randint(-4, 5, (n, k), device=DEV).float(), block_rows=BLOCK if b_block else 1)
    res = torch.randint(-128, 129, (m, n), device=DEV).bfloat16()
    want = (a.dequantize().double() @ b.dequantize().double().t() + res.double()).to(BF16)
    for _ in range(8):
        assert torch.equal(fp8_gemm(a, b, residual=res), want)
    _no_errors()
