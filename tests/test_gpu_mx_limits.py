"""Operands beyond 2^28 elements along their blocks, where their index in bits passes 32 bits."""
import pytest
import torch

from custom_matmul_kernels_b200 import MXDenseBMMCUDA, MXQuantizeCUDA

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("side", ["right", "left"])
def test_long_block_axis(dev, side):
    n, dtype = (1 << 28) + 200, torch.bfloat16
    X = torch.zeros((1, 1, n), device=dev, dtype=dtype)
    g = torch.Generator(dev).manual_seed(1)
    for at in (0, (1 << 27) - 100, (1 << 28) - 100, n - 200):
        X[0, 0, at:at + 200] = torch.randn(200, device=dev, generator=g).to(dtype)
    Q = MXQuantizeCUDA(8)(X)
    want = Q.dequantize(dtype)
    del X
    A = torch.full((1, 1, 1), 2.0, device=dev, dtype=dtype)  # one term per result: exact
    C = MXDenseBMMCUDA()(A, Q) if side == "right" else MXDenseBMMCUDA()(Q.mT, A).view(1, 1, n)
    assert torch.equal(C, want * 2)
    assert bool(C[0, 0, (1 << 28) - 100:(1 << 28)].any()) and bool(C[0, 0, -200:].any())
