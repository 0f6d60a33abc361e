"""4-bit products whose 128-row tiles, k shared, just fit the SMs at once, and just do not: kernels change there."""
import pytest
import torch

from custom_matmul_kernels_b200 import MXBMMCUDA, MXQuantizeCUDA

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("l,m,n,k", [(1, 128, 4736, 8200), (1, 128, 4864, 8200), (1, 512, 5120, 4100), (3, 130, 3100, 4096), (1, 1024, 2500, 5000)])
def test_products(dev, l, m, n, k, dtype):
    g = torch.Generator(dev).manual_seed(m + n)
    A4 = MXQuantizeCUDA(4)(torch.randn((l, m, k), device=dev, generator=g))
    B4 = MXQuantizeCUDA(4)(torch.randn((l, n, k), device=dev, generator=g)).mT
    a, b = A4.dequantize().double(), B4.dequantize().double()
    want, mag = a @ b, a.abs() @ b.abs()
    C = MXBMMCUDA(out_dtype=dtype)(A4, B4)
    fi = torch.finfo(dtype)
    # one rounding of the type, 2^-23 of the terms' magnitudes per fp32 addition
    tol = want.abs() * (fi.eps / 2) + mag * (k * 2.0 ** -23) * (1 + fi.eps)
    assert bool(((C.double() - want).abs() <= tol).all())
    assert torch.equal(MXBMMCUDA(out_dtype=dtype)(A4, B4), C)
