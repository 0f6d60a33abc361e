"""The differentiable products have no forward mode: a tangent is refused, with or without reverse-mode gradients, and
not dropped."""
import pytest
import torch
from torch.autograd import forward_ad

from custom_matmul_kernels_b200 import CheckpointBMMCUDA, MXBMMCUDA, MXQuantizeCUDA


@pytest.mark.parametrize("grad", [False, True])
def test_checkpoint_refuses_before_anything_else(lib, grad):
    A, B = torch.ones(1, 2, 3), torch.ones(1, 3, 4)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(A.requires_grad_(grad), torch.ones(1, 2, 3))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            CheckpointBMMCUDA()(dual, B)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            CheckpointBMMCUDA()(A, forward_ad.make_dual(B, torch.ones(1, 3, 4)))


@pytest.mark.gpu
@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_products_refuse(dev, dtype, grad):
    A, B = torch.randn(1, 8, 64, device=dev, dtype=dtype), torch.randn(1, 64, 16, device=dev, dtype=dtype)
    W = MXQuantizeCUDA(4)(B, dim=-2)
    want = MXBMMCUDA()(A, W), CheckpointBMMCUDA()(A, B)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(A.detach().requires_grad_(grad), torch.ones_like(A))
        for call in (lambda: MXBMMCUDA()(dual, W), lambda: CheckpointBMMCUDA()(dual, B),
                     lambda: CheckpointBMMCUDA()(A, forward_ad.make_dual(B, torch.ones_like(B)))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        # operands without a tangent pass inside the same level
        got = MXBMMCUDA()(A, W), CheckpointBMMCUDA()(A, B)
    assert all(torch.equal(g, w) for g, w in zip(got, want))
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(lambda x: MXBMMCUDA()(x, W), (A,), (torch.ones_like(A),))


@pytest.mark.gpu
def test_backward_passes_refuse(dev):
    A, B = torch.randn(1, 8, 64, device=dev, requires_grad=True), torch.randn(1, 64, 16, device=dev, requires_grad=True)
    W = MXQuantizeCUDA(4)(B.detach(), dim=-2)
    for C in (MXBMMCUDA()(A, W), CheckpointBMMCUDA()(A, B)):
        with forward_ad.dual_level():
            dC = forward_ad.make_dual(torch.ones_like(C), torch.ones_like(C))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                torch.autograd.grad(C, A, dC)
