"""The same inputs give the same bits, whatever ran before: the wide products (CTA pairs), over and over, with other
work and other operands between."""
import pytest
import torch

from custom_matmul_kernels_b200 import CheckpointBMMCUDA, MXBMMCUDA, MXDenseBMMCUDA, MXQuantizeCUDA

pytestmark = pytest.mark.gpu


def rnd(shape, seed, dev, dtype):
    g = torch.Generator(dev).manual_seed(seed)
    return torch.randn(shape, device=dev, generator=g).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,k,n", [(4096, 2048, 2048), (2900, 2312, 3000)])
def test_wide_products_repeat(dev, m, k, n, dtype):
    A, B, dC = rnd((1, m, k), 1, dev, dtype), rnd((1, k, n), 2, dev, dtype), rnd((1, m, n), 3, dev, dtype)
    A8, A4, W = MXQuantizeCUDA(8)(A), MXQuantizeCUDA(4)(A), MXQuantizeCUDA(4)(B, dim=-2)
    other = MXQuantizeCUDA(8)(rnd((1, m, k), 4, dev, dtype))
    calls = {
        "dense": lambda: CheckpointBMMCUDA()(A.detach().requires_grad_(), B).detach(),
        "8-bit, left": lambda: MXDenseBMMCUDA()(A8.mT, dC),
        "8-bit, right": lambda: MXDenseBMMCUDA()(dC.transpose(1, 2), A8),
        "4-bit, left": lambda: MXDenseBMMCUDA()(A4.mT, dC),
        "4-bit, right": lambda: MXDenseBMMCUDA()(dC, W.mT),
        "4-bit product": lambda: MXBMMCUDA(out_dtype=dtype)(A4, W),
        "4-bit product of a tensor": lambda: MXBMMCUDA()(A, W),
    }
    first = {name: call() for name, call in calls.items()}
    wrong = torch.zeros(len(calls), device=dev, dtype=torch.int64)
    for i in range(30):
        if i % 3 == 1:
            MXDenseBMMCUDA()(other.mT, dC)
        for j, (name, call) in enumerate(calls.items()):
            wrong[j] += (call() != first[name]).sum()
    assert wrong.tolist() == [0] * len(calls), dict(zip(calls, wrong.tolist()))


def test_training_step_repeats(dev):
    """Forward and backward pass of a wide projection, with a step on other operands between."""
    def operands(seed):
        return [rnd(s, seed + i, dev, torch.bfloat16) for i, s in enumerate(((1, 8192, 4096), (1, 4096, 4096), (1, 8192, 4096)))]

    def step(A, B, dC):
        A, B = A.detach().requires_grad_(), B.detach().requires_grad_()
        C = CheckpointBMMCUDA()(A, B)
        return (C.detach(),) + torch.autograd.grad(C, (A, B), dC)

    one, two = operands(1), operands(11)
    first, wrong = step(*one), torch.zeros(3, device=dev, dtype=torch.int64)
    for _ in range(25):
        step(*two)
        for j, (x, y) in enumerate(zip(step(*one), first)):
            wrong[j] += (x != y).sum()
    assert wrong.tolist() == [0, 0, 0]
