"""Codes and scales have batch strides of their own: either may be one matrix for every batch while the other is not.

Tolerances as in test_gpu_mx.py: one rounding of the result's type and 2^-23 of the terms' magnitudes per fp32 addition."""
import itertools

import pytest
import torch

from custom_matmul_kernels_b200 import MXBMMCUDA, MXDenseBMMCUDA, MXTensor
from oracle import mx_semantics as S

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
MIXED = list(itertools.product((False, True), repeat=2))


def mixed(l, rows, k, bits, dev, one_code, one_scale, dim=-1):
    """(operand with the asked strides of 0, the same with copies, its float64 values [l, rows, k])."""
    codes, scales = zip(*(S.random_mx(rows, k, bits, 7 + i, lo=121, hi=126) for i in range(l)))
    codes = [codes[0]] * l if one_code else list(codes)
    scales = [scales[0]] * l if one_scale else list(scales)
    packed = [S.pack(c, s, bits) for c, s in zip(codes, scales)]
    C, E = (torch.stack([p[i] for p in packed]).to(dev) for i in (0, 1))
    copies = MXTensor(C, E, bits=bits, k=k, dim=dim)
    got = MXTensor(C[:1].expand(l, -1, -1) if one_code else C, E[:1].expand(l, -1, -1, -1) if one_scale else E, bits=bits, k=k,
                   dim=dim)
    assert (got.codes.stride(0) == 0) == one_code and (got.scales.stride(0) == 0) == one_scale
    return got, copies, torch.stack([S.values(c, s, bits) for c, s in zip(codes, scales)])


def assert_close(got, want, magnitude, K):
    fi = torch.finfo(got.dtype)
    tol = want.abs() * (fi.eps / 2) + magnitude * (K * 2.0 ** -23) * (1 + fi.eps) + fi.smallest_normal * fi.eps
    err = (got.detach().double().cpu() - want).abs()
    assert bool((err <= tol).all()), f"off by {float((err / tol).max()):.3g} tolerances"


@pytest.mark.parametrize("one_code,one_scale", MIXED)
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("l,m,j,c", [(3, 5, 70, 40), (2, 130, 96, 200), (2, 60, 4000, 100), (3, 1100, 70, 1300)])
def test_dense_product(dev, l, m, j, c, dtype, bits, one_code, one_scale):
    """Single tiles, long sums shared by clusters, and tiles on CTA pairs; the microscaled operand on either side."""
    Q, copies, q = mixed(l, j, c, bits, dev, one_code, one_scale)
    g = torch.Generator().manual_seed(3)
    P = (torch.randn((l, m, j), generator=g) * 0.5).to(dtype)
    want, mag = P.double() @ q, P.double().abs() @ q.abs()
    for X in (P.to(dev), P.transpose(1, 2).contiguous().to(dev).transpose(1, 2)):
        C, D = MXDenseBMMCUDA()(X, Q), MXDenseBMMCUDA()(Q.mT, X.transpose(1, 2))
        assert torch.equal(C, MXDenseBMMCUDA()(X, copies)) and torch.equal(D, MXDenseBMMCUDA()(copies.mT, X.transpose(1, 2)))
        assert_close(C, want, mag, j)
        assert_close(D, want.transpose(1, 2), mag.transpose(1, 2), j)


@pytest.mark.parametrize("one_code,one_scale", MIXED)
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("l,m,n,k", [(3, 1, 40, 64), (2, 70, 150, 300), (4, 640, 520, 96)])
def test_four_bit_product_and_its_gradient(dev, l, m, n, k, dtype, one_code, one_scale):
    W, copies, w = mixed(l, n, k, 4, dev, one_code, one_scale, dim=-2)
    g = torch.Generator().manual_seed(4)
    A, dC = torch.randn((l, m, k), generator=g).to(dtype), torch.randn((l, m, n), generator=g).to(dtype)
    got = []
    for operand in (W, copies):
        x = A.to(dev).requires_grad_()
        C = MXBMMCUDA()(x, operand)
        got.append((C.detach(),) + torch.autograd.grad(C, x, dC.to(dev)))
    assert all(torch.equal(a, b) for a, b in zip(*got))
    a = torch.stack([S.values(*S.quantize(x, 4), 4) for x in A])
    assert_close(got[0][0], a @ w.transpose(1, 2), a.abs() @ w.abs().transpose(1, 2), k)
    # the fp32 gradient's product splits each term in three
    assert_close(got[0][1], dC.double() @ w, dC.double().abs() @ w.abs(), n * (8 if dtype == F32 else 1))


@pytest.mark.parametrize("one_code,one_scale", MIXED)
@pytest.mark.parametrize("bits", [4, 8])
def test_both_operands_and_dequantisation(dev, bits, one_code, one_scale):
    Q, _, q = mixed(3, 140, 300, bits, dev, one_code, one_scale)
    for dtype in (F32, F16, BF16):
        assert torch.equal(Q.dequantize(dtype).cpu(), q.to(F32).to(dtype))
    if bits == 4:
        for m in (4, 150):
            A, _, a = mixed(3, m, 300, 4, dev, one_scale, one_code)
            C = MXBMMCUDA()(A, Q.mT)
            assert_close(C, a @ q.transpose(1, 2), a.abs() @ q.abs().transpose(1, 2), 300)
