"""The 8-bit codes 0x7f and 0xff, which the quantiser does not write but a caller's MXTensor may hold, read as NaN in
every type, at every scale and in every product; their neighbours keep their values."""
import pytest
import torch

from custom_matmul_kernels_b200 import MXDenseBMMCUDA, MXTensor
from oracle import mx_semantics as S

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def with_nan(rows, k, dev, at, lo, hi):
    codes, scales = S.random_mx(rows, k, 8, 5, lo=lo, hi=hi)
    for i, (r, c) in enumerate(at):
        codes[r, c] = 127 + 128 * (i % 2)
    p = S.pack(codes, scales, 8)
    return MXTensor(p[0].to(dev), p[1].to(dev), bits=8, k=k), S.values(codes, scales, 8)


@pytest.mark.parametrize("lo,hi", [(118, 122), (0, 8), (128, 133)])  # the last two partly beyond fp16 and the fast forms
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,k", [(1, 1), (5, 33), (130, 272), (128, 128)])
def test_dequantised(dev, rows, k, dtype, lo, hi):
    at = {(0, 0), (rows - 1, k - 1), (rows // 2, k // 2), (rows // 2, min(k - 1, k // 2 + 3)), (rows // 3, k // 5)}
    Q, v = with_nan(rows, k, dev, sorted(at), lo, hi)
    got = Q.dequantize(dtype).cpu()
    want = v.to(F32).to(dtype)
    assert torch.equal(torch.isnan(got), torch.isnan(v))
    keep = ~torch.isnan(v)
    assert torch.equal(got[keep], want[keep])


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("m,j,c", [(7, 40, 70), (60, 4000, 100), (2100, 200, 2300)])
def test_products(dev, m, j, c, dtype):
    """Single tiles, sums shared by clusters, CTA pairs."""
    at = [(0, 0), (j - 1, c - 1), (j // 2, c // 3)]
    Q, q = with_nan(j, c, dev, at, 119, 123)
    clean, _ = with_nan(j, c, dev, [], 119, 123)
    g = torch.Generator().manual_seed(3)
    P = torch.randn((m, j), generator=g).to(dtype).to(dev)
    columns = torch.zeros(c, dtype=torch.bool)
    columns[[x for _, x in at]] = True
    for X in (P, P.t().contiguous().t()):
        for got, want in ((MXDenseBMMCUDA()(X, Q), MXDenseBMMCUDA()(X, clean)),
                          (MXDenseBMMCUDA()(Q.mT, X.t()).t(), MXDenseBMMCUDA()(clean.mT, X.t()).t())):
            assert bool(torch.isnan(got[:, columns]).all())
            assert torch.equal(got[:, ~columns], want[:, ~columns]) and not bool(torch.isnan(want).any())
