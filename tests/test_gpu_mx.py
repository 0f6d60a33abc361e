"""Microscaled operators on the GPU against their plain 64-bit forms.

Tolerances count roundings. A result type rounds once: half a step, eps / 2 relative. The fp32 sums
of a product of K terms are off by at most K * 2^-23 of the sum of the terms' magnitudes (every
addition may truncate at one step, 2^-23, of a partial sum, which that sum bounds)."""
import pytest
import torch

from custom_matmul_kernels_b200 import (BMMCUDA, CheckpointBMMCUDA, MXBMMCUDA, MXDenseBMMCUDA, MXQuantizeCUDA, MXTensor)
from oracle import mx_semantics as S

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def rnd(shape, seed, dtype=F32, spread=1.5):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * torch.exp(spread * torch.randn(shape[:-1] + (1,), generator=g))
    return x.to(dtype)


def stored(X, bits):
    """Oracle storage of X [l, rows, k]."""
    out = [S.pack(*S.quantize(x, bits), bits) for x in X]
    return torch.stack([o[0] for o in out]), torch.stack([o[1] for o in out])


def as_mx(rows, k, bits, seed, dev, l=1, dim=-1, **kw):
    parts = [S.random_mx(rows, k, bits, seed + i, **kw) for i in range(l)]
    packed = [S.pack(c, s, bits) for c, s in parts]
    vals = torch.stack([S.values(c, s, bits) for c, s in parts])
    t = MXTensor(torch.stack([p[0] for p in packed]).to(dev), torch.stack([p[1] for p in packed]).to(dev), bits=bits, k=k,
                 dim=dim)
    return t, vals


def assert_sum_close(got, want, magnitude, K, dtype):
    """|got - want| <= rounding of the type + K * 2^-23 of the sum of magnitudes."""
    tol = want.abs() * (torch.finfo(dtype).eps / 2) + magnitude * (K * 2.0 ** -23) * (1 + torch.finfo(dtype).eps)
    tol = tol + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps  # half a step below the normal range
    err = (got.double().cpu() - want).abs()
    assert bool((err <= tol).all()), f"off by {float((err / tol).max()):.3g} tolerances"


# ---- quantisation -----------------------------------------------------------------------------
SHAPES = [(1, 1, 1), (1, 1, 31), (2, 3, 33), (1, 128, 128), (1, 129, 160), (3, 77, 257), (1, 200, 96), (2, 5, 1000)]


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("l,rows,k", SHAPES)
def test_quantize_storage(dev, l, rows, k, dtype, bits):
    X = rnd((l, rows, k), rows * 1000 + k, dtype)
    if rows > 2:
        X[0, 1] = 0
    codes, scales = stored(X, bits)
    q = MXQuantizeCUDA(bits)(X.to(dev))
    assert q.shape == (l, rows, k) and q.dim == -1
    assert torch.equal(q.codes.cpu(), codes) and torch.equal(q.scales.cpu(), scales)
    # along the other axis: the transposed matrix gives the same storage
    for Xt in (X.transpose(1, 2).contiguous().to(dev), X.to(dev).transpose(1, 2)):
        qt = MXQuantizeCUDA(bits)(Xt, dim=-2)
        assert qt.shape == (l, k, rows)
        assert torch.equal(qt.codes.cpu(), codes) and torch.equal(qt.scales.cpu(), scales)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_quantize_range_of_the_type(dev, dtype, bits):
    """Blocks at the ends of the type's range: subnormals, the largest values, signed zeros."""
    fi = torch.finfo(dtype)
    tiny = fi.smallest_normal * fi.eps
    rows = [[0.0] * 32, [-0.0] * 32, [tiny] * 32, [3 * tiny, -tiny] * 16, [fi.smallest_normal] * 32, [fi.max, -fi.max] * 16,
            [fi.max * (1 - fi.eps), 1.0] * 16, [fi.max / 2, tiny] * 16, [1.75, 448.0] * 16, [1.7500001, 449.0] * 16,
            [7.99, 6.0, 5.0, 2.5] * 8, [1.0, 0.25, 0.75, -1.25] * 8]
    X = torch.tensor(rows, dtype=torch.float64).clamp(-fi.max, fi.max).to(dtype)[None]
    codes, scales = stored(X, bits)
    q = MXQuantizeCUDA(bits)(X.to(dev))
    assert torch.equal(q.codes.cpu(), codes) and torch.equal(q.scales.cpu(), scales)
    want = S.values(*S.quantize(X[0], bits), bits)
    back = q.dequantize(F32)[0].cpu().double()
    assert torch.equal(back, want)
    if bits == 8:  # kept values are values of the source's type
        assert torch.equal(q.dequantize(dtype)[0].cpu().double(), want)


@pytest.mark.parametrize("bits", [4, 8])
def test_quantize_non_finite_blocks(dev, bits):
    X = torch.ones(4, 96)
    X[0, 5], X[1, 40], X[2, 70], X[2, 3] = float("nan"), float("inf"), float("-inf"), float("nan")
    back = MXQuantizeCUDA(bits)(X.to(dev)).dequantize().cpu()
    want = torch.ones(4, 96)
    want[0, :32] = want[1, 32:64] = want[2, 64:] = want[2, :32] = float("nan")
    assert torch.equal(torch.isnan(back), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(back), torch.nan_to_num(want))
    back = MXQuantizeCUDA(bits)(X.t().to(dev).contiguous(), dim=-2).dequantize().cpu().t()
    assert torch.equal(torch.isnan(back), torch.isnan(want))


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_quantize_strides(dev, dtype, bits):
    """Pitches, offsets and orders that vector loads cannot take."""
    base = rnd((3, 150, 301), 5, dtype).to(dev)
    for X in (base[:, :, 1:], base[:, 3:, :64], base[::2, :, :256], base[:, ::2], base[:, :, ::3], base[0], base[1, 7:8],
              base[:1].expand(4, -1, -1), base.permute(1, 0, 2), base[:, :, 5:6]):
        for dim in (-1, -2):
            q, w = MXQuantizeCUDA(bits)(X, dim=dim), MXQuantizeCUDA(bits)(X.contiguous().clone(), dim=dim)
            assert torch.equal(q.codes, w.codes) and torch.equal(q.scales, w.scales)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("l,rows,k", [(1, 1, 1), (2, 130, 100), (1, 40, 264)])
def test_dequantize(dev, l, rows, k, dtype, bits):
    q, v = as_mx(rows, k, bits, 3, dev, l)
    assert torch.equal(q.dequantize(dtype).cpu(), v.to(F32).to(dtype))  # the fp32 value is exact
    assert torch.equal(q.mT.dequantize(dtype).cpu(), v.transpose(1, 2).to(F32).to(dtype))


# ---- 4-bit product ------------------------------------------------------------------------------
PRODUCTS = [(1, 1, 1, 1), (1, 1, 129, 33), (2, 3, 5, 64), (1, 16, 200, 257), (1, 17, 128, 128), (3, 33, 70, 500),
            (1, 64, 130, 96), (1, 65, 1, 31), (2, 128, 128, 256), (1, 129, 257, 640), (1, 300, 400, 1111), (4, 100, 1, 300)]


@pytest.mark.parametrize("l,m,n,k", PRODUCTS)
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_product_of_microscaled(dev, l, m, n, k, dtype):
    A, a = as_mx(m, k, 4, 11, dev, l, lo=121, hi=125)
    B, b = as_mx(n, k, 4, 977, dev, l, dim=-2, lo=121, hi=125)
    C = MXBMMCUDA(out_dtype=dtype)(A, B)
    assert C.shape == (l, m, n) and C.dtype == dtype
    want = a @ b.transpose(1, 2)
    assert_sum_close(C, want, a.abs() @ b.abs().transpose(1, 2), k, dtype)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("l,m,n,k", [(1, 2300, 2500, 700), (2, 2048, 1536, 1280), (9, 1100, 300, 130)])
def test_product_many_tiles(dev, l, m, n, k, dtype):
    """Enough tiles for CTA pairs (256 x 256 tiles); the plain form runs in float64 on the GPU."""
    A, a = as_mx(m, k, 4, 11, dev, l, lo=121, hi=125)
    B, b = as_mx(n, k, 4, 977, dev, l, dim=-2, lo=121, hi=125)
    a, b = a.to(dev), b.to(dev)
    C = MXBMMCUDA(out_dtype=dtype)(A, B)
    assert_sum_close(C, (a @ b.transpose(1, 2)).cpu(), (a.abs() @ b.abs().transpose(1, 2)).cpu(), k, dtype)
    if l == 1:  # shared across batches, and a scale and a NaN block in every corner
        A3 = MXTensor(A.codes.expand(2, -1, -1), A.scales.expand(2, -1, -1, -1), k=k)
        B3 = MXTensor(B.codes.repeat(2, 1, 1), B.scales.repeat(2, 1, 1, 1), k=k, dim=-2)
        assert torch.equal(MXBMMCUDA(out_dtype=dtype)(A3, B3), C.expand(2, -1, -1))
        S2 = A.scales.clone()
        S2.view(-1)[-512 + (m - 1) % 32 * 16 + (m - 1) % 128 // 32 * 4] = 255
        C2 = MXBMMCUDA(out_dtype=dtype)(MXTensor(A.codes, S2, k=k), B)
        assert bool(torch.isnan(C2[0, -1]).all()) and torch.equal(C2[0, :-1], C[0, :-1])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("l,m,n,k", [(1, 65, 130, 2500), (1, 128, 256, 9000), (2, 200, 500, 1800), (1, 300, 900, 4100), (1, 129, 1, 520)])
def test_product_split_tiles(dev, l, m, n, k, dtype):
    """Few whole tiles: k split over clusters, several tiles of rows."""
    A, a = as_mx(m, k, 4, 11, dev, l, lo=121, hi=125)
    B, b = as_mx(n, k, 4, 977, dev, l, dim=-2, lo=121, hi=125)
    a, b = a.to(dev), b.to(dev)
    C = MXBMMCUDA(out_dtype=dtype)(A, B)
    assert_sum_close(C, (a @ b.transpose(1, 2)).cpu(), (a.abs() @ b.abs().transpose(1, 2)).cpu(), k, dtype)
    assert torch.equal(MXBMMCUDA(out_dtype=dtype)(A, B), C)


@pytest.mark.parametrize("m", [1, 16, 40, 200])
def test_product_exact_integers(dev, m):
    """Scales of one: every sum is a multiple of 1/4 below 2^22, so the result is exact."""
    A, a = as_mx(m, 2000, 4, 1, dev, lo=127, hi=128)
    B, b = as_mx(300, 2000, 4, 2, dev, dim=-2, lo=127, hi=128)
    assert torch.equal(MXBMMCUDA()(A, B).cpu().double(), a @ b.transpose(1, 2))


@pytest.mark.parametrize("m", [1, 30, 150])
def test_product_scales_place(dev, m):
    """One non-zero block per row, with a scale that names row and block: a scale that is
    read from another place shows."""
    n, k = 300, 1000
    nb = (k + 31) // 32
    ca, sa = torch.zeros((m, k), dtype=torch.int64), torch.zeros((m, nb), dtype=torch.int64)
    cb, sb = torch.zeros((n, k), dtype=torch.int64), torch.zeros((n, nb), dtype=torch.int64)
    for r in range(m):
        b = r % nb
        ca[r, 32 * b:32 * b + 1] = 2
        sa[r] = 110 + (torch.arange(nb) * 7 + r) % 17
    for r in range(n):
        cb[r] = 2
        sb[r] = 115 + (torch.arange(nb) * 5 + r * 3) % 13
    pa, pb = S.pack(ca, sa, 4), S.pack(cb, sb, 4)
    C = MXBMMCUDA()(MXTensor(pa[0].to(dev), pa[1].to(dev), k=k), MXTensor(pb[0].to(dev), pb[1].to(dev), k=k, dim=-2))
    assert torch.equal(C.cpu().double(), S.values(ca, sa, 4) @ S.values(cb, sb, 4).t())


def test_product_nan_blocks_stay_in_their_rows(dev):
    for m in (5, 150):
        ca, sa = S.random_mx(m, 600, 4, 1)
        cb, sb = S.random_mx(140, 600, 4, 2)
        sa[2, 18], sb[131, 0] = 255, 255
        pa, pb = S.pack(ca, sa, 4), S.pack(cb, sb, 4)
        C = MXBMMCUDA()(MXTensor(pa[0].to(dev), pa[1].to(dev), k=600), MXTensor(pb[0].to(dev), pb[1].to(dev), k=600, dim=-2))
        want = S.values(ca, sa, 4) @ S.values(cb, sb, 4).t()
        assert torch.equal(torch.isnan(C.cpu()), torch.isnan(want))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("l,m,n,k", [(1, 1, 300, 260), (1, 16, 130, 512), (2, 40, 140, 333), (1, 200, 260, 700)])
def test_product_of_a_tensor(dev, l, m, n, k, dtype):
    X = rnd((l, m, k), 31, dtype)
    B, b = as_mx(n, k, 4, 9, dev, l, dim=-2, lo=119, hi=123)
    a = torch.stack([S.values(*S.quantize(x, 4), 4) for x in X])
    want = a @ b.transpose(1, 2)
    C = MXBMMCUDA()(X.to(dev), B)
    assert C.dtype == dtype
    assert_sum_close(C, want, a.abs() @ b.abs().transpose(1, 2), k, dtype)
    if l == 1:
        B2 = MXTensor(B.codes[0], B.scales[0], k=k, dim=-2)
        assert torch.equal(MXBMMCUDA()(X[0].to(dev), B2), C[0])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("m", [1, 3, 16, 17, 64])
@pytest.mark.parametrize("l,n,k", [(1, 1, 1), (1, 130, 31), (1, 200, 256), (1, 100, 257), (2, 129, 2500), (1, 128, 9000), (40, 300, 600)])
def test_product_few_rows(dev, l, m, n, k, dtype):
    """One kernel for up to 64 rows: k split over clusters of 1 to 8 CTAs, ragged everywhere; the plain
    form takes the values that the quantiser (tested above) gives."""
    X = rnd((l, m, k), 31 + m, dtype).to(dev)
    if m > 2:
        X[0, 1] = 0
    B, b = as_mx(n, k, 4, 9, dev, l, dim=-2, lo=119, hi=123)
    a, b = MXQuantizeCUDA(4)(X).dequantize().double(), b.to(dev)
    want, mag = (a @ b.transpose(1, 2)).cpu(), (a.abs() @ b.abs().transpose(1, 2)).cpu()
    C = MXBMMCUDA()(X, B)
    assert_sum_close(C, want, mag, k, dtype)
    for _ in range(2):  # the order of the sums does not depend on timing
        assert torch.equal(MXBMMCUDA()(X, B), C)
    wide = torch.zeros((l, m, k + 3), dtype=dtype, device=dev)
    wide[:, :, 1:k + 1] = X
    assert torch.equal(MXBMMCUDA()(wide[:, :, 1:k + 1], B), C)  # rows at any alignment
    one = MXTensor(B.codes[:1].expand(l, -1, -1), B.scales[:1].expand(l, -1, -1, -1), k=k, dim=-2)
    assert torch.equal(MXBMMCUDA()(X, one)[0], C[0])
    A4 = MXQuantizeCUDA(4)(X)  # the same kernel on codes
    C4 = MXBMMCUDA(out_dtype=dtype)(A4, B)
    assert_sum_close(C4, want, mag, k, dtype)
    assert torch.equal(MXBMMCUDA(out_dtype=dtype)(A4, B), C4)
    if k > 64:  # the other layout goes through the workspace
        assert_sum_close(MXBMMCUDA()(X.transpose(1, 2).contiguous().transpose(1, 2), B), want, mag, k, dtype)


@pytest.mark.parametrize("m,n,k", [(1, 64, 1 << 18), (1, 40, 1 << 19), (9, 19000, 1100), (64, 19000, 520)])
def test_product_few_rows_long(dev, m, n, k):
    """A k of which no CTA can keep its rows beside the ring, and more tiles than SMs."""
    X = rnd((1, m, k), 3, BF16).to(dev)
    g = torch.Generator("cuda").manual_seed(1)
    W = MXQuantizeCUDA(4)(torch.randn((1, n, k), device=dev, generator=g, dtype=BF16)).mT
    a, b = MXQuantizeCUDA(4)(X).dequantize(), W.dequantize()
    want, mag = torch.zeros(1, m, n, dtype=torch.float64, device=dev), torch.zeros(1, m, n, dtype=torch.float64, device=dev)
    for i in range(0, k, 1 << 16):
        x, y = a[:, :, i:i + (1 << 16)].double(), b[:, i:i + (1 << 16)].double()
        want += x @ y
        mag += x.abs() @ y.abs()
    assert_sum_close(MXBMMCUDA()(X, W), want.cpu(), mag.cpu(), k, BF16)


def test_product_few_rows_non_finite(dev):
    """A row with an infinity or a NaN is NaN in its whole row and leaves the others alone."""
    X = rnd((1, 8, 3000), 3)
    B, b = as_mx(200, 3000, 4, 9, dev, dim=-2, lo=119, hi=123)
    clean = MXBMMCUDA()(X.to(dev), B)
    X[0, 2, 2999], X[0, 5, 0] = float("inf"), float("nan")
    C = MXBMMCUDA()(X.to(dev), B)
    assert bool(torch.isnan(C[0, [2, 5]]).all())
    keep = [0, 1, 3, 4, 6, 7]
    assert torch.equal(C[0, keep], clean[0, keep])


def test_product_shared_operands(dev):
    """Batch strides of 0 on either side give what copies give."""
    for m in (4, 150):
        A, _ = as_mx(m, 300, 4, 1, dev)
        B, _ = as_mx(260, 300, 4, 2, dev, 3, dim=-2)
        A3 = MXTensor(A.codes.expand(3, -1, -1), A.scales.expand(3, -1, -1, -1), k=300)
        Ac = MXTensor(A.codes.repeat(3, 1, 1), A.scales.repeat(3, 1, 1, 1), k=300)
        assert A3.codes.stride(0) == 0
        assert torch.equal(MXBMMCUDA()(A3, B), MXBMMCUDA()(Ac, B))
        assert torch.equal(MXBMMCUDA()(B.mT, A3.mT), MXBMMCUDA()(B.mT, Ac.mT))


def test_first_call_of_a_thread(dev):
    """A thread that has made no CUDA call yet (as the one of a backward pass) has no context for
    the tensor maps; shapes of its own, so that no cached map serves it."""
    import threading
    got = {}

    def work():
        W, w = as_mx(173, 231, 4, 5, dev, dim=-2, lo=120, hi=124)
        X = torch.ones(1, 19, 231, device=dev)
        got["mx"] = MXBMMCUDA()(X, W), torch.ones(1, 19, 231).double() @ w.transpose(1, 2)
        got["f32"] = BMMCUDA()(torch.ones(1, 37, 44, device=dev), torch.ones(1, 44, 76, device=dev)), torch.full((1, 37, 76), 44.0)

    t = threading.Thread(target=work)
    t.start()
    t.join()
    for g, w in got.values():
        assert torch.allclose(g.cpu().double(), w.double(), rtol=1e-4, atol=1e-4)
    assert len(got) == 2


def test_product_empty(dev):
    B, _ = as_mx(40, 64, 4, 1, dev, dim=-2)
    assert MXBMMCUDA()(torch.empty(1, 0, 64, device=dev), B).shape == (1, 0, 40)
    q = MXQuantizeCUDA(4)(torch.empty(0, 5, 64, device=dev))
    assert q.shape == (0, 5, 64) and q.dequantize().shape == (0, 5, 64)


# ---- gradients -----------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("l,m,j,c", [(1, 1, 1, 1), (1, 64, 64, 64), (2, 70, 130, 200), (1, 300, 129, 257), (3, 5, 1000, 33),
                                     (1, 257, 640, 300), (2, 1000, 200, 2600)])
@pytest.mark.parametrize("bits", [4, 8])
def test_dense_product(dev, l, m, j, c, dtype, bits):
    """One microscaled operand on either side, both layouts of the other."""
    P = rnd((l, m, j), 3, dtype, 0.3)  # a [l, m, j] tensor
    Q, q = as_mx(j, c, bits, 17, dev, l, lo=120, hi=124)
    want, mag = P.double() @ q, P.double().abs() @ q.abs()
    for X in (P.to(dev), P.transpose(1, 2).contiguous().to(dev).transpose(1, 2)):
        C = MXDenseBMMCUDA()(X, Q)
        assert C.shape == (l, m, c) and C.dtype == dtype
        assert_sum_close(C, want, mag, j, dtype)
        D = MXDenseBMMCUDA()(Q.mT, X.transpose(1, 2))
        assert D.shape == (l, c, m)
        assert_sum_close(D, want.transpose(1, 2), mag.transpose(1, 2), j, dtype)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("bits", [4, 8])
def test_dense_product_many_tiles(dev, dtype, bits):
    """Enough tiles for CTA pairs (256 x 256 tiles); the plain form runs in float64 on the GPU."""
    m, j, c = 2000, 200, 2300
    P = rnd((1, m, j), 3, dtype, 0.3).to(dev)
    Q, q = as_mx(j, c, bits, 17, dev, 1, lo=120, hi=124)
    q = q.to(dev)
    want, mag = P.double() @ q, P.double().abs() @ q.abs()
    for X in (P, P.transpose(1, 2).contiguous().transpose(1, 2)):
        assert_sum_close(MXDenseBMMCUDA()(X, Q), want.cpu(), mag.cpu(), j, dtype)
        assert_sum_close(MXDenseBMMCUDA()(Q.mT, X.transpose(1, 2)), want.transpose(1, 2).cpu(), mag.transpose(1, 2).cpu(),
                         j, dtype)
    if bits == 8:  # the dense products of a training step, in its three layouts
        for transposed in (False, True):
            A = rnd((1, 2100, 2050), 5, dtype, 0.3).to(dev).requires_grad_()
            B = rnd((1, 2050, 2310), 6, dtype, 0.3).to(dev)
            B = (B.transpose(1, 2).contiguous().transpose(1, 2) if transposed else B).detach().requires_grad_()
            dC = rnd((1, 2100, 2310), 7, dtype, 0.3).to(dev)
            C = CheckpointBMMCUDA()(A, B)
            dA, dB = torch.autograd.grad(C, (A, B), dC)
            a, b, d = A.detach().double(), B.detach().double(), dC.double()
            a8 = MXQuantizeCUDA(8)(A.detach()).dequantize().double()
            for got, x, y in ((C, a, b), (dA, d, b.transpose(1, 2)), (dB, a8.transpose(1, 2), d)):
                assert_sum_close(got.detach(), (x @ y).cpu(), (x.abs() @ y.abs()).cpu(), x.shape[2], dtype)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("l,m,j,c", [(7, 6, 86, 14244), (7, 23, 199, 5477), (3, 500, 70, 2900)])
def test_dense_product_short_sums(dev, l, m, j, c, bits):
    """Many tiles of one to four stages each: the expanding warps' groups overtake one another at every turn."""
    P = rnd((l, m, j), 3, BF16, 0.3).to(dev)
    Q = MXQuantizeCUDA(bits)(rnd((l, j, c), 4, BF16, 0.3).to(dev))
    q, p = Q.dequantize().double(), P.double()
    want, mag = (p @ q).cpu(), (p.abs() @ q.abs()).cpu()
    first = MXDenseBMMCUDA()(P, Q)
    assert_sum_close(first, want, mag, j, BF16)
    flipped = MXDenseBMMCUDA()(Q.mT, P.transpose(1, 2))
    assert_sum_close(flipped, want.transpose(1, 2), mag.transpose(1, 2), j, BF16)
    for _ in range(40):
        assert torch.equal(MXDenseBMMCUDA()(P, Q), first)
        assert torch.equal(MXDenseBMMCUDA()(Q.mT, P.transpose(1, 2)), flipped)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("l,m,j,c", [(1, 64, 5000, 130), (2, 200, 3001, 33), (1, 1, 9000, 700), (1, 129, 2600, 257)])
def test_dense_product_long_sums(dev, l, m, j, c, dtype):
    """Few tiles and a long sum: clusters share it; every layout, both widths, and the dense products."""
    P = rnd((l, m, j), 3, dtype, 0.3).to(dev)
    R = rnd((l, j, c), 4, dtype, 0.3).to(dev)
    p, r = P.double(), R.double()
    for bits in (4, 8):
        Q = MXQuantizeCUDA(bits)(R)
        q = Q.dequantize(dtype).double()
        want, mag = (p @ q).cpu(), (p.abs() @ q.abs()).cpu()
        for X in (P, P.transpose(1, 2).contiguous().transpose(1, 2)):
            C, D = MXDenseBMMCUDA()(X, Q), MXDenseBMMCUDA()(Q.mT, X.transpose(1, 2))
            assert_sum_close(C, want, mag, j, dtype)
            assert_sum_close(D, want.transpose(1, 2), mag.transpose(1, 2), j, dtype)
            assert torch.equal(MXDenseBMMCUDA()(X, Q), C)
    for X in (P, P.transpose(1, 2).contiguous().transpose(1, 2)):
        for Y in (R, R.transpose(1, 2).contiguous().transpose(1, 2)):
            C = CheckpointBMMCUDA()(X.requires_grad_(), Y)
            assert_sum_close(C.detach(), (p @ r).cpu(), (p.abs() @ r.abs()).cpu(), j, dtype)


@pytest.mark.parametrize("n", [1, 2, 3, 4, 6, 129, 130, 131, 132, 134, 136, 195, 196, 198, 257, 258, 260])
@pytest.mark.parametrize("l,m", [(1, 3), (1, 150), (3, 97), (1, 20001)])
def test_result_rows_at_every_alignment(dev, l, m, n):
    """Result rows 2, 4, 8 and 16 bytes apart from a line, in every kernel that writes them, and their last pieces."""
    k = 96
    A, B = rnd((l, m, k), 5, BF16).to(dev), rnd((l, k, n), 6, BF16).to(dev)
    A4, B4, B8 = MXQuantizeCUDA(4)(A), MXQuantizeCUDA(4)(B, dim=-2), MXQuantizeCUDA(8)(B)
    a, b = A4.dequantize(F32).double(), B4.dequantize(F32).double()
    want, mag = (a @ b).cpu(), (a.abs() @ b.abs()).cpu()
    for dtype in (F32, F16, BF16):
        C = MXBMMCUDA(out_dtype=dtype)(A4, B4).cpu()
        # fp16 ends at 65504: a sum of 65520 or more rounds to infinity (20001 x 3 has four: the largest is 80999)
        over = want.abs() >= 65520 if dtype == F16 else torch.zeros_like(want, dtype=torch.bool)
        assert torch.equal(C[over].double(), want[over].sign() * float("inf"))
        assert_sum_close(C.masked_fill(over, 0), want.masked_fill(over, 0), mag, k, dtype)
    a, b = A.double(), B8.dequantize(BF16).double()
    assert_sum_close(MXDenseBMMCUDA()(A, B8), (a @ b).cpu(), (a.abs() @ b.abs()).cpu(), k, BF16)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("l,m,n,k", [(1, 5, 40, 64), (2, 130, 200, 300)])
def test_frozen_weights_gradient(dev, l, m, n, k, dtype):
    W, w = as_mx(n, k, 4, 5, dev, l, dim=-2, lo=120, hi=124)
    X = rnd((l, m, k), 8, dtype, 0.5).to(dev).requires_grad_()
    dC = rnd((l, m, n), 9, dtype, 0.3)
    C = MXBMMCUDA()(X, W)
    assert torch.equal(C.detach(), MXBMMCUDA()(X.detach(), W))
    dX, = torch.autograd.grad(C, X, dC.to(dev))
    tol_k = n * (1 if dtype != F32 else 8)  # the fp32 product splits each term in three
    assert_sum_close(dX, dC.double() @ w, dC.double().abs() @ w.abs(), tol_k, dtype)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("l,m,n,k", [(1, 1, 1, 1), (1, 64, 96, 128), (2, 77, 130, 33), (1, 300, 257, 200), (1, 700, 530, 600)])
def test_checkpoint_gradients(dev, l, m, n, k, dtype):
    A, B, dC = rnd((l, m, k), 1, dtype, 0.5), rnd((l, k, n), 2, dtype, 0.2), rnd((l, m, n), 3, dtype, 0.2)
    a8 = torch.stack([S.values(*S.quantize(x, 8), 8) for x in A])
    Ad, Bd = A.to(dev).requires_grad_(), B.to(dev).requires_grad_()
    C = CheckpointBMMCUDA()(Ad, Bd)
    dA, dB = torch.autograd.grad(C, (Ad, Bd), dC.to(dev))
    f = 8 if dtype == F32 else 1  # the fp32 product splits each term in three
    a, b, d = A.double(), B.double(), dC.double()
    assert_sum_close(C.detach(), a @ b, a.abs() @ b.abs(), f * k, dtype)
    assert_sum_close(dA, d @ b.transpose(1, 2), d.abs() @ b.abs().transpose(1, 2), f * n, dtype)
    assert_sum_close(dB, a8.transpose(1, 2) @ d, a8.abs().transpose(1, 2) @ d.abs(), f * m, dtype)
    # B stored transposed (a weight [n, k] used as its own transpose)
    Wd = B.transpose(1, 2).contiguous().to(dev).requires_grad_()
    Ct = CheckpointBMMCUDA()(Ad, Wd.transpose(1, 2))
    dA2, dW = torch.autograd.grad(Ct, (Ad, Wd), dC.to(dev))
    assert_sum_close(Ct.detach(), a @ b, a.abs() @ b.abs(), f * k, dtype)
    assert_sum_close(dA2, d @ b.transpose(1, 2), d.abs() @ b.abs().transpose(1, 2), f * n, dtype)
    assert_sum_close(dW, d.transpose(1, 2) @ a8, d.abs().transpose(1, 2) @ a8.abs(), f * m, dtype)


def test_checkpoint_keeps_eight_bits(dev):
    """What waits for the backward pass: B, and A at 33/32 byte per element; released by it."""
    A = torch.randn(1, 512, 1024, device=dev, dtype=BF16).requires_grad_()
    B = torch.randn(1, 1024, 256, device=dev, dtype=BF16).requires_grad_()
    kept = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t) or t, lambda t: t):
        C = CheckpointBMMCUDA()(A, B)
    assert sum(t.numel() for t in kept if t.dtype == torch.uint8) == 512 * 1024 * 33 // 32
    assert [t.shape for t in kept if t.dtype != torch.uint8] == [B.shape]
    C.sum().backward()  # an expanded gradient
    with pytest.raises(RuntimeError, match="second time"):
        C.sum().backward()


@pytest.mark.parametrize("need", ["A", "B"])
def test_checkpoint_one_gradient(dev, need):
    A, B = rnd((2, 70, 96), 1, BF16, 0.5).to(dev), rnd((2, 96, 64), 2, BF16, 0.5).to(dev)
    both = [t.clone().requires_grad_() for t in (A, B)]
    want = torch.autograd.grad(CheckpointBMMCUDA()(*both).square().sum(), both)
    one = [A.clone().requires_grad_(need == "A"), B.clone().requires_grad_(need == "B")]
    C = CheckpointBMMCUDA()(*one)
    got, = torch.autograd.grad(C.square().sum(), [t for t in one if t.requires_grad])
    assert torch.equal(got, want[need == "B"])
    with torch.no_grad():
        assert not CheckpointBMMCUDA()(*both).requires_grad


def test_checkpoint_broadcast_and_2d(dev):
    """One B for every batch: its gradient is the sum over the batches; 2-D operands."""
    A, B = rnd((3, 40, 64), 1, BF16, 0.5).to(dev), rnd((64, 48), 2, BF16, 0.5).to(dev).requires_grad_()
    dC = rnd((3, 40, 48), 3, BF16, 0.5).to(dev)
    C = CheckpointBMMCUDA()(A, B.expand(3, -1, -1))
    dB, = torch.autograd.grad(C, B, dC)
    each = []
    for i in range(3):
        Ci = CheckpointBMMCUDA()(A[i], B)
        assert torch.equal(Ci, C[i])
        each.append(torch.autograd.grad(Ci, B, dC[i])[0])
    want = torch.stack(each).double().sum(0)
    # three results of half a step each, and the sum's own rounding
    tol = torch.stack(each).double().abs().sum(0) * torch.finfo(BF16).eps / 2 + want.abs() * torch.finfo(BF16).eps
    assert bool(((dB.double() - want).abs() <= tol + 1e-6).all())


@pytest.mark.parametrize("kind", ["checkpoint", "frozen"])
def test_gradient_by_differences(dev, kind):
    """L = sum(C * D) is linear in each operand, so (L(x + h) - L(x - h)) / 2h is its derivative; operands
    whose quantisation is exact (small integers in blocks with a 4 or a 448) and fp32 products."""
    g = torch.Generator().manual_seed(5)
    A = torch.randint(-2, 3, (1, 6, 64), generator=g).float()
    D = torch.randint(-3, 4, (1, 6, 40), generator=g).float()
    if kind == "checkpoint":
        B = torch.randint(-2, 3, (1, 64, 40), generator=g).float()
        Ad, Bd = A.to(dev).requires_grad_(), B.to(dev).requires_grad_()
        dA, dB = torch.autograd.grad((CheckpointBMMCUDA()(Ad, Bd) * D.to(dev)).sum(), (Ad, Bd))
        run = lambda a, b: float((CheckpointBMMCUDA()(a.to(dev), b.to(dev)).cpu() * D).double().sum())  # noqa: E731
        for i, j in ((0, 0), (3, 17), (5, 63)):
            h = torch.zeros_like(A)
            h[0, i, j] = 1.0
            assert (run(A + h, B) - run(A - h, B)) / 2 == float(dA[0, i, j])
        for i, j in ((0, 0), (31, 20), (63, 39)):
            h = torch.zeros_like(B)
            h[0, i, j] = 1.0
            assert (run(A, B + h) - run(A, B - h)) / 2 == float(dB[0, i, j])
    else:
        A[:, :, ::32] = 4.0  # every block's scale stays 1, and 0, 1, 2, 3 are elements
        W, _ = as_mx(40, 64, 4, 3, dev, dim=-2, lo=127, hi=128)
        Ad = A.to(dev).requires_grad_()
        dA, = torch.autograd.grad((MXBMMCUDA()(Ad, W) * D.to(dev)).sum(), Ad)
        run = lambda a: float((MXBMMCUDA()(a.to(dev), W).cpu() * D).double().sum())  # noqa: E731
        for i, j in ((0, 1), (3, 17), (5, 63)):
            h = torch.zeros_like(A)
            h[0, i, j] = 1.0
            assert (run(A + h) - run(A - h)) / 2 == float(dA[0, i, j])


def test_written_weights_are_noticed(dev):
    W, _ = as_mx(40, 64, 4, 3, dev, dim=-2)
    A = torch.randn(1, 4, 64, device=dev, requires_grad=True)
    C = MXBMMCUDA()(A, W)
    W.codes.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(C.sum(), A)


def test_higher_order_is_refused(dev):
    A = torch.randn(1, 4, 64, device=dev, requires_grad=True)
    B = torch.randn(1, 64, 8, device=dev, requires_grad=True)
    g, = torch.autograd.grad(CheckpointBMMCUDA()(A, B).square().sum(), A, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()


# ---- as they are used together ---------------------------------------------------------------------
def test_training_step_captured(dev):
    """Two projections, one over frozen 4-bit weights and one with its activations in 8 bits, forward
    and backward in one CUDA graph: replays follow the inputs, and equal the eager step bit for bit."""
    W = MXQuantizeCUDA(4)(rnd((1, 192, 256), 4, BF16, 0.2).to(dev), dim=-2)
    A, B = rnd((1, 300, 192), 1, BF16, 0.5).to(dev).requires_grad_(), rnd((1, 256, 128), 2, BF16, 0.2).to(dev).requires_grad_()
    dC = rnd((1, 300, 128), 3, BF16, 0.2).to(dev)

    def step(a, b):
        H = MXBMMCUDA()(a, W)
        C = CheckpointBMMCUDA()(H, b)
        return (C.detach(),) + torch.autograd.grad(C, (a, b), dC)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(A, B)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(A, B)
    for seed in (11, 12):
        with torch.no_grad():
            A.copy_(rnd((1, 300, 192), seed, BF16, 0.5))
            B.copy_(rnd((1, 256, 128), seed + 100, BF16, 0.2))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        want = step(A.detach().clone().requires_grad_(), B.detach().clone().requires_grad_())
        assert all(torch.equal(g, w) for g, w in zip(got, want))


def test_decoding_captured_on_another_stream(dev):
    """A decoding step (few rows, fused) and a longer product share weights on two streams and in two graphs."""
    W = MXQuantizeCUDA(4)(rnd((1, 512, 640), 4, BF16, 0.2).to(dev), dim=-2)
    x, y = rnd((1, 3, 512), 1, BF16).to(dev), rnd((1, 200, 512), 2, BF16).to(dev)
    want = MXBMMCUDA()(x, W), MXBMMCUDA()(y, W)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for t in (x, y, x, y):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(MXBMMCUDA()(t, W))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for i, o in enumerate(outs):
        assert torch.equal(o, want[i % 2])


@pytest.mark.parametrize("m", [3, 100, 2300])
def test_operands_written_right_before(dev, m):
    """Every operand is rewritten by the kernel ahead of the product, over and over; the products may start early, but
    read what is there when that kernel is done."""
    k, n = 512, 2304
    A, B = torch.zeros(1, m, k, device=dev, dtype=BF16), torch.zeros(1, k, n, device=dev, dtype=BF16)
    W = MXQuantizeCUDA(4)(torch.zeros(1, k, n, device=dev), dim=-2)
    one = MXQuantizeCUDA(4)(torch.ones(1, k, n, device=dev), dim=-2)
    along = MXQuantizeCUDA(4)(torch.ones(1, k, n, device=dev))
    big = torch.zeros(1 << 26, device=dev, dtype=torch.uint8)
    outs = []
    for i in range(24):
        big.zero_()
        if i % 3 == 0:
            A.fill_(i + 1.0)
            W.codes.copy_(one.codes)
            W.scales.copy_(one.scales)
        elif i % 3 == 1:
            W.scales.fill_(127 + i % 5)  # 4 * 2^(i % 5), the codes being those of 4 (ones scaled by 1/4)
        else:
            B.fill_(i + 1.0)
        outs.append((i, MXBMMCUDA()(A, W), MXBMMCUDA()(MXQuantizeCUDA(4)(A), W),
                     CheckpointBMMCUDA()(A.requires_grad_(), B).detach(), MXDenseBMMCUDA()(A.detach(), along)))
        A = A.detach()
    a, w, b = 0.0, 0.0, 0.0
    for i, y, z, c, d in outs:
        if i % 3 == 0:
            a, w = i + 1.0, 1.0
        elif i % 3 == 1:
            w = 4.0 * 2.0 ** (i % 5)
        else:
            b = i + 1.0
        # all elements of a row alike; A itself is rounded to 4 bits in y and z
        a4 = float(S.values(*S.quantize(torch.full((1, 32), a, dtype=BF16), 4), 4)[0, 0])
        assert float(y.min()) == float(y.max()) == float(torch.tensor(a4 * w * k).to(BF16)), i
        assert float(z.min()) == float(z.max()) == a4 * w * k, i
        assert float(c.min()) == float(c.max()) == float(torch.tensor(a * b * k).to(BF16)), i
        assert float(d.min()) == float(d.max()) == float(torch.tensor(a * k).to(BF16)), i


def test_offsets_past_32_bits(dev):
    """Sources, codes and results of more than 2^32 bytes, looked at where they end."""
    # quantised and back: 36000 x 131072, 4.7 GB of 8-bit codes, 9.4 GB on either side
    rows, k = 36000, 1 << 17
    X = torch.zeros((1, rows, k), device=dev, dtype=BF16)
    X[0, -200:] = rnd((200, k), 5, BF16).to(dev)
    q = MXQuantizeCUDA(8)(X)
    want = MXQuantizeCUDA(8)(X[:, -200:].clone()).dequantize(BF16)
    back = q.dequantize(BF16)
    assert q.codes.numel() > 1 << 32
    assert torch.equal(back[:, -200:], want) and not bool(back[:, -500:-200].any())
    # the weights' gradient over all of it: only the last rows count
    dC = torch.randn((1, rows, 64), device=dev, dtype=BF16)
    got = MXDenseBMMCUDA()(q.mT, dC)
    v, d = want.double().transpose(1, 2), dC[:, -200:].double()
    assert_sum_close(got, (v @ d).cpu(), (v.abs() @ d.abs()).cpu(), 200, BF16)
    del back, q, got, v
    # weights of 4.7 GB of 4-bit codes: few rows and many
    W = MXQuantizeCUDA(4)(X.expand(2, -1, -1).reshape(1, 2 * rows, k)).mT  # [1, k, 72000], both halves alike
    assert W.codes.numel() > 1 << 32
    del X
    torch.cuda.empty_cache()
    for m in (2, 130):
        A = torch.randn((1, m, k), device=dev, dtype=BF16)
        C = MXBMMCUDA()(A, W)
        assert torch.equal(C[:, :, rows - 200:rows], C[:, :, -200:]) and bool(C[:, :, -200:].any())
        assert not bool(C[:, :, rows:-200].any())
    del W, C
    torch.cuda.empty_cache()
    # a result of 2.6e9 elements
    m = n = 51000
    A, B = rnd((1, m, 64), 1, BF16).to(dev), rnd((1, n, 64), 2, BF16).to(dev)
    QA, QB = MXQuantizeCUDA(4)(A), MXQuantizeCUDA(4)(B).mT
    C = MXBMMCUDA(out_dtype=BF16)(QA, QB)
    tail = MXBMMCUDA(out_dtype=BF16)(MXQuantizeCUDA(4)(A[:, -300:].clone()), QB)
    assert torch.equal(C[:, -300:], tail)
    D = MXDenseBMMCUDA()(A, MXQuantizeCUDA(4)(B.transpose(1, 2).contiguous()))
    tail = MXDenseBMMCUDA()(A[:, -300:].clone(), MXQuantizeCUDA(4)(B.transpose(1, 2).contiguous()))
    assert torch.equal(D[:, -300:], tail)


def test_product_with_itself_and_slices(dev):
    X = rnd((4, 70, 96), 3, BF16).to(dev)
    q = MXQuantizeCUDA(4)(X)
    v = q.dequantize().double()
    for A, a in ((q, v), (MXTensor(q.codes[1:3], q.scales[1:3], k=96), v[1:3])):
        C = MXBMMCUDA()(A, A.mT)
        assert_sum_close(C, (a @ a.transpose(1, 2)).cpu(), (a.abs() @ a.abs().transpose(1, 2)).cpu(), 96, F32)


def test_library_reports_no_trouble(dev, lib):
    assert lib.fbmm_check(None) == 0, lib.fbmm_last_error()


# ---- refusals ----------------------------------------------------------------------------------------
def test_refusals(dev):
    X = torch.randn(2, 8, 64, device=dev)
    W = MXQuantizeCUDA(4)(torch.randn(2, 64, 16, device=dev), dim=-2)
    P = MXBMMCUDA()
    with pytest.raises(ValueError, match="batch sizes"):
        P(X[:1], W)
    with pytest.raises(ValueError, match="inner dimensions"):
        P(X[:, :, :32], W)
    with pytest.raises(ValueError, match="same number of dimensions"):
        P(X[0], W)
    with pytest.raises(ValueError, match="dim=-2"):
        P(X[:, :, :16], W.mT)
    with pytest.raises(ValueError, match="4-bit"):
        P(X, MXQuantizeCUDA(8)(torch.randn(2, 64, 16, device=dev), dim=-2))
    with pytest.raises(ValueError, match="A must hold"):
        P(MXQuantizeCUDA(8)(X), W)
    with pytest.raises(TypeError):
        P(X, torch.randn(2, 64, 16, device=dev))
    with pytest.raises(TypeError):
        P(X.double(), W)
    with pytest.raises(ValueError, match="CUDA"):
        P(X.cpu(), W)
    D = MXDenseBMMCUDA()
    with pytest.raises(TypeError):
        D(X.half(), X.half())
    with pytest.raises(TypeError):
        D(torch.randn(2, 8, 16, device=dev), W.mT)  # fp32
    with pytest.raises(ValueError, match="own axis"):
        D(X.half(), W)
    with pytest.raises(ValueError, match="2d or 3d"):
        MXQuantizeCUDA(4)(X[0, 0])
    with pytest.raises(ValueError, match="empty"):
        MXQuantizeCUDA(4)(X[:, :, :0])
    with pytest.raises(TypeError):
        MXQuantizeCUDA(4)(X.double())
    with pytest.raises(TypeError):
        W.dequantize(torch.float64)
    with pytest.raises(ValueError, match="what k"):
        MXTensor(W.codes, W.scales, k=65)
    with pytest.raises(ValueError, match="scales have shape"):
        MXTensor(W.codes, W.scales[:, :, :, :256], k=64)
    with pytest.raises(TypeError):
        MXTensor(W.codes.int(), W.scales, k=64)
    with pytest.raises(TypeError):
        CheckpointBMMCUDA()(X.double().requires_grad_(), X.double().transpose(1, 2))
    with pytest.raises(ValueError, match="inner dimensions"):
        CheckpointBMMCUDA()(X.requires_grad_(), X)


def test_unaligned_storage_is_copied(dev):
    """Codes and scales at odd addresses or batch strides give what aligned ones give."""
    B, _ = as_mx(40, 96, 4, 3, dev, 2, dim=-2)
    A = torch.randn(2, 5, 96, device=dev)
    want = MXBMMCUDA()(A, B)
    raw = torch.empty(B.codes.numel() + 1, dtype=torch.uint8, device=dev)
    raw[1:] = B.codes.reshape(-1)
    odd = MXTensor(raw[1:].view_as(B.codes), B.scales, k=96, dim=-2)
    assert torch.equal(MXBMMCUDA()(A, odd), want)
    wide = torch.zeros(2, 41, B.codes.shape[2] + 1, dtype=torch.uint8, device=dev)
    wide[:, :40, :-1] = B.codes
    assert torch.equal(MXBMMCUDA()(A, MXTensor(wide[:, :40, :-1], B.scales, k=96, dim=-2)), want)
