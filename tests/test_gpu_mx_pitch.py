"""The C entries with results and sources inside larger buffers: a pitch wider than a row, space between batches,
layout letters of either case. What lies between rows and batches stays as it was; the values are those of the
dense layout."""
import pytest
import torch

from custom_matmul_kernels_b200 import MXBMMCUDA, MXDenseBMMCUDA, MXQuantizeCUDA
from custom_matmul_kernels_b200 import mx

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
CODE = {F32: 0, F16: 1, BF16: 2}
MARK = 77.0


def rnd(shape, seed, dev, dtype):
    g = torch.Generator(dev).manual_seed(seed)
    return torch.randn(shape, device=dev, generator=g).to(dtype)


def frame(l, m, n, pad, gap, offset, dtype, dev):
    """(buffer, view [l, m, n] in it, pitch, batch stride): every element of the buffer is MARK."""
    ld = n + pad
    step = m * ld + gap
    buf = torch.full((offset + l * step + 64,), MARK, device=dev, dtype=dtype)
    return buf, buf.as_strided((l, m, n), (step, ld, 1), offset), ld, step


def assert_framed(buf, view, want):
    assert torch.equal(view, want)
    view.fill_(MARK)
    assert bool((buf == MARK).all())


@pytest.mark.parametrize("pad,gap,offset", [(0, 0, 0), (1, 3, 1), (2, 0, 2), (4, 8, 4), (8, 16, 8), (61, 5, 3)])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("l,m,n,k", [(2, 5, 70, 300), (1, 40, 200, 64), (2, 100, 130, 4000), (3, 300, 200, 96), (1, 2300, 2309, 70)])
def test_four_bit_product(dev, lib, l, m, n, k, dtype, pad, gap, offset):
    """Few rows (quantised inside, and codes), shared k, single tiles, CTA pairs."""
    A, W = rnd((l, m, k), 1, dev, dtype), MXQuantizeCUDA(4)(rnd((l, n, k), 2, dev, F32)).mT
    A4 = MXQuantizeCUDA(4)(A)
    buf, C, ld, step = frame(l, m, n, pad, gap, offset, dtype, dev)
    mx._call("fbmm_mx4_bmm", dev.index or 0, *A4._arguments(), *W._arguments(), C.data_ptr(), CODE[dtype], ld, step, l, m, n, k)
    assert_framed(buf, C, MXBMMCUDA(out_dtype=dtype)(A4, W))
    for letter, X, ldx in ((ord("N"), A, k), (ord("T"), A.transpose(1, 2).contiguous(), m)):
        need = lib.fbmm_mx4_bmm_tensor_workspace_bytes(l, m, n, k, letter)
        ws = torch.empty(max(need, 16), dtype=torch.uint8, device=dev)
        mx._call("fbmm_mx4_bmm_tensor", dev.index or 0, X.data_ptr(), CODE[dtype], letter, ldx, m * k, *W._arguments(), C.data_ptr(),
                 CODE[dtype], ld, step, l, m, n, k, ws.data_ptr(), need)
        wrapped = X if letter == ord("N") else X.transpose(1, 2)
        assert_framed(buf, C, MXBMMCUDA()(wrapped, W))


@pytest.mark.parametrize("pad,gap,offset", [(0, 0, 0), (1, 3, 1), (2, 0, 2), (4, 8, 4), (8, 16, 8), (61, 5, 3)])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("l,m,n,k", [(2, 5, 70, 300), (2, 100, 130, 4000), (3, 300, 200, 96), (1, 2300, 2309, 70)])
def test_dense_products(dev, l, m, n, k, dtype, pad, gap, offset):
    """Results and the dense operands framed alike; operands that have to be repacked among them."""
    A, B = rnd((l, m, k), 1, dev, dtype), rnd((l, k, n), 2, dev, dtype)
    QB, QA = MXQuantizeCUDA(8)(B), MXQuantizeCUDA(4)(A.transpose(1, 2).contiguous())  # QA.mT: [l, m, k], blocks along m
    _, a, lda, sa = frame(l, m, k, pad, gap, offset, dtype, dev)
    _, b, ldb, sb = frame(l, k, n, pad, gap, offset, dtype, dev)
    a.copy_(A), b.copy_(B)
    lib = mx.load_library()
    need_a, need_b = (lib.fbmm_x16_repack_bytes(x.data_ptr(), ld, s, l, rows, cols)
                      for x, ld, s, rows, cols in ((a, lda, sa, m, k), (b, ldb, sb, k, n)))
    ws = torch.empty(need_a + need_b + 16, dtype=torch.uint8, device=dev)
    buf, C, ld, step = frame(l, m, n, pad, gap, offset, dtype, dev)
    tail = C.data_ptr(), ld, step, l, m, n, k, ws.data_ptr()
    index = dev.index or 0
    mx._call("fbmm_dense_bmm_x16", index, a.data_ptr(), ord("N"), lda, sa, b.data_ptr(), ord("n"), ldb, sb, CODE[dtype], *tail,
             need_a + need_b)
    assert_framed(buf, C, mx._dense_bmm(A, B))
    mx._call("fbmm_dense_mx_bmm_x16", index, a.data_ptr(), ord("n"), lda, sa, CODE[dtype], *QB._arguments(), 8, *tail, need_a)
    assert_framed(buf, C, MXDenseBMMCUDA()(A, QB))
    mx._call("fbmm_mx_dense_bmm_x16", index, *QA._arguments(), 4, b.data_ptr(), ldb, sb, CODE[dtype], *tail, need_b)
    assert_framed(buf, C, MXDenseBMMCUDA()(QA.mT, B))


@pytest.mark.parametrize("pad,gap,offset", [(0, 0, 0), (1, 3, 1), (2, 0, 2), (4, 8, 4), (8, 16, 8), (61, 5, 3)])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("l,rows,k", [(2, 5, 33), (1, 130, 256), (3, 200, 301)])
def test_quantise_and_back(dev, l, rows, k, bits, dtype, pad, gap, offset):
    X = rnd((l, rows, k), 1, dev, dtype)
    want = MXQuantizeCUDA(bits)(X)
    index = dev.index or 0
    per, groups = want._sizes()
    for letter in "NTnt":
        shape = (l, rows, k) if letter in "Nn" else (l, k, rows)
        _, x, ld, step = frame(*shape, pad, gap, offset, dtype, dev)
        x.copy_(X if letter in "Nn" else X.transpose(1, 2))
        codes = torch.full((l * per + 64,), 0xa5, dtype=torch.uint8, device=dev)
        scales = torch.full((l * groups + 64,), 0xa5, dtype=torch.uint8, device=dev)
        mx._call("fbmm_mx_quantize", index, x.data_ptr(), CODE[dtype], ord(letter), ld, step, bits, codes.data_ptr(),
                 scales.data_ptr(), l, rows, k)
        assert torch.equal(codes[:-64], want.codes.reshape(-1)) and torch.equal(scales[:-64], want.scales.reshape(-1))
        assert bool((codes[-64:] == 0xa5).all()) and bool((scales[-64:] == 0xa5).all())
    buf, out, ld, step = frame(l, rows, k, pad, gap, offset, dtype, dev)
    mx._call("fbmm_mx_dequantize", index, *want._arguments(), bits, out.data_ptr(), CODE[dtype], ld, step, l, rows, k)
    assert_framed(buf, out, want.dequantize(dtype))
