"""Microscaled operators without a GPU: the plain forms against each other, the C entries' sizes and
refusals (all of them before any CUDA call), the wrappers' refusals of host tensors."""
import math

import pytest
import torch

from custom_matmul_kernels_b200 import CheckpointBMMCUDA, MXBMMCUDA, MXDenseBMMCUDA, MXQuantizeCUDA, MXTensor
from custom_matmul_kernels_b200 import custom_kernel as ck
from oracle import mx_semantics as S

OK_PTR = 1 << 20  # aligned, never read: every call below is refused first


@pytest.mark.parametrize("bits,grid", [(4, S.E2M1), (8, S.E4M3)])
def test_plain_rounding_is_nearest_even(bits, grid):
    """The vector form of the oracle against a search, at grid points, midpoints and between."""
    ys = []
    for a, b in zip(grid, grid[1:]):
        ys += [a, (a + b) / 2, (a + b) / 2 * (1 - 1e-6), (a + b) / 2 * (1 + 1e-6)]
    ys += [grid[-1], grid[-1] * 1.01]
    top = grid[-1] if bits == 8 else 4.0  # a block whose scale is 1
    for i in range(0, len(ys), 31):
        part = ys[i:i + 31]
        X = torch.tensor(part + [top] + [0.0] * (31 - len(part)), dtype=torch.float32)[None]
        e = S.block_exponent(float(X.max()), bits, torch.float32)
        codes, scales = S.quantize(X, bits)
        assert int(scales) == e + 127
        want = [S.nearest_code(float(x) * 2.0 ** -e, grid) for x in X[0]]
        assert codes[0].tolist() == want


def test_plain_scale_rules():
    for t in (torch.float32, torch.bfloat16, torch.float16):
        for amax in (1.0, 1.75, 1.7578125, 1.9921875, 3.0, 6.0, 7.0, 448.0, 449.0, 0.0078125):
            e4, e8 = S.block_exponent(amax, 4, t), S.block_exponent(amax, 8, t)
            assert 4 * 2.0 ** e4 <= amax < 8 * 2.0 ** e4
            assert amax <= 448 * 2.0 ** e8 and (e8 == S.LOW8[t] or amax > 448 * 2.0 ** (e8 - 1))
    assert S.block_exponent(0.0, 4, torch.float32) == -127


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_kept_values_are_values_of_the_source_type(dtype):
    """8 bits: element * scale is exact in the source's type, over its whole range."""
    fi = torch.finfo(dtype)
    X = torch.logspace(math.log2(fi.smallest_normal * fi.eps), math.log2(fi.max), 992, base=2.0, dtype=torch.float64)
    X = X.clamp(max=fi.max).to(dtype).view(31, 32)
    v = S.values(*S.quantize(X, 8), 8)
    assert bool(torch.isfinite(v).all()) and torch.equal(v.to(dtype).double(), v)


def test_pack_places():
    codes = torch.arange(130 * 160).view(130, 160) % 16
    scales = torch.arange(130 * 5).view(130, 5) % 200
    c, s = S.pack(codes, scales, 4)
    assert c.shape == (130, 80) and s.shape == (2, 2, 512)
    assert int(c[7, 3]) == int(codes[7, 6]) + 16 * int(codes[7, 7])
    for r, b in ((0, 0), (31, 3), (32, 0), (127, 4), (128, 1), (129, 4)):
        assert int(s[r // 128, b // 4, r % 32 * 16 + r % 128 // 32 * 4 + b % 4]) == int(scales[r, b])


def test_sizes(lib):
    assert lib.fbmm_mx_codes_bytes(2, 5, 33, 4) == 2 * 5 * 32
    assert lib.fbmm_mx_codes_bytes(2, 5, 33, 8) == 2 * 5 * 64
    assert lib.fbmm_mx_codes_bytes(1, 5, 33, 5) == 0 and lib.fbmm_mx_codes_bytes(1, 0, 33, 4) == 0
    assert lib.fbmm_mx_scales_bytes(2, 129, 129) == 2 * 2 * 2 * 512
    assert lib.fbmm_mx_scales_bytes(1, 1, 1) == 512 and lib.fbmm_mx_scales_bytes(0, 1, 1) == 0
    n, t = ord("n"), ord("t")
    need = lib.fbmm_mx4_bmm_tensor_workspace_bytes
    assert need(1, 1, 4096, 4096, n) == 0                      # quantised inside the product
    assert need(1, 1, 4096, 4096, t) == 2048 + 32 * 512        # not from the other layout
    assert need(2, 300, 64, 100, n) == (2 * 300 * 64 + 255) // 256 * 256 + 2 * 3 * 512
    assert need(1, 1, 64, 1 << 20, n) > 0                      # its rows would not fit beside the ring
    assert need(1, 0, 64, 64, n) == 0


def _quantize(lib, X=OK_PTR, dtype=0, layout=ord("n"), ld=64, bits=4, codes=OK_PTR, scales=OK_PTR, l=1, rows=8, k=64, step=512):
    return lib.fbmm_mx_quantize(None, X, dtype, layout, ld, step, bits, codes, scales, l, rows, k)


def test_quantize_refusals(lib):
    for kw in ({"X": None}, {"dtype": 3}, {"layout": ord("x")}, {"ld": 63}, {"bits": 6}, {"codes": None}, {"scales": None},
               {"l": 0}, {"rows": -1}, {"k": 0}, {"layout": ord("t"), "ld": 7}, {"l": 2, "step": -1}, {"k": (1 << 29) + 1, "ld": 1 << 30}):
        assert _quantize(lib, **kw) == ck.FBMM_ERR_INVALID, kw
    for kw in ({"X": OK_PTR + 2}, {"codes": OK_PTR + 8}, {"scales": OK_PTR + 1}):
        assert _quantize(lib, **kw) == ck.FBMM_ERR_ALIGN, kw
    assert _quantize(lib, X=OK_PTR + 1, dtype=1) == ck.FBMM_ERR_ALIGN


def _dequantize(lib, codes=OK_PTR, sc=256, scales=OK_PTR, ss=512, bits=4, out=OK_PTR, dtype=0, ldo=64, so=512, l=1, rows=8, k=64):
    return lib.fbmm_mx_dequantize(None, codes, sc, scales, ss, bits, out, dtype, ldo, so, l, rows, k)


def test_dequantize_refusals(lib):
    for kw in ({"codes": None}, {"scales": None}, {"bits": 16}, {"out": None}, {"dtype": -1}, {"ldo": 63}, {"l": 2, "so": 511},
               {"rows": 0}):
        assert _dequantize(lib, **kw) == ck.FBMM_ERR_INVALID, kw
    for kw in ({"codes": OK_PTR + 4}, {"out": OK_PTR + 2}, {"l": 2, "sc": 257}, {"l": 2, "ss": -16}):
        assert _dequantize(lib, **kw) == ck.FBMM_ERR_ALIGN, kw


def _product(lib, a=OK_PTR, sa=256, a_s=OK_PTR, sas=512, b=OK_PTR, sb=256, bs=OK_PTR, sbs=512, C=OK_PTR, dtype=0, ldc=8, sc=64,
             l=1, m=8, n=8, k=64):
    return lib.fbmm_mx4_bmm(None, a, sa, a_s, sas, b, sb, bs, sbs, C, dtype, ldc, sc, l, m, n, k)


def test_product_refusals(lib):
    for kw in ({"a": None}, {"bs": None}, {"C": None}, {"dtype": 4}, {"ldc": 7}, {"l": 2, "sc": 63}, {"m": 0}, {"n": -3}, {"k": 0},
               {"m": 0x7fffffff}):
        assert _product(lib, **kw) == ck.FBMM_ERR_INVALID, kw
    for kw in ({"b": OK_PTR + 1}, {"a_s": OK_PTR + 8}, {"C": OK_PTR + 2}, {"l": 2, "sa": 8}, {"l": 2, "sbs": -512}):
        assert _product(lib, **kw) == ck.FBMM_ERR_ALIGN, kw
    args = [None, OK_PTR, 0, ord("n"), 64, 64 * 300, OK_PTR, 256, OK_PTR, 512, OK_PTR, 0, 8, 2400, 1, 300, 8, 64]
    assert lib.fbmm_mx4_bmm_tensor(*args, None, 0) == ck.FBMM_ERR_WORKSPACE
    assert lib.fbmm_mx4_bmm_tensor(*args, OK_PTR, 100) == ck.FBMM_ERR_WORKSPACE
    args[1] = None
    assert lib.fbmm_mx4_bmm_tensor(*args, OK_PTR, 1 << 30) == ck.FBMM_ERR_INVALID


def test_dense_refusals(lib):
    n, t = ord("n"), ord("t")

    def dense(A=OK_PTR, la=n, lda=64, sa=512, B=OK_PTR, lb=n, ldb=8, sb=512, dtype=2, C=OK_PTR, ldc=8, sc=64, l=1, m=8, nn=8, k=64,
              ws=None, size=0):
        return lib.fbmm_dense_bmm_x16(None, A, la, lda, sa, B, lb, ldb, sb, dtype, C, ldc, sc, l, m, nn, k, ws, size)

    for kw in ({"A": None}, {"la": 0}, {"lda": 56}, {"lb": t, "ldb": 56}, {"dtype": 0}, {"C": None}, {"ldc": 7}, {"l": 2, "sc": 10},
               {"k": 0}, {"la": t, "lda": 0}):
        assert dense(**kw) == ck.FBMM_ERR_INVALID, kw
    assert dense(l=2, sa=-8) == ck.FBMM_ERR_INVALID
    for kw in ({"A": OK_PTR + 1}, {"C": OK_PTR + 1}, {"ws": OK_PTR + 8, "size": 1 << 20}):
        assert dense(**kw) == ck.FBMM_ERR_ALIGN, kw
    # storage that needs repacking: refused without a workspace, or with one that is too small
    for kw, bytes_ in (({"A": OK_PTR + 8}, 8 * 64 * 2), ({"lda": 65}, 8 * 64 * 2), ({"l": 2, "sb": 4}, 2 * 64 * 8 * 2)):
        assert dense(**kw) == ck.FBMM_ERR_ALIGN, kw
        assert dense(ws=OK_PTR, size=bytes_ - 1, **kw) == ck.FBMM_ERR_WORKSPACE, kw
    assert lib.fbmm_x16_repack_bytes(OK_PTR, 64, 512, 2, 8, 60) == 0
    assert lib.fbmm_x16_repack_bytes(OK_PTR, 61, 488, 2, 8, 60) == 2 * 8 * 64 * 2
    assert lib.fbmm_x16_repack_bytes(OK_PTR, 61, 0, 2, 8, 60) == 8 * 64 * 2  # one matrix for every batch
    assert lib.fbmm_x16_repack_bytes(OK_PTR, 64, 4, 1, 8, 60) == 0 and lib.fbmm_x16_repack_bytes(OK_PTR, 64, 4, 0, 8, 60) == 0
    rc = lib.fbmm_dense_mx_bmm_x16(None, OK_PTR, n, 64, 512, 2, OK_PTR, 256, OK_PTR, 512, 3, OK_PTR, 8, 64, 1, 8, 8, 64, None, 0)
    assert rc == ck.FBMM_ERR_INVALID and b"bits" in lib.fbmm_last_error()
    rc = lib.fbmm_dense_mx_bmm_x16(None, OK_PTR, n, 64, 512, 2, OK_PTR + 8, 256, OK_PTR, 512, 4, OK_PTR, 8, 64, 1, 8, 8, 64, None, 0)
    assert rc == ck.FBMM_ERR_ALIGN
    rc = lib.fbmm_mx_dense_bmm_x16(None, None, 256, OK_PTR, 512, 8, OK_PTR, 8, 64, 1, OK_PTR, 8, 64, 1, 8, 8, 64, None, 0)
    assert rc == ck.FBMM_ERR_INVALID


def test_wrappers_refuse_host_tensors(lib):
    X = torch.zeros(2, 4, 64)
    codes, scales = torch.zeros(2, 4, 32, dtype=torch.uint8), torch.zeros(2, 1, 1, 512, dtype=torch.uint8)
    with pytest.raises(ValueError, match="CUDA"):
        MXQuantizeCUDA(4)(X)
    with pytest.raises(ValueError, match="CUDA"):
        MXTensor(codes, scales, k=64)
    with pytest.raises(ValueError, match="CUDA"):
        CheckpointBMMCUDA()(X.requires_grad_(), X.transpose(1, 2))
    with pytest.raises(TypeError):
        MXBMMCUDA()(X, X)
    with pytest.raises(TypeError):
        MXDenseBMMCUDA()(X, X)
    with pytest.raises(ValueError, match="bits"):
        MXQuantizeCUDA(5)
    with pytest.raises(TypeError):
        MXBMMCUDA(out_dtype=torch.float64)
