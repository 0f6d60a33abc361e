"""Microscaled operands: 4- and 8-bit elements with a power-of-two scale per block of 32, products
that read them, and a training product that keeps its activations in 8 bits.

The reference stops at fp32 (its kernels take float* only, kernels/bmm.cu:185); these are the
narrow forms of the same batched product.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from .bmm import BMMCUDA
from .custom_kernel import FBMM_BF16, FBMM_F16, FBMM_F32, CustomKernel, check

_DTYPES = {torch.float32: FBMM_F32, torch.float16: FBMM_F16, torch.bfloat16: FBMM_BF16}
_X16 = (torch.float16, torch.bfloat16)
BLOCK = 32


def _code(dtype: torch.dtype) -> int:
    code = _DTYPES.get(dtype)
    if code is None:
        raise TypeError(f"dtype {dtype} is not one of float32, float16, bfloat16")
    return code


class MXTensor:
    """A [l, r, c] (or [r, c]) matrix held as microscaled elements.

    ``codes`` uint8 [l, rows, ceil(k / 32) * 32 * bits / 8] and ``scales`` uint8
    [l, ceil(rows / 128), ceil(k / 128), 512] as ``include/fbmm.h`` lays them out; k is the extent
    of the axis the blocks run along, ``dim``: -1 (the matrix is [l, rows, k]) or -2 (it is
    [l, k, rows], held k-contiguous all the same). A batch stride of 0 (an expanded tensor)
    serves every batch with one matrix. 2-D codes with 3-D scales make a 2-D matrix."""

    __slots__ = ("codes", "scales", "bits", "k", "dim", "two_d")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, bits: int = 4, k: int | None = None, dim: int = -1):
        if bits not in (4, 8):
            raise ValueError("bits must be 4 or 8")
        if dim not in (-1, -2):
            raise ValueError("dim must be -1 or -2")
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
            raise TypeError("codes and scales must be uint8")
        two_d = codes.dim() == 2
        if codes.dim() not in (2, 3) or scales.dim() != codes.dim() + 1:
            raise ValueError("codes must be 2d or 3d and scales one dimension more")
        if codes.device.type != "cuda" or scales.device != codes.device:
            raise ValueError("codes and scales must be CUDA tensors on one device")
        if two_d:
            codes, scales = codes[None], scales[None]
        l, rows, pitch = codes.shape
        if k is None:
            k = pitch * 8 // bits
        blocks = (k + BLOCK - 1) // BLOCK
        if k <= 0 or pitch != blocks * (4 * bits):
            raise ValueError(f"codes have {pitch} bytes per row, which is not what k = {k} takes at {bits} bits")
        want = (l, (rows + 127) // 128, (blocks + 3) // 4, 512)
        if tuple(scales.shape) != want:
            raise ValueError(f"scales have shape {tuple(scales.shape)}, expected {want}")
        self.codes = self._addressable(codes)
        self.scales = self._addressable(scales)
        self.bits, self.k, self.dim, self.two_d = bits, k, dim, two_d

    @staticmethod
    def _addressable(t: torch.Tensor) -> torch.Tensor:
        # dense within a batch, batches a multiple of 16 bytes apart (or one for all), 16-byte base
        if t.numel() == 0:
            return t
        if t[0].is_contiguous() and t.data_ptr() % 16 == 0 and (t.shape[0] == 1 or t.stride(0) % 16 == 0):
            return t
        return t.clone(memory_format=torch.contiguous_format)

    @property
    def device(self) -> torch.device:
        return self.codes.device

    @property
    def rows(self) -> int:
        return self.codes.shape[1]

    @property
    def shape(self) -> tuple:
        l, rows = self.codes.shape[:2]
        s = (rows, self.k) if self.dim == -1 else (self.k, rows)
        return s if self.two_d else (l,) + s

    @property
    def mT(self) -> "MXTensor":
        """The transposed matrix: the same storage with the blocks along the other axis."""
        return self._with(-3 - self.dim)

    def _with(self, dim: int) -> "MXTensor":
        t = object.__new__(MXTensor)
        t.codes, t.scales, t.bits, t.k, t.dim, t.two_d = self.codes, self.scales, self.bits, self.k, dim, self.two_d
        return t

    def _strides(self):
        """Batch strides of codes and scales in bytes (0: one matrix for every batch)."""
        return self.codes.stride(0), self.scales.stride(0)

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """Element times scale, rounded once to `dtype`; with dim=-2 a transposed view of
        k-contiguous storage."""
        return MXQuantizeCUDA(self.bits).dequantize(self, dtype)

    def __repr__(self) -> str:
        return f"MXTensor(shape={self.shape}, bits={self.bits}, dim={self.dim}, device={self.device})"


class MXQuantizeCUDA(CustomKernel):
    """``MXQuantizeCUDA(bits)(X, dim) -> MXTensor``: X [l, r, c] or [r, c], fp32 / fp16 / bf16, as
    4-bit (e2m1) or 8-bit (e4m3) elements with one power-of-two scale per 32 elements along
    `dim` (-1 or -2).

    4 bits: the scale is 2^(floor(log2 a) - 2) of the block's largest magnitude a; elements above
    six scales saturate. 8 bits: the least power of two that keeps a within 448 scales, bounded so
    that every element times its scale is a value of X's type. Elements round to nearest, ties to
    even. A block that holds an infinity or a NaN reads back as NaN throughout. The result is for
    ``MXBMMCUDA`` when quantised along the axis that the product sums over. No gradient flows
    through this call."""

    def __init__(self, bits: int = 4):
        super().__init__()
        if bits not in (4, 8):
            raise ValueError("bits must be 4 or 8")
        self.bits = bits

    def __call__(self, X: torch.Tensor, dim: int = -1) -> MXTensor:
        if dim not in (-1, -2):
            raise ValueError("dim must be -1 or -2")
        two_d = X.dim() == 2
        if X.dim() not in (2, 3):
            raise ValueError("X needs to be 2d or 3d")
        dtype = _code(X.dtype)
        if X.device.type != "cuda":
            raise ValueError("X must be a CUDA tensor")
        X3 = X[None] if two_d else X
        if dim == -2:
            X3 = X3.transpose(1, 2)  # [l, rows, k] whichever axis the blocks run along
        l, rows, k = X3.shape
        if k == 0:
            raise ValueError("the axis the blocks run along is empty")
        pitch = (k + BLOCK - 1) // BLOCK * (4 * self.bits)
        q = object.__new__(MXTensor)
        q.codes = torch.empty((l, rows, pitch), dtype=torch.uint8, device=X.device)
        q.scales = torch.empty((l, (rows + 127) // 128, (k + 127) // 128, 512), dtype=torch.uint8, device=X.device)
        q.bits, q.k, q.dim, q.two_d = self.bits, k, dim, two_d
        if l == 0 or rows == 0:
            return q
        sl, sr, sk = X3.stride()
        if sk == 1 and (sr >= k or rows == 1):
            layout, ld = ord("n"), max(sr, k)
        elif sr == 1 and (sk >= rows or k == 1):
            layout, ld = ord("t"), max(sk, rows)
        else:
            X3 = X3.contiguous()
            sl, layout, ld = rows * k, ord("n"), k
        with torch.cuda.device(X.device):
            check(self.lib.fbmm_mx_quantize(self.stream_ptr(X.device), X3.data_ptr(), dtype, layout, ld, sl, self.bits,
                                            q.codes.data_ptr(), q.scales.data_ptr(), l, rows, k))
        return q

    def dequantize(self, q: MXTensor, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        code = _code(dtype)
        l, rows = q.codes.shape[:2]
        out = torch.empty((l, rows, q.k), dtype=dtype, device=q.device)
        if out.numel():
            sc, ss = q._strides()
            with torch.cuda.device(q.device):
                check(self.lib.fbmm_mx_dequantize(self.stream_ptr(q.device), q.codes.data_ptr(), sc, q.scales.data_ptr(),
                                                  ss, q.bits, out.data_ptr(), code, q.k, rows * q.k, l, rows, q.k))
        if q.dim == -2:
            out = out.transpose(1, 2)
        return out[0] if q.two_d else out


def _check_product(a_shape, b_shape, a_device, b_device):
    if len(a_shape) != len(b_shape):
        raise ValueError("A and B need the same number of dimensions")
    if len(a_shape) == 3 and a_shape[0] != b_shape[0]:
        raise ValueError(f"batch sizes differ: {a_shape[0]} vs {b_shape[0]}")
    if a_shape[-1] != b_shape[-2]:
        raise ValueError(f"inner dimensions differ: A {tuple(a_shape)} B {tuple(b_shape)}")
    if a_device != b_device:
        raise ValueError("A and B must be on the same device")


class MXDenseBMMCUDA(CustomKernel):
    """``MXDenseBMMCUDA()(P, Q) -> C``: fp16 / bf16 P [l, m, j] times a microscaled Q [l, j, c] whose
    blocks run along c (``dim=-1``), C in P's type. Q's elements times their scales enter as values of
    P's type, which is exact for bf16 and, for fp16, wherever they are fp16 values. This is the
    product of both backward passes below: the gradient of activations through 4-bit weights, and
    of weights from activations kept in 8 bits."""

    def __call__(self, P: torch.Tensor, Q: MXTensor) -> torch.Tensor:
        if not isinstance(Q, MXTensor):
            raise TypeError("Q must be an MXTensor")
        if P.dtype not in _X16:
            raise TypeError(f"dtype {P.dtype} is not one of float16, bfloat16")
        if P.dim() not in (2, 3):
            raise ValueError("P needs to be 2d or 3d")
        if P.device.type != "cuda":
            raise ValueError("P must be a CUDA tensor")
        _check_product(P.shape, Q.shape, P.device, Q.device)
        if Q.dim != -1:
            raise ValueError("Q's blocks must run along its last axis (dim=-1)")
        return BMMCUDA()(P, Q.dequantize(P.dtype))


class _MXProduct(torch.autograd.Function):
    """C = Q4(A) @ W, differentiable in A: straight through the rounding, dA = dC @ W^T."""

    @staticmethod
    def forward(ctx, A, W, out_dtype):
        ctx.W, ctx.dtype = W, A.dtype
        ctx.save_for_backward(W.codes, W.scales)
        return _mx_product(MXQuantizeCUDA(4)(A), W, out_dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, dC):
        ctx.saved_tensors  # raises if the weights were written to since the forward pass
        W = ctx.W.mT
        if ctx.dtype in _X16:
            return MXDenseBMMCUDA()(dC.to(ctx.dtype), W), None, None
        return BMMCUDA()(dC.to(ctx.dtype), W.dequantize(ctx.dtype)), None, None


def _mx_product(A: MXTensor, B: MXTensor, out_dtype: torch.dtype) -> torch.Tensor:
    kernel = CustomKernel()
    l, m, _ = A.codes.shape
    n = B.rows
    C = torch.empty((l, m, n), dtype=out_dtype, device=A.device)
    if C.numel():
        sa, sas = A._strides()
        sb, sbs = B._strides()
        with torch.cuda.device(A.device):
            check(kernel.lib.fbmm_mx4_bmm(
                kernel.stream_ptr(A.device), A.codes.data_ptr(), sa, A.scales.data_ptr(), sas, B.codes.data_ptr(), sb,
                B.scales.data_ptr(), sbs, C.data_ptr(), _code(out_dtype), n, m * n, l, m, n, A.k))
    return C[0] if A.two_d else C


class MXBMMCUDA(CustomKernel):
    """``MXBMMCUDA(out_dtype)(A, B) -> C``: A [l, m, k] times B [l, k, n], both with 4-bit elements
    (``MXTensor``, blocks along k: ``dim=-1`` for A, ``dim=-2`` for B). A may be a fp32 / fp16 /
    bf16 tensor, which is quantised first; C then has its type unless `out_dtype` says
    otherwise, and is differentiable in A (the gradient passes straight through A's rounding:
    dA = dC @ B^T with B's values). With a microscaled A, C is fp32 unless `out_dtype` says
    otherwise. Products and scales are exact, sums are kept in fp32, C is rounded once."""

    def __init__(self, out_dtype: torch.dtype | None = None):
        super().__init__()
        if out_dtype is not None:
            _code(out_dtype)
        self.out_dtype = out_dtype

    def __call__(self, A, B: MXTensor) -> torch.Tensor:
        if not isinstance(B, MXTensor):
            raise TypeError("B must be an MXTensor")
        _check_product(A.shape, B.shape, A.device, B.device)
        if B.bits != 4 or B.dim != -2:
            raise ValueError("B must hold 4-bit elements with their blocks along k (dim=-2)")
        if isinstance(A, MXTensor):
            if A.bits != 4 or A.dim != -1:
                raise ValueError("A must hold 4-bit elements with their blocks along k (dim=-1)")
            return _mx_product(A, B, self.out_dtype or torch.float32)
        _code(A.dtype)
        out_dtype = self.out_dtype or A.dtype
        if A.requires_grad and torch.is_grad_enabled():
            return _MXProduct.apply(A, B, out_dtype)
        return _mx_product(MXQuantizeCUDA(4)(A), B, out_dtype)


class _CheckpointProduct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, A, B):
        C = BMMCUDA()(A, B)
        ctx.a_shape, ctx.dtype = A.shape, A.dtype
        ctx.q = None
        if ctx.needs_input_grad[1] and A.shape[2] != 0:
            ctx.q = MXQuantizeCUDA(8)(A)
        if ctx.needs_input_grad[0]:
            ctx.save_for_backward(B)
        return C

    @staticmethod
    @once_differentiable
    def backward(ctx, dC):
        dA = dB = None
        l, m, k = ctx.a_shape
        n = dC.shape[2]
        if ctx.needs_input_grad[0]:
            B, = ctx.saved_tensors
            dA = BMMCUDA()(dC, B.transpose(1, 2))
        if ctx.needs_input_grad[1]:
            if ctx.q is None or m == 0 or n == 0 or l == 0:
                dB = torch.zeros((l, k, n), dtype=ctx.dtype, device=dC.device)
            elif ctx.dtype in _X16:
                dB = MXDenseBMMCUDA()(dC.transpose(1, 2), ctx.q).transpose(1, 2)
            else:
                dB = BMMCUDA()(ctx.q.dequantize(ctx.dtype).transpose(1, 2), dC)
        return dA, dB


class CheckpointBMMCUDA(BMMCUDA):
    """``CheckpointBMMCUDA()(A, B) -> C``: the product of ``BMMCUDA`` (fp32, fp16, bf16; 2-D or 3-D)
    with a backward pass for which the activations A are kept in 8 bits (``MXQuantizeCUDA(8)``
    along k: 1.03 bytes per element) instead of their own type. C and dA = dC @ B^T are what the full
    A gives; dB = A8^T @ dC uses the kept values, each within 2^-4 of its own size or, where it is
    far below its block's largest, within half of the block's finest step. A itself is not
    kept; B is. Differentiable once."""

    def __call__(self, A: torch.Tensor, B: torch.Tensor) -> torch.Tensor:
        if not (torch.is_grad_enabled() and (A.requires_grad or B.requires_grad)):
            return super().__call__(A, B)
        A3, B3, two_d = self.check_inputs(A, B, (torch.float32,) + _X16)
        C = _CheckpointProduct.apply(A3, B3)
        return C[0] if two_d else C
