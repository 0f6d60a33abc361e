"""Microscaled operands: 4- and 8-bit elements with a power-of-two scale per block of 32, products
that read them, and a training product that keeps its activations in 8 bits.

The reference stops at fp32 (its kernels take float* only, kernels/bmm.cu:185); these are the
narrow forms of the same batched product.

All calls work on the stream that is current on their tensors' device and can be captured into CUDA
graphs, backward passes too. As for every torch operation, an eager graph of the same leaves must
not be alive while a backward pass is captured: torch then ends the capture with an error.
"""
from __future__ import annotations

import functools

import torch
from torch.autograd.forward_ad import unpack_dual
from torch.autograd.function import once_differentiable

from .bmm import BMMCUDA
from .custom_kernel import FBMM_BF16, FBMM_F16, FBMM_F32, CustomKernel, check, load_library

_DTYPES = {torch.float32: FBMM_F32, torch.float16: FBMM_F16, torch.bfloat16: FBMM_BF16}
_X16 = (torch.float16, torch.bfloat16)
_N, _T = ord("n"), ord("t")
BLOCK = 32


def _code(dtype: torch.dtype) -> int:
    code = _DTYPES.get(dtype)
    if code is None:
        raise TypeError(f"dtype {dtype} is not one of float32, float16, bfloat16")
    return code


try:  # the stream's handle without a Stream object around it (2 us less per call)
    _raw_stream = torch._C._cuda_getCurrentRawStream
except AttributeError:
    def _raw_stream(index: int) -> int:
        return torch.cuda.current_stream(index).cuda_stream


_functions = {}


def _function(name: str):
    """The library's entry point `name` (load_library raises where the library is not built)."""
    fn = _functions[name] = getattr(load_library(), name)
    return fn


def _call(name: str, index: int, *args) -> None:
    """One library call on the stream that is current on device `index`; the device is only switched
    when it is not the current one (the switch costs more than the call)."""
    fn = _functions.get(name) or _function(name)
    if torch.cuda.current_device() == index:
        rc = fn(_raw_stream(index), *args)
    else:
        with torch.cuda.device(index):
            rc = fn(_raw_stream(index), *args)
    if rc:
        check(rc)


def _dense_layout(X: torch.Tensor):
    """(tensor, layout letter, pitch, batch stride) of a [l, r, c] tensor whose last ('n') or middle
    ('t') axis is contiguous; any other order is copied."""
    l, r, c = X.shape
    sl, sr, sc = X.stride()
    if (sc == 1 or c == 1) and (sr >= c or r == 1):
        return X, _N, max(sr, c), sl
    if (sr == 1 or r == 1) and (sc >= r or c == 1):
        return X, _T, max(sc, r), sl
    return X.contiguous(), _N, c, r * c


def _x16_layout(X: torch.Tensor):
    """The same with the bytes of workspace that the 16-bit products repack it in: 0 for storage that
    their copies can address (base, pitch and batch stride multiples of 16 bytes)."""
    X, letter, ld, step = _dense_layout(X)
    l, r, c = X.shape
    batched = l > 1 and step != 0
    if X.data_ptr() % 16 == 0 and ld % 8 == 0 and not (batched and step % 8):
        return X, letter, ld, step, 0
    outer, inner = (r, c) if letter == _N else (c, r)
    return X, letter, ld, step, ((l if batched else 1) * outer * ((inner + 7) // 8 * 16) + 255) // 256 * 256


class MXTensor:
    """A [l, r, c] (or [r, c]) matrix held as microscaled elements.

    ``codes`` uint8 [l, rows, ceil(k / 32) * 32 * bits / 8] and ``scales`` uint8
    [l, ceil(rows / 128), ceil(k / 128), 512] as ``include/fbmm.h`` lays them out; k is the extent
    of the axis the blocks run along, ``dim``: -1 (the matrix is [l, rows, k]) or -2 (it is
    [l, k, rows], held k-contiguous all the same). A batch stride of 0 (an expanded tensor)
    serves every batch with one matrix. 2-D codes with 3-D scales make a 2-D matrix. The codes
    behind k must be zero, and so must the scale bytes of rows and blocks that do not exist, as
    ``MXQuantizeCUDA`` leaves them: the 4-bit products multiply the padding behind k too, where a scale
    byte of 255 would make a whole row of the result NaN. A scale byte of 255 makes its block NaN; an
    8-bit code of 0x7f or 0xff is NaN by itself."""

    # Storage is either the caller's two tensors or one buffer (codes, then scales), of which `codes`
    # and `scales` are views made when asked for: one allocation per quantisation.
    __slots__ = ("_buffer", "_codes", "_scales", "_l", "rows", "bits", "k", "dim", "two_d")

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
        if not codes.is_cuda or not scales.is_cuda or codes.get_device() != scales.get_device():
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
        if scales.shape != want:
            raise ValueError(f"scales have shape {tuple(scales.shape)}, expected {want}")
        self._buffer = None
        self._codes = self._addressable(codes, rows * pitch)
        self._scales = self._addressable(scales, want[1] * want[2] * 512)
        self._l, self.rows, self.bits, self.k, self.dim, self.two_d = l, rows, bits, k, dim, two_d

    @staticmethod
    def _addressable(t: torch.Tensor, per_batch: int) -> torch.Tensor:
        """t itself where its batches are dense, lie 16 bytes apart (or are one) and start aligned."""
        if t.is_contiguous() and t.data_ptr() % 16 == 0:
            return t
        step = t.stride(0)
        if (t.numel() and t[0].is_contiguous() and t.data_ptr() % 16 == 0
                and (t.shape[0] == 1 or step == 0 or (step >= per_batch and step % 16 == 0))):
            return t
        return t.clone(memory_format=torch.contiguous_format)

    @classmethod
    def _around(cls, tensors, l, rows, k, bits, dim, two_d) -> "MXTensor":
        """One made of `_tensors()` of another (a buffer, or codes and scales)."""
        t = object.__new__(cls)
        if len(tensors) == 1:
            t._buffer, t._codes, t._scales = tensors[0], None, None
        else:
            t._buffer, (t._codes, t._scales) = None, tensors
        t._l, t.rows, t.bits, t.k, t.dim, t.two_d = l, rows, bits, k, dim, two_d
        return t

    def _tensors(self) -> tuple:
        return (self._codes, self._scales) if self._buffer is None else (self._buffer,)

    def _sizes(self):
        """Bytes per batch of codes and scales."""
        blocks = (self.k + BLOCK - 1) // BLOCK
        return self.rows * blocks * (4 * self.bits), (self.rows + 127) // 128 * ((blocks + 3) // 4) * 512

    @property
    def codes(self) -> torch.Tensor:
        if self._codes is None:
            per, _ = self._sizes()
            self._codes = self._buffer[:self._l * per].view(self._l, self.rows, (self.k + BLOCK - 1) // BLOCK * (4 * self.bits))
        return self._codes

    @property
    def scales(self) -> torch.Tensor:
        if self._scales is None:
            per, _ = self._sizes()
            self._scales = self._buffer[self._l * per:].view(self._l, (self.rows + 127) // 128, (self.k + 127) // 128, 512)
        return self._scales

    @property
    def device(self) -> torch.device:
        return self._tensors()[0].device

    @property
    def shape(self) -> tuple:
        s = (self.rows, self.k) if self.dim == -1 else (self.k, self.rows)
        return s if self.two_d else (self._l,) + s

    @property
    def mT(self) -> "MXTensor":
        """The transposed matrix: the same storage with the blocks along the other axis."""
        return self._around(self._tensors(), self._l, self.rows, self.k, self.bits, -3 - self.dim, self.two_d)

    def _arguments(self):
        """codes, their batch stride, scales, their batch stride (bytes; 0: one matrix for all)."""
        if self._buffer is None:
            return self._codes.data_ptr(), self._codes.stride(0), self._scales.data_ptr(), self._scales.stride(0)
        per, groups = self._sizes()
        at = self._buffer.data_ptr()
        return at, per, at + self._l * per, groups  # a row of codes is a multiple of 16 bytes

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """Element times scale, rounded once to `dtype`; with dim=-2 a transposed view of
        k-contiguous storage."""
        code = _code(dtype)
        l, rows, k = self._l, self.rows, self.k
        t = self._tensors()[0]
        out = t.new_empty((l, rows, k), dtype=dtype)
        if l and rows:
            codes, sc, scales, ss = self._arguments()
            _call("fbmm_mx_dequantize", t.get_device(), codes, sc, scales, ss, self.bits, out.data_ptr(), code, k, rows * k,
                  l, rows, k)
        if self.dim == -2:
            out = out.transpose(1, 2)
        return out[0] if self.two_d else out

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
        if not X.is_cuda:
            raise ValueError("X must be a CUDA tensor")
        X3 = X[None] if two_d else X
        if dim == -2:
            X3 = X3.transpose(1, 2)  # [l, rows, k] whichever axis the blocks run along
        l, rows, k = X3.shape
        if k == 0:
            raise ValueError("the axis the blocks run along is empty")
        q = MXTensor._around((None,), l, rows, k, self.bits, dim, two_d)
        codes, scales = q._sizes()
        q._buffer = X.new_empty(l * (codes + scales), dtype=torch.uint8)
        if l and rows:
            X3, layout, ld, step = _dense_layout(X3)
            at = q._buffer.data_ptr()
            _call("fbmm_mx_quantize", X.get_device(), X3.data_ptr(), dtype, layout, ld, step, self.bits, at, at + l * codes, l,
                  rows, k)
        return q


def _check_product(A, B) -> bool:
    """Shapes and devices of a product with a microscaled operand; True for 2-D operands."""
    a, b = A.shape, B.shape
    if len(a) != len(b):
        raise ValueError("A and B need the same number of dimensions")
    if len(a) not in (2, 3):
        raise ValueError("A and B need to be 2d or 3d")
    if len(a) == 3 and a[0] != b[0]:
        raise ValueError(f"batch sizes differ: {a[0]} vs {b[0]}")
    if a[-1] != b[-2]:
        raise ValueError(f"inner dimensions differ: A {tuple(a)} B {tuple(b)}")
    for X in (A, B):
        if isinstance(X, torch.Tensor) and not X.is_cuda:
            raise ValueError("A and B must be CUDA tensors")
    if _index(A) != _index(B):
        raise ValueError("A and B must be on the same device")
    return len(a) == 2


def _index(X) -> int:
    """Device index of a tensor or MXTensor."""
    return (X if isinstance(X, torch.Tensor) else X._tensors()[0]).get_device()


def _dense_bmm(A: torch.Tensor, B: torch.Tensor) -> torch.Tensor:
    """16-bit [l, m, k] @ [l, k, n] in any storage order, k > 0."""
    l, m, k = A.shape
    n = B.shape[2]
    C = A.new_empty((l, m, n))
    if l and m and n:
        a, la, lda, sa, need_a = _x16_layout(A)
        b, lb, ldb, sb, need_b = _x16_layout(B)
        need = need_a + need_b
        ws = A.new_empty(need, dtype=torch.uint8) if need else None
        _call("fbmm_dense_bmm_x16", A.get_device(), a.data_ptr(), la, lda, sa, b.data_ptr(), lb, ldb, sb, _DTYPES[A.dtype],
              C.data_ptr(), n, m * n, l, m, n, k, ws.data_ptr() if need else None, need)
    return C


class MXDenseBMMCUDA(CustomKernel):
    """``MXDenseBMMCUDA()(A, B) -> C``: A [l, m, k] @ B [l, k, n] with one fp16 / bf16 tensor and
    one ``MXTensor`` (4 or 8 bits) whose blocks run along its own axis of C (``dim=-2`` for A,
    ``dim=-1`` for B); C in the tensor's type, fp32 sums. The microscaled elements times their
    scales enter as values of that type: exact for bf16, and for fp16 wherever they are fp16
    values. These are the products of the backward passes below: activations' gradient through
    4-bit weights, weights' gradient from activations kept in 8 bits. No gradient flows through."""

    def __call__(self, A, B) -> torch.Tensor:
        if isinstance(A, MXTensor) == isinstance(B, MXTensor):
            raise TypeError("one of A and B must be an MXTensor, the other a tensor")
        two_d = _check_product(A, B)
        mx, dense = (A, B) if isinstance(A, MXTensor) else (B, A)
        if dense.dtype not in _X16:
            raise TypeError(f"dtype {dense.dtype} is not one of float16, bfloat16")
        if mx.dim != (-2 if mx is A else -1):
            raise ValueError("the blocks must run along the operand's own axis of C (dim=-2 for A, dim=-1 for B)")
        D = dense[None] if two_d else dense
        l, m, n = D.shape[0], A.shape[-2], B.shape[-1]
        k = A.shape[-1]
        C = D.new_empty((l, m, n))
        if C.numel() == 0 or k == 0:
            C.zero_()
        else:
            d, letter, ld, step, need = _x16_layout(D)
            if mx is A and letter != _N:
                d, letter, ld, step, need = _x16_layout(D.contiguous())
            ws = D.new_empty(need, dtype=torch.uint8) if need else None
            tail = C.data_ptr(), n, m * n, l, m, n, k, ws.data_ptr() if need else None, need
            if mx is B:
                _call("fbmm_dense_mx_bmm_x16", D.get_device(), d.data_ptr(), letter, ld, step, _DTYPES[D.dtype],
                      *mx._arguments(), mx.bits, *tail)
            else:
                _call("fbmm_mx_dense_bmm_x16", D.get_device(), *mx._arguments(), mx.bits, d.data_ptr(), ld, step,
                      _DTYPES[D.dtype], *tail)
        return C[0] if two_d else C


@functools.lru_cache(maxsize=4096)
def _product_workspace(index: int, l: int, m: int, n: int, k: int, layout: int) -> int:
    """Scratch bytes of a product with a tensor on device `index`, by whose SM count the library decides whether the
    rows are quantised inside the product."""
    with torch.cuda.device(index):
        return load_library().fbmm_mx4_bmm_tensor_workspace_bytes(l, m, n, k, layout)


def _mx4_product(A, B: MXTensor, out_dtype: torch.dtype) -> torch.Tensor:
    two_d = B.two_d
    n, k = B.rows, B.k
    if isinstance(A, MXTensor):
        l, m, t = A._l, A.rows, A._tensors()[0]
    else:
        t = A[None] if two_d else A
        l, m, _ = t.shape
    C = t.new_empty((l, m, n), dtype=out_dtype)
    if l and m and n:
        result = C.data_ptr(), _DTYPES[out_dtype], n, m * n, l, m, n, k
        if isinstance(A, MXTensor):
            _call("fbmm_mx4_bmm", t.get_device(), *A._arguments(), *B._arguments(), *result)
        else:
            t, layout, ld, step = _dense_layout(t)
            need = _product_workspace(t.get_device(), l, m, n, k, layout)
            ws = t.new_empty(need, dtype=torch.uint8) if need else None
            _call("fbmm_mx4_bmm_tensor", t.get_device(), t.data_ptr(), _DTYPES[t.dtype], layout, ld, step, *B._arguments(),
                  *result, ws.data_ptr() if need else None, need)
    return C[0] if two_d else C


def _refuse_tangents(*tensors) -> None:
    """The differentiable products have reverse mode only; without this a tangent would be dropped."""
    for t in tensors:
        if unpack_dual(t).tangent is not None:
            raise NotImplementedError("this product has no forward-mode derivative: its operands must not carry a tangent")


def _once(backward):
    """A backward pass that can itself not be differentiated. The wrapper that says so to a graph
    of higher order (10 us a call) is only entered where such a graph is being made."""
    guarded = once_differentiable(backward)

    def run(ctx, dC):
        _refuse_tangents(dC)
        return guarded(ctx, dC) if torch.is_grad_enabled() else backward(ctx, dC)
    return run


class _MX4Product(torch.autograd.Function):
    """C = Q4(A) @ B, differentiable in A: straight through the rounding, dA = dC @ B^T."""

    @staticmethod
    def forward(ctx, A, B, out_dtype):
        ctx.dtype, ctx.shape = A.dtype, (B._l, B.rows, B.k, 4, -1, B.two_d)  # of B^T, [l, n, k]
        ctx.save_for_backward(*B._tensors())
        return _mx4_product(A, B, out_dtype)

    @staticmethod
    @_once
    def backward(ctx, dC):
        BT = MXTensor._around(ctx.saved_tensors, *ctx.shape)
        dC = dC.to(ctx.dtype)
        if ctx.dtype in _X16:
            return MXDenseBMMCUDA()(dC, BT), None, None
        return BMMCUDA()(dC, BT.dequantize(ctx.dtype)), None, None


class MXBMMCUDA(CustomKernel):
    """``MXBMMCUDA(out_dtype)(A, B) -> C``: A [l, m, k] times B [l, k, n], both with 4-bit elements
    (``MXTensor``, blocks along k: ``dim=-1`` for A, ``dim=-2`` for B). A may be a fp32 / fp16 /
    bf16 tensor, which is quantised on the way; C then has its type unless `out_dtype` says
    otherwise, and is differentiable in A (the gradient passes straight through A's rounding:
    dA = dC @ B^T with B's values, computed in A's type; forward-mode tangents are refused). With a
    microscaled A, C is fp32 unless `out_dtype` says otherwise. Products and scales are exact, sums
    are kept in fp32, C is rounded once."""

    def __init__(self, out_dtype: torch.dtype | None = None):
        super().__init__()
        if out_dtype is not None:
            _code(out_dtype)
        self.out_dtype = out_dtype

    def __call__(self, A, B: MXTensor) -> torch.Tensor:
        if not isinstance(B, MXTensor):
            raise TypeError("B must be an MXTensor")
        _check_product(A, B)
        if B.bits != 4 or B.dim != -2:
            raise ValueError("B must hold 4-bit elements with their blocks along k (dim=-2)")
        if isinstance(A, MXTensor):
            if A.bits != 4 or A.dim != -1:
                raise ValueError("A must hold 4-bit elements with their blocks along k (dim=-1)")
            return _mx4_product(A, B, self.out_dtype or torch.float32)
        _code(A.dtype)
        _refuse_tangents(A)
        out_dtype = self.out_dtype or A.dtype
        if A.requires_grad and torch.is_grad_enabled():
            return _MX4Product.apply(A, B, out_dtype)
        return _mx4_product(A, B, out_dtype)


class _CheckpointProduct(torch.autograd.Function):
    """Operands are 3-D with every extent positive."""

    @staticmethod
    def forward(ctx, A, B):
        C = _dense_bmm(A, B) if A.dtype in _X16 else BMMCUDA()(A, B)
        need_a, need_b = ctx.needs_input_grad
        ctx.shape = (*A.shape, 8, -1, False)
        ctx.b_transposed = B.stride(2) != 1 and B.stride(1) == 1
        ctx.save_for_backward(B if need_a else None, *(MXQuantizeCUDA(8)(A)._tensors() if need_b else ()))
        return C

    @staticmethod
    @_once
    def backward(ctx, dC):
        B, *kept = ctx.saved_tensors
        x16 = dC.dtype in _X16
        dA = dB = None
        if B is not None:
            BT = B.transpose(1, 2)
            dA = _dense_bmm(dC, BT) if x16 else BMMCUDA()(dC, BT)
        if kept:
            A8 = MXTensor._around(kept, *ctx.shape)
            if not x16:
                dB = BMMCUDA()(A8.mT.dequantize(dC.dtype), dC)
            elif ctx.b_transposed:  # in B's own storage order
                dB = MXDenseBMMCUDA()(dC.transpose(1, 2), A8).transpose(1, 2)
            else:
                dB = MXDenseBMMCUDA()(A8.mT, dC)
        return dA, dB


class CheckpointBMMCUDA(BMMCUDA):
    """``CheckpointBMMCUDA()(A, B) -> C``: the product of ``BMMCUDA`` (fp32, fp16, bf16; 2-D or 3-D)
    with a backward pass for which the activations A are kept in 8 bits (``MXQuantizeCUDA(8)``
    along k: 1.03 bytes per element) instead of their own type. C and dA = dC @ B^T are what the full
    A gives; dB = A8^T @ dC uses the kept values, each within 2^-4 of its own size or, where it is
    far below its block's largest, within half of the block's finest step. A itself is not
    kept; B is. Differentiable once, in reverse mode (forward-mode tangents are refused). Without a
    gradient to compute it is ``BMMCUDA``."""

    def __call__(self, A: torch.Tensor, B: torch.Tensor) -> torch.Tensor:
        _refuse_tangents(A, B)
        if not (torch.is_grad_enabled() and (A.requires_grad or B.requires_grad)):
            return super().__call__(A, B)
        A3, B3, two_d = self.check_inputs(A, B, (torch.float32,) + _X16)
        l, m, k = A3.shape
        if min(l, m, k, B3.shape[2]) == 0:
            C = torch.bmm(A3, B3)  # nothing to compute or to keep: empty, or zeros with zero gradients
        else:
            C = _CheckpointProduct.apply(A3, B3)
        return C[0] if two_d else C
