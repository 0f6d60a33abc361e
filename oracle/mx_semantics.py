"""Plain 64-bit forms of the microscaled operators (test infrastructure only).

Quantisation by search over every element value, storage index by index, products in float64.
"""
from __future__ import annotations

import math

import torch

E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
E4M3 = [j * 2.0 ** -9 for j in range(8)] + [(8 + j) * 2.0 ** (x - 10) for x in range(1, 16) for j in range(8)][:-1]
LOW8 = {torch.float32: -127, torch.bfloat16: -124, torch.float16: -15}


def block_exponent(amax: float, bits: int, dtype: torch.dtype) -> int:
    """Exponent of the scale of a block whose largest magnitude is amax (finite)."""
    if bits == 4:
        return -127 if amax == 0 else max(math.frexp(amax)[1] - 3, -127)
    if amax == 0:
        return LOW8[dtype]
    e = math.frexp(amax)[1] - 9
    if amax > 448 * 2.0 ** e:
        e += 1
    return max(e, LOW8[dtype])


def nearest_code(y: float, grid) -> int:
    """Index of the grid value nearest to y >= 0; a tie goes to the even index; saturating."""
    if y >= grid[-1]:
        return len(grid) - 1
    hi = next(i for i, g in enumerate(grid) if g >= y)
    if grid[hi] == y:
        return hi
    lo = hi - 1
    up, down = grid[hi] - y, y - grid[lo]
    return hi if up < down or (up == down and hi % 2 == 0) else lo


def quantize(X: torch.Tensor, bits: int):
    """X [rows, k] on the CPU -> (codes int64 [rows, k], scale bytes int64 [rows, blocks]).
    A code is the element's index in its value table with the sign above it."""
    grid = E2M1 if bits == 4 else E4M3
    rows, k = X.shape
    nb = (k + 31) // 32
    codes = torch.zeros((rows, k), dtype=torch.int64)
    scales = torch.zeros((rows, nb), dtype=torch.int64)
    g = torch.tensor(grid, dtype=torch.float64)
    for r in range(rows):
        for b in range(nb):
            x = X[r, 32 * b:32 * b + 32].double()
            if not bool(torch.isfinite(x).all()):
                scales[r, b] = 255
                continue
            e = block_exponent(float(x.abs().max()), bits, X.dtype)
            scales[r, b] = e + 127
            y = x.abs() * 2.0 ** -e
            if bits == 8 and e == (8 if X.dtype == torch.float16 else 120):
                y = y.clamp(max=240.0)
            # the vector form of nearest_code
            hi = torch.searchsorted(g, y).clamp(max=len(grid) - 1)
            lo = (hi - 1).clamp(min=0)
            up, down = g[hi] - y, y - g[lo]
            at = torch.where((up < down) | ((up == down) & (hi % 2 == 0)) | (y > g[-1]), hi, lo)
            codes[r, 32 * b:32 * b + 32] = at + torch.signbit(x).long() * (8 if bits == 4 else 128)
    return codes, scales


def values(codes: torch.Tensor, scales: torch.Tensor, bits: int) -> torch.Tensor:
    """float64 values of (codes [.., k], scale bytes [.., blocks])."""
    grid = torch.tensor(E2M1 if bits == 4 else E4M3 + [math.nan], dtype=torch.float64)
    half = 8 if bits == 4 else 128
    v = grid[codes % half] * torch.where(codes >= half, -1.0, 1.0)
    e = scales.repeat_interleave(32, -1)[..., :codes.shape[-1]]
    return torch.where(e == 255, math.nan, v * torch.pow(2.0, e.double() - 127))


def pack(codes: torch.Tensor, scales: torch.Tensor, bits: int):
    """Storage of one matrix: codes uint8 [rows, pitch], scales uint8 [row groups, k groups, 512]."""
    rows, k = codes.shape
    nb = (k + 31) // 32
    full = torch.zeros((rows, nb * 32), dtype=torch.int64)
    full[:, :k] = codes
    stored = full if bits == 8 else full[:, 0::2] + 16 * full[:, 1::2]
    rg, kg = (rows + 127) // 128, (k + 127) // 128
    S = torch.zeros(rg * kg * 512, dtype=torch.int64)
    r = torch.arange(rows)[:, None]
    b = torch.arange(nb)[None, :]
    S[(r // 128 * kg + b // 4) * 512 + r % 32 * 16 + r % 128 // 32 * 4 + b % 4] = scales
    return stored.to(torch.uint8), S.view(rg, kg, 512).to(torch.uint8)


def random_mx(rows: int, k: int, bits: int, seed: int, lo: int = 120, hi: int = 131):
    """Random codes (no NaN) and scale bytes in [lo, hi)."""
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 16 if bits == 4 else 256, (rows, k), generator=g)
    if bits == 8:
        codes[codes % 128 == 127] = 5
    scales = torch.randint(lo, hi, (rows, (k + 31) // 32), generator=g)
    return codes, scales
