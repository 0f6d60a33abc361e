"""Cases of the microscaled operators, their plain forms and their values in 64 bits.

Three operators: ``quantize`` (a tensor to 4- or 8-bit elements with one power-of-two scale per
block of 32, and back), ``product`` (activations times 4-bit weights, both operands 4-bit on the
tensor cores) and ``step`` (forward and backward pass of a product: over frozen 4-bit weights, or
with its activations kept in 8 bits for the backward pass).

Storage of a matrix of ``rows`` x ``k`` (blocks run along k, which is contiguous): ``codes`` uint8
[l, rows, ceil(k / 32) * 32 * bits / 8], two 4-bit elements per byte, the lower k in the low half;
``scales`` uint8 [l, ceil(rows / 128), ceil(k / 128), 512], the scale of row r and block b of a
128 x 4 group at byte (r % 32) * 16 + (r // 32) * 4 + b, a byte E standing for 2^(E - 127).
"""
import math

import torch

own = False

TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
BLOCK = 32


def listed():
    return [
        # the hidden states of 16 sequences at one decoding step, before a 4-bit projection
        {"name": "quantize4 decode", "op": "quantize", "bits": 4, "dtype": "bfloat16", "l": 1, "rows": 16, "k": 4096, "dim": -1},
        # the activations of a long prompt
        {"name": "quantize4 prompt", "op": "quantize", "bits": 4, "dtype": "bfloat16", "l": 1, "rows": 8192, "k": 8192, "dim": -1},
        # fp32 master weights stored [k][n], laid out once per update; a ragged width
        {"name": "quantize4 weights", "op": "quantize", "bits": 4, "dtype": "float32", "l": 1, "rows": 5001, "k": 4096, "dim": -2},
        # a batch of odd-sized activations kept for a backward pass
        {"name": "quantize8 ragged", "op": "quantize", "bits": 8, "dtype": "float16", "l": 3, "rows": 1003, "k": 1111, "dim": -1},
        # one token through a 4-bit projection
        {"name": "product one token", "op": "product", "dtype": "bfloat16", "l": 1, "m": 1, "n": 4096, "k": 4096},
        # a decoding step of 16 sequences through a wide one
        {"name": "product 16 tokens", "op": "product", "dtype": "bfloat16", "l": 1, "m": 16, "n": 16384, "k": 8192},
        # eight weight matrices, each with the 77 tokens that were sent to it
        {"name": "product batched", "op": "product", "dtype": "float16", "l": 8, "m": 77, "n": 2048, "k": 1408},
        # ragged in every direction, fp32 results
        {"name": "product ragged fp32", "op": "product", "dtype": "float32", "l": 1, "m": 1000, "n": 1999, "k": 2081},
        # a long prompt
        {"name": "product prompt", "op": "product", "dtype": "bfloat16", "l": 1, "m": 8192, "n": 8192, "k": 8192},
        # fine-tuning over frozen 4-bit weights: product and gradient of the activations
        {"name": "step frozen", "op": "step", "keep": 4, "dtype": "bfloat16", "l": 1, "m": 4096, "n": 4096, "k": 4096},
        # training step of a projection whose activations wait for the backward pass in 8 bits
        {"name": "step checkpoint", "op": "step", "keep": 8, "dtype": "bfloat16", "l": 1, "m": 8192, "n": 4096, "k": 4096},
        # the same at small odd sizes, a batch of two, fp16
        {"name": "step checkpoint small", "op": "step", "keep": 8, "dtype": "float16", "l": 2, "m": 333, "n": 520, "k": 203},
    ]


def _log_uniform(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["quantize", "product", "product", "step"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    if op == "quantize":
        l, rows, k = rng.choice([1, 1, 2, 5]), _log_uniform(rng, 1, 8192), _log_uniform(rng, 32, 8192)
        if l * rows * k > 8192 * 8192:
            l = 1
        return {"op": op, "bits": rng.choice([4, 8]), "dtype": dtype, "l": l, "rows": rows, "k": k, "dim": rng.choice([-1, -1, -2])}
    if op == "product":
        l, m = rng.choice([1, 1, 1, 4, 8]), _log_uniform(rng, 1, 8192)
        n, k = _log_uniform(rng, 64, 8192), _log_uniform(rng, 64, 8192)
        if l * m * n * k > 8192 ** 3 or l * n * k > 1 << 28:
            l = 1
        return {"op": op, "dtype": dtype, "l": l, "m": m, "n": n, "k": k}
    return {"op": op, "keep": rng.choice([4, 8]), "dtype": rng.choice(["bfloat16", "float16"]), "l": rng.choice([1, 1, 2]),
            "m": _log_uniform(rng, 64, 4096), "n": _log_uniform(rng, 64, 4096), "k": _log_uniform(rng, 64, 4096)}


# ---- storage -------------------------------------------------------------------------------


def _tile_scales(E):
    """[l, rows, blocks] scale bytes -> [l, ceil(rows / 128), ceil(blocks / 4), 512]."""
    l, rows, kb = E.shape
    rt, kt = -(-rows // 128), -(-kb // 4)
    full = torch.zeros((l, rt * 128, kt * 4), dtype=torch.uint8, device=E.device)
    full[:, :rows, :kb] = E
    return full.view(l, rt, 4, 32, kt, 4).permute(0, 1, 4, 3, 2, 5).reshape(l, rt, kt, 512).contiguous()


def _untile_scales(S, rows, kb):
    l, rt, kt, _ = S.shape
    return S.view(l, rt, kt, 32, 4, 4).permute(0, 1, 4, 3, 2, 5).reshape(l, rt * 128, kt * 4)[:, :rows, :kb]


def _blocks(X, to):
    """X [l, rows, k] -> [l, rows, blocks, 32] in type `to`, zeros behind k."""
    l, rows, k = X.shape
    kb = -(-k // BLOCK)
    if kb * BLOCK == k:
        return X.to(to).reshape(l, rows, kb, BLOCK)
    out = torch.zeros((l, rows, kb * BLOCK), dtype=to, device=X.device)
    out[:, :, :k] = X
    return out.view(l, rows, kb, BLOCK)


def _power(e):
    """2^e in 32 bits, exactly, e in -127 .. 127."""
    half = torch.div(e, 2, rounding_mode="floor")
    return ((half + 127) << 23).view(torch.float32) * ((e - half + 127) << 23).view(torch.float32)


def _element(y, bits):
    """Nearest element value (ties to even) of |y|, saturating."""
    if bits == 4:  # 0, 0.5, 1, 1.5, 2, 3, 4, 6
        step = torch.where(y < 2, 0.5, torch.where(y < 4, 1.0, 2.0))
        return torch.clamp(torch.round(y / step) * step, max=6.0)
    _, e = torch.frexp(y)  # 4 significant bits, steps no finer than 2^-9
    step = _power(torch.clamp(e - 4, min=-9))
    return torch.clamp(torch.round(y / step) * step, max=448.0)


def _scale_exponent(amax, bits, dtype):
    """4 bits: floor(log2 amax) - 2 (the largest may saturate). 8 bits: the least that keeps amax
    within 448 steps, and none so small that a value could not be held in the source's type."""
    frac, e = torch.frexp(amax)  # amax = frac * 2^e, frac in [0.5, 1)
    if bits == 4:
        return torch.where(amax > 0, torch.clamp(e - 3, min=-127), -127)
    low = {"float32": -127, "bfloat16": -124, "float16": -15}[dtype]
    e = e - 9 + (frac > 0.875).to(e.dtype)
    return torch.where(amax > 0, torch.clamp(e, min=low), low)


def _quantized(X, bits, dtype):
    """(values, exponents) of X [l, rows, k] in X's computing type: values [l, rows, blocks, 32]."""
    amax = X.abs().amax(-1, keepdim=True)
    e = _scale_exponent(amax, bits, dtype)
    q = _element((X * _power(-e)).abs(), bits)
    if bits == 8:  # a value that would round up beyond the source's type stays below it
        q = torch.where(e == (8 if dtype == "float16" else 120), torch.clamp(q, max=240.0), q)
    return torch.copysign(q * _power(e), X), e


def _weights(l, n, k, seed):
    """Codes and scales of random 4-bit weights [l, n, k], as a checkpoint holds them."""
    g = torch.Generator("cuda").manual_seed(seed)
    kb = -(-k // BLOCK)
    # elements of normal weights after scaling: magnitude codes 0..7 with falling probabilities
    p = torch.tensor([0.11, 0.20, 0.18, 0.15, 0.17, 0.11, 0.05, 0.03], device="cuda")
    mag = torch.bucketize(torch.rand((l, n, kb * BLOCK), device="cuda", generator=g), torch.cumsum(p, 0)[:-1]).to(torch.uint8)
    c = mag | (torch.randint(0, 2, mag.shape, device="cuda", generator=g, dtype=torch.uint8) << 3)
    c[:, :, k:] = 0
    codes = (c[:, :, 0::2] | (c[:, :, 1::2] << 4)).contiguous()
    E = torch.randint(119, 122, (l, n, kb), device="cuda", generator=g, dtype=torch.int32).to(torch.uint8)
    return codes, _tile_scales(E)


def _decoded(codes, scales, k):
    """Values [l, n, k] of 4-bit codes."""
    l, n, half = codes.shape
    c = torch.stack((codes & 15, codes >> 4), -1).reshape(l, n, half * 2)
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)
    E = _untile_scales(scales, n, half // 16).to(torch.int32) - 127
    v = grid[c.to(torch.int32)].view(l, n, half // 16, BLOCK)
    return (v * _power(E[..., None])).reshape(l, n, half * 2)[:, :, :k]


def _activations(shape, dtype, seed):
    """Normal values whose rows differ in size, with a few large channels and some empty rows."""
    g = torch.Generator("cuda").manual_seed(seed)
    x = torch.randn(shape, device="cuda", generator=g)
    x *= torch.exp(0.5 * torch.randn(shape[:-1] + (1,), device="cuda", generator=g))
    x *= torch.where(torch.rand((shape[-1],), device="cuda", generator=g) < 0.01, 12.0, 1.0)
    if shape[-2] > 4:
        x *= (torch.rand(shape[:-1] + (1,), device="cuda", generator=g) > 0.02)
    return x.to(TYPES[dtype])


# ---- the interface -------------------------------------------------------------------------


def prepare(case, seed):
    s = dict(case)
    l = case["l"]
    if case["op"] == "quantize":
        X = _activations((l, case["rows"], case["k"]), case["dtype"], seed)
        s["X"] = X if case["dim"] == -1 else X.transpose(1, 2).contiguous()
        return s
    m, n, k = case["m"], case["n"], case["k"]
    s["A"] = _activations((l, m, k), case["dtype"], seed)
    if case["op"] == "product" or case["keep"] == 4:
        s["codes"], s["scales"] = _weights(l, n, k, seed + 1000003)
    else:
        g = torch.Generator("cuda").manual_seed(seed + 1000003)
        s["B"] = (torch.randn((l, k, n), device="cuda", generator=g) * k ** -0.5).to(TYPES[case["dtype"]])
    if case["op"] == "step":
        g = torch.Generator("cuda").manual_seed(seed + 2000003)
        s["dC"] = (torch.randn((l, m, n), device="cuda", generator=g) * 0.1).to(TYPES[case["dtype"]])
        s["A"].requires_grad_()
        if case["keep"] == 8:
            s["B"].requires_grad_()
    return s


def _run_own(s):
    from custom_matmul_kernels_b200 import CheckpointBMMCUDA, MXBMMCUDA, MXQuantizeCUDA, MXTensor
    if s["op"] == "quantize":
        return MXQuantizeCUDA(bits=s["bits"])(s["X"], dim=s["dim"]).dequantize(s["X"].dtype)
    if s["op"] == "step" and s["keep"] == 8:
        C = CheckpointBMMCUDA()(s["A"], s["B"])
        dA, dB = torch.autograd.grad(C, (s["A"], s["B"]), s["dC"])
        return {"C": C, "dA": dA, "dB": dB}
    W = MXTensor(s["codes"], s["scales"], bits=4, k=s["k"], dim=-2)  # logical [l, k, n]
    C = MXBMMCUDA()(s["A"], W)
    if s["op"] == "product":
        return C
    dA, = torch.autograd.grad(C, (s["A"],), s["dC"])
    return {"C": C, "dA": dA}


def run(state):
    if own:
        return _run_own(state)
    s = state
    f32 = torch.float32
    if s["op"] == "quantize":
        X = s["X"] if s["dim"] == -1 else s["X"].transpose(1, 2)
        l, rows, k = X.shape
        V = _quantized(_blocks(X, f32), s["bits"], s["dtype"])[0].reshape(l, rows, -1)[:, :, :k].to(X.dtype)
        return V if s["dim"] == -1 else V.transpose(1, 2)
    with torch.no_grad():
        A, l, m, k = s["A"], s["l"], s["m"], s["k"]
        if s["op"] == "step" and s["keep"] == 8:
            A32, B32, dC32 = A.to(f32), s["B"].to(f32), s["dC"].to(f32)
            A8 = _quantized(_blocks(A, f32), 8, s["dtype"])[0].reshape(l, m, -1)[:, :, :k]
            return {"C": torch.bmm(A32, B32).to(A.dtype), "dA": torch.bmm(dC32, B32.transpose(1, 2)).to(A.dtype),
                    "dB": torch.bmm(A8.transpose(1, 2), dC32).to(A.dtype)}
        W = _decoded(s["codes"], s["scales"], k)
        A4 = _quantized(_blocks(A, f32), 4, s["dtype"])[0].reshape(l, m, -1)[:, :, :k]
        C = torch.bmm(A4, W.transpose(1, 2)).to(A.dtype)
        if s["op"] == "product":
            return C
        return {"C": C, "dA": torch.bmm(s["dC"].to(f32), W).to(A.dtype)}  # straight through A's rounding


def _exact_power(e):
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _exact_quantized(X, bits, dtype):
    """Values of X [l, rows, k] by search among all element values, in 64 bits."""
    l, rows, k = X.shape
    B = _blocks(X, torch.float64)
    amax = B.abs().amax(-1, keepdim=True)
    if bits == 4:
        grid = [0, 0.5, 1, 1.5, 2, 3, 4, 6]
        e = (amax.view(torch.int64) >> 52) - 1025  # floor(log2(amax)) - 2, from the exponent's own bits
    else:
        grid = [j * 2.0 ** -9 for j in range(8)] + [(8 + j) * 2.0 ** (x - 10) for x in range(1, 16) for j in range(8)][:-1]
        e = (amax.view(torch.int64) >> 52) - 1030  # the larger of the two candidates
        e = torch.where(amax <= 448 * _exact_power(e - 1), e - 1, e)
        e = e.clamp(min={"float32": -127, "bfloat16": -124, "float16": -15}[dtype])
    e = torch.where(amax > 0, e, torch.zeros_like(e))
    y = (B * _exact_power(-e)).abs()
    g = torch.tensor(grid, dtype=torch.float64, device=X.device)
    if bits == 8 and dtype == "float16":
        y = torch.where(e == 8, y.clamp(max=240.0), y)
    hi = torch.searchsorted(g, y).clamp(max=len(grid) - 1)
    lo = (hi - 1).clamp(min=0)
    up, down = g[hi] - y, y - g[lo]
    at = torch.where((up < down) | ((up == down) & (hi % 2 == 0)) | (y > g[-1]), hi, lo)
    return (torch.sign(B) * g[at] * _exact_power(e)).reshape(l, rows, -1)[:, :, :k]


def exact(case, seed):
    s = prepare(case, seed)
    f64 = torch.float64
    if case["op"] == "quantize":
        X = s["X"] if case["dim"] == -1 else s["X"].transpose(1, 2)
        V = _exact_quantized(X, case["bits"], case["dtype"])
        return V if case["dim"] == -1 else V.transpose(1, 2)
    with torch.no_grad():
        A, k = s["A"], case["k"]
        if case["op"] == "step" and case["keep"] == 8:
            B, dC = s["B"].to(f64), s["dC"].to(f64)
            A8 = _exact_quantized(A, 8, case["dtype"])
            return {"C": A.to(f64) @ B, "dA": dC @ B.transpose(1, 2), "dB": A8.transpose(1, 2) @ dC}
        c = s["codes"].to(torch.int64)
        c = torch.stack((c % 16, c // 16), -1).flatten(2)
        mag, sign = c % 8, 1.0 - 2.0 * (c // 8).to(f64)
        v = torch.where(mag < 2, 0.5 * mag, _exact_power(mag // 2 - 1) * (1 + 0.5 * (mag % 2)))  # 2 exponent bits, 1 of mantissa
        r = torch.arange(case["n"], device="cuda")[:, None]
        b = torch.arange(c.shape[2] // BLOCK, device="cuda")[None, :]
        at = (r // 128 * s["scales"].shape[2] + b // 4) * 512 + r % 32 * 16 + r % 128 // 32 * 4 + b % 4
        e = s["scales"].flatten(1)[:, at.flatten()].view(-1, *at.shape).to(f64) - 127
        W = (sign * v * torch.repeat_interleave(_exact_power(e), BLOCK, -1))[:, :, :k]
        del c, mag, sign, v
        C = _exact_quantized(A, 4, case["dtype"]) @ W.transpose(1, 2)
        return C if case["op"] == "product" else {"C": C, "dA": s["dC"].to(f64) @ W}


def work(case):
    size = torch.finfo(TYPES[case["dtype"]]).bits // 8
    l = case["l"]
    if case["op"] == "quantize":  # read, codes and scales written and read again, values written
        n = l * case["rows"] * case["k"]
        return {"bytes": 2 * n * size + 2 * n * (case["bits"] / 8 + 1 / BLOCK), "flops": 4 * n}
    m, n, k = case["m"], case["n"], case["k"]
    mnk = 2.0 * l * m * n * k
    w4 = n * k * (0.5 + 1 / BLOCK)
    if case["op"] == "product":
        return {"bytes": l * (w4 + size * (m * k + m * n)), "flops": mnk}
    if case["keep"] == 4:  # A in, C out, dC in, dA out
        return {"bytes": l * (w4 + size * (2 * m * k + 2 * m * n)), "flops": 2 * mnk}
    a8 = m * k * (1 + 1 / BLOCK)  # written by the forward pass, read by the backward pass
    return {"bytes": l * (size * (2 * m * k + 2 * k * n + 2 * m * n) + 2 * a8), "flops": 3 * mnk}
