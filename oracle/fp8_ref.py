"""The 8-bit block format and its products in 64 bits on the CPU, from their definition.

A block is 128 consecutive columns of a row (weights: 128 x 128).  Its scale is 2^e, e the smallest integer >= -126 for which the
largest finite magnitude is at most MAX * 2^e (0 without one); an element is x * 2^-e rounded to nearest even.
"""
from __future__ import annotations

import math

import torch

BLOCK = 128
MAX = {"e4m3": 448.0, "e5m2": 57344.0}
DIGITS = {"e4m3": (3, -6), "e5m2": (2, -14)}          # fraction bits, exponent of the smallest normal number
TYPE = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}


def exponent(block: torch.Tensor, fmt: str) -> int:
    """e of one block."""
    b = block.double().abs()
    b = b[torch.isfinite(b)]
    top = float(b.max()) if b.numel() else 0.0
    if top == 0.0:
        return 0
    m, e = math.frexp(top / MAX[fmt])                  # top / MAX = m * 2^e, 0.5 <= m < 1 (MAX has three bits: nearly exact)
    e = e - 1
    while top > MAX[fmt] * math.ldexp(1.0, e):
        e += 1
    while top <= MAX[fmt] * math.ldexp(1.0, e - 1):
        e -= 1
    return max(e, -126)


def round8(u: torch.Tensor, fmt: str) -> torch.Tensor:
    """u (fp64, at most MAX where finite) to the nearest 8-bit value, ties to even."""
    digits, low = DIGITS[fmt]
    _, e = torch.frexp(torch.where(torch.isfinite(u), u, 1.0))
    step = torch.ldexp(torch.ones_like(u), (e - 1).clamp_min(low) - digits)
    r = torch.round(u / step) * step
    if fmt == "e4m3":
        r = torch.where(torch.isinf(u), float("nan"), r)
    return r


def pack_rows(x: torch.Tensor, fmt: str = "e4m3"):
    """(values fp64 like x, exponents (rows, blocks)) of a tensor packed by rows."""
    c = x.shape[-1]
    v = x.double().reshape(-1, c).clone()
    kb = -(-c // BLOCK)
    ex = torch.zeros((v.shape[0], kb), dtype=torch.int64)
    for r in range(v.shape[0]):
        for k in range(kb):
            s = slice(k * BLOCK, min(c, (k + 1) * BLOCK))
            e = exponent(v[r, s], fmt)
            ex[r, k] = e
            v[r, s] = round8(v[r, s] * math.ldexp(1.0, -e), fmt) * math.ldexp(1.0, e)
    return v.reshape(x.shape), ex


def pack_weight(w: torch.Tensor):
    """(values fp64, exponents (row blocks, column blocks)) of a weight."""
    n, k = w.shape
    v = w.double().clone()
    ex = torch.zeros((-(-n // BLOCK), -(-k // BLOCK)), dtype=torch.int64)
    for i in range(ex.shape[0]):
        for j in range(ex.shape[1]):
            s = (slice(i * BLOCK, (i + 1) * BLOCK), slice(j * BLOCK, (j + 1) * BLOCK))
            e = exponent(v[s], "e4m3")
            ex[i, j] = e
            v[s] = round8(v[s] * math.ldexp(1.0, -e), "e4m3") * math.ldexp(1.0, e)
    return v, ex


def stored(values: torch.Tensor, ex: torch.Tensor, fmt: str = "e4m3", rows_per_scale: int = 1):
    """(bytes, scale bytes) of the stored format, padding included, for values and exponents of pack_rows / pack_weight."""
    c = values.shape[-1]
    v = values.reshape(-1, c)
    e = ex.repeat_interleave(rows_per_scale, 0)[:v.shape[0]].repeat_interleave(BLOCK, 1)[:, :c]
    q = torch.zeros((v.shape[0], (c + 15) // 16 * 16), dtype=torch.uint8)
    q[:, :c] = torch.ldexp(v, -e).float().to(TYPE[fmt]).view(torch.uint8)
    s = torch.full((ex.shape[0], (ex.shape[1] + 3) // 4 * 4), 127, dtype=torch.uint8)
    s[:, :ex.shape[1]] = (ex + 127).to(torch.uint8)
    return q, s


def silu(t: torch.Tensor) -> torch.Tensor:
    return t * torch.sigmoid(t)
