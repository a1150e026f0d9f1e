"""CPU restatement in 64 bits of the operators on a paged key/value cache.  TEST INFRASTRUCTURE ONLY.

Written from the formulas: rotary positions as products of complex numbers, attention row by row over the tokens
that a row sees.  Inputs of any floating type are taken at their values; results are float64.  Checked by
tests/test_paged.py against closed forms before the kernels are held to it.
"""
from __future__ import annotations

import numpy as np
import torch


def rotary(x: torch.Tensor, positions: torch.Tensor, frequencies, factor: float = 1.0, interleaved: bool = False) -> torch.Tensor:
    """x [T, heads, dim]; the first 2 len(frequencies) values of a head turned."""
    x = x.double().cpu()
    r = 2 * len(frequencies)
    angle = positions.cpu().numpy().astype(np.float64)[:, None] * np.asarray(frequencies, dtype=np.float64)[None, :]
    turn = torch.from_numpy(factor * np.exp(1j * angle))[:, None, :]
    y = x.clone()
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if interleaved else (x[..., :r // 2], x[..., r // 2:r])
    z = torch.complex(a.contiguous(), b.contiguous()) * turn
    if interleaved:
        y[..., 0:r:2], y[..., 1:r:2] = z.real, z.imag
    else:
        y[..., :r // 2], y[..., r // 2:r] = z.real, z.imag
    return y


def attention(q, k_pages, v_pages, tables, lengths, scale, window=0):
    """(out, sum of weights times |values|, largest sum of |scale q k| of a head) for every row and head, float64.  Only what a
    row sees is looked at."""
    q, tables, lengths = q.double().cpu(), tables.cpu().long(), lengths.cpu().tolist()
    rows, heads, dim = q.shape
    _, kv, ps, _ = k_pages.shape
    out, size, most = torch.zeros(rows, heads, dim, dtype=torch.float64), torch.zeros(rows, heads, dim, dtype=torch.float64), torch.zeros(
        rows, heads, dtype=torch.float64)
    for r, n in enumerate(lengths):
        first = max(0, n - window) if window else 0
        if n <= first:
            continue
        t = torch.arange(first, n)
        page = tables[r][t // ps]
        dev = k_pages.device
        k, v = (p[page.to(dev), :, (t % ps).to(dev)].double().cpu() for p in (k_pages, v_pages))      # [tokens, kv, dim]
        for h in range(heads):
            kh, vh = k[:, h * kv // heads], v[:, h * kv // heads]
            s = scale * (kh @ q[r, h])
            p = torch.softmax(s, 0)
            out[r, h], size[r, h] = p @ vh, p @ vh.abs()
            most[r, h] = (abs(scale) * (kh.abs() @ q[r, h].abs())).max()
    return out, size, most


def attention_bound(want, size, most, dtype, dim, tokens):
    """How far a kernel that rounds its output once may be from `want`: half a step of the output; a score's fp32 sum is off by
    (dim + 4) 2^-24 of its terms, which moves a weight by as much (twice: numerator and denominator); a weight
    in two values of the type by the square of half a step; exponentials and their sums by 2^-21 and tokens 2^-24 (twice)."""
    half = torch.finfo(dtype).eps / 2
    weight = 2 * ((dim + 4) * 2.0 ** -24 * most + 2.0 ** -21 + tokens * 2.0 ** -24) + half ** 2
    return half * want.abs() + size * weight[..., None] * (1 + half) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
