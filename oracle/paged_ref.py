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


def tokens_as_rows(starts, lengths, tables, groups=None, prefixes=None, page_size=None):
    """(rows, lengths, tables) of the new tokens of a batch as rows of one token each: what `attention` above takes.  A row with a prefix reads it through
    the table of the first row of its group that has tokens."""
    starts, lengths, tables = [int(x) for x in starts], [int(n) for n in lengths], tables.cpu().clone()
    if groups is not None:
        for g, prefix in enumerate(prefixes.tolist()):
            rows = [r for r in range(int(groups[g]), int(groups[g + 1])) if lengths[r] > 0 and starts[r + 1] > starts[r]]
            for r in rows:
                # as far as the first new token of each sees; a page that the prefix ends in is shared as a whole only where it is the same page
                cut = max(0, min([prefix] + [lengths[x] - (starts[x + 1] - starts[x]) + 1 for x in rows]))
                tables[r, :cut // page_size] = tables[rows[0], :cut // page_size]
    row, length = [], []
    for r, n in enumerate(lengths):
        c = starts[r + 1] - starts[r]
        for i in range(c):
            row.append(r)
            length.append(max(0, n - (c - 1 - i)) if n > 0 else 0)
    return row, torch.tensor(length, dtype=torch.int64), tables[row] if row else tables[:0]


def prefix_bound(want, size, most, dtype, dim, tokens, largest):
    """attention_bound for weights p that are rounded to the type, p (1 + d) with d up to half a step, in the sum of values and in that of weights:
    sum p (1 + d) v / sum p (1 + d) is off from sum p v / sum p = o by  sum p d (v - o) / sum p (1 + d),  at most half a step of the sum of
    p |v| and |o|, over 1 - half a step.  float16 holds 2^(s - m + 14): those above 2^-28 of the largest to half a step, and of the others all but 2^-39 each."""
    half = torch.finfo(dtype).eps / 2
    lost = tokens * 2.0 ** -39 * largest if dtype == torch.float16 else 0.0
    return attention_bound(want, size, most, dtype, dim, tokens) + half * (1 + 2 * half) * (size + want.abs()) + lost


def extend_tables(tables, lengths, counts, free, taken, page_size, tokens=None):
    """Token by token; None where something does not fit.  (tables, lengths, taken, starts, positions, slots) as lists."""
    tables = [list(map(int, row)) for row in tables]
    width = len(tables[0]) if tables else 0
    packed = tokens is not None
    if any(n < 0 or c < 0 or n + c > width * page_size or (not packed and c > 1) for n, c in zip(lengths, counts)):
        return None
    if taken < 0 or (packed and sum(counts) > tokens):
        return None
    starts, positions, slots = [], [], []
    for r, (n, c) in enumerate(zip(lengths, counts)):
        starts.append(len(positions))
        for t in range(n, n + c):
            if t % page_size == 0:
                if taken >= len(free):
                    return None
                tables[r][t // page_size] = int(free[taken])
                taken += 1
            positions.append(t)
            slots.append(tables[r][t // page_size] * page_size + t % page_size)
        if not packed and c == 0:
            positions.append(0)
            slots.append(-1)
    starts.append(len(positions))
    if packed:
        positions += [0] * (tokens - len(positions))
        slots += [-1] * (tokens - len(slots))
    return tables, [n + c for n, c in zip(lengths, counts)], taken, starts, positions, slots
