"""Plain restatements of a step's other operators (fa2.rotary.rotary_qk, fa2.pages): float64 norms and rotations by
several axes with the error bounds their tests hold the kernels to, and pages taken and given back in Python."""

import torch

from . import serving


def norm(x, weight, eps):
    """x [..., D] in float64, every row divided by its root mean square and weighted (weight None: as it is)."""
    x = x.double()
    if weight is None:
        return x
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight.double()


def turn(x, positions, freqs, interleaved=False, scale=1.0, axes=None, weight=None, eps=0.0):
    """x [T, H, D] normalised and rotated: (result, bound), both float64. positions [T], or [axes, T] with axes.

    The bound of a kernel's value, in units of 2^-24 relative to |a cos| + |b sin|. The sum of D <= 128 squares: 8 products and
    sums of a lane, at most 2 units each if they are cut off, and 4 sums of lanes, together 20, half of that in its root; the mean
    and eps 1, the root's estimate 2 (one unit in its last place), x * r * weight 2, cos or sin, its product and the sum 3: 18, and 24 with
    what second order adds. Then the rounding to the type: half a step, which is at least half the type's least subnormal value
    (2^-25 for fp16, 2^-134 for bf16, whose least normal value is float's own: there each of float's 8 roundings on the way is off by up to 2^-150,
    with weights up to 16 together less than 2^-142)."""
    half = freqs.numel()
    angle = (positions.double()[:, None] if axes is None else positions.double()[axes.long()].t()) * freqs.double()
    cos, sin = (torch.cos(angle) * scale)[:, None], (torch.sin(angle) * scale)[:, None]
    y = norm(x, weight, eps).clone()
    i = torch.arange(half, device=x.device)
    a_at, b_at = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    a, b = y[..., a_at], y[..., b_at]
    size = y.abs()
    size[..., a_at] = a.abs() * cos.abs() + b.abs() * sin.abs()
    size[..., b_at] = b.abs() * cos.abs() + a.abs() * sin.abs()
    y[..., a_at], y[..., b_at] = a * cos - b * sin, b * cos + a * sin
    u = serving.HALF_STEP[x.dtype]
    return y, u * y.abs() * (1 + u) + 24 * serving.F32 * size + (2.0 ** -25 if x.dtype == torch.float16 else 2.0 ** -134 + 2.0 ** -142)


def release(free, count, table, first, last):
    """(free, count) after entries first[s] .. last[s] - 1 of every row of table that are pages go on top."""
    free = list(free)
    for row, a, b in zip(table, first, last):
        for page in row[max(a, 0):min(b, len(row))] if b > 0 else []:
            if 0 <= page < len(free):
                if count < len(free):
                    free[count] = page
                count = min(count + 1, len(free))
    return free, count


def extend(free, count, table, lens, new, page_size, n_tokens):
    """(count, cu, lens, positions, slots, table) of the new tokens, a page at a time."""
    count = min(max(count, 0), len(free))
    table = [list(row) for row in table]
    lens, new = [max(x, 0) for x in lens], [max(x, 0) for x in new]
    width = len(table[0])
    needs = []  # (sequence, entry)
    for s, (a, n) in enumerate(zip(lens, new)):
        needs += [(s, e) for e in range(min(-(-a // page_size), width), min(-(-(a + n) // page_size), width))]
    base = max(count - len(needs), 0)
    for i, (s, e) in enumerate(needs):
        table[s][e] = free[base + i] if base + i < count else -1
    cu, positions, slots = [0], [], []
    for row, a, n in zip(table, lens, new):
        cu.append(cu[-1] + n)
        for p in range(a, a + n):
            page = row[p // page_size] if p // page_size < width else -1
            positions.append(p)
            slots.append(page * page_size + p % page_size if 0 <= page < len(free) else -1)
    pad = n_tokens - cu[-1]
    return (base, cu, [a + n for a, n in zip(lens, new)], (positions + [-1] * pad)[:n_tokens], (slots + [-1] * pad)[:n_tokens], table)
