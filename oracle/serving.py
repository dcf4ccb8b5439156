"""Plain float64 restatements of the serving operators (fa2.rotary, fa2.paged, fa2.packed), and the error
bounds that their tests hold the kernels to. One sequence, one head at a time where that is the clearest form;
runs on the device its tensors are on.
"""

import math

import torch

# half a step of rounding, relative to the value
HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
F32 = 2.0 ** -24


def rotate(x, positions, freqs, interleaved=False, scale=1.0):
    """x [..., T, D] (float64 result): the first 2 len(freqs) values rotated by positions [T] * freqs."""
    x = x.double().clone()
    half = freqs.numel()
    angle = positions.double()[:, None] * freqs.double()
    cos, sin = torch.cos(angle) * scale, torch.sin(angle) * scale
    i = torch.arange(half, device=x.device)
    a_at, b_at = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    a, b = x[..., a_at], x[..., b_at]
    x[..., a_at], x[..., b_at] = a * cos - b * sin, b * cos + a * sin
    return x


def to_e4m3(x, dtype):
    """Rows x [..., D] (float64) as the cache holds them: (e4m3 values as float64, exponents e), x ~ values * 2^e.

    e is the least integer with max|x| <= 448 * 2^e over the finite values, at least -126 and at most 8 (fp16) or 120
    (bf16), where magnitudes end at 240. e4m3: exponents -6 .. 8, three bits of mantissa, ties to even.
    """
    finite = torch.where(x.isfinite(), x.abs(), torch.zeros_like(x))
    top = finite.amax(-1, keepdim=True)
    m, k = torch.frexp(top / 448.0)  # 448 = 7 * 2^6: exact where it decides
    e = torch.where(m == 0.5, k - 1, k)
    most = 8 if dtype == torch.float16 else 120
    e = torch.where(top == 0, torch.full_like(e, -126), e).clamp(-126, most)
    y = x * torch.exp2(-e.double())
    limit = torch.where(e == most, 240.0, 448.0).double()
    y = torch.maximum(torch.minimum(y, limit), -limit)
    p = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -9))).clamp(min=-6)
    step = torch.exp2(p - 3)
    y = torch.round(y / step) * step
    return torch.where(x.isfinite(), y, torch.full_like(y, math.nan)), e[..., 0]


def attention(q, k, v, causal, sm_scale=None):
    """One sequence: q [n, H_q, D] over k, v [m, H_kv, D], the causal mask aligned at the end. Float64 out
    [n, H_q, D], lse [H_q, n], and for the bounds: the weights' sum of |v|, [n, H_q, D], and the largest sum of
    |q_d k_d| * sm_scale of a row, [n, H_q, 1]. Values of keys that a row does not see do not enter its result."""
    n, h_q, D = q.shape
    m, h_kv = k.shape[:2]
    sm_scale = D ** -0.5 if sm_scale is None else sm_scale
    out = torch.zeros(n, h_q, D, dtype=torch.float64, device=q.device)
    size = torch.zeros_like(out)
    lse = torch.full((h_q, n), -math.inf, dtype=torch.float64, device=q.device)
    big = torch.zeros(n, h_q, 1, dtype=torch.float64, device=q.device)
    if n == 0 or m == 0:
        return out, lse, size, big
    see = torch.ones(n, m, dtype=torch.bool, device=q.device)
    if causal:
        see = torch.arange(m, device=q.device) <= torch.arange(n, device=q.device)[:, None] + (m - n)
    some = see.any(1)
    group = h_q // h_kv
    for h in range(h_kv):  # the group of query heads of a KV head at once
        heads = slice(h * group, (h + 1) * group)
        qh, kt, vh = q[:, heads].double().reshape(n * group, D), k[:, h].double().t().contiguous(), v[:, h].double()
        sees = see.repeat_interleave(group, 0)
        any_ = some.repeat_interleave(group)
        s = (qh @ kt * sm_scale).masked_fill(~sees, -math.inf)
        w = torch.where(sees, torch.softmax(s, 1), 0.0)
        fine = vh.isfinite().all(1)
        o = w[:, fine] @ vh[fine]
        for j in (~fine).nonzero()[:, 0].tolist():  # infinite and NaN values: only where they are seen
            o += torch.where(sees[:, j, None], w[:, j, None] * vh[j], 0.0)
        out[:, heads] = torch.where(any_[:, None], o, 0.0).view(n, group, D)
        size[:, heads] = torch.where(any_[:, None], w[:, fine] @ vh[fine].abs(), 0.0).view(n, group, D)
        lse[heads] = torch.where(any_, torch.logsumexp(s, 1), -math.inf).view(n, group).t()
        score = (qh.abs() @ kt.abs()).masked_fill(~sees, 0.0).nan_to_num(0, 0, 0).amax(1) * sm_scale
        big[:, heads, 0] = score.view(n, group)
    return out, lse, size, big


def attention_bounds(out, size, big, dtype, head_dim, n_kv, v_max):
    """How far a kernel's (out, lse) may be off, elementwise. With u half a step of the 16-bit type: each weight
    is rounded to it (u in the sum of products, u in the sum it is divided by), and the output once (u). A
    score of float32 sums of exact products is off by (D + 4) 2^-24 of its sum of magnitudes, the softmax by
    twice that, its exp2, scale and sums of n_kv terms by (n_kv + 16) 2^-23. fp16 weights below 2^-14 of the
    row's reference are rounded to 2^-25 absolutely, whatever their size."""
    u = HALF_STEP[dtype]
    score = 2 * (head_dim + 4) * F32 * big
    tol = size * (2 * u * (1 + u) + score + (n_kv + 16) * 2 * F32) + u * out.abs() * (1 + 4 * u) + 2.0 ** -30
    if dtype == torch.float16:
        tol = tol + n_kv * 2.0 ** -25 * v_max + 2.0 ** -25
    return tol, (score[..., 0].t() + (n_kv + 16) * 2 * F32)


class Pages:
    """Sequences of given lengths spread over a cache's pages in a shuffled order: block table, and where each
    token lies. Entries of the table past a sequence's pages are -1."""

    def __init__(self, lens, page_size, n_pages=None, extra=2, seed=0, device="cpu", first_page=0):
        g = torch.Generator().manual_seed(seed)
        need = [-(-n // page_size) for n in lens]
        self.n_pages = n_pages or (first_page + sum(need) + extra)
        order = (torch.randperm(self.n_pages - first_page, generator=g)[:sum(need)] + first_page).to(torch.int32)
        self.table = torch.full((len(lens), max(need + [0]) + 1), -1, dtype=torch.int32)
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = order[at:at + n]
            at += n
        self.page_size = page_size
        self.table = self.table.to(device)

    def at(self, s, positions):
        """(page, row) of sequence s's tokens at `positions`"""
        return self.table[s].long()[positions // self.page_size], positions % self.page_size
