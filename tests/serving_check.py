"""Shared by the tests of the serving operators: packed inputs, caches in every layout, and the comparison of
attention with oracle/serving.py's float64 form under its derived bounds."""

import torch

from oracle import serving as oracle

CACHES = ("16bit", "e4m3")


def cumulative(lens, device="cuda"):
    cu = torch.zeros(len(lens) + 1, dtype=torch.int32)
    cu[1:] = torch.tensor(lens, dtype=torch.int64).cumsum(0)
    return cu.to(device)


def randn(shape, dtype, seed, device="cuda", scale=1.0):
    g = torch.Generator(device=device).manual_seed(seed)
    return (torch.randn(shape, device=device, generator=g) * scale).to(dtype)


def make_cache(pages, h_kv, page_size, D, dtype, e4m3, seed=0, storage="hnd", device="cuda"):
    """A KVCache of random values, and of NaN wherever a test leaves them: storage "nhd" is
    [pages, page_size, H_kv, D] seen through transpose."""
    from fa2.paged import KVCache

    shape = (pages, h_kv, page_size, D) if storage == "hnd" else (pages, page_size, h_kv, D)
    tensors = []
    for i in range(2):
        x = randn(shape, torch.float32, seed + i, device)
        if not e4m3:
            t = x.to(dtype)
            tensors.append((t if storage == "hnd" else t.transpose(1, 2), None))
            continue
        values, e = oracle.to_e4m3(x.double(), dtype)
        t = values.float().to(torch.float8_e4m3fn)
        e = (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)
        tensors.append((t, e) if storage == "hnd" else (t.transpose(1, 2), e.transpose(1, 2)))
    return KVCache(tensors[0][0], tensors[1][0], tensors[0][1], tensors[1][1])


def bytes_of(t):
    """t's bits, for comparison and assignment by index (8-bit floats have neither)"""
    return t.view(torch.uint8) if t.element_size() == 1 else t


def cached(cache, which, page, row):
    """float64 values [n, H_kv, D] of the cache's k or v at (page, row)"""
    t, scale = getattr(cache, which), getattr(cache, which + "_scale")
    x = bytes_of(t)[page, :, row]
    if scale is None:
        return x.double()
    e = scale.view(torch.uint8)[page, :, row].double() - 127
    return x.view(torch.float8_e4m3fn).double() * torch.exp2(e)[..., None]


def check_attention(out, lse, q, k_of, v_of, cu, causal, dtype, sm_scale=None):
    """out and lse (or None) of packed q against float64, sequence by sequence; k_of(s), v_of(s) give float64
    [n_kv, H_kv, D]."""
    D = q.shape[-1]
    cu = cu.tolist()
    for s in range(len(cu) - 1):
        rows = slice(cu[s], cu[s + 1])
        if cu[s] == cu[s + 1]:
            continue
        k, v = k_of(s), v_of(s)
        want, want_lse, size, big = oracle.attention(q[rows], k, v, causal, sm_scale)
        v_max = v.abs().nan_to_num(0, 0, 0).max().item() if v.numel() else 0.0
        tol, lse_tol = oracle.attention_bounds(want, size, big, dtype, D, k.shape[0], v_max)
        got = out[rows].double()
        assert torch.equal(got.isnan(), want.isnan()), f"sequence {s}: NaN in other places"
        assert torch.equal(got.isinf(), want.isinf()), f"sequence {s}: infinities in other places"
        fine = want.isfinite()
        off = ((got - want).abs() / tol)[fine]
        assert off.numel() == 0 or off.max().item() <= 1.0, f"sequence {s}: {off.max().item():.2f} of the bound"
        if lse is not None:
            got_lse = lse[:, rows].double()
            assert torch.equal(got_lse.isfinite(), want_lse.isfinite()), f"sequence {s}: lse"
            assert torch.equal(got_lse.isnan(), want_lse.isnan()), f"sequence {s}: lse NaN"
            ok = want_lse.isfinite()
            off = ((got_lse - want_lse).abs() / (lse_tol + 4 * oracle.F32 * (1 + want_lse.abs())))[ok]
            assert off.numel() == 0 or off.max().item() <= 1.0, f"sequence {s}: lse {off.max().item():.2f} of the bound"
