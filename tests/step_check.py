"""Shared by the tests of windows, common prefixes and a step's pages: attention compared with oracle/serving.py's float64
form under its derived bounds, a window included."""

import torch

from oracle import serving as oracle
from serving_check import cached


def check_rows(out, lse, q, k_of, v_of, cu, dtype, causal=True, window=None, sinks=0, sm_scale=None, joined=0):
    """out and lse (or None) of packed q, sequence by sequence; k_of(s), v_of(s) give float64 [n_kv, H_kv, D]. joined: roundings
    in float32 beside those of oracle.attention_bounds, in its unit of 2^-23 of the sum of weighted magnitudes."""
    D = q.shape[-1]
    cu = cu.tolist()
    for s in range(len(cu) - 1):
        rows = slice(cu[s], cu[s + 1])
        if cu[s] == cu[s + 1]:
            continue
        k, v = k_of(s), v_of(s)
        want, want_lse, size, big = oracle.attention(q[rows], k, v, causal, sm_scale, window, sinks)
        v_max = v.abs().nan_to_num(0, 0, 0).max().item() if v.numel() else 0.0
        tol, lse_tol = oracle.attention_bounds(want, size, big, dtype, D, k.shape[0] + joined, v_max)
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


def check_paged_rows(out, lse, q, cache, pages, lens, cu, dtype, **kw):
    """... of a paged cache (oracle.Pages), whose entries that are no page are read as page 0 (they are not seen)."""
    def tokens(which):
        def of(s):
            page, row = pages.at(s, torch.arange(lens[s], device=q.device))
            return cached(cache, which, page.clamp(min=0), row)
        return of
    check_rows(out, lse, q, tokens("k"), tokens("v"), cu, dtype, **kw)


def hide_pages(pages, lens, new, window, sinks, entry=-1):
    """A copy of the table in which the pages that no row of the call sees are no pages any more."""
    table, P = pages.table.clone(), pages.page_size
    for s, (n_kv, n) in enumerate(zip(lens, new)):
        low = max(n_kv - n - window + 1, 0) // P
        table[s, min(-(-sinks // P), low):low] = entry
    return table
