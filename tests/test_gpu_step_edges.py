"""GPU tests of calls at the edges of what windows, common prefixes, turned writes and rotations document: row starts that are not
the tensors', rows past them, results past 2^32 bytes, queries of no heads, keys that are not finite."""

import math

import pytest
import torch

from oracle import serving as oracle
from oracle import step as step_oracle
from serving_check import bytes_of, cached, cumulative, make_cache, randn
from step_check import check_paged_rows, check_rows
from test_gpu_shared import JOINED, batch, tokens
from test_gpu_turn import check, plan_of, positions_of, weight_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("form", ["shared", "window", "mixed", "packed"])
@pytest.mark.parametrize("before,behind", [(3, 0), (0, 5), (37, 130)])
def test_rows_of_no_sequence(form, before, behind):
    """Row starts that begin behind the first rows and end before the last: those rows stay as they are."""
    from fa2.packed import attention_packed
    from fa2.paged import attention_paged
    D, dtype, h_q, h_kv = 128, torch.bfloat16, 28, 4
    new, lens = ([1] * 24 + [2048], [2300 + i for i in range(24)] + [2100]) if form == "mixed" else ([1, 40, 3], [700, 640, 650])
    pages, cache, cu, seqlens, table = batch(new, lens, 576 if form == "shared" else 0, 64, h_kv, D, dtype, False)
    cu += before
    T = before + sum(new) + behind
    q, out = randn((T, h_q, D), dtype, 3), torch.full((T, h_q, D), 9.0, dtype=dtype, device="cuda")
    kw = dict(window=1900, sinks=5)
    if form == "packed":
        k, v = (randn((T, h_kv, D), dtype, i) for i in (4, 5))
        _, lse = attention_packed(q, k, v, cu, window=50, sinks=2, out=out, return_lse=True)
        of = [lambda s, t=t: t[int(cu[s]):int(cu[s + 1])].double() for t in (k, v)]
        check_rows(out, lse, q, *of, cu, dtype, window=50, sinks=2)
    elif form == "shared":
        _, lse = attention_paged(q, cache, table, cu, seqlens, shared=tokens(580), out=out, return_lse=True)
        check_paged_rows(out, lse, q, cache, pages, lens, cu, dtype, joined=JOINED)
    else:
        _, lse = attention_paged(q, cache, table, cu, seqlens, out=out, return_lse=True, **kw)
        check_paged_rows(out, lse, q, cache, pages, lens, cu, dtype, **kw)
    assert (out[:before] == 9.0).all() and (out[T - behind:] == 9.0).all()


@pytest.mark.parametrize("form", ["shared", "window"])
def test_row_starts_past_the_rows(form):
    """Row starts past the tensors' end are held to it: the sequences have the rows that there are."""
    from fa2.paged import attention_paged
    D, dtype, lens = 64, torch.float16, [700, 640, 650]
    pages, cache, cu, seqlens, table = batch([1, 1, 1], lens, 512 if form == "shared" else 0, 64, 2, D, dtype, False)
    cu = torch.tensor([0, 5, 9, 2000], dtype=torch.int32, device="cuda")
    q = randn((20, 8, D), dtype, 3)
    kw = dict(shared=tokens(512)) if form == "shared" else dict(window=90, sinks=1)
    out, lse = attention_paged(q, cache, table, cu, seqlens, return_lse=True, **kw)
    check_paged_rows(out, lse, q, cache, pages, lens, cu.clamp(max=20), dtype, joined=JOINED,
                     **({} if form == "shared" else kw))


def test_shared_results_past_32_bits():
    """150000 rows' results in float, 5 GB of workspace, in as many sequences: the same as without sharing, to the bounds of both."""
    from fa2.paged import attention_paged
    n, D, dtype, page_size, prefix, h_q, h_kv = 150000, 128, torch.bfloat16, 64, 128, 32, 8
    cache = make_cache(6, h_kv, page_size, D, dtype, False)
    table = torch.tensor([[4, 1, 0], [4, 1, 2], [4, 1, 3]], dtype=torch.int32, device="cuda").repeat(n // 3, 1)
    g = torch.Generator().manual_seed(1)
    seqlens = (prefix + 1 + torch.randint(0, 63, (n,), generator=g)).int().cuda()
    cu = torch.arange(n + 1, dtype=torch.int32, device="cuda")
    q = randn((n, h_q, D), dtype, 3)
    got, lse = attention_paged(q, cache, table, cu, seqlens, shared=tokens(prefix), return_lse=True)
    want, want_lse = attention_paged(q, cache, table, cu, seqlens, return_lse=True)
    # both are within 4 half steps of the weighted magnitudes (weights, their sum, the output) of float64, |v| <= 6; log-sum-exps
    # within 2 (D + 4) 2^-24 of a row's sum of |q_d k_d| / sqrt(D), at most 40, and (n_kv + 16) 2^-23
    assert (got.float() - want.float()).abs().max() <= 8 * 2.0 ** -8 * 6
    assert (lse - want_lse).abs().max() <= 2 * (2 * 132 * 40 * 2.0 ** -24 + 208 * 2.0 ** -23)
    for s in (0, 1, 2, 74998, 74999, n - 3, n - 2, n - 1):
        length = int(seqlens[s])
        page, row = table[s].long()[torch.arange(length, device="cuda") // page_size], torch.arange(length, device="cuda") % page_size
        one = torch.tensor([0, 1], dtype=torch.int32)
        check_rows(got[s:s + 1], lse[:, s:s + 1], q[s:s + 1], lambda _: cached(cache, "k", page, row), lambda _: cached(cache, "v", page, row),
                   one, dtype, joined=JOINED)


def test_queries_of_no_heads():
    from fa2.rotary import HeadNorm, rotary_qk
    plan, norm = plan_of(64, 3), HeadNorm(weight_of(64, 1))
    k, positions = randn((30, 2, 64), torch.float16, 1), positions_of(3, (30,), 1)
    q, got = rotary_qk(k[:, :0], k, positions, plan, k_norm=norm)
    assert q.shape == (30, 0, 64)
    check(got, k, positions, plan, norm)
    got, none = rotary_qk(k, k[:, :0], positions, plan, q_norm=norm)
    assert none.shape == (30, 0, 64)
    check(got, k, positions, plan, norm)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("normed", [False, True])
def test_turned_keys_that_are_not_finite(dtype, e4m3, normed):
    """Infinite and NaN values, zeros and the type's largest and least ones, in rows of their own."""
    from fa2.paged import cache_write
    from fa2.rotary import HeadNorm
    D, page_size, T = 64, 64, 40
    plan, norm = plan_of(32, 3), HeadNorm(weight_of(D, 2), 1e-6) if normed else None
    info = torch.finfo(dtype)
    pages = oracle.Pages([T], page_size, device="cuda")
    cu, seqlens = cumulative([T]), torch.tensor([T], dtype=torch.int32, device="cuda")
    k, v = randn((T, 2, D), dtype, 1), randn((T, 2, D), dtype, 2)
    for i, x in enumerate((math.inf, -math.inf, math.nan, info.max, info.smallest_normal * info.eps)):
        k[3 * i, 0, 7 * i] = x
        k[3 * i + 1, 1, 40 + i] = x
    k[20:24] = 0
    k[24, 0] = info.max / 2
    positions = positions_of(3, (T,), 1)
    cache = make_cache(pages.n_pages, 2, page_size, D, dtype, e4m3)
    cache_write(cache, k, v, pages.table, cu, seqlens, rotary=plan, k_norm=norm, positions=positions)
    weight, eps = norm or (None, 0.0)
    turned, tol = step_oracle.turn(k, positions, plan.freqs, False, plan.scale, plan.axes, weight, eps)
    page, row = pages.at(0, torch.arange(T, device="cuda"))
    got = cached(cache, "k", page, row)
    if e4m3:
        values, e = oracle.to_e4m3(turned, dtype)
        assert torch.equal(cache.k_scale.view(torch.uint8)[page, :, row].long(), (e + 127).long())
        want = values * torch.exp2(e.double())[..., None]
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(), want.nan_to_num())
        assert torch.equal(got.isnan(), ~turned.isfinite())
    else:
        rounded = turned.to(dtype).double()  # (sums of the largest values leave the type's range)
        assert torch.equal(got.isnan(), rounded.isnan())
        near = rounded.isfinite() & got.isfinite()
        assert ((got - turned).abs() <= tol)[near].all()
        assert (turned.abs() >= info.max * (1 - 2.0 ** -7))[~near & ~rounded.isnan()].all()
