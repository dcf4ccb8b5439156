"""GPU tests of attention with a sliding window and sinks, over packed rows and over pages, against the float64 oracle under
its derived bounds."""

import math

import pytest
import torch

from oracle import serving as oracle
from serving_check import cumulative, make_cache, randn
from step_check import check_paged_rows, check_rows, hide_pages

pytestmark = pytest.mark.gpu
DTYPES = [torch.float16, torch.bfloat16]
# windows from a single key on, on tiles' borders and beside them, longer than any sequence; sinks likewise
WINDOWS = [(1, 0), (1, 1), (5, 64), (64, 0), (65, 4), (300, 70), (5000, 3)]


def packed(lens, h_q, h_kv, D, dtype, seed=0):
    T = sum(lens)
    return (randn((T, h_q, D), dtype, seed), randn((T, h_kv, D), dtype, seed + 1), randn((T, h_kv, D), dtype, seed + 2),
            cumulative(lens))


def of_rows(t, cu):
    cu = cu.tolist()
    return lambda s: t[cu[s]:cu[s + 1]].double()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [16, 32, 64, 128])
@pytest.mark.parametrize("h_q,h_kv", [(4, 4), (8, 2), (7, 1)])
def test_packed(dtype, D, h_q, h_kv):
    """Few rows (four waves that take keys in turn) and more than the GPU has CUs for (128-row tiles)."""
    from fa2.packed import attention_packed
    for lens in ([1], [130, 1, 0, 63, 64, 65], [700, 300], [129 + 11 * i for i in range(24)]):
        q, k, v, cu = packed(lens, h_q, h_kv, D, dtype, len(lens))
        for window, sinks in WINDOWS:
            out, lse = attention_packed(q, k, v, cu, window=window, sinks=sinks, return_lse=True)
            check_rows(out, lse, q, of_rows(k, cu), of_rows(v, cu), cu, dtype, window=window, sinks=sinks)


@pytest.mark.parametrize("D", [64, 128])
def test_packed_long(D):
    from fa2.packed import attention_packed
    lens = [3000, 1, 2500]
    q, k, v, cu = packed(lens, 8, 2, D, torch.bfloat16)
    for window, sinks in ((128, 4), (1000, 0), (1024, 200), (2999, 1)):
        out, lse = attention_packed(q, k, v, cu, window=window, sinks=sinks, return_lse=True, sm_scale=0.3)
        check_rows(out, lse, q, of_rows(k, cu), of_rows(v, cu), cu, torch.bfloat16, window=window, sinks=sinks, sm_scale=0.3)


def test_packed_other_keys():
    """Keys of their own lengths: rows that see no key, sequences without keys, rows behind the last sequence."""
    from fa2.packed import attention_packed
    n_q, n_kv, D, dtype = [5, 40, 7, 300], [200, 10, 0, 333], 64, torch.float16
    q, cu, cu_kv = randn((sum(n_q) + 3, 6, D), dtype, 1), cumulative(n_q), cumulative(n_kv)
    k, v = randn((sum(n_kv), 2, D), dtype, 2), randn((sum(n_kv), 2, D), dtype, 3)
    for window, sinks in WINDOWS:
        out = torch.full_like(q, 9.0)
        got, lse = attention_packed(q, k, v, cu, cu_kv, window=window, sinks=sinks, return_lse=True, out=out)
        assert got is out and (out[-3:] == 9.0).all()
        check_rows(out, lse, q, of_rows(k, cu_kv), of_rows(v, cu_kv), cu, dtype, window=window, sinks=sinks)


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("h_q", [2, 32])
def test_packed_hidden_values_do_not_matter(bad, h_q):
    """Infinite and NaN keys and values: rows that do not see them stay as they are, the others are the oracle's."""
    from fa2.packed import attention_packed
    lens, dtype, window, sinks = [600, 200], torch.bfloat16, 100, 4
    q, k, v, cu = packed(lens, h_q, 2, 64, dtype)
    clean = attention_packed(q, k, v, cu, window=window, sinks=sinks)
    v[300] = bad
    k[650] = bad
    out, lse = attention_packed(q, k, v, cu, window=window, sinks=sinks, return_lse=True)
    check_rows(out, lse if not math.isinf(bad) else None, q, of_rows(k, cu), of_rows(v, cu), cu, dtype, window=window, sinks=sinks)
    hidden = [i for i in range(800) if not (300 <= i < 400 or 650 <= i < 750)]
    assert torch.isfinite(out[hidden]).all()
    assert (out[hidden].float() - clean[hidden].float()).abs().max() < 0.05


def test_as_all_keys():
    """A window of every key there is: what attention without one gives, to the bounds of both."""
    from fa2.packed import attention_packed
    q, k, v, cu = packed([500, 20], 4, 2, 128, torch.float16)
    out = attention_packed(q, k, v, cu, window=1 << 40)
    check_rows(out, None, q, of_rows(k, cu), of_rows(v, cu), cu, torch.float16)
    assert torch.equal(attention_packed(q, k, v, cu, window=(1 << 31) - 1, sinks=1 << 50), out)


@pytest.mark.parametrize("window,sinks", [(1 << 40, 0), ((1 << 31) - 1, 3), ((1 << 31) - 20, 1 << 40)])
@pytest.mark.parametrize("h_q", [2, 24])
def test_largest_windows_of_rows_without_keys(window, sinks, h_q):
    """The largest windows there are, in row tiles that begin with rows that see no key: packed rows with fewer keys than rows, and
    sequences with fewer tokens in the cache than rows."""
    from fa2.packed import attention_packed
    from fa2.paged import attention_paged
    n_q, n_kv, D, dtype = [40, 300, 7, 900], [10, 131, 0, 899], 64, torch.bfloat16
    q, cu, cu_kv = randn((sum(n_q), h_q, D), dtype, 1), cumulative(n_q), cumulative(n_kv)
    k, v = randn((sum(n_kv), 2, D), dtype, 2), randn((sum(n_kv), 2, D), dtype, 3)
    out, lse = attention_packed(q, k, v, cu, cu_kv, window=window, sinks=sinks, return_lse=True)
    check_rows(out, lse, q, of_rows(k, cu_kv), of_rows(v, cu_kv), cu, dtype, window=window, sinks=sinks)
    pages = oracle.Pages(n_kv, 16, seed=1, device="cuda")
    cache = make_cache(pages.n_pages, 2, 16, D, dtype, False, 5, "hnd")
    seqlens = torch.tensor(n_kv, dtype=torch.int32, device="cuda")
    out, lse = attention_paged(q, cache, pages.table, cu, seqlens, window=window, sinks=sinks, return_lse=True)
    check_paged_rows(out, lse, q, cache, pages, n_kv, cu, dtype, window=window, sinks=sinks)


# ------------------------------------------------------------------------------------------
# pages
# ------------------------------------------------------------------------------------------

STEPS = [([1], [1]), ([1, 1, 1, 1], [1, 77, 900, 64]), ([5, 0, 33, 1, 128], [5, 9, 700, 1, 400]),
         ([1] * 40, [1 + 37 * i for i in range(40)]), ([200, 1, 1], [1500, 2000, 3])]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("D,page_size", [(16, 64), (32, 32), (64, 16), (128, 16), (128, 128)])
@pytest.mark.parametrize("h_q,h_kv", [(2, 2), (8, 2), (7, 1)])
def test_paged(dtype, e4m3, D, page_size, h_q, h_kv):
    """Pages that no row sees are no pages (a negative entry, one far past the cache, a page of NaN); wide tables, whose
    sequences' keys several workgroups share, as well."""
    from fa2.paged import attention_paged
    for seed, (new, lens) in enumerate(STEPS):
        pages = oracle.Pages(lens, page_size, seed=seed, device="cuda")
        cache = make_cache(pages.n_pages, h_kv, page_size, D, dtype, e4m3, seed, ("hnd", "nhd")[seed % 2])
        cu, seqlens = cumulative(new), torch.tensor(lens, dtype=torch.int32, device="cuda")
        q = randn((sum(new), h_q, D), dtype, seed)
        for window, sinks in ((1, 0), (17, 1), (64, 0), (130, 33), (600, 5), (5000, 0)):
            for entry, columns in ((-1, 0), (1 << 30, 5000 // page_size)):
                table = hide_pages(pages, lens, new, window, sinks, entry)
                table = torch.nn.functional.pad(table, (0, columns), value=-7)
                out, lse = attention_paged(q, cache, table, cu, seqlens, window=window, sinks=sinks, return_lse=True)
                check_paged_rows(out, lse, q, cache, pages, lens, cu, dtype, window=window, sinks=sinks)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("dtype,D,page_size", [(torch.bfloat16, 128, 32), (torch.float16, 64, 16), (torch.float16, 128, 64)])
@pytest.mark.parametrize("new,lens", [([1, 1], [9000, 20]), ([1], [30000]), ([300, 1, 1, 64], [5000, 3000, 1, 2100]), ([700], [9001])])
@pytest.mark.parametrize("window,sinks", [(4096, 4), (2500, 0), (1, 3000)])
def test_paged_long(e4m3, dtype, D, page_size, new, lens, window, sinks):
    from fa2.paged import attention_paged
    pages = oracle.Pages(lens, page_size, device="cuda")
    cache = make_cache(pages.n_pages, 2, page_size, D, dtype, e4m3)
    cu, seqlens = cumulative(new), torch.tensor(lens, dtype=torch.int32, device="cuda")
    q = randn((sum(new), 8, D), dtype, 3)
    table = hide_pages(pages, lens, new, window, sinks)
    out, lse = attention_paged(q, cache, table, cu, seqlens, window=window, sinks=sinks, return_lse=True)
    check_paged_rows(out, lse, q, cache, pages, lens, cu, dtype, window=window, sinks=sinks)


def test_paged_freed_pages_hold_anything():
    """NaN in freed pages, and in the tokens of seen pages that no row sees: nothing of them reaches a row."""
    from fa2.paged import attention_paged
    page_size, D, dtype, window, sinks = 16, 64, torch.float16, 100, 20
    new, lens = [1, 40], [700, 800]
    pages = oracle.Pages(lens, page_size, device="cuda")
    cache = make_cache(pages.n_pages, 2, page_size, D, dtype, False)
    q, cu = randn((41, 8, D), dtype, 1), cumulative(new)
    seqlens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    want = attention_paged(q, cache, pages.table, cu, seqlens, window=window, sinks=sinks)
    for s in range(2):
        hidden = torch.arange(sinks, lens[s] - new[s] - window + 1, device="cuda")
        page, row = pages.at(s, hidden)
        cache.k[page, :, row] = math.nan
        cache.v[page, :, row] = math.nan
    got = attention_paged(q, cache, pages.table, cu, seqlens, window=window, sinks=sinks)
    check_paged_rows(got, None, q, cache, pages, lens, cu, dtype, window=window, sinks=sinks)
    assert (got.float() - want.float()).abs().max() < 0.01


def test_paged_page_outside_the_cache():
    """A seen page that is none: its rows are NaN, other sequences' are not."""
    from fa2.paged import attention_paged
    page_size, D, dtype = 16, 64, torch.bfloat16
    new, lens = [1, 1], [300, 300]
    pages = oracle.Pages(lens, page_size, device="cuda")
    cache = make_cache(pages.n_pages, 2, page_size, D, dtype, False)
    table = pages.table.clone()
    table[0, 17] = 1 << 20  # tokens 272 .. 287
    out = attention_paged(randn((2, 4, D), dtype, 1), cache, table, cumulative(new),
                          torch.tensor(lens, dtype=torch.int32, device="cuda"), window=40)
    assert out[0].isnan().all() and torch.isfinite(out[1]).all()


def test_graph_follows_lengths():
    """A captured call on tensors that change between replays, checked at each."""
    from fa2.paged import attention_paged
    page_size, D, dtype, window, sinks = 16, 128, torch.bfloat16, 200, 8
    longest = [2000, 1200, 900]
    pages = oracle.Pages(longest, page_size, device="cuda")
    cache = make_cache(pages.n_pages, 2, page_size, D, dtype, False)
    q, cu = randn((3, 8, D), dtype, 1), cumulative([1, 1, 1])
    seqlens = torch.tensor([10, 20, 30], dtype=torch.int32, device="cuda")
    attention_paged(q, cache, pages.table, cu, seqlens, window=window, sinks=sinks)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = attention_paged(q, cache, pages.table, cu, seqlens, window=window, sinks=sinks, return_lse=True)
    for lens in ([10, 20, 30], [2000, 1, 900], [1999, 1200, 201]):
        seqlens.copy_(torch.tensor(lens, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        check_paged_rows(out, lse, q, cache, pages, lens, cu, dtype, window=window, sinks=sinks)


def test_layouts_and_both_ways_to_the_kernels(monkeypatch):
    """Odd storage, an out of its own, q itself, and the Python way: the same bits."""
    from fa2 import _lib
    from fa2.packed import attention_packed
    q, k, v, cu = packed([300, 45], 8, 2, 64, torch.bfloat16)
    want = attention_packed(q, k, v, cu, window=50, sinks=3)
    wide = torch.zeros(345, 8, 128, dtype=q.dtype, device="cuda")[..., ::2].copy_(q)
    assert torch.equal(attention_packed(wide, k, v, cu, window=50, sinks=3), want)
    turned = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(attention_packed(turned, k, v, cu, window=50, sinks=3), want)
    mine = q.clone()
    assert attention_packed(mine, k, v, cu, window=50, sinks=3, out=mine) is mine and torch.equal(mine, want)
    monkeypatch.setattr(_lib, "native", None)
    assert torch.equal(attention_packed(q, k, v, cu, window=50, sinks=3), want)


def test_streams_at_once():
    """Calls of different sizes on two streams at once: each as alone."""
    from fa2.paged import attention_paged
    page_size, D, dtype = 16, 64, torch.float16
    calls = []
    for seed, (new, lens) in enumerate((([1] * 8, [3000] * 8), ([256], [2500]))):
        pages = oracle.Pages(lens, page_size, seed=seed, device="cuda")
        cache = make_cache(pages.n_pages, 2, page_size, D, dtype, False, seed)
        args = (randn((sum(new), 8, D), dtype, seed), cache, pages.table, cumulative(new),
                torch.tensor(lens, dtype=torch.int32, device="cuda"))
        calls.append((args, attention_paged(*args, window=1800, sinks=5)))
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    results = [[] for _ in calls]
    for _ in range(5):
        for (args, _), stream, got in zip(calls, streams, results):
            with torch.cuda.stream(stream):
                got.append(attention_paged(*args, window=1800, sinks=5))
    torch.cuda.synchronize()
    for (_, want), got in zip(calls, results):
        assert all(torch.equal(x, want) for x in got)
