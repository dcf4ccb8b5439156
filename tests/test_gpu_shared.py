"""GPU tests of attention_paged for a batch that shares a prefix, against the float64 oracle over every sequence's own
tokens."""

import math

import pytest
import torch

from oracle import serving as oracle
from serving_check import cumulative, make_cache, randn
from step_check import check_paged_rows

pytestmark = pytest.mark.gpu
DTYPES = [torch.float16, torch.bfloat16]
# Joining the two parts of a row: two exponentials, four products, two sums and an inverse in float32 at most, half a unit of 2^-23
# each
JOINED = 8


def batch(new, lens, prefix, page_size, h_kv, D, dtype, e4m3, seed=0, storage="hnd"):
    """Sequences whose first prefix // page_size pages are the same: (pages, cache, cu, seqlens, table). In the table, which is what
    the call gets, only the first sequence with new tokens names them."""
    pages = oracle.Pages(lens, page_size, seed=seed, device="cuda")
    common = prefix // page_size
    having = [s for s, n in enumerate(new) if n]
    longest = max(having, key=lambda s: lens[s])
    for s in having:
        assert lens[s] >= common * page_size
        pages.table[s, :common] = pages.table[longest, :common].clone()
    table = pages.table.clone()
    for s in having[1:]:
        table[s, :common] = -3
    cache = make_cache(pages.n_pages, h_kv, page_size, D, dtype, e4m3, seed, storage)
    return pages, cache, cumulative(new), torch.tensor(lens, dtype=torch.int32, device="cuda"), table


def tokens(n):
    return torch.tensor([n], dtype=torch.int32, device="cuda")


# (new tokens, tokens in the cache, shared): a row, a few rows (four waves that take keys in turn), more than 32 rows; a prefix of no
# whole page, of one, of many; sequences with hardly more than the prefix, and without new tokens
CASES = [([1], [100], 70), ([1, 1], [300, 257], 256), ([1, 1, 1], [129, 128 + 5, 400], 128), ([3, 0, 2, 17], [500, 0, 403, 450], 399),
         ([1] * 40, [600 + 7 * i for i in range(40)], 555), ([5] * 16, [1030 + i for i in range(16)], 1024), ([130, 1], [800, 700], 640)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("D,page_size", [(16, 64), (32, 32), (64, 16), (128, 16), (128, 128)])
@pytest.mark.parametrize("h_q,h_kv", [(2, 2), (8, 2), (7, 1)])
def test_shared(dtype, e4m3, D, page_size, h_q, h_kv):
    """... with tables wide enough that several workgroups share the keys, too."""
    from fa2.paged import attention_paged
    for seed, (new, lens, prefix) in enumerate(CASES):
        pages, cache, cu, seqlens, table = batch(new, lens, prefix, page_size, h_kv, D, dtype, e4m3, seed, ("hnd", "nhd")[seed % 2])
        q = randn((sum(new) + 2, h_q, D), dtype, seed)
        for columns in (0, 4000 // page_size):
            wide = torch.nn.functional.pad(table, (0, columns), value=-7)
            out = torch.full_like(q, 9.0)
            _, lse = attention_paged(q, cache, wide, cu, seqlens, shared=tokens(prefix), return_lse=True, out=out)
            assert (out[-2:] == 9.0).all()
            check_paged_rows(out, lse, q, cache, pages, lens, cu, dtype, joined=JOINED)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("dtype,D,page_size", [(torch.bfloat16, 128, 32), (torch.float16, 64, 16), (torch.float16, 128, 64)])
@pytest.mark.parametrize("new,lens,prefix", [([1, 1], [9000, 8300], 8192), ([1] * 64, [4100 + 10 * i for i in range(64)], 4099),
                                             ([4] * 9, [12000 + i * i for i in range(9)], 11990), ([300, 1, 64], [3000, 2700, 2800], 2650)])
def test_shared_long(e4m3, dtype, D, page_size, new, lens, prefix):
    from fa2.paged import attention_paged
    pages, cache, cu, seqlens, table = batch(new, lens, prefix, page_size, 2, D, dtype, e4m3)
    q = randn((sum(new), 8, D), dtype, 3)
    out, lse = attention_paged(q, cache, table, cu, seqlens, shared=tokens(prefix), return_lse=True)
    check_paged_rows(out, lse, q, cache, pages, lens, cu, dtype, joined=JOINED)
    out = attention_paged(q, cache, table, cu, seqlens, shared=tokens(prefix), causal=False, sm_scale=0.05)
    check_paged_rows(out, None, q, cache, pages, lens, cu, dtype, causal=False, sm_scale=0.05, joined=JOINED)


def test_as_much_as_all_rows_see():
    """A number past what every sequence has before its new tokens counts as that, and a negative one as none; the
    first sequences may have no new tokens and no pages."""
    from fa2.paged import attention_paged
    page_size, D, dtype = 16, 64, torch.bfloat16
    new, lens = [0, 2, 5, 1], [0, 300, 290, 500]
    pages, cache, cu, seqlens, table = batch(new, lens, 285, page_size, 2, D, dtype, False)
    q = randn((8, 8, D), dtype, 1)
    for n in (285, 286, 290, 1000, (1 << 31) - 1):  # 285 tokens lie before every new one: 17 whole pages
        out = attention_paged(q, cache, table, cu, seqlens, shared=tokens(n))
        check_paged_rows(out, None, q, cache, pages, lens, cu, dtype, joined=JOINED)
    for n in (0, -5, 15, 16, 40):  # ... (here every sequence's table names the pages that are not common)
        out = attention_paged(q, cache, pages.table, cu, seqlens, shared=tokens(n))
        check_paged_rows(out, None, q, cache, pages, lens, cu, dtype, joined=JOINED)


def test_sequences_shorter_than_their_rows():
    """More new rows than tokens in the cache: nothing is common, rows before the start see no key."""
    from fa2.paged import attention_paged
    page_size, D, dtype = 16, 64, torch.float16
    new, lens = [4, 1], [2, 200]
    pages = oracle.Pages(lens, page_size, device="cuda")
    cache = make_cache(pages.n_pages, 2, page_size, D, dtype, False)
    cu, seqlens, q = cumulative(new), torch.tensor(lens, dtype=torch.int32, device="cuda"), randn((5, 4, D), dtype, 1)
    out, lse = attention_paged(q, cache, pages.table, cu, seqlens, shared=tokens(100), return_lse=True)
    check_paged_rows(out, lse, q, cache, pages, lens, cu, dtype, joined=JOINED)
    assert (out[:2] == 0).all() and (lse[:, :2] == -math.inf).all()


@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("bad", [math.inf, math.nan])
@pytest.mark.parametrize("where", [5, 270])  # in the prefix, behind it
def test_not_finite(which, bad, where):
    """An infinite or NaN value in a token: the rows that see it, of one sequence or of all, and no others."""
    from fa2.paged import attention_paged
    page_size, D, dtype = 16, 64, torch.bfloat16
    new, lens = [1, 3, 1], [300, 280, 400]
    pages, cache, cu, seqlens, table = batch(new, lens, 256, page_size, 2, D, dtype, False)
    page, row = pages.at(1, torch.tensor([where], device="cuda"))
    getattr(cache, which)[page, :, row] = bad
    q = randn((5, 8, D), dtype, 1)
    for columns in (0, 200):
        wide = torch.nn.functional.pad(table, (0, columns), value=-7)
        out, lse = attention_paged(q, cache, wide, cu, seqlens, shared=tokens(256), return_lse=True)
        lse = None if which == "k" and math.isinf(bad) else lse  # (an infinite score's is infinite, a NaN one's NaN)
        check_paged_rows(out, lse, q, cache, pages, lens, cu, dtype, joined=JOINED)


@pytest.mark.parametrize("columns", [0, 300])
def test_page_outside_the_cache(columns):
    """In the prefix, all rows are NaN; behind it, those of its sequence."""
    from fa2.paged import attention_paged
    page_size, D, dtype = 16, 64, torch.float16
    new, lens = [1] * 20, [400] * 20
    pages, cache, cu, seqlens, table = batch(new, lens, 256, page_size, 2, D, dtype, False)
    q = randn((20, 8, D), dtype, 1)
    table = torch.nn.functional.pad(table, (0, columns), value=-7)
    own = table.clone()
    own[7, 20] = pages.n_pages
    out, lse = attention_paged(q, cache, own, cu, seqlens, shared=tokens(256), return_lse=True)
    assert out[7].isnan().all() and lse[:, 7].isnan().all()
    rest = [s for s in range(20) if s != 7]
    assert torch.isfinite(out[rest]).all() and torch.isfinite(lse[:, rest]).all()
    table[0, 3] = -1
    out, lse = attention_paged(q, cache, table, cu, seqlens, shared=tokens(256), return_lse=True)
    assert out.isnan().all() and lse.isnan().all()


def test_graph_follows_lengths_and_prefix():
    from fa2.paged import attention_paged
    page_size, D, dtype = 16, 128, torch.bfloat16
    lens = [2000, 1900, 2100]
    pages, cache, cu, seqlens, table = batch([1, 1, 1], lens, 1800, page_size, 2, D, dtype, False)
    q, n = randn((3, 8, D), dtype, 1), tokens(1800)
    attention_paged(q, cache, table, cu, seqlens, shared=n)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = attention_paged(q, cache, pages.table, cu, seqlens, shared=n, return_lse=True)
    for now, prefix in ((lens, 1800), ([1805, 1900, 2100], 1600), ([1900, 1801, 1850], 0), (lens, 1800)):
        seqlens.copy_(torch.tensor(now, dtype=torch.int32))
        n.fill_(prefix)
        graph.replay()
        torch.cuda.synchronize()
        check_paged_rows(out, lse, q, cache, pages, now, cu, dtype, joined=JOINED)
        assert torch.equal(attention_paged(q, cache, pages.table, cu, seqlens, shared=n), out)


def test_streams_at_once_and_both_ways_to_the_kernels(monkeypatch):
    from fa2 import _lib
    from fa2.paged import attention_paged
    calls = []
    for seed, (new, lens, prefix) in enumerate((([1] * 30, [3000 + i for i in range(30)], 2900), ([5] * 8, [1500] * 8, 1400))):
        pages, cache, cu, seqlens, table = batch(new, lens, prefix, 16, 2, 64, torch.float16, False, seed)
        args = (randn((sum(new), 8, 64), torch.float16, seed), cache, table, cu, seqlens)
        calls.append((args, tokens(prefix), attention_paged(*args, shared=tokens(prefix))))
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    results = [[] for _ in calls]
    for _ in range(5):
        for (args, n, _), stream, got in zip(calls, streams, results):
            with torch.cuda.stream(stream):
                got.append(attention_paged(*args, shared=n))
    torch.cuda.synchronize()
    for (_, _, want), got in zip(calls, results):
        assert all(torch.equal(x, want) for x in got)
    monkeypatch.setattr(_lib, "native", None)
    for args, n, want in calls:
        assert torch.equal(attention_paged(*args, shared=n), want)
        mine = args[0].clone()
        assert attention_paged(mine, *args[1:], shared=n, out=mine) is mine and torch.equal(mine, want)
