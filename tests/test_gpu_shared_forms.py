"""GPU tests of attention behind a common prefix in the forms that its plan chooses: 32- or 128-row workgroups for the prefix and
for the keys behind it, tiles that the shares cut, batches of more sequences than a wave holds."""

import math

import pytest
import torch

from serving_check import randn
from step_check import check_paged_rows
from test_gpu_shared import DTYPES, JOINED, batch, tokens

pytestmark = pytest.mark.gpu


def many(n, rows, shortest, prefix, seed):
    """n sequences with `rows` new tokens and lengths of their own, the shortest one just behind the prefix: (new, lens)"""
    g = torch.Generator().manual_seed(seed)
    lens = (prefix + 40 + torch.randint(0, 90, (n,), generator=g)).tolist()
    lens[shortest] = prefix + rows + 3
    return [rows] * n, lens


@pytest.mark.parametrize("dtype,e4m3", [(torch.float16, False), (torch.bfloat16, False), (torch.bfloat16, True)])
@pytest.mark.parametrize("D,h_q,h_kv", [(128, 8, 2), (64, 7, 1), (16, 3, 3)])
@pytest.mark.parametrize("rows", [1, 3, 40])
@pytest.mark.parametrize("n,shortest", [(65, 64), (130, 100), (257, 256)])
def test_more_sequences_than_a_wave_holds(dtype, e4m3, D, h_q, h_kv, rows, n, shortest):
    """The least length past the first 64 sequences, which the number of shared tokens exceeds: only what all have in front of
    their own rows is common."""
    from fa2.paged import attention_paged
    page_size, prefix = 64, 448
    new, lens = many(n, rows, shortest, prefix, n + rows)
    pages, cache, cu, seqlens, table = batch(new, lens, prefix, page_size, h_kv, D, dtype, e4m3)
    q = randn((sum(new) + 1, h_q, D), dtype, 3)
    for count in (prefix, 10 ** 6):
        out = torch.full_like(q, 9.0)
        _, lse = attention_paged(q, cache, table, cu, seqlens, shared=tokens(count), return_lse=True, out=out)
        assert (out[-1] == 9.0).all()
        check_paged_rows(out, lse, q, cache, pages, lens, cu, dtype, joined=JOINED)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("n,empty", [(130, 64), (200, 129), (257, 256)])
def test_first_rows_in_a_later_block(e4m3, n, empty):
    """The first 64, 129 or 256 sequences have no new tokens: the prefix's pages are those of a later one. One of those behind it has
    none either, and one fewer tokens than the others."""
    from fa2.paged import attention_paged
    page_size, prefix, D, dtype = 32, 256, 64, torch.bfloat16
    new, lens = many(n, 1, n - 1, prefix, n)
    new[:empty] = [0] * empty
    if n > empty + 3:
        new[empty + 2], new[empty + 3] = 0, 5
    lens[0], lens[empty - 1] = 0, 7
    pages, cache, cu, seqlens, table = batch(new, lens, prefix, page_size, 2, D, dtype, e4m3)
    q = randn((sum(new), 8, D), dtype, 3)
    out, lse = attention_paged(q, cache, table, cu, seqlens, shared=tokens(prefix + 5), return_lse=True)
    check_paged_rows(out, lse, q, cache, pages, lens, cu, dtype, joined=JOINED)


def test_long_keys_of_their_own_in_many_sequences():
    """Shares of the keys behind the prefix that end inside tiles, in blocks of sequences behind the first."""
    from fa2.paged import attention_paged
    page_size, prefix, D, dtype = 64, 320, 128, torch.bfloat16
    new, lens = [1] * 140, [prefix + 5 + (3000 if i % 45 == 40 else 60) for i in range(140)]
    for rows in (1, 2):
        pages, cache, cu, seqlens, table = batch([n * rows for n in new], lens, prefix, page_size, 1, D, dtype, False, rows)
        q = randn((140 * rows, 4, D), dtype, rows)
        out, lse = attention_paged(q, cache, table, cu, seqlens, shared=tokens(prefix), return_lse=True)
        check_paged_rows(out, lse, q, cache, pages, lens, cu, dtype, joined=JOINED)


# Rows of a KV head (4 query heads each): at most 32 in all; at most 32 a sequence; more. The prefix is cut in many pieces, and
# what lies behind it where one sequence has most of it.
FORMS = [([1, 3, 1], [4200, 4116, 7000]), ([5] * 9, [4200 + i for i in range(8)] + [9000]), ([60, 1, 44], [4300, 4200, 6000])]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("D,page_size", [(16, 64), (32, 32), (64, 16), (128, 128)])
@pytest.mark.parametrize("new,lens", FORMS)
def test_cut_tiles(dtype, e4m3, D, page_size, new, lens):
    from fa2.paged import attention_paged
    prefix = 4100
    pages, cache, cu, seqlens, table = batch(new, lens, prefix, page_size, 2, D, dtype, e4m3)
    q = randn((sum(new), 8, D), dtype, 3)
    for causal in (True, False):
        out, lse = attention_paged(q, cache, table, cu, seqlens, shared=tokens(prefix), causal=causal, return_lse=True)
        check_paged_rows(out, lse, q, cache, pages, lens, cu, dtype, causal=causal, joined=JOINED)


@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("where", [5, 2100, 4150])  # in the prefix, in a later piece of it, behind it
@pytest.mark.parametrize("new,lens", FORMS)
def test_not_finite(which, bad, where, new, lens):
    """An infinite or NaN value in a token: the rows that see it, of one sequence or of all, and no others."""
    from fa2.paged import attention_paged
    page_size, D, dtype, prefix = 16, 64, torch.bfloat16, 4096
    pages, cache, cu, seqlens, table = batch(new, lens, prefix, page_size, 2, D, dtype, False)
    page, row = pages.at(2, torch.tensor([where], device="cuda"))
    getattr(cache, which)[page, :, row] = bad
    q = randn((sum(new), 8, D), dtype, 1)
    out, lse = attention_paged(q, cache, table, cu, seqlens, shared=tokens(prefix), return_lse=True)
    lse = None if which == "k" and math.isinf(bad) else lse  # (an infinite score's is infinite, a NaN one's NaN)
    check_paged_rows(out, lse, q, cache, pages, lens, cu, dtype, joined=JOINED)


@pytest.mark.parametrize("entry", [-1, 1 << 30])
@pytest.mark.parametrize("new,lens", FORMS)
def test_page_outside_the_cache(entry, new, lens):
    """In the prefix, all rows are NaN; behind it, those of its sequence (which all see it)."""
    from fa2.paged import attention_paged
    page_size, D, dtype, prefix = 16, 64, torch.float16, 4096
    pages, cache, cu, seqlens, table = batch(new, lens, prefix, page_size, 2, D, dtype, False)
    q = randn((sum(new), 8, D), dtype, 1)
    own = table.clone()
    own[2, 4096 // 16] = entry
    out, lse = attention_paged(q, cache, own, cu, seqlens, shared=tokens(prefix), return_lse=True)
    mine = torch.zeros(sum(new), dtype=torch.bool, device="cuda")
    mine[int(cu[2]):int(cu[3])] = True
    assert out[mine].isnan().all() and lse[:, mine].isnan().all()
    assert torch.isfinite(out[~mine]).all() and torch.isfinite(lse[:, ~mine]).all()
    table[0, 130] = entry
    out, lse = attention_paged(q, cache, table, cu, seqlens, shared=tokens(prefix), return_lse=True)
    assert out.isnan().all() and lse.isnan().all()
