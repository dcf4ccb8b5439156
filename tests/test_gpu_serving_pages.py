"""GPU tests of what a paged cache may hold beside ordinary tokens: table entries that are no page, wherever they lie among the
workgroups that share a sequence's keys, and infinite and NaN values in keys that rows see; and of rows that belong to no sequence.
"""

import pytest
import torch

from oracle import serving as oracle
from serving_check import CACHES, bytes_of, cached, check_attention, cumulative, make_cache, randn

pytestmark = pytest.mark.gpu


# (new tokens, tokens in the cache) of the sequences: steps of one token (32-row workgroups) and a chunk beside steps (128-row
# ones), over keys that several workgroups share; and steps and chunks that nobody shares, as their table is narrow
CALLS = {"shared steps": ([1, 1, 1], [4000, 2500, 3333]), "shared chunk": ([300, 1, 40], [3000, 2500, 2000]),
         "steps": ([1, 1, 4], [1500, 700, 600]), "chunk": ([300, 1, 40], [1500, 700, 600])}


def call_of(name, page_size, D, dtype, e4m3, h_q=8, h_kv=2, seed=0):
    new, lens = CALLS[name]
    pages = oracle.Pages(lens, page_size, seed=seed, device="cuda")
    pages.table = pages.table[:, :-(-max(lens) // page_size)].contiguous()
    cache = make_cache(pages.n_pages, h_kv, page_size, D, dtype, e4m3, seed)
    q = randn((sum(new), h_q, D), dtype, 30 + seed)
    return new, lens, pages, cache, q, cumulative(new), torch.tensor(lens, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("D,page_size", [(128, 128), (64, 256), (32, 64), (128, 16)])
@pytest.mark.parametrize("call", CALLS)
def test_rows_that_see_an_entry_that_is_no_page_are_nan(call, D, page_size, e4m3):
    """One such entry, at every place of a sequence's table in turn, and runs of them up to a whole row: the rows that see its
    tokens are NaN, their log-sum-exp too, and the other sequences as they were. A page of 128 tokens of head_dim 128 is a
    tile for each of the four waves that take tiles in turn, so that none of them has a sum to show for its keys."""
    from fa2.paged import attention_paged
    new, lens, pages, cache, q, cu, seqlens = call_of(call, page_size, D, torch.bfloat16, e4m3)
    want, want_lse = attention_paged(q, cache, pages.table, cu, seqlens, return_lse=True)
    assert want.isfinite().all() and want_lse.isfinite().all()
    s, first = 0, cu.tolist()
    need = -(-lens[s] // page_size)
    runs = [(i, i + 1) for i in range(0, need, max(1, need // 24))] + [(need // 3, need), (0, need), (need // 4, need // 2)]
    for a, b in runs:
        table = pages.table.clone()
        table[s, a:b] = -1
        out, lse = attention_paged(q, cache, table, cu, seqlens, return_lse=True)
        # row i of the sequence sees its tokens up to lens - new + i
        sees = [first[s] + i for i in range(new[s]) if lens[s] - new[s] + i >= a * page_size]
        assert out[sees].isnan().all() and lse[:, sees].isnan().all(), (a, b)
        assert torch.equal(attention_paged(q, cache, table, cu, seqlens)[sees].isnan(), out[sees].isnan())
        others = [t for t in range(q.shape[0]) if not first[s] <= t < first[s + 1]]
        assert torch.equal(out[others], want[others]) and torch.equal(lse[:, others], want_lse[:, others]), (a, b)


BAD = {"inf": float("inf"), "-inf": float("-inf"), "nan": float("nan")}


@pytest.mark.parametrize("dtype,D,page_size", [(torch.float16, 64, 16), (torch.bfloat16, 128, 64), (torch.float16, 128, 16),
                                               (torch.bfloat16, 16, 64), (torch.float16, 32, 128)])
@pytest.mark.parametrize("cache_type", CACHES)
@pytest.mark.parametrize("call", CALLS)
def test_values_that_are_not_finite(call, cache_type, dtype, D, page_size):
    """An infinite or NaN value or key of a cached token (e4m3: NaN, and a scale that is none) reaches the rows that see it, and
    no other: at the first token, within a tile, at the last token that every row sees and at the last one, which only the
    last row does."""
    from fa2.paged import attention_paged
    e4m3 = cache_type == "e4m3"
    new, lens, pages, cache, q, cu, seqlens = call_of(call, page_size, D, dtype, e4m3)
    q = torch.where(q == 0, torch.ones_like(q), q)
    s = 0
    for which in ("k", "v"):
        for at in (0, lens[s] // 2 + 5, lens[s] - new[s], lens[s] - 1):
            page, row = (x.item() for x in pages.at(s, torch.tensor(at, device="cuda")))
            for name in (("nan", "scale") if e4m3 else BAD):
                one = cache._replace(**{which: cache._asdict()[which].clone()})
                if name == "scale":  # e8m0 has NaN too
                    scale = getattr(cache, which + "_scale").view(torch.uint8).clone()
                    scale[page, 1, row] = 255
                    one = one._replace(**{which + "_scale": scale.view(torch.float8_e8m0fnu)})
                else:
                    bytes_of(getattr(one, which))[page, 1, row, D // 2] = 0x7f if e4m3 else BAD[name]
                for causal in (True, False):
                    out, lse = attention_paged(q, one, pages.table, cu, seqlens, causal=causal, return_lse=True)

                    def values(part, n):
                        x = cached(one, part, *pages.at(n, torch.arange(lens[n], device="cuda"))).to(dtype).double()
                        if name == "scale" and part == which and n == s:
                            x[at, 1] = float("nan")
                        return x
                    check_attention(out, lse, q, lambda n: values("k", n), lambda n: values("v", n), cu, causal, dtype)
                    assert torch.equal(attention_paged(q, one, pages.table, cu, seqlens, causal=causal).nan_to_num(5.0),
                                       out.nan_to_num(5.0))


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("n_seq,group", [(5, 40), (64, 2), (65, 1), (200, 3)])
def test_rows_of_no_sequence(n_seq, group, e4m3):
    """Rows before the first sequence and behind the last, and rows before their sequence's start, stay as they are in every
    operator's output; sequences without rows lie between the others, more than 64 of them side by side among 200."""
    from fa2.packed import attention_packed
    from fa2.paged import attention_paged, cache_read, cache_write
    from fa2.rotary import rotary, rotary_plan
    D, page_size, h_kv, dtype, first = 64, 32, 2, torch.bfloat16, 37
    new = [3 + s % 5 if s in (1, 2, n_seq // 2, n_seq - 1) else 0 for s in range(n_seq)]
    lens = [n - 2 if s == 2 else n + 11 * (s % 7) for s, n in enumerate(new)]  # sequence 2: two rows before its start
    pages = oracle.Pages(lens, page_size, device="cuda")
    cache = make_cache(pages.n_pages, h_kv, page_size, D, dtype, e4m3)
    cu, seqlens = cumulative(new) + first, torch.tensor(lens, dtype=torch.int32, device="cuda")
    at, T = cu.tolist(), first + sum(new) + 9
    q, k, v = (randn((T, h, D), dtype, i) for i, h in enumerate((h_kv * group, h_kv, h_kv)))
    position = torch.full((T,), -1, device="cuda")
    for s, n in enumerate(new):
        position[at[s]:at[s + 1]] = torch.arange(lens[s] - n, lens[s], device="cuda")
    placed = position >= 0
    plan = rotary_plan(D)
    q_out, k_out, v_out, out = (torch.full_like(t, 7.0) for t in (q, k, v, q))
    cache_write(cache, k, v, pages.table, cu, seqlens, rotary=plan, q=q, q_out=q_out)
    cache_read(cache, pages.table, cu, seqlens, T, out=(k_out, v_out))
    assert torch.equal(q_out[placed], rotary(q, position, plan)[placed])
    if not e4m3:
        assert torch.equal(k_out[placed], rotary(k, position, plan)[placed]) and torch.equal(v_out[placed], v[placed])
    for t in (q_out, k_out, v_out):
        assert (t[~placed] == 7.0).all()

    def rows_of_none(t):
        return torch.cat([t[:first], t[at[-1]:]])
    for causal in (True, False):
        _, lse = attention_paged(q, cache, pages.table, cu, seqlens, causal=causal, return_lse=True, out=out.fill_(7.0))
        assert (rows_of_none(out) == 7.0).all()

        def of(which):
            return lambda s: cached(cache, which, *pages.at(s, torch.arange(lens[s], device="cuda"))).to(dtype).double()
        check_attention(out, lse, q, of("k"), of("v"), cu, causal, dtype)
        _, lse = attention_packed(q, k, v, cu, causal=causal, return_lse=True, out=out.fill_(7.0))
        assert (rows_of_none(out) == 7.0).all()
        check_attention(out, lse, q, lambda s: k[at[s]:at[s + 1]].double(), lambda s: v[at[s]:at[s + 1]].double(), cu, causal,
                        dtype)
