"""GPU tests of windows over chunks of prompts beside single tokens, whose rows fill the GPU: 128-row workgroups for the
chunks and a 32-row one for each sequence of few rows, in one launch."""

import pytest
import torch

from oracle import serving as oracle
from serving_check import cumulative, make_cache, randn
from step_check import check_paged_rows, hide_pages

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("dtype,D,page_size", [(torch.bfloat16, 128, 32), (torch.float16, 64, 16), (torch.bfloat16, 32, 64), (torch.float16, 16, 64)])
@pytest.mark.parametrize("h_q,h_kv", [(28, 4), (16, 16)])
def test_chunks_beside_steps(e4m3, dtype, D, page_size, h_q, h_kv):
    """Sequences on both sides of 32 rows of a KV head, and of exactly 32; empty ones among them; more than 64 sequences."""
    from fa2.paged import attention_paged
    group = h_q // h_kv
    for new, lens in (([1] * 9 + [2500, 0, 32 // group, 1] + [33] + [1] * 3, [2300 + 7 * i for i in range(9)] + [2600, 0, 900, 1] + [40] + [1700] * 3),
                      ([1] * 40 + [1800] + [2] * 40 + [700], [1600 + i for i in range(40)] + [1800] + [50 + i for i in range(40)] + [5000])):
        pages = oracle.Pages(lens, page_size, device="cuda")
        cache = make_cache(pages.n_pages, h_kv, page_size, D, dtype, e4m3)
        cu, seqlens = cumulative(new), torch.tensor(lens, dtype=torch.int32, device="cuda")
        q = randn((sum(new) + 1, h_q, D), dtype, 3)
        for window, sinks in ((1900, 5), (1500, 0)):
            table = hide_pages(pages, lens, new, window, sinks)
            out = torch.full_like(q, 9.0)
            _, lse = attention_paged(q, cache, table, cu, seqlens, window=window, sinks=sinks, return_lse=True, out=out)
            assert (out[-1] == 9.0).all()
            check_paged_rows(out, lse, q, cache, pages, lens, cu, dtype, window=window, sinks=sinks)
        out = attention_paged(q, cache, table, cu, seqlens, window=window, sinks=sinks)  # (an instance of its own)
        check_paged_rows(out, None, q, cache, pages, lens, cu, dtype, window=window, sinks=sinks)
