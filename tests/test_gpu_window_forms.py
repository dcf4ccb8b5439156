"""GPU tests of windows over 16-bit pages with heads of 128, chunks of prompts beside single tokens, around the sizes at which the
chunks get 128-row workgroups and each sequence of few rows a 32-row one, in one launch."""

import pytest
import torch

from oracle import serving as oracle
from serving_check import cumulative, make_cache, randn
from step_check import check_paged_rows, hide_pages

pytestmark = pytest.mark.gpu
CUS = 256


def is_mixed(h_q, h_kv, n, n_seq, window, sinks):
    """Whether a batch of n rows is one of both forms (csrc/serve_host.hpp's window_plan)."""
    rows, shares, keys = n * h_q // h_kv // 128, 2 * CUS // h_kv, window + sinks + 128
    whole = rows <= shares and (keys + 256) * (shares - rows) <= 640 * shares
    return rows * h_kv >= CUS and whole and rows + n_seq > shares and n_seq * h_kv <= CUS


# (new tokens, tokens in the cache): many or few of the few, sequences of exactly 32 rows of a KV head and one more, empty ones, rows
# before their sequence's start
BATCHES = [(28, 4, [1] * 12 + [2040, 0, 4, 5] + [1] * 12, [2300 + 7 * i for i in range(12)] + [2600, 0, 900, 40] + [1700 + i for i in range(12)], True),
           (28, 4, [1] * 20 + [1000, 0, 1000, 2], [6000 + i for i in range(20)] + [1500, 9, 998, 2], True),
           (16, 16, [1] * 5 + [3400, 32, 0, 33] + [1] * 3, [2100 + i for i in range(5)] + [5000, 40, 0, 2000] + [1, 64, 3000], True),
           (28, 4, [1] * 24 + [2500], [2300] * 24 + [2500], False), (28, 4, [1] * 24 + [1500], [2300] * 24 + [1500], False),
           (28, 4, [1] * 70 + [2048], [2300] * 70 + [2100], False), (8, 2, [1] * 3 + [8192], [40] * 3 + [9000], True)]


@pytest.mark.parametrize("dtype,page_size", [(torch.bfloat16, 32), (torch.float16, 128)])
@pytest.mark.parametrize("h_q,h_kv,new,lens,mixed", BATCHES)
def test_chunks_beside_steps(dtype, page_size, h_q, h_kv, new, lens, mixed):
    from fa2.paged import attention_paged
    D = 128
    pages = oracle.Pages(lens, page_size, device="cuda")
    cache = make_cache(pages.n_pages, h_kv, page_size, D, dtype, False)
    cu, seqlens = cumulative(new), torch.tensor(lens, dtype=torch.int32, device="cuda")
    q = randn((sum(new) + 1, h_q, D), dtype, 3)
    if torch.cuda.get_device_properties(0).multi_processor_count == CUS:
        assert is_mixed(h_q, h_kv, len(q), len(new), 1900, 5) == mixed
    for window, sinks in ((1900, 5), (1500, 0)):
        table = hide_pages(pages, lens, new, window, sinks)
        out = torch.full_like(q, 9.0)
        _, lse = attention_paged(q, cache, table, cu, seqlens, window=window, sinks=sinks, return_lse=True, out=out)
        assert (out[-1] == 9.0).all()
        check_paged_rows(out, lse, q, cache, pages, lens, cu, dtype, window=window, sinks=sinks)
    out = attention_paged(q, cache, table, cu, seqlens, window=window, sinks=sinks)  # (an instance of its own)
    check_paged_rows(out, None, q, cache, pages, lens, cu, dtype, window=window, sinks=sinks)
