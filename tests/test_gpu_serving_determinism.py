"""Run-to-run determinism of every instance of the ragged attention kernel, the ones that spill registers to scratch among them
(tests/test_serving_resources.py). Scratch loads and stores count in the same vmcnt counter as the kernel's hand-placed waits, so
a wrong count would show up as a read of K, V or a spilled value before it landed: the output would change from launch to
launch. Each instance runs a grid that fills the GPU three times, which gives the same bits, and within the bound of two kernels
what the other way to its rows gives: pages and packed rows hold the same tokens.
"""

import pytest
import torch

from oracle import serving as oracle
from serving_check import cumulative, make_cache, randn

pytestmark = pytest.mark.gpu

# new tokens and tokens of the sequences. 128-row workgroups: prompts and chunks. 32-row ones: a prompt of few row tiles, steps
CALLS = {("packed", 4): ([1500, 900, 1, 2100], [1500, 900, 1, 2100]), ("packed", 1): ([700], [700]),
         ("16bit", 4): ([1000, 1, 500, 77], [9000, 3000, 5000, 77]), ("16bit", 1): ([1] * 48, [500 + 150 * i for i in range(48)])}


@pytest.mark.parametrize("lse", [False, True])
@pytest.mark.parametrize("row_waves", [1, 4])
@pytest.mark.parametrize("source", ["packed", "16bit", "e4m3"])
@pytest.mark.parametrize("D", [16, 32, 64, 128])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_every_instance_gives_the_same_bits(dtype, D, source, row_waves, lse):
    from fa2.packed import attention_packed
    from fa2.paged import attention_paged, cache_read
    new, lens = CALLS[(source if source == "packed" else "16bit", row_waves)]
    h_q, h_kv, page_size = 16, 8 if row_waves == 4 else 4, 64
    pages = oracle.Pages(lens, page_size, device="cuda")
    cache = make_cache(pages.n_pages, h_kv, page_size, D, dtype, source == "e4m3")
    seqlens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    q, cu, cu_kv = randn((sum(new), h_q, D), dtype, 3), cumulative(new), cumulative(lens)
    k, v = cache_read(cache, pages.table, cu_kv, seqlens, sum(lens), dtype=dtype)

    def packed():
        return attention_packed(q, k, v, cu, cu_kv, return_lse=lse)

    def paged():
        return attention_paged(q, cache, pages.table, cu, seqlens, return_lse=lse)
    run, other = (packed, paged) if source == "packed" else (paged, packed)
    first = run()
    torch.cuda.synchronize()
    for _ in range(2):
        again = run()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(again, first)) if lse else torch.equal(again, first)
    out, want = (first[0], other()[0]) if lse else (first, other())
    assert out.isfinite().all()
    # two kernels, each off by three roundings at most of values around the largest |v|
    assert (out.double() - want.double()).abs().max() <= 8 * oracle.HALF_STEP[dtype] * v.abs().max()
