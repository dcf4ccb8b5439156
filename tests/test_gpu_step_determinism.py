"""GPU tests that every instance of the attention kernels of windows and common prefixes gives the same bits each time, and
that calls from several host threads at once are each as alone."""

import threading

import pytest
import torch

from oracle import serving as oracle
from serving_check import cumulative, make_cache, randn

pytestmark = pytest.mark.gpu
# (new, tokens in the cache, h_q, h_kv): of a window the 32-row form, the 128-row one and both at once; of a prefix 32 rows for both passes, 128
# and 32, and 128
CALLS = {"few": ([1] * 5, [3000 + i for i in range(5)], 8, 2), "many": ([300, 64], [2900, 3000], 8, 2),
         "mixed": ([3000, 1, 1, 2], [3100, 3000, 2950, 2980], 16, 16), "shared few": ([1] * 5, [3000 + i for i in range(5)], 8, 2),
         "shared steps": ([1] * 40, [2900 + 3 * i for i in range(40)], 8, 2), "shared chunks": ([100] * 4, [3100 + i for i in range(4)], 8, 2)}


def call_of(name, dtype, D, e4m3, lse):
    from fa2.paged import attention_paged
    new, lens, h_q, h_kv = CALLS[name]
    pages = oracle.Pages(lens, 64, device="cuda")
    shared = name.startswith("shared")
    if shared:
        pages.table[:, :40] = pages.table[0, :40].clone()
    cache = make_cache(pages.n_pages, h_kv, 64, D, dtype, e4m3)
    args = (randn((sum(new), h_q, D), dtype, 1), cache, pages.table, cumulative(new), torch.tensor(lens, dtype=torch.int32, device="cuda"))
    kw = dict(shared=torch.tensor([2560], dtype=torch.int32, device="cuda")) if shared else dict(window=2000, sinks=3)
    return lambda: attention_paged(*args, return_lse=lse, **kw)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [16, 32, 64, 128])
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("lse", [False, True])
@pytest.mark.parametrize("name", CALLS)
def test_the_same_bits(dtype, D, e4m3, lse, name):
    call = call_of(name, dtype, D, e4m3, lse)
    first = call()
    for _ in range(2):
        again = call()
        pairs = zip(again, first) if lse else [(again, first)]
        assert all(torch.equal(a, b) for a, b in pairs)


def test_threads_at_once():
    calls = [call_of(name, torch.bfloat16, 64, False, True) for name in CALLS]
    want = [call() for call in calls]
    torch.cuda.synchronize()
    wrong = []

    def work(call, w):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            got = [call() for _ in range(6)]
        stream.synchronize()
        if not all(torch.equal(a, b) for g in got for a, b in zip(g, w)):
            wrong.append(call)

    threads = [threading.Thread(target=work, args=x) for x in zip(calls, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
