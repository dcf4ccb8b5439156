"""GPU test of the serving operators called from several host threads at once, each on a stream of its own."""

import threading

import pytest
import torch

from oracle import serving as oracle
from serving_check import cumulative, make_cache, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("native", [True, False])
def test_threads_at_once(native, monkeypatch):
    """Natively (the interpreter runs other threads meanwhile) and through ctypes, the same bits as one after another; a
    refused call beside them raises its own error in its own thread."""
    from fa2 import _lib
    from fa2.packed import attention_packed
    from fa2.paged import attention_paged, cache_read
    from fa2.rotary import rotary, rotary_plan
    if not native:
        monkeypatch.setattr(_lib, "native", None)
    plan, dtype, D = rotary_plan(64), torch.bfloat16, 64
    jobs = []
    for i in range(4):
        new, lens = [1 + i] * 5, [700 * i + 100 + 31 * j for j in range(5)]
        pages = oracle.Pages(lens, 16, seed=i, device="cuda")
        cache = make_cache(pages.n_pages, 2, 16, D, dtype, i % 2 == 1, i)
        cu, seqlens = cumulative(new), torch.tensor(lens, dtype=torch.int32, device="cuda")
        q, k = randn((sum(new), 8, D), dtype, i), randn((sum(new), 2, D), dtype, 9 + i)
        positions = torch.arange(sum(new), device="cuda")

        def job(q=q, k=k, cache=cache, table=pages.table, cu=cu, seqlens=seqlens, positions=positions):
            return (rotary(q, positions, plan), attention_packed(q, k, k, cu), attention_paged(q, cache, table, cu, seqlens),
                    *cache_read(cache, table, cu, seqlens, q.shape[0], dtype=dtype))
        jobs.append(job)
    want = [job() for job in jobs]
    torch.cuda.synchronize()
    got, errors = [[] for _ in jobs], []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got[i].append(jobs[i]())
        except Exception as e:
            errors.append(e)

    def refused():
        x = torch.zeros(4, 2, D, dtype=dtype, device="cuda")
        for _ in range(20):
            try:
                rotary(x, torch.arange(4, device="cuda"), plan, out=x[:1].expand(4, 2, D))
                errors.append("not refused")
            except RuntimeError as e:
                if "stride of 0" not in str(e):
                    errors.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    bad = threading.Thread(target=refused)
    for t in (*threads, bad):
        t.start()
    for t in (*threads, bad):
        t.join()
    torch.cuda.synchronize()
    assert not errors, errors
    for results, w in zip(got, want):
        assert len(results) == 20
        for r in results:
            assert all(torch.equal(a, b) for a, b in zip(r, w))
