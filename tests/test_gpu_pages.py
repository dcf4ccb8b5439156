"""GPU tests of a step's pages (fa2.pages) against Python lists, of two calls at once and captured ones, and of whole
serving loops: pages taken, keys normalised, rotated and written, attention over them, pages given back."""

import random

import pytest
import torch

from oracle import step as step_oracle
from serving_check import randn
from step_check import check_rows

pytestmark = pytest.mark.gpu


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def pool_of(free, count):
    from fa2.pages import PagePool
    return PagePool(i32(free), i32([count]))


def check_extend(free, count, table, lens, new, page_size, n_tokens, padding=0):
    from fa2.pages import pages_extend
    pool = pool_of(free, count)
    wide = torch.full((len(table), len(table[0]) + padding), 77, dtype=torch.int32, device="cuda")
    t = wide[:, :len(table[0])]
    t.copy_(i32(table))
    was = pool.free.clone(), i32(lens)
    seqlens, fresh = i32(lens), i32(new)
    step = pages_extend(pool, t, seqlens, fresh, page_size, n_tokens)
    base, cu, after, positions, slots, want_table = step_oracle.extend(free, count, table, lens, new, page_size, n_tokens)
    assert step.pool.count.tolist() == [base] and step.pool.free is pool.free
    assert step.cu_seqlens.tolist() == cu and step.seqlens.tolist() == after
    assert step.positions.tolist() == positions and step.positions.dtype == torch.int32
    assert step.slots.tolist() == slots and step.slots.dtype == torch.int64
    assert t.tolist() == want_table
    assert (wide[:, len(table[0]):] == 77).all()
    assert torch.equal(pool.free, was[0]) and torch.equal(seqlens, was[1]) and pool.count.tolist() == [count]
    return step


def sequences(rng, n, page_size, most, columns, n_pages):
    """n sequences of up to `most` tokens over distinct pages: (free, count, table, lens)"""
    order = list(range(n_pages))
    rng.shuffle(order)
    table, lens = [[-1] * columns for _ in range(n)], []
    for row in table:
        tokens = min(rng.choice([0, 1, page_size, rng.randint(0, most)]), len(order) * page_size)
        held = min(-(-tokens // page_size), columns)
        for e in range(held):
            row[e] = order.pop()
        lens.append(tokens)
    return order + [0] * (n_pages - len(order)), len(order), table, lens


@pytest.mark.parametrize("page_size", [1, 16, 64, 4096])
@pytest.mark.parametrize("n", [1, 2, 63, 256, 257, 700])
def test_extend(n, page_size):
    rng = random.Random(n * 1000 + page_size)
    for most_new in (1, 3, 5 * page_size):
        columns = rng.randint(1, 20)
        free, count, table, lens = sequences(rng, n, page_size, 6 * page_size, columns, 40 * n + 7)
        new = [rng.choice([0, 1, rng.randint(0, most_new)]) for _ in range(n)]
        total = sum(new)
        check_extend(free, count, table, lens, new, page_size, total)
        check_extend(free, count, table, lens, new, page_size, total + 300, padding=3)  # rows of no sequence
        check_extend(free, count, table, lens, new, page_size, total // 2)              # more tokens than rows
        check_extend(free, rng.randint(0, 3), table, lens, new, page_size, total)       # too few pages
        check_extend(free, 0, table, lens, new, page_size, total)


def test_extend_long():
    """A long prompt among single tokens: many stripes of rows, of few sequences."""
    rng = random.Random(5)
    free, count, table, lens = sequences(rng, 9, 16, 1000, 3000, 10000)
    check_extend(free, count, table, lens, [1, 30000, 1, 0, 2000, 1, 1, 1, 5], 16, 32010)


def test_extend_odd_numbers():
    """Negative lengths and numbers, a count past the pool, entries that are no page, sums past 2^31, no columns."""
    from fa2.pages import PagePool, pages_extend
    check_extend(list(range(10)), 99, [[-1, -1], [5, -1]], [-4, 16], [20, -3], 16, 20)
    check_extend(list(range(10)), -1, [[-1, -1], [5, -1]], [0, 3], [20, 1], 16, 21)
    check_extend(list(range(10)), 4, [[1 << 30, -9], [5, 4]], [3, 30], [2, 1], 16, 3)
    step = pages_extend(PagePool.full(4), i32([[-1], [-1], [-1]]), i32([(1 << 31) - 1, 5, 7]), i32([(1 << 31) - 1, (1 << 31) - 1, 3]), 16, 5)
    assert step.seqlens.tolist() == [(1 << 31) - 1, (1 << 31) - 1, 10] and step.cu_seqlens.tolist() == [0] + [(1 << 31) - 1] * 3
    assert step.positions.tolist() == [(1 << 31) - 1] * 5 and step.slots.tolist() == [-1] * 5
    none = torch.empty(3, 0, dtype=torch.int32, device="cuda")
    step = pages_extend(PagePool.full(4), none, i32([0, 1, 2]), i32([1, 1, 1]), 16, 4)
    assert step.slots.tolist() == [-1] * 4 and step.positions.tolist() == [0, 1, 2, -1] and step.pool.count.tolist() == [4]
    step = pages_extend(PagePool.full(4), none[:0], i32([]), i32([]), 16, 2)
    assert step.cu_seqlens.tolist() == [0] and step.slots.tolist() == [-1, -1] and step.pool.count.tolist() == [4]
    step = pages_extend(PagePool.full(0), i32([[3]]), i32([0]), i32([2]), 16, 2)  # a pool of no pages
    assert step.slots.tolist() == [-1, -1] and step.pool.count.tolist() == [0]


@pytest.mark.parametrize("n", [1, 3, 64, 300])
def test_release(n):
    from fa2.pages import pages_release
    rng = random.Random(n)
    for _ in range(4):
        columns = rng.choice([1, 7, 130])
        free, count, table, lens = sequences(rng, n, 16, 16 * columns, columns, 60 * n)
        first = [rng.choice([0, 0, rng.randint(-2, columns)]) for _ in range(n)]
        last = [rng.choice([0, -(-x // 16), columns + 2, rng.randint(-3, columns)]) for x in lens]
        pool, t = pool_of(free, count), i32(table)
        got = pages_release(pool, t, i32(first), i32(last))
        want, want_count = step_oracle.release(free, count, table, first, last)
        assert got.count.tolist() == [want_count] and got.free is pool.free and got.free.tolist() == want
        assert t.tolist() == table and pool.count.tolist() == [count]


def test_release_wide():
    """Tables too wide for one launch: the same."""
    from fa2.pages import pages_release
    rng = random.Random(9)
    n, columns = 300, 1000
    free, count, table, lens = sequences(rng, n, 16, 2000, columns, 40 * n)
    first, last = [rng.choice([0, 3]) for _ in range(n)], [rng.choice([0, -(-x // 16), columns]) for x in lens]
    got = pages_release(pool_of(free, count), i32(table), i32(first), i32(last))
    want, want_count = step_oracle.release(free, count, table, first, last)
    assert got.count.tolist() == [want_count] and got.free.tolist() == want


def test_release_more_than_the_pool_holds():
    from fa2.pages import pages_release
    pool = pool_of([0, 1, 2, 3], 3)
    got = pages_release(pool, i32([[0, 1, 9], [2, -1, 3]]), i32([0, 0]), i32([3, 3]))
    assert got.count.tolist() == [4] and got.free.tolist() == [0, 1, 2, 0]
    empty = torch.empty(0, 3, dtype=torch.int32, device="cuda")
    assert pages_release(pool, empty, i32([]), i32([])).count.tolist() == [3]


def test_both_ways_streams_and_graphs(monkeypatch):
    from fa2 import _lib
    from fa2.pages import pages_extend, pages_release
    rng = random.Random(1)
    free, count, table, lens = sequences(rng, 40, 16, 300, 30, 2000)
    new = [rng.randint(0, 40) for _ in range(40)]

    def all_of():
        pool, t = pool_of(free, count), i32(table)
        step = pages_extend(pool, t, i32(lens), i32(new), 16, sum(new) + 3)
        back = pages_release(step.pool, t, i32([0] * 40), i32([3] * 40))
        return [step.pool.count, *step[1:], t, back.free, back.count]
    want = all_of()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    torch.cuda.synchronize()
    for _ in range(4):
        for stream in streams:
            with torch.cuda.stream(stream):
                got.append(all_of())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))
    pool, t, seqlens, fresh = pool_of(free, count), i32(table), i32(lens), i32(new)
    last = i32([0] * 40)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step = pages_extend(pool, t, seqlens, fresh, 16, 1600)
        back = pages_release(step.pool, t, torch.zeros_like(last), last)
        seqlens.copy_(step.seqlens)
        pool.count.copy_(back.count)
    state = free, count, table, lens
    for _ in range(4):  # every replay goes on from the one before
        more = [rng.randint(0, 3) for _ in range(40)]
        gone = [rng.choice([0, 0, 2]) for _ in range(40)]
        fresh.copy_(i32(more))
        last.copy_(i32(gone))
        graph.replay()
        torch.cuda.synchronize()
        base, cu, after, positions, slots, entries = step_oracle.extend(*state, more, 16, 1600)
        stack, total = step_oracle.release(state[0], base, entries, [0] * 40, gone)
        assert step.cu_seqlens.tolist() == cu and step.slots.tolist() == slots and step.positions.tolist() == positions
        assert t.tolist() == entries and pool.free.tolist() == stack and pool.count.tolist() == [total]
        assert seqlens.tolist() == after
        state = stack, total, entries, after
    monkeypatch.setattr(_lib, "native", None)
    assert all(torch.equal(a, b) for a, b in zip(all_of(), want))


# ------------------------------------------------------------------------------------------
# serving loops
# ------------------------------------------------------------------------------------------

@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("window", [None, 50])
def test_serving_loop(e4m3, window):
    """Sequences that come, grow by prompts and steps and end, over a pool hardly larger than they need: the pages of one are
    the next one's. Rows are the oracle's over each sequence's own history; with a window, pages that have left it go back
    while the sequence runs. Images' positions of three axes, heads normalised."""
    from fa2.paged import KVCache, attention_paged, cache_read, cache_write
    from fa2.pages import PagePool, pages_extend, pages_release
    from fa2.rotary import HeadNorm, rotary_plan
    S, columns, page_size, h_q, h_k, D, dtype, sinks = 6, 40, 16 if not e4m3 else 32, 4, 2, 64, torch.bfloat16, 5
    rng = random.Random(3)
    plan = rotary_plan(64, axes=[0] * 8 + [1] * 12 + [2] * 12)
    norms = dict(q_norm=HeadNorm(1 + 0.1 * randn((D,), torch.float32, 1)), k_norm=HeadNorm(1 + 0.1 * randn((D,), torch.float32, 2)))
    n_pages = 60 if window is None else 45
    cache = KVCache.empty(n_pages, h_k, page_size, D, torch.float8_e4m3fn if e4m3 else dtype)
    pool = PagePool.full(n_pages)
    table, seqlens = torch.full((S, columns), -1, dtype=torch.int32, device="cuda"), i32([0] * S)
    given = [0] * S   # entries (behind the sinks' pages) that have gone back
    history = [[] for _ in range(S)]  # per sequence: (k, v) float64 of every token, as the cache holds them
    for turn in range(25):
        lens = [len(h) for h in history]
        ended = [len(h) > 120 for h in history]
        # pages back: of ended sequences what they still hold, of running ones what has left the window
        first, last = [0] * S, [0] * S
        sink_pages = -(-sinks // page_size)
        for s in range(S):
            if ended[s]:
                first[s], last[s] = given[s], -(-lens[s] // page_size)
            elif window is not None:
                first[s], last[s] = max(given[s], sink_pages), max((lens[s] - window + 1) // page_size, 0)
                last[s] = max(last[s], first[s])
        pool = pages_release(pool, table, i32(first), i32(last))
        for s in range(S):
            if ended[s] and given[s]:  # the sinks' pages, in front of what went back before
                pool = pages_release(pool, table, i32([0] * S), i32([sink_pages if x == s else 0 for x in range(S)]))
            if ended[s]:
                history[s], given[s] = [], 0
            elif last[s] > first[s]:
                given[s] = last[s]
        seqlens = i32([len(h) for h in history])
        new = [0 if rng.random() < 0.2 else rng.choice([1, 1, 2, rng.randint(1, 60) if not h else 1]) for h in history]
        T = sum(new)
        step = pages_extend(pool, table, seqlens, i32(new), page_size, T)
        pool, seqlens = step.pool, step.seqlens
        if T == 0:
            continue
        q, k, v = (randn((T, h, D), dtype, 100 * turn + i) for i, h in enumerate((h_q, h_k, h_k)))
        positions = torch.stack([step.positions, step.positions // 3, step.positions % 7])
        q = cache_write(cache, k, v, table, step.cu_seqlens, seqlens, rotary=plan, q=q, positions=positions, **norms)
        assert (step.slots >= 0).all() and len(set(step.slots.tolist())) == T
        kw = {} if window is None else dict(window=window, sinks=sinks)
        out, lse = attention_paged(q, cache, table, step.cu_seqlens, seqlens, return_lse=True, **kw)
        written = cache_read(cache, table, step.cu_seqlens, seqlens, T, dtype=dtype)
        cu = step.cu_seqlens.tolist()
        for s in range(S):
            for t in range(cu[s], cu[s + 1]):
                history[s].append((written[0][t].double(), written[1][t].double()))
        of = [lambda s, i=i: torch.stack([x[i] for x in history[s]]) for i in range(2)]
        check_rows(out, lse, q, *of, step.cu_seqlens, dtype, window=window, sinks=sinks if window else 0)
    live = {int(p) for s in range(S) for e, p in enumerate(table[s].tolist())
            if e < -(-len(history[s]) // page_size) and not (-(-sinks // page_size) <= e < given[s])}
    free = pool.free[:int(pool.count)].tolist()
    assert len(set(free)) == len(free) and not live & set(free) and len(live) + len(free) == n_pages


def test_shared_prefix_loop():
    """One prompt, then a batch of answers behind it whose tables all name its pages; shared and plain attention agree to the
    bounds of both with the oracle, and the answers' own pages go back at the end."""
    from fa2.paged import KVCache, attention_paged, cache_read, cache_write
    from fa2.pages import PagePool, pages_extend, pages_release
    from fa2.rotary import HeadNorm, rotary_plan
    S, page_size, h_q, h_k, D, dtype, prompt = 12, 16, 8, 2, 128, torch.float16, 515
    plan, norm = rotary_plan(128), HeadNorm(1 + 0.1 * randn((D,), torch.float32, 1))
    cache, pool = KVCache.empty(120, h_k, page_size, D, dtype), PagePool.full(120)
    one = torch.full((1, 40), -1, dtype=torch.int32, device="cuda")
    step = pages_extend(pool, one, i32([0]), i32([prompt]), page_size, prompt)
    q, k, v = (randn((prompt, h, D), dtype, i) for i, h in enumerate((h_q, h_k, h_k)))
    cache_write(cache, k, v, one, step.cu_seqlens, step.seqlens, rotary=plan, k_norm=norm)
    common = prompt // page_size
    first_k, first_v = cache_read(cache, one, step.cu_seqlens, step.seqlens, prompt)
    # the batch begins with the whole pages of the prompt; its last tokens are written again, for each
    table = torch.full((S, 40), -1, dtype=torch.int32, device="cuda")
    table[:, :common] = one[0, :common]
    lens, pool = i32([common * page_size] * S), step.pool
    tail = prompt - common * page_size
    history = [([first_k[:common * page_size].double()], [first_v[:common * page_size].double()]) for _ in range(S)]
    shared = i32([prompt])
    for turn in range(20):
        n = tail if turn == 0 else 1
        step = pages_extend(pool, table, lens, i32([n] * S), page_size, n * S)
        pool, lens = step.pool, step.seqlens
        q, k, v = (randn((n * S, h, D), dtype, 1000 + 10 * turn + i) for i, h in enumerate((h_q, h_k, h_k)))
        q = cache_write(cache, k, v, table, step.cu_seqlens, lens, rotary=plan, q=q, k_norm=norm, q_norm=norm)
        out, lse = attention_paged(q, cache, table, step.cu_seqlens, lens, shared=shared, return_lse=True)
        written = cache_read(cache, table, step.cu_seqlens, lens, n * S)
        for s in range(S):
            for x, w in zip(history[s], written):
                x.append(w[s * n:(s + 1) * n].double())
        of = [lambda s, i=i: torch.cat(history[s][i]) for i in range(2)]
        check_rows(out, lse, q, *of, step.cu_seqlens, dtype, joined=8)
        plain = attention_paged(q, cache, table, step.cu_seqlens, lens)
        check_rows(plain, None, q, *of, step.cu_seqlens, dtype)
    count = int(pool.count)
    pool = pages_release(pool, table, i32([common] * S), (lens + page_size - 1) // page_size)
    assert int(pool.count) == 120 - common - 1  # the prompt's own pages are the only ones still out
    assert int(pool.count) > count and len(set(pool.free[:int(pool.count)].tolist())) == int(pool.count)
