"""GPU tests of normalised rotations by one position or several axes (fa2.rotary.rotary_qk, and cache_write with norms and
positions), against float64 under derived bounds."""

import math

import pytest
import torch

from oracle import serving as oracle
from oracle import step as step_oracle
from serving_check import bytes_of, cached, cumulative, make_cache, randn

pytestmark = pytest.mark.gpu
DTYPES = [torch.float16, torch.bfloat16]


def plan_of(rot, axes, interleaved=False, scale=1.0):
    from fa2.rotary import rotary_plan
    of = None if axes == 1 else [i * axes // (rot // 2) if i % 3 else i % axes for i in range(rot // 2)]
    return rotary_plan(rot, 10000.0, interleaved=interleaved, axes=of)._replace(scale=scale)


def weight_of(D, seed):
    return 1.0 + 0.3 * randn((D,), torch.float32, seed)


def positions_of(axes, shape, seed, far=1 << 20):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-5, far, (*((axes,) if axes > 1 else ()), *shape), generator=g).cuda()


def check(got, x, positions, plan, norm):
    """got and x [T, H, D], positions [T] or [axes, T]"""
    weight, eps = (None, 0.0) if norm is None else norm
    want, tol = step_oracle.turn(x, positions, plan.freqs, plan.interleaved, plan.scale, plan.axes, weight, eps)
    off = (got.double() - want).abs()
    assert (off <= tol).all(), (off / tol).max()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,rot", [(16, 16), (32, 16), (64, 48), (64, 64), (128, 32), (128, 96), (128, 128)])
@pytest.mark.parametrize("axes", [1, 2, 3])
def test_rotary_qk(dtype, interleaved, D, rot, axes):
    from fa2.rotary import HeadNorm, rotary, rotary_qk
    plan = plan_of(rot, axes, interleaved, 1.25)
    norms = HeadNorm(weight_of(D, 7)), HeadNorm(weight_of(D, 8), 1e-5)
    for seed, (T, h_q, h_k) in enumerate([(1, 1, 1), (3, 5, 2), (37, 32, 8), (130, 7, 1)]):
        q, k = randn((T, h_q, D), dtype, seed), randn((T, h_k, D), dtype, 50 + seed, scale=5.0)
        positions = positions_of(axes, (T,), seed)
        for q_norm, k_norm in ((None, None), (norms[0], norms[1]), (None, norms[1])):
            got_q, got_k = rotary_qk(q, k, positions, plan, q_norm=q_norm, k_norm=k_norm)
            check(got_q, q, positions, plan, q_norm)
            check(got_k, k, positions, plan, k_norm)
            if q_norm is None:
                assert torch.equal(got_q[..., rot:], q[..., rot:])  # neither: copied
            assert all(torch.equal(a, b) for a, b in zip(rotary_qk(q, k, positions.int(), plan, q_norm=q_norm, k_norm=k_norm),
                                                         (got_q, got_k)))
            assert torch.equal(rotary(q, positions, plan, norm=q_norm), got_q)
            alone, nothing = rotary_qk(k, None, positions, plan, q_norm=k_norm)
            assert nothing is None and torch.equal(alone, got_k)
            mine = q.clone(), k.clone()  # in place
            out = rotary_qk(*mine, positions, plan, q_norm=q_norm, k_norm=k_norm, q_out=mine[0], k_out=mine[1])
            assert out[0] is mine[0] and out[1] is mine[1]
            assert torch.equal(mine[0], got_q) and torch.equal(mine[1], got_k)


def test_one_axis_as_rotary():
    """Without norms and axes the values are rotary()'s, bit for bit; three axes of one position too."""
    from fa2.rotary import rotary, rotary_plan, rotary_qk
    q, k = randn((60, 8, 128), torch.bfloat16, 1), randn((60, 2, 128), torch.bfloat16, 2)
    positions = torch.arange(60, device="cuda") * 977
    plan = rotary_plan(128)
    want = rotary(q, positions, plan), rotary(k, positions, plan)
    assert all(torch.equal(a, b) for a, b in zip(rotary_qk(q, k, positions, plan), want))
    three = rotary_plan(128, axes=[0, 1, 2] * 21 + [0])
    assert all(torch.equal(a, b) for a, b in zip(rotary_qk(q, k, positions.expand(3, 60), three), want))
    wild = three._replace(axes=torch.where(three.axes == 2, 1 << 30, torch.where(three.axes == 0, -7, 1)).int())
    apart = torch.stack([positions, positions + 5, positions + 11])
    assert all(torch.equal(a, b) for a, b in zip(rotary_qk(q, k, apart, wild), rotary_qk(q, k, apart, three)))  # the nearest axis


@pytest.mark.parametrize("axes", [1, 3])
def test_layouts(axes):
    """[B, H, N, D] with positions of a row or of the batch, transposed and offset storage, outputs of their own."""
    from fa2.rotary import HeadNorm, rotary_qk
    plan, norms = plan_of(64, axes), dict(q_norm=HeadNorm(weight_of(64, 1)), k_norm=HeadNorm(weight_of(64, 2)))
    q, k = randn((3, 4, 50, 64), torch.bfloat16, 1), randn((3, 2, 50, 64), torch.bfloat16, 2)
    both = positions_of(axes, (3, 50), 5)
    got = rotary_qk(q, k, both, plan, **norms)
    for b in range(3):
        mine = both[b] if axes == 1 else both[:, b]
        check(got[0][b].transpose(0, 1), q[b].transpose(0, 1), mine, plan, norms["q_norm"])
        check(got[1][b].transpose(0, 1), k[b].transpose(0, 1), mine, plan, norms["k_norm"])
        assert all(torch.equal(a[b], g[b]) for a, g in zip(rotary_qk(q, k, mine, plan, **norms), got))
    bnhd = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k)]
    assert all(torch.equal(a, g) for a, g in zip(rotary_qk(*bnhd, both, plan, **norms), got))
    out = [torch.full((3, 50, h, 64), 9.0, dtype=q.dtype, device="cuda").transpose(1, 2) for h in (4, 2)]
    made = rotary_qk(*bnhd, both, plan, **norms, q_out=out[0], k_out=out[1])
    assert all(m is o and torch.equal(o, g) for m, o, g in zip(made, out, got))

    def odd(t):  # not 16-byte aligned: through copies
        return torch.zeros(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(t.shape).copy_(t)
    mine = odd(q), odd(k)
    assert all(torch.equal(a, g) for a, g in zip(rotary_qk(*mine, both, plan, **norms), got))
    made = rotary_qk(*mine, both, plan, **norms, q_out=mine[0], k_out=mine[1])
    assert all(m is o and torch.equal(o, g) for m, o, g in zip(made, mine, got))
    strided = both.repeat_interleave(2, -1)[..., ::2]
    assert all(torch.equal(a, g) for a, g in zip(rotary_qk(q, k, strided, plan, **norms), got))
    empty = rotary_qk(q[:, :, :0], k[:, :, :0], both[..., :0], plan, **norms)
    assert empty[0].shape == (3, 4, 0, 64) and empty[1].shape == (3, 2, 0, 64)


@pytest.mark.parametrize("dtype", DTYPES)
def test_norm_extremes(dtype):
    """Heads of zeros, of the least and largest values (whose squares no float holds, in bf16), with infinities and NaN."""
    from fa2.rotary import HeadNorm, rotary_plan, rotary_qk
    D = 64
    info = torch.finfo(dtype)
    rows = [[0.0], [info.smallest_normal * info.eps], [info.max], [info.max] * D, [-info.max, 1.0, info.max / 2], [1e-3] * D,
            [math.inf, 1.0], [math.nan, 2.0], [1.0, -math.inf, math.nan]]
    x = torch.zeros(len(rows), 1, D, dtype=dtype, device="cuda")
    for i, r in enumerate(rows):
        x[i, 0, :len(r)] = torch.tensor(r, device="cuda").to(dtype)
    plan, norm = rotary_plan(32), HeadNorm(weight_of(D, 3), 1e-12)
    positions = torch.arange(len(rows), device="cuda")
    got, _ = rotary_qk(x, None, positions, plan, q_norm=norm)
    want, tol = step_oracle.turn(x, positions, plan.freqs, weight=norm.weight, eps=norm.eps)
    assert torch.equal(got.isnan(), want.isnan())
    fine = ~want.isnan()
    assert ((got.double() - want).abs() <= tol)[fine].all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_norm_of_small_values(dtype):
    """Heads of values on both sides of the type's least normal one, whose squares are its sum; and of one large value among them."""
    from fa2.rotary import HeadNorm, rotary_plan, rotary_qk
    D = 128
    least = torch.finfo(dtype).smallest_normal
    g = torch.Generator().manual_seed(1)
    x = ((torch.rand(40, 3, D, generator=g, dtype=torch.float64) - 0.5) * 4 * least).to(dtype).cuda()
    x[:, 1, 5] = least
    x[:, 2, 77] = 1.0
    plan, norm = rotary_plan(64), HeadNorm(weight_of(D, 3), 1e-30 if dtype == torch.float16 else 1e-300)
    positions = torch.arange(40, device="cuda")
    got, _ = rotary_qk(x, None, positions, plan, q_norm=norm)
    want, tol = step_oracle.turn(x, positions, plan.freqs, weight=norm.weight, eps=norm.eps)
    assert ((got.double() - want).abs() <= tol).all(), ((got.double() - want).abs() / tol).max()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("eps", [5e-324, 1e-300, 1e-78, 1e-76, 1e-40, 1e300])
@pytest.mark.parametrize("interleaved", [False, True])
def test_norm_least_values(dtype, eps, interleaved):
    """The least eps there are, and the largest: rows of zeros are zeros, rows of the type's least values as any others."""
    from fa2.rotary import HeadNorm, rotary_plan, rotary_qk
    D = 64
    least = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    g = torch.Generator().manual_seed(2)
    x = torch.zeros(60, 2, D, dtype=torch.float64)
    for t in range(1, 60):  # (with one value, a few and all; up to 2^40 times the least)
        n = (1, 5, D)[t % 3]
        x[t, 0, torch.randperm(D, generator=g)[:n]] = torch.randint(-9, 10, (n,), generator=g).double() * least * 2.0 ** (t * 2 // 3)
        x[t, 1] = least * (1 if t % 2 else -3)
    x = x.to(dtype).cuda()
    plan, norm = rotary_plan(48, interleaved=interleaved), HeadNorm(weight_of(D, 3), eps)
    positions = torch.arange(60, device="cuda")
    got, _ = rotary_qk(x, None, positions, plan, q_norm=norm)
    want, tol = step_oracle.turn(x, positions, plan.freqs, interleaved, weight=norm.weight, eps=norm.eps)
    assert (got[0] == 0).all() and torch.equal(got.isnan(), want.isnan())
    fine = ~want.isnan()  # (fp16's largest rows hold infinities)
    assert fine[:40].all() and ((got.double() - want).abs() <= tol)[fine].all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("eps", [1e29, 1e31, 1e38, 1e39, 1e60, 1e72, 1e76, 1e100, 1e200, 1.7e308])
@pytest.mark.parametrize("interleaved", [False, True])
def test_norm_large_eps(dtype, eps, interleaved):
    """An eps past float's range, beside ordinary values and the type's largest: results are small, not zero."""
    from fa2.rotary import HeadNorm, rotary_plan, rotary_qk
    D = 64
    g = torch.Generator().manual_seed(2)
    top = torch.finfo(dtype).max
    size = torch.tensor([1.0, 2.0 ** 15, top, top / 2, *([2.0 ** 60, 2.0 ** 100, 2.0 ** 120, 2.0 ** -60] if dtype == torch.bfloat16 else [0.1])],
                        dtype=torch.float64)[:, None, None]
    x = (size * (torch.rand(len(size), 2, D, generator=g, dtype=torch.float64) * 2 - 1)).to(dtype).cuda()
    plan, norm = rotary_plan(48, interleaved=interleaved), HeadNorm(weight_of(D, 3), eps)
    positions = torch.arange(len(x), device="cuda")
    got, _ = rotary_qk(x, None, positions, plan, q_norm=norm)
    want, tol = step_oracle.turn(x, positions, plan.freqs, interleaved, weight=norm.weight, eps=norm.eps)
    assert ((got.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("D,rot,interleaved", [(128, 128, False), (64, 32, True), (32, 16, False), (16, 16, True)])
@pytest.mark.parametrize("axes", [1, 3])
def test_cache_write(dtype, e4m3, D, rot, interleaved, axes):
    """What lands in the cache, its scales, and q; other bytes and rows of no sequence as they were."""
    from fa2.paged import cache_write
    from fa2.rotary import HeadNorm
    page_size, h_q, h_k = 64, 6, 2
    plan = plan_of(rot, axes, interleaved, 1.1)
    for seed, (new, lens) in enumerate([([1, 1, 1], [1, 65, 300]), ([40, 0, 129], [40, 7, 500]), ([17] * 30, [17 + i for i in range(30)])]):
        pages = oracle.Pages(lens, page_size, seed=seed, device="cuda")
        cu, seqlens = cumulative(new), torch.tensor(lens, dtype=torch.int32, device="cuda")
        T = sum(new) + 2
        q, k, v = (randn((T, h, D), dtype, 10 * seed + i, scale=3.0) for i, h in enumerate((h_q, h_k, h_k)))
        norms = dict(q_norm=HeadNorm(weight_of(D, 1), 1e-5), k_norm=HeadNorm(weight_of(D, 2)))
        own = torch.cat([torch.arange(n - m, n) for m, n in zip(new, lens)] + [torch.zeros(2, dtype=torch.int64)]).cuda()
        # by the positions in the sequences (one axis), and by the caller's
        for positions in ([None] if axes == 1 else []) + [positions_of(axes, (T,), seed), positions_of(axes, (T,), seed).int()]:
            for kw in (norms, dict(k_norm=norms["k_norm"]), *([] if positions is None else [{}])):
                cache = make_cache(pages.n_pages, h_k, page_size, D, dtype, e4m3, seed)
                before = [None if t is None else bytes_of(t).clone() for t in cache]
                q_out = torch.full_like(q, 9.0)
                made = cache_write(cache, k, v, pages.table, cu, seqlens, rotary=plan, q=q, q_out=q_out, positions=positions, **kw)
                assert made is q_out and (q_out[-2:] == 9.0).all()
                at = own if positions is None else positions
                check(q_out[:-2], q[:-2], at[..., :-2], plan, kw.get("q_norm"))
                weight, eps = kw.get("k_norm") or (None, 0.0)
                turned, _ = step_oracle.turn(k, at, plan.freqs, interleaved, plan.scale, plan.axes, weight, eps)
                for s, n in enumerate(new):
                    rows = slice(int(cu[s]), int(cu[s + 1]))
                    page, row = pages.at(s, own[rows])
                    if e4m3:
                        for name, x in (("k", turned[rows]), ("v", v[rows].double())):
                            values, e = oracle.to_e4m3(x, dtype)
                            assert torch.equal(getattr(cache, name + "_scale").view(torch.uint8)[page, :, row].long(), (e + 127).long())
                            assert torch.equal(cached(cache, name, page, row), values * torch.exp2(e.double())[..., None])
                    else:
                        check(cached(cache, "k", page, row).to(dtype), k[rows], at[..., rows], plan, kw.get("k_norm"))
                        assert torch.equal(cached(cache, "v", page, row), v[rows].double())
                    for t, was in zip(cache, before):
                        if t is not None:
                            was[page, :, row] = bytes_of(t)[page, :, row]
                assert all(t is None or torch.equal(bytes_of(t), was) for t, was in zip(cache, before))
                assert cache_write(cache, k, v, pages.table, cu, seqlens, rotary=plan, q=q.clone(), positions=positions, **kw).shape == q.shape
                if "q_norm" not in kw:
                    assert cache_write(cache, k, v, pages.table, cu, seqlens, rotary=plan, positions=positions, **kw) is None


def test_cache_write_without_turning_is_as_before():
    """A caller's positions that are the sequences' own, no norm: the bytes of the plain call."""
    from fa2.paged import cache_write
    from fa2.rotary import rotary_plan
    new, lens, D, dtype = [30, 1], [200, 90], 64, torch.bfloat16
    pages = oracle.Pages(lens, 64, device="cuda")
    cu, seqlens = cumulative(new), torch.tensor(lens, dtype=torch.int32, device="cuda")
    q, k, v = (randn((31, h, D), dtype, h) for h in (8, 2, 2))
    own = torch.cat([torch.arange(170, 200), torch.tensor([89])]).cuda()
    for e4m3 in (False, True):
        caches, made = [make_cache(pages.n_pages, 2, 64, D, dtype, e4m3) for _ in range(2)], []
        for cache, positions in zip(caches, (None, own)):
            made.append(cache_write(cache, k, v, pages.table, cu, seqlens, rotary=rotary_plan(64), q=q, positions=positions))
        assert torch.equal(*made)
        assert all(a is None or torch.equal(bytes_of(a), bytes_of(b)) for a, b in zip(*caches))


def test_both_ways_to_the_kernels(monkeypatch):
    from fa2 import _lib
    from fa2.paged import cache_write
    from fa2.rotary import HeadNorm, rotary_qk
    plan, norms = plan_of(64, 3), dict(q_norm=HeadNorm(weight_of(64, 1)), k_norm=HeadNorm(weight_of(64, 2)))
    q, k, v = (randn((40, h, 64), torch.float16, h) for h in (8, 2, 3))
    v = v[:, :2]
    positions = positions_of(3, (40,), 1)
    pages = oracle.Pages([40], 64, device="cuda")
    cu, seqlens = cumulative([40]), torch.tensor([40], dtype=torch.int32, device="cuda")

    def all_of():
        cache = make_cache(pages.n_pages, 2, 64, 64, torch.float16, True)
        q_out = cache_write(cache, k, v, pages.table, cu, seqlens, rotary=plan, q=q, positions=positions, **norms)
        return [*rotary_qk(q, k, positions, plan, **norms), q_out, *map(bytes_of, cache)]
    want = all_of()
    monkeypatch.setattr(_lib, "native", None)
    assert all(torch.equal(a, b) for a, b in zip(all_of(), want))


def test_graph_and_streams():
    """A captured call follows its tensors; calls on two streams at once are each as alone."""
    from fa2.rotary import HeadNorm, rotary_qk
    plan, norms = plan_of(128, 3), dict(q_norm=HeadNorm(weight_of(128, 1)), k_norm=HeadNorm(weight_of(128, 2)))
    q, k, positions = randn((300, 8, 128), torch.bfloat16, 1), randn((300, 2, 128), torch.bfloat16, 2), positions_of(3, (300,), 1)
    rotary_qk(q, k, positions, plan, **norms)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = rotary_qk(q, k, positions, plan, **norms)
    for seed in range(3):
        positions.copy_(positions_of(3, (300,), seed))
        q.copy_(randn(q.shape, q.dtype, seed))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(rotary_qk(q, k, positions, plan, **norms), out))
    calls = [(randn((n, 8, 128), torch.bfloat16, n), randn((n, 2, 128), torch.bfloat16, n), positions_of(3, (n,), n)) for n in (5, 4000)]
    want = [rotary_qk(*c, plan, **norms) for c in calls]
    streams, got = [torch.cuda.Stream() for _ in calls], []
    torch.cuda.synchronize()
    for _ in range(5):
        for c, w, stream in zip(calls, want, streams):
            with torch.cuda.stream(stream):
                got.append((rotary_qk(*c, plan, **norms), w))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g, w in got for a, b in zip(g, w))


@pytest.mark.parametrize("shape", ["packed", "batch"])
def test_most_tokens(shape):
    """As many tokens of one head of 16 as a launch holds threads for, 8 GiB written: every group of tokens is its own, the last,
    partial one too."""
    from fa2.rotary import HeadNorm, rotary_qk
    N, D = 16 * (((1 << 32) - 1) // 256) - 5, 16
    x = randn((1, 1, D), torch.bfloat16, 1)
    plan, norm = plan_of(D, 1), HeadNorm(weight_of(D, 1))
    out = torch.full((N, 1, D), 9.0, dtype=x.dtype, device="cuda")
    positions = torch.tensor([7], device="cuda")  # every token's
    q, o = x.expand(N, 1, D), out
    if shape == "batch":
        q, o = (t.transpose(0, 1).unsqueeze(0) for t in (q, o))
    made, _ = rotary_qk(q, None, positions.expand(N), plan, q_norm=norm, q_out=o)
    assert made is o
    want, _ = rotary_qk(x, None, positions, plan, q_norm=norm)
    check(want, x, positions, plan, norm)
    for rows in out.split(1 << 24):
        assert torch.equal(rows, want.expand(rows.shape))
