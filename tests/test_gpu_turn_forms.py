"""GPU tests of how normalised rotations and turned cache writes are dealt to workgroups, against float64: a token's rows over
several workgroups, several passes over its heads in one, several tokens in one with a last group that is not full."""

import pytest
import torch

from oracle import serving as oracle
from oracle import step as step_oracle
from serving_check import bytes_of, cached, cumulative, make_cache, randn
from test_gpu_turn import DTYPES, check, plan_of, positions_of, weight_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,rot,h_q,h_k", [(128, 128, 32, 8), (128, 64, 28, 4), (64, 64, 40, 40), (16, 16, 150, 3)])
def test_rotary_qk(dtype, interleaved, D, rot, h_q, h_k):
    """More heads than a pass takes: a workgroup a pass (few tokens), or all of a token's in one (from 512 workgroups on), with a
    token a workgroup and with several."""
    from fa2.rotary import HeadNorm, rotary_qk
    plan, norms = plan_of(rot, 3, interleaved), (HeadNorm(weight_of(D, 7)), HeadNorm(weight_of(D, 8), 1e-5))
    for T in (5, 511, 700, 2500, 5001):
        q, k = randn((T, h_q, D), dtype, T), randn((T, h_k, D), dtype, T + 1, scale=5.0)
        positions = positions_of(3, (T,), T)
        for q_norm, k_norm in ((norms[0], norms[1]), (norms[0], None)):
            got_q, got_k = rotary_qk(q, k, positions, plan, q_norm=q_norm, k_norm=k_norm)
            check(got_q, q, positions, plan, q_norm)
            check(got_k, k, positions, plan, k_norm)
        mine = q.clone(), k.clone()
        rotary_qk(*mine, positions, plan, q_norm=q_norm, k_norm=k_norm, q_out=mine[0], k_out=mine[1])
        assert torch.equal(mine[0], got_q) and torch.equal(mine[1], got_k)
    B = 3  # groups of tokens end with their batch row
    q, k, positions = (t[:4998] for t in (q, k, positions.t()))
    q, k = (t.view(B, 1666, -1, D).transpose(1, 2) for t in (q, k))
    positions = positions.view(B, 1666, 3).permute(2, 0, 1)
    both = rotary_qk(q, k, positions, plan, q_norm=q_norm, k_norm=k_norm)
    assert all(torch.equal(b.transpose(1, 2).reshape(4998, -1, D), g[:4998]) for b, g in zip(both, (got_q, got_k)))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("D,rot,interleaved,h_q,h_k", [(128, 128, False, 32, 8), (128, 64, True, 28, 4), (64, 64, False, 40, 40),
                                                      (16, 16, True, 130, 3)])
def test_cache_write(dtype, e4m3, D, rot, interleaved, h_q, h_k):
    """Heads that take several passes: of few tokens, dealt to several workgroups; of 700, in one workgroup a token; of more, in
    one of several tokens, whose scales are stored together."""
    from fa2.paged import cache_write
    from fa2.rotary import HeadNorm
    page_size = 64
    plan = plan_of(rot, 3, interleaved, 1.1)
    norms = dict(q_norm=HeadNorm(weight_of(D, 1), 1e-5), k_norm=HeadNorm(weight_of(D, 2)))
    for seed, (new, lens) in enumerate([([1, 1, 3], [1, 65, 300]), ([300, 0, 400], [300, 7, 450]), ([3000, 17, 1], [3010, 17, 65]),
                                        ([9000, 41], [9000, 50])]):
        pages = oracle.Pages(lens, page_size, seed=seed, device="cuda")
        cu, seqlens = cumulative(new), torch.tensor(lens, dtype=torch.int32, device="cuda")
        T = sum(new) + 2
        q, k, v = (randn((T, h, D), dtype, 10 * seed + i, scale=3.0) for i, h in enumerate((h_q, h_k, h_k)))
        positions = positions_of(3, (T,), seed)
        cache = make_cache(pages.n_pages, h_k, page_size, D, dtype, e4m3, seed)
        before = [None if t is None else bytes_of(t).clone() for t in cache]
        q_out = torch.full_like(q, 9.0)
        cache_write(cache, k, v, pages.table, cu, seqlens, rotary=plan, q=q, q_out=q_out, positions=positions, **norms)
        assert (q_out[-2:] == 9.0).all()
        check(q_out[:-2], q[:-2], positions[:, :-2], plan, norms["q_norm"])
        turned, _ = step_oracle.turn(k, positions, plan.freqs, interleaved, plan.scale, plan.axes, *norms["k_norm"])
        for s, (n, length) in enumerate(zip(new, lens)):
            rows = slice(int(cu[s]), int(cu[s + 1]))
            page, row = pages.at(s, torch.arange(length - n, length, device="cuda"))
            if e4m3:
                for name, x in (("k", turned[rows]), ("v", v[rows].double())):
                    values, e = oracle.to_e4m3(x, dtype)
                    assert torch.equal(getattr(cache, name + "_scale").view(torch.uint8)[page, :, row].long(), (e + 127).long())
                    assert torch.equal(cached(cache, name, page, row), values * torch.exp2(e.double())[..., None])
            else:
                check(cached(cache, "k", page, row).to(dtype), k[rows], positions[:, rows], plan, norms["k_norm"])
                assert torch.equal(cached(cache, "v", page, row), v[rows].double())
            for t, was in zip(cache, before):
                if t is not None:
                    was[page, :, row] = bytes_of(t)[page, :, row]
        assert all(t is None or torch.equal(bytes_of(t), was) for t, was in zip(cache, before))
        mine = q.clone()
        assert cache_write(cache, k, v, pages.table, cu, seqlens, rotary=plan, q=mine, q_out=mine, positions=positions, **norms) is mine
        assert torch.equal(mine[:-2], q_out[:-2]) and torch.equal(mine[-2:], q[-2:])
