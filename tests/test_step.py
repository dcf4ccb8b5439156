"""CPU tests of windows, common prefixes, normalised rotations and a step's pages: the plans of several axes, the oracle's own
pieces, and every refusal, in Python and at the C ABI (which stop before any GPU call)."""

import ctypes
import math
import os

import pytest
import torch

from fa2 import _lib
from fa2.packed import attention_packed
from fa2.paged import KVCache, attention_paged, cache_write
from fa2.pages import PagePool, pages_extend, pages_release
from fa2.rotary import HeadNorm, rotary, rotary_plan, rotary_qk
from oracle import serving as oracle
from oracle import step as step_oracle

needs_lib = pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH), reason="libfa2_fwd.so not built")


# ------------------------------------------------------------------------------------------
# the oracle, and plans
# ------------------------------------------------------------------------------------------

@pytest.mark.parametrize("window,sinks", [(1, 0), (3, 2), (4, 100), (100, 0)])
def test_oracle_window(window, sinks):
    """A row at a time, over the keys that it sees by the definition."""
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(n, h, 16, generator=g, dtype=torch.float64) for n, h in ((5, 4), (9, 2), (9, 2)))
    out, lse, _, _ = oracle.attention(q, k, v, True, None, window, sinks)
    for i in range(5):
        last = i + 4
        keys = [n for n in range(9) if n <= last and (n > last - window or n < sinks)]
        for h in range(4):
            s = k[keys, h // 2] @ q[i, h] / 4.0
            assert torch.allclose(out[i, h], torch.softmax(s, 0) @ v[keys, h // 2], rtol=1e-12)
            assert math.isclose(lse[h, i], torch.logsumexp(s, 0), rel_tol=1e-12)


def test_oracle_turn():
    """Three axes of one position are one axis; a norm leaves heads of root mean square one; pairs turn by their own axis."""
    g = torch.Generator().manual_seed(1)
    x = torch.randn(6, 3, 32, generator=g).half()
    freqs, positions = rotary_plan(32, device="cpu").freqs, torch.arange(6)
    axes = torch.tensor([0, 1, 2, 0] * 4, dtype=torch.int32)
    one, _ = step_oracle.turn(x, positions, freqs)
    assert torch.allclose(one, oracle.rotate(x.transpose(0, 1), positions, freqs).transpose(0, 1), rtol=1e-12)
    assert torch.equal(step_oracle.turn(x, positions.expand(3, 6), freqs, axes=axes)[0], one)
    y, _ = step_oracle.turn(x, positions, freqs, weight=torch.ones(32), eps=0.0)
    assert torch.allclose((y * y).mean(-1), torch.ones(6, 3, dtype=torch.float64), rtol=1e-12)
    apart = torch.stack([positions, torch.zeros_like(positions), torch.zeros_like(positions)])
    z, _ = step_oracle.turn(x, apart, freqs, axes=axes)
    still = (axes != 0).repeat(2)
    assert torch.equal(z[..., still], x.double()[..., still])
    assert torch.equal(z[..., ~still], one[..., ~still])


def test_oracle_pages():
    base, cu, lens, positions, slots, table = step_oracle.extend([7, 3, 5, 9, 0, 0, 0, 0, 0, 0], 4, [[1, -1, -1], [-1, -1, -1]], [4, 0], [2, 5], 4, 8)
    assert (base, cu, lens) == (1, [0, 2, 7], [6, 5]) and table == [[1, 3, -1], [5, 9, -1]]
    assert positions == [4, 5, 0, 1, 2, 3, 4, -1] and slots == [12, 13, 20, 21, 22, 23, 36, -1]
    assert step_oracle.release([7, 0, 0, 0], 1, [[3, -1, 2], [1, 9, 0]], [1, 0], [3, 2]) == ([7, 2, 1, 0], 3)


def test_plan_axes():
    plan = rotary_plan(32, axes=[0] * 4 + [1] * 6 + [2] * 6, device="cpu")
    assert plan.axes.dtype == torch.int32 and plan.axes.tolist() == [0] * 4 + [1] * 6 + [2] * 6
    assert rotary_plan(32, device="cpu").axes is None
    for axes in ([0] * 15, [0] * 17, [-1] + [0] * 15, [0.5] * 16):
        with pytest.raises(ValueError, match="axes"):
            rotary_plan(32, axes=axes, device="cpu")


# ------------------------------------------------------------------------------------------
# refusals in Python
# ------------------------------------------------------------------------------------------

def rows(*shape):
    return torch.zeros(shape, dtype=torch.bfloat16)


def i32(*x):
    return torch.tensor(x, dtype=torch.int32)


def step():
    return KVCache.empty(4, 2, 16, 64, device="cpu"), torch.zeros(1, 2, dtype=torch.int32), i32(0, 3), i32(3)


def test_window_refusals():
    q, k, cu = rows(3, 4, 64), rows(3, 2, 64), i32(0, 3)
    for kw in (dict(window=0), dict(window=-4), dict(window=4, sinks=-1), dict(sinks=4), dict(window=4, causal=False)):
        with pytest.raises(ValueError):
            attention_packed(q, k, k, cu, **kw)
    for kw in (dict(window=4.0), dict(window=4, sinks=1.5), dict(window="4")):
        with pytest.raises(TypeError):
            attention_packed(q, k, k, cu, **kw)
    with pytest.raises(RuntimeError, match="GPU"):
        attention_packed(q, k, k, cu, window=4, sinks=1)
    from fa2.packed import _window
    assert _window(1 << 40, 1 << 40, True) == ((1 << 31) - 1, (1 << 31) - 1) and _window(None, 0, False) == (None, 0)


def test_paged_refusals(monkeypatch):
    """The checks of attention_paged on CPU tensors: the cache's own, of its device, is stepped over."""
    from fa2 import paged
    cache, table, cu, lens = step()
    q = rows(3, 4, 64)
    with pytest.raises(RuntimeError, match="GPU"):
        attention_paged(q, cache, table, cu, lens, window=4)
    monkeypatch.setattr(paged, "_check_cache", lambda cache, dtype: None)
    for kw in (dict(window=0), dict(sinks=1), dict(window=4, causal=False), dict(window=4, shared=i32(3))):
        with pytest.raises(ValueError):
            attention_paged(q, cache, table, cu, lens, **kw)
    for bad in (torch.zeros(1), i32(1, 2), torch.zeros(1, dtype=torch.int64)):
        with pytest.raises(AssertionError, match="shared"):
            attention_paged(q, cache, table, cu, lens, shared=bad)


def test_rotary_qk_refusals():
    q, k, positions, plan = rows(3, 4, 64), rows(3, 2, 64), torch.arange(3), rotary_plan(64, device="cpu")
    norm = HeadNorm(torch.ones(64))
    with pytest.raises(RuntimeError, match="GPU"):
        rotary_qk(q, k, positions, plan)
    with pytest.raises(RuntimeError, match="GPU"):
        rotary(q, positions, plan, norm=norm)
    for bad in (dict(q=q.float()), dict(q=rows(3, 4, 48), k=rows(3, 2, 48)), dict(k=rows(4, 2, 64)), dict(k=rows(3, 2, 32)),
                dict(k=k.half()), dict(k=rows(1, 2, 3, 64)), dict(k=None, k_norm=norm), dict(k=None, k_out=k),
                dict(q_out=q[:2]), dict(k_out=k.half())):
        with pytest.raises(AssertionError):
            rotary_qk(**{"q": q, "k": k, "positions": positions, "plan": plan, **bad})


def test_turn_checks():
    from fa2.rotary import _check_axes, _check_norm, _positions
    cpu, plan = torch.device("cpu"), rotary_plan(64, device="cpu")
    three = rotary_plan(64, axes=[0, 1, 2, 1] * 8, device="cpu")
    assert _check_axes(plan, cpu) is None and _check_norm(None, "q_norm", 64, cpu) is None
    for axes in (three.axes.long(), three.axes[:8], three.axes.view(2, 16)):
        with pytest.raises(AssertionError, match="axes"):
            _check_axes(plan._replace(axes=axes), cpu)
    with pytest.raises(RuntimeError, match="axes"):
        _check_axes(three, torch.device("meta"))
    for weight in (torch.ones(32), torch.ones(64).half(), torch.ones(1, 64)):
        with pytest.raises(AssertionError, match="k_norm"):
            _check_norm(HeadNorm(weight), "k_norm", 64, cpu)
    for eps in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError, match="eps"):
            _check_norm(HeadNorm(torch.ones(64), eps), "q_norm", 64, cpu)
    with pytest.raises(RuntimeError, match="weight"):
        _check_norm(HeadNorm(torch.ones(64)), "q_norm", 64, torch.device("meta"))
    assert _positions(torch.arange(5), plan, 2, 5, False).shape == (1, 2, 5)
    assert _positions(torch.zeros(3, 2, 5, dtype=torch.int32), three, 2, 5, False).shape == (3, 2, 5)
    assert _positions(torch.zeros(3, 5, dtype=torch.int32), three, 1, 5, True).shape == (3, 1, 5)
    for positions, p in ((torch.arange(4), plan), (torch.zeros(2, 5, dtype=torch.int32), plan), (torch.arange(5), three),
                         (torch.zeros(0, 5, dtype=torch.int32), three), (torch.arange(5.0), plan)):
        with pytest.raises(AssertionError, match="positions"):
            _positions(positions, p, 1, 5, True)


def test_cache_write_refusals(monkeypatch):
    from fa2 import paged
    cache, table, cu, lens = step()
    monkeypatch.setattr(paged, "_check_cache", lambda cache, dtype: None)
    k, q, plan, norm = rows(3, 2, 64), rows(3, 4, 64), rotary_plan(64, device="cpu"), HeadNorm(torch.ones(64))
    three = rotary_plan(64, axes=[0, 1, 2, 1] * 8, device="cpu")
    for kw in (dict(k_norm=norm), dict(positions=torch.arange(3)), dict(rotary=plan, q_norm=norm),
               dict(rotary=plan, positions=torch.arange(4)), dict(rotary=three, positions=torch.arange(3)),
               dict(rotary=plan, k_norm=HeadNorm(torch.ones(32)))):
        with pytest.raises(AssertionError):
            cache_write(cache, k, k, table, cu, lens, **kw)
    for kw in (dict(rotary=three), dict(rotary=plan, q=q, q_norm=HeadNorm(torch.ones(64), 0.0))):
        with pytest.raises(ValueError):
            cache_write(cache, k, k, table, cu, lens, **kw)


def test_pages_refusals():
    pool, table, lens = PagePool.full(8, device="cpu"), torch.zeros(2, 3, dtype=torch.int32), i32(1, 2)
    assert pool.free.tolist() == list(range(8)) and pool.count.tolist() == [8]
    with pytest.raises(RuntimeError, match="GPU"):
        pages_extend(pool, table, lens, lens, 16, 3)
    with pytest.raises(RuntimeError, match="GPU"):
        pages_release(pool, table, lens, lens)
    for bad in (pool._replace(free=pool.free.long()), pool._replace(free=pool.free.view(2, 4)), pool._replace(count=i32(1, 2)),
                pool._replace(count=torch.ones(1))):
        for call in (lambda: pages_extend(bad, table, lens, lens, 16, 3), lambda: pages_release(bad, table, lens, lens)):
            with pytest.raises(AssertionError, match="pool"):
                call()
    for bad in (table.long(), table[0]):
        with pytest.raises(AssertionError, match="block_table"):
            pages_extend(pool, bad, lens, lens, 16, 3)


def test_pages_checks(monkeypatch):
    """The checks behind the device's."""
    from fa2 import pages
    pool, table, lens = PagePool.full(8, device="cpu"), torch.zeros(2, 3, dtype=torch.int32), i32(1, 2)
    monkeypatch.setattr(pages, "_check", lambda pool, table: torch.device("cpu"))
    for page_size in (0, 3, -16, 1 << 21):
        with pytest.raises(ValueError, match="page_size"):
            pages_extend(pool, table, lens, lens, page_size, 3)
    with pytest.raises(ValueError, match="n_tokens"):
        pages_extend(pool, table, lens, lens, 16, -1)
    with pytest.raises(AssertionError):
        pages_extend(pool, table, lens[:1], lens, 16, 3)
    with pytest.raises(AssertionError):
        pages_extend(pool, table, lens.long(), lens.long(), 16, 3)
    with pytest.raises(AssertionError):
        pages_release(pool, table, lens, lens[:1])


# ------------------------------------------------------------------------------------------
# refusals of the C ABI: no pointer here is read, every call stops at the checks or has nothing to do
# ------------------------------------------------------------------------------------------

P = 1 << 20  # a 16-byte aligned address that nothing reads


def c_cache(**kw):
    c = _lib.Cache(P, P, None, None, (2048, 1024, 64), (2048, 1024, 64), (0, 0, 0), (0, 0, 0), 4, 2, 16, 64, 1)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def c_seq(**kw):
    s = _lib.Sequences(P, P, P, 2, 2, 3, 2)
    for k, v in kw.items():
        setattr(s, k, v)
    return s


def c_turn(**kw):
    t = _lib.Turn(_lib.Rotation(P, 32, 0, 1.0), None, None, None, 0.0, 0.0, 1)
    for k, v in kw.items():
        setattr(t, k, v)
    return t


def strides(*s):
    return (ctypes.c_int64 * len(s))(*s)


@needs_lib
def test_c_window_refusals():
    s = strides(256, 64)

    def packed(window=4, sinks=0, q=P, n=3, h_q=4, scale=0.1):
        return _lib.lib().fa2_attn_packed_window(q, P, P, P, s, s, s, s, P, None, 2, n, n, h_q, 4, 64, 1, window, sinks, scale, None, None)

    def paged(window=4, sinks=0, q=P, n=3, h_q=4, cache=c_cache(), **seq):
        return _lib.lib().fa2_attn_paged_window(q, P, s, s, ctypes.byref(cache), ctypes.byref(c_seq(n_tokens=n, **seq)), h_q, 1,
                                                window, sinks, 0.1, None, None, 0, None)
    for call in (packed, paged):
        for kw in (dict(window=0), dict(window=-1), dict(sinks=-1), dict(q=None), dict(h_q=3)):
            assert call(**kw) == -1 and _lib.last_error(), kw
        assert call(q=P + 8) == -2
        assert call(n=0) == 0 and _lib.last_error() == ""
    assert packed(scale=0.0) == -1
    long = dict(max_pages=4096, table_stride=4096)
    assert paged(window=2000, **long) == -1 and "workspace" in _lib.last_error()
    need = _lib.paged_window_workspace_bytes(4, 2, 64, torch.bfloat16, 3, 2, 4096 * 16, 2000, 0, 256)
    assert need == _lib.paged_workspace_bytes(4, 2, 64, torch.bfloat16, 3, 2, 4096 * 16, 256) > 0
    assert _lib.paged_window_workspace_bytes(4, 2, 64, torch.bfloat16, 3, 2, 4096 * 16, 500, 4, 256) == 0  # few keys: none are shared
    assert _lib.paged_window_workspace_bytes(4, 2, 64, torch.bfloat16, 3, 2, 4096 * 16, 0, 0, 256) == 0
    assert paged(cache=c_cache(page_size=24)) == -1


@needs_lib
def test_c_shared_refusals():
    s = strides(256, 64)

    def shared(n=P, q=P, ws=P, n_ws=1 << 40, h_q=4, tokens=3, **seq):
        return _lib.lib().fa2_attn_paged_shared(q, P, s, s, ctypes.byref(c_cache()), ctypes.byref(c_seq(n_tokens=tokens, **seq)), n, h_q,
                                                1, 1, 0.1, None, ws, n_ws, None)
    assert shared(n=None) == -1 and "shared" in _lib.last_error()
    assert shared(n=P + 2) == -2
    assert shared(q=None) == -1 and shared(h_q=3) == -1 and shared(lens=None) == -1
    need = _lib.paged_shared_workspace_bytes(4, 2, 64, 3, 2, 256)
    assert need >= 2 * 3 * 4 * 68 * 4  # a row's results over the prefix and behind it, in float
    assert shared(ws=None) == -1 and str(need) in _lib.last_error()
    assert shared(n_ws=need - 1) == -1 and str(need) in _lib.last_error()
    assert shared(ws=P + 128) == -2
    assert shared(tokens=0) == 0 and shared(n_seq=0) == 0
    for h_q, D, n, n_seq, cus in ((3, 64, 3, 2, 256), (4, 48, 3, 2, 256), (4, 64, 0, 2, 256), (4, 64, 3, 0, 256), (4, 64, 3, 2, 0)):
        assert _lib.paged_shared_workspace_bytes(h_q, 2, D, n, n_seq, cus) == 0


BAD_TURNS = [(dict(n_axes=0), -1), (dict(n_axes=3), -1), (dict(axes=P + 2, n_axes=3), -2), (dict(q_weight=P + 2, q_eps=1e-6), -2),
             (dict(q_weight=P), -1), (dict(k_weight=P, k_eps=-1.0), -1), (dict(k_weight=P, k_eps=math.inf), -1),
             (dict(rotation=_lib.Rotation(None, 32, 0, 1.0)), -2), (dict(rotation=_lib.Rotation(P, 12, 0, 1.0)), -1),
             (dict(rotation=_lib.Rotation(P, 40, 0, 1.0)), -1), (dict(rotation=_lib.Rotation(P, 32, 0, math.nan)), -1)]


@needs_lib
def test_c_rotary_qk_refusals():
    r = strides(768, 64, 256)

    def qk(q=P, k=P, qo=P, ko=P, st=r, so=r, pos=P, size=8, turn=c_turn(), B=1, h_q=4, h_k=4, n=3, D=64, dtype=1):
        return _lib.lib().fa2_rotary_qk(q, k, qo, ko, st, r, so, r, pos, size, strides(0, 0, 1),
                                        None if turn is None else ctypes.byref(turn), B, h_q, h_k, n, D, dtype, None)
    for kw in (dict(q=None), dict(k=None), dict(qo=None), dict(ko=None), dict(pos=None), dict(size=2), dict(turn=None), dict(B=-1),
               dict(h_q=-1), dict(h_k=-1), dict(n=-1), dict(D=24), dict(dtype=2), dict(so=strides(768, 0, 256)), dict(h_q=1 << 25)):
        assert qk(**kw) == -1 and _lib.last_error(), kw
    for turn, code in BAD_TURNS:
        assert qk(turn=c_turn(**turn)) == code and _lib.last_error(), turn
    assert qk(q=P + 4) == -2 and qk(pos=P + 4) == -2 and qk(st=strides(768, 60, 256)) == -2
    assert qk(B=0) == 0 and qk(n=0) == 0 and qk(h_q=0, h_k=0) == 0


@needs_lib
def test_c_cache_write_turned_refusals():
    s = strides(128, 64)

    def write(k=P, q=None, qo=None, h_q=4, pos=None, size=0, turn=c_turn(), cache=c_cache(), **seq):
        return _lib.lib().fa2_cache_write_turned(ctypes.byref(cache), ctypes.byref(c_seq(**seq)), k, P, s, s, q, qo, s, s, h_q, pos, size,
                                                 strides(0, 1), None if turn is None else ctypes.byref(turn), 1, None)
    assert write(turn=None) == -1 and write(k=None) == -1 and write(q=P, qo=None) == -1 and write(q=P, qo=P, h_q=0) == -1
    assert write(pos=P, size=2) == -1 and write(pos=P + 4, size=8) == -2
    assert write(turn=c_turn(axes=P, n_axes=3)) == -1 and "positions" in _lib.last_error()
    for turn, code in BAD_TURNS:
        assert write(turn=c_turn(**turn)) == code and _lib.last_error(), turn
    assert write(cache=c_cache(v_stride=(0, 1024, 64))) == -1 and "stride of 0" in _lib.last_error()
    assert write(n_tokens=0) == 0 and write(n_seq=0) == 0


@needs_lib
def test_c_pages_refusals():
    def extend(free=P, n_pages=8, count=P, out=P, table=P, stride=3, n_seq=2, columns=3, page=16, lens=P, new=P, after=P, cu=P,
               pos=P, slots=P, n=4):
        return _lib.lib().fa2_pages_extend(free, n_pages, count, out, table, stride, n_seq, columns, page, lens, new, after, cu, pos, slots,
                                           n, None)
    for kw in (dict(free=None), dict(count=None), dict(out=None), dict(table=None), dict(lens=None), dict(new=None), dict(after=None),
               dict(cu=None), dict(pos=None), dict(slots=None), dict(n_pages=-1), dict(stride=-1), dict(stride=0), dict(n_seq=0),
               dict(columns=-1), dict(page=0), dict(page=24), dict(page=1 << 21), dict(n=-1)):
        assert extend(**kw) == -1 and _lib.last_error(), kw
    for kw in (dict(free=P + 2), dict(table=P + 1), dict(slots=P + 4), dict(cu=P + 2)):
        assert extend(**kw) == -2 and _lib.last_error(), kw

    def release(free=P, n_pages=8, count=P, out=P, table=P, stride=3, n_seq=2, columns=3, first=P, last=P, ws=P):
        return _lib.lib().fa2_pages_release(free, n_pages, count, out, table, stride, n_seq, columns, first, last, ws, None)
    for kw in (dict(free=None), dict(count=None), dict(out=None), dict(table=None), dict(first=None), dict(last=None), dict(ws=None),
               dict(n_pages=-1), dict(stride=-1), dict(n_seq=0), dict(columns=-1)):
        assert release(**kw) == -1 and _lib.last_error(), kw
    assert release(last=P + 2) == -2 and release(ws=P + 1) == -2
