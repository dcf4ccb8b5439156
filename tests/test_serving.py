"""CPU tests of the serving operators: the frequencies of scaled rotations, the oracle's own pieces, and every
refusal, in Python and at the C ABI (which stop before any GPU call).
"""

import ctypes
import math
import os

import pytest
import torch

from fa2 import _lib
from fa2.packed import attention_packed
from fa2.paged import KVCache, attention_paged, cache_read, cache_write
from fa2.rotary import Rotary, rotary, rotary_plan
from oracle import serving as oracle

needs_lib = pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH), reason="libfa2_fwd.so not built")


# ------------------------------------------------------------------------------------------
# frequencies
# ------------------------------------------------------------------------------------------

def test_rotary_plan_frequencies():
    plan = rotary_plan(64, 10000.0, device="cpu")
    assert plan.freqs.dtype == torch.float64 and plan.freqs.shape == (32,) and plan.scale == 1.0
    assert plan.freqs[0] == 1.0
    assert torch.allclose(plan.freqs.log(), -torch.arange(32, dtype=torch.float64) * math.log(10000.0) / 32, rtol=1e-14)
    linear = rotary_plan(64, scaling="linear", factor=4.0, device="cpu")
    assert torch.equal(linear.freqs, plan.freqs / 4)
    base = rotary_plan(64, scaling="base", factor=4.0, device="cpu").freqs
    assert base[0] == 1.0 and math.isclose(base[-1], plan.freqs[-1] / 4, rel_tol=1e-12)


@pytest.mark.parametrize("scaling", ["blend", "smooth"])
def test_rotary_plan_keeps_fast_pairs(scaling):
    plain = rotary_plan(128, device="cpu").freqs
    plan = rotary_plan(128, scaling=scaling, factor=8.0, trained_length=4096, device="cpu")
    turns = 4096 * plain / (2 * math.pi)
    ratio = plan.freqs / plain
    assert torch.equal(ratio[turns >= 40], torch.ones_like(ratio[turns >= 40]))
    assert torch.allclose(ratio[turns <= 0.8], torch.full_like(ratio[turns <= 0.8], 1 / 8), rtol=1e-14)
    assert (ratio.diff() <= 1e-15).all()  # the slower, the more stretched
    assert plan.scale == (0.1 * math.log(8.0) + 1.0 if scaling == "blend" else 1.0)
    same = rotary_plan(128, scaling=scaling, factor=1.0, trained_length=4096, device="cpu")
    assert torch.allclose(same.freqs, plain, rtol=1e-14) and same.scale == 1.0


@pytest.mark.parametrize("kw", [dict(rot_dim=24), dict(rot_dim=0), dict(base=1.0), dict(factor=0.0), dict(scaling="other"),
                                dict(scaling="blend", factor=2.0), dict(scaling="smooth", trained_length=0),
                                dict(scaling="blend", trained_length=100, fast=1.0, slow=2.0)])
def test_rotary_plan_refuses(kw):
    with pytest.raises(ValueError):
        rotary_plan(**{"rot_dim": 64, "device": "cpu", **kw})


# ------------------------------------------------------------------------------------------
# the oracle
# ------------------------------------------------------------------------------------------

def test_oracle_rotation_keeps_norms_and_differences():
    """Rotated by m and n, a query and a key meet as if by m - n and 0."""
    g = torch.Generator().manual_seed(0)
    q, k = torch.randn(1, 1, 32, generator=g), torch.randn(1, 1, 32, generator=g)
    freqs = rotary_plan(32, device="cpu").freqs
    for inter in (False, True):
        a, b = (oracle.rotate(t, torch.tensor([p]), freqs, inter) for t, p in ((q, 117), (k, 100)))
        c, d = (oracle.rotate(t, torch.tensor([p]), freqs, inter) for t, p in ((q, 17), (k, 0)))
        assert torch.allclose((a * b).sum(), (c * d).sum(), rtol=1e-12)
        assert torch.allclose(a.norm(), q.double().norm(), rtol=1e-12)


def test_oracle_e4m3_is_the_types_rounding():
    """Against torch's conversion wherever no saturation is involved, and 2^e the least that holds the row."""
    g = torch.Generator().manual_seed(0)
    x = torch.randn(500, 32, generator=g).double() * torch.exp2(torch.randint(-20, 20, (500, 1), generator=g).double())
    values, e = oracle.to_e4m3(x, torch.bfloat16)
    y = x * torch.exp2(-e.double())[:, None]
    assert torch.equal(values, y.float().to(torch.float8_e4m3fn).double())
    top = x.abs().amax(1)
    assert (top <= 448 * torch.exp2(e.double())).all() and (top > 448 * torch.exp2(e.double() - 1)).all()


def test_oracle_attention_matches_plain_softmax():
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(n, h, 16, generator=g) for n, h in ((5, 4), (9, 2), (9, 2)))
    out, lse, _, _ = oracle.attention(q, k, v, True)
    s = torch.einsum("nhd,mhd->hnm", q.double(), k.double().repeat_interleave(2, 1)) / 4
    s.masked_fill_(torch.arange(9) > torch.arange(5)[:, None] + 4, -math.inf)
    assert torch.allclose(lse, s.logsumexp(-1))
    assert torch.allclose(out, torch.einsum("hnm,mhd->nhd", s.softmax(-1), v.double().repeat_interleave(2, 1)))
    v[7, 0, 3] = math.nan  # seen by the rows from 3 on
    out = oracle.attention(q, k, v, True)[0]
    assert out[3:, :2, 3].isnan().all() and out.isnan().sum() == 4


# ------------------------------------------------------------------------------------------
# refusals in Python
# ------------------------------------------------------------------------------------------

def cpu_step(e4m3=False, D=64, page_size=16, dtype=torch.bfloat16):
    cache = KVCache.empty(4, 2, page_size, D, torch.float8_e4m3fn if e4m3 else dtype, device="cpu")
    table = torch.zeros(2, 2, dtype=torch.int32)
    cu, lens = torch.tensor([0, 1, 3], dtype=torch.int32), torch.tensor([5, 9], dtype=torch.int32)
    return cache, table, cu, lens


def test_cpu_tensors_fail_loudly():
    x = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    cache, table, cu, lens = cpu_step()
    with pytest.raises(RuntimeError, match="GPU"):
        rotary(x, torch.arange(3), rotary_plan(64, device="cpu"))
    with pytest.raises(RuntimeError, match="GPU"):
        attention_packed(x, x, x, cu)
    for call in (lambda: cache_write(cache, x, x, table, cu, lens), lambda: cache_read(cache, table, cu, lens, 3),
                 lambda: attention_paged(x, cache, table, cu, lens)):
        with pytest.raises(RuntimeError, match="GPU"):
            call()


@pytest.mark.parametrize("bad", ["rank", "dtype", "head_dim", "gqa", "kv_shape", "kv_rows", "cu_dtype", "cu_empty", "cu_kv"])
def test_packed_refuses(bad):
    q, k = torch.zeros(3, 4, 64, dtype=torch.float16), torch.zeros(3, 2, 64, dtype=torch.float16)
    v, cu, cu_kv = k, torch.tensor([0, 3], dtype=torch.int32), None
    if bad == "rank":
        q = q[None]
    elif bad == "dtype":
        k = v = k.bfloat16()
    elif bad == "head_dim":
        q, k, v = (t[..., :48] for t in (q, k, v))
    elif bad == "gqa":
        q = q[:, :3]
    elif bad == "kv_shape":
        v = v[:2]
    elif bad == "kv_rows":
        k = v = k[:2]
    elif bad == "cu_empty":
        cu = cu[:0]
    elif bad == "cu_kv":
        cu_kv = cu[:1]
    elif bad == "cu_dtype":
        from fa2.packed import _index
        with pytest.raises(AssertionError):
            _index(cu.long(), "cu_seqlens", cu.device)
        with pytest.raises(AssertionError):
            _index(cu[None], "cu_seqlens", cu.device)
        return
    with pytest.raises(AssertionError):
        attention_packed(q, k, v, cu, cu_kv)
    with pytest.raises(ValueError, match="sm_scale"):
        attention_packed(torch.zeros(3, 4, 64, dtype=torch.float16), *[torch.zeros(3, 2, 64, dtype=torch.float16)] * 2,
                         torch.tensor([0, 3], dtype=torch.int32), sm_scale=0.0)


def test_cache_refuses():
    """What a cache must be is checked before anything else of a call."""
    from fa2.paged import _check_cache
    good = cpu_step()[0]
    with pytest.raises(AssertionError, match="own type"):
        _check_cache(good, torch.float16)
    with pytest.raises(AssertionError, match="shape"):
        _check_cache(good._replace(v=good.v[:2]), torch.bfloat16)
    for shape in ((4, 2, 24, 64), (4, 2, 8, 128), (4, 2, 16, 16), (0, 2, 16, 64)):
        t = torch.zeros(shape, dtype=torch.bfloat16)
        with pytest.raises(ValueError, match="page_size"):
            _check_cache(KVCache(t, t), torch.bfloat16)
    t = torch.zeros(4, 2, 16, 72, dtype=torch.bfloat16)[..., :64]
    _strided = torch.zeros(4, 2, 16, 68, dtype=torch.bfloat16)[..., :64]
    with pytest.raises(ValueError, match="stride"):
        _check_cache(KVCache(t, _strided), torch.bfloat16)
    e4m3 = cpu_step(True)[0]
    with pytest.raises(AssertionError, match="k_scale"):
        _check_cache(e4m3._replace(k_scale=None), torch.bfloat16)
    with pytest.raises(AssertionError, match="v_scale"):
        _check_cache(e4m3._replace(v_scale=e4m3.v_scale.view(torch.uint8)), torch.bfloat16)
    with pytest.raises(AssertionError):
        KVCache.empty(4, 2, 16, 64, torch.float32, device="cpu")
    with pytest.raises(AssertionError, match="dtype"):
        cache_read(e4m3, *cpu_step()[1:], 3)


def test_plan_and_position_refusals():
    from fa2.rotary import _check_plan
    cpu = torch.device("cpu")
    for n in (0, 4, 40):
        with pytest.raises(ValueError, match="rotation covers"):
            _check_plan(Rotary(torch.ones(n, dtype=torch.float64)), 64, cpu)
    with pytest.raises(AssertionError, match="float64"):
        _check_plan(Rotary(torch.ones(32)), 64, cpu)
    with pytest.raises(ValueError, match="scale"):
        _check_plan(Rotary(torch.ones(32, dtype=torch.float64), False, math.inf), 64, cpu)
    x = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    plan = rotary_plan(64, device="cpu")
    for positions in (torch.arange(3.0), torch.arange(4), torch.zeros(3, 1, dtype=torch.int64)):
        with pytest.raises(AssertionError):
            rotary(x, positions, plan)
    with pytest.raises(AssertionError):
        rotary(x.float(), torch.arange(3), plan)
    with pytest.raises(AssertionError):
        rotary(x, torch.arange(3), plan, out=torch.zeros(3, 2, 64, dtype=torch.float16))


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


def strides(*s):
    return (ctypes.c_int64 * len(s))(*s)


def write(cache, seq, k=P, dtype=1, q=None, q_out=None, rotation=None, h_q=4, ks=None):
    s = strides(128, 64)
    return _lib.lib().fa2_cache_write(ctypes.byref(cache), ctypes.byref(seq), k, P, ks or s, s, q, q_out, s, s, h_q,
                                      None if rotation is None else ctypes.byref(rotation), dtype, None)


def paged(cache, seq, q=P, dtype=1, h_q=4, scale=0.1, lse=None, ws=P, n_ws=1 << 40):
    s = strides(256, 64)
    return _lib.lib().fa2_attn_paged(q, P, s, s, ctypes.byref(cache), ctypes.byref(seq), h_q, dtype, 1, scale, lse, ws, n_ws, None)


@needs_lib
@pytest.mark.parametrize("change,code", [
    (dict(cache_dtype=0), -1), (dict(cache_dtype=3), -1), (dict(cache_dtype=2), -1), (dict(n_pages=0), -1),
    (dict(h_kv=0), -1), (dict(page_size=24), -1), (dict(page_size=8), -1), (dict(page_size=1 << 21), -1),
    (dict(head_dim=48), -1), (dict(head_dim=16), -1), (dict(k=None), -1), (dict(v=P + 8), -2),
    (dict(k_stride=(2048, 1024, 60)), -2), (dict(v_stride=(-2048, 1024, 64)), -2), (dict(k_stride=(2048, 1024, 1 << 23)), -1),
    (dict(cache_dtype=2, k_scale=P, v_scale=P, k_stride=(2048, 1024, 72)), -2),
    (dict(cache_dtype=2, k_scale=P, v_scale=P, k_scale_stride=(-1, 0, 0)), -1),
    (dict(cache_dtype=2, k_scale=P, v_scale=P, v_scale_stride=(32, 16, 1 << 23)), -1)])
def test_c_cache_refusals(change, code):
    cache = c_cache(**change)
    s = strides(128, 64)
    assert write(cache, c_seq()) == code and _lib.last_error()
    assert paged(cache, c_seq()) == code and _lib.last_error()
    assert _lib.lib().fa2_cache_read(ctypes.byref(cache), ctypes.byref(c_seq()), P, P, s, s, 1, None) == code


@needs_lib
@pytest.mark.parametrize("change", [dict(n_seq=-1), dict(n_tokens=-1), dict(max_pages=-1), dict(table_stride=-1),
                                    dict(max_pages=1 << 27), dict(cu=None), dict(lens=None), dict(table=None)])
def test_c_sequences_refusals(change):
    assert write(c_cache(), c_seq(**change)) == -1 and _lib.last_error()
    assert paged(c_cache(), c_seq(**change)) == -1 and _lib.last_error()


@needs_lib
def test_c_call_refusals():
    rot = _lib.Rotation(P, 32, 0, 1.0)
    assert write(c_cache(), c_seq(), k=P + 2) == -2
    assert write(c_cache(), c_seq(), ks=strides(130, 64)) == -2
    assert write(c_cache(), c_seq(), dtype=2) == -1
    assert write(c_cache(), c_seq(), q=P, q_out=P) == -1  # no rotation
    assert write(c_cache(), c_seq(), q=P, q_out=None, rotation=rot) == -1
    assert write(c_cache(), c_seq(), q=P, q_out=P, rotation=rot, h_q=0) == -1
    for bad in (_lib.Rotation(P, 4, 0, 1.0), _lib.Rotation(P, 36, 0, 1.0), _lib.Rotation(P, 40, 0, 1.0),
                _lib.Rotation(P, 2 ** 31 - 8, 0, 1.0), _lib.Rotation(P, 32, 0, math.inf)):
        assert write(c_cache(), c_seq(), rotation=bad) == -1
    assert write(c_cache(), c_seq(), rotation=_lib.Rotation(P + 4, 32, 0, 1.0)) == -2
    assert paged(c_cache(), c_seq(), h_q=3) == -1 and "GQA" in _lib.last_error()
    assert paged(c_cache(), c_seq(), h_q=0) == -1
    assert paged(c_cache(), c_seq(), scale=0.0) == -1 and "qk_scale" in _lib.last_error()
    assert paged(c_cache(), c_seq(), scale=math.inf) == -1
    assert paged(c_cache(), c_seq(), q=None) == -1
    assert paged(c_cache(), c_seq(), lse=P + 2) == -2
    assert paged(c_cache(), c_seq(n_tokens=1 << 30), h_q=8) == -1  # 2^32 rows of a KV head
    need = _lib.paged_workspace_bytes(4, 2, 64, torch.bfloat16, 3, 2, 4096, 256)
    assert need > 0
    long = c_seq(max_pages=256, table_stride=256)  # (the two pages of c_seq() need none)
    assert paged(c_cache(), long, ws=None) == -1 and "workspace" in _lib.last_error()
    assert paged(c_cache(), long, n_ws=need - 1) == -1 and str(need) in _lib.last_error()
    assert paged(c_cache(), long, ws=P + 128) == -2
    for h_q, D, n, n_seq, cus in ((3, 64, 3, 2, 256), (4, 48, 3, 2, 256), (4, 64, 0, 2, 256), (4, 64, 3, 0, 256), (4, 64, 3, 2, 0)):
        assert _lib.paged_workspace_bytes(h_q, 2, D, torch.bfloat16, n, n_seq, 4096, cus) == 0
    assert _lib.paged_workspace_bytes(4, 2, 64, torch.bfloat16, 3, 2, 1536, 256) == 0  # no sequence is long enough
    assert _lib.paged_workspace_bytes(32, 8, 128, torch.float8_e4m3fn, 1 << 20, 4, 1 << 20, 256) == 0  # row tiles enough: none are shared
    assert _lib.lib().fa2_cache_write(None, None, P, P, None, None, None, None, None, None, 0, None, 1, None) == -1
    # rows that are written have places of their own
    for stride in ((0, 1024, 64), (2048, 0, 64), (2048, 1024, 0)):
        assert write(c_cache(v_stride=stride), c_seq()) == -1 and "stride of 0" in _lib.last_error()
    e4m3 = dict(cache_dtype=2, k_scale=P, v_scale=P, v_scale_stride=(32, 16, 1))
    assert write(c_cache(**e4m3), c_seq()) == -1 and "stride of 0" in _lib.last_error()
    s, one = strides(256, 64), strides(0, 64)
    assert _lib.lib().fa2_cache_read(ctypes.byref(c_cache()), ctypes.byref(c_seq()), P, P, s, one, 1, None) == -1
    assert _lib.lib().fa2_attn_paged(P, P, s, one, ctypes.byref(c_cache()), ctypes.byref(c_seq()), 4, 1, 1, 0.1, None, None,
                                     0, None) == -1 and "stride of 0" in _lib.last_error()
    assert _lib.lib().fa2_attn_packed(P, P, P, P, s, s, s, one, P, None, 2, 3, 3, 4, 4, 64, 1, 1, 0.1, None, None) == -1
    three = strides(768, 64, 0)
    assert _lib.lib().fa2_rotary(P, P, strides(768, 64, 256), three, P, 4, strides(0, 1), ctypes.byref(rot), 1, 4, 3, 64, 1,
                                 None) == -1 and "stride of 0" in _lib.last_error()
    # nothing to do
    assert write(c_cache(), c_seq(n_tokens=0)) == 0 and write(c_cache(), c_seq(n_seq=0, cu=None)) == 0
    assert paged(c_cache(), c_seq(n_tokens=0)) == 0 and _lib.last_error() == ""


@needs_lib
def test_c_packed_and_rotary_refusals():
    s = strides(256, 64)

    def packed(q=P, n_seq=2, n=3, n_kv=3, cu=P, cu_kv=None, h_q=4, h_kv=4, D=64, dtype=0, scale=0.1, ks=s):
        return _lib.lib().fa2_attn_packed(q, P, P, P, s, ks, s, s, cu, cu_kv, n_seq, n, n_kv, h_q, h_kv, D, dtype, 1, scale,
                                          None, None)
    for kw in (dict(q=None), dict(n_seq=-1), dict(n=-1), dict(n_kv=-1), dict(n_kv=4), dict(cu=None), dict(h_q=3), dict(h_kv=0),
               dict(D=8), dict(dtype=2), dict(scale=-1.0), dict(ks=strides(1 << 23, 64)),
               dict(n=2 ** 31 - 300, n_kv=2 ** 31 - 300, n_seq=2 ** 31 - 1)):
        assert packed(**kw) == -1 and _lib.last_error(), kw
    assert packed(q=P + 8) == -2 and packed(ks=strides(4, 64)) == -2
    assert packed(n=0, n_kv=0) == 0 and packed(n_seq=0) == 0

    r = strides(0, 64, 128)

    def turn(x=P, out=P, pos=P, size=8, rot=_lib.Rotation(P, 32, 0, 1.0), B=1, H=2, N=3, D=64, dtype=1, st=r):
        return _lib.lib().fa2_rotary(x, out, st, r, pos, size, strides(0, 1), None if rot is None else ctypes.byref(rot), B,
                                     H, N, D, dtype, None)
    for kw in (dict(x=None), dict(out=None), dict(pos=None), dict(size=2), dict(rot=None), dict(B=-1), dict(H=-1), dict(N=-1),
               dict(D=24), dict(dtype=2), dict(rot=_lib.Rotation(None, 0, 0, 1.0)), dict(D=32)):
        assert turn(**kw) == -1 and _lib.last_error(), kw
    assert turn(x=P + 4) == -2 and turn(pos=P + 4) == -2 and turn(st=strides(0, 60, 128)) == -2
    assert turn(B=0) == 0 and turn(N=0) == 0
