"""GPU tests of the serving operators: rotary positions (fa2.rotary), the paged cache written and read back, and
attention over it (fa2.paged), and attention over packed sequences (fa2.packed), each against float64
(oracle/serving.py) under bounds derived there, and all of them together as a serving loop uses them.
"""

import math

import pytest
import torch

from oracle import serving as oracle
from serving_check import bytes_of, cached, check_attention, cumulative, make_cache, randn

pytestmark = pytest.mark.gpu
DTYPES = [torch.float16, torch.bfloat16]
DIMS = [16, 32, 64, 128]


def plan_of(rot, interleaved=False, scale=1.0, base=10000.0):
    from fa2.rotary import rotary_plan
    return rotary_plan(rot, base, interleaved=interleaved)._replace(scale=scale)


# ------------------------------------------------------------------------------------------
# rotary positions
# ------------------------------------------------------------------------------------------

def check_rotary(got, x, positions, plan):
    """One rounding to the type (u), and products and cosines in float32 (8 * 2^-24 of their magnitudes)."""
    want = oracle.rotate(x, positions, plan.freqs, plan.interleaved, plan.scale)
    ones = oracle.rotate(x.abs(), torch.zeros_like(positions), plan.freqs, plan.interleaved, 1.0)
    half = plan.freqs.numel()
    size = ones.clone()
    i = torch.arange(half, device=x.device)
    a, b = (2 * i, 2 * i + 1) if plan.interleaved else (i, i + half)
    size[..., a] = size[..., b] = (ones[..., a] + ones[..., b]) * max(1.0, abs(plan.scale))
    u = oracle.HALF_STEP[x.dtype]
    tol = u * want.abs() * (1 + u) + 8 * oracle.F32 * size + 2.0 ** -25
    assert ((got.double() - want).abs() <= tol).all(), ((got.double() - want).abs() / tol).max()
    assert torch.equal(got[..., 2 * half:], x[..., 2 * half:])  # not rotated: copied


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,rot", [(16, 16), (32, 16), (64, 48), (64, 64), (128, 32), (128, 96), (128, 128)])
def test_rotary(dtype, interleaved, D, rot):
    from fa2.rotary import rotary
    plan = plan_of(rot, interleaved, 1.25)
    for seed, (T, H) in enumerate([(1, 1), (3, 5), (37, 32), (130, 7)]):
        x = randn((T, H, D), dtype, seed)
        g = torch.Generator().manual_seed(seed)
        positions = torch.randint(-5, 1 << 20, (T,), generator=g).cuda()
        got = rotary(x, positions, plan)
        check_rotary(got.transpose(0, 1), x.transpose(0, 1), positions, plan)
        assert torch.equal(rotary(x, positions.int(), plan), got)
        assert torch.equal(rotary(x, positions, plan, out=x), got) and torch.equal(x, got)  # in place


def test_rotary_layouts():
    """[B, H, N, D] with positions of a row or of the batch, transposed and offset storage, an out of its own."""
    from fa2.rotary import rotary
    plan = plan_of(64)
    x = randn((3, 4, 50, 64), torch.bfloat16, 1)
    positions = torch.arange(50, device="cuda") * 1001
    both = torch.stack([positions, positions + 7, positions.flip(0)])
    got = rotary(x, both, plan)
    for b in range(3):
        check_rotary(got[b], x[b], both[b], plan)
    assert torch.equal(rotary(x, positions, plan)[0], got[0])
    bnhd = x.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(rotary(bnhd, both, plan), got)
    out = torch.full((3, 50, 4, 64), 9.0, dtype=x.dtype, device="cuda").transpose(1, 2)
    assert rotary(bnhd, both, plan, out=out) is out and torch.equal(out, got)
    odd = torch.zeros(3 * 4 * 50 * 64 + 1, dtype=x.dtype, device="cuda")[1:].view(3, 4, 50, 64)
    odd.copy_(x)  # not 16-byte aligned: through copies
    assert torch.equal(rotary(odd, both, plan), got)
    assert rotary(odd, both, plan, out=odd) is odd and torch.equal(odd, got)
    assert rotary(x[:, :, :0], positions[:0], plan).shape == (3, 4, 0, 64)


# ------------------------------------------------------------------------------------------
# the cache, written and read back
# ------------------------------------------------------------------------------------------

def step_of(new, lens, page_size, seed=0, **kw):
    pages = oracle.Pages(lens, page_size, seed=seed, device="cuda", **kw)
    return pages, cumulative(new), torch.tensor(lens, dtype=torch.int32, device="cuda")


STEPS = [([1], [1]), ([1, 1, 1, 1], [1, 77, 300, 64]), ([5, 0, 33, 1, 128], [5, 9, 100, 1, 400]),
         ([17] * 70, [17 + i for i in range(70)])]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("D,page_size,storage", [(16, 64, "hnd"), (32, 32, "nhd"), (64, 16, "hnd"), (64, 64, "nhd"),
                                                 (128, 16, "nhd"), (128, 256, "hnd")])
def test_cache_write_and_read(dtype, e4m3, D, page_size, storage):
    """Every value and scale byte that a place holds, and every other byte of the cache as it was; then the same
    tokens back."""
    from fa2.paged import cache_read, cache_write
    for seed, (new, lens) in enumerate(STEPS):
        h_kv = 1 + seed
        pages, cu, seqlens = step_of(new, lens, page_size, seed)
        cache = make_cache(pages.n_pages, h_kv, page_size, D, dtype, e4m3, seed, storage)
        before = [None if t is None else bytes_of(t).clone() for t in cache]
        T = sum(new) + 3  # three rows of no sequence behind the last one
        k, v = randn((T, h_kv, D), dtype, 10 + seed), randn((T, h_kv, D), dtype, 20 + seed, scale=30.0)
        assert cache_write(cache, k, v, pages.table, cu, seqlens) is None
        dense_k, dense_v = (torch.full((T, h_kv, D), 7.0, dtype=dtype, device="cuda") for _ in "kv")
        cache_read(cache, pages.table, cu, seqlens, T, out=(dense_k, dense_v))
        start = cu.tolist()
        for s, n in enumerate(new):
            rows = slice(start[s], start[s + 1])
            page, row = pages.at(s, torch.arange(lens[s] - n, lens[s], device="cuda"))
            for x, dense, name, i in ((k, dense_k, "k", 0), (v, dense_v, "v", 1)):
                if e4m3:
                    values, e = oracle.to_e4m3(x[rows].double(), dtype)
                    scale = getattr(cache, name + "_scale").view(torch.uint8)
                    assert torch.equal(scale[page, :, row].long(), (e + 127).long())
                    want = values * torch.exp2(e.double())[..., None]
                    before[i + 2][page, :, row] = scale[page, :, row]
                else:
                    want = x[rows].double()
                assert torch.equal(cached(cache, name, page, row), want)
                assert torch.equal(dense[rows].double(), want)
                before[i][page, :, row] = bytes_of(getattr(cache, name))[page, :, row]
        assert (dense_k[start[-1]:] == 7.0).all() and (dense_v[start[-1]:] == 7.0).all()
        for t, was in zip(cache, before):
            assert t is None or torch.equal(bytes_of(t), was)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("interleaved,rot", [(False, 64), (True, 64), (False, 16), (True, 32)])
def test_cache_write_rotates(dtype, e4m3, interleaved, rot):
    """k rotated by its position in the sequence before it is rounded (once), v not, q beside it."""
    from fa2.paged import cache_write
    new, lens, D, page_size = [3, 1, 40], [3, 5000, 900], 64, 32
    pages, cu, seqlens = step_of(new, lens, page_size)
    cache = make_cache(pages.n_pages, 2, page_size, D, dtype, e4m3)
    plan = plan_of(rot, interleaved, 1.1)
    T = sum(new) + 2
    k, v, q = randn((T, 2, D), dtype, 1), randn((T, 2, D), dtype, 2), randn((T, 10, D), dtype, 3)
    q_out = torch.full_like(q, 7.0)
    assert cache_write(cache, k, v, pages.table, cu, seqlens, rotary=plan, q=q, q_out=q_out) is q_out
    assert (q_out[-2:] == 7.0).all()
    start = cu.tolist()
    for s, n in enumerate(new):
        rows = slice(start[s], start[s + 1])
        positions = torch.arange(lens[s] - n, lens[s], device="cuda")
        page, row = pages.at(s, positions)
        check_rotary(q_out[rows].transpose(0, 1), q[rows].transpose(0, 1), positions, plan)
        turned = oracle.rotate(k[rows].transpose(0, 1), positions, plan.freqs, interleaved, 1.1).transpose(0, 1)
        if e4m3:
            values, e = oracle.to_e4m3(turned, dtype)
            assert torch.equal(cache.k_scale.view(torch.uint8)[page, :, row].long(), (e + 127).long())
            assert torch.equal(cached(cache, "k", page, row), values * torch.exp2(e.double())[..., None])
            values, e = oracle.to_e4m3(v[rows].double(), dtype)
            assert torch.equal(cached(cache, "v", page, row), values * torch.exp2(e.double())[..., None])
        else:
            check_rotary(cached(cache, "k", page, row).to(dtype).transpose(0, 1), k[rows].transpose(0, 1),
                         positions, plan)
            assert torch.equal(cached(cache, "v", page, row), v[rows].double())
    assert cache_write(cache, k, v, pages.table, cu, seqlens, rotary=plan, q=q, q_out=q) is q  # in place
    assert torch.equal(q[:-2], q_out[:-2])


@pytest.mark.parametrize("dtype", DTYPES)
def test_e4m3_extremes(dtype):
    """Rows of zeros, of the type's least and largest values, of one value at each side of a power of two, with
    infinities and NaN: what is stored is the oracle's, and finite wherever the row was."""
    from fa2.paged import cache_read, cache_write
    D, page_size = 64, 16
    info = torch.finfo(dtype)
    tiny = info.smallest_normal * info.eps  # the least subnormal
    rows = [[0.0], [tiny], [-tiny, info.smallest_normal], [info.max], [-info.max, 1.0, info.max / 2],
            [math.inf, 1.0, -3.0], [-math.inf, math.nan], [math.nan, 0.1, 200.0], [448.0], [449.0, 447.0, 1.0],
            [0.875, 0.0009765625], [1.75 * 2.0 ** 12, 2.0 ** -3], [57344.0, 61440.0, 32.0], [17.0, 18.0, 19.0, 216.0, 232.0, 240.0]]
    k = torch.zeros(len(rows), 1, D, dtype=dtype, device="cuda")
    for i, r in enumerate(rows):
        k[i, 0, :len(r)] = torch.tensor(r, device="cuda").to(dtype)
    pages, cu, seqlens = step_of([len(rows)], [len(rows)], page_size)
    cache = make_cache(pages.n_pages, 1, page_size, D, dtype, True)
    cache_write(cache, k, k.neg(), pages.table, cu, seqlens)
    back_k, back_v = cache_read(cache, pages.table, cu, seqlens, len(rows), dtype=dtype)
    page, row = pages.at(0, torch.arange(len(rows), device="cuda"))
    for x, back, name in ((k, back_k, "k"), (k.neg(), back_v, "v")):
        values, e = oracle.to_e4m3(x.double(), dtype)
        assert torch.equal(getattr(cache, name + "_scale").view(torch.uint8)[page, :, row].long(), (e + 127).long())
        want = values * torch.exp2(e.double())[..., None]
        assert torch.equal(cached(cache, name, page, row).nan_to_num(9e9), want.nan_to_num(9e9))
        assert torch.equal(back.isnan(), ~x.isfinite()) and not back.isinf().any()
        assert torch.equal(back.nan_to_num(1.0), want.to(dtype).nan_to_num(1.0))


@pytest.mark.parametrize("e4m3", [False, True])
def test_cache_places_that_are_not_there(e4m3):
    """Entries outside the cache, positions past the table, sequences shorter than their new tokens and index
    vectors that do not ascend: nothing outside the places that exist is written, and reads of the others
    are zeros."""
    from fa2.paged import cache_read, cache_write
    D, page_size, dtype = 64, 16, torch.bfloat16
    cache = make_cache(6, 2, page_size, D, dtype, e4m3)
    before = [None if t is None else bytes_of(t).clone() for t in cache]
    table = torch.tensor([[0, 6, 1], [-1, 2, 1 << 30], [3, -2 ** 31, 5]], dtype=torch.int32, device="cuda")
    new, lens = [40, 20, 6], [40, 60, 4]  # the last: two rows before position 0
    cu, seqlens = cumulative(new), torch.tensor(lens, dtype=torch.int32, device="cuda")
    k, v = randn((66, 2, D), dtype, 1), randn((66, 2, D), dtype, 2)
    cache_write(cache, k, v, table, cu, seqlens)
    out = tuple(torch.full_like(k, 7.0) for _ in "kv")
    cache_read(cache, table, cu, seqlens, 66, out=out)
    for s in range(3):
        for j in range(new[s]):
            t, pos = sum(new[:s]) + j, lens[s] - new[s] + j
            if pos < 0:
                assert (out[0][t] == 7.0).all()
                continue
            page = table[s, pos // page_size].item() if pos // page_size < 3 else -1
            if not 0 <= page < 6:
                assert (out[0][t] == 0).all() and (out[1][t] == 0).all()
                continue
            want = k[t].double()
            if e4m3:
                values, e = oracle.to_e4m3(want, dtype)
                want = values * torch.exp2(e.double())[..., None]
            assert torch.equal(out[0][t].double(), want)
            for i, t2 in enumerate(cache):
                if t2 is not None:
                    before[i][page, :, pos % page_size] = bytes_of(t2)[page, :, pos % page_size]
    for t, was in zip(cache, before):
        assert t is None or torch.equal(bytes_of(t), was)
    wild = torch.tensor([70, -3, 1 << 30, 12], dtype=torch.int32, device="cuda")
    cache_read(cache, table, wild, seqlens, 66, dtype=dtype)
    q = randn((66, 4, D), dtype, 3)
    from fa2.paged import attention_paged
    attention_paged(q, cache, table, wild, seqlens)
    torch.cuda.synchronize()


# ------------------------------------------------------------------------------------------
# attention over packed sequences
# ------------------------------------------------------------------------------------------

PACKED = [[1], [0, 1, 0, 2], [31, 32, 33], [64, 1, 127, 128, 129], [300, 7, 0, 1000], [5] * 67]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", DIMS)
@pytest.mark.parametrize("h_q,h_kv", [(1, 1), (4, 4), (8, 2), (7, 1), (16, 8)])
@pytest.mark.parametrize("causal", [True, False])
def test_packed(dtype, D, h_q, h_kv, causal):
    from fa2.packed import attention_packed
    for seed, lens in enumerate(PACKED):
        T, cu = sum(lens) + 2, cumulative(lens)
        q, k, v = randn((T, h_q, D), dtype, seed), randn((T, h_kv, D), dtype, 50 + seed), randn((T, h_kv, D), dtype, 90 + seed)
        k[-2:], v[-2:] = math.nan, math.inf  # rows of no sequence
        out = torch.full_like(q, 7.0)
        got, lse = attention_packed(q, k, v, cu, causal=causal, return_lse=True, out=out)
        assert got is out and (out[-2:] == 7.0).all()
        at = cu.tolist()
        check_attention(out, lse, q, lambda s: k[at[s]:at[s + 1]].double(), lambda s: v[at[s]:at[s + 1]].double(), cu,
                        causal, dtype)
        assert torch.equal(attention_packed(q, k, v, cu, causal=causal)[:-2], out[:-2])


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens", [[2500, 1, 777, 1300], [300, 0, 1, 700, 129, 128, 0, 511, 90, 0], [7 * i % 400 for i in range(64)],
                                  [200 + i for i in range(20)] * 4], ids=len)
def test_packed_long(causal, D, lens):
    from fa2.packed import attention_packed
    T, cu = sum(lens), cumulative(lens)
    q, k, v = (randn((T, h, D), torch.bfloat16, i) for i, h in enumerate((8, 2, 2)))
    out, lse = attention_packed(q, k, v, cu, causal=causal, return_lse=True)
    at = cu.tolist()
    check_attention(out, lse, q, lambda s: k[at[s]:at[s + 1]].double(), lambda s: v[at[s]:at[s + 1]].double(), cu, causal,
                    torch.bfloat16)


@pytest.mark.parametrize("causal", [True, False])
def test_packed_other_keys(causal):
    """Sequences of k and v of their own lengths: more keys than rows, fewer (rows that see none), and none."""
    from fa2.packed import attention_packed
    n_q, n_kv, D, dtype = [5, 40, 33, 0, 1, 70], [300, 8, 33, 9, 0, 1], 64, torch.float16
    cu, cu_kv = cumulative(n_q), cumulative(n_kv)
    q = randn((sum(n_q), 6, D), dtype, 1)
    k, v = randn((sum(n_kv), 3, D), dtype, 2), randn((sum(n_kv), 3, D), dtype, 3)
    out, lse = attention_packed(q, k, v, cu, cu_kv, causal=causal, sm_scale=0.3, return_lse=True)
    at = cu_kv.tolist()
    check_attention(out, lse, q, lambda s: k[at[s]:at[s + 1]].double(), lambda s: v[at[s]:at[s + 1]].double(), cu, causal,
                    dtype, 0.3)


def test_packed_layouts():
    """Parts of one QKV projection, heads outermost, and storage that the 16-byte loads cannot address."""
    from fa2.packed import attention_packed
    lens, D, dtype = [100, 1, 63], 64, torch.bfloat16
    T, cu = sum(lens), cumulative(lens)
    qkv = randn((T, 8 + 2 + 2, D), dtype, 5)
    q, k, v = qkv[:, :8], qkv[:, 8:10], qkv[:, 10:]
    want = attention_packed(q.contiguous(), k.contiguous(), v.contiguous(), cu)
    assert torch.equal(attention_packed(q, k, v, cu), want)
    heads = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]
    assert torch.equal(attention_packed(*heads, cu), want)
    wide = torch.empty(T, 12, D + 4, dtype=dtype, device="cuda")
    wide[..., :D] = qkv
    assert torch.equal(attention_packed(wide[:, :8, :D], wide[:, 8:10, :D], wide[:, 10:, :D], cu), want)
    out = torch.full((T, 8, D + 4), 7.0, dtype=dtype, device="cuda")
    attention_packed(q, k, v, cu, out=out[..., :D])
    assert torch.equal(out[..., :D], want) and (out[..., D:] == 7.0).all()
    assert torch.equal(attention_packed(q, k, v, cumulative([T, 0, 0])), attention_packed(q, k, v, cumulative([T])))


@pytest.mark.parametrize("D", [16, 64, 128])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_packed_not_finite(D, bad):
    """An infinite or NaN value or key reaches the rows that see it, and no other: not the rows before it in the
    same tile, and not the next sequence."""
    from fa2.packed import attention_packed
    lens, dtype = [150, 90], torch.float16
    cu = cumulative(lens)
    q, k, v = (randn((240, 2, D), dtype, i) for i in range(3))
    q = torch.where(q == 0, torch.ones_like(q), q)
    for which in ("v", "k"):
        for at in (0, 70, 149, 150, 239):
            kb, vb = k.clone(), v.clone()
            (vb if which == "v" else kb)[at, 1, D // 2] = bad
            for causal in (True, False):
                out, lse = attention_packed(q, kb, vb, cu, causal=causal, return_lse=True)
                c = cu.tolist()
                check_attention(out, lse, q, lambda s: kb[c[s]:c[s + 1]].double(), lambda s: vb[c[s]:c[s + 1]].double(),
                                cu, causal, dtype)


def test_packed_indices_that_do_not_ascend():
    """Whatever cu_seqlens holds, no row outside the tensors is touched (they end where their memory does)."""
    from fa2.packed import attention_packed
    q, k, v = (randn((64, 2, 32), torch.float16, i) for i in range(3))
    for bad in ([5, 1 << 30, -7, 64], [64, 0, 64, 0], [-2 ** 31, 2 ** 31 - 1, 3, 2 ** 31 - 1]):
        cu = torch.tensor(bad, dtype=torch.int32, device="cuda")
        attention_packed(q, k, v, cu)
        attention_packed(q, k, v, cumulative([20, 20, 24]), cu)
    torch.cuda.synchronize()


# ------------------------------------------------------------------------------------------
# attention over the paged cache
# ------------------------------------------------------------------------------------------

PAGED = [([1], [1]), ([1] * 5, [1, 33, 64, 700, 129]), ([4, 0, 1, 40, 129], [4, 50, 1000, 41, 129]),
         ([3, 5, 2], [1, 0, 2])]
MANY = [([1] * 66, [2 + 5 * i for i in range(66)]), ([40] * 70, [20 + 7 * i for i in range(70)])]


def widened(table, page_size, keys=1600):
    """The table with entries behind the last pages for sequences of `keys` tokens: workgroups share the work of calls
    whose sequences may be long"""
    more = max(-(-keys // page_size) - table.shape[1], 0)
    return torch.cat([table, torch.full((table.shape[0], more), -1, dtype=torch.int32, device=table.device)], 1)


def check_paged(q, cache, pages, cu, lens, causal, dtype, out, lse, sm_scale=None):
    def of(which):
        return lambda s: cached(cache, which, *pages.at(s, torch.arange(lens[s], device="cuda"))).to(dtype).double()
    check_attention(out, lse, q, of("k"), of("v"), cu, causal, dtype, sm_scale)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("D,page_size", [(16, 64), (32, 32), (64, 16), (64, 128), (128, 16), (128, 64)])
@pytest.mark.parametrize("h_q,h_kv", [(2, 2), (8, 2), (7, 1), (16, 8)])
def test_paged(dtype, e4m3, D, page_size, h_q, h_kv):
    check_paged_calls(PAGED, dtype, e4m3, D, page_size, h_q, h_kv)


@pytest.mark.parametrize("dtype,e4m3,D,page_size,h_q,h_kv", [(torch.float16, False, 64, 16, 8, 2), (torch.bfloat16, True, 128, 64, 2, 2),
                                                             (torch.bfloat16, False, 16, 32, 7, 1)])
def test_paged_many_sequences(dtype, e4m3, D, page_size, h_q, h_kv):
    """More than 64: a workgroup looks for its rows 64 sequences at a time"""
    check_paged_calls(MANY, dtype, e4m3, D, page_size, h_q, h_kv)


def check_paged_calls(steps, dtype, e4m3, D, page_size, h_q, h_kv):
    from fa2.paged import attention_paged
    for seed, (new, lens) in enumerate(steps):
        pages, cu, seqlens = step_of(new, lens, page_size, seed)
        cache = make_cache(pages.n_pages, h_kv, page_size, D, dtype, e4m3, seed, ("hnd", "nhd")[seed % 2])
        for s, n in enumerate(lens):  # rows behind a sequence's last token hold NaN
            if n % page_size:
                page, row = pages.at(s, torch.arange(n, -(-n // page_size) * page_size, device="cuda"))
                for t in (cache.k, cache.v):
                    bytes_of(t)[page, :, row] = 0x7f if e4m3 else math.nan
        T = sum(new) + 2
        q, out = randn((T, h_q, D), dtype, 30 + seed), torch.full((T, h_q, D), 7.0, dtype=dtype, device="cuda")
        for causal, table in ((c, t) for t in (pages.table, widened(pages.table, page_size)) for c in (True, False)):
            got, lse = attention_paged(q, cache, table, cu, seqlens, causal=causal, return_lse=True, out=out.fill_(7.0))
            assert got is out and (out[-2:] == 7.0).all()
            check_paged(q, cache, pages, cu, lens, causal, dtype, out, lse)
            assert torch.equal(attention_paged(q, cache, table, cu, seqlens, causal=causal)[:-2], out[:-2])


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("dtype,D,page_size", [(torch.bfloat16, 128, 32), (torch.float16, 64, 16), (torch.bfloat16, 32, 64),
                                               (torch.float16, 16, 128)])
@pytest.mark.parametrize("new,lens", [([1, 1], [9000, 20]), ([1], [30000]), ([3], [12345]), ([300, 1, 1, 64], [5000, 3000, 1, 2100]), ([600], [4321]),
                                      ([200, 0, 1, 700], [100, 50, 6000, 350]), ([30] * 66 + [400], [40] * 66 + [5000])])
def test_paged_long(e4m3, dtype, D, page_size, new, lens):
    from fa2.paged import attention_paged
    pages, cu, seqlens = step_of(new, lens, page_size)
    cache = make_cache(pages.n_pages, 2, page_size, D, dtype, e4m3)
    q = randn((sum(new), 8, D), dtype, 3)
    for causal in (True, False):
        out, lse = attention_paged(q, cache, pages.table, cu, seqlens, causal=causal, return_lse=True, sm_scale=0.2)
        check_paged(q, cache, pages, cu, lens, causal, dtype, out, lse, 0.2)


@pytest.mark.parametrize("wide", [False, True])
def test_paged_page_outside_the_cache(wide):
    """A table entry that is no page makes the rows that see its tokens NaN, and leaves the others; one behind the last
    token is never read."""
    from fa2.paged import attention_paged
    D, page_size, dtype = 64, 16, torch.float16
    for e4m3 in (False, True):
        new, lens = [1, 30, 1], [200, 200, 200]
        pages, cu, seqlens = step_of(new, lens, page_size)
        cache = make_cache(pages.n_pages, 2, page_size, D, dtype, e4m3)
        q = randn((32, 4, D), dtype, 3)
        whole = pages.table if not wide else widened(pages.table, page_size)
        want = attention_paged(q, cache, whole, cu, seqlens)
        assert want.isfinite().all()
        for bad in (-1, pages.n_pages, 1 << 30, -2 ** 31):
            table = whole.clone()
            table[0, 3] = table[1, 12] = bad  # tokens 48 .. 63, and 192 .. 199 (rows 22 and on see them)
            out, lse = attention_paged(q, cache, table, cu, seqlens, return_lse=True)
            assert out[0].isnan().all() and lse[:, 0].isnan().all()
            assert out[23:31].isnan().all()
            assert torch.equal(out[31], want[31])


def test_paged_far_offsets():
    """Pages past 2^31 elements and 2^32 bytes of the cache."""
    from fa2.paged import KVCache, attention_paged, cache_read, cache_write
    D, page_size, h_kv = 128, 64, 8
    n_pages = (1 << 31) // (D * page_size * h_kv) + 40
    for dtype, kv in ((torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float8_e4m3fn)):
        cache = KVCache.empty(n_pages, h_kv, page_size, D, kv)
        new, lens = [70, 1], [70, 500]
        pages, cu, seqlens = step_of(new, lens, page_size, n_pages=n_pages, first_page=n_pages - 30)
        k, v, q = (randn((71, h, D), dtype, i) for i, h in enumerate((h_kv, h_kv, 16)))
        cache_write(cache, k, v, pages.table, cu, seqlens)
        out = attention_paged(q, cache, pages.table, cu, seqlens)
        check_paged(q, cache, pages, cu, lens, True, dtype, out, None)
        back = cache_read(cache, pages.table, cu, seqlens, 71, dtype=dtype)
        u = 2.0 ** -4 if kv == torch.float8_e4m3fn else 0.0
        assert ((back[0].double() - k.double()).abs() <= u * k.double().abs() + u * 2.0 ** -10).all()
        del cache


# ------------------------------------------------------------------------------------------
# together
# ------------------------------------------------------------------------------------------

def serve(cache, pages, lens, x, plan, chunks):
    """A serving loop over `chunks` ([new tokens of each sequence] per step): x(s, a, b) gives the rows of tokens a .. b
    of sequence s (q, k, v). Returns every sequence's outputs."""
    from fa2.paged import attention_paged, cache_write
    done, outs = [0] * len(lens), [[] for _ in lens]
    for new in chunks:
        parts = [x(s, done[s], done[s] + n) for s, n in enumerate(new)]
        q, k, v = (torch.cat([p[i] for p in parts]) for i in range(3))
        done = [d + n for d, n in zip(done, new)]
        cu, seqlens = cumulative(new), torch.tensor(done, dtype=torch.int32, device="cuda")
        q = cache_write(cache, k, v, pages.table, cu, seqlens, rotary=plan, q=q)
        out = attention_paged(q, cache, pages.table, cu, seqlens)
        for s, o in enumerate(out.split(new)):
            outs[s].append(o)
    assert done == lens
    return [torch.cat(o) for o in outs]


@pytest.mark.parametrize("e4m3", [False, True])
def test_chunks_and_steps_as_one_prompt(e4m3):
    """Prompts in chunks and then token by token through rotary, cache and paged attention, against attention over
    the whole packed prompts, rotated by rotary(), with the cache's own k and v read back."""
    from fa2.kernel import attention
    from fa2.packed import attention_packed
    from fa2.paged import KVCache, cache_read
    from fa2.rotary import rotary
    lens, D, h_q, h_kv, page_size, dtype = [70, 33, 1, 150], 64, 8, 2, 16, torch.bfloat16
    T, whole = sum(lens), cumulative(lens)
    at = whole.tolist()
    q, k, v = randn((T, h_q, D), dtype, 1), randn((T, h_kv, D), dtype, 2), randn((T, h_kv, D), dtype, 3)
    pages = oracle.Pages(lens, page_size, device="cuda")
    cache = KVCache.empty(pages.n_pages, h_kv, page_size, D, torch.float8_e4m3fn if e4m3 else dtype)
    plan = plan_of(64)

    def rows(s, a, b):
        return [t[at[s] + a:at[s] + b] for t in (q, k, v)]
    chunks = [[64, 33, 0, 100], [4, 0, 1, 48], [1, 0, 0, 1], [1, 0, 0, 1]]
    outs = serve(cache, pages, lens, rows, plan, chunks)
    positions = torch.cat([torch.arange(n, device="cuda") for n in lens])
    q_ = rotary(q, positions, plan)
    seqlens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    k_, v_ = cache_read(cache, pages.table, whole, seqlens, T, dtype=dtype)
    if not e4m3:
        assert torch.equal(k_, rotary(k, positions, plan)) and torch.equal(v_, v)
    check_attention(torch.cat(outs), None, q_, lambda s: k_[at[s]:at[s + 1]].double(),
                    lambda s: v_[at[s]:at[s + 1]].double(), whole, True, dtype)
    packed = attention_packed(q_, k_, v_, whole)
    u = oracle.HALF_STEP[dtype]
    for s in range(len(lens)):  # the dense operator on each prompt alone
        r = slice(at[s], at[s + 1])
        dense = attention(*(t[r].transpose(0, 1)[None] for t in (q_, k_, v_)), causal=True)[0].transpose(0, 1)
        for other in (packed[r], outs[s]):
            # two kernels, each off by three roundings at most of values around the largest |v| of the row
            assert (other.double() - dense.double()).abs().max() <= 8 * u * v_[r].abs().max()


@pytest.mark.parametrize("columns", [40, 120])  # (of 16 tokens: a workgroup per row tile, or equal shares)
def test_graph_follows_lengths(columns):
    """A step captured once and replayed with other lengths, tables and values, a padded batch among them: rows behind the
    last sequence keep what they held."""
    from fa2.paged import KVCache, attention_paged, cache_write
    D, h_q, h_kv, page_size, dtype, S, T = 128, 8, 2, 16, torch.bfloat16, 6, 40
    plan = plan_of(128)
    q, k, v = (torch.zeros(T, h, D, dtype=dtype, device="cuda") for h in (h_q, h_kv, h_kv))
    cu = torch.zeros(S + 1, dtype=torch.int32, device="cuda")
    seqlens = torch.zeros(S, dtype=torch.int32, device="cuda")
    table = torch.zeros(S, columns, dtype=torch.int32, device="cuda")
    out, q_out = torch.zeros_like(q), torch.zeros_like(q)
    caches = [KVCache.empty(300, h_kv, page_size, D, t) for t in (dtype, torch.float8_e4m3fn)]

    def step(cache):
        cache_write(cache, k, v, table, cu, seqlens, rotary=plan, q=q, q_out=q_out)
        return attention_paged(q_out, cache, table, cu, seqlens, out=out)
    for cache in caches:
        step(cache)
        torch.cuda.synchronize()
        graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream), torch.cuda.graph(graph, stream=stream):
            step(cache)
        torch.cuda.synchronize()
        for seed, (new, lens) in enumerate([([1] * 6, [5, 600, 40, 1, 16, 17]), ([30, 1, 1, 0, 0, 0], [300, 9, 64, 0, 0, 0]),
                                            ([0] * 6, [0] * 6), ([1, 1, 1, 1, 1, 1], [640, 1, 2, 3, 4, 5])]):
            for t, h in ((q, h_q), (k, h_kv), (v, h_kv)):
                t.copy_(randn((T, h, D), dtype, seed))
            pages = oracle.Pages(lens, page_size, n_pages=300, seed=seed, device="cuda")
            table.fill_(-1)
            table[:, :pages.table.shape[1]] = pages.table[:, :columns]
            cu.copy_(cumulative(new)), seqlens.copy_(torch.tensor(lens, dtype=torch.int32))
            start = [t if t is None else t.clone() for t in cache]
            out.fill_(7.0), q_out.fill_(5.0)
            graph.replay()
            torch.cuda.synchronize()
            got, got_q, n = out.clone(), q_out.clone(), sum(new)
            after = [None if t is None else bytes_of(t).clone() for t in cache]
            assert (got[n:] == 7.0).all() and (got_q[n:] == 5.0).all()
            for t, was in zip(cache, start):
                if t is not None:
                    bytes_of(t).copy_(bytes_of(was))
            out.fill_(7.0), q_out.fill_(5.0)
            step(cache)
            torch.cuda.synchronize()
            assert torch.equal(out, got) and torch.equal(q_out, got_q)
            assert all(t is None or torch.equal(bytes_of(t), was) for t, was in zip(cache, after))


def test_streams_at_once():
    """Calls on several streams at once, each with its own tensors, equal the same calls one after another."""
    from fa2.packed import attention_packed
    from fa2.paged import attention_paged
    D, dtype = 64, torch.float16
    jobs = []
    for i in range(4):
        new, lens = [1 + i] * 9, [100 + 300 * i + 7 * j for j in range(9)]
        pages, cu, seqlens = step_of(new, lens, 16, seed=i)
        cache = make_cache(pages.n_pages, 2, 16, D, dtype, i % 2 == 1, i)
        q = randn((sum(new), 8, D), dtype, i)
        qp, kp, vp = (randn((500, h, D), dtype, 10 * i + h) for h in (8, 2, 2))
        jobs.append((lambda q=q, c=cache, t=pages.table, u=cu, s=seqlens: attention_paged(q, c, t, u, s),
                     lambda q=qp, k=kp, v=vp, u=cumulative([200, 300]): attention_packed(q, k, v, u)))
    want = [(a(), b()) for a, b in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    got = [[] for _ in jobs]
    for _ in range(5):
        for i, (s, (a, b)) in enumerate(zip(streams, jobs)):
            with torch.cuda.stream(s):
                got[i].append((a(), b()))
    torch.cuda.synchronize()
    for i, w in enumerate(want):
        for g in got[i]:
            assert torch.equal(g[0], w[0]) and torch.equal(g[1], w[1])


def calls_of_each(seed=0, dtype=torch.bfloat16, e4m3=True):
    """Every operator's call on tensors of its own, as functions of `out` (a tensor to write, or None)"""
    from fa2.packed import attention_packed
    from fa2.paged import attention_paged, cache_read, cache_write
    from fa2.rotary import rotary
    D, page_size, new, lens = 64, 64, [3, 0, 40, 1], [30, 5, 900, 1]
    pages, cu, seqlens = step_of(new, lens, page_size, seed)
    table = widened(pages.table, page_size)
    cache = make_cache(pages.n_pages, 2, page_size, D, dtype, e4m3, seed)
    T = sum(new)
    q, k, v = (randn((T, h, D), dtype, seed + i) for i, h in enumerate((8, 2, 2)))
    positions = torch.arange(T, device="cuda")
    return {"rotary": lambda out=None: rotary(q, positions, plan_of(32, True, 0.5), out=out),
            "cache_write": lambda out=None: cache_write(cache, k, v, table, cu, seqlens, rotary=plan_of(64), q=q, q_out=out),
            "cache_read": lambda out=None: cache_read(cache, table, cu, seqlens, T, dtype=dtype,
                                                      out=None if out is None else (out[:, :2], k.clone()))[0],
            "packed": lambda out=None: attention_packed(q, k, v, cu, out=out),
            "packed lse": lambda out=None: attention_packed(q, k, v, cu, causal=False, sm_scale=0.3, return_lse=True, out=out)[1],
            "paged": lambda out=None: attention_paged(q, cache, table, cu, seqlens, out=out),
            "paged lse": lambda out=None: attention_paged(q, cache, table, cu, seqlens, return_lse=True, out=out)[1]}


@pytest.mark.parametrize("e4m3", [False, True])
def test_both_ways_to_the_kernels(e4m3, monkeypatch):
    """The native calls and the ones through ctypes launch the same."""
    from fa2 import _lib
    assert _lib.native is not None
    native = {name: call() for name, call in calls_of_each(e4m3=e4m3).items()}
    monkeypatch.setattr(_lib, "native", None)
    for name, call in calls_of_each(e4m3=e4m3).items():
        assert torch.equal(call(), native[name]), name


@pytest.mark.parametrize("layout", ["dense", "odd storage", "every other value", "other order"])
def test_out_of_any_layout(layout):
    """An out that the kernels cannot address is written through a copy; what lies between its values stays."""
    for name, call in calls_of_each().items():
        want = call()
        if name.endswith("lse"):
            continue
        shape = (44, 8, 64)
        if layout == "dense":
            store = torch.full(shape, 3.0, dtype=torch.bfloat16, device="cuda")
            out = store
        elif layout == "odd storage":
            store = torch.full((44 * 8 * 64 + 1,), 3.0, dtype=torch.bfloat16, device="cuda")
            out = store[1:].view(shape)
        elif layout == "every other value":
            store = torch.full((44, 8, 128), 3.0, dtype=torch.bfloat16, device="cuda")
            out = store[..., ::2]
        else:
            store = torch.full((8, 44, 64), 3.0, dtype=torch.bfloat16, device="cuda")
            out = store.transpose(0, 1)
        got = call(out)
        assert torch.equal(got, want), name
        assert torch.equal(out[:, :want.shape[1]], want), name
        if layout == "every other value":
            assert (store[..., 1::2] == 3.0).all(), name


def test_out_in_place_and_broadcast():
    """out may be the call's own q; a broadcast one is refused."""
    from fa2.packed import attention_packed
    from fa2.paged import attention_paged, cache_read, cache_write
    from fa2.rotary import rotary
    for new, lens in (([1] * 6, [700, 3, 64, 1, 2000, 90]), ([300, 1, 70], [2500, 800, 70])):
        pages, cu, seqlens = step_of(new, lens, 32)
        for D, e4m3 in ((64, False), (128, True)):
            cache = make_cache(pages.n_pages, 2, 32, D, torch.float16, e4m3)
            T = sum(new)
            q, k = randn((T, 8, D), torch.float16, 5), randn((T, 2, D), torch.float16, 6)
            for call in (lambda q, out: attention_paged(q, cache, pages.table, cu, seqlens, out=out),
                         lambda q, out: attention_packed(q, k, k, cu, out=out),
                         lambda q, out: rotary(q, torch.arange(T, device="cuda"), plan_of(D), out=out)):
                want = call(q, None)
                x = q.clone()
                assert torch.equal(call(x, x), want)
                with pytest.raises(RuntimeError, match="stride of 0"):
                    call(q, x[:, :1].expand(T, 8, D))
            with pytest.raises(RuntimeError, match="stride of 0"):
                cache_write(cache._replace(k=cache.k[:1].expand_as(cache.k)), k, k, pages.table, cu, seqlens)
            with pytest.raises(RuntimeError, match="stride of 0"):
                cache_read(cache, pages.table, cu, seqlens, T, out=(k, k[:1].expand(T, 2, D)))
            # reading from heads that share their rows is fine
            one = cache._replace(**{n: t[:, :1].expand(t.shape) for n, t in zip(cache._fields, cache) if t is not None})
            apart = cache._replace(**{n: bytes_of(t).contiguous().view(t.dtype) for n, t in zip(one._fields, one) if t is not None})
            assert torch.equal(attention_paged(q, one, pages.table, cu, seqlens),
                               attention_paged(q, apart, pages.table, cu, seqlens))


def test_tables_without_columns():
    """No sequence has a token in the cache: rows get 0, nothing is written, zeros are read."""
    from fa2.paged import attention_paged, cache_read, cache_write
    cache = make_cache(2, 2, 16, 64, torch.float16, False)
    before = [bytes_of(t).clone() for t in (cache.k, cache.v)]
    cu, table = cumulative([3, 1]), torch.zeros(2, 0, dtype=torch.int32, device="cuda")
    seqlens = torch.tensor([3, 9], dtype=torch.int32, device="cuda")
    q, k = randn((4, 4, 64), torch.float16, 1), randn((4, 2, 64), torch.float16, 2)
    out, lse = attention_paged(q, cache, table, cu, seqlens, return_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()
    cache_write(cache, k, k, table, cu, seqlens)
    assert all(torch.equal(bytes_of(t), b) for t, b in zip((cache.k, cache.v), before))
    assert all((t == 0).all() for t in cache_read(cache, table, cu, seqlens, 4))


def test_lengths_past_the_table():
    from fa2.paged import attention_paged
    for most, new in ((128, [1, 5]), (2048, [1, 300])):
        pages, cu, seqlens = step_of(new, [most, 60 + new[1]], 32)
        table = pages.table[:, :most // 32].contiguous()
        for e4m3 in (False, True):
            cache = make_cache(pages.n_pages, 2, 32, 64, torch.bfloat16, e4m3)
            q = randn((sum(new), 8, 64), torch.bfloat16, 1)
            long = torch.tensor([2 ** 31 - 1, 60 + new[1]], dtype=torch.int32, device="cuda")
            for causal in (True, False):
                assert torch.equal(attention_paged(q, cache, table, cu, long, causal=causal),
                                   attention_paged(q, cache, table, cu, seqlens, causal=causal))


def test_two_graphs_of_one_pool():
    """Two captured steps that share a memory pool, replayed in turn with other lengths and eager calls between."""
    from fa2.paged import attention_paged
    D, dtype, page_size = 128, torch.float16, 32
    jobs = []
    stream, pool = torch.cuda.Stream(), None
    for i, new in enumerate(([1] * 8, [90, 1, 200, 1])):
        most = [2000 + 100 * j for j in range(len(new))]
        pages, cu, _ = step_of(new, most, page_size, seed=i)
        cache = make_cache(pages.n_pages, 2, page_size, D, dtype, i == 1, i)
        seqlens = torch.tensor(most, dtype=torch.int32, device="cuda")
        q = randn((sum(new), 8, D), dtype, i)
        out = torch.zeros_like(q)

        def call(q=q, cache=cache, table=pages.table, cu=cu, seqlens=seqlens, out=None):
            return attention_paged(q, cache, table, cu, seqlens, out=out)
        call()
        torch.cuda.synchronize()
        stream.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(stream), torch.cuda.graph(graph, pool=pool, stream=stream):
            call(out=out)
        pool = graph.pool()
        jobs.append((graph, call, seqlens, most, out))
    torch.cuda.synchronize()
    for round_ in range(4):
        for graph, call, seqlens, most, out in jobs:
            seqlens.copy_(torch.tensor([max(n - 631 * round_ * (j % 3), 300) for j, n in enumerate(most)], dtype=torch.int32))
            out.fill_(9.0)
            graph.replay()
            assert torch.equal(out, call())
    torch.cuda.synchronize()
