"""The serving operators beside the attention forward, as measured cases: rotary positions, a paged K/V
cache as it is written (16-bit, or e4m3 with a power-of-two scale per token and head) and read back,
attention over packed prompts, and attention of new tokens over the paged cache.

Every operator has a plain form in elementary torch operations, in float32 and rounded once at the end
(float64 for the angles of far positions and for values that are rounded to 8 bits), and the call that a
user makes of the package (`own`). listed() holds twelve cases, draw() more of the same ranges.

Sequences are packed: `cu` [S + 1] holds each sequence's first row, and `lens` [S] the tokens of each in
the cache, the new ones included. Their lengths follow from the case alone (_lengths); values and page
tables from the seed.
"""

import math
import os
import random
import sys

import torch

own = False

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "triton-fa2-forward_amd")
_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _modules():
    """The package's public modules (only where `own` is true)."""
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import fa2.packed
    import fa2.paged
    import fa2.rotary
    return fa2


# ------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------

def _rotary(name, tokens, heads, dim, rot, dtype, interleaved, far, factor=1.0):
    """tokens at positions up to `far`; the first `rot` of dim values are rotated, pairs (i, i + rot / 2) or
    (2 i, 2 i + 1); factor > 1: frequencies stretched for a longer context, as rotary_frequencies does."""
    return dict(name=name, kind="rotary", tokens=tokens, heads=heads, dim=dim, rot=rot, dtype=dtype,
                interleaved=interleaved, far=far, factor=factor)


def _write(name, seqs, new, old, h_q, h_kv, dim, page, dtype, e4m3, rot, interleaved):
    """up to `new` tokens of each sequence behind up to `old` in the cache: q and k rotated, k and v written
    into pages, and the written tokens read back."""
    return dict(name=name, kind="write", seqs=seqs, new=new, old=old, h_q=h_q, h_kv=h_kv, dim=dim, page=page,
                dtype=dtype, e4m3=e4m3, rot=rot, interleaved=interleaved)


def _read(name, seqs, old, h_kv, dim, page, dtype, e4m3):
    """whole sequences of up to `old` tokens out of the cache, dense and packed."""
    return dict(name=name, kind="read", seqs=seqs, old=old, h_kv=h_kv, dim=dim, page=page, dtype=dtype, e4m3=e4m3)


def _packed(name, seqs, new, h_q, h_kv, dim, dtype, causal, lse):
    """attention over packed sequences of up to `new` tokens."""
    return dict(name=name, kind="packed", seqs=seqs, new=new, h_q=h_q, h_kv=h_kv, dim=dim, dtype=dtype,
                causal=causal, lse=lse)


def _paged(name, seqs, new, one, old, h_q, h_kv, dim, page, dtype, e4m3, lse):
    """attention over a paged cache: `one` sequences of a single new token, the others of up to `new`, each
    behind up to `old` tokens."""
    return dict(name=name, kind="paged", seqs=seqs, new=new, one=one, old=old, h_q=h_q, h_kv=h_kv, dim=dim,
                page=page, dtype=dtype, e4m3=e4m3, lse=lse)


def listed():
    return [
        # a decoding step's queries before attention: the call's own latency
        _rotary("rotary-step", 16, 32, 128, 128, "bf16", False, 31987),
        # a long prompt's queries, half of each head rotated in neighbouring pairs, stretched positions
        _rotary("rotary-prompt-16k", 16384, 32, 128, 64, "fp16", True, 131072, 4.0),
        # a decoding step of a large batch into an e4m3 cache
        _write("write-step-e4m3", 64, 1, 4095, 32, 8, 128, 16, "bf16", True, 128, False),
        # ragged prompts straight into 16-bit pages, odd lengths, a small head with a rotated quarter
        _write("write-prompts-fp16", 12, 1000, 333, 28, 4, 64, 32, "fp16", False, 16, True),
        # long conversations out of the e4m3 cache, as a move to another machine or a dense pass needs them
        _read("read-e4m3-32k", 4, 31987, 8, 128, 64, "bf16", True),
        # a few short prompts of a small model in one call
        _packed("packed-short", 5, 100, 16, 16, 64, "fp16", True, False),
        # a batch of prompts of different lengths with grouped heads
        _packed("packed-gqa-2k", 8, 2048, 32, 8, 128, "bf16", True, False),
        # long documents packed for training or scoring, every head with its own K/V; the log-sum-exp too
        _packed("packed-8k-d64-lse", 4, 8192, 16, 16, 64, "fp16", True, True),
        # one token for each of a batch of sequences, 16-bit pages of 16 tokens
        _paged("paged-step-4k", 16, 1, 16, 4095, 32, 8, 128, 16, "bf16", False, False),
        # one token for each of a large ragged batch out of an e4m3 cache
        _paged("paged-step-e4m3-16k", 64, 1, 64, 16000, 32, 8, 128, 64, "bf16", True, False),
        # a chunk of a long prompt beside the steps of running sequences
        _paged("paged-mixed-8k", 25, 500, 24, 8192, 28, 4, 128, 32, "fp16", False, False),
        # the chunks of two long prompts, e4m3 cache; the log-sum-exp merges them with other parts
        _paged("paged-chunk-e4m3-32k", 2, 2048, 0, 31987, 32, 8, 128, 64, "bf16", True, True),
    ]


def _spread(n, most, salt):
    """n lengths in 1 .. most, `most` among them, spread evenly over the range, in a mixed order."""
    turn = (0.7548776662466927, 0.5698402909980532)[salt]
    return [most if i == n // 2 else 1 + int((most - 1) * ((0.5 + turn * (i + 1)) % 1.0)) for i in range(n)]


def _lengths(case):
    """(new, old): each sequence's new tokens, and its tokens in the cache before them."""
    n, kind = case["seqs"], case["kind"]
    if kind == "read":
        return _spread(n, case["old"], 0), [0] * n
    new = _spread(n, case["new"], 0)
    if kind == "paged":
        one = case["one"]
        new = [1] * (one // 2) + _spread(n - one, case["new"], 0) + [1] * (one - one // 2)
    return new, [0] * n if kind == "packed" else _spread(n, case["old"], 1)


def _pairs(new, old, causal):
    return sum(n * o + n * (n + 1) // 2 if causal else n * (n + o) for n, o in zip(new, old))


def work(case):
    """What a pass cannot do without: inputs read once, outputs written once (a cache that is written and
    read back once each way), 2 products of 2 FLOP per visible pair and dim, 3 FLOP per rotated value."""
    kind, dim = case["kind"], case["dim"]
    if kind == "rotary":
        values = case["tokens"] * case["heads"] * dim
        return {"bytes": 4 * values + 8 * case["tokens"] + 4 * case["rot"],
                "flops": 3 * case["tokens"] * case["heads"] * case["rot"]}
    new, old = _lengths(case)
    tokens, total = sum(new), sum(new) + sum(old)
    if kind == "packed":
        rows = tokens * case["h_q"]
        return {"bytes": 4 * rows * dim + 4 * tokens * case["h_kv"] * dim + (4 * rows if case["lse"] else 0),
                "flops": 4 * case["h_q"] * dim * _pairs(new, old, case["causal"])}
    row = case["h_kv"] * (dim + 1 if case["e4m3"] else 2 * dim)  # one token's K (or V) in the cache
    dense = case["h_kv"] * 2 * dim
    if kind == "read":
        return {"bytes": 2 * tokens * (row + dense), "flops": 0}
    if kind == "write":
        return {"bytes": 2 * tokens * (2 * row + 2 * dense) + 4 * tokens * case["h_q"] * dim,
                "flops": 3 * tokens * (case["h_q"] + case["h_kv"]) * case["rot"]}
    rows = tokens * case["h_q"]
    return {"bytes": 4 * rows * dim + 2 * total * row + (4 * rows if case["lse"] else 0),
            "flops": 4 * case["h_q"] * dim * _pairs(new, old, True)}


# A drawn case costs at most this, each a little below the largest listed case's: FLOP, bytes, and score
# elements of sequences padded to the longest.
_MAX_FLOPS = 0.9e12
_MAX_BYTES = 1 << 28
_MAX_SCORES = 4 << 30


def _scores(case):
    new, old = _lengths(case)
    return case["seqs"] * case["h_q"] * max(new) * max(n + o for n, o in zip(new, old))


def draw(rng):
    def log_int(lo, hi):
        return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))

    kind = rng.choice(["rotary", "write", "read", "packed", "packed", "paged", "paged", "paged"])
    h_kv, group = rng.choice([(4, 1), (8, 1), (16, 1), (4, 2), (2, 4), (8, 4), (4, 5), (4, 7), (4, 8), (1, 16)])
    h_q, dim, dtype = h_kv * group, rng.choice([32, 64, 64, 128, 128, 128]), rng.choice(["bf16", "fp16"])
    rot = rng.choice([r for r in (16, 32, 64, 96, 128) if r <= dim])
    page, e4m3, interleaved = rng.choice([32, 32, 64, 128]), rng.random() < 0.5, rng.random() < 0.5
    if kind == "rotary":
        case = _rotary(None, log_int(1, 32768), h_q, dim, rot, dtype, interleaved, log_int(64, 1 << 20),
                       rng.choice([1.0, 1.0, 2.0, 8.0]))
    elif kind == "write":
        case = _write(None, log_int(1, 128), rng.choice([1, log_int(2, 4096)]), log_int(1, 8192), h_q, h_kv, dim,
                      page, dtype, e4m3, rot, interleaved)
    elif kind == "read":
        case = _read(None, log_int(1, 32), log_int(1, 32768), h_kv, dim, page, dtype, e4m3)
    elif kind == "packed":
        case = _packed(None, log_int(1, 64), log_int(1, 8192), h_q, h_kv, dim, dtype, rng.random() < 0.8,
                       rng.random() < 0.3)
    else:
        seqs, new = log_int(1, 128), rng.choice([1, 1, log_int(2, 2048)])
        one = seqs if new == 1 else rng.choice([0, seqs // 2, seqs - 1])
        case = _paged(None, seqs, new, one, log_int(1, 32768), h_q, h_kv, dim, page, dtype, e4m3,
                      rng.random() < 0.3)
    def most():
        w = work(case)
        return max(w["flops"] / _MAX_FLOPS, w["bytes"] / _MAX_BYTES,
                   _scores(case) / _MAX_SCORES if kind in ("packed", "paged") else 0)
    while most() > 1:
        if kind == "rotary":
            case["tokens"] = int(case["tokens"] * 0.7)
        elif case["seqs"] > 1 and rng.random() < 0.5:
            case["seqs"] = max(1, int(case["seqs"] * 0.7))
            if kind == "paged":
                case["one"] = min(case["one"], case["seqs"])
        else:
            case.update({k: max(1, int(case[k] * 0.8)) for k in ("new", "old") if k in case})
    del case["name"]
    return case


# ------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------

def _frequencies(rot, factor):
    """float64 radians per position of every rotated pair, base 10000, and the factor of the rotated values.
    factor > 1 stretches the context that the frequencies were trained for (4096 positions here): pairs that
    turn at least 32 times within it keep their frequency, those that turn at most once are divided by
    factor, and between the two the share goes with the pair's index; the values grow by
    sqrt-temperature 0.1 ln(factor) + 1."""
    i = torch.arange(rot // 2, dtype=torch.float64)
    freqs = 10000.0 ** (-2.0 * i / rot)
    if factor == 1.0:
        return freqs, 1.0
    pair = [rot * math.log(4096.0 / (2.0 * math.pi * turns)) / (2.0 * math.log(10000.0)) for turns in (32.0, 1.0)]
    low, high = max(math.floor(pair[0]), 0), min(math.ceil(pair[1]), rot - 1)
    ramp = ((i - low) / max(high - low, 1e-3)).clamp(0, 1)
    return freqs * (1 - ramp) + freqs / factor * ramp, 0.1 * math.log(factor) + 1.0


def _e4m3_cache(shape, scale, g):
    """Pages of e4m3 values of N(0, 1) rows, and their scales' bytes (2^(byte - 127)); a sequence's tail of its
    last page holds other tokens' leavings, as pages do."""
    x = torch.randn(shape, device="cuda", generator=g) * scale
    e = torch.frexp(x.abs().amax(-1) / 448.0)[1]
    return (x * torch.exp2(-e.float())[..., None]).to(torch.float8_e4m3fn), (e + 127).to(torch.uint8)


def _state(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, dim = _DTYPES[case["dtype"]], case["dim"]

    def randn(*shape):
        return torch.randn(shape, device="cuda", generator=g).to(dtype)

    s = {"kind": case["kind"]}
    if case["kind"] == "rotary":
        freqs, factor = _frequencies(case["rot"], case["factor"])
        s.update(x=randn(case["tokens"], case["heads"], dim), freqs=freqs.cuda(), scale=factor,
                 interleaved=case["interleaved"],
                 positions=torch.randint(0, case["far"] + 1, (case["tokens"],), device="cuda", generator=g))
        return s
    new, old = _lengths(case)
    lens = [n + o for n, o in zip(new, old)]
    tokens = sum(new)
    cu = torch.zeros(len(new) + 1, dtype=torch.int32)
    cu[1:] = torch.tensor(new).cumsum(0)
    s.update(cu=cu.cuda(), tokens=tokens, longest=max(new))
    if case["kind"] == "packed":
        s.update(q=randn(tokens, case["h_q"], dim), k=randn(tokens, case["h_kv"], dim),
                 v=randn(tokens, case["h_kv"], dim), causal=case["causal"], lse=case["lse"])
        return s
    page = case["page"]
    width = -(-max(lens) // page)  # pages of the longest sequence
    pages = sum(-(-n // page) for n in lens)
    order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
    table = torch.zeros(len(lens), width, dtype=torch.int32, device="cuda")
    used = torch.arange(width)[None] < torch.tensor([-(-n // page) for n in lens])[:, None]
    table[used.cuda()] = order
    s.update(table=table, lens=torch.tensor(lens, dtype=torch.int32).cuda(), longest_kv=max(lens))
    shape = (pages, case["h_kv"], page, dim)
    if case["e4m3"]:
        s["k_cache"], s["k_scale"] = _e4m3_cache(shape, 1.0, g)
        s["v_cache"], s["v_scale"] = _e4m3_cache(shape, 0.7, g)
        s.update({n: s[n].view(torch.float8_e8m0fnu) for n in ("k_scale", "v_scale")})
    else:
        s.update(k_cache=randn(*shape), v_cache=randn(*shape), k_scale=None, v_scale=None)
    s["dtype"] = dtype
    if case["kind"] == "write":
        freqs, factor = _frequencies(case["rot"], 1.0)
        s.update(k=randn(tokens, case["h_kv"], dim), v=randn(tokens, case["h_kv"], dim), freqs=freqs.cuda(),
                 q=randn(tokens, case["h_q"], dim), scale=factor, interleaved=case["interleaved"])
    elif case["kind"] == "paged":
        s.update(q=randn(tokens, case["h_q"], dim), lse=case["lse"])
    return s


def prepare(case, seed):
    return _state(case, seed)


# ------------------------------------------------------------------------------------------
# plain forms
# ------------------------------------------------------------------------------------------

def _rotate(x, positions, s):
    """x [T, H, D] with its first 2 * len(freqs) values rotated, in float64."""
    angle = positions.double()[:, None] * s["freqs"]
    cos, sin = (angle.cos() * s["scale"])[:, None], (angle.sin() * s["scale"])[:, None]
    x = x.double()
    rot = 2 * s["freqs"].numel()
    if s["interleaved"]:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, x[..., rot:]], -1)


def _places(s):
    """(sequence, position) of every packed row."""
    rows = torch.arange(s["tokens"], device="cuda")
    seq = torch.searchsorted(s["cu"][1:].long(), rows, right=True)
    return seq, s["lens"].long()[seq] - s["cu"].long()[seq + 1] + rows


def _store(cache, scale, x, page, at):
    """x [T, H, D] into cache [pages, H, P, D] at (page, at), quantised to e4m3 where it has scales."""
    if scale is None:
        cache[page, :, at] = x.to(cache.dtype)
        return
    m, e = torch.frexp(x.abs().amax(-1) / 448.0)
    e = torch.where(m == 0.5, e - 1, e)
    scale.view(torch.uint8)[page, :, at] = (e + 127).to(torch.uint8)
    cache.view(torch.uint8)[page, :, at] = torch.ldexp(x, -e[..., None]).to(cache.dtype).view(torch.uint8)


def _values(cache, scale, page, at):
    """The values that rows (page, at) of every head stand for, in float32: [rows..., H, D]."""
    if scale is None:
        return cache[page, :, at].float()
    e = scale.view(torch.uint8)[page, :, at].float() - 127.0
    return cache.view(torch.uint8)[page, :, at].view(torch.float8_e4m3fn).float() * torch.exp2(e)[..., None]


def _attend(q, k, v, cu, lens, s, causal):
    """q [T, H_q, D] over k, v [S, L, H_kv, D] (float32), sequence s's first lens[s] keys; its rows are the last
    of them. Sequences are padded to the longest."""
    n_seq, length, h_kv, dim = k.shape
    h_q, most = q.shape[1], s["longest"]
    start, n_q = cu[:-1].long(), (cu[1:] - cu[:-1]).long()
    j = torch.arange(most, device="cuda")
    row = (start[:, None] + j).clamp(max=q.shape[0] - 1)
    group = h_q // h_kv
    qs = q.float()[row].view(n_seq, most, h_kv, group, dim).permute(0, 2, 3, 1, 4)
    qs = qs.reshape(n_seq * h_kv, group * most, dim) / math.sqrt(dim)
    kt = k.permute(0, 2, 3, 1).reshape(n_seq * h_kv, dim, length)
    score = torch.bmm(qs, kt).view(n_seq, h_kv, group, most, length)
    n = torch.arange(length, device="cuda")
    last = lens.long()[:, None] - 1 + ((j - n_q[:, None] + 1).clamp(max=0) if causal else 0 * j)
    score.masked_fill_((n > last[..., None])[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    score.sub_(top).exp_()
    total = score.sum(-1, keepdim=True)
    out = torch.bmm(score.view(n_seq * h_kv, group * most, length),
                    v.transpose(1, 2).reshape(n_seq * h_kv, length, dim))
    out = out.view(n_seq, h_kv, group, most, dim) / total
    lse = (top + total.log())[..., 0]
    keep = j < n_q[:, None]
    out = out.permute(0, 3, 1, 2, 4).reshape(n_seq, most, h_q, dim)[keep].to(q.dtype)
    lse = lse.permute(0, 3, 1, 2).reshape(n_seq, most, h_q)[keep].t().contiguous()
    return (out, lse) if s["lse"] else out


def _plain(s):
    kind = s["kind"]
    if kind == "rotary":
        return _rotate(s["x"], s["positions"], s).to(s["x"].dtype)
    if kind == "packed":
        row = (s["cu"][:-1].long()[:, None] + torch.arange(s["longest"], device="cuda")).clamp(max=s["tokens"] - 1)
        return _attend(s["q"], s["k"].float()[row], s["v"].float()[row], s["cu"], s["cu"][1:] - s["cu"][:-1], s,
                       s["causal"])
    page = s["k_cache"].shape[2]
    if kind == "paged":
        n = torch.arange(s["longest_kv"], device="cuda")
        at = (s["table"].long()[:, n // page], n % page)
        return _attend(s["q"], _values(s["k_cache"], s["k_scale"], *at), _values(s["v_cache"], s["v_scale"], *at),
                       s["cu"], s["lens"], s, True)
    seq, position = _places(s)
    at = (s["table"].long()[seq, position // page], position % page)
    q = []
    if kind == "write":
        _store(s["k_cache"], s["k_scale"], _rotate(s["k"], position, s), *at)
        _store(s["v_cache"], s["v_scale"], s["v"].double(), *at)
        q = [_rotate(s["q"], position, s).to(s["dtype"])]
    return [_values(s["k_cache"], s["k_scale"], *at).to(s["dtype"]),
            _values(s["v_cache"], s["v_scale"], *at).to(s["dtype"]), *q]


def run(state):
    s = state
    if not own:
        return _plain(s)
    fa2, kind = _modules(), s["kind"]
    if kind == "rotary":
        plan = fa2.rotary.Rotary(s["freqs"], s["interleaved"], s["scale"])
        return fa2.rotary.rotary(s["x"], s["positions"], plan)
    if kind == "packed":
        return fa2.packed.attention_packed(s["q"], s["k"], s["v"], s["cu"], causal=s["causal"],
                                           return_lse=s["lse"])
    cache = fa2.paged.KVCache(s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"])
    if kind == "paged":
        return fa2.paged.attention_paged(s["q"], cache, s["table"], s["cu"], s["lens"], return_lse=s["lse"])
    q = []
    if kind == "write":
        plan = fa2.rotary.Rotary(s["freqs"], s["interleaved"], s["scale"])
        q = [fa2.paged.cache_write(cache, s["k"], s["v"], s["table"], s["cu"], s["lens"], rotary=plan, q=s["q"])]
    return [*fa2.paged.cache_read(cache, s["table"], s["cu"], s["lens"], s["tokens"], dtype=s["dtype"]), *q]


# ------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ------------------------------------------------------------------------------------------

def _exact_rotary(x, positions, freqs, interleaved, scale):
    """Every pair as a complex number times scale * exp(i angle)."""
    half = freqs.numel()
    out = x.double().clone()
    turn = torch.polar(torch.full_like(positions, scale, dtype=torch.float64)[:, None].expand(-1, half).contiguous(),
                       torch.outer(positions.double(), freqs))[:, None]
    first, second = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    z = torch.complex(out[..., first].contiguous(), out[..., second].contiguous()) * turn
    out[..., first], out[..., second] = z.real, z.imag
    return out


def _exact_e4m3(x):
    """x [..., D] rounded to the nearest of 2^e times an e4m3 value (ties to even), e the least with every
    |x| <= 448 * 2^e: a value of exponent p >= -6 has steps of 2^(p - 3)."""
    top = x.abs().amax(-1, keepdim=True)
    e = torch.floor(torch.log2(top)) - 8
    e = torch.where(top > 448 * torch.exp2(e), e + 1, e)
    y = x * torch.exp2(-e)
    p = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -9))).clamp(min=-6)
    step = torch.exp2(p - 3)
    return torch.round(y / step) * step * torch.exp2(e)


def _exact_attention(q, k, v, causal):
    """One sequence: q [n, H_q, D] are the last of the m keys k, v [m, H_kv, D]. (out [n, H_q, D], lse [H_q, n])"""
    n, h_q, dim = q.shape
    m, h_kv = k.shape[:2]
    out, lse = torch.empty_like(q), torch.empty(h_q, n, dtype=torch.float64, device="cuda")
    rows = max(1, (1 << 27) // m)
    for h in range(h_q):
        kt, vh = k[:, h // (h_q // h_kv)].t().contiguous(), v[:, h // (h_q // h_kv)].contiguous()
        for r in range(0, n, rows):
            score = q[r:r + rows, h].contiguous() @ kt * dim ** -0.5
            if causal:
                see = torch.arange(r, r + score.shape[0], device="cuda") + (m - n)
                score.masked_fill_(torch.arange(m, device="cuda") > see[:, None], -math.inf)
            lse[h, r:r + rows] = torch.logsumexp(score, 1)
            out[r:r + rows, h] = torch.exp(score - lse[h, r:r + rows, None]) @ vh
    return out, lse


def exact(case, seed):
    s = _state(case, seed)
    if case["kind"] == "rotary":
        return _exact_rotary(s["x"], s["positions"], s["freqs"], s["interleaved"], s["scale"])
    new, old = _lengths(case)
    starts = [sum(new[:i]) for i in range(len(new))]
    if case["kind"] in ("read", "write"):
        positions = torch.cat([torch.arange(o, o + n, device="cuda") for n, o in zip(new, old)])
    if case["kind"] == "write":
        k = _exact_rotary(s["k"], positions, s["freqs"], s["interleaved"], s["scale"])
        v = s["v"].double()
        q = _exact_rotary(s["q"], positions, s["freqs"], s["interleaved"], s["scale"])
        return [_exact_e4m3(k), _exact_e4m3(v), q] if case["e4m3"] else [k, v, q]

    def dense(cache, scale, i):
        """Sequence i's tokens [n, H, D]."""
        length = new[i] + old[i]
        pages = s["table"][i, :-(-length // case["page"])].long()
        x = cache.view(torch.uint8)[pages].view(torch.float8_e4m3fn) if case["e4m3"] else cache[pages]
        x = x.double()
        if case["e4m3"]:
            x = x * torch.exp2(scale.view(torch.uint8)[pages].double() - 127)[..., None]
        return x.transpose(1, 2).reshape(-1, case["h_kv"], case["dim"])[:length]

    if case["kind"] == "read":
        return [torch.cat([dense(s[n + "_cache"], s[n + "_scale"], i) for i in range(len(new))]) for n in ("k", "v")]
    causal = case["kind"] == "paged" or case["causal"]
    outs = []
    for i, (n, first) in enumerate(zip(new, starts)):
        rows = slice(first, first + n)
        if case["kind"] == "packed":
            k, v = s["k"][rows].double(), s["v"][rows].double()
        else:
            k, v = dense(s["k_cache"], s["k_scale"], i), dense(s["v_cache"], s["v_scale"], i)
        outs.append(_exact_attention(s["q"][rows].double(), k, v, causal))
    out, lse = torch.cat([o for o, _ in outs]), torch.cat([x for _, x in outs], 1)
    return (out, lse) if case["lse"] else out
