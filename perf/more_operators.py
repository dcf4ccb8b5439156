"""More operators of a serving step, as measured cases: attention with a sliding window and a few first tokens
that stay visible (packed prompts, and over the paged cache), attention of a batch that shares a long prefix, queries
and keys normalised per head and rotated in one pass (by one position, or by several axes' positions; out of place and
on the way into the cache), and a step's pages: finished sequences' given back, new tokens' taken.

Every operator has a plain form in elementary torch operations, in float32 and rounded once at the end (float64
for angles and for values that are rounded to 8 bits), and the call that a user makes of the package (`own`).
listed() holds twelve cases, draw() more of the same ranges.

Sequences are packed: `cu` [S + 1] holds each sequence's first row, and `lens` [S] the tokens of each in the cache,
the new ones included. Their lengths follow from the case alone (_lengths); values and page tables from the seed.
"""

import math
import os
import sys

import torch

own = False

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "triton-fa2-forward_amd")
_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
_EPS = 1e-6  # of the norms


def _modules():
    """The package's public modules (only where `own` is true)."""
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import fa2.packed
    import fa2.paged
    import fa2.pages
    import fa2.rotary
    return fa2


# ------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------

def _packed(name, seqs, new, h_q, h_kv, dim, dtype, window, sinks, lse):
    """packed sequences of up to `new` tokens; a token sees the `window` newest up to itself, and the first `sinks`."""
    return dict(name=name, kind="packed", seqs=seqs, new=new, h_q=h_q, h_kv=h_kv, dim=dim, dtype=dtype,
                window=window, sinks=sinks, lse=lse)


def _paged(name, seqs, new, one, old, h_q, h_kv, dim, page, dtype, e4m3, window, sinks, lse):
    """the same over a paged cache: `one` sequences of a single new token, the others of up to `new`, each behind up to
    `old` tokens, of which the cache holds the pages that are still seen."""
    return dict(name=name, kind="paged", seqs=seqs, new=new, one=one, old=old, h_q=h_q, h_kv=h_kv, dim=dim, page=page,
                dtype=dtype, e4m3=e4m3, window=window, sinks=sinks, lse=lse)


def _shared(name, seqs, new, prefix, old, h_q, h_kv, dim, page, dtype, e4m3, lse):
    """a batch behind one prefix of `prefix` tokens: up to `new` new tokens each, behind up to `old` of its own."""
    return dict(name=name, kind="shared", seqs=seqs, new=new, prefix=prefix, old=old, h_q=h_q, h_kv=h_kv, dim=dim,
                page=page, dtype=dtype, e4m3=e4m3, lse=lse)


def _turn(name, tokens, h_q, h_kv, dim, rot, dtype, interleaved, axes, far, norm):
    """q and k, each head normalised (norm) and its first `rot` values rotated, by `axes` positions a token."""
    return dict(name=name, kind="turn", tokens=tokens, h_q=h_q, h_kv=h_kv, dim=dim, rot=rot, dtype=dtype,
                interleaved=interleaved, axes=axes, far=far, norm=norm)


def _write(name, seqs, new, old, h_q, h_kv, dim, page, dtype, e4m3, rot, interleaved, axes):
    """up to `new` tokens of each sequence behind up to `old` in the cache: q and k normalised and rotated (axes 1: by
    their positions in the sequence), k and v written into pages, and the written tokens read back."""
    return dict(name=name, kind="write", seqs=seqs, new=new, old=old, h_q=h_q, h_kv=h_kv, dim=dim, page=page,
                dtype=dtype, e4m3=e4m3, rot=rot, interleaved=interleaved, axes=axes)


def _tables(name, seqs, new, old, page, done):
    """the pages of `done` finished sequences given back, and those of up to `new` new tokens of each of the others,
    behind up to `old` in the cache, taken and entered: row starts, lengths, positions and slots of the step."""
    return dict(name=name, kind="tables", seqs=seqs, new=new, old=old, page=page, done=done)


def listed():
    return [
        # a few prompts of a small model whose layers see 128 tokens back
        _packed("window-short-d64", 5, 1000, 16, 16, 64, "fp16", 128, 0, False),
        # long prompts with grouped heads, a window of 1024 and four sinks; the log-sum-exp too
        _packed("window-8k-sinks", 4, 8192, 32, 8, 128, "bf16", 1024, 4, True),
        # one token for each of a large batch of long conversations, e4m3 cache that has dropped what left the window
        _paged("window-step-e4m3-16k", 64, 1, 64, 16000, 32, 8, 128, 64, "bf16", True, 4096, 4, False),
        # a chunk of a long prompt beside the steps of running sequences
        _paged("window-mixed-32k", 25, 2048, 24, 31987, 28, 4, 128, 32, "fp16", False, 2048, 64, False),
        # a batch of answers to one long document, one token each
        _shared("shared-step-8k", 32, 1, 8192, 500, 32, 8, 128, 16, "bf16", False, False),
        # short drafts to be checked behind one very long prefix, e4m3 cache; the log-sum-exp too
        _shared("shared-draft-e4m3-32k", 16, 5, 31987, 300, 28, 4, 128, 64, "fp16", True, True),
        # a decoding step's queries and keys before attention: the call's own latency
        _turn("norm-step", 16, 32, 8, 128, 128, "bf16", False, 1, 31987, True),
        # a long prompt of images and text
        _turn("axes-prompt-16k", 16384, 32, 8, 128, 128, "fp16", False, 3, 16384, True),
        # a decoding step of a large batch into an e4m3 cache
        _write("norm-write-step-e4m3", 64, 1, 4095, 32, 8, 128, 64, "bf16", True, 128, False, 1),
        # ragged prompts of video straight into 16-bit pages, half of each head rotated in neighbouring pairs
        _write("axes-write-prompts", 12, 1000, 333, 28, 4, 128, 32, "fp16", False, 64, True, 3),
        # a decoding step of a large batch, eight sequences of which have ended
        _tables("tables-step-256", 256, 1, 8192, 16, 8),
        # a batch of long prompts admitted where another has ended
        _tables("tables-prompts-2k", 100, 2048, 4096, 64, 50),
    ]


def _spread(n, most, salt):
    """n lengths in 1 .. most, `most` among them, spread evenly over the range, in a mixed order."""
    turn = (0.7548776662466927, 0.5698402909980532)[salt]
    return [most if i == n // 2 else 1 + int((most - 1) * ((0.5 + turn * (i + 1)) % 1.0)) for i in range(n)]


def _lengths(case):
    """(new, old): each sequence's new tokens, and its tokens in the cache before them (behind the prefix, if any)."""
    n, kind = case["seqs"], case["kind"]
    new = _spread(n, case["new"], 0)
    if kind == "paged":
        one = case["one"]
        new = [1] * (one // 2) + _spread(n - one, case["new"], 0) + [1] * (one - one // 2)
    if kind == "packed":
        return new, [0] * n
    old = _spread(n, case["old"], 1)
    if kind == "tables":
        ended = [i * n // case["done"] for i in range(case["done"])] if case["done"] else []
        new = [0 if i in set(ended) else x for i, x in enumerate(new)]
    return new, [x + case["prefix"] for x in old] if kind == "shared" else old


def _seen(new, old, case):
    """(pairs of a row and a key that it sees, keys that some row sees), summed over the sequences."""
    pairs = keys = 0
    for n, o in zip(new, old):
        if "window" not in case:
            pairs += n * o + n * (n + 1) // 2
            keys += n + o
            continue
        w, first = case["window"], case["sinks"]
        for p in (range(o, o + n) if n else ()):
            low = max(p - w + 1, 0)
            pairs += p + 1 - low + min(low, first)
        low = max(o - w + 1, 0)
        keys += o + n - low + min(low, first)
    return pairs, keys


def work(case):
    """What a pass cannot do without: inputs read once, outputs written once (a cache that is written and
    read back once each way), 2 products of 2 FLOP per visible pair and dim, 3 FLOP per rotated value and 4
    per normalised one."""
    kind = case["kind"]
    if kind == "tables":
        new, old = _lengths(case)
        page, tokens, seqs = case["page"], sum(new), case["seqs"]
        taken = sum(-(-(n + o) // page) - -(-o // page) for n, o in zip(new, old))
        given = sum(-(-o // page) for n, o in zip(new, old) if n == 0)
        return {"bytes": 8 * taken + 8 * given + 24 * seqs + 12 * tokens, "flops": 0}
    dim = case["dim"]
    if kind == "turn":
        values = case["tokens"] * (case["h_q"] + case["h_kv"]) * dim
        return {"bytes": 4 * values + 8 * case["axes"] * case["tokens"] + 4 * case["rot"] + (8 * dim if case["norm"] else 0),
                "flops": 3 * values * case["rot"] // dim + (4 * values if case["norm"] else 0)}
    new, old = _lengths(case)
    tokens = sum(new)
    rows = tokens * case["h_q"]
    dense = case["h_kv"] * 2 * dim
    if kind == "packed":
        pairs, _ = _seen(new, old, case)
        return {"bytes": 4 * rows * dim + 2 * tokens * dense + (4 * rows if case["lse"] else 0),
                "flops": 4 * case["h_q"] * dim * pairs}
    row = case["h_kv"] * (dim + 1 if case["e4m3"] else 2 * dim)  # one token's K (or V) in the cache
    if kind == "write":
        return {"bytes": 2 * tokens * (2 * row + 2 * dense) + 4 * rows * dim + 8 * case["axes"] * tokens,
                "flops": tokens * (case["h_q"] + case["h_kv"]) * (3 * case["rot"] + 4 * dim)}
    pairs, keys = _seen(new, old, case)
    if kind == "shared":
        keys -= (case["seqs"] - 1) * (case["prefix"] // case["page"] * case["page"])
    return {"bytes": 4 * rows * dim + 2 * keys * row + (4 * rows if case["lse"] else 0),
            "flops": 4 * case["h_q"] * dim * pairs}


# A drawn case costs at most this, each a little below the largest listed case's: FLOP, bytes, and score
# elements of sequences padded to the longest.
_MAX_FLOPS = 0.21e12
_MAX_BYTES = 1 << 28
_MAX_SCORES = 4 << 30


def _scores(case):
    new, old = _lengths(case)
    return case["seqs"] * case["h_q"] * max(new) * max(n + o for n, o in zip(new, old))


def draw(rng):
    def log_int(lo, hi):
        return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))

    kind = rng.choice(["packed", "packed", "paged", "paged", "shared", "shared", "turn", "write", "tables"])
    h_kv, group = rng.choice([(4, 1), (8, 1), (16, 1), (4, 2), (2, 4), (8, 4), (4, 5), (4, 7), (4, 8), (1, 16)])
    h_q, dim, dtype = h_kv * group, rng.choice([32, 64, 64, 128, 128, 128]), rng.choice(["bf16", "fp16"])
    rot = rng.choice([r for r in (16, 32, 64, 96, 128) if r <= dim])
    page, e4m3, interleaved = rng.choice([32, 32, 64, 128]), rng.random() < 0.5, rng.random() < 0.5
    window, sinks, lse = log_int(16, 8192), rng.choice([0, 0, 1, 4, log_int(2, 256)]), rng.random() < 0.3
    axes = rng.choice([1, 2, 3])
    if kind == "packed":
        case = _packed(None, log_int(1, 64), log_int(1, 8192), h_q, h_kv, dim, dtype, window, sinks, lse)
    elif kind == "paged":
        seqs, new = log_int(1, 128), rng.choice([1, 1, log_int(2, 2048)])
        one = seqs if new == 1 else rng.choice([0, seqs // 2, seqs - 1])
        case = _paged(None, seqs, new, one, log_int(1, 32768), h_q, h_kv, dim, page, dtype, e4m3, window, sinks, lse)
    elif kind == "shared":
        case = _shared(None, log_int(2, 128), rng.choice([1, 1, log_int(2, 64)]), log_int(64, 32768), log_int(1, 2048),
                       h_q, h_kv, dim, page, dtype, e4m3, lse)
    elif kind == "turn":
        case = _turn(None, log_int(1, 16384), h_q, h_kv, dim, rot, dtype, interleaved, axes, log_int(64, 1 << 20),
                     rng.random() < 0.7)
    elif kind == "write":
        case = _write(None, log_int(1, 128), rng.choice([1, log_int(2, 4096)]), log_int(1, 8192), h_q, h_kv, dim,
                      page, dtype, e4m3, rot, interleaved, axes)
    else:
        seqs = log_int(2, 1024)
        case = _tables(None, seqs, rng.choice([1, log_int(2, 2048)]), log_int(1, 16384), rng.choice([16, 32, 64, 128]),
                       rng.choice([0, 1, seqs // 2]))

    def most():
        if kind == "tables":
            return sum(_lengths(case)[0]) / 100000
        w = work(case)
        return max(w["flops"] / _MAX_FLOPS, w["bytes"] / _MAX_BYTES,
                   _scores(case) / _MAX_SCORES if kind in ("packed", "paged", "shared") else 0)

    while most() > 1:
        if kind == "turn":
            case["tokens"] = int(case["tokens"] * 0.7)
        elif case["seqs"] > 2 and rng.random() < 0.5:
            case["seqs"] = max(2, int(case["seqs"] * 0.7))
            case.update({k: min(case[k], case["seqs"] - (k == "done")) for k in ("one", "done") if k in case})
        else:
            case.update({k: max(1, int(case[k] * 0.8)) for k in ("new", "old") if k in case})
    del case["name"]
    return case


# ------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------

def _frequencies(rot):
    """float64 radians per position of every rotated pair, base 10000."""
    return 10000.0 ** (-2.0 * torch.arange(rot // 2, dtype=torch.float64) / rot)


def _axes(rot, axes):
    """The axis that each pair turns by: a quarter of the pairs by the first, the rest in equal blocks by the
    others."""
    half = rot // 2
    if axes == 1:
        return None
    first = half // 4
    return torch.tensor([0 if i < first else 1 + (i - first) * (axes - 1) // (half - first) for i in range(half)],
                        dtype=torch.int32, device="cuda")


def _e4m3_cache(shape, scale, g):
    """Pages of e4m3 values of N(0, 1) rows, and their scales' bytes (2^(byte - 127)); a sequence's tail of its
    last page holds other tokens' leavings, as pages do."""
    x = torch.randn(shape, device="cuda", generator=g) * scale
    e = torch.frexp(x.abs().amax(-1) / 448.0)[1]
    return (x * torch.exp2(-e.float())[..., None]).to(torch.float8_e4m3fn), (e + 127).to(torch.uint8)


def _places_in_pages(case, new, old):
    """bool [S, W]: the entries of the page table that are pages (of a window: those that a row sees)."""
    page = case["page"]
    width = -(-max(n + o for n, o in zip(new, old)) // page)
    used = torch.zeros(len(new), width, dtype=torch.bool)
    for s, (n, o) in enumerate(zip(new, old)):
        used[s, :-(-(n + o) // page)] = True
        if "window" in case:
            low = max(o - case["window"] + 1, 0) // page
            used[s, min(low, -(-case["sinks"] // page)):low] = False
    return used


def _tables_state(case, g):
    new, old = _lengths(case)
    page, n = case["page"], len(new)
    held = [-(-o // page) for o in old]
    width = max(-(-(a + o) // page) for a, o in zip(new, old))
    spare = sum(-(-(a + o) // page) for a, o in zip(new, old)) - sum(held) + 64
    order = torch.randperm(sum(held) + spare, device="cuda", generator=g).to(torch.int32)
    table = torch.full((n, width), -1, dtype=torch.int32, device="cuda")
    used = torch.arange(width)[None] < torch.tensor(held)[:, None]
    table[used.cuda()] = order[:sum(held)]
    free = torch.zeros_like(order)
    free[:spare] = order[sum(held):]
    given = torch.tensor([h if a == 0 else 0 for h, a in zip(held, new)], dtype=torch.int32)
    lens = torch.tensor([0 if a == 0 else o for a, o in zip(new, old)], dtype=torch.int32)
    return {"kind": "tables", "page": page, "tokens": sum(new), "table": table, "free": free,
            "count": torch.tensor([spare], dtype=torch.int32, device="cuda"), "given": given.cuda(),
            "none": torch.zeros_like(given).cuda(), "lens": lens.cuda(),
            "new": torch.tensor(new, dtype=torch.int32).cuda()}


def _state(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if case["kind"] == "tables":
        return _tables_state(case, g)
    dtype, dim, kind = _DTYPES[case["dtype"]], case["dim"], case["kind"]

    def randn(*shape):
        return torch.randn(shape, device="cuda", generator=g).to(dtype)

    s = {"kind": kind, "dtype": dtype, "lse": case.get("lse"), "window": case.get("window"), "sinks": case.get("sinks", 0)}
    if kind in ("turn", "write"):
        s.update(freqs=_frequencies(case["rot"]).cuda(), interleaved=case["interleaved"], axes=_axes(case["rot"], case["axes"]))
        if case.get("norm", True):
            s.update({n: 1.0 + 0.2 * torch.randn(dim, device="cuda", generator=g) for n in ("q_weight", "k_weight")})
        else:
            s.update(q_weight=None, k_weight=None)

    def positions(tokens, far):
        """Images' and videos' positions: each axis runs over a range of its own; text: one position."""
        if case["axes"] == 1:
            return torch.randint(0, far + 1, (tokens,), device="cuda", generator=g)
        p = torch.randint(0, far + 1, (case["axes"], tokens), device="cuda", generator=g)
        p[1:] //= 16
        return p

    if kind == "turn":
        s.update(q=randn(case["tokens"], case["h_q"], dim), k=randn(case["tokens"], case["h_kv"], dim),
                 positions=positions(case["tokens"], case["far"]))
        return s
    new, old = _lengths(case)
    lens = [n + o for n, o in zip(new, old)]
    tokens = sum(new)
    cu = torch.zeros(len(new) + 1, dtype=torch.int32)
    cu[1:] = torch.tensor(new).cumsum(0)
    s.update(cu=cu.cuda(), tokens=tokens, longest=max(new), q=randn(tokens, case["h_q"], dim))
    if kind == "packed":
        s.update(k=randn(tokens, case["h_kv"], dim), v=randn(tokens, case["h_kv"], dim))
        return s
    page = case["page"]
    used = _places_in_pages(case, new, old)
    common = case.get("prefix", 0) // page
    used[1:, :common] = False
    pages = int(used.sum())
    table = torch.full(used.shape, -1, dtype=torch.int32, device="cuda")
    table[used.cuda()] = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
    table[:, :common] = table[0, :common]
    s.update(table=table, lens=torch.tensor(lens, dtype=torch.int32).cuda(), longest_kv=max(lens))
    if kind == "shared":
        s["shared"] = torch.tensor([case["prefix"]], dtype=torch.int32).cuda()
    shape = (pages, case["h_kv"], page, dim)
    if case["e4m3"]:
        s["k_cache"], s["k_scale"] = _e4m3_cache(shape, 1.0, g)
        s["v_cache"], s["v_scale"] = _e4m3_cache(shape, 0.7, g)
        s.update({n: s[n].view(torch.float8_e8m0fnu) for n in ("k_scale", "v_scale")})
    else:
        s.update(k_cache=randn(*shape), v_cache=randn(*shape), k_scale=None, v_scale=None)
    if kind == "write":
        s.update(k=randn(tokens, case["h_kv"], dim), v=randn(tokens, case["h_kv"], dim),
                 positions=positions(tokens, case["old"]) if case["axes"] > 1 else None)
    return s


def prepare(case, seed):
    return _state(case, seed)


# ------------------------------------------------------------------------------------------
# plain forms
# ------------------------------------------------------------------------------------------

def _normed(x, weight):
    """x [T, H, D] in float64, every head divided by its root mean square, times weight."""
    x = x.double()
    if weight is None:
        return x
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS) * weight.double()


def _rotate(x, positions, s):
    """x [T, H, D] (float64) with its first 2 * len(freqs) values rotated by positions [T], or [axes, T]."""
    if s["axes"] is None:
        angle = positions.double()[:, None] * s["freqs"]
    else:
        angle = positions.double()[s["axes"].long()].t() * s["freqs"]
    cos, sin = angle.cos()[:, None], angle.sin()[:, None]
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


def _attend(q, k, v, cu, lens, s):
    """q [T, H_q, D] over k, v [S, L, H_kv, D] (float32), sequence s's first lens[s] keys; its rows are the last
    of them, each sees up to its own key, of a window the newest and the first ones. Sequences are padded to the longest."""
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
    last = (lens.long()[:, None] - 1 + (j - n_q[:, None] + 1).clamp(max=0))[..., None]
    hidden = n > last
    if s["window"] is not None:
        hidden |= (n <= last - s["window"]) & (n >= s["sinks"])
    score.masked_fill_(hidden[:, None, None], -math.inf)
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


def _plain_tables(s):
    """Given-back pages go on top of the free ones, a sequence's in order after those of the sequence before; pages are
    taken from the top together, in the order of the sequences' needs."""
    page, table, lens, new = s["page"], s["table"], s["lens"].long(), s["new"].long()
    column = torch.arange(table.shape[1], device="cuda")
    given = table[(column >= s["none"][:, None]) & (column < s["given"][:, None])]
    count = int(s["count"])
    free = s["free"].clone()
    free[count:count + given.numel()] = given
    count += given.numel()
    held, want = (lens + page - 1) // page, (lens + new + page - 1) // page
    fresh = (column >= held[:, None]) & (column < want[:, None])
    need = int((want - held).sum())
    table = table.clone()
    table[fresh] = free[count - need:count]
    cu = torch.zeros(lens.numel() + 1, dtype=torch.int64, device="cuda")
    cu[1:] = new.cumsum(0)
    rows = torch.arange(s["tokens"], device="cuda")
    seq = torch.searchsorted(cu[1:], rows, right=True)
    position = lens[seq] + rows - cu[seq]
    slot = table[seq, position // page].long() * page + position % page
    return [table, cu.int(), (lens + new).int(), position.int(), slot, free,
            torch.tensor([count - need], dtype=torch.int32, device="cuda")]


def _plain(s):
    kind = s["kind"]
    if kind == "tables":
        return _plain_tables(s)
    if kind == "turn":
        return [_rotate(_normed(s[n], s[n + "_weight"]), s["positions"], s).to(s["dtype"]) for n in ("q", "k")]
    if kind == "packed":
        row = (s["cu"][:-1].long()[:, None] + torch.arange(s["longest"], device="cuda")).clamp(max=s["tokens"] - 1)
        return _attend(s["q"], s["k"].float()[row], s["v"].float()[row], s["cu"], s["cu"][1:] - s["cu"][:-1], s)
    page = s["k_cache"].shape[2]
    if kind in ("paged", "shared"):
        n = torch.arange(s["longest_kv"], device="cuda")
        at = (s["table"].long().clamp(min=0)[:, n // page], n % page)
        return _attend(s["q"], _values(s["k_cache"], s["k_scale"], *at), _values(s["v_cache"], s["v_scale"], *at),
                       s["cu"], s["lens"], s)
    seq, position = _places(s)
    at = (s["table"].long()[seq, position // page], position % page)
    turn = position if s["positions"] is None else s["positions"]
    _store(s["k_cache"], s["k_scale"], _rotate(_normed(s["k"], s["k_weight"]), turn, s), *at)
    _store(s["v_cache"], s["v_scale"], s["v"].double(), *at)
    return [_values(s["k_cache"], s["k_scale"], *at).to(s["dtype"]),
            _values(s["v_cache"], s["v_scale"], *at).to(s["dtype"]),
            _rotate(_normed(s["q"], s["q_weight"]), turn, s).to(s["dtype"])]


def run(state):
    s = state
    if not own:
        return _plain(s)
    fa2, kind = _modules(), s["kind"]
    if kind == "tables":
        pool = fa2.pages.PagePool(s["free"], s["count"])
        pool = fa2.pages.pages_release(pool, s["table"], s["none"], s["given"])
        step = fa2.pages.pages_extend(pool, s["table"], s["lens"], s["new"], s["page"], s["tokens"])
        return [s["table"], step.cu_seqlens, step.seqlens, step.positions, step.slots, step.pool.free, step.pool.count]
    if kind in ("turn", "write"):
        plan = fa2.rotary.Rotary(s["freqs"], s["interleaved"], 1.0, s["axes"])
        q_norm, k_norm = (None if s[n] is None else fa2.rotary.HeadNorm(s[n], _EPS) for n in ("q_weight", "k_weight"))
    if kind == "turn":
        return fa2.rotary.rotary_qk(s["q"], s["k"], s["positions"], plan, q_norm=q_norm, k_norm=k_norm)
    if kind == "packed":
        return fa2.packed.attention_packed(s["q"], s["k"], s["v"], s["cu"], window=s["window"], sinks=s["sinks"],
                                           return_lse=s["lse"])
    cache = fa2.paged.KVCache(s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"])
    if kind == "paged":
        return fa2.paged.attention_paged(s["q"], cache, s["table"], s["cu"], s["lens"], window=s["window"],
                                         sinks=s["sinks"], return_lse=s["lse"])
    if kind == "shared":
        return fa2.paged.attention_paged(s["q"], cache, s["table"], s["cu"], s["lens"], shared=s["shared"],
                                         return_lse=s["lse"])
    q = fa2.paged.cache_write(cache, s["k"], s["v"], s["table"], s["cu"], s["lens"], rotary=plan, q=s["q"],
                              q_norm=q_norm, k_norm=k_norm, positions=s["positions"])
    return [*fa2.paged.cache_read(cache, s["table"], s["cu"], s["lens"], s["tokens"], dtype=s["dtype"]), q]


# ------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ------------------------------------------------------------------------------------------

def _exact_turn(x, weight, angles, interleaved):
    """Heads divided by sqrt(mean of squares + eps) and times weight; then every pair as a complex number times
    exp(i angle), angles [T, rot / 2]."""
    out = x.double().clone()
    if weight is not None:
        size = torch.sqrt(out.pow(2).sum(-1) / out.shape[-1] + _EPS)
        out = torch.einsum("thd,d->thd", out / size[..., None], weight.double())
    half = angles.shape[1]
    turn = torch.polar(torch.ones_like(angles), angles)[:, None]
    first, second = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    z = torch.complex(out[..., first].contiguous(), out[..., second].contiguous()) * turn
    out[..., first], out[..., second] = z.real, z.imag
    return out


def _exact_angles(s, positions):
    if s["axes"] is None:
        return torch.outer(positions.double(), s["freqs"])
    return torch.stack([positions[a].double() * f for a, f in zip(s["axes"].tolist(), s["freqs"].tolist())], 1)


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


def _exact_attention(q, key_of, value_of, m, window, sinks):
    """One sequence: q [n, H_q, D] are the last of m keys; key_of(h, i) gives K [len(i), D] of KV head h at positions
    i, value_of V. Only keys that a block of rows sees are looked at. (out [n, H_q, D], lse [H_q, n])"""
    n, h_q, dim = q.shape
    h_kv = key_of(None, None)
    group = h_q // h_kv
    out, lse = torch.empty_like(q), torch.empty(h_q, n, dtype=torch.float64, device="cuda")
    rows = max(1, (1 << 25) // m) if window is None else max(256, min(window, 2048))
    for r in range(0, n, rows):
        own_key = torch.arange(m - n + r, m - n + min(r + rows, n), device="cuda")
        low = 0 if window is None else max(int(own_key[0]) - window + 1, 0)
        keys = torch.cat([torch.arange(min(sinks, low), device="cuda"), torch.arange(low, int(own_key[-1]) + 1, device="cuda")])
        see = keys <= own_key[:, None]
        if window is not None:
            see &= (keys > own_key[:, None] - window) | (keys < sinks)
        for h in range(h_kv):
            kt, vh = key_of(h, keys).t().contiguous(), value_of(h, keys)
            for x in range(h * group, (h + 1) * group):
                score = q[r:r + rows, x].contiguous() @ kt * dim ** -0.5
                score = torch.where(see, score, torch.full_like(score, -math.inf))
                lse[x, r:r + rows] = torch.logsumexp(score, 1)
                out[r:r + rows, x] = torch.exp(score - lse[x, r:r + rows, None]) @ vh
    return out, lse


def _exact_tables(case, seed):
    """The step in Python, a token at a time where that is the clearest form."""
    s = _state(case, seed)
    page = s["page"]
    table, free, count = s["table"].tolist(), s["free"].tolist(), int(s["count"])
    for row, n in zip(table, s["given"].tolist()):
        for p in row[:n]:
            free[count] = p
            count += 1
    lens, new = s["lens"].tolist(), s["new"].tolist()
    needs = [-(-(a + n) // page) - -(-a // page) for a, n in zip(lens, new)]
    at = count = count - sum(needs)
    cu, positions, slots = [0], [], []
    for row, a, n, need in zip(table, lens, new, needs):
        held = -(-a // page)
        for i in range(need):
            row[held + i] = free[at]
            at += 1
        for p in range(a, a + n):
            positions.append(p)
            slots.append(row[p // page] * page + p % page)
        cu.append(cu[-1] + n)

    def i32(x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")
    return [i32(table), i32(cu), i32([a + n for a, n in zip(lens, new)]), i32(positions),
            torch.tensor(slots, dtype=torch.int64, device="cuda"), i32(free), i32([count])]


def exact(case, seed):
    if case["kind"] == "tables":
        return _exact_tables(case, seed)
    s = _state(case, seed)
    if case["kind"] == "turn":
        angles = _exact_angles(s, s["positions"])
        return [_exact_turn(s[n], s[n + "_weight"], angles, s["interleaved"]) for n in ("q", "k")]
    new, old = _lengths(case)
    starts = [sum(new[:i]) for i in range(len(new))]
    if case["kind"] == "write":
        positions = s["positions"]
        if positions is None:
            positions = torch.cat([torch.arange(o, o + n, device="cuda") for n, o in zip(new, old)])
        angles = _exact_angles(s, positions)
        q, k = (_exact_turn(s[n], s[n + "_weight"], angles, s["interleaved"]) for n in ("q", "k"))
        v = s["v"].double()
        return [_exact_e4m3(k), _exact_e4m3(v), q] if case["e4m3"] else [k, v, q]

    def reader(name, i, rows):
        """f(h, keys): KV head h's K or V of sequence i at `keys`, float64; f(None, None): the number of KV heads"""
        def read(h, keys):
            if h is None:
                return case["h_kv"]
            if case["kind"] == "packed":
                return s[name][rows][keys, h].double()
            page, at = s["table"][i].long()[keys // case["page"]], keys % case["page"]
            if not case["e4m3"]:
                return s[name + "_cache"][page, h, at].double()
            x = s[name + "_cache"].view(torch.uint8)[page, h, at].view(torch.float8_e4m3fn).double()
            return x * torch.exp2(s[name + "_scale"].view(torch.uint8)[page, h, at].double() - 127)[:, None]
        return read

    outs = []
    for i, (n, o, first) in enumerate(zip(new, old, starts)):
        rows = slice(first, first + n)
        outs.append(_exact_attention(s["q"][rows].double(), reader("k", i, rows), reader("v", i, rows), n + o,
                                     s["window"], s["sinks"]))
    out, lse = torch.cat([o for o, _ in outs]), torch.cat([x for _, x in outs], 1)
    return (out, lse) if case["lse"] else out
