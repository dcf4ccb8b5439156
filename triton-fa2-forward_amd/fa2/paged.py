"""A paged K/V cache and attention over it on AMD MI355X (gfx950).

A KVCache holds the tokens of many sequences in pages of a fixed number of tokens, in 16 bits, or in 8:
e4m3 with a power-of-two scale for each token and head, which costs no rounding of its own. cache_write() puts
new tokens into their pages (keys rotated on the way, see fa2.rotary), attention_paged() is the attention of
the new tokens over everything that their sequences have in the cache, cache_read() takes tokens out again.

All three take the same description of a step: the packed rows of the sequences' newest tokens (cu_seqlens), how
many tokens each sequence has in the cache, these included (seqlens), and its pages (block_table). It is read on
the device: nothing is copied to the host, and a captured graph follows what the tensors hold at each
replay. The HIP kernels are csrc/serve_cache.hip and csrc/attn_ragged.hpp behind include/fa2_fwd.h.
"""

from typing import NamedTuple, Optional

import torch

from . import _lib
from .kernel import _cu_count
from .packed import _index, _output, _rows, _scale, _window
from .rotary import _check_axes, _check_norm, _check_plan, _positions

_16BIT = (torch.float16, torch.bfloat16)


class KVCache(NamedTuple):
    """k, v: [pages, H_kv, page_size, D], fp16, bf16 or float8_e4m3fn, any strides with a unit one for D (a
    [pages, page_size, H_kv, D] storage by transpose(1, 2)); k_scale, v_scale: float8_e8m0fnu
    [pages, H_kv, page_size] with e4m3, else None. page_size: a power of two from 16 to 2^20, and at least 1 KiB
    of a head's rows. A page extends over less than 2^31 bytes, and lies less than that from the next."""
    k: torch.Tensor
    v: torch.Tensor
    k_scale: Optional[torch.Tensor] = None
    v_scale: Optional[torch.Tensor] = None

    @classmethod
    def empty(cls, pages, h_kv, page_size, head_dim, dtype=torch.bfloat16, device="cuda"):
        """A cache of `pages` pages: zeros, so that no page holds what was in memory before."""
        assert dtype in _16BIT or dtype == torch.float8_e4m3fn
        shape = (pages, h_kv, page_size, head_dim)
        if dtype in _16BIT:
            return cls(*(torch.zeros(shape, dtype=dtype, device=device) for _ in "kv"))
        return cls(*(torch.zeros(shape, dtype=torch.uint8, device=device).view(dtype) for _ in "kv"),
                   *(torch.full(shape[:3], 127, dtype=torch.uint8, device=device).view(torch.float8_e8m0fnu)
                     for _ in "kv"))


def _check_cache(cache, dtype):
    """The cache's sizes and types, for rows of `dtype`."""
    k, v = cache.k, cache.v
    assert k.dim() == 4 and v.shape == k.shape and v.dtype == k.dtype, "a cache's k and v are of one shape and type"
    pages, _, page_size, D = k.shape
    assert D in (16, 32, 64, 128), "head_dim must be a power of two in [16, 128]"
    assert dtype in _16BIT
    e4m3 = k.dtype == torch.float8_e4m3fn
    assert e4m3 or k.dtype == dtype, "a 16-bit cache is of the rows' own type"
    if pages < 1 or page_size < 16 or page_size & (page_size - 1) or page_size * D * (1 if e4m3 else 2) < 1024:
        raise ValueError("page_size must be a power of two of at least 16 with at least 1024 bytes of a head's "
                         f"rows, and at least one page, got {pages} pages of {page_size} tokens")
    step = 16 if e4m3 else 8
    for name, t in (("k", k), ("v", v)):
        # written in place, so never copied: what the kernels cannot address is refused
        if t.data_ptr() % 16 or t.stride(3) != 1 or any(n > 1 and s % step for n, s in zip(t.shape[:3], t.stride())):
            raise ValueError(f"the cache's {name} must be 16-byte aligned, with a unit stride for head_dim and the "
                             f"others multiples of {step} elements, got {t.stride()}")
        if t.stride(2) > 1 << 22:
            raise ValueError(f"the cache's {name} has a token stride above 2^22 elements")
    if e4m3:
        for name, t in (("k_scale", cache.k_scale), ("v_scale", cache.v_scale)):
            assert t is not None and t.shape == k.shape[:3] and t.dtype == torch.float8_e8m0fnu, (
                f"an e4m3 cache has a float8_e8m0fnu {name} [pages, H_kv, page_size]")
    for t in cache:
        if t is not None and (not t.is_cuda or t.device != k.device):
            raise RuntimeError(f"a cache's tensors must be on one GPU, got {k.device} and {t.device}")


def _step(cache, block_table, cu_seqlens, seqlens, n_tokens):
    """The C ABI's descriptions of the cache and of the sequences over it (and what keeps them alive)."""
    device = cache.k.device
    assert block_table.dim() == 2 and block_table.dtype == torch.int32, "block_table is int32 [S, pages]"
    assert cu_seqlens.numel() == seqlens.numel() + 1 == block_table.shape[0] + 1, (
        "cu_seqlens holds S + 1 entries, seqlens and block_table S")
    if block_table.device != device:
        raise RuntimeError(f"block_table must be on {device}, got {block_table.device}")
    cu, lens = _index(cu_seqlens, "cu_seqlens", device), _index(seqlens, "seqlens", device)
    table = block_table if block_table.stride(1) == 1 or block_table.shape[1] == 1 else block_table.contiguous()
    return _lib.cache_of(cache), _lib.sequences_of(cu, lens, table, n_tokens), (cu, lens, table)


def _check_kv(cache, k, v):
    assert k.dim() == 3 and k.shape == v.shape and k.dtype == v.dtype
    assert tuple(k.shape[1:]) == (cache.k.shape[1], cache.k.shape[3]), "k and v are [T, H_kv, D] of the cache's"
    if k.device != cache.k.device or v.device != cache.k.device:
        raise RuntimeError(f"k and v must be on {cache.k.device}, got {k.device} and {v.device}")


def cache_write(cache, k, v, block_table, cu_seqlens, seqlens, *, rotary=None, q=None, q_out=None, q_norm=None,
                k_norm=None, positions=None):
    """Write the new tokens' k and v [T, H_kv, D] into their places in the cache.

    block_table: int32 [S, pages], the pages of every sequence in order; cu_seqlens: int32 [S + 1], sequence s's new
    tokens are rows cu_seqlens[s] .. cu_seqlens[s + 1] - 1; seqlens: int32 [S], its tokens in the cache, the new ones
    included (the first new one goes to position seqlens[s] minus their number).
    rotary: a fa2.rotary.Rotary; k is rotated by its position before it is written, and so is q [T, H_q, D], if given,
        into q_out (a new tensor; q_out=q rotates in place), which is returned.
    q_norm, k_norm: a fa2.rotary.HeadNorm (with rotary): every head of q, or of k, is normalised before it is rotated.
    positions: int32 or int64 [T], or with a plan's axes [axes, T] (which it needs): what q and k are rotated by, in the place
        of the position in the sequence.
    An e4m3 cache rounds each token and head once, against its own power-of-two scale (the least that holds its
    largest finite value); what is not finite becomes NaN.
    Not written: tokens past the table or in a page outside the cache, rows of no sequence, and rows before their
    sequence's start (where it has more rows than tokens in the cache); q_out is left as it is at the last two (undefined
    in a new one). Two tokens in one place are the caller's to avoid.
    """
    turned = positions is not None or q_norm is not None or k_norm is not None or (
        rotary is not None and rotary.axes is not None)
    if _lib.native is not None:  # the common call, made natively; None: not one of those
        plan = (None, False, 1.0, None) if rotary is None else (rotary.freqs, rotary.interleaved, rotary.scale, rotary.axes)
        args = (*cache, block_table, cu_seqlens, seqlens, k, v, *plan, q, q_out)
        if turned:
            result = _lib.native.cache_write_turned(*args, *(q_norm or (None, 0.0)), *(k_norm or (None, 0.0)), positions)
        else:
            result = _lib.native.cache_write(*args)
        if result is not None:
            return q_out if q is None or q_out is not None else result
    _check_cache(cache, k.dtype)
    _check_kv(cache, k, v)
    T, D = k.shape[0], k.shape[2]
    device = cache.k.device
    rotation = keep = None
    if rotary is not None:
        keep = _check_plan(rotary, D, device)
        rotation = _lib.Rotation(keep.data_ptr(), keep.numel(), rotary.interleaved, rotary.scale)
    assert q is not None or q_out is None, "q_out is q's"
    if turned:
        assert rotary is not None, "norms and positions are of a rotation: they need a rotary plan"
        assert q is not None or q_norm is None, "q_norm is q's"
        axes = _check_axes(rotary, device)
        norms = _check_norm(q_norm, "q_norm", D, device), _check_norm(k_norm, "k_norm", D, device)
        if positions is not None:
            if positions.device != device:
                raise RuntimeError(f"positions must be on {device}, got {positions.device}")
            positions = _positions(positions, rotary, 1, T, True)[:, 0]
        elif axes is not None:
            raise ValueError("a plan's axes need positions")
        turn = _lib.turn_of(rotary, keep, axes, 1 if positions is None else positions.shape[0], *norms)
    o_ = None
    if q is not None:
        assert rotary is not None, "q is taken to be rotated: it needs a rotary plan"
        assert q.dim() == 3 and q.shape[0] == T and q.shape[2] == D and q.dtype == k.dtype and q.shape[1] > 0
        if q.device != device:
            raise RuntimeError(f"q must be on {device}, got {q.device}")
        q_out, o_ = _output(q, q_out)
    c, s, alive = _step(cache, block_table, cu_seqlens, seqlens, T)
    if T:
        rows = _rows(k), _rows(v), None if q is None else _rows(q), o_
        with torch.cuda.device(device):
            stream = torch.cuda.current_stream(device).cuda_stream
            if turned:
                _lib.cache_write_turned(c, s, *rows, positions, turn, stream)
            else:
                _lib.cache_write(c, s, *rows, rotation, stream)
        if o_ is not q_out:
            q_out.copy_(o_)
    return q_out


def cache_read(cache, block_table, cu_seqlens, seqlens, n_tokens, *, dtype=None, out=None):
    """The sequences' last tokens out of the cache, dense: (k, v), each [n_tokens, H_kv, D].

    Takes the tokens that cache_write would write for the same block_table, cu_seqlens and seqlens; whole
    sequences with cu_seqlens the running sum of seqlens. n_tokens: rows of the result (cu_seqlens[-1], which is not
    copied to the host to find out). dtype: fp16 or bf16, for an e4m3 cache (a 16-bit one gives its own).
    Tokens past the table or in a page outside the cache read as zeros; rows of no sequence or before their
    sequence's start are left as they are in out=(k, v) (undefined in new ones).
    """
    if dtype is None:
        assert cache.k.dtype in _16BIT or out is not None, "an e4m3 cache needs the dtype to read it as"
        dtype = cache.k.dtype if out is None else out[0].dtype
    if out is None and _lib.native is not None:  # the common call, made natively; None: not one of those
        result = _lib.native.cache_read(*cache, block_table, cu_seqlens, seqlens, n_tokens, dtype)
        if result is not None:
            return result
    _check_cache(cache, dtype)
    if n_tokens < 0:
        raise ValueError(f"n_tokens must not be negative, got {n_tokens}")
    shape = (n_tokens, cache.k.shape[1], cache.k.shape[3])
    if out is None:
        out = tuple(torch.empty(shape, dtype=dtype, device=cache.k.device) for _ in "kv")
    k, v = out
    assert tuple(k.shape) == shape and k.dtype == dtype, "out holds k and v, [n_tokens, H_kv, D] each"
    _check_kv(cache, k, v)
    c, s, alive = _step(cache, block_table, cu_seqlens, seqlens, n_tokens)
    if n_tokens:
        k_, v_ = _rows(k), _rows(v)
        with torch.cuda.device(k.device):
            _lib.cache_read(c, s, k_, v_, torch.cuda.current_stream(k.device).cuda_stream)
        for t, t_ in ((k, k_), (v, v_)):
            if t_ is not t:
                t.copy_(t_)
    return k, v


def attention_paged(q, cache, block_table, cu_seqlens, seqlens, *, causal=True, window=None, sinks=0, shared=None,
                    sm_scale=None, return_lse=False, out=None):
    """Attention of the new tokens q [T, H_q, D] over all their sequences' tokens in the cache.

    block_table, cu_seqlens and seqlens as in cache_write, which has put the new tokens' own k and v there; one
    new token per sequence is a decoding step, a part of a prompt a chunk, and both may be in one call. q is of the
    cache's type, or fp16 or bf16 with an e4m3 cache. causal: the sequence's last new token sees all of its tokens,
    the one before it all but the last. A row that sees no key gets 0, and a log-sum-exp of -inf; rows past the last
    sequence are left as they are in out (undefined in a new one). A sequence of more tokens than its row of the
    table holds counts as one of as many. A page outside the cache makes the rows that see its tokens NaN, and may
    make other rows of its sequence NaN.
    window: (with causal) a row whose last key is n sees the `window` newest, n - window + 1 .. n, and the sequence's first
        `sinks`; entries of the table whose pages no row sees are not looked at, and their pages may be others' by now.
    shared: int32 [1] on the GPU, a number of tokens that all sequences begin with and that lie in the same pages: those are
        read once for the whole batch, from the table's row of the first sequence that has new tokens. As many count as
        whole pages hold and as lie before every sequence's new tokens. Not with a window. It pays for long prefixes and few
        new tokens a sequence; rows of hundreds share their sequence's keys as it is, and are faster without it. The workspace
        holds every row's results twice in float, beside the pieces of cut row tiles.
    return_lse: also return the natural-log log-sum-exp of every row's scaled scores, fp32 [H_q, T].
    out: of q's shape and type, in any layout without shared elements; q itself is allowed, and no other memory that
        the call reads.
    """
    if _lib.native is not None:  # the common call, made natively; None: not one of those
        result = _lib.native.attn_paged(*cache, block_table, cu_seqlens, seqlens, q, causal, sm_scale, return_lse, out,
                                        window, sinks, shared)
        if result is not None:
            return result if out is None else (out, result[1]) if return_lse else out
    assert q.dim() == 3
    T, H_q, D = q.shape
    _check_cache(cache, q.dtype)
    H_kv = cache.k.shape[1]
    assert D == cache.k.shape[3], "q and the cache are of one head_dim"
    assert H_kv > 0 and H_q % H_kv == 0, "GQA needs H_q divisible by H_kv"
    if q.device != cache.k.device:
        raise RuntimeError(f"q must be on {cache.k.device}, got {q.device}")
    qk_scale = _scale(sm_scale, D)
    window, sinks = _window(window, sinks, causal)
    if shared is not None:
        if window is not None:
            raise ValueError("a shared prefix and a window exclude each other")
        assert shared.dtype == torch.int32 and shared.numel() == 1, "shared is int32 [1]"
        if shared.device != q.device:
            raise RuntimeError(f"shared must be on {q.device}, got {shared.device}")
    out, o_ = _output(q, out)
    lse = torch.empty((H_q, T), dtype=torch.float32, device=q.device) if return_lse else None
    c, s, alive = _step(cache, block_table, cu_seqlens, seqlens, T)
    if out.numel():
        sizes = (H_q, H_kv, D, cache.k.dtype, T, seqlens.numel(), block_table.shape[1] * cache.k.shape[2])
        cus = _cu_count(q.device)
        if shared is not None:
            n = _lib.paged_shared_workspace_bytes(H_q, H_kv, D, T, seqlens.numel(), cus)
        elif window is not None:
            n = _lib.paged_window_workspace_bytes(*sizes, window, sinks, cus)
        else:
            n = _lib.paged_workspace_bytes(*sizes, cus)
        ws = torch.empty(n, dtype=torch.uint8, device=q.device) if n else None
        with torch.cuda.device(q.device):
            stream = torch.cuda.current_stream(q.device).cuda_stream
            if shared is not None and seqlens.numel():
                _lib.attn_paged_shared(_rows(q), o_, c, s, shared, causal, qk_scale, lse, ws, stream)
            elif window is not None:
                _lib.attn_paged_window(_rows(q), o_, c, s, window, sinks, qk_scale, lse, ws, stream)
            else:
                _lib.attn_paged(_rows(q), o_, c, s, causal, qk_scale, lse, ws, stream)
        if o_ is not out:
            out.copy_(o_)
    return (out, lse) if return_lse else out
