"""Attention over packed sequences on AMD MI355X (gfx950): attention() for sequences of different lengths in
one call, without padding.

The rows of all sequences lie back to back in [tokens, heads, head_dim] tensors; cu_seqlens says where each
starts. The arithmetic runs in the HIP kernels of csrc/attn_ragged.hpp behind fa2_attn_packed of
include/fa2_fwd.h. Lengths are read on the device: no copy to the host, and a captured graph follows the
lengths that its tensors hold at each replay.
"""

import math
import operator

import torch

from . import _lib
from .kernel import _MAX_KV_ROW_STRIDE, LOG2E

_MOST = (1 << 31) - 1  # more tokens than any sequence has


def _rows(t, max_row_stride=None):
    """t [tokens, heads, head_dim] itself if the kernels' 16-byte loads can address it, else a dense copy
    (fa2.kernel._loadable for packed rows)."""
    ok = t.data_ptr() % 16 == 0 and (t.is_contiguous() or (
        t.stride(-1) == 1 and all(n == 1 or s % 8 == 0 for n, s in zip(t.shape[:2], t.stride()[:2]))
        and (max_row_stride is None or t.shape[0] == 1 or t.stride(0) <= max_row_stride)))
    return t if ok else t.clone(memory_format=torch.contiguous_format)


def _index(t, name, device):
    """An int32 index vector of the call, dense."""
    assert t.dim() == 1 and t.dtype == torch.int32, f"{name} is an int32 vector"
    if t.device != device:
        raise RuntimeError(f"{name} must be on {device}, got {t.device}")
    return t.contiguous()


def _scale(sm_scale, head_dim):
    if sm_scale is None:
        sm_scale = 1.0 / math.sqrt(head_dim)
    if not sm_scale > 0:
        raise ValueError(f"sm_scale must be positive (the row max is scaled after it is taken), got {sm_scale}")
    return sm_scale * LOG2E


def _window(window, sinks, causal):
    """(window, sinks) of a call as the C ABI takes them; (None, 0): all keys."""
    if window is None:
        if sinks:
            raise ValueError("sinks are the tokens that stay visible beside a window")
        return None, 0
    window, sinks = operator.index(window), operator.index(sinks)
    if window < 1 or sinks < 0:
        raise ValueError(f"window must be positive and sinks not negative, got {window} and {sinks}")
    if not causal:
        raise ValueError("a window needs the causal mask")
    return min(window, _MOST), min(sinks, _MOST)


def _output(q, out):
    """(the caller's out, the tensor the kernel writes): the same, or a copy that holds out's rows where the
    kernel cannot address out."""
    if out is None:
        out = torch.empty_like(q)
    assert out.shape == q.shape and out.dtype == q.dtype, "out must be of q's shape and type"
    if out.device != q.device:
        raise RuntimeError(f"out must be on {q.device}, got {out.device}")
    return out, _rows(out)


def attention_packed(q, k, v, cu_seqlens, cu_seqlens_kv=None, *, causal=True, window=None, sinks=0, sm_scale=None,
                     return_lse=False, out=None):
    """softmax(Q K^T * sm_scale [+ causal mask]) V within each of the packed sequences.

    q: [T, H_q, D]; k, v: [T_kv, H_kv, D], fp16 or bf16, D in (16, 32, 64, 128), H_q % H_kv == 0; returns out
    [T, H_q, D], laid out like q.
    cu_seqlens: int32 [S + 1] on the GPU, ascending: sequence s owns rows cu_seqlens[s] .. cu_seqlens[s + 1] - 1 of
        q, and of k and v unless cu_seqlens_kv gives theirs. Rows of no sequence are left as they are in
        out (undefined in a new one).
    causal: row i of a sequence sees its keys up to i + n_kv - n_q (with one cu_seqlens: up to its own).
        A row that sees no key gets 0, and a log-sum-exp of -inf.
    window: (with causal) a row whose last key is n sees the `window` newest, n - window + 1 .. n, and the sequence's first
        `sinks`; keys that no row sees are not read.
    return_lse: also return the natural-log log-sum-exp of every row's scaled scores, fp32 [H_q, T].
    out: of q's shape and type, in any layout without shared elements; q itself is allowed, and no other memory that
        the call reads.
    """
    if _lib.native is not None:  # the common call, made natively; None: not one of those
        result = _lib.native.attn_packed(q, k, v, cu_seqlens, cu_seqlens_kv, causal, sm_scale, return_lse, out, window, sinks)
        if result is not None:
            return result if out is None else (out, result[1]) if return_lse else out
    assert q.dim() == k.dim() == v.dim() == 3
    T, H_q, D = q.shape
    T_kv, H_kv, Dk = k.shape
    assert v.shape == k.shape and Dk == D
    assert q.dtype == k.dtype == v.dtype and q.dtype in (torch.float16, torch.bfloat16)
    assert H_kv > 0 and H_q % H_kv == 0, "GQA needs H_q divisible by H_kv"
    assert D in (16, 32, 64, 128), "head_dim must be a power of two in [16, 128]"
    assert cu_seqlens.numel() >= 1, "cu_seqlens holds S + 1 entries"
    if cu_seqlens_kv is None:
        assert T_kv == T, "k and v of another length than q need cu_seqlens_kv"
    else:
        assert cu_seqlens_kv.shape == cu_seqlens.shape, "cu_seqlens_kv holds as many entries as cu_seqlens"
    qk_scale = _scale(sm_scale, D)
    window, sinks = _window(window, sinks, causal)
    if not (q.is_cuda and k.is_cuda and v.is_cuda):
        raise RuntimeError("fa2.packed.attention_packed runs on the GPU (gfx950 HIP kernel); got CPU tensors")
    if not q.device == k.device == v.device:
        raise RuntimeError(f"q, k, v must be on one device, got {q.device}, {k.device}, {v.device}")
    cu = _index(cu_seqlens, "cu_seqlens", q.device)
    cu_kv = None if cu_seqlens_kv is None else _index(cu_seqlens_kv, "cu_seqlens_kv", q.device)
    out, o_ = _output(q, out)
    lse = torch.empty((H_q, T), dtype=torch.float32, device=q.device) if return_lse else None
    if out.numel():
        tensors = (_rows(q), _rows(k, _MAX_KV_ROW_STRIDE), _rows(v, _MAX_KV_ROW_STRIDE), o_, cu, cu_kv)
        with torch.cuda.device(q.device):
            stream = torch.cuda.current_stream(q.device).cuda_stream
            if window is None:
                _lib.attn_packed(*tensors, causal, qk_scale, lse, stream)
            else:
                _lib.attn_packed_window(*tensors, window, sinks, qk_scale, lse, stream)
        if o_ is not out:
            out.copy_(o_)
    return (out, lse) if return_lse else out
