"""ctypes binding of libfa2_fwd.so, the C ABI declared in include/fa2_fwd.h.

The library is built in-tree by triton-fa2-forward_amd/csrc/build.py and sits next to this
file. torch is imported first so that its HIP runtime (SONAME libamdhip64.so.7) is the one
already loaded when the library is opened: the library then launches on exactly the streams
torch hands out.
"""

import ctypes
import os
import sys

import torch  # noqa: F401  (must be loaded before the HIP library, see above)

LIB_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "libfa2_fwd.so")

# C-ABI symbols declared in include/fa2_fwd.h, with (restype, argtypes).
_i32, _i64, _i64p, _vp = ctypes.c_int32, ctypes.c_int64, ctypes.POINTER(ctypes.c_int64), ctypes.c_void_p
_i64x3 = ctypes.c_int64 * 3


class Cache(ctypes.Structure):
    """fa2_cache"""
    _fields_ = [("k", _vp), ("v", _vp), ("k_scale", _vp), ("v_scale", _vp), ("k_stride", _i64x3),
                ("v_stride", _i64x3), ("k_scale_stride", _i64x3), ("v_scale_stride", _i64x3), ("n_pages", _i32),
                ("h_kv", _i32), ("page_size", _i32), ("head_dim", _i32), ("cache_dtype", _i32)]


class Sequences(ctypes.Structure):
    """fa2_sequences"""
    _fields_ = [("cu", _vp), ("lens", _vp), ("table", _vp), ("table_stride", ctypes.c_int64), ("n_seq", _i32),
                ("n_tokens", _i32), ("max_pages", _i32)]


class Rotation(ctypes.Structure):
    """fa2_rotation"""
    _fields_ = [("freqs", _vp), ("half", _i32), ("interleaved", _i32), ("scale", ctypes.c_double)]


class Turn(ctypes.Structure):
    """fa2_turn"""
    _fields_ = [("rotation", Rotation), ("axes", _vp), ("q_weight", _vp), ("k_weight", _vp), ("q_eps", ctypes.c_double),
                ("k_eps", ctypes.c_double), ("n_axes", _i32)]


_cachep, _seqp, _rotp, _turnp = (ctypes.POINTER(t) for t in (Cache, Sequences, Rotation, Turn))
SIGNATURES = {
    "fa2_attn_fwd": (ctypes.c_int, [_vp, _vp, _vp, _vp, _i64p, _i64p, _i64p, _i64p,
                                    _i32, _i32, _i32, _i32, _i32, _i32, _i32, _i32, _i32,
                                    _i32, _i32, ctypes.c_float, _vp]),
    "fa2_attn_fwd_ex": (ctypes.c_int, [_vp, _vp, _vp, _vp, _i64p, _i64p, _i64p, _i64p,
                                       _i32, _i32, _i32, _i32, _i32, _i32, _i32, _i32, _i32,
                                       _i32, _i32, ctypes.c_float, _vp, _i32, _vp,
                                       ctypes.c_size_t, _vp]),
    "fa2_attn_fwd_noalloc": (ctypes.c_int, [_vp, _vp, _vp, _vp, _i64p, _i64p, _i64p, _i64p,
                                            _i32, _i32, _i32, _i32, _i32, _i32, _i32, _i32, _i32,
                                            _i32, _i32, ctypes.c_float, _vp, _i32, _vp]),
    "fa2_workspace_bytes": (ctypes.c_size_t, [_i32, _i32, _i32, _i32, _i32]),
    "fa2_workspace_bytes_for": (ctypes.c_size_t, [_i32, _i32, _i32, _i32, _i32, _i32, _i32,
                                                  _i32, _i32]),
    "fa2_num_splits": (_i32, [_i32, _i32, _i32, _i32, _i32, _i32, _i32, _i32, _i32, _i32]),
    "fa2_launch_splits": (_i32, [_i32] * 11),
    "fa2_default_config": (ctypes.c_int, [_i32, ctypes.POINTER(_i32), ctypes.POINTER(_i32),
                                          ctypes.POINTER(_i32), ctypes.POINTER(_i32)]),
    "fa2_should_pack_gqa": (ctypes.c_int, [_i32, _i32, _i32]),
    "fa2_rotary": (ctypes.c_int, [_vp, _vp, _i64p, _i64p, _vp, _i32, _i64p, _rotp, _i32, _i32, _i32, _i32, _i32,
                                  _vp]),
    "fa2_cache_write": (ctypes.c_int, [_cachep, _seqp, _vp, _vp, _i64p, _i64p, _vp, _vp, _i64p, _i64p, _i32, _rotp,
                                       _i32, _vp]),
    "fa2_cache_read": (ctypes.c_int, [_cachep, _seqp, _vp, _vp, _i64p, _i64p, _i32, _vp]),
    "fa2_attn_packed": (ctypes.c_int, [_vp, _vp, _vp, _vp, _i64p, _i64p, _i64p, _i64p, _vp, _vp, _i32, _i32, _i32,
                                       _i32, _i32, _i32, _i32, _i32, ctypes.c_float, _vp, _vp]),
    "fa2_attn_paged": (ctypes.c_int, [_vp, _vp, _i64p, _i64p, _cachep, _seqp, _i32, _i32, _i32, ctypes.c_float,
                                      _vp, _vp, ctypes.c_size_t, _vp]),
    "fa2_paged_workspace_bytes": (ctypes.c_size_t, [_i32] * 6 + [_i64, _i32]),
    "fa2_attn_packed_window": (ctypes.c_int, [_vp, _vp, _vp, _vp, _i64p, _i64p, _i64p, _i64p, _vp, _vp, _i32, _i32, _i32,
                                              _i32, _i32, _i32, _i32, _i32, _i32, ctypes.c_float, _vp, _vp]),
    "fa2_attn_paged_window": (ctypes.c_int, [_vp, _vp, _i64p, _i64p, _cachep, _seqp, _i32, _i32, _i32, _i32, ctypes.c_float,
                                             _vp, _vp, ctypes.c_size_t, _vp]),
    "fa2_paged_window_workspace_bytes": (ctypes.c_size_t, [_i32] * 6 + [_i64, _i32, _i32, _i32]),
    "fa2_attn_paged_shared": (ctypes.c_int, [_vp, _vp, _i64p, _i64p, _cachep, _seqp, _vp, _i32, _i32, _i32, ctypes.c_float,
                                             _vp, _vp, ctypes.c_size_t, _vp]),
    "fa2_paged_shared_workspace_bytes": (ctypes.c_size_t, [_i32] * 6),
    "fa2_rotary_qk": (ctypes.c_int, [_vp] * 4 + [_i64p] * 4 + [_vp, _i32, _i64p, _turnp] + [_i32] * 6 + [_vp]),
    "fa2_cache_write_turned": (ctypes.c_int, [_cachep, _seqp, _vp, _vp, _i64p, _i64p, _vp, _vp, _i64p, _i64p, _i32, _vp,
                                              _i32, _i64p, _turnp, _i32, _vp]),
    "fa2_pages_extend": (ctypes.c_int, [_vp, _i32, _vp, _vp, _vp, _i64, _i32, _i32, _i32] + [_vp] * 6 + [_i32, _vp]),
    "fa2_pages_release": (ctypes.c_int, [_vp, _i32, _vp, _vp, _vp, _i64, _i32, _i32, _vp, _vp, _vp, _vp]),
    "fa2_last_error": (ctypes.c_char_p, []),
    "fa2_version": (ctypes.c_char_p, []),
}

DTYPE_CODE = {torch.float16: 0, torch.bfloat16: 1}
CACHE_DTYPE_CODE = {**DTYPE_CODE, torch.float8_e4m3fn: 2}

_LIB = None


def lib():
    """The loaded library. Raises RuntimeError when it has not been built."""
    global _LIB
    if _LIB is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(
                f"{LIB_PATH} is missing; build the HIP library first: "
                "python triton-fa2-forward_amd/csrc/build.py")
        handle = ctypes.CDLL(LIB_PATH)
        for name, (restype, argtypes) in SIGNATURES.items():
            fn = getattr(handle, name)
            fn.restype = restype
            fn.argtypes = argtypes
        _LIB = handle
    return _LIB


def build_id():
    """The torch and the Python that the native call must have been built for: it reads tensors by
    their C++ layout, which another build of either can change without a missing symbol."""
    return "torch {} {} python {}.{}".format(torch.__version__, torch.version.git_version,
                                             *sys.version_info[:2])


def _load_native():
    """The native common calls (csrc/fa2_torch.cpp), built beside the library; None where they are missing
    or were built for another torch or Python: the Python functions then make every call themselves, through
    ctypes."""
    try:
        from . import _torch_call
    except ImportError:
        return None
    return _torch_call if getattr(_torch_call, "built_for", None) == build_id() else None


native = _load_native()  # the serving operators' (fa2.rotary, fa2.packed, fa2.paged)


def _load_fast_call():
    """attention()'s native common call, or None."""
    module = _load_native()
    return None if module is None else module.call


fast_call = _load_fast_call()


def last_error():
    return lib().fa2_last_error().decode(errors="replace")


_STRIDES = {}


def _strides(t):
    """The element strides as the C array the ABI takes (four; the entry points of packed rows and of the
    cache read the first two or three). The stride of a size-1 dimension never
    enters an address; pass 0 so that only the strides the kernel actually steps by are checked
    against the 16-byte rule. The arrays are cached per (shape, strides): the library only reads
    them during the call, and building one costs more than the rest of a small call."""
    key = (t.shape, t.stride())
    arr = _STRIDES.get(key)
    if arr is None:
        if len(_STRIDES) >= 1024:
            _STRIDES.clear()
        arr = (ctypes.c_int64 * 4)(*(0 if n == 1 else s for n, s in zip(key[0], key[1])))
        _STRIDES[key] = arr
    return arr


def attn_fwd(q, k, v, out, causal, pack, block_m, block_n, qk_scale, stream):
    """Call fa2_attn_fwd on tensors that already satisfy the C contract."""
    B, H_q, N_q, D = q.shape
    H_kv, N_kv = k.shape[1], k.shape[2]
    rc = lib().fa2_attn_fwd(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
        _strides(q), _strides(k), _strides(v), _strides(out),
        B, H_q, H_kv, N_q, N_kv, D, DTYPE_CODE[q.dtype], int(bool(causal)), pack,
        block_m, block_n, qk_scale, stream)
    if rc != 0:
        raise RuntimeError(f"fa2_attn_fwd failed ({rc}): {last_error()}")


def attn_fwd_ex(q, k, v, out, causal, pack, block_m, block_n, qk_scale, lse, num_splits,
                workspace, stream):
    """Call fa2_attn_fwd_ex: lse (fp32 [B, H_q, N_q]) and workspace (uint8) may be None."""
    B, H_q, N_q, D = q.shape
    H_kv, N_kv = k.shape[1], k.shape[2]
    rc = lib().fa2_attn_fwd_ex(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
        _strides(q), _strides(k), _strides(v), _strides(out),
        B, H_q, H_kv, N_q, N_kv, D, DTYPE_CODE[q.dtype], int(bool(causal)), pack,
        block_m, block_n, qk_scale, None if lse is None else lse.data_ptr(), num_splits,
        None if workspace is None else workspace.data_ptr(),
        0 if workspace is None else workspace.numel(), stream)
    if rc != 0:
        raise RuntimeError(f"fa2_attn_fwd_ex failed ({rc}): {last_error()}")


def attn_fwd_noalloc(q, k, v, out, causal, pack, block_m, block_n, qk_scale, lse, num_splits,
                     stream):
    """Call fa2_attn_fwd_noalloc: fa2_attn_fwd_ex with the library's own scratch as the
    workspace (no allocation anywhere); lse (fp32 [B, H_q, N_q]) may be None."""
    B, H_q, N_q, D = q.shape
    H_kv, N_kv = k.shape[1], k.shape[2]
    rc = lib().fa2_attn_fwd_noalloc(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
        _strides(q), _strides(k), _strides(v), _strides(out),
        B, H_q, H_kv, N_q, N_kv, D, DTYPE_CODE[q.dtype], int(bool(causal)), pack,
        block_m, block_n, qk_scale, None if lse is None else lse.data_ptr(), num_splits, stream)
    if rc != 0:
        raise RuntimeError(f"fa2_attn_fwd_noalloc failed ({rc}): {last_error()}")


def workspace_bytes(B, H_q, N_q, D, num_splits):
    return int(lib().fa2_workspace_bytes(B, H_q, N_q, D, num_splits))


_WS_FOR = {}


def workspace_bytes_for(B, H_q, H_kv, N_q, N_kv, D, dtype, causal, num_splits):
    """fa2_workspace_bytes_for, cached per shape (it is host policy, a pure function)."""
    key = (B, H_q, H_kv, N_q, N_kv, D, dtype, bool(causal), num_splits)
    n = _WS_FOR.get(key)
    if n is None:
        if len(_WS_FOR) >= 1024:
            _WS_FOR.clear()
        n = int(lib().fa2_workspace_bytes_for(B, H_q, H_kv, N_q, N_kv, D, DTYPE_CODE[dtype],
                                              int(bool(causal)), num_splits))
        _WS_FOR[key] = n
    return n


def num_splits(B, H_q, H_kv, N_q, N_kv, D, causal, block_m, block_n, num_cus):
    return int(lib().fa2_num_splits(B, H_q, H_kv, N_q, N_kv, D, int(bool(causal)), block_m,
                                    block_n, num_cus))


# ---- serving: packed sequences, the paged cache, rotary positions

def _ptr(t):
    return None if t is None else t.data_ptr()


def _int32(**sizes):
    """Sizes as the C ABI takes them: a larger one would lose its upper bits on the way there."""
    for name, n in sizes.items():
        if not 0 <= n < 1 << 31:
            raise ValueError(f"{name} must be below 2^31, got {n}")


def _checked(rc, name):
    if rc != 0:
        raise RuntimeError(f"{name} failed ({rc}): {last_error()}")


def cache_of(cache):
    """The C description of a fa2.paged.KVCache that satisfies its checks."""
    pages, h_kv, page_size, head_dim = cache.k.shape
    _int32(pages=pages, H_kv=h_kv, page_size=page_size)

    def strides(t):
        return _i64x3(*([0] * 3 if t is None else (0 if n == 1 else s for n, s in zip(t.shape[:3], t.stride()))))

    return Cache(_ptr(cache.k), _ptr(cache.v), _ptr(cache.k_scale), _ptr(cache.v_scale), strides(cache.k),
                 strides(cache.v), strides(cache.k_scale), strides(cache.v_scale), pages, h_kv, page_size,
                 head_dim, CACHE_DTYPE_CODE[cache.k.dtype])


def sequences_of(cu, lens, table, n_tokens):
    """The C description of sequences over a cache (dense int32 tensors; table rows any distance apart)."""
    _int32(sequences=lens.numel(), tokens=n_tokens, table_columns=table.shape[1])
    return Sequences(_ptr(cu), _ptr(lens), _ptr(table), 0 if table.shape[0] == 1 else table.stride(0),
                     lens.numel(), n_tokens, table.shape[1])


def rotary(x, out, positions, rotation, stream):
    """Call fa2_rotary on [B, H, N, D] tensors and positions [B, N]."""
    B, H, N, D = x.shape
    _int32(B=B, H=H, N=N)
    _checked(lib().fa2_rotary(x.data_ptr(), out.data_ptr(), _strides(x), _strides(out), positions.data_ptr(),
                              positions.element_size(), (ctypes.c_int64 * 2)(*positions.stride()),
                              ctypes.byref(rotation), B, H, N, D, DTYPE_CODE[x.dtype], stream), "fa2_rotary")


def cache_write(cache, seq, k, v, q, q_out, rotation, stream):
    """Call fa2_cache_write; q, q_out and rotation may be None."""
    _int32(H_q=0 if q is None else q.shape[1])
    _checked(lib().fa2_cache_write(
        ctypes.byref(cache), ctypes.byref(seq), k.data_ptr(), v.data_ptr(), _strides(k), _strides(v), _ptr(q),
        _ptr(q_out), None if q is None else _strides(q), None if q is None else _strides(q_out),
        0 if q is None else q.shape[1], None if rotation is None else ctypes.byref(rotation), DTYPE_CODE[k.dtype],
        stream), "fa2_cache_write")


def cache_read(cache, seq, k, v, stream):
    """Call fa2_cache_read."""
    _checked(lib().fa2_cache_read(ctypes.byref(cache), ctypes.byref(seq), k.data_ptr(), v.data_ptr(), _strides(k),
                                  _strides(v), DTYPE_CODE[k.dtype], stream), "fa2_cache_read")


def attn_packed(q, k, v, out, cu, cu_kv, causal, qk_scale, lse, stream):
    """Call fa2_attn_packed; cu_kv and lse may be None."""
    T, H_q, D = q.shape
    _int32(T=T, H_q=H_q, T_kv=k.shape[0], H_kv=k.shape[1], sequences=cu.numel() - 1)
    _checked(lib().fa2_attn_packed(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), _strides(q), _strides(k), _strides(v),
        _strides(out), cu.data_ptr(), _ptr(cu_kv), cu.numel() - 1, T, k.shape[0], H_q, k.shape[1], D,
        DTYPE_CODE[q.dtype], int(bool(causal)), qk_scale, _ptr(lse), stream), "fa2_attn_packed")


def paged_workspace_bytes(H_q, H_kv, D, cache_dtype, n_tokens, n_seq, max_keys, num_cus):
    return int(lib().fa2_paged_workspace_bytes(H_q, H_kv, D, CACHE_DTYPE_CODE[cache_dtype], n_tokens, n_seq, max_keys,
                                               num_cus))


def attn_paged(q, out, cache, seq, causal, qk_scale, lse, workspace, stream):
    """Call fa2_attn_paged; lse and workspace (uint8) may be None."""
    _int32(H_q=q.shape[1])
    _checked(lib().fa2_attn_paged(q.data_ptr(), out.data_ptr(), _strides(q), _strides(out), ctypes.byref(cache),
                                  ctypes.byref(seq), q.shape[1], DTYPE_CODE[q.dtype], int(bool(causal)), qk_scale,
                                  _ptr(lse), _ptr(workspace), 0 if workspace is None else workspace.numel(), stream),
             "fa2_attn_paged")


# ---- a step beyond that: windows, a common prefix, normalised rotations of several axes, pages

def turn_of(plan, freqs, axes, n_axes, q_norm, k_norm):
    """The C description of a fa2.rotary.Rotary and the heads' norms (checked; None: no norm)."""
    q_weight, q_eps = (None, 0.0) if q_norm is None else q_norm
    k_weight, k_eps = (None, 0.0) if k_norm is None else k_norm
    return Turn(Rotation(freqs.data_ptr(), freqs.numel(), plan.interleaved, plan.scale), _ptr(axes), _ptr(q_weight),
                _ptr(k_weight), q_eps, k_eps, n_axes)


def rotary_qk(q, k, q_out, k_out, positions, turn, stream):
    """Call fa2_rotary_qk on [B, H, N, D] tensors (k and k_out may be None) and positions [axes, B, N]."""
    B, H, N, D = q.shape
    H_k = 0 if k is None else k.shape[1]
    _int32(B=B, H_q=H, H_k=H_k, N=N)
    none = (ctypes.c_int64 * 4)()
    _checked(lib().fa2_rotary_qk(
        q.data_ptr(), _ptr(k), q_out.data_ptr(), _ptr(k_out), _strides(q), none if k is None else _strides(k),
        _strides(q_out), none if k is None else _strides(k_out), positions.data_ptr(), positions.element_size(),
        (ctypes.c_int64 * 3)(*positions.stride()), ctypes.byref(turn), B, H, H_k, N, D, DTYPE_CODE[q.dtype], stream),
        "fa2_rotary_qk")


def cache_write_turned(cache, seq, k, v, q, q_out, positions, turn, stream):
    """Call fa2_cache_write_turned; q and q_out, and positions [axes, T], may be None."""
    _int32(H_q=0 if q is None else q.shape[1])
    _checked(lib().fa2_cache_write_turned(
        ctypes.byref(cache), ctypes.byref(seq), k.data_ptr(), v.data_ptr(), _strides(k), _strides(v), _ptr(q), _ptr(q_out),
        None if q is None else _strides(q), None if q is None else _strides(q_out), 0 if q is None else q.shape[1],
        _ptr(positions), 0 if positions is None else positions.element_size(),
        None if positions is None else (ctypes.c_int64 * 2)(*positions.stride()), ctypes.byref(turn), DTYPE_CODE[k.dtype],
        stream), "fa2_cache_write_turned")


def attn_packed_window(q, k, v, out, cu, cu_kv, window, sinks, qk_scale, lse, stream):
    """Call fa2_attn_packed_window; cu_kv and lse may be None."""
    T, H_q, D = q.shape
    _int32(T=T, H_q=H_q, T_kv=k.shape[0], H_kv=k.shape[1], sequences=cu.numel() - 1)
    _checked(lib().fa2_attn_packed_window(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), _strides(q), _strides(k), _strides(v),
        _strides(out), cu.data_ptr(), _ptr(cu_kv), cu.numel() - 1, T, k.shape[0], H_q, k.shape[1], D,
        DTYPE_CODE[q.dtype], window, sinks, qk_scale, _ptr(lse), stream), "fa2_attn_packed_window")


def paged_window_workspace_bytes(H_q, H_kv, D, cache_dtype, n_tokens, n_seq, max_keys, window, sinks, num_cus):
    return int(lib().fa2_paged_window_workspace_bytes(H_q, H_kv, D, CACHE_DTYPE_CODE[cache_dtype], n_tokens, n_seq, max_keys,
                                                      window, sinks, num_cus))


def attn_paged_window(q, out, cache, seq, window, sinks, qk_scale, lse, workspace, stream):
    """Call fa2_attn_paged_window; lse and workspace (uint8) may be None."""
    _int32(H_q=q.shape[1])
    _checked(lib().fa2_attn_paged_window(
        q.data_ptr(), out.data_ptr(), _strides(q), _strides(out), ctypes.byref(cache), ctypes.byref(seq), q.shape[1],
        DTYPE_CODE[q.dtype], window, sinks, qk_scale, _ptr(lse), _ptr(workspace),
        0 if workspace is None else workspace.numel(), stream), "fa2_attn_paged_window")


def paged_shared_workspace_bytes(H_q, H_kv, D, n_tokens, n_seq, num_cus):
    return int(lib().fa2_paged_shared_workspace_bytes(H_q, H_kv, D, n_tokens, n_seq, num_cus))


def attn_paged_shared(q, out, cache, seq, shared, causal, qk_scale, lse, workspace, stream):
    """Call fa2_attn_paged_shared; lse may be None."""
    _int32(H_q=q.shape[1])
    _checked(lib().fa2_attn_paged_shared(
        q.data_ptr(), out.data_ptr(), _strides(q), _strides(out), ctypes.byref(cache), ctypes.byref(seq), shared.data_ptr(),
        q.shape[1], DTYPE_CODE[q.dtype], int(bool(causal)), qk_scale, _ptr(lse), _ptr(workspace), workspace.numel(), stream),
        "fa2_attn_paged_shared")


def pages_extend(free, count, count_out, table, page_size, lens, new_tokens, lens_out, cu_out, positions, slots, stream):
    """Call fa2_pages_extend on int32 tensors (slots int64) that satisfy fa2.pages' checks."""
    S, P = table.shape
    _int32(pages=free.numel(), sequences=S, table_columns=P, page_size=page_size, n_tokens=slots.numel())
    _checked(lib().fa2_pages_extend(
        free.data_ptr(), free.numel(), count.data_ptr(), count_out.data_ptr(), table.data_ptr(), 0 if S == 1 else table.stride(0),
        S, P, page_size, lens.data_ptr(), new_tokens.data_ptr(), lens_out.data_ptr(), cu_out.data_ptr(), positions.data_ptr(),
        slots.data_ptr(), slots.numel(), stream), "fa2_pages_extend")


def pages_release(free, count, count_out, table, first, last, workspace, stream):
    """Call fa2_pages_release on int32 tensors that satisfy fa2.pages' checks."""
    S, P = table.shape
    _int32(pages=free.numel(), sequences=S, table_columns=P)
    _checked(lib().fa2_pages_release(
        free.data_ptr(), free.numel(), count.data_ptr(), count_out.data_ptr(), table.data_ptr(), 0 if S == 1 else table.stride(0),
        S, P, first.data_ptr(), last.data_ptr(), workspace.data_ptr(), stream), "fa2_pages_release")
