"""Rotary positions on AMD MI355X (gfx950): the rotation of queries and keys that comes before attention().

rotary() rotates the first values of every head, in pairs, by angles that grow with the token's position;
rotary_plan() makes the frequencies, plain or scaled for longer contexts than they were trained for. The
arithmetic runs in one HIP kernel (csrc/serve_cache.hip) behind fa2_rotary of include/fa2_fwd.h; angles are
formed in float64, so positions of a million tokens cost no accuracy. fa2.paged.cache_write rotates keys
and queries by the same plan on their way into a cache.

rotary_qk() makes queries and keys of a layer ready in one launch (csrc/serve_turn.hip): each head first divided by its
root mean square and weighted, if asked for, then rotated, by one position a token or, with a plan of several
axes, by a position of its own on each (time, height and width of images and video).
"""

import math
from typing import NamedTuple, Optional

import torch

from . import _lib
from .kernel import _loadable


class _Plan(NamedTuple):
    freqs: torch.Tensor
    interleaved: bool = False
    scale: float = 1.0


class _AxesPlan(NamedTuple):
    freqs: torch.Tensor
    interleaved: bool = False
    scale: float = 1.0
    axes: Optional[torch.Tensor] = None


class Rotary(_Plan):
    """Frequencies and form of a rotation, kept by the caller for every layer.

    freqs: float64 [rot_dim / 2] on the GPU, radians per position; rot_dim a multiple of 16, at most head_dim.
    interleaved: pairs (2 i, 2 i + 1) instead of (i, i + rot_dim / 2).
    scale: factor on the rotated values (scaled contexts).
    axes: int32 [rot_dim / 2] on the GPU, the axis by whose position each pair is rotated (below the number of axes of the
        positions it is used with; others count as the nearest). None: one position a token.

    A named tuple of the first three, and of all four (an AxesRotary) with axes.
    """
    __slots__ = ()
    axes = None

    def __new__(cls, freqs, interleaved=False, scale=1.0, axes=None):
        if axes is not None:
            return tuple.__new__(AxesRotary, (freqs, interleaved, scale, axes))
        return tuple.__new__(cls, (freqs, interleaved, scale))

    def _replace(self, *, axes=None, **values):
        return Rotary(*super()._replace(**values), axes)


class AxesRotary(_AxesPlan, Rotary):
    """A Rotary with axes."""
    __slots__ = ()


class HeadNorm(NamedTuple):
    """A norm of every head: x / sqrt(mean x^2 + eps) * weight. weight: float32 [head_dim] on the GPU, dense; eps positive."""
    weight: torch.Tensor
    eps: float = 1e-6


def rotary_plan(rot_dim, base=10000.0, *, scaling=None, factor=1.0, trained_length=None, fast=32.0, slow=1.0,
                interleaved=False, axes=None, device="cuda"):
    """The Rotary of base^(-2 i / rot_dim), i < rot_dim / 2, scaled for contexts `factor` times as long.

    scaling: None, or
      "linear"  every frequency divided by factor (positions interpolated);
      "base"    base * factor^(rot_dim / (rot_dim - 2)): the slowest pair turns as under "linear", the
                fastest keeps its frequency;
      "blend"   pairs that turn at least `fast` times within trained_length keep their frequency, those that turn at
                most `slow` times are divided by factor, between them the share goes linearly with the
                pair's index; values are scaled by 0.1 ln(factor) + 1 (YaRN, arXiv 2309.00071);
      "smooth"  as "blend", with the share linear in the number of turns and no scale of the values.
    axes: for positions of several axes, the axis of each of the rot_dim / 2 pairs: [0] * 16 + [1] * 24 + [2] * 24 gives
        time the fastest quarter and height and width equal blocks, [0, 1, 2] * 21 + [0] takes turns.
    """
    if rot_dim % 16 or rot_dim <= 0:
        raise ValueError(f"rot_dim must be a positive multiple of 16, got {rot_dim}")
    if not (base > 1 and factor > 0 and math.isfinite(base) and math.isfinite(factor)):
        raise ValueError(f"base must be above 1 and factor positive, got {base} and {factor}")
    if scaling not in (None, "linear", "base", "blend", "smooth"):
        raise ValueError(f'scaling must be None, "linear", "base", "blend" or "smooth", got {scaling!r}')
    if scaling == "base":
        base = base * factor ** (rot_dim / (rot_dim - 2))
    i = torch.arange(rot_dim // 2, dtype=torch.float64)
    freqs = float(base) ** (-2.0 * i / rot_dim)
    scale = 1.0
    if scaling == "linear":
        freqs = freqs / factor
    elif scaling in ("blend", "smooth"):
        if not trained_length or trained_length <= 0:
            raise ValueError(f'scaling "{scaling}" needs the trained_length of the frequencies')
        if not fast > slow > 0:
            raise ValueError(f"fast and slow must be fast > slow > 0, got {fast} and {slow}")
        if scaling == "blend":
            # the pair index at which a pair turns x times within trained_length
            def pair(x):
                return rot_dim * math.log(trained_length / (2 * math.pi * x)) / (2 * math.log(base))
            low, high = max(math.floor(pair(fast)), 0), min(math.ceil(pair(slow)), rot_dim - 1)
            keep = 1 - ((i - low) / max(high - low, 1e-3)).clamp(0, 1)
            scale = 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0
        else:
            turns = trained_length * freqs / (2 * math.pi)
            keep = ((turns - slow) / (fast - slow)).clamp(0, 1)
        freqs = freqs * keep + freqs / factor * (1 - keep)
    if axes is not None:
        axes = torch.as_tensor(axes)
        if axes.shape != freqs.shape or axes.is_floating_point() or bool((axes < 0).any()):
            raise ValueError(f"axes must name an axis for each of the {rot_dim // 2} pairs")
        axes = axes.to(device=device, dtype=torch.int32)
    return Rotary(freqs.to(device), interleaved, scale, axes)


def _check_plan(plan, head_dim, device):
    """The plan's frequencies as the kernels take them: float64, dense, on the tensors' device."""
    f = plan.freqs
    assert f.dim() == 1 and f.dtype == torch.float64, "a Rotary's freqs are float64 [rot_dim / 2]"
    rot = 2 * f.numel()
    if rot % 16 or not 0 < rot <= head_dim:
        raise ValueError(f"a rotation covers 16, 32, ... up to head_dim ({head_dim}) values, got {rot}")
    if not math.isfinite(plan.scale):
        raise ValueError(f"a Rotary's scale must be finite, got {plan.scale}")
    if f.device != device:
        raise RuntimeError(f"the Rotary's freqs must be on {device}, got {f.device}")
    return f.contiguous()


def _check_axes(plan, device):
    """The plan's axes as the kernels take them (None: one)."""
    if plan.axes is None:
        return None
    assert plan.axes.dim() == 1 and plan.axes.dtype == torch.int32 and plan.axes.numel() == plan.freqs.numel(), (
        "a Rotary's axes are int32 [rot_dim / 2]")
    if plan.axes.device != device:
        raise RuntimeError(f"the Rotary's axes must be on {device}, got {plan.axes.device}")
    return plan.axes.contiguous()


def _check_norm(norm, name, head_dim, device):
    """A HeadNorm as the kernels take it: (weight, eps), or None."""
    if norm is None:
        return None
    weight, eps = norm
    assert weight.dtype == torch.float32 and tuple(weight.shape) == (head_dim,), (
        f"{name}'s weight is float32 [head_dim]")
    if not (eps > 0 and math.isfinite(eps)):
        raise ValueError(f"{name}'s eps must be positive and finite, got {eps}")
    if weight.device != device:
        raise RuntimeError(f"{name}'s weight must be on {device}, got {weight.device}")
    return weight.contiguous(), float(eps)


def rotary(x, positions, plan, *, norm=None, out=None):
    """x with the first 2 * len(plan.freqs) values of every head rotated by its token's position.

    x: fp16 or bf16, [B, H, N, D] with positions [N] or [B, N], or packed [T, H, D] with positions [T];
    positions: int32 or int64; a plan with axes takes them of every axis, [axes, N], [axes, B, N] or [axes, T].
    norm: a HeadNorm, applied to every head first. Returns out, laid out like x; out=x works in place. A pair (a, b) at
    position p becomes scale * (a cos - b sin, b cos + a sin) of the angle p * freqs[i].
    """
    if norm is not None or plan.axes is not None:
        return rotary_qk(x, None, positions, plan, q_norm=norm, q_out=out)[0]
    if _lib.native is not None:  # the common call, made natively; None: not one of those
        result = _lib.native.rotary(x, positions, plan.freqs, plan.interleaved, plan.scale, out)
        if result is not None:
            return result if out is None else out
    assert x.dim() in (3, 4) and x.dtype in (torch.float16, torch.bfloat16)
    D = x.shape[-1]
    assert D in (16, 32, 64, 128), "head_dim must be a power of two in [16, 128]"
    assert positions.dtype in (torch.int32, torch.int64), "positions are int32 or int64"
    x4 = x if x.dim() == 4 else x.transpose(0, 1).unsqueeze(0)
    B, H, N, _ = x4.shape
    assert tuple(positions.shape) in ((N,), (B, N)) if x.dim() == 4 else tuple(positions.shape) == (N,), (
        "positions are one per token")
    if out is not None:
        assert out.shape == x.shape and out.dtype == x.dtype, "out must be of x's shape and type"
    if not (x.is_cuda and positions.is_cuda and (out is None or out.is_cuda)):
        raise RuntimeError("fa2.rotary.rotary runs on the GPU (gfx950 HIP kernel); got CPU tensors")
    if not x.device == positions.device == (x.device if out is None else out.device):
        raise RuntimeError(f"x, positions and out must be on one device, got {x.device} and {positions.device}")
    freqs = _check_plan(plan, D, x.device)
    if out is None:
        out = torch.empty_like(x)
    if x.numel() == 0:
        return out
    x_ = _loadable(x4)
    o4 = out if out.dim() == 4 else out.transpose(0, 1).unsqueeze(0)
    o_ = _loadable(o4)
    pos = positions.expand(B, N)
    with torch.cuda.device(x.device):
        _lib.rotary(x_, o_, pos, _lib.Rotation(freqs.data_ptr(), freqs.numel(), plan.interleaved, plan.scale),
                    torch.cuda.current_stream(x.device).cuda_stream)
    if o_ is not o4:
        o4.copy_(o_)
    return out


def _positions(positions, plan, B, N, packed):
    """positions as the kernels take them: [axes, B, N], strides of 0 where they repeat."""
    assert positions.dtype in (torch.int32, torch.int64), "positions are int32 or int64"
    if plan.axes is None:
        positions = positions[None]
    shapes = ((N,),) if packed else ((N,), (B, N))
    assert tuple(positions.shape[1:]) in shapes and positions.shape[0] > 0, (
        "positions are one per token, and with a plan's axes one per axis and token")
    if positions.dim() == 2:
        positions = positions[:, None]
    return positions.expand(positions.shape[0], B, N)


def rotary_qk(q, k, positions, plan, *, q_norm=None, k_norm=None, q_out=None, k_out=None):
    """(q, k) ready for attention: every head normalised (q_norm, k_norm: a HeadNorm, or None), then rotated as rotary()
    does, in one launch.

    q: fp16 or bf16 [B, H_q, N, D], k [B, H_k, N, D], or packed [T, H_q, D] and [T, H_k, D]; k may be None.
    positions as for rotary(). Returns (q_out, k_out), laid out like q and k; q_out=q and k_out=k work in place, and no other
    memory that the call reads may be written. Sums and products are held in 32 bits or more, and a value is rounded once.
    """
    if _lib.native is not None:  # the common call, made natively; None: not one of those
        result = _lib.native.rotary_qk(q, k, positions, plan.freqs, plan.interleaved, plan.scale, plan.axes,
                                       *(q_norm or (None, 0.0)), *(k_norm or (None, 0.0)), q_out, k_out)
        if result is not None:
            return result[0] if q_out is None else q_out, result[1] if k_out is None else k_out
    assert q.dim() in (3, 4) and q.dtype in (torch.float16, torch.bfloat16)
    D = q.shape[-1]
    assert D in (16, 32, 64, 128), "head_dim must be a power of two in [16, 128]"
    packed = q.dim() == 3

    def four(t):
        return t.transpose(0, 1).unsqueeze(0) if packed else t

    B, _, N, _ = four(q).shape
    if k is None:
        assert k_norm is None and k_out is None, "k_norm and k_out are k's"
    else:
        assert k.dim() == q.dim() and k.dtype == q.dtype and k.shape[-1] == D and four(k).shape[0] == B and (
            four(k).shape[2] == N), "q and k are of one type and of the same tokens and head_dim"
    for t, o in ((q, q_out), (k, k_out)):
        if o is not None:
            assert o.shape == t.shape and o.dtype == t.dtype, "out must be of its input's shape and type"
    tensors = [t for t in (q, k, positions, q_out, k_out) if t is not None]
    if not all(t.is_cuda for t in tensors):
        raise RuntimeError("fa2.rotary.rotary_qk runs on the GPU (gfx950 HIP kernel); got CPU tensors")
    if not all(t.device == q.device for t in tensors):
        raise RuntimeError(f"q, k, positions and the outputs must be on one device, got {[str(t.device) for t in tensors]}")
    freqs, axes = _check_plan(plan, D, q.device), _check_axes(plan, q.device)
    pos = _positions(positions, plan, B, N, packed)
    norms = _check_norm(q_norm, "q_norm", D, q.device), _check_norm(k_norm, "k_norm", D, q.device)
    q_out = torch.empty_like(q) if q_out is None else q_out
    if k is not None and k_out is None:
        k_out = torch.empty_like(k)
    if B * N == 0 or q.numel() + (0 if k is None else k.numel()) == 0:
        return q_out, k_out
    q4, k4 = (None if t is None else _loadable(four(t)) for t in (q, k))
    qo4, ko4 = (None if t is None else four(t) for t in (q_out, k_out))
    qo_, ko_ = (None if t is None else _loadable(t) for t in (qo4, ko4))
    turn = _lib.turn_of(plan, freqs, axes, pos.shape[0], *norms)
    with torch.cuda.device(q.device):
        _lib.rotary_qk(q4, k4, qo_, ko_, pos, turn, torch.cuda.current_stream(q.device).cuda_stream)
    for to, made in ((qo4, qo_), (ko4, ko_)):
        if made is not to:
            to.copy_(made)
    return q_out, k_out
