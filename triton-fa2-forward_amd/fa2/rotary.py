"""Rotary positions on AMD MI355X (gfx950): the rotation of queries and keys that comes before attention().

rotary() rotates the first values of every head, in pairs, by angles that grow with the token's position;
rotary_plan() makes the frequencies, plain or scaled for longer contexts than they were trained for. The
arithmetic runs in one HIP kernel (csrc/serve_cache.hip) behind fa2_rotary of include/fa2_fwd.h; angles are
formed in float64, so positions of a million tokens cost no accuracy. fa2.paged.cache_write rotates keys
and queries by the same plan on their way into a cache.
"""

import math
from typing import NamedTuple

import torch

from . import _lib
from .kernel import _loadable


class Rotary(NamedTuple):
    """Frequencies and form of a rotation, kept by the caller for every layer.

    freqs: float64 [rot_dim / 2] on the GPU, radians per position; rot_dim a multiple of 16, at most head_dim.
    interleaved: pairs (2 i, 2 i + 1) instead of (i, i + rot_dim / 2).
    scale: factor on the rotated values (scaled contexts).
    """
    freqs: torch.Tensor
    interleaved: bool = False
    scale: float = 1.0


def rotary_plan(rot_dim, base=10000.0, *, scaling=None, factor=1.0, trained_length=None, fast=32.0, slow=1.0,
                interleaved=False, device="cuda"):
    """The Rotary of base^(-2 i / rot_dim), i < rot_dim / 2, scaled for contexts `factor` times as long.

    scaling: None, or
      "linear"  every frequency divided by factor (positions interpolated);
      "base"    base * factor^(rot_dim / (rot_dim - 2)): the slowest pair turns as under "linear", the
                fastest keeps its frequency;
      "blend"   pairs that turn at least `fast` times within trained_length keep their frequency, those that turn at
                most `slow` times are divided by factor, between them the share goes linearly with the
                pair's index; values are scaled by 0.1 ln(factor) + 1 (YaRN, arXiv 2309.00071);
      "smooth"  as "blend", with the share linear in the number of turns and no scale of the values.
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
    return Rotary(freqs.to(device), interleaved, scale)


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


def rotary(x, positions, plan, *, out=None):
    """x with the first 2 * len(plan.freqs) values of every head rotated by its token's position.

    x: fp16 or bf16, [B, H, N, D] with positions [N] or [B, N], or packed [T, H, D] with positions [T];
    positions: int32 or int64. Returns out, laid out like x; out=x rotates in place. A pair (a, b) at
    position p becomes scale * (a cos - b sin, b cos + a sin) of the angle p * freqs[i].
    """
    if _lib.native is not None:  # the common call, made natively; None: not one of those
        result = _lib.native.rotary(x, positions, *plan, out)
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
