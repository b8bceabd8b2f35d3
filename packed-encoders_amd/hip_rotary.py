"""Rotary positions as an operator of its own: either pair layout, part of the head, scaled frequencies,
with a gradient (``csrc/pe_paged_rope.h``).

``hip_attention.rope_qkv`` serves the packed encoder's layers (split-half pairs over the whole head, from
bf16 tables, out of the packed projection). ``rotary`` serves models whose heads turn otherwise: the angle
comes from a position and a frequency inside the kernel, so there are no tables, and positions may reach
far (the angle is reduced in 64 bits). ``paged.paged_append`` does the same rotation on the way into a
paged cache.
"""

from __future__ import annotations

import ctypes
import math

import torch
from torch import Tensor

from . import _lib
from ._native import native_for

_DTYPES = {torch.bfloat16: _lib.ROTARY_BF16, torch.float16: _lib.ROTARY_FP16, torch.float32: _lib.ROTARY_FP32}


def _check_frequencies(inv_freq: Tensor, d: int, device) -> int:
    if not isinstance(inv_freq, Tensor) or inv_freq.ndim != 1 or inv_freq.dtype != torch.float32:
        raise ValueError("inv_freq must be a 1-D float32 tensor, one frequency per pair")
    if inv_freq.device != device:
        raise ValueError("inv_freq must be on the rotated tensor's device")
    half = inv_freq.numel()
    if not 1 <= half <= _lib.ROTARY_MAX_PAIRS or 2 * half > d:
        raise ValueError(f"{half} pairs do not fit a head of {d} (at most {_lib.ROTARY_MAX_PAIRS} pairs)")
    return half


def _check(x: Tensor, positions: Tensor, inv_freq: Tensor) -> None:
    if x.ndim < 2:
        raise ValueError("rotary expects [..., heads, head_dim]")
    if x.dtype not in _DTYPES:
        raise ValueError(f"rotary takes bfloat16, float16 or float32, not {x.dtype}")
    if not isinstance(positions, Tensor) or positions.dtype not in (torch.int64, torch.int32):
        raise ValueError("positions must be an int64 or int32 tensor")
    if positions.device != x.device:
        raise ValueError("positions must be on x's device")
    lead = x.shape[:-2]
    if positions.ndim > len(lead) or any(p not in (1, n) for p, n in zip(positions.shape[::-1], lead[::-1])):
        raise ValueError(f"positions {tuple(positions.shape)} do not broadcast to {tuple(lead)}")
    if max(x.shape[-2:]) >= 2**31:
        raise ValueError("rotary's heads and head_dim fit 32 bits")
    _check_frequencies(inv_freq, x.shape[-1], x.device)


def _rotary_impl(x: Tensor, positions: Tensor, inv_freq: Tensor, interleaved: bool, inverse: bool,
                 scale: float) -> Tensor:
    _check(x, positions, inv_freq)
    out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if out.numel() == 0:
        return out
    rows = x.reshape(-1, *x.shape[-2:])
    if rows.stride(-1) != 1:
        rows = rows.contiguous()
    positions = positions.expand(x.shape[:-2]).reshape(-1).contiguous()
    inv_freq = inv_freq.contiguous()
    a = _lib.RotaryArgs()
    a.struct_size = ctypes.sizeof(_lib.RotaryArgs)
    a.dtype = _DTYPES[x.dtype]
    a.x, a.out, a.positions, a.inv_freq = rows.data_ptr(), out.data_ptr(), positions.data_ptr(), inv_freq.data_ptr()
    a.x_stride_token, a.x_stride_head = rows.stride(0), rows.stride(1)
    a.n_tokens, a.n_heads, a.head_dim = rows.shape
    a.half = inv_freq.numel()
    a.positions_32 = int(positions.dtype == torch.int32)
    a.interleaved, a.inverse, a.scale = int(interleaved), int(inverse), float(scale)
    with torch.cuda.device(x.device):
        stream = torch.cuda.current_stream(x.device).cuda_stream
        _lib.check(_lib.library().pe_rotary_fwd(ctypes.byref(a), stream), "pe_rotary_fwd")
    return out


def _rotary_meta(x: Tensor, positions: Tensor, inv_freq: Tensor, interleaved: bool, inverse: bool,
                 scale: float) -> Tensor:
    return torch.empty(x.shape, dtype=x.dtype, device=x.device)


def _rotate(x: Tensor, positions: Tensor, inv_freq: Tensor, interleaved: bool, inverse: bool, scale: float) -> Tensor:
    native = native_for(x)
    if native is not None:
        out = native.rotary(x, positions, inv_freq, interleaved, inverse, scale)
        if out is not None:
            return out
    return torch.ops.pe_hip.rotary(x, positions, inv_freq, interleaved, inverse, scale)


class _Rotary(torch.autograd.Function):
    """The rotation; its gradient is the rotation by the opposite angle (and so is that one's)."""

    @staticmethod
    def forward(ctx, x, positions, inv_freq, interleaved, inverse, scale):
        ctx.save_for_backward(positions, inv_freq)
        ctx.options = (interleaved, inverse, scale)
        return _rotate(x, positions, inv_freq, interleaved, inverse, scale)

    @staticmethod
    def backward(ctx, grad):
        positions, inv_freq = ctx.saved_tensors
        interleaved, inverse, scale = ctx.options
        return _apply(grad, positions, inv_freq, interleaved, not inverse, scale), None, None, None, None, None


def _apply(x: Tensor, positions: Tensor, inv_freq: Tensor, interleaved: bool, inverse: bool, scale: float) -> Tensor:
    if torch.is_grad_enabled() and isinstance(inv_freq, Tensor) and inv_freq.requires_grad:
        raise ValueError("rotary has no gradient for inv_freq")
    if torch.is_grad_enabled() and x.requires_grad:
        return _Rotary.apply(x, positions, inv_freq, interleaved, inverse, scale)
    return _rotate(x, positions, inv_freq, interleaved, inverse, scale)


def rotary(x: Tensor, positions: Tensor, inv_freq: Tensor, *, interleaved: bool = False,
           scale: float = 1.0) -> Tensor:
    """Rotary positions of ``x [..., heads, head_dim]`` (bfloat16, float16 or float32, on the GPU).

    ``inv_freq`` (float32 ``[R / 2]``) gives one frequency per pair of the head's first R elements, the
    others are copied: pairs ``(i, i + R / 2)``, or ``(2 i, 2 i + 1)`` with ``interleaved``. Pair i of a token
    at position s turns by ``s * inv_freq[i]``, ``(a, b) -> scale * (a cos - b sin, b cos + a sin)``, in 32 bits
    with the angle reduced in 64, rounded once. ``positions`` (int64 or int32, any sign) broadcasts to
    ``x.shape[:-2]``. ``rotary_frequencies`` makes ``inv_freq`` and ``scale``, also for long contexts.

    Returns a new contiguous tensor; differentiable in ``x``. ``ValueError`` for other arguments."""
    if not isinstance(x, Tensor) or x.device.type == "cpu":
        raise ValueError("rotary runs on the HIP device")
    return _apply(x, positions, inv_freq, bool(interleaved), False, float(scale))


def rotary_frequencies(rot_dim: int, theta: float, *, scaling: str | None = None, factor: float = 1.0,
                       original: int | None = None, beta_fast: float = 32.0, beta_slow: float = 1.0,
                       low: float = 1.0, high: float = 4.0, device=None) -> tuple[Tensor, float]:
    """``(inv_freq, scale)`` for ``rotary`` on ``rot_dim`` elements of a head: ``theta ** (-2 i / rot_dim)``,
    stretched by ``factor`` for contexts longer than the trained one (``original`` positions):

    - ``"linear"``: every frequency divided by ``factor``;
    - ``"ntk"``: the base raised to ``theta * factor ** (R / (R - 2))``, so that the slowest pair is divided by
      ``factor`` and the fastest kept;
    - ``"ramp"``: pairs that turn more than ``beta_fast`` times over ``original`` are kept, those that turn
      fewer than ``beta_slow`` times divided, a linear ramp over the pairs between; ``scale`` becomes
      ``0.1 ln(factor) + 1``;
    - ``"bands"``: pairs of a wavelength below ``original / high`` are kept, those above ``original / low``
      divided, the others interpolated by ``original`` over their wavelength."""
    rot_dim, factor, theta = int(rot_dim), float(factor), float(theta)
    if rot_dim < 2 or rot_dim % 2 or not theta > 0.0 or not factor >= 1.0:
        raise ValueError("rotary_frequencies needs an even rot_dim, a positive theta and a factor of at least 1")
    if scaling not in (None, "linear", "ntk", "ramp", "bands"):
        raise ValueError(f"unknown scaling {scaling!r}")
    if scaling in ("ramp", "bands") and (original is None or original < 1):
        raise ValueError(f"scaling {scaling!r} needs the original context length")
    if scaling == "ramp" and not (theta > 1.0 and beta_fast >= beta_slow > 0.0):
        raise ValueError("scaling 'ramp' needs a theta above 1 and beta_fast >= beta_slow > 0")
    if scaling == "bands" and not high > low > 0.0:
        raise ValueError("scaling 'bands' needs high > low > 0")
    if scaling == "ntk":
        if rot_dim < 4:
            raise ValueError("scaling 'ntk' needs a rot_dim of at least 4")
        theta *= factor ** (rot_dim / (rot_dim - 2))
    inv = theta ** (-torch.arange(0, rot_dim, 2, dtype=torch.float64) / rot_dim)
    scale = 1.0
    if scaling == "linear":
        inv = inv / factor
    elif scaling == "ramp":
        def pair(turns: float) -> float:  # the (fractional) pair that turns that often over the original context
            return rot_dim * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(theta))

        first, last = max(math.floor(pair(beta_fast)), 0), min(math.ceil(pair(beta_slow)), rot_dim - 1)
        index = torch.arange(rot_dim // 2, dtype=torch.float64)
        divided = ((index - first) / max(last - first, 1e-3)).clamp(0.0, 1.0)
        inv = inv * (1.0 - divided) + inv / factor * divided
        scale = 0.1 * math.log(factor) + 1.0
    elif scaling == "bands":
        wavelength = 2 * math.pi / inv
        kept = ((original / wavelength - low) / (high - low)).clamp(0.0, 1.0)
        inv = inv * kept + inv / factor * (1.0 - kept)
    return inv.float().to(device), scale


def _register() -> None:
    lib = torch.library.Library("pe_hip", "FRAGMENT")
    try:
        lib.define("rotary(Tensor x, Tensor positions, Tensor inv_freq, bool interleaved, bool inverse, float scale) "
                   "-> Tensor")
    except RuntimeError:
        return  # already defined by an earlier import in this process
    lib.impl("rotary", _rotary_impl, "CUDA")
    lib.impl("rotary", _rotary_meta, "Meta")
    globals()["_TORCH_LIBRARY"] = lib


_register()

__all__ = ["rotary", "rotary_frequencies"]
