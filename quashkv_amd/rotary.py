"""Rotary positions of query and key rows, before a cache takes the keys.

    turns = rotary_turns(rotary_frequencies(128, base=500000.0), device="cuda")
    plan = store.plan(new_lens, rows)
    q, k = rotary(q, k, plan.positions, turns)
    store.append(k, v, plan)

Pair i of a head's first R coordinates turns by position * w_i radians.  The kernel takes w_i
as turns in units of 2^-64 (int64): the product with a position, modulo a turn, is then exact at
any position, where a 32-bit product of radians is 0.06 off at a million tokens.
"""

from __future__ import annotations

import math
from typing import Optional, Sequence, Union

import torch

from . import _native as N
from .paged8 import _call, _one_device, _want

_TWO_PI_E64 = 62831853071795864769252867665590057683943387987502116419498891846  # 2 pi 10^64


def rotary_frequencies(dim: int, base: float = 10000.0, scaling: Optional[str] = None,
                       factor: float = 1.0, original: int = 8192, low: float = 1.0,
                       high: float = 32.0) -> list[float]:
    """Radians per position of the dim / 2 pairs: w_i = base^(-2 i / dim), for contexts
    ``factor`` times the ``original`` length changed by ``scaling``:

    * None: as they are;
    * "linear": w_i / factor (positions interpolated);
    * "ntk": base * factor^(dim / (dim - 2)), which leaves the shortest wave and makes the longest
      ``factor`` times as long;
    * "ramp": by the turns t_i = original * w_i / 2 pi that a pair makes within the original
      context: as they are from ``high`` turns on, w_i / factor up to ``low`` turns, and
      between them weighted by (t_i - low) / (high - low)."""
    if dim < 2 or dim % 2:
        raise ValueError(f"the rotated part must be a positive even number; got {dim}")
    if not (base > 0 and factor > 0 and original > 0):
        raise ValueError(f"base, factor and original must be positive; got {base}, {factor}, "
                         f"{original}")
    if scaling == "ntk":
        if dim == 2:
            raise ValueError("ntk scaling needs more than one pair")
        base = base * factor ** (dim / (dim - 2))
    w = [base ** (-2 * i / dim) for i in range(dim // 2)]
    if scaling is None or scaling == "ntk":
        return w
    if scaling == "linear":
        return [x / factor for x in w]
    if scaling == "ramp":
        if not high > low:
            raise ValueError(f"high ({high}) must lie above low ({low})")
        out = []
        for x in w:
            keep = min(max((original * x / (2 * math.pi) - low) / (high - low), 0.0), 1.0)
            out.append(x * (keep + (1 - keep) / factor))
        return out
    raise ValueError(f"scaling {scaling!r} must be None, 'linear', 'ntk' or 'ramp'")


def rotary_turns(frequencies: Union[Sequence[float], torch.Tensor], device=None) -> torch.Tensor:
    """Radians per position (a list, or a tensor as models hold them) as the (R / 2,) int64
    tensor of turns that :func:`rotary` takes, rounded to 2^-64 of a turn."""
    if isinstance(frequencies, torch.Tensor):
        frequencies = frequencies.detach().double().reshape(-1).tolist()
    out = []
    for w in frequencies:
        n, d = float(w).as_integer_ratio()      # (raises for NaN and infinities)
        t = (2 * n * 10 ** 64 * 2 ** 64 + d * _TWO_PI_E64) // (2 * d * _TWO_PI_E64) % 2 ** 64
        out.append(t - 2 ** 64 if t >= 2 ** 63 else t)
    return torch.tensor(out, dtype=torch.int64, device=device)


def _out(x: torch.Tensor, shape: torch.Size, out: torch.Tensor, what: str) -> tuple:
    """Strides of an output for rows like x."""
    if out.dtype is not x.dtype or out.shape != shape:
        raise ValueError(f"{what} must be {x.dtype} of shape {tuple(shape)}; got {out.dtype} "
                         f"{tuple(out.shape)}")
    rows, heads, d = shape
    ts, hs, ls = out.stride()
    if ls != 1 and rows * heads > 0:
        raise ValueError(f"{what} must have a dense last axis")
    (near, n), (far, m) = sorted(((ts, rows), (hs, heads)))
    if n > 1 and near < d or m > 1 and far < d + near * (n - 1):
        raise ValueError(f"{what}'s rows or heads overlap")
    return ts, hs


class _Rotary(torch.autograd.Function):
    """rotary with its gradient: the same rows' map by the negative angles."""

    @staticmethod
    def forward(ctx, q, k, positions, turns, factor, interleaved, inverse):
        ctx.set_materialize_grads(False)
        # (a plan's positions are the next step's before a backward pass asks for them)
        ctx.save_for_backward(positions.clone(), turns)
        ctx.args = factor, interleaved, not inverse
        return rotary(q, k, positions, turns, factor, interleaved, inverse)

    @staticmethod
    def backward(ctx, dq, dk):
        positions, turns = ctx.saved_tensors
        dq, dk = (g if need else None for g, need in zip((dq, dk), ctx.needs_input_grad))
        if dq is None and dk is not None:
            dk, _ = rotary(dk, None, positions, turns, *ctx.args)
        elif dq is not None:
            dq, dk = rotary(dq, dk, positions, turns, *ctx.args)
        return dq, dk, None, None, None, None, None


def rotary(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor,
           turns: torch.Tensor, factor: float = 1.0, interleaved: bool = False,
           inverse: bool = False, q_out: Optional[torch.Tensor] = None,
           k_out: Optional[torch.Tensor] = None) -> tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Rows q (rows, Hq, d) and k (rows, Hk, d; None: no keys) of one type (fp32, fp16 or bf16;
    any row and head strides) turned by their positions ((rows,) int32, as a page plan has
    them): pair i of a head's first R = 2 * turns.numel() coordinates -- (i, i + R / 2), or
    (2 i, 2 i + 1) where ``interleaved`` -- by positions * turns[i], times ``factor``
    (which contexts scaled by a ramp take on sine and cosine).  The others are copied.

    ``inverse``: by the negative angles, times ``factor`` all the same: the gradient of a
    call, and where factor is 1 what undoes it.  ``q_out`` / ``k_out`` may be q / k
    themselves, but not overlap them otherwise.

    Autograd goes through results that the call makes; with ``q_out`` or ``k_out`` none of the
    tensors may require a gradient (but under torch.no_grad())."""
    if torch.is_grad_enabled() and (q.requires_grad or k is not None and k.requires_grad
                                    or q_out is not None and q_out.requires_grad
                                    or k_out is not None and k_out.requires_grad):
        if q_out is not None or k_out is not None:
            raise ValueError("q_out and k_out take no gradients, and a tensor of the call "
                             "requires one: leave them out, or call it under torch.no_grad()")
        return _Rotary.apply(q, k, positions, turns, factor, interleaved, inverse)
    dev = _one_device("rotary", q, k, positions, turns, q_out, k_out)
    shape, dtype = q.shape, q.dtype
    if len(shape) != 3:
        raise ValueError(f"queries must be (rows, heads, head_dim); got {tuple(shape)}")
    rows, Hq, d = shape
    ts, hs, ls = q.stride()
    x = q
    if ls != 1:
        x = q.contiguous()
        ts, hs, ls = x.stride()
    if q_out is None:
        q_out, to, ho = torch.empty_like(q, memory_format=torch.contiguous_format), Hq * d, d
    else:
        to, ho = _out(q, shape, q_out, "q_out")
    if k is None:
        if k_out is not None:
            raise ValueError("k_out needs keys")
        keys, keys_out = (None, 0, 0, 0), (None, 0, 0)
    else:
        y, other = k, k.shape
        if len(other) != 3 or other[0] != rows or other[2] != d or k.dtype is not dtype:
            raise ValueError(f"keys must be {dtype} of shape ({rows}, heads, {d}); got {k.dtype} "
                             f"{tuple(other)}")
        Hk = other[1]
        kts, khs, kls = k.stride()
        if kls != 1:
            y = k.contiguous()
            kts, khs, kls = y.stride()
        if k_out is None:
            k_out = torch.empty_like(k, memory_format=torch.contiguous_format)
            kto, kho = Hk * d, d
        else:
            kto, kho = _out(k, other, k_out, "k_out")
        keys, keys_out = (y.data_ptr(), kts, khs, Hk), (k_out.data_ptr(), kto, kho)
    _want(positions, "positions", torch.int32, (rows,))
    if turns.dim() != 1:
        raise ValueError("turns must be a 1-D int64 tensor")
    _want(turns, "turns", torch.int64)
    _call(dev, N.lib().qkv_rotary, N.dtype_code(dtype), x.data_ptr(), ts, hs, Hq, *keys, rows, d,
          2 * turns.numel(), positions.data_ptr(), turns.data_ptr(), float(factor),
          1 if interleaved else 0, 1 if inverse else 0, q_out.data_ptr(), to, ho, *keys_out)
    return q_out, k_out
