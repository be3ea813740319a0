"""Rotary positions of a reader model's queries and keys, on one axis or several.

A token of text has one position; a patch of a page image has a page, a line and a
column, each of which turns its own part of a head's dims.
"""
from __future__ import annotations

import math

from maxsim_amd import _native
from maxsim_amd.kvcache import _cuda_device


# A turn, 2 pi, over 10^-49.
_TURN = 2 * 31415926535897932384626433832795028841971693993751


def _fixed_turns(frequency: float) -> int:
    """Turns per position, in 2^-64, whole turns dropped: the exact quotient rounded once."""
    numerator, denominator = frequency.as_integer_ratio()
    numerator, denominator = numerator * 10**49 << 64, denominator * _TURN
    return (2 * numerator + denominator) // (2 * denominator) % 2**64


class Rotary:
    """Turns pairs of dims by their position's angle: pair i of frequency f_i becomes
    ``(x cos t - y sin t, x sin t + y cos t)`` with ``t = f_i * position``.

    The first ``rotary_dim`` dims of a head of ``head_dim`` (default: all; at most 256)
    make rotary_dim / 2 pairs, ``(i, i + rotary_dim / 2)`` or, with ``adjacent``,
    ``(2 i, 2 i + 1)``; the other dims stay as they are.  ``frequencies`` gives each
    pair's (default ``base ** (-2 i / rotary_dim)``), ``axes`` the axis that its
    position is on (default 0), for instance ``[0] * 16 + [1] * 24 + [2] * 24``.

    The angle's fraction of a turn is taken in 64-bit fixed point, so that far
    positions are as exact as near ones."""

    def __init__(self, head_dim: int, *, base: float = 10000.0, rotary_dim: int | None = None, axes=None,
                 frequencies=None, adjacent: bool = False, device="cuda"):
        import torch

        head_dim = int(head_dim)
        rotary_dim = head_dim if rotary_dim is None else int(rotary_dim)
        if rotary_dim < 2 or rotary_dim % 2 or rotary_dim > head_dim:
            raise ValueError("rotary_dim must be even, and between 2 and head_dim")
        if head_dim > 256:
            raise NotImplementedError("head_dim must be at most 256")
        pairs = rotary_dim // 2
        if frequencies is None:
            if not (math.isfinite(base) and base > 0):
                raise ValueError("base must be positive")
            frequencies = [float(base) ** (-2.0 * i / rotary_dim) for i in range(pairs)]
        else:
            frequencies = [float(f) for f in frequencies]
        axes = [0] * pairs if axes is None else [int(a) for a in axes]
        if len(frequencies) != pairs or len(axes) != pairs:
            raise ValueError("frequencies and axes must have one entry for each of rotary_dim / 2 pairs")
        if not all(math.isfinite(f) for f in frequencies):
            raise ValueError("frequencies must be finite")
        if min(axes) < 0 or max(axes) >= pairs:
            raise ValueError("axes must be numbered from 0, and be no more than the pairs")
        self.device = _cuda_device(device)
        self.head_dim, self.rotary_dim = head_dim, rotary_dim
        self.num_axes, self.adjacent = max(axes) + 1, bool(adjacent)
        turns = [_fixed_turns(f) for f in frequencies]  # kept as two's complement numbers
        self._turns = torch.tensor([t - 2**64 if t >= 2**63 else t for t in turns], dtype=torch.int64,
                                   device=self.device)
        self._axes = torch.tensor(axes, dtype=torch.int32, device=self.device)
        self._calls = _native.tensor_calls()
        self._handle = self._calls.rotary(self._turns, self._axes, head_dim, self.num_axes, self.adjacent)

    def __call__(self, q, k, positions, out=None):
        """(q, k) turned: [rows, heads, head_dim] and [rows, kv_heads, head_dim] of one
        type (float32, float16 or bfloat16, any strides with dense rows; k may be
        None), by ``positions`` int32 [num_axes, rows] ([rows] for one axis; any
        numbers).  Computed in single precision, rounded once.  ``out`` is a pair of
        tensors to write, which may be the inputs themselves and must not overlap them
        otherwise.  Enqueued on the current stream; records no gradients."""
        q_out, k_out = (None, None) if out is None else out
        return self._calls.rotate(self._handle, q, k, positions, q_out, k_out)
