"""Rotary positions on int16 query and key rows (nsrl_rotary_rows).

The reference's models learn their positions or have none.  Here the queries and
keys of a Q|K|V projection turn before an attention called by itself (`apply` on
the q | k columns), and the gradients of its backward turn back
(`backward=True`); `cache.prenorm_attention_decode_block_q4` takes a plan.  The
fused transformer block, `train.TrainModel` and the generators take none.

The angles are 64-bit fractions of a turn, so positions far into a long
context lose nothing, and cos and sin are integer functions of them (the
recipe is in include/nsrl_b200.h): results do not depend on the machine.
"""
from __future__ import annotations

import ctypes as C
import decimal
from typing import List, Optional

import torch

from . import core

LAYOUTS = {"half": 0, "interleaved": 1}
SCALINGS = ("none", "linear", "ntk", "by_parts")


class RotaryC(C.Structure):
    _fields_ = [("turns", C.c_void_p), ("rotary_dim", C.c_size_t), ("interleaved", C.c_int32),
                ("amplitude", C.c_int32)]


def _lib():
    L = core.lib()
    if not getattr(L, "_rotary_bound", False):
        vp, sz = C.c_void_p, C.c_size_t
        L.nsrl_rotary_rows.argtypes = [vp, sz, sz, sz, sz, C.POINTER(RotaryC), vp, sz, C.c_int, vp, sz, vp]
        L._rotary_bound = True
    return L


def turns_per_position(rotary_dim: int, base=10000, scaling="none", factor=1, original_len=0, low=1,
                       high=4) -> List[int]:
    """Turns per position of each pair in units of 2^-64 turn, rounded to nearest:
    base^(-2 i / rotary_dim) / (2 pi), for contexts `factor` times the trained one
      linear    divided by factor
      ntk       with base * factor^(rotary_dim / (rotary_dim - 2)), which leaves the
                fastest pair and divides the slowest by factor
      by_parts  whole for pairs that make at least `high` turns over original_len
                positions, divided by factor at `low` turns or fewer, between them
                in proportion.
    Computed with 60 decimal digits, so the rounding is the exact one."""
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError("rotary_dim must be even and at least 2")
    if scaling not in SCALINGS:
        raise ValueError(f"scaling must be one of {SCALINGS}")
    with decimal.localcontext() as ctx:
        ctx.prec = 60
        D = decimal.Decimal
        two_pi = 2 * D("3.14159265358979323846264338327950288419716939937510582097494459")
        factor, base = D(factor), D(base)
        if factor <= 0 or base <= 0:
            raise ValueError("base and factor must be positive")
        if scaling == "by_parts" and (original_len <= 0 or not high > low):
            raise ValueError("by_parts needs original_len > 0 and high > low")
        if scaling == "ntk" and rotary_dim > 2:
            base *= factor ** (D(rotary_dim) / D(rotary_dim - 2))
        out = []
        for i in range(rotary_dim // 2):
            turn = base ** (-D(2 * i) / D(rotary_dim)) / two_pi
            if scaling == "linear":
                turn /= factor
            elif scaling == "by_parts":
                whole = (D(original_len) * turn - D(low)) / (D(high) - D(low))
                whole = min(D(1), max(D(0), whole))
                turn *= whole + (1 - whole) / factor
            out.append(int((turn * (1 << 64)).to_integral_value(decimal.ROUND_HALF_EVEN)) % (1 << 64))
    return out


class Rotary:
    """The angles of one model: made once, used by every layer and step.

    amplitude multiplies cos and sin (long-context recipes that raise the
    logits put the square root of their factor here), in Q30 below 2."""

    def __init__(self, head_dim: int, rotary_dim: Optional[int] = None, base=10000, layout: str = "half",
                 scaling: str = "none", factor=1, original_len=0, low=1, high=4, amplitude: float = 1.0):
        rotary_dim = head_dim if rotary_dim is None else rotary_dim
        if layout not in LAYOUTS:
            raise ValueError(f"layout must be one of {tuple(LAYOUTS)}")
        if not 2 <= rotary_dim <= head_dim <= 1024:
            raise ValueError("need 2 <= rotary_dim <= head_dim <= 1024")
        q30 = int(decimal.Decimal(amplitude) * (1 << 30) + decimal.Decimal("0.5"))
        if not 1 <= q30 < 1 << 31:
            raise ValueError("amplitude must be positive and below 2")
        self.head_dim, self.rotary_dim = head_dim, rotary_dim
        turns = turns_per_position(rotary_dim, base, scaling, factor, original_len, low, high)
        self.turns = torch.tensor([t - (1 << 64) if t >> 63 else t for t in turns], dtype=torch.int64,
                                  device=core._dev())
        self._c = RotaryC(self.turns.data_ptr(), rotary_dim, LAYOUTS[layout], q30)
        self._ref = C.byref(self._c)

    def c(self) -> RotaryC:
        return self._c

    def apply(self, x: torch.Tensor, heads: int, positions: Optional[torch.Tensor] = None, seq_len: int = 0,
              backward: bool = False, out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
        """Turns the first heads * head_dim columns of the int16 rows x [rows, >= heads * head_dim].

        positions: int32 [rows], or None for row % seq_len.  out may be x (in
        place); by default a new [rows, heads * head_dim] tensor.  Enqueues on
        the current stream without waiting; None on an invalid shape."""
        L, dev = _lib(), torch.cuda.current_device()
        cols = heads * self.head_dim
        rows = x.shape[0]
        xp, ldx = core._rows(x, rows, cols, dev, "x")
        pp = None if positions is None else core._array(positions, torch.int32, (rows,), dev, "positions")
        if self.turns.get_device() != dev:
            core._refuse(self.turns, torch.int64, dev, "the rotary plan", "on the current device")
        if out is None:
            out = torch.empty((rows, cols), dtype=torch.int16, device=x.device)
        yp, ldy = core._rows(out, rows, cols, dev, "out")
        if rows == 0:
            return out
        r = L.nsrl_rotary_rows(xp, rows, heads, self.head_dim, ldx, self._ref, pp, seq_len,
                               1 if backward else 0, yp, ldy, core._raw_stream(dev))
        if r == core.NSRL_OK:
            return out
        if r == core.NSRL_INVALID_SHAPE:
            return None
        core._check(r)
