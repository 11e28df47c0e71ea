"""spl_sage.rotary -- rotary positions along a sequence, or on several axes.

The tables and options of SageAttention.rotary and SageAttention.cache_append
(sage_rotary_table, sage_rotary_apply and their forms for several axes in
include/sage_hip.h; no counterpart in the reference, whose 2D tables are
spl_sage.qkv's). Device buffers are torch tensors.
"""
from __future__ import annotations

import ctypes as C
import enum
from dataclasses import dataclass
from typing import Optional

import numpy as np

from . import SageError, _abi, _check, _elems_from
from ._abi import lib


class RotaryLayout(enum.IntEnum):
    """Half rotates channels (i, i + rot / 2), Pairs (2 i, 2 i + 1)."""

    Half = 0
    Pairs = 1


class ScalingKind(enum.IntEnum):
    None_ = 0
    Linear = 1
    Ntk = 2
    Yarn = 3


@dataclass(frozen=True)
class RotaryScaling:
    """Contexts `factor` times longer than the model was trained on; original
    (its positions), beta_fast and beta_slow are YaRN's. 0: the default."""

    kind: ScalingKind
    factor: float
    original: float = 0.0
    beta_fast: float = 0.0
    beta_slow: float = 0.0
    attention: float = 0.0

    def _c(self) -> _abi.sage_rotary_scaling:
        return _abi.sage_rotary_scaling(int(self.kind), self.factor, self.original, self.beta_fast, self.beta_slow,
                                        self.attention)


@dataclass
class RotaryTable:
    """cos and sin per (position, pair), float32 [positions][rot/2][2] on the host."""

    rot: int
    positions: int
    cos_sin: np.ndarray

    @staticmethod
    def new(rot: int, positions: int, base: float = 10000.0, scaling: Optional[RotaryScaling] = None) -> "RotaryTable":
        out = np.empty((max(positions, 0), max(rot, 0) // 2, 2), np.float32)
        sc = None if scaling is None else C.byref(scaling._c())
        _check(lib().sage_rotary_table(rot, positions, float(base), sc, out.ctypes.data, out.size))
        return RotaryTable(rot, positions, out)

    @staticmethod
    def axes(sections, positions: int, base: float = 10000.0, scaling: Optional[RotaryScaling] = None,
             dealt: bool = False, per_axis: bool = False) -> "RotaryTable":
        """The table of AxesRotary: sections pairs of each axis, whose frequencies
        are the whole head's, or each axis's own (per_axis)."""
        c = (C.c_uint64 * max(len(sections), 1))(*(max(n, 0) for n in sections))
        rot = 2 * sum(c)
        out = np.empty((max(positions, 0), rot // 2, 2), np.float32)
        sc = None if scaling is None else C.byref(scaling._c())
        _check(lib().sage_rotary_axes_table(c, len(sections), int(dealt), int(per_axis), positions, float(base), sc,
                                            out.ctypes.data, out.size))
        return RotaryTable(rot, positions, out)

    def upload(self, device="cuda"):
        import torch

        return torch.from_numpy(np.ascontiguousarray(self.cos_sin).reshape(-1)).to(device)


def _ints(t, what: str) -> tuple:
    """(address, elements) of a contiguous int32 device tensor."""
    import torch

    if t.dtype != torch.int32 or not t.is_contiguous():
        raise SageError(1, f"{what} must be a contiguous int32 device tensor, got {t.dtype}")
    return t.data_ptr(), t.numel()


def _device_of(what: str, *tensors) -> int:
    """The device that all the tensors are on; -1: host memory."""
    if any(t.device != tensors[0].device for t in tensors):
        raise SageError(1, f"{what} are on different devices")
    return tensors[0].get_device()


def _floats(t, what: str) -> tuple:
    import torch

    if t.dtype != torch.float32 or not t.is_contiguous():
        raise SageError(1, f"{what} must be a contiguous float32 device tensor, got {t.dtype}")
    return t.data_ptr(), t.numel()


@dataclass(frozen=True)
class Rotary:
    """An uploaded RotaryTable with its layout, and the rows' positions (int32
    device tensor; None: the token's index, or its slot in cache_append). Made
    once for its tensors, whose contents may change."""

    table: object
    rot: int
    layout: RotaryLayout = RotaryLayout.Half
    positions: object = None

    APPLY, APPEND = "sage_rotary_apply", "sage_cache_append"  # the calls that take it

    def __post_init__(self):
        t, m = _floats(self.table, "the rotary table")
        p, n = (None, 0) if self.positions is None else _ints(self.positions, "rotary positions")
        c = _abi.sage_rotary(t, m, self.rot, int(self.layout), p, n)
        object.__setattr__(self, "_struct", c)
        at = (self.table,) if self.positions is None else (self.table, self.positions)
        object.__setattr__(self, "_device", _device_of("the rotary table and positions", *at))


class AxisLayout(enum.IntEnum):
    """Half rotates channels (i, i + rot / 2), Pairs (2 i, 2 i + 1), AxisHalf the
    halves within each axis's channels."""

    Half = 0
    Pairs = 1
    AxisHalf = 2


@dataclass(frozen=True)
class AxesRotary:
    """Rotary positions with one to four axes, wherever a Rotary is taken: an
    uploaded RotaryTable.axes, the pairs of each axis, and the rows' positions,
    int32 [axes][rows] on the device (rows of it may be apart). dealt: the pairs
    go to the axes in turn, else in runs. Made once for its tensors, whose contents may change."""

    table: object
    sections: tuple
    positions: object
    layout: AxisLayout = AxisLayout.Half
    dealt: bool = False

    APPLY, APPEND = "sage_rotary_axes_apply", "sage_cache_append_axes"  # the calls that take it

    def __post_init__(self):
        import torch

        t, m = _floats(self.table, "the rotary table")
        x = self.positions
        if x.dtype != torch.int32 or x.dim() != 2 or x.shape[0] != len(self.sections) or (x.shape[1] > 1 and x.stride(1) != 1):
            raise SageError(1, "rotary positions must be an int32 device tensor [axes][rows] with contiguous rows, got "
                               f"{x.dtype} {tuple(x.shape)}")
        if not 1 <= len(self.sections) <= 4:
            raise SageError(1, f"rotary: {len(self.sections)} axes (1 to 4 are supported)")
        rows, stride = x.shape[1], x.shape[1] if x.shape[0] == 1 else x.stride(0)
        if x.shape[0] > 1 and stride < rows:
            raise SageError(1, "the axes' rotary positions overlap")
        c = _abi.sage_rotary_axes(t, m, (C.c_uint64 * 4)(*(max(n, 0) for n in self.sections)), len(self.sections),
                                  int(self.layout), int(self.dealt), x.data_ptr(), (x.shape[0] - 1) * stride + rows, stride)
        object.__setattr__(self, "_struct", c)
        object.__setattr__(self, "_device", _device_of("the rotary table and positions", self.table, x))


__all__ = ["RotaryLayout", "ScalingKind", "RotaryScaling", "RotaryTable", "Rotary", "AxisLayout", "AxesRotary"]
