"""spl_sage.rotary -- rotary positions along a sequence.

The tables and options of SageAttention.rotary and SageAttention.cache_append
(sage_rotary_table, sage_rotary_apply in include/sage_hip.h; no counterpart in
the reference, whose 2D tables are spl_sage.qkv's). Device buffers are torch
tensors.
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


@dataclass(frozen=True)
class Rotary:
    """An uploaded RotaryTable with its layout, and the rows' positions (int32
    device tensor; None: the token's index, or its slot in cache_append). Made
    once for its tensors, whose contents may change."""

    table: object
    rot: int
    layout: RotaryLayout = RotaryLayout.Half
    positions: object = None

    def __post_init__(self):
        import torch

        if self.table.dtype != torch.float32 or not self.table.is_contiguous():
            raise SageError(1, f"the rotary table must be a contiguous float32 device tensor, got {self.table.dtype}")
        p, n = (None, 0) if self.positions is None else _ints(self.positions, "rotary positions")
        c = _abi.sage_rotary(self.table.data_ptr(), self.table.numel(), self.rot, int(self.layout), p, n)
        object.__setattr__(self, "_struct", c)
        at = (self.table,) if self.positions is None else (self.table, self.positions)
        object.__setattr__(self, "_device", _device_of("the rotary table and positions", *at))


__all__ = ["RotaryLayout", "ScalingKind", "RotaryScaling", "RotaryTable", "Rotary"]
