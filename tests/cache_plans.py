"""Which kernel an attention call over the paged cache runs: the library's own
rule (cache_plan, sage_cache.hpp), which needs no GPU. Tests name the kernel
that they mean, so that a change of the rule cannot leave them without it."""
from __future__ import annotations

import ctypes as C

TOKENS = 64  # of a tile of the chunk kernel, and of a wave's step in the other


class Plan(C.Structure):
    _fields_ = [("chunks", C.c_bool), ("whole", C.c_bool), ("wgs", C.c_int), ("part_rows", C.c_uint64),
                ("wide", C.c_bool)]

    @property
    def kind(self) -> str:
        if self.chunks:
            return "splits" if self.wgs > 1 else "chunk"
        return ("wide" if self.wide else "whole") if self.whole else "shares"


def plan(shape, head_dim: int) -> Plan:
    from spl_sage._abi import lib

    f = lib()._ZN4sage10cache_planEiiiiiii
    f.restype, f.argtypes = Plan, [C.c_int] * 7
    return f(head_dim, shape.batch, shape.rows, shape.heads, shape.kv_heads, shape.max_new,
             shape.max_pages * shape.page_tokens)
