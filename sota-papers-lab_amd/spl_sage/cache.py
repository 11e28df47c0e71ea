"""spl_sage.cache -- a paged 4-bit key/value cache and the attention over it.

The types of SageAttention.cache_append, cache_read, cache_workspace and
cache_attend (sage_cache_* in include/sage_hip.h; no counterpart in the
reference). Q, K, V and outputs are [1][row][head][head_dim] views (Tensor,
TensorMut): the sequences' rows packed one behind the other. Device buffers are
torch tensors.
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass

from . import SageError, _abi, _check, _layouts_differ
from ._abi import lib
from .rotary import _device_of, _ints

BLOCK = 32  # channels a scale


@dataclass(frozen=True)
class CacheShape:
    """sage_cache_shape: sequences, packed rows, most rows of a sequence, query
    and KV heads, pages of the pool, tokens a page, columns of the page table."""

    batch: int
    rows: int
    max_new: int
    heads: int
    kv_heads: int
    pages: int
    page_tokens: int
    max_pages: int

    def __post_init__(self):
        c = _abi.sage_cache_shape(self.batch, self.rows, self.max_new, self.heads, self.kv_heads, self.pages,
                                  self.page_tokens, self.max_pages)
        object.__setattr__(self, "_struct", c)
        object.__setattr__(self, "_layout", (self.pages, self.kv_heads, self.page_tokens))

    def _c(self) -> _abi.sage_cache_shape:
        return self._struct

    def sizes(self, head_dim: int) -> tuple:
        """Bytes of the codes and of the scales, each for K and for V."""
        codes, scales = C.c_uint64(), C.c_uint64()
        _check(lib().sage_cache_sizes(C.byref(self._c()), head_dim, C.byref(codes), C.byref(scales)))
        return codes.value, scales.value


def _bytes(t, what: str) -> tuple:
    import torch

    if t.dtype != torch.uint8 or not t.is_contiguous():
        raise SageError(1, f"{what} must be a contiguous uint8 device tensor, got {t.dtype}")
    return t.data_ptr(), t.numel()


@dataclass(frozen=True)
class PagedCache:
    """The pool: uint8 device tensors [pages][kv_heads][page_tokens][head_dim/2]
    (codes) and [..][head_dim/32] (scales), of the shape's pages or more. Made
    once for its tensors; one pool serves steps of any shape with its
    page_tokens and kv_heads (with_shape): another's rows lie elsewhere in it,
    and tensors of four dimensions refuse it."""

    shape: CacheShape
    k_codes: object
    k_scales: object
    v_codes: object
    v_scales: object

    @staticmethod
    def new(shape: CacheShape, head_dim: int, device="cuda") -> "PagedCache":
        """A pool of zeros, which torch's current stream fills."""
        import torch

        shape.sizes(head_dim)  # its refusals
        dims = (shape.pages, shape.kv_heads, shape.page_tokens)
        z = lambda n: torch.zeros(*dims, n, dtype=torch.uint8, device=device)  # noqa: E731
        return PagedCache(shape, z(head_dim // 2), z(head_dim // BLOCK), z(head_dim // 2), z(head_dim // BLOCK))

    def with_shape(self, shape: CacheShape) -> "PagedCache":
        return PagedCache(shape, self.k_codes, self.k_scales, self.v_codes, self.v_scales)

    def __post_init__(self):
        kc, ks = _bytes(self.k_codes, "cache K codes"), _bytes(self.k_scales, "cache K scales")
        vc, vs = _bytes(self.v_codes, "cache V codes"), _bytes(self.v_scales, "cache V scales")
        dims = None  # of a row's codes and scales, where the tensors say them
        for pair in ((self.k_codes, self.k_scales), (self.v_codes, self.v_scales)):
            for t, channels in zip(pair, (2, BLOCK)):
                if t.dim() != 4:
                    continue
                if t.shape[0] < self.shape.pages or tuple(t.shape[1:3]) != self.shape._layout[1:]:
                    raise _layouts_differ("the cache's tensors and shape", tuple(t.shape[:3]), self.shape._layout)
                if dims not in (None, t.shape[3] * channels):
                    raise SageError(1, f"the cache's tensors are of head dims {dims} and {t.shape[3] * channels}")
                dims = t.shape[3] * channels
        object.__setattr__(self, "_head_dim", dims)
        c = _abi.sage_cache(kc[0], ks[0], vc[0], vs[0], min(kc[1], vc[1]), min(ks[1], vs[1]))
        object.__setattr__(self, "_struct", c)
        object.__setattr__(self, "_device", _device_of("the cache's buffers", self.k_codes, self.k_scales, self.v_codes,
                                                       self.v_scales))


@dataclass(frozen=True)
class CacheIndex:
    """int32 device tensors: starts [batch + 1], lengths [batch] (this step's
    rows included), page_table [batch][max_pages]. Made once for its tensors,
    whose contents change from step to step."""

    starts: object
    lengths: object
    page_table: object

    def __post_init__(self):
        c = _abi.sage_cache_index(*_ints(self.starts, "cache starts"), *_ints(self.lengths, "cache lengths"),
                                  *_ints(self.page_table, "cache page table"))
        object.__setattr__(self, "_struct", c)
        object.__setattr__(self, "_cols", self.page_table.shape[1] if self.page_table.dim() == 2 else None)
        object.__setattr__(self, "_device", _device_of("the cache's index", self.starts, self.lengths, self.page_table))


class CacheWorkspace:
    """What cache_attend keeps between its kernels, for one shape; one call at a time uses it."""

    def __init__(self, sa, shape: CacheShape):
        h = C.c_void_p()
        _check(lib().sage_cache_workspace_new(sa._h, C.byref(shape._c()), C.byref(h)))
        self._h = h.value
        self.shape = shape
        # Bound now: at interpreter exit the module's globals may be gone before __del__ runs.
        self._destroy = lib().sage_cache_workspace_destroy

    def __del__(self):
        h, self._h = getattr(self, "_h", None), None
        destroy = getattr(self, "_destroy", None)
        if h and destroy is not None:
            destroy(h)

    def bytes(self) -> int:
        return lib().sage_cache_workspace_bytes(self._h)


__all__ = ["BLOCK", "CacheShape", "PagedCache", "CacheIndex", "CacheWorkspace"]
