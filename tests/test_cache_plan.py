"""The rule that picks the attention kernel of a cache call, on the CPU."""
from __future__ import annotations

import pytest

from cache_plans import plan


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("batch,max_new,heads,kv,tokens,kind", [
    (1, 1, 32, 8, 256, "whole"),       # one step
    (1, 1, 32, 8, 1024, "wide"),       # a short sequence on few units
    (64, 1, 32, 8, 1024, "whole"),     # 512 units
    (1, 1, 32, 8, 4096, "shares"),
    (600, 1, 8, 2, 65536, "whole"),    # more sequences than shares are found among
    (1, 16, 32, 8, 20000, "shares"),   # 64 columns
    (1, 17, 32, 8, 20000, "splits"),   # 68
    (3, 40, 8, 2, 2048, "shares"),     # few tiles over few keys
    (4, 2048, 32, 8, 8192, "chunk"),
    (6, 1500, 16, 16, 1024, "chunk"),  # tiles that fill the chip, whatever the keys
])
def test_kernel_of_a_shape(d, batch, max_new, heads, kv, tokens, kind):
    from spl_sage import cache as K

    shape = K.CacheShape(batch, batch * max_new, max_new, heads, kv, 10, 256, tokens // 256 + (tokens % 256 > 0))
    p = plan(shape, d)
    assert p.kind == kind
    # What the workspace holds follows from it.
    rows = {"splits": p.wgs * shape.rows * heads, "shares": 2 * p.wgs * 16}
    assert p.part_rows == rows.get(kind, 0) and p.wgs >= 1
