"""The kernels that the picks and the attention over them are built as, on the CPU: a call can launch every one of them, and
none but the named one uses scratch memory, by the compiler's own account."""
from __future__ import annotations

import re

import pytest

from test_device_asm import assembly
from test_gpu_pick import plan


def kernels(unit, name):
    """{template arguments: (VGPRs, scratch bytes)} of the unit's kernels of that name."""
    out = {}
    for k in re.split(r"\n  - ", assembly(unit).split(".amdgpu_metadata")[1]):
        m = re.search(rf"\.name:\s+\S*?{len(name)}{name}I((?:L[ib]\d+E)+)E", k)
        if m:
            get = lambda f: int(re.search(rf"\.{f}:\s+(\d+)", k).group(1))  # noqa: E731
            args = tuple(int(x) for x in re.findall(r"L[ib](\d+)E", m.group(1)))
            out[args] = get("vgpr_count"), get("private_segment_fixed_size")
    return out


def test_units_of_32_columns():
    """Head dim, bf16 parts of a query, pages of a step and more: fp16 queries of 128 channels run in units of 16."""
    got = kernels("sage_cache_picked.hip.o", "picked_chunk")
    assert set(got) == {(d, parts, big) for d, parts in ((64, 1), (64, 2), (128, 1)) for big in (0, 1)}
    assert all(vgprs <= 256 and scratch == 0 for vgprs, scratch in got.values()), got


def test_units_of_16_columns():
    got = {k: v for k, v in kernels("sage_cache_attn.hip.o", "cache_attn").items() if k[3]}
    assert set(got) == {(d, parts, waves, 1) for d in (64, 128) for parts in (1, 2) for waves in (4, 8)}
    assert all(vgprs <= 256 and scratch == 0 for vgprs, scratch in got.values()), got


@pytest.mark.parametrize("name,want", [
    ("row_pick_kernel", {(d, tiles, keys) for d in (64, 128) for tiles in (1, 2, 4) for keys in (4, 8, 16, 32)}),
    ("score_kernel", {(64, 4), (128, 4)}),
    ("score_tile_kernel", {(64,), (128,)}),
    ("pick_kernel", {(1, 4), (1, 8), (1, 16), (4, 16), (16, 32)}),
    ("bounds_kernel", {(64, 1), (64, 2), (64, 4), (64, 8), (128, 2), (128, 4), (128, 8)})])
def test_picks(name, want):
    """row_pick_kernel<128, 4, 32> keeps two registers in memory."""
    got = kernels("sage_cache_pick.hip.o", name)
    assert set(got) == want
    for args, (vgprs, scratch) in got.items():
        assert scratch <= (12 if (name, args) == ("row_pick_kernel", (128, 4, 32)) else 0), (args, vgprs, scratch)


@pytest.mark.parametrize("d,group,page,least", [(128, 4, 64, 64), (128, 4, 32, 256), (128, 4, 16, 256), (128, 8, 64, 256),
                                                (64, 8, 64, 64), (64, 4, 128, 64), (64, 4, 16, 256)])
def test_units_of_32_columns_where_there_are_many(d, group, page, least):
    """On both sides of the number of units (rows * group / 32 * KV heads) from which a call runs in them."""
    from spl_sage import cache as C

    for rows, chunks in ((32 // group * (least // 8), True), (32 // group * (least // 8 - 1), False)):
        shape = C.CacheShape(1, rows, rows, 8 * group, 8, 1024, page, 256)
        assert plan(shape, d, 32).chunks == chunks, rows
