"""The entry points of a step's index, rotary axes, page bounds and picked pages
on the CPU: their C structs and refusals (tests/cpp/pick_host.cpp, under the
sanitizers), Python's own checks, and the oracle of the GPU tests against second
forms."""
from __future__ import annotations

import ctypes as C
import math
import os
import subprocess

import numpy as np
import pytest

import cache_oracle as O
import pick_oracle as P
from test_cpp_host import SAN_BIN, SAN_ENV
from test_host_api import HEADER

STRUCTS = {
    "sage_rotary_axes": ["table", "table_len", "sections", "axes", "layout", "dealt", "positions", "positions_len",
                         "positions_stride"],
    "sage_cache_requests": ["news", "news_len", "past", "past_len"],
    "sage_cache_free": ["pages", "pages_len", "state", "state_len"],
    "sage_cache_step": ["starts", "starts_len", "lengths", "lengths_len", "page_table", "page_table_len", "positions",
                        "positions_len", "slots", "slots_len", "sequences", "sequences_len", "state", "state_len",
                        "scratch", "scratch_len"],
    "sage_cache_bounds": ["codes", "scales", "codes_len", "scales_len"],
    "sage_pick_options": ["first", "last", "causal"],
}


def test_refusals_under_sanitizers():
    exe = SAN_BIN.parent / "pick_host"
    assert exe.exists(), f"{exe} is not built; run `python __graft_entry__.py` (build)"
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120, env={**os.environ, **SAN_ENV})
    assert r.returncode == 0, r.stdout + r.stderr
    assert "runtime error" not in r.stderr and "Sanitizer" not in r.stderr, r.stderr


def test_ctypes_structs_match_the_c_layout(tmp_path):
    from spl_sage import _abi

    lines = ['#include <stdio.h>', '#include <stddef.h>', f'#include "{HEADER}"', "int main(void) {"]
    for s, fields in STRUCTS.items():
        lines.append(f'printf("{s} %zu\\n", sizeof({s}));')
        lines += [f'printf("{s}.{f} %zu\\n", offsetof({s}, {f}));' for f in fields]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-std=c11", "-Wall", "-o", str(exe), str(src)], check=True)
    got = dict(x.split() for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines())
    for s, fields in STRUCTS.items():
        cls = getattr(_abi, s)
        assert int(got[s]) == C.sizeof(cls) and [f for f, _ in cls._fields_] == fields
        for f in fields:
            assert int(got[f"{s}.{f}"]) == getattr(cls, f).offset, f"{s}.{f}"


@pytest.mark.parametrize("sections", [(16, 24, 24), (5,), (3, 1), (1, 2, 3, 4)])
@pytest.mark.parametrize("dealt", [False, True])
@pytest.mark.parametrize("per_axis", [False, True])
@pytest.mark.parametrize("kind", ["none", "linear", "yarn"])
def test_axes_tables(sections, dealt, per_axis, kind):
    """The angles from their definitions in 64 bits; cos and sin are off by their angle's error and half an fp32 step."""
    from spl_sage import rotary as R

    n, f, original = 900, 8.0, 512.0
    sc = None if kind == "none" else R.RotaryScaling(R.ScalingKind[kind.title()], f, original)
    t = R.RotaryTable.axes(sections, n, 5e5, sc, dealt, per_axis)
    pairs = sum(sections)
    whole = O.angles(2 * pairs, n, 5e5, kind, f, original)
    own = [O.angles(2 * s, n, 5e5, kind, f, original) for s in sections]
    a = np.stack([own[x][:, j] if per_axis else whole[:, i] for i, (x, j) in enumerate(P.axis_of(sections, dealt))], 1)
    m = 0.1 * math.log(f) + 1 if kind == "yarn" else 1.0
    assert t.cos_sin.shape == (n, pairs, 2) and t.rot == 2 * pairs
    tol = m * (2.0 ** -24 + n * 2.0 ** -48)
    assert np.abs(t.cos_sin[..., 0] - m * np.cos(a)).max() <= tol and np.abs(t.cos_sin[..., 1] - m * np.sin(a)).max() <= tol


def test_axes_of_one_are_the_plain_table():
    from spl_sage import rotary as R

    for per_axis in (False, True):
        assert (R.RotaryTable.axes((32,), 50, per_axis=per_axis).cos_sin == R.RotaryTable.new(64, 50).cos_sin).all()


def _fakes():
    import torch

    import spl_sage as S
    from spl_sage import cache as K

    sa = object.__new__(S.SageAttention)  # no GPU here: the checks come before the handle's use
    sa._h, sa._device, sa._head_dim = None, -1, 64
    shape = K.CacheShape(2, 4, 2, 4, 2, 8, 32, 3)
    ints = lambda *n: torch.zeros(*n, dtype=torch.int32)  # noqa: E731
    x = torch.zeros(1, 4, 4, 64, dtype=torch.bfloat16)
    ws = type("", (), {"_h": None, "shape": shape, "top": 2})
    return torch, S, K, sa, shape, ints, S.Tensor(x), S.TensorMut(x), ws


def test_wrong_types_are_refused():
    from spl_sage import rotary as R

    torch, S, K, sa, shape, ints, *_ = _fakes()
    table = torch.zeros(16)
    with pytest.raises(S.SageError, match="float32"):
        R.AxesRotary(table.double(), (2, 2), ints(2, 4))
    for bad in (ints(4), ints(3, 4), ints(4, 2).t()[:, ::2], torch.zeros(2, 4, dtype=torch.int64)):
        with pytest.raises(S.SageError, match="rotary positions must be an int32"):
            R.AxesRotary(table, (2, 2), bad)
    with pytest.raises(S.SageError, match="overlap"):
        R.AxesRotary(table, (2, 2), ints(1, 4).expand(2, 4))
    with pytest.raises(S.SageError, match="5 axes"):
        R.AxesRotary(table, (1,) * 5, ints(5, 4))
    with pytest.raises(S.SageError, match="0 axes"):
        R.AxesRotary(table, (), ints(0, 4))
    r = R.AxesRotary(table, (2, 2), ints(2, 9)[:, 2:6])
    assert r._struct.positions_stride == 9 and r._struct.positions_len == 13
    with pytest.raises(S.SageError, match="int32"):
        K.FreePages(ints(4).long(), ints(4))
    t = K.CacheTables.new(shape, device="cpu")
    with pytest.raises(S.SageError, match="int64"):
        K.CacheTables(shape, t.starts, t.lengths, t.page_table, t.positions, t.positions, t.sequences, t.state, t.scratch)
    with pytest.raises(S.SageError, match="4 columns, the shape 3"):
        K.CacheTables.new(shape, device="cpu", page_table=ints(2, 4))
    b = K.PageBounds.new(shape, 64, device="cpu")
    with pytest.raises(S.SageError, match="int8"):
        K.PageBounds(shape, b.codes.to(torch.uint8), b.scales)
    with pytest.raises(S.SageError, match="uint8"):
        K.PageBounds(shape, b.codes, b.scales.int())
    with pytest.raises(S.SageError, match="do not fit 9 pages"):
        b.with_shape(K.CacheShape(2, 4, 2, 4, 2, 9, 32, 3))
    with pytest.raises(S.SageError, match="int32"):
        K.Picked(torch.zeros(4, 2, 2))


def test_layouts_and_devices_that_differ_are_refused():
    """Before the library is called, whichever argument it is."""
    torch, S, K, sa, shape, ints, t, m, ws = _fakes()
    from spl_sage import rotary as R

    class Far:
        _device, strides, columns = 1, None, ints(4, 2, 2)
        data = property(lambda self: self)

        def get_device(self):
            return 1

    Far.shape = shape
    index = K.CacheIndex(ints(3), ints(2), ints(2, 3))
    pool, bounds = K.PagedCache.new(shape, 64, device="cpu"), K.PageBounds.new(shape, 64, device="cpu")
    picked = K.Picked(ints(4, 2, 2))
    tables, free = K.CacheTables.new(shape, device="cpu"), K.FreePages.new(8, device="cpu")
    axes = R.AxesRotary(torch.zeros(16), (2, 2), ints(2, 4))
    calls = [((tables, ints(2), ints(2), free), sa.cache_tables),
             ((pool, index, bounds), sa.cache_bounds),
             ((bounds, index, t, picked), lambda *a: sa.cache_pick(ws, *a)),
             ((pool, index, picked, t, m), lambda *a: sa.cache_attend_picked(ws, *a)),
             ((axes, t, m), lambda *a: sa.rotary(S.Shape(1, 4, 4), *a)),
             ((pool, index, t, t, axes, t, m), sa.cache_append)]
    for args, call in calls:
        with pytest.raises(S.SageError, match="null argument"):  # the library's own, behind every check here
            call(*args)
        sa._device = 0
        with pytest.raises(S.SageError, match="in host memory, the context on device 0"):
            call(*args)
        sa._device = -1
        for n, a in enumerate(args):
            far = Far()
            if isinstance(a, torch.Tensor):
                continue  # (below)
            with pytest.raises(S.SageError, match="on device 1, the context on device -1"):
                call(*args[:n], far, *args[n + 1:])
    sa._device = -1
    wide = K.CacheIndex(ints(3), ints(2), ints(2, 4))
    for call in (lambda: sa.cache_bounds(pool, wide, bounds), lambda: sa.cache_pick(ws, bounds, wide, t, picked),
                 lambda: sa.cache_attend_picked(ws, pool, wide, picked, t, m)):
        with pytest.raises(S.SageError, match="4 columns, the shape 3"):
            call()
    far = K.PageBounds.new(shape, 128, device="cpu")
    other = K.PageBounds.new(K.CacheShape(2, 4, 2, 4, 4, 8, 32, 3), 64, device="cpu")
    for call in (lambda b: sa.cache_bounds(pool, index, b), lambda b: sa.cache_pick(ws, b, index, t, picked)):
        with pytest.raises(S.SageError, match="bounds are made for head dim 128"):
            call(far)
        with pytest.raises(S.SageError, match="8 pages and 4 KV heads"):
            call(other)
    for bad in (ints(4, 2, 3), ints(4, 1, 4)):
        for call in (lambda p: sa.cache_pick(ws, bounds, index, t, p), lambda p: sa.cache_attend_picked(ws, pool, index, p, t, m)):
            with pytest.raises(S.SageError, match="2 of 2 KV heads a row are expected"):
                call(K.Picked(bad))


# ------------------------------------------------------------------ the oracle


def test_oracle_tables():
    """A step by hand: pages of 16, a request with 17 tokens that gets 20 more, one that ends, a new one."""
    table = np.array([[4, 7, -1], [2, -1, -1], [-1, -1, -1]])
    got = P.tables([20, -1, 3], [17, 5, 0], [9, 8, 0, 0, 6], [4, 3], table, 16, 25)
    assert got["starts"] == [0, 20, 20, 23] and got["lengths"] == [37, 0, 3]
    assert got["page_table"] == [[4, 7, 6], [2, -1, -1], [9, -1, -1]] and got["ring"] == [9, 8, 2, 0, 6]
    assert got["state"] == [1, 2, 0, 0]
    assert got["positions"][:3] == [17, 18, 19] and got["positions"][19:] == [36, 0, 1, 2, 0, 0]
    assert got["slots"][0] == 7 * 16 + 1 and got["slots"][15:] == [96, 97, 98, 99, 100, 144, 145, 146, -1, -1]
    assert got["sequences"] == [0] * 20 + [2] * 3 + [-1] * 2
    void = P.tables([20, -1, 30], [17, 5, 0], [9, 8, 0, 0, 6], [4, 2], table, 16, 25)
    assert void["state"] == [4, 3, 1, 25] and void["starts"] == [0] * 4 and void["lengths"] == [17, 0, 0]


def test_oracle_axes_of_one_are_the_plain_rotation():
    rng = np.random.default_rng(0)
    x, pos = rng.standard_normal((9, 2, 40)), rng.integers(0, 30, 9)
    cs = rng.standard_normal((30, 16, 2))
    for layout, pairs in (("Half", False), ("Pairs", True), ("AxisHalf", False)):
        assert (P.rotate_axes(x, cs, pos[None], (16,), layout, False) == O.rotate(x, cs, pos, 32, pairs)).all()
        y = P.rotate_axes(x, cs, np.stack([pos, pos]), (5, 11), layout, False)
        assert ((y == O.rotate(x, cs, pos, 32, pairs)).all()) == (layout != "AxisHalf")
    i, j = P.channels((2, 3), "AxisHalf")
    assert i.tolist() == [0, 1, 4, 5, 6] and j.tolist() == [2, 3, 7, 8, 9]
    assert [a for a, _ in P.axis_of((1, 3, 2), True)] == [0, 1, 2, 1, 2, 1]


def test_oracle_bounds_hold():
    """No product of a query with a key of the page is above the page's bound, and the bound of one key is its product."""
    rng = np.random.default_rng(1)
    k = rng.standard_normal((16, 64)) * np.exp2(rng.integers(-3, 4, (16, 1)))
    codes, scales, v = O.quantise(k)
    hi, lo, top = P.page_bounds(codes, scales)
    unit = 2.0 ** (top - 127) / 16
    assert (v <= hi * unit).all() and (v >= lo * unit).all() and (v.max(0) > (hi - 1.0) * unit).all()
    q = rng.standard_normal((5, 64))
    assert ((q @ v.T).max(1) <= np.maximum(q * (hi * unit), q * (lo * unit)).sum(1) + 1e-9).all()
    one = P.page_bounds(codes[:1], np.full_like(scales[:1], scales.max()))
    assert (one[0] == one[1]).all()  # whole sixteenths of their own scale
    scales[3, 1] = 255
    hi, lo, _ = P.page_bounds(codes, scales)
    assert (hi[32:] == 127).all() and (lo[32:] == -127).all() and (np.abs(hi[:32]) <= 96).all()


def test_oracle_query_codes():
    q = np.array([[127.0, -0.5, 0.25], [1.5, 2.5, -3.5]])
    assert P.query_codes(q).tolist() == [[127, 0, 0], [2, 2, -4]]
    assert np.abs(P.query_codes(q * 1.01)).max() == 64 and np.abs(P.query_codes(q * 2.0 ** -140)).max() <= 127
    assert (P.query_codes(np.array([[np.inf, 1.0]])) == 0).all() and (P.query_codes(np.zeros((2, 2))) == 0).all()
