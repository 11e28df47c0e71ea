"""The rotary and paged-cache entry points on the CPU: their C structs, tables
and refusals, the index lookups on bad indexes (tests/cpp/cache_host.cpp, under
the sanitizers), and the oracle of the GPU tests against second forms."""
from __future__ import annotations

import ctypes as C
import math
import os
import subprocess

import numpy as np
import pytest

import cache_oracle as O
from test_cpp_host import SAN_BIN, SAN_ENV
from test_host_api import HEADER

STRUCTS = {
    "sage_rotary_scaling": ["kind", "factor", "original", "beta_fast", "beta_slow", "attention"],
    "sage_rotary": ["table", "table_len", "rot", "layout", "positions", "positions_len"],
    "sage_cache_shape": ["batch", "rows", "max_new", "heads", "kv_heads", "pages", "page_tokens", "max_pages"],
    "sage_cache": ["k_codes", "k_scales", "v_codes", "v_scales", "codes_len", "scales_len"],
    "sage_cache_index": ["starts", "starts_len", "lengths", "lengths_len", "page_table", "page_table_len"],
    "sage_cache_options": ["softmax_scale", "has_softmax_scale", "causal"],
}


def test_refusals_and_index_lookups_under_sanitizers():
    exe = SAN_BIN.parent / "cache_host"
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


@pytest.mark.parametrize("rot", [2, 4, 20, 64, 128])
@pytest.mark.parametrize("kind", ["none", "linear", "ntk", "yarn"])
def test_tables(rot, kind):
    """The angles from their definitions in 64 bits; cos and sin of them are off by their angle's error and half an
    fp32 step. Positions up to 200000: an angle there is known to 200000 * 2^-52 or so."""
    from spl_sage import SageError
    from spl_sage import rotary as R

    n, f, original = 200_001 if rot == 64 else 3001, 8.0, 512.0
    sc = None if kind == "none" else R.RotaryScaling(R.ScalingKind[kind.title()], f, original)
    if kind == "ntk" and rot == 2:
        with pytest.raises(SageError, match="NTK"):
            R.RotaryTable.new(rot, n, 5e5, sc)
        return
    t = R.RotaryTable.new(rot, n, 5e5, sc).cos_sin
    a = O.angles(rot, n, 5e5, kind, f, original)
    m = 0.1 * math.log(f) + 1 if kind == "yarn" else 1.0
    assert t.shape == (n, rot // 2, 2) and t.dtype == np.float32
    tol = m * (2.0 ** -24 + n * 2.0 ** -48)
    assert np.abs(t[..., 0] - m * np.cos(a)).max() <= tol and np.abs(t[..., 1] - m * np.sin(a)).max() <= tol


def test_yarn_ends():
    """Pairs that turn often keep their angle, slow ones are interpolated; an attention factor replaces the default."""
    from spl_sage import rotary as R

    t = R.RotaryTable.new(128, 50, scaling=R.RotaryScaling(R.ScalingKind.Yarn, 4.0, 4096.0, attention=2.0)).cos_sin
    plain = R.RotaryTable.new(128, 50).cos_sin
    slow = R.RotaryTable.new(128, 50, scaling=R.RotaryScaling(R.ScalingKind.Linear, 4.0)).cos_sin
    assert np.allclose(t[:, 0], 2 * plain[:, 0], rtol=0, atol=1e-6) and np.allclose(t[:, -1], 2 * slow[:, -1], rtol=0, atol=1e-6)


def test_wrong_types_are_refused():
    import torch

    from spl_sage import SageError
    from spl_sage import cache as K
    from spl_sage import rotary as R

    with pytest.raises(SageError, match="float32"):
        R.Rotary(torch.zeros(8, dtype=torch.float64), 4)
    with pytest.raises(SageError, match="int32"):
        R.Rotary(torch.zeros(8), 4, positions=torch.zeros(4, dtype=torch.int64))
    i = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(SageError, match="int32"):
        K.CacheIndex(i, i, i.view(2, 2).t())
    shape = K.CacheShape(1, 1, 1, 1, 1, 1, 16, 1)
    assert shape.sizes(64) == (512, 32)
    c = K.PagedCache.new(shape, 64, device="cpu")
    with pytest.raises(SageError, match="uint8"):
        K.PagedCache(shape, c.k_codes.to(torch.int8), c.k_scales, c.v_codes, c.v_scales)
    with pytest.raises(SageError, match="pages of 17 tokens"):
        K.PagedCache.new(K.CacheShape(1, 1, 1, 1, 1, 1, 17, 1), 64, device="cpu")


class _Far:
    """A handle or tensor of device 1, as far as the check sees it."""

    _device, strides = 1, None
    data = property(lambda self: self)

    def get_device(self):
        return 1


def test_tensors_out_of_reach_are_refused():
    """Host memory, another device's and channels apart: refused before the library is called, whichever tensor it is."""
    import torch

    import spl_sage as S
    from spl_sage import cache as K
    from spl_sage import rotary as R

    sa = object.__new__(S.SageAttention)  # no GPU here: the checks come before the handle's use
    sa._h = None
    i = torch.zeros(2, dtype=torch.int32)
    shape = K.CacheShape(1, 1, 1, 1, 1, 1, 16, 1)
    pool, index, r = K.PagedCache.new(shape, 64, device="cpu"), K.CacheIndex(i, i, i), R.Rotary(torch.zeros(8), 4)
    x = torch.zeros(1, 1, 1, 64, dtype=torch.bfloat16)
    t, m = S.Tensor(x), S.TensorMut(x)
    ws = type("", (), {"_h": None})

    class Far(_Far):
        shape = pool.shape

    calls = [((pool, index, t, m), lambda *a: sa.cache_attend(ws, *a)),
             ((r, t, m), lambda *a: sa.rotary(S.Shape(1, 1, 1), *a)),
             ((pool, index, t, t, r, t, m), sa.cache_append),
             ((pool, index, t, t), sa.cache_append),
             ((pool, index, m, m), sa.cache_read)]
    for args, call in calls:
        sa._device = 0
        with pytest.raises(S.SageError, match="in host memory, the context on device 0"):
            call(*args)
        sa._device = -1  # host memory passes for the device's
        for n in range(len(args)):
            with pytest.raises(S.SageError, match="on device 1, the context on device -1"):
                call(*args[:n], Far(), *args[n + 1:])
    with pytest.raises(S.SageError, match="channels"):
        sa.cache_read(pool, index, m, S.TensorMut(torch.zeros(1, 1, 64, 8, dtype=torch.bfloat16).transpose(2, 3)))


def test_handles_of_one_device():
    import torch

    from spl_sage import SageError
    from spl_sage import cache as K
    from spl_sage import rotary as R

    i, far = torch.zeros(2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32, device="meta")
    assert R._device_of("all", i, i) == -1
    with pytest.raises(SageError, match="the cache's index are on different devices"):
        R._device_of("the cache's index", i, far)
    assert K.CacheIndex(i, i, i)._device == -1


def test_oracle_quantiser():
    """Known answers, ties to the even code, the scale's edge at 1.5 * 2^k, NaN blocks, and no level nearer."""
    x = np.zeros((6, 32))
    x[0, :10] = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, -5.0, 0.2500001]
    x[1, 0], x[2, 0] = 6.0 * 2.0 ** 9, 6.0001 * 2.0 ** 9
    x[3, 4], x[4, 31] = np.inf, np.nan
    x[5, 0] = 2.0 ** -133
    codes, scales, v = O.quantise(x)
    assert scales[:, 0].tolist() == [127, 136, 137, 255, 255, 1]
    assert v[0, :10].tolist() == [0, 1, 1, 2, 2, 4, 4, 6, -4, 0.5]
    assert np.isnan(v[3]).all() and np.isnan(v[4]).all() and v[1, 0] == 6 * 512 and v[2, 0] == 6 * 512
    y = np.random.default_rng(0).standard_normal((500, 64)) * 10
    codes, scales, v = O.quantise(y)
    step = np.exp2(scales.astype(float) - 127).repeat(32, -1)
    best = np.min(np.abs(np.abs(y)[..., None] - O.LEVELS * step[..., None]), -1)
    assert np.allclose(np.abs(v - y), best, rtol=0, atol=1e-12) and (np.abs(y) <= 6 * step).all()


def test_oracle_attention_is_the_softmax():
    """Against the textbook form on one sequence without pages."""
    rng = np.random.default_rng(0)
    n, kv, d = 40, 2, 64
    k, v, q = rng.standard_normal((n, kv, d)), rng.standard_normal((n, kv, d)), rng.standard_normal((5, 4, d))
    pad = lambda x: np.concatenate([x, np.full((8, kv, d), np.nan)]).reshape(3, 16, kv, d).transpose(0, 2, 1, 3)  # noqa: E731
    got, _, _ = O.attend(q, pad(k), pad(v), [0, 5], [n], np.array([[0, 1, 2]]), 16, True, 0.1, np.zeros((5, 4, d)))
    for h in range(4):
        x = 0.1 * q[:, h] @ k[:, h // 2].T
        x[np.arange(n)[None] > np.arange(n - 5, n)[:, None]] = -np.inf
        p = np.exp(x) / np.exp(x).sum(1, keepdims=True)
        assert np.allclose(got[:, h], p @ v[:, h // 2], rtol=1e-12, atol=1e-12)


def test_layouts_that_differ_are_refused():
    """A pool, workspace or page table of another layout, whose buffers are long enough: refused before the library is
    called."""
    import torch

    import spl_sage as S
    from spl_sage import cache as K

    sa = object.__new__(S.SageAttention)  # no GPU here: the checks come before the handle's use
    sa._h, sa._device, sa._head_dim = None, -1, 64
    shape = K.CacheShape(2, 4, 2, 4, 2, 8, 32, 3)
    pool = K.PagedCache.new(shape, 64, device="cpu")
    ints = lambda *n: torch.zeros(*n, dtype=torch.int32)  # noqa: E731
    index = K.CacheIndex(ints(3), ints(2), ints(2, 3))
    x = torch.zeros(1, 4, 4, 64, dtype=torch.bfloat16)
    t, m = S.Tensor(x), S.TensorMut(x)
    ws = lambda h: type("", (), {"_h": None, "shape": h})  # noqa: E731

    # A step of any size over the same pool passes the checks, up to the library's own.
    for h in (shape, K.CacheShape(1, 1, 1, 2, 2, 8, 32, 3)):
        with pytest.raises(S.SageError, match="null argument"):
            sa.cache_attend(ws(h), pool.with_shape(h), index, t, m)
    fewer = K.CacheShape(2, 4, 2, 4, 2, 7, 32, 3)  # the same places, other pages that are there
    for h in (K.CacheShape(2, 4, 2, 4, 2, 16, 16, 6), K.CacheShape(2, 4, 2, 4, 4, 4, 32, 3), K.CacheShape(2, 4, 2, 4, 2, 9, 32, 3), fewer):
        if h is fewer:
            with pytest.raises(S.SageError, match="null argument"):
                sa.cache_attend(ws(h), pool.with_shape(h), index, t, m)
        else:
            with pytest.raises(S.SageError, match="the cache's tensors and shape differ"):
                pool.with_shape(h)
        with pytest.raises(S.SageError, match="the workspace and the cache differ"):
            sa.cache_attend(ws(h), pool, index, t, m)
    wide = K.CacheIndex(ints(3), ints(2), ints(2, 4))
    calls = [lambda p, i: sa.cache_attend(ws(shape), p, i, t, m), lambda p, i: sa.cache_append(p, i, t, t),
             lambda p, i: sa.cache_read(p, i, m, m)]
    for call in calls:
        with pytest.raises(S.SageError, match="4 columns, the shape 3"):
            call(pool, wide)
        with pytest.raises(S.SageError, match="made for head dim 128, the context for 64"):
            call(K.PagedCache.new(shape, 128, device="cpu"), index)
        with pytest.raises(S.SageError, match="null argument"):
            call(pool, index)
    big = K.PagedCache.new(shape, 128, device="cpu")
    with pytest.raises(S.SageError, match="head dims 128 and 64"):
        K.PagedCache(shape, big.k_codes, big.k_scales, pool.v_codes, pool.v_scales)
    # Tensors that say no layout are the caller's word.
    flat = K.PagedCache(shape, *(getattr(pool, n).flatten() for n in ("k_codes", "k_scales", "v_codes", "v_scales")))
    with pytest.raises(S.SageError, match="null argument"):
        sa.cache_read(flat, K.CacheIndex(ints(3), ints(2), ints(6)), m, m)
