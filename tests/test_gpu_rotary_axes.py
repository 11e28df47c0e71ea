"""Rotary positions with several axes on the GPU against float64 numpy
(pick_oracle): every layout, dealing and type, in place, strided, transposed, and
inside the append, where the codes are those of the rotation followed by an append."""
from __future__ import annotations

import numpy as np
import pytest

import cache_oracle as O
import pick_oracle as P
from conftest import from_device16
from test_gpu_cache import BATCHES, Pool, close_to_rounding, decode16, draw16, ints

pytestmark = pytest.mark.gpu
SECTIONS = {64: [(8, 12, 12), (12, 10, 10), (32,), (8, 8, 8), (3, 1), (8, 8, 8, 8)],
            128: [(16, 24, 24), (22, 21, 21), (64,), (16, 16, 16), (7, 2, 30, 5), (24, 40)]}
WAYS = [("Half", False), ("Half", True), ("Pairs", False), ("Pairs", True), ("AxisHalf", False)]


def axes_rotary(torch, table, sections, pos, layout, dealt):
    from spl_sage import rotary as R

    return R.AxesRotary(table.upload(), sections, ints(torch, pos), R.AxisLayout[layout], dealt)


@pytest.mark.parametrize("t", ["bf16", "f16"])
@pytest.mark.parametrize("d,which", [(d, i) for d in (64, 128) for i in range(6)])
@pytest.mark.parametrize("layout,dealt", WAYS)
def test_axes(torch_gpu, t, d, which, layout, dealt):
    import spl_sage as S
    from spl_sage import rotary as R

    torch, sections = torch_gpu, SECTIONS[d][which]
    rng = np.random.default_rng(d + which)
    sa = S.SageAttention(torch.cuda.current_stream(), d)
    table = R.RotaryTable.axes(sections, 300, dealt=dealt, per_axis=which % 2 == 0)
    rot = 2 * sum(sections)
    for batch, tokens, heads in ((1, 1, 1), (2, 37, 5), (1, 130, 9)):
        x, xv = draw16(torch, rng, (batch, tokens, heads, d), t)
        pos = rng.integers(0, 300, (len(sections), batch * tokens))
        r = axes_rotary(torch, table, sections, pos, layout, dealt)
        for transpose in (False, True):
            out = torch.full_like(x, 7.0)
            sa.rotary(S.Shape(batch, heads, tokens), r, S.Tensor(x), S.TensorMut(out), transpose)
            got = decode16(from_device16(out), t).reshape(-1, heads, d)
            flat = xv.reshape(-1, heads, d)
            want = P.rotate_axes(flat, table.cos_sin, pos, sections, layout, dealt, transpose)
            terms = np.abs(flat).max(-1, keepdims=True) * 2.0
            close_to_rounding(got, want, np.broadcast_to(terms, want.shape), t)
            assert (got[..., rot:] == flat[..., rot:]).all()


@pytest.mark.parametrize("layout", ["Half", "Pairs"])
def test_equal_positions_are_one_axis(torch_gpu, layout):
    """Rows whose positions are alike on all axes (text) turn bit for bit as with one axis."""
    import spl_sage as S
    from spl_sage import rotary as R

    torch, d, sections = torch_gpu, 128, (16, 24, 24)
    rng = np.random.default_rng(0)
    sa = S.SageAttention(torch.cuda.current_stream(), d)
    x, _ = draw16(torch, rng, (1, 77, 6, d), "bf16")
    pos = rng.integers(0, 500, 77)
    table = R.RotaryTable.new(d, 500)
    outs = [torch.empty_like(x) for _ in range(3)]
    sa.rotary(S.Shape(1, 6, 77), R.Rotary(table.upload(), d, R.RotaryLayout[layout], ints(torch, pos)), S.Tensor(x), S.TensorMut(outs[0]))
    for dealt in (False, True):
        r = axes_rotary(torch, R.RotaryTable.axes(sections, 500, dealt=dealt), sections, np.stack([pos] * 3), layout, dealt)
        sa.rotary(S.Shape(1, 6, 77), r, S.Tensor(x), S.TensorMut(outs[1 + dealt]))
        assert torch.equal(outs[0], outs[1 + dealt])


@pytest.mark.parametrize("layout,dealt", WAYS)
def test_in_place_strided_and_outside(torch_gpu, layout, dealt):
    """Heads inside fused rows, x itself as the output, positions that are rows of a longer tensor, and positions that
    the table does not hold: their axis's channels alone become NaN."""
    import spl_sage as S
    from spl_sage import rotary as R

    torch, d, sections = torch_gpu, 64, (4, 10, 10)
    rng = np.random.default_rng(3)
    sa = S.SageAttention(torch.cuda.current_stream(), d)
    table = R.RotaryTable.axes(sections, 40, dealt=dealt)
    long = ints(torch, rng.integers(0, 40, (3, 90)))
    r = R.AxesRotary(table.upload(), sections, long[:, 11:77], R.AxisLayout[layout], dealt)
    fused, fv = draw16(torch, rng, (2, 33, 10, d), "f16")
    pos = long[:, 11:77].cpu().numpy()
    want = P.rotate_axes(fv[:, :, 2:9].reshape(66, 7, d), table.cos_sin, pos, sections, layout, dealt)
    terms = np.broadcast_to(np.abs(fv).max() * 2, want.shape)
    keep = fused.clone()
    out = torch.zeros(2, 7, 33, d, dtype=fused.dtype, device="cuda")
    part = fused[:, :, 2:9]
    sa.rotary(S.Shape(2, 7, 33), r, S.Tensor(part), S.TensorMut(out, S.Strides.bhtd(33, 7, d)))
    close_to_rounding(decode16(from_device16(out.transpose(1, 2).contiguous()), "f16").reshape(66, 7, d), want, terms, "f16")
    sa.rotary(S.Shape(2, 7, 33), r, S.Tensor(part), S.TensorMut(part))
    assert torch.equal(part, out.transpose(1, 2))
    assert torch.equal(fused[:, :, :2], keep[:, :, :2]) and torch.equal(fused[:, :, 9:], keep[:, :, 9:])
    pos = np.array([[0, -1, 5, 39], [40, 3, 5, 39], [7, 8, 2 ** 31 - 1, 39]])
    x = torch.ones(1, 4, 3, d, dtype=torch.bfloat16, device="cuda")
    out = torch.zeros_like(x)
    sa.rotary(S.Shape(1, 3, 4), axes_rotary(torch, table, sections, pos, layout, dealt), S.Tensor(x), S.TensorMut(out))
    want = P.rotate_axes(np.ones((4, 3, d)), table.cos_sin, pos, sections, layout, dealt)
    assert (torch.isnan(out[0]).cpu().numpy() == np.isnan(want)).all() and np.isnan(want).sum() == 3 * 2 * (4 + 10 + 10)


@pytest.mark.parametrize("layout,dealt", WAYS)
def test_transpose_is_the_gradient(torch_gpu, layout, dealt):
    """<y', R x> = <R^T y', x>, and R's difference quotients along single channels."""
    import spl_sage as S
    from spl_sage import rotary as R

    torch, d, sections = torch_gpu, 64, (8, 12, 12)
    rng = np.random.default_rng(5)
    sa = S.SageAttention(torch.cuda.current_stream(), d)
    table = R.RotaryTable.axes(sections, 200, scaling=R.RotaryScaling(R.ScalingKind.Yarn, 4.0, 64.0), dealt=dealt)
    r = axes_rotary(torch, table, sections, rng.integers(0, 200, (3, 40)), layout, dealt)
    x, xv = draw16(torch, rng, (1, 40, 3, d), "f16")
    g, gv = draw16(torch, rng, (1, 40, 3, d), "f16")
    y, gx = torch.empty_like(x), torch.empty_like(x)
    sa.rotary(S.Shape(1, 3, 40), r, S.Tensor(x), S.TensorMut(y))
    sa.rotary(S.Shape(1, 3, 40), r, S.Tensor(g), S.TensorMut(gx), transpose=True)
    yv, gxv = y.double().cpu().numpy(), gx.double().cpu().numpy()
    # Each side's outputs are off by half a step at most, and half a subnormal's.
    tol = 2.0 ** -10 * (np.abs(gv * yv).sum(-1) + np.abs(gxv * xv).sum(-1)) + 1e-5
    assert (np.abs((gv * yv).sum(-1) - (gxv * xv).sum(-1)) <= tol).all()
    for c in (0, 9, 40, d - 1):  # R is linear: (R(x + e) - R(x)) . g / |e| = (R^T g)_c, with |e| = 4
        x2 = x.clone()
        x2[..., c] += 4.0
        e = (x2[..., c].double() - x[..., c].double()).cpu().numpy()
        y2 = torch.empty_like(x)
        sa.rotary(S.Shape(1, 3, 40), r, S.Tensor(x2), S.TensorMut(y2))
        y2v = y2.double().cpu().numpy()
        slope = ((y2v - yv) * gv).sum(-1) / e
        tol = 2.0 ** -11 * (((np.abs(y2v) + np.abs(yv)) * np.abs(gv)).sum(-1) / np.abs(e) + np.abs(gxv[..., c])) + 1e-5
        assert (np.abs(slope - gxv[..., c]) <= tol).all()


@pytest.mark.parametrize("t", ["bf16", "f16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("layout,dealt", WAYS)
@pytest.mark.parametrize("which", range(len(BATCHES)))
def test_append_with_axes(torch_gpu, t, d, layout, dealt, which):
    """Codes and scales are those of the keys that rotary() turns, the queries come out as from rotary(), and every
    other byte and row stays."""
    import spl_sage as S
    from spl_sage import rotary as R

    torch = torch_gpu
    starts, lengths = BATCHES[which]
    kv, heads, rows = 3, 6, starts[-1] + 4
    rng = np.random.default_rng(which * 100 + d)
    sa = S.SageAttention(torch.cuda.current_stream(), d)
    for sections in SECTIONS[d][:2]:
        p = Pool(torch, d, starts, lengths, kv, 16, heads, rows, seed=which)
        fused, _ = draw16(torch, rng, (rows, heads + 2 * kv, d), t, 3.0)
        q, k, v = fused[None, :, :heads], fused[None, :, heads:heads + kv], fused[None, :, heads + kv:]
        r = axes_rotary(torch, R.RotaryTable.axes(sections, 600, dealt=dealt), sections, rng.integers(0, 600, (len(sections), rows)),
                        layout, dealt)
        q_out = torch.full((1, rows, heads, d), 9.0, dtype=fused.dtype, device="cuda")
        sa.cache_append(p.cache, p.index, S.Tensor(k), S.Tensor(v), r, S.Tensor(q), S.TensorMut(q_out))
        kk, qq = torch.empty_like(k), torch.empty_like(q)
        sa.rotary(S.Shape(1, kv, rows), r, S.Tensor(k), S.TensorMut(kk))
        sa.rotary(S.Shape(1, heads, rows), r, S.Tensor(q), S.TensorMut(qq))
        cells = p.cells()
        mine = [c[0] for c in cells]
        assert torch.equal(q_out[0, mine], qq[0, mine])
        assert (q_out[0, sorted(set(range(rows)) - set(mine))] == 9.0).all()
        for side, x in (("k", kk), ("v", v)):
            codes, scales, _ = O.quantise(x[0].double().cpu().numpy())
            for row, pg, tok, _ in cells:
                if pg >= 0:
                    p.host[side + "_codes"][pg, :, tok] = codes[row]
                    p.host[side + "_scales"][pg, :, tok] = scales[row]
            for name in (side + "_codes", side + "_scales"):
                assert (p.device(name) == p.host[name]).all(), name
