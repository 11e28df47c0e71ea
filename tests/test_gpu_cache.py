"""Rotary positions, and the paged 4-bit cache's writes and reads, on the GPU
against float64 numpy (cache_oracle): rotations to a rounding of their type,
codes, scales and values read back exactly."""
from __future__ import annotations

import numpy as np
import pytest

import cache_oracle as O
from conftest import from_device16, to_device16

pytestmark = pytest.mark.gpu
DT = {"bf16": 0, "f16": 1}


def decode16(u, t):
    u = np.asarray(u, np.uint16)
    if t == "f16":
        return u.view(np.float16).astype(np.float64)
    return (u.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def draw16(torch, rng, shape, t, scale=1.0):
    """Device tensor of normal draws and its float64 values."""
    x = torch.from_numpy((rng.standard_normal(shape) * scale).astype(np.float32)).to(
        torch.bfloat16 if t == "bf16" else torch.float16).cuda()
    return x, x.double().cpu().numpy()


def ints(torch, v):
    return torch.tensor(np.asarray(v).tolist(), dtype=torch.int32, device="cuda")


def close_to_rounding(got, want, terms, t):
    """A sum of two products in fp32 (three roundings, each of at most the terms' size) rounded once to t."""
    tol = O.HALF_STEP[t] * (np.abs(want) + terms * 2.0 ** -22) + terms * 2.0 ** -22
    tol += 2.0 ** -25 if t == "f16" else 0.0
    assert (np.isnan(got) == np.isnan(want)).all()
    bad = ~((np.abs(got - want) <= tol) | np.isnan(want))
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4], got[bad][:4], want[bad][:4])


@pytest.mark.parametrize("t", ["bf16", "f16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rot", [None, 2, 20, 32, 48, 62])
@pytest.mark.parametrize("pairs", [False, True])
def test_rotary(torch_gpu, t, d, rot, pairs):
    import spl_sage as S
    from spl_sage import rotary as R

    torch, rot = torch_gpu, rot or d
    rng = np.random.default_rng(rot * 7 + d + pairs)
    sa = S.SageAttention(torch.cuda.current_stream(), d)
    table = R.RotaryTable.new(rot, 500)
    for batch, tokens, heads in ((1, 1, 1), (2, 37, 5), (1, 130, 9)):
        x, xv = draw16(torch, rng, (batch, tokens, heads, d), t)
        pos = rng.integers(0, 500, batch * tokens)
        r = R.Rotary(table.upload(), rot, R.RotaryLayout(int(pairs)), ints(torch, pos))
        for transpose in (False, True):
            out = torch.full_like(x, 7.0)
            sa.rotary(S.Shape(batch, heads, tokens), r, S.Tensor(x), S.TensorMut(out), transpose)
            got = decode16(from_device16(out), t).reshape(-1, heads, d)
            flat = xv.reshape(-1, heads, d)
            want = O.rotate(flat, table.cos_sin, pos, rot, pairs, transpose)
            terms = np.abs(flat).max(-1, keepdims=True) * 2.0
            close_to_rounding(got, want, np.broadcast_to(terms, want.shape), t)
            assert (got[..., rot:] == flat[..., rot:]).all()


def test_rotary_in_place_strided_and_default_positions(torch_gpu):
    """Heads inside fused rows, head-major rows, and x itself as the output; positions by index."""
    import spl_sage as S
    from spl_sage import rotary as R

    torch, d, rot = torch_gpu, 128, 64
    rng = np.random.default_rng(3)
    sa = S.SageAttention(torch.cuda.current_stream(), d)
    table = R.RotaryTable.new(rot, 64)
    r = R.Rotary(table.upload(), rot)
    fused, fv = draw16(torch, rng, (2, 33, 10, d), "bf16")
    want = O.rotate(fv[:, :, 2:9].reshape(66, 7, d), table.cos_sin, np.tile(np.arange(33), 2), rot, False)
    terms = np.broadcast_to(np.abs(fv).max() * 2, want.shape)
    out = torch.zeros(2, 7, 33, d, dtype=torch.bfloat16, device="cuda")
    part = fused[:, :, 2:9]
    sa.rotary(S.Shape(2, 7, 33), r, S.Tensor(part), S.TensorMut(out, S.Strides.bhtd(33, 7, d)))
    close_to_rounding(decode16(from_device16(out.transpose(1, 2).contiguous()), "bf16").reshape(66, 7, d), want, terms, "bf16")
    keep = fused.clone()
    sa.rotary(S.Shape(2, 7, 33), r, S.Tensor(part), S.TensorMut(part))
    assert torch.equal(part, out.transpose(1, 2))
    assert torch.equal(fused[:, :, :2], keep[:, :, :2]) and torch.equal(fused[:, :, 9:], keep[:, :, 9:])


def test_rotary_positions_outside_the_table_are_nan(torch_gpu):
    import spl_sage as S
    from spl_sage import rotary as R

    torch, d, rot = torch_gpu, 64, 32
    sa = S.SageAttention(torch.cuda.current_stream(), d)
    table = R.RotaryTable.new(rot, 10)
    x = torch.ones(1, 5, 3, d, dtype=torch.float16, device="cuda")
    pos = [-1, 0, 9, 10, 2 ** 31 - 1]
    out = torch.zeros_like(x)
    sa.rotary(S.Shape(1, 3, 5), R.Rotary(table.upload(), rot, R.RotaryLayout.Pairs, ints(torch, pos)), S.Tensor(x),
              S.TensorMut(out))
    nan = torch.isnan(out[0])
    for i, p in enumerate(pos):
        assert nan[i, :, :rot].all() == (not 0 <= p < 10) and not nan[i, :, rot:].any()


def test_rotary_transpose_is_the_gradient(torch_gpu):
    """<y', R x> = <R^T y', x> for random x, y', and R's difference quotients along single channels."""
    import spl_sage as S
    from spl_sage import rotary as R

    torch, d = torch_gpu, 64
    rng = np.random.default_rng(5)
    sa = S.SageAttention(torch.cuda.current_stream(), d)
    table = R.RotaryTable.new(d, 200, scaling=R.RotaryScaling(R.ScalingKind.Yarn, 4.0, 64.0))
    pos = rng.integers(0, 200, 40)
    for layout in R.RotaryLayout:
        r = R.Rotary(table.upload(), d, layout, ints(torch, pos))
        x, xv = draw16(torch, rng, (1, 40, 3, d), "f16")
        g, gv = draw16(torch, rng, (1, 40, 3, d), "f16")
        y, gx = torch.empty_like(x), torch.empty_like(x)
        sa.rotary(S.Shape(1, 3, 40), r, S.Tensor(x), S.TensorMut(y))
        sa.rotary(S.Shape(1, 3, 40), r, S.Tensor(g), S.TensorMut(gx), transpose=True)
        yv, gxv = y.double().cpu().numpy(), gx.double().cpu().numpy()
        # Each side's outputs are off by half a step at most, and half a subnormal's.
        tol = 2.0 ** -10 * (np.abs(gv * yv).sum(-1) + np.abs(gxv * xv).sum(-1)) + 1e-5
        assert (np.abs((gv * yv).sum(-1) - (gxv * xv).sum(-1)) <= tol).all()
        for c in (0, 5, d // 2, d - 1):  # R is linear: (R(x + e) - R(x)) . g / |e| = (R^T g)_c, with |e| = 4
            x2 = x.clone()
            x2[..., c] += 4.0
            e = (x2[..., c].double() - x[..., c].double()).cpu().numpy()
            y2 = torch.empty_like(x)
            sa.rotary(S.Shape(1, 3, 40), r, S.Tensor(x2), S.TensorMut(y2))
            y2v = y2.double().cpu().numpy()
            slope = ((y2v - yv) * gv).sum(-1) / e
            tol = 2.0 ** -11 * (((np.abs(y2v) + np.abs(yv)) * np.abs(gv)).sum(-1) / np.abs(e) + np.abs(gxv[..., c])) + 1e-5
            assert (np.abs(slope - gxv[..., c]) <= tol).all()


class Pool:
    """A batch over a pool with shuffled pages, host copies beside the device's."""

    def __init__(self, torch, d, starts, lengths, kv, page, heads=None, rows=None, extra_cols=1, seed=0, spare=3, max_new=None):
        from spl_sage import cache as C

        rng = np.random.default_rng(seed)
        b = len(lengths)
        cols = max(-(-max(max(lengths), 1) // page), 1) + extra_cols
        pages = b * cols + spare
        self.starts, self.lengths, self.page = list(starts), list(lengths), page
        self.table = rng.permutation(pages)[:b * cols].reshape(b, cols).astype(np.int32)
        self.rows = starts[-1] if rows is None else rows
        most = max([starts[i + 1] - starts[i] for i in range(b)] + [0]) if max_new is None else max_new
        self.shape = C.CacheShape(b, self.rows, most, heads or kv, kv, pages, page, cols)
        self.pages, self.d, self.kv = pages, d, kv
        fill = lambda n, hi: rng.integers(0, hi, (pages, kv, page, n)).astype(np.uint8)  # noqa: E731
        self.host = {"k_codes": fill(d // 2, 256), "k_scales": fill(d // 32, 14) + 120, "v_codes": fill(d // 2, 256),
                     "v_scales": fill(d // 32, 14) + 120}
        self.torch = torch
        self.upload()

    def upload(self):
        from spl_sage import cache as C

        torch = self.torch
        self.cache = C.PagedCache(self.shape, **{n: torch.from_numpy(x.copy()).cuda() for n, x in self.host.items()})
        self.index = C.CacheIndex(ints(torch, self.starts), ints(torch, self.lengths), ints(torch, self.table))

    def values(self, side):
        return O.values(self.host[side + "_codes"], self.host[side + "_scales"])

    def cells(self):
        return O.cells(self.starts, self.lengths, self.table, self.page, self.pages, self.rows)

    def device(self, name):
        return getattr(self.cache, name).cpu().numpy()


BATCHES = [
    ([0, 1], [1]),
    ([0, 1, 2, 3, 4, 5], [1, 17, 300, 16, 64]),                # a step of one token each
    ([0, 5, 5, 42, 43, 170], [5, 9, 40, 100, 127]),            # ragged, one without rows
    ([3, 10, 30], [7, 300]),                                   # rows before the first sequence and behind the last
]


@pytest.mark.parametrize("t", ["bf16", "f16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("which", range(len(BATCHES)))
def test_append_and_read(torch_gpu, t, d, page, which):
    """Codes and scales of the appended rows equal the oracle's, every other byte is untouched, and reading gives the
    values that they stand for; keys rotated on the way equal rotary() followed by an append."""
    import spl_sage as S
    from spl_sage import rotary as R

    torch = torch_gpu
    starts, lengths = BATCHES[which]
    kv, heads, rows = 3, 6, starts[-1] + 4
    rng = np.random.default_rng(which * 100 + page + d)
    sa = S.SageAttention(torch.cuda.current_stream(), d)
    for rot, pairs in ((0, False), (d, False), (d // 2, True), (20, False)):
        p = Pool(torch, d, starts, lengths, kv, page, heads, rows, seed=which)
        fused, _ = draw16(torch, rng, (rows, heads + 2 * kv, d), t, 3.0)
        q, k, v = fused[None, :, :heads], fused[None, :, heads:heads + kv], fused[None, :, heads + kv:]
        r = None
        if rot:
            table = R.RotaryTable.new(rot, 600)
            r = R.Rotary(table.upload(), rot, R.RotaryLayout(int(pairs)))
        q_out = torch.full((1, rows, heads, d), 9.0, dtype=fused.dtype, device="cuda")
        if rot:
            sa.cache_append(p.cache, p.index, S.Tensor(k), S.Tensor(v), r, S.Tensor(q), S.TensorMut(q_out))
        else:
            sa.cache_append(p.cache, p.index, S.Tensor(k), S.Tensor(v))
        kk, qq = k, q
        cells = p.cells()
        if rot:  # the same rows by rotary()
            pos = np.zeros(rows, int)
            for row, _, _, slot in cells:
                pos[row] = slot
            rr = R.Rotary(r.table, rot, r.layout, ints(torch, pos))
            kk, qq = torch.empty_like(k), torch.empty_like(q)
            sa.rotary(S.Shape(1, kv, rows), rr, S.Tensor(k), S.TensorMut(kk))
            sa.rotary(S.Shape(1, heads, rows), rr, S.Tensor(q), S.TensorMut(qq))
            mine = [c[0] for c in cells]
            assert torch.equal(q_out[0, mine], qq[0, mine])
            others = sorted(set(range(rows)) - set(mine))
            assert (q_out[0, others] == 9.0).all()
        for side, x in (("k", kk), ("v", v)):
            codes, scales, vals = O.quantise(x[0].double().cpu().numpy())
            for row, pg, tok, _ in cells:
                if pg >= 0:
                    p.host[side + "_codes"][pg, :, tok] = codes[row]
                    p.host[side + "_scales"][pg, :, tok] = scales[row]
            for name in (side + "_codes", side + "_scales"):
                got = p.device(name)
                bad = got != p.host[name]
                assert not bad.any(), (name, np.argwhere(bad)[:4], got[bad][:4], p.host[name][bad][:4])
        ko, vo = (torch.full((1, rows, kv, d), 5.0, dtype=fused.dtype, device="cuda") for _ in range(2))
        sa.cache_read(p.cache, p.index, S.TensorMut(ko), S.TensorMut(vo))
        for side, got in (("k", ko), ("v", vo)):
            want = np.full((rows, kv, d), 5.0)
            val = p.values(side)
            for row, pg, tok, _ in cells:
                want[row] = val[pg, :, tok] if pg >= 0 else 0
            assert (decode16(from_device16(got[0]), t) == want).all()


@pytest.mark.parametrize("d", [64, 128])
def test_codec_on_every_value(torch_gpu, d):
    """Every 16-bit value of both types, in blocks of all kinds: sorted (one magnitude a block), shuffled (blocks with
    large and small ones), zeros of both signs, subnormals, infinities and NaN."""
    import spl_sage as S

    torch = torch_gpu
    sa = S.SageAttention(torch.cuda.current_stream(), d)
    rng = np.random.default_rng(1)
    u = np.arange(65536, dtype=np.uint16)
    for t in ("bf16", "f16"):
        finite = u[np.isfinite(decode16(u, t))]
        finite = np.concatenate([finite, finite[:-len(finite) % 128]])
        near = finite[np.argsort(np.abs(decode16(finite, t)), kind="stable")]
        sets = [u, finite, near, rng.permutation(finite)]
        for s in sets:
            x = s[:len(s) // d * d].reshape(1, -1, 1, d)
            rows = x.shape[1]
            p = Pool(torch, d, [0, rows], [rows], 1, 256, seed=2)
            k = to_device16(torch, x, DT[t])
            sa.cache_append(p.cache, p.index, S.Tensor(k), S.Tensor(k))
            codes, scales, vals = O.quantise(decode16(x[0], t))
            pg = p.table[0, np.arange(rows) // 256]
            at = (pg, 0, np.arange(rows) % 256)
            for side in "kv":
                got_s, got_c = p.device(side + "_scales")[at], p.device(side + "_codes")[at]
                assert (got_s == scales[:, 0]).all(), np.argwhere(got_s != scales[:, 0])[:3]
                bad = got_c != codes[:, 0]
                assert not bad.any(), (t, np.argwhere(bad)[:3], got_c[bad][:3], codes[:, 0][bad][:3])
            out = [torch.empty_like(k) for _ in range(2)]
            sa.cache_read(p.cache, p.index, *(S.TensorMut(o) for o in out))
            got = out[0].double().cpu().numpy()
            want = torch.from_numpy(vals[None]).to(k.dtype).double().numpy()
            assert ((got == want) | (np.isnan(got) & np.isnan(want))).all()
            assert torch.equal(out[0].view(torch.int16), out[1].view(torch.int16))


def test_slots_that_hold_nothing(torch_gpu):
    """Slots before 0 and past the page table, and pages outside the pool: nothing is written, zeros are read."""
    import spl_sage as S

    torch, d, kv, page = torch_gpu, 64, 2, 16
    sa = S.SageAttention(torch.cuda.current_stream(), d)
    starts, lengths = [0, 10, 60, 90], [4, 70, 40]  # the first: six rows before slot 0
    p = Pool(torch, d, starts, lengths, kv, page, extra_cols=0, seed=4)
    p.table[1, 2], p.table[1, 3], p.table[2, 1] = -1, p.pages, -2 ** 31
    p.lengths[1] = p.table.shape[1] * page + 7  # the last seven rows are past the page table
    p.upload()
    rng = np.random.default_rng(0)
    k, _ = draw16(torch, rng, (1, 90, kv, d), "bf16")
    v, _ = draw16(torch, rng, (1, 90, kv, d), "bf16")
    sa.cache_append(p.cache, p.index, S.Tensor(k), S.Tensor(v))
    cells = p.cells()
    assert sum(c[1] < 0 for c in cells) > 20 and sum(c[1] >= 0 for c in cells) > 20
    for side, x in (("k", k), ("v", v)):
        codes, scales, _ = O.quantise(x[0].double().cpu().numpy())
        for row, pg, tok, _ in cells:
            if pg >= 0:
                p.host[side + "_codes"][pg, :, tok], p.host[side + "_scales"][pg, :, tok] = codes[row], scales[row]
        assert (p.device(side + "_codes") == p.host[side + "_codes"]).all()
        assert (p.device(side + "_scales") == p.host[side + "_scales"]).all()
    ko, vo = (torch.full((1, 90, kv, d), 5.0, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    sa.cache_read(p.cache, p.index, S.TensorMut(ko), S.TensorMut(vo))
    val = p.values("k")
    for row, pg, tok, _ in cells:
        want = val[pg, :, tok] if pg >= 0 else np.zeros((kv, d))
        assert (ko[0, row].double().cpu().numpy() == want).all()


def test_many_sequences(torch_gpu):
    """More sequences than a workgroup looks over at once, some without rows."""
    import spl_sage as S

    torch, d, kv = torch_gpu, 64, 1
    rng = np.random.default_rng(8)
    sa = S.SageAttention(torch.cuda.current_stream(), d)
    for b in (63, 64, 65, 1500):
        news = rng.integers(0, 4, b)
        starts = np.concatenate([[0], np.cumsum(news)]).tolist()
        lengths = (news + rng.integers(0, 20, b)).tolist()
        p = Pool(torch, d, starts, lengths, kv, 16, seed=b)
        k, kvv = draw16(torch, rng, (1, starts[-1], kv, d), "f16")
        sa.cache_append(p.cache, p.index, S.Tensor(k), S.Tensor(k))
        codes, scales, _ = O.quantise(kvv[0])
        for row, pg, tok, _ in p.cells():
            p.host["k_codes"][pg, :, tok], p.host["k_scales"][pg, :, tok] = codes[row], scales[row]
        assert (p.device("k_codes") == p.host["k_codes"]).all() and (p.device("k_scales") == p.host["k_scales"]).all()


def test_rotary_of_the_most_rows(torch_gpu):
    """2^26 - 4 rows, the last count whose launch is allowed, over themselves: every 2^20th row and the ends turn, and the
    rest is what was there (zeros); one row more is refused."""
    import spl_sage as S
    from spl_sage import rotary as R

    torch, d, rows = torch_gpu, 64, 2 ** 26 - 4
    rng = np.random.default_rng(0)
    at = sorted({0, 1, 2, 3, *range(5, rows, 2 ** 20), rows - 4, rows - 3, rows - 2, rows - 1})
    x = torch.zeros(1, rows + 1, 1, d, dtype=torch.bfloat16, device="cuda")
    some, sv = draw16(torch, rng, (len(at), 1, d), "bf16")
    index = torch.tensor(at, device="cuda")
    x[0, index] = some
    x[0, rows] = 7.0
    table = R.RotaryTable.new(d, 100)
    pos = torch.zeros(rows + 1, dtype=torch.int32, device="cuda")
    want_pos = rng.integers(0, 100, len(at))
    pos[index] = ints(torch, want_pos)
    sa = S.SageAttention(torch.cuda.current_stream(), d)
    r = R.Rotary(table.upload(), d, R.RotaryLayout.Half, pos)
    with pytest.raises(S.SageError, match="exceed the launch grid"):
        sa.rotary(S.Shape(1, 1, rows + 1), r, S.Tensor(x), S.TensorMut(x))
    sa.rotary(S.Shape(1, 1, rows), r, S.Tensor(x), S.TensorMut(x))
    want = O.rotate(sv, table.cos_sin, want_pos, d, False)
    terms = O.rotate(np.abs(sv), np.abs(table.cos_sin) * [1, -1], want_pos, d, False)  # |a c| + |b s|
    got = x[0, index].double().cpu().numpy()
    assert (np.abs(got - want) <= O.HALF_STEP["bf16"] * (np.abs(want) + 2.0 ** -20) + np.abs(terms).max() * 2.0 ** -22).all()
    x[0, index] = 0
    assert (x[0, rows] == 7.0).all() and not x[0, :rows].any()
