"""Bounds of the pages' keys, picked pages and the attention over them on the GPU,
against numpy in 64 bits (pick_oracle): bounds and picks equal, the attention
within the bound that its roundings give."""
from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest

import cache_oracle as O
import pick_oracle as P
from cache_rows import queries, spread, tolerance
from test_gpu_cache import BATCHES, Pool, draw16, ints

pytestmark = pytest.mark.gpu


def bounds_of(torch, p, seed=0):
    """Bounds of other bytes, and their host copies."""
    from spl_sage import cache as C

    rng = np.random.default_rng(seed)
    codes = rng.integers(-128, 128, (p.pages, p.kv, 2, p.d)).astype(np.int8)
    scales = rng.integers(0, 256, (p.pages, p.kv)).astype(np.uint8)
    return C.PageBounds(p.shape, torch.from_numpy(codes.copy()).cuda(), torch.from_numpy(scales.copy()).cuda()), codes, scales


def check_bounds(torch, p):
    import spl_sage as S

    sa = S.SageAttention(torch.cuda.current_stream(), p.d)
    b, codes, scales = bounds_of(torch, p)
    sa.cache_bounds(p.cache, p.index, b)
    n = 0
    for seq, col, held in P.touched(p.starts, p.lengths, p.page, p.table.shape[1], p.shape.max_new):
        page = int(p.table[seq, col])
        if not 0 <= page < p.pages:
            continue
        n += 1
        for g in range(p.kv):
            codes[page, g, 0], codes[page, g, 1], scales[page, g] = P.page_bounds(
                p.host["k_codes"][page, g, :held], p.host["k_scales"][page, g, :held])
    for got, want in ((b.codes, codes), (b.scales, scales)):
        got = got.cpu().numpy()
        bad = got != want
        assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4], got[bad][:4], want[bad][:4])
    return n


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("which", range(len(BATCHES)))
def test_bounds(torch_gpu, d, page, which):
    starts, lengths = BATCHES[which]
    p = Pool(torch_gpu, d, starts, lengths, 3, page, 6, starts[-1] + 4, seed=which)
    assert check_bounds(torch_gpu, p) > 0


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("page", [16, 64, 256])
def test_bounds_of_every_scale(torch_gpu, d, page):
    """Blocks of NaN, all of a page NaN, scales from one end to the other beside each other, zeros, one token, and
    tokens behind the length that would change everything."""
    torch = torch_gpu
    rng = np.random.default_rng(page + d)
    p = Pool(torch, d, [0, 40, 41, 400, 460], [300, 1, 359, 77], 2, page, 4, seed=1)
    s = rng.integers(1, 255, p.host["k_scales"].shape)
    s = np.where(rng.random(s.shape) < 0.02, 255, s)
    near = rng.integers(118, 128, s.shape)
    s = np.where(np.arange(p.pages)[:, None, None, None] % 2 == 0, s, near).astype(np.uint8)
    s[p.table[0, 0]] = 255
    s[p.table[2, 0], 0], s[p.table[2, 0], 1, :, 0] = 0, 255
    p.host["k_scales"] = s
    p.host["k_codes"][p.table[2, 0], 0] = 0
    p.upload()
    check_bounds(torch, p)


def test_bounds_of_bad_indexes(torch_gpu):
    """Pages that are not there, slots before 0, lengths past the table and rows past max_new: their pages stay."""
    torch = torch_gpu
    p = Pool(torch, 64, [0, 50, 90, 95, 200], [30, 60, 5000, 110], 2, 16, 2, seed=2, max_new=60)
    p.table[1, 2], p.table[3, 1], p.table[3, 4] = -1, p.pages, 2 ** 31 - 1
    p.upload()
    assert check_bounds(torch, p) > 0


# ------------------------------------------------------------------ picks


def check_pick(torch, p, q, qv, b, codes, scales, top, first, last, causal):
    import spl_sage as S
    from spl_sage import cache as C

    sa = S.SageAttention(torch.cuda.current_stream(), p.d)
    ws = sa.cache_pick_workspace(p.shape, top)
    out = torch.full((p.rows, p.kv, top), -9, dtype=torch.int32, device="cuda")
    sa.cache_pick(ws, b, p.index, S.Tensor(q), C.Picked(out), first, last, causal)
    torch.cuda.synchronize()  # the workspace lives to the end of the call's work
    want = P.pick(qv[0], codes[:, :, 0], codes[:, :, 1], scales, p.starts, p.lengths, p.table, p.page, p.pages, top, first,
                  last, causal, np.full((p.rows, p.kv, top), -9), p.shape.max_new)
    got = out.cpu().numpy()
    bad = got != want
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:3], got[bad][:6], want[bad][:6])
    return out


def drawn(torch, p, t, seed, near=True):
    """Bounds whose pages are close to each other, and queries."""
    rng = np.random.default_rng(seed)
    b, codes, scales = bounds_of(torch, p, seed)
    if near:
        codes[:] = np.clip(rng.normal(0, 30, codes.shape), -96, 96)
        codes[:, :, 0] = np.maximum(codes[:, :, 0], codes[:, :, 1])
        scales[:] = rng.integers(126, 129, scales.shape)
        b.codes.copy_(torch.from_numpy(codes)), b.scales.copy_(torch.from_numpy(scales))
    q, qv = draw16(torch, rng, (1, p.rows, p.shape.heads, p.d), t)
    return q, qv, b, codes, scales


@pytest.mark.parametrize("t", ["bf16", "f16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("group", [1, 2, 3, 4, 7, 8, 16, 17, 40])
@pytest.mark.parametrize("causal", [True, False])
def test_picks(torch_gpu, t, d, group, causal):
    """Ragged sequences with and without rows, steps and chunks, groups of all sizes."""
    torch = torch_gpu
    kv = 2
    p = Pool(torch, d, [0, 1, 1, 40, 42, 43], [300, 50, 400, 2, 16], kv, 16, kv * group, 47, seed=group)
    for top, first, last in ((4, 1, 1), (6, 0, 2), (3, 2, 1), (30, 1, 2)):
        check_pick(torch, p, *drawn(torch, p, t, group * 10 + top), top, first, last, causal)


@pytest.mark.parametrize("cols", [255, 256, 257, 1024, 1025, 4096, 4100, 32768])
def test_picks_of_wide_tables(torch_gpu, cols):
    """Every kernel of the selection, at both ends of its widths; a short sequence beside the long one."""
    torch = torch_gpu
    long = cols * 16 - 5
    p = Pool(torch, 64, [0, 1, 3, 4], [long, 700, 33], 1, 16, 2, extra_cols=0, spare=0, seed=cols)
    q, qv, b, codes, scales = drawn(torch, p, "bf16", cols)
    for top, first, last in ((32, 1, 2), (256, 0, 1)):
        check_pick(torch, p, q, qv, b, codes, scales, top, first, last, True)


def test_picks_of_equal_scores(torch_gpu):
    """Bounds that are all alike, in halves alike, and queries of zeros: the lowest columns; and pages that are not there
    come last, the lower column first."""
    torch = torch_gpu
    p = Pool(torch, 128, [0, 2, 20], [900, 1500], 2, 16, 8, seed=3)
    q, qv, b, codes, scales = drawn(torch, p, "bf16", 3)
    codes[:], scales[:] = 5, 127
    for half in (False, True):
        if half:
            codes[::2, :, :, :7] = -6
            p.table[:, 3:50:2] = np.array([[-1], [2 ** 30]])
            p.upload()
        b.codes.copy_(torch.from_numpy(codes)), b.scales.copy_(torch.from_numpy(scales))
        for top in (5, 20, 48):
            check_pick(torch, p, q, qv, b, codes, scales, top, 1, 2, True)
    q.zero_()
    check_pick(torch, p, q, q.double().cpu().numpy(), b, codes, scales, 9, 0, 1, True)


def test_picks_at_the_ends_of_the_types(torch_gpu):
    """Scales from one end to the other, queries of the types' ends, subnormal ones, infinities and NaN."""
    torch = torch_gpu
    for t in ("bf16", "f16"):
        p = Pool(torch, 64, [0, 14, 20], [700, 900], 2, 16, 4, seed=4)
        q, qv, b, codes, scales = drawn(torch, p, t, 4, near=False)
        dt = q.dtype
        big = torch.finfo(dt).max
        for row, size in enumerate((big, -big, 2.0 ** -14, 2.0 ** -24, 2.0 ** -126, 2.0 ** -133, 127.0, 127.5, 254.0)):
            q[0, row] = (torch.sign(q[0, row].float()) * torch.rand_like(q[0, row].float()) * size).to(dt)
            q[0, row, 1, 3] = size
        q[0, 10, 0, 5], q[0, 11, 3, 7], q[0, 12, 2, 0] = math.inf, math.nan, -math.inf
        check_pick(torch, p, q, q.double().cpu().numpy(), b, codes, scales, 7, 1, 1, True)


def test_picks_of_strided_queries_and_bad_indexes(torch_gpu):
    """Queries inside fused rows, head-major; slots before 0, lengths past the table, rows past max_new and of no sequence."""
    import spl_sage as S
    from spl_sage import cache as C

    torch, d = torch_gpu, 128
    p = Pool(torch, d, [3, 53, 90, 95, 130], [30, 160, 5000, 500], 2, 16, 4, 140, seed=5, max_new=31)
    q, qv, b, codes, scales = drawn(torch, p, "bf16", 5)
    want = check_pick(torch, p, q, qv, b, codes, scales, 4, 1, 1, True)
    fused = torch.zeros(1, 140, 9, d, dtype=q.dtype, device="cuda")
    fused[:, :, 3:7] = q
    major = q.transpose(1, 2).contiguous()
    sa = S.SageAttention(torch.cuda.current_stream(), d)
    ws = sa.cache_pick_workspace(p.shape, 4)
    for view in (S.Tensor(fused[:, :, 3:7]), S.Tensor(major, S.Strides.bhtd(140, 4, d))):
        out = torch.full_like(want, -9)
        sa.cache_pick(ws, b, p.index, view, C.Picked(out), 1, 1, True)
        assert torch.equal(out, want)
    torch.cuda.synchronize()


def test_picks_in_windows(torch_gpu):
    """More scores than are kept at a time: rows in several turns, over sequences' ends."""
    from spl_sage._abi import lib

    torch = torch_gpu
    cols, kv = 20000, 2
    p = Pool(torch, 64, [0, 1, 900, 1700], [cols * 16, 200 * 16 + 899, 21 * 16 + 800], kv, 16, kv, extra_cols=0, spare=0, seed=6)
    f = lib()._ZN4sage11pick_windowEiii
    f.restype, f.argtypes = ctypes.c_int, [ctypes.c_int] * 3
    window = f(p.rows, kv, cols)
    assert 900 < window < p.rows  # (the second sequence's rows are in the first turn, the third's in both)
    q, qv, b, codes, scales = drawn(torch, p, "bf16", 6)
    import spl_sage as S
    from spl_sage import cache as C

    sa = S.SageAttention(torch.cuda.current_stream(), 64)
    ws = sa.cache_pick_workspace(p.shape, 12)
    out = torch.full((p.rows, kv, 12), -9, dtype=torch.int32, device="cuda")
    sa.cache_pick(ws, b, p.index, S.Tensor(q), C.Picked(out), 1, 1, True)
    got = out.cpu().numpy()
    rows = [0, 1, 2, 899, 900, window - 1, window, 1698, 1699]
    for row in rows:  # the oracle row by row
        seq = 0 if row < 1 else 1 if row < 900 else 2
        at = p.starts[seq]
        one = P.pick(qv[0][row:row + 1], codes[:, :, 0], codes[:, :, 1], scales, [0, 1],
                     [p.lengths[seq] - (p.starts[seq + 1] - at) + row - at + 1], p.table[seq:seq + 1], 16, p.pages, 12, 1, 1, True,
                     np.full((1, kv, 12), -9), 1)
        assert (got[row] == one[0]).all(), row


# ------------------------------------------------------------------ the attention


def attend(p, qv, picked, causal, scale, out):
    """float64 attention of every row over its picked columns (cache_rows.attend's results)."""
    rows, heads, _ = qv.shape
    kv, vv = p.values("k"), p.values("v")
    size, reach, count, top = np.zeros_like(out), np.zeros((rows, heads)), np.zeros((rows, heads)), np.zeros_like(out)
    group = heads // p.kv
    for b, length in enumerate(p.lengths):
        n = p.starts[b + 1] - p.starts[b]
        k, there = O.sequence(kv, p.table[b], length, p.page)
        v, _ = O.sequence(vv, p.table[b], length, p.page)
        for j in range(min(n, p.shape.max_new)):
            row = p.starts[b] + j
            if not 0 <= row < rows:
                continue
            limit = max(0, min(len(k), length - n + j + 1)) if causal else len(k)
            for g in range(p.kv):
                h = slice(g * group, (g + 1) * group)
                seen = there & P.seen_by(picked[row, g], limit, p.page, len(k))
                if not seen.any():
                    out[row, h] = 0
                    continue
                kk, vs = k[seen, g], v[seen, g]
                with np.errstate(invalid="ignore", over="ignore"):
                    x = (qv[row, h] @ kk.T) * scale
                    w = np.exp(x - x.max(-1, keepdims=True))
                    w /= w.sum(-1, keepdims=True)
                    out[row, h], size[row, h] = w @ vs, w @ np.abs(vs)
                    r = (np.abs(qv[row, h]) @ np.abs(kk).T) * abs(scale)
                reach[row, h] = np.where(np.isfinite(r), r, 0).max(-1)
                count[row, h], top[row, h] = seen.sum(), np.abs(vs).max(0)
    return out, size, reach, count, top


class Plan(ctypes.Structure):
    _fields_ = [("chunks", ctypes.c_bool), ("wide", ctypes.c_bool), ("splits", ctypes.c_int), ("parts", ctypes.c_int),
                ("lds", ctypes.c_uint), ("chunk_lds", ctypes.c_uint), ("part_rows", ctypes.c_uint64)]


def plan(shape, d, top):
    """How the call runs: the library's own rule."""
    from spl_sage._abi import lib

    f = lib()._ZN4sage11picked_planEiiiiiiiii
    f.restype, f.argtypes = Plan, [ctypes.c_int] * 9
    return f(d, shape.batch, shape.rows, shape.heads, shape.kv_heads, shape.max_new, shape.max_pages, shape.page_tokens, top)


def in_chunks(p, top, q_type):
    return plan(p.shape, p.d, top).chunks and not (p.d == 128 and q_type == "f16")


def fp16_weights(p, top, q_type, out_type):
    """Chunks of rows with a bf16 output round their weights to fp16 (where V's scales allow)."""
    return out_type == "bf16" and in_chunks(p, top, q_type)


def type_of(torch, x):
    return "bf16" if x.dtype == torch.bfloat16 else "f16"


def run_attend(torch, p, q, picked, out_type, causal=True, scale=None, out=None):
    import spl_sage as S
    from spl_sage import cache as C

    sa = S.SageAttention(torch.cuda.current_stream(), p.d)
    if out is None:
        out = torch.full(q.shape, 3.0, dtype=torch.bfloat16 if out_type == "bf16" else torch.float16, device="cuda")
    ws = sa.cache_pick_workspace(p.shape, picked.shape[2])
    sa.cache_attend_picked(ws, p.cache, p.index, C.Picked(ints(torch, picked)), S.Tensor(q), S.TensorMut(out), scale, causal)
    torch.cuda.synchronize()  # the workspace lives to the end of the call's work
    return out


def check_attend(torch, p, q, qv, picked, out_type, causal=True, scale=None, out=None):
    out = run_attend(torch, p, q, picked, out_type, causal, scale, out)
    s = 1 / math.sqrt(p.d) if scale is None else scale
    want, size, reach, count, top = attend(p, qv[0], picked, causal, s, np.full(qv[0].shape, 3.0))
    got = out[0].double().cpu().numpy()
    assert (np.isnan(got) == np.isnan(want)).all(), np.argwhere(np.isnan(got) != np.isnan(want))[:4]
    with np.errstate(invalid="ignore"):
        tol = tolerance(want, size, reach, count, top, p.d, out_type, fp16_weights(p, picked.shape[2], type_of(torch, q), out_type))
        # From 65520 on, half a step past its greatest value, fp16 has infinity.
        past = (np.abs(want) >= 65520 + tol) & (out_type == "f16")
        assert (got[past] == np.sign(want[past]) * np.inf).all()
        near = (np.abs(want) >= 65520 - tol) & (out_type == "f16")  # (either side of it)
        bad = ~(np.abs(got - want) <= tol) & ~np.isnan(want) & ~near
    assert not bad.any(), (int(bad.sum()), bad.size, np.argwhere(bad)[:4], got[bad][:4], want[bad][:4], tol[bad][:4])
    return out


def some_columns(rng, p, top, causal=True, shared=0.5, order="sorted"):
    """Columns for every row and KV head: some that a sequence's rows share, the row's last one, others its own."""
    out = np.full((p.rows, p.kv, top), -1, np.int32)
    for b, length in enumerate(p.lengths):
        n = p.starts[b + 1] - p.starts[b]
        common = rng.permutation(max(1, -(-max(length, 1) // p.page)))
        for j in range(n):
            row = p.starts[b] + j
            if not 0 <= row < p.rows:
                continue
            count = -(-max(0, length - n + j + 1 if causal else length) // p.page)
            for g in range(p.kv):
                mine = [c for c in common if c < count][:int(top * shared)]
                rest = [c for c in rng.permutation(count) if c not in mine]
                cols = ([count - 1] if count else []) + [c for c in mine + rest if c != count - 1]
                cols = cols[:top]
                out[row, g, :len(cols)] = sorted(cols) if order == "sorted" else cols
    return out


# (new rows, lengths, tokens a page, extra columns): steps, ragged chunks, one long sequence
SHAPES = {
    "steps": ([1, 1, 0, 1, 1], [200, 33, 7, 100, 1], 16, 1),
    "chunks": ([40, 3, 0, 70], [600, 3, 100, 330], 32, 2),
    "long": ([1, 2], [9000, 3001], 64, 0),
    "pages": ([5, 1], [1500, 700], 256, 0),
}


def shaped(torch, name, d, kv, group, seed=0, rows_behind=2):
    news, lengths, page, extra = SHAPES[name]
    starts = np.concatenate([[0], np.cumsum(news)]).tolist()
    return Pool(torch, d, starts, lengths, kv, page, kv * group, starts[-1] + rows_behind, extra_cols=extra, seed=seed)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("name", SHAPES)
@pytest.mark.parametrize("group", [1, 3, 4, 8, 16, 20])
@pytest.mark.parametrize("q_type,out_type,causal", [("bf16", "bf16", True), ("f16", "f16", False), ("f16", "bf16", True)])
def test_attention(torch_gpu, d, name, group, q_type, out_type, causal):
    torch = torch_gpu
    rng = np.random.default_rng(group + d)
    p = shaped(torch, name, d, 2, group, seed=group)
    spread(p, rng)
    for top in (1, 7, 40):
        q, qv = queries(torch, rng, p, q_type)
        check_attend(torch, p, q, qv, some_columns(rng, p, top, causal), out_type, causal)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("page", [16, 32, 64, 256])
@pytest.mark.parametrize("group", [1, 3, 8])
@pytest.mark.parametrize("q_type,out_type,causal", [("bf16", "bf16", True), ("f16", "f16", False), ("f16", "bf16", True), ("bf16", "f16", True)])
def test_attention_in_chunks(torch_gpu, d, page, group, q_type, out_type, causal):
    """Units of 32 columns, of which the shape allows enough to choose them: ragged chunks, pages of part of a step and more."""
    torch = torch_gpu
    rng = np.random.default_rng(group + d)
    p = Pool(torch, d, [0, 37, 38, 38, 103], [1300, 3, 100, 330], 2, page, 2 * group, 105, extra_cols=2, seed=group, max_new=1100)
    spread(p, rng)
    q, qv = queries(torch, rng, p, q_type)
    for top in (3, 14):
        assert plan(p.shape, d, top).chunks
        check_attend(torch, p, q, qv, some_columns(rng, p, top, causal), out_type, causal)


@pytest.mark.parametrize("d,page", [(64, 16), (128, 64)])
@pytest.mark.parametrize("rows", [258, 270, 512, 523])
def test_units_past_whole_rounds(torch_gpu, d, page, rows):
    """Just as many units as fill the chip, a few over, which are cut into parts, and hundreds."""
    torch = torch_gpu
    rng = np.random.default_rng(rows)
    p = Pool(torch, d, [0, rows - 250, rows - 249, rows], [rows + 100, 5, 600], 16, page, 64, rows + 3, seed=rows)
    spread(p, rng)
    q, qv = queries(torch, rng, p, "bf16")
    assert plan(p.shape, d, 8).chunks
    check_attend(torch, p, q, qv, some_columns(rng, p, 8), "bf16")


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("d", [64, 128])
def test_values_past_fp16_in_chunks(torch_gpu, d, page):
    """A block of V past fp16, and one of NaN, behind pages that fp16 holds: the weights go on as bf16 parts."""
    torch = torch_gpu
    rng = np.random.default_rng(d + page)
    p = Pool(torch, d, [0, 60, 100], [2000, 1500], 2, page, 8, extra_cols=0, seed=4, max_new=1100)
    spread(p, rng)
    for b, col in ((0, 1500 // page), (1, 700 // page)):
        p.host["v_scales"][p.table[b, col], :, 3, 1] = 165
        p.host["v_scales"][p.table[b, col], 1, 5, 0] = 90
    p.host["v_scales"][p.table[1, 1000 // page], 0, 7, d // 32 - 1] = 255
    p.upload()
    q, qv = queries(torch, rng, p, "bf16")
    picked = some_columns(rng, p, 40 if page == 16 else 14)
    assert plan(p.shape, d, picked.shape[2]).chunks
    check_attend(torch, p, q, qv, picked, "bf16")
    check_attend(torch, p, q, qv, picked, "f16")


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("name", ["steps", "chunks"])
def test_lists_in_any_order(torch_gpu, d, name):
    """Unsorted, with columns twice, ones that the row does not see, outside the table, holes, and lists of nothing: what
    the sorted list of the visible ones gives, bit for bit."""
    torch = torch_gpu
    rng = np.random.default_rng(d)
    p = shaped(torch, name, d, 2, 4)
    spread(p, rng)
    q, qv = queries(torch, rng, p, "bf16")
    plain = some_columns(rng, p, 9)
    plain[1] = -1  # a row that sees nothing
    cols = p.table.shape[1]
    want = check_attend(torch, p, q, qv, np.pad(plain, ((0, 0), (0, 0), (0, 8)), constant_values=-1), "bf16")
    odd = np.full((p.rows, p.kv, 17), -1, np.int32)
    for r in range(p.rows):
        for g in range(p.kv):
            x = plain[r, g]
            junk = [-1, -2 ** 31, cols, cols + 5, 2 ** 31 - 1, -7, x[0], x[-1]]
            odd[r, g] = rng.permutation(np.concatenate([x, junk]))
    assert torch.equal(want, check_attend(torch, p, q, qv, odd, "bf16"))
    odd = np.repeat(plain, 2, -1)[..., :18]
    assert torch.equal(want, run_attend(torch, p, q, odd, "bf16"))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("max_new,q_type", [(16, "bf16"), (16, "f16"), (2080, "bf16"), (2080, "f16")])
def test_the_widest_table_and_the_longest_lists(torch_gpu, d, max_new, q_type):
    """Lists of 256 pages that 16 rows share little of, under 32768 columns: the most that a unit's lists take of LDS, with
    eight waves and, as the shape allows units enough, with four."""
    torch = torch_gpu
    rng = np.random.default_rng(max_new)
    p = Pool(torch, d, [0, 16], [9000], 2, 16, 2, seed=3, extra_cols=32768 - 563, max_new=max_new)
    assert p.table.shape[1] == 32768 and not plan(p.shape, d, 256).chunks
    assert plan(p.shape, d, 256).wide == (max_new == 16)
    spread(p, rng)
    q, qv = queries(torch, rng, p, q_type)
    check_attend(torch, p, q, qv, some_columns(rng, p, 256, shared=0.1), "bf16")


def test_a_workspace_that_the_card_has_no_room_for(torch_gpu):
    """8 TB of partial rows: refused, and the next calls do not report it again."""
    import spl_sage as S
    from spl_sage import cache as C

    torch = torch_gpu
    rng = np.random.default_rng(0)
    sa = S.SageAttention(torch.cuda.current_stream(), 128)
    large = C.CacheShape(1, 4000000, 1, 64, 1, 4, 256, 4000)
    with pytest.raises(S.SageError, match="allocate pick workspace"):
        sa.cache_pick_workspace(large, 256)
    p = shaped(torch, "steps", 128, 2, 4)
    spread(p, rng)
    q, qv = queries(torch, rng, p, "bf16")
    check_attend(torch, p, q, qv, some_columns(rng, p, 7), "bf16")


@pytest.mark.parametrize("page", [16, 256])
def test_every_page_is_the_whole_attention(torch_gpu, page):
    """Rows that pick all their pages, up to the most that a pick can hold."""
    torch = torch_gpu
    rng = np.random.default_rng(page)
    p = Pool(torch, 64, [0, 1, 9], [255 * page + 3 if page == 16 else 2000, 70], 2, page, 4, seed=1)
    spread(p, rng)
    q, qv = queries(torch, rng, p, "bf16")
    every = np.full((p.rows, p.kv, 256), -1, np.int32)
    every[...] = np.where(np.arange(256) < p.table.shape[1], np.arange(256), -1)
    check_attend(torch, p, q, qv, every, "bf16")
    for softmax_scale in (0.0, -0.3, 2.0):
        check_attend(torch, p, q, qv, every, "bf16", scale=softmax_scale)


@pytest.mark.parametrize("name", ["steps", "chunks", "long"])
@pytest.mark.parametrize("d", [64, 128])
def test_nan_missing_pages_and_shifts(torch_gpu, name, d):
    """NaN blocks of V and K reach the rows that see them and no others; infinities' scales count as NaN; pages that are
    not there are not seen; V's exponents from small to large."""
    torch = torch_gpu
    rng = np.random.default_rng(d)
    p = shaped(torch, name, d, 2, 4, seed=2)
    spread(p, rng, v_shift=rng.integers(-30, 30, (1, 1, 1, d // 32)))
    bad = rng.random(p.host["v_scales"].shape) < 0.004
    p.host["v_scales"] = np.where(bad, rng.choice([253, 254, 255], bad.shape), p.host["v_scales"]).astype(np.uint8)
    kbad = rng.random(p.host["k_scales"].shape) < 0.0005
    p.host["k_scales"] = np.where(kbad, 255, p.host["k_scales"]).astype(np.uint8)
    p.table[0, 1], p.table[-1, 0], p.table[-1, 3 % p.table.shape[1]] = -1, p.pages, 2 ** 31 - 1
    p.upload()
    q, qv = queries(torch, rng, p, "bf16", sizes=(0.5, 1.0, 0.0, 2.0))
    picked = some_columns(rng, p, 12)
    host = dict(p.host)
    p.host["v_scales"] = np.where(p.host["v_scales"] >= 253, 255, p.host["v_scales"]).astype(np.uint8)  # as the call counts them
    out = run_attend(torch, p, q, picked, "bf16")
    want, size, reach, count, top = attend(p, qv[0], picked, True, 1 / math.sqrt(d), np.full(qv[0].shape, 3.0))
    got = out[0].double().cpu().numpy()
    assert (np.isnan(got) == np.isnan(want)).all() and np.isnan(want).any() and not np.isnan(want).all()
    with np.errstate(invalid="ignore"):
        tol = tolerance(want, size, reach, count, top, d, "bf16", fp16_weights(p, 12, "bf16", "bf16"))
        assert ((np.abs(got - want) <= tol) | np.isnan(want)).all()
    p.host = host


def test_in_place_strided_and_bad_indexes(torch_gpu):
    """out = q; rows before the first and behind the last sequence stay; slots before 0; lengths past the table; rows past max_new."""
    import spl_sage as S
    from spl_sage import cache as C

    torch, d = torch_gpu, 128
    rng = np.random.default_rng(7)
    p = Pool(torch, d, [3, 53, 90, 95, 130], [30, 160, 5000, 500], 2, 16, 4, 140, seed=5, max_new=31)
    spread(p, rng)
    q, qv = queries(torch, rng, p, "bf16")
    picked = rng.integers(-2, p.table.shape[1] + 1, (140, 2, 6)).astype(np.int32)
    want = check_attend(torch, p, q, qv, picked, "bf16")
    fused = torch.zeros(1, 140, 9, d, dtype=q.dtype, device="cuda")
    fused[:, :, 3:7] = q
    keep = fused.clone()
    sa = S.SageAttention(torch.cuda.current_stream(), d)
    ws = sa.cache_pick_workspace(p.shape, 6)
    part = fused[:, :, 3:7]
    sa.cache_attend_picked(ws, p.cache, p.index, C.Picked(ints(torch, picked)), S.Tensor(part), S.TensorMut(part))
    torch.cuda.synchronize()
    has = (want[0] != 3.0).any(-1).any(-1)
    assert torch.equal(part[0][has], want[0][has]) and torch.equal(part[0][~has], q[0][~has])
    assert torch.equal(fused[:, :, :3], keep[:, :, :3]) and torch.equal(fused[:, :, 7:], keep[:, :, 7:])
