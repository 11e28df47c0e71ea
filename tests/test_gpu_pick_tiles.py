"""Every kernel that makes a pick, against the whole lists of the oracle: one launch with 1, 2 and 4 tiles of rows a
workgroup and keys for 256 to 2048 columns, and two launches, whose scores are made by tiles of several rows."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

import pick_oracle as P
from test_gpu_cache import Pool
from test_gpu_pick import drawn

GROUPS = [1, 2, 3, 4, 7, 8, 16]
COLUMNS = [200, 500, 1000, 2000, 2100]
# New rows of a sequence that the shape allows, columns of the page table, heads of a KV head.
CASES = ([(1100, c, g) for c in COLUMNS for g in GROUPS] + [(130, c, g) for c in COLUMNS for g in (7, 16)] +
         [(40, c, g) for c in COLUMNS for g in (1, 2, 4, 8, 16)] + [(12, 1000, 1), (12, 1000, 2)] +
         # (all of the keys that 64 KB, and that a wave's lanes, hold)
         [(1100, 1024, 4), (1100, 512, 2), (1100, 2048, 3), (1100, 2048, 8), (130, 2048, 16), (40, 1024, 1)])


def tiles(batch, group, kv_heads, max_new, max_pages):
    """Tiles of 16 columns a workgroup where one launch serves the call, else 0: the library's own rule."""
    import torch  # noqa: F401  (its runtime first: the library joins it)
    from spl_sage._abi import lib

    f = lib()._ZN4sage10pick_tilesEiiiii
    f.restype, f.argtypes = ctypes.c_int, [ctypes.c_int] * 5
    return f(batch, group, kv_heads, max_new, max_pages)


def way(most, cols, group):
    """Tiles, columns that a wave's keys are for, columns of a tile that a row takes (their binary logarithm)."""
    return tiles(4, group, 2, most, cols), next(w for w in (256, 512, 1024, 2048, 4096) if cols <= w), (group - 1).bit_length()


def test_the_cases_reach_every_kernel():
    reached = {way(*case) for case in CASES}
    assert {r[:2] for r in reached} >= {(t, w) for t in (1, 2, 4) for w in (256, 512, 1024, 2048)}
    assert reached >= {(0, 4096, slots) for slots in range(5)}
    assert {r[2] for r in reached if r[0] == 4} == {1, 2, 3, 4} and {r[2] for r in reached if r[0] == 1} == {0, 1, 2, 3, 4}


def test_the_oracle_of_all_rows_is_the_oracle_of_one():
    rng = np.random.default_rng(0)
    pages, kv, d, rows = 90, 2, 64, 9
    codes = rng.integers(-9, 10, (2, pages, kv, d))
    hi, lo = codes.max(0), codes.min(0)
    scales = rng.integers(126, 129, (pages, kv))
    table = rng.integers(-1, pages + 1, (1, 70))
    for heads in (2, 6):
        q = rng.standard_normal((rows, heads, d))
        q[4] = 0
        want = P.pick(q, hi, lo, scales, [0, rows], [1111], table, 16, pages, 20, 2, 3, True, np.zeros((rows, kv, 20), int), rows)
        score = P.scores(q, hi, lo, scales, table[0], pages)
        for j in range(rows):
            for g in range(kv):
                assert (P.greatest(score[j, g, :-(-(1111 - rows + j + 1) // 16)], 20, 2, 3) == want[j, g]).all()
    assert P.greatest(score[0, 0, :2], 4, 0, 1).tolist() == [0, 1, -1, -1]


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("most,cols,group", CASES)
def test_lists_of_every_kernel(torch_gpu, d, most, cols, group):
    """Chunks that end inside a tile and fill several workgroups, sequences of one row and of none beside them; lists that
    fit a lane's keys and longer ones, of which all but one page are always picked, and a page that is not there."""
    import spl_sage as S
    from spl_sage import cache as C

    torch, kv = torch_gpu, 2
    news = (min(most, 70), 1, 0, min(most, 39))
    lengths = [cols * 16 - 3, cols * 8 + 1, 7, 39 + 5 * 16]
    starts = np.concatenate([[0], np.cumsum(news)]).tolist()
    p = Pool(torch, d, starts, lengths, kv, 16, kv * group, starts[-1] + 2, extra_cols=0, seed=cols + group, max_new=most)
    p.table[0, 5] = -1
    p.upload()
    q, qv, b, codes, scales = drawn(torch, p, "bf16" if (group + cols // 100) % 2 else "f16", cols + group)
    sa = S.SageAttention(torch.cuda.current_stream(), d)
    want = {}  # row: its slots, its scores
    for seq, n in enumerate(news):
        if not n:
            continue
        here = slice(starts[seq], starts[seq] + n)
        all_rows = P.scores(qv[0][here], codes[:, :, 0], codes[:, :, 1], scales, p.table[seq], p.pages)
        want.update({starts[seq] + j: (lengths[seq] - n + j + 1, all_rows[j]) for j in range(n)})
    for top, first, last in ((32, 1, 2), (64, 0, 1), (4, 2, 1), (150, 1, 1)):
        ws = sa.cache_pick_workspace(p.shape, top)
        out = torch.full((p.rows, kv, top), -9, dtype=torch.int32, device="cuda")
        sa.cache_pick(ws, b, p.index, S.Tensor(q), C.Picked(out), first, last, True)
        got = out.cpu().numpy()
        assert (got[starts[-1]:] == -9).all()
        for row, (seen, score) in want.items():
            for g in range(kv):
                lists = P.greatest(score[g, :-(-seen // 16)], top, first, last)
                assert (got[row, g] == lists).all(), (row, g, top, np.argwhere(got[row, g] != lists)[:3])
