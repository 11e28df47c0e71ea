"""Every kernel of the attention over the paged cache, named by the library's own
rule (cache_rows.WAYS), against float64 with a bound for each row: types, masks,
groups, pages, scales, NaN, pages that are not there, rows past the limits, views,
and joins of parts that all carry weight."""
from __future__ import annotations

import math

import numpy as np
import pytest

import cache_rows as R
from cache_plans import plan
from test_gpu_cache import Pool, draw16

pytestmark = pytest.mark.gpu

# The kernels whose sequences are cut, or whose rows fill tiles of 128 columns.
LARGE = ["shares", "chunk", "splits"]


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("t,out_t", [("bf16", "bf16"), ("f16", "bf16"), ("bf16", "f16"), ("f16", "f16")])
@pytest.mark.parametrize("way", list(R.WAYS))
def test_no_mask(torch_gpu, way, d, t, out_t):
    rng = np.random.default_rng(d + 1)
    p = R.batch(torch_gpu, way, d, causal=False, rows_behind=3, seed=1)
    R.spread(p, rng)
    q, qv = R.queries(torch_gpu, rng, p, t)
    out = R.check(torch_gpu, p, q, qv, out_t, causal=False)
    assert (out[0, p.starts[-1]:] == 3.0).all()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("kv,group", [(1, 1), (3, 1), (2, 3), (1, 8), (8, 4), (1, 17)])
@pytest.mark.parametrize("way", LARGE)
def test_heads(torch_gpu, way, d, kv, group):
    """KV heads (the grid's fastest) and groups, which set a tile's columns: chunks of more than one tile of them."""
    rng = np.random.default_rng(kv * 100 + group)
    news, lengths, page, cols, most = R.WAYS[way]
    if way == "chunk":  # tiles to fill the chip whatever the heads
        most = 128 * 90 // (kv * group) * kv
    if way == "splits":
        news = [x * 4 // group + 1 for x in news]
    if way == "shares":
        news = [min(x, 64 // group) for x in news]
    starts = np.concatenate([[0], np.cumsum(news)]).tolist()
    p = Pool(torch_gpu, d, starts, [max(n, x) for n, x in zip(news, lengths)], kv, page, kv * group, seed=2, max_new=most,
             extra_cols=cols - -(-max(lengths) // page))
    assert plan(p.shape, d).kind == way
    R.spread(p, rng)
    t, out_t = [("bf16", "bf16"), ("f16", "bf16"), ("bf16", "f16"), ("f16", "f16")][(kv + group) % 4]
    q, qv = R.queries(torch_gpu, rng, p, t, (0.5, 0.0, 1.0, 3.0, 0.25))
    R.check(torch_gpu, p, q, qv, out_t)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("most,kind", [(1100, "chunk"), (70, "splits"), (16, "shares")])
def test_pages(torch_gpu, d, page, most, kind):
    """Lengths around the ends of pages and tiles."""
    rng = np.random.default_rng(page)
    news = [min(x, most) for x in (70, 2, 33, 17)]
    lengths = [page * 5 + 1, page - 1, 511, 64 * 9]
    starts = np.concatenate([[0], np.cumsum(news)]).tolist()
    p = Pool(torch_gpu, d, starts, [max(n, x) for n, x in zip(news, lengths)], 2, page, 8, seed=3, max_new=most,
             extra_cols=4096 // page - -(-max(*lengths, *news) // page))
    assert plan(p.shape, d).kind == kind
    R.spread(p, rng)
    q, qv = R.queries(torch_gpu, rng, p, "bf16")
    R.check(torch_gpu, p, q, qv, "bf16")


@pytest.mark.parametrize("scale", [0.0, -0.3, 1.0])
@pytest.mark.parametrize("t", ["bf16", "f16"])
@pytest.mark.parametrize("way", LARGE)
def test_softmax_scales(torch_gpu, way, t, scale):
    rng = np.random.default_rng(4)
    p = R.batch(torch_gpu, way, 128, seed=4)
    R.spread(p, rng)
    q, qv = R.queries(torch_gpu, rng, p, t, (0.1, 0.5, 1.0, 0.0))
    R.check(torch_gpu, p, q, qv, t, scale=scale)


def marked(p, b, slot, side, head, block, byte):
    p.host[side + "_scales"][p.table[b, slot // p.page], head, slot % p.page, block] = byte


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("t", ["bf16", "f16"])
@pytest.mark.parametrize("way", LARGE)
def test_nan_where_it_is_seen(torch_gpu, way, d, t):
    """NaN blocks, and V blocks of 2^126 and 2^127, of tokens that all rows, some rows or no row sees; NaN and infinity in
    queries: NaN reaches the rows, heads and channels that see it and no other."""
    rng = np.random.default_rng(d)
    p = R.batch(torch_gpu, way, d, seed=5)
    R.spread(p, rng)
    for b, n in enumerate(p.lengths):  # behind every length
        for slot in range(n, min(n + 300, p.table.shape[1] * p.page)):
            for side in "kv":
                marked(p, b, slot, side, slice(None), slice(None), 255 if slot % 2 else 253 + (slot // 2) % 2)
    n, new = p.lengths[0], p.starts[1] - p.starts[0]
    last = d // 32 - 1
    marked(p, 0, n - 1, "v", 1, last, 255)       # the last row of the sequence alone
    marked(p, 0, 130, "v", 0, 0, 253)            # all its rows
    marked(p, 0, n - new // 2 - 1, "k", 1, 0, 255)  # half its rows, in one KV head
    marked(p, 3, p.lengths[3] - 1, "v", 0, last, 254)
    p.upload()
    q, _ = R.queries(torch_gpu, rng, p, t)
    q[0, -1, 2, 3] = math.inf
    q[0, p.starts[1], 5, 0] = math.nan
    out = R.run(torch_gpu, p, q, t)
    v = p.host["v_scales"]
    v[v >= 253] = 255  # what they count as
    p.upload()
    want = R.check(torch_gpu, p, q, q.double().cpu().numpy(), t)
    assert torch_gpu.equal(torch_gpu.isnan(out), torch_gpu.isnan(want))
    assert torch_gpu.equal(out.nan_to_num(7.0), want.nan_to_num(7.0))
    assert 0 < torch_gpu.isnan(out).sum() < out.numel() // 2


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("way", LARGE)
def test_pages_that_are_not_there(torch_gpu, way, d, causal):
    """Their tokens are not attended to, nor slots past the page table; a sequence of nothing else gives zeros."""
    rng = np.random.default_rng(6)
    p = R.batch(torch_gpu, way, d, seed=6)
    R.spread(p, rng)
    cols = p.table.shape[1]
    p.table[0, 1::3] = -1
    p.table[0, 2] = p.pages
    p.table[1, :] = [2 ** 31 - 1, -2 ** 31][way == "chunk"]
    p.table[3, 0] = -2 ** 31
    p.lengths[3] = cols * p.page + 50
    p.upload()
    q, qv = R.queries(torch_gpu, rng, p, "bf16")
    out = R.check(torch_gpu, p, q, qv, "bf16", causal=causal)
    assert (out[0, p.starts[1]:p.starts[2]] == 0).all()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("kind,most,cols", [("shares", 8, 16), ("chunk", 5600, 9), ("splits", 45, 16)])
def test_rows_past_the_limits(torch_gpu, kind, most, cols, d):
    """Rows past max_new and past the packed rows, rows before the first sequence, lengths below the new rows (the first
    of them see nothing), sequences without rows or tokens."""
    rng = np.random.default_rng(7)
    starts, lengths = [2, 62, 62, 130, 131, 190], [40, 50, 400, 0, 75]
    p = Pool(torch_gpu, d, starts, lengths, 2, 256, 4, rows=170, extra_cols=cols - 2, seed=7, max_new=most)
    assert plan(p.shape, d).kind == kind
    R.spread(p, rng)
    q, qv = R.queries(torch_gpu, rng, p, "f16")
    out = R.check(torch_gpu, p, q, qv, "f16")
    assert (out[0, :2] == 3.0).all() and (out[0, 130] == 0).all()
    assert (out[0, 2:min(most, 20) + 2] == 0).all()
    if most < 60:
        assert (out[0, 2 + most:62] == 3.0).all()


@pytest.mark.parametrize("t", ["bf16", "f16"])
@pytest.mark.parametrize("way", LARGE)
def test_views_and_in_place(torch_gpu, way, t):
    """Queries inside fused rows, head-major outputs, the output over the queries: the same bits."""
    import spl_sage as S

    torch, d = torch_gpu, 64
    rng = np.random.default_rng(8)
    p = R.batch(torch, way, d, seed=8)
    R.spread(p, rng)
    rows, heads = p.rows, p.shape.heads
    fused, fv = draw16(torch, rng, (1, rows, heads + 4, d), t)
    q, qv = fused[:, :, 2:2 + heads], fv[:, :, 2:2 + heads]
    want = R.check(torch, p, q, qv, t)
    assert torch.equal(want, R.run(torch, p, q, t))  # the same bits again
    R.check(torch, p, q, qv, "f16" if t == "bf16" else "bf16")
    sa = S.SageAttention(torch.cuda.current_stream(), d)
    ws = sa.cache_workspace(p.shape)
    out = torch.zeros(1, heads, rows, d, dtype=q.dtype, device="cuda")
    sa.cache_attend(ws, p.cache, p.index, S.Tensor(q), S.TensorMut(out, S.Strides.bhtd(rows, heads, d)))
    assert torch.equal(out.transpose(1, 2), want)
    keep = fused.clone()
    sa.cache_attend(ws, p.cache, p.index, S.Tensor(q), S.TensorMut(q))
    assert torch.equal(q, want)
    assert torch.equal(fused[:, :, :2], keep[:, :, :2]) and torch.equal(fused[:, :, 2 + heads:], keep[:, :, 2 + heads:])


# Joins: sequences, new rows, KV heads, group and columns of 256 tokens, and whether a workgroup joins a column's
# parts (SHARE) or a group of lanes does.
JOINS = {
    "shares, a workgroup": ([9001, 3, 2048, 513, 0, 4097], 1, 2, 4, 40),
    "shares, lanes": ([3000, 1, 257, 2048] * 5, 2, 2, 4, 16),
    "splits, a workgroup": ([9001, 700, 4096], 40, 2, 4, 40),
    "splits, lanes": ([4000, 300, 2600], 90, 2, 4, 16),
}


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("t", ["bf16", "f16"])
@pytest.mark.parametrize("name", list(JOINS))
def test_joins_of_parts_that_all_carry_weight(torch_gpu, name, t, d):
    """Positive values under weights all alike, nearly alike and uneven: a part left out or weighed wrongly shows in
    every channel."""
    lengths, new, kv, group, cols = JOINS[name]
    rng = np.random.default_rng(9)
    news = [min(new, x) for x in lengths]
    starts = np.concatenate([[0], np.cumsum(news)]).tolist()
    p = Pool(torch_gpu, d, starts, lengths, kv, 256, kv * group, extra_cols=cols - -(-max(lengths) // 256), seed=9,
             max_new=new)
    plan_ = plan(p.shape, d)
    assert plan_.kind == name.split(",")[0]
    joined = (plan_.wgs > 8 and new * kv * group * len(lengths) <= 2048) if plan_.chunks else \
        -(-new * group // 16) * kv * len(lengths) <= 32
    assert joined == ("workgroup" in name)
    R.spread(p, rng, positive=True)
    q, qv = R.queries(torch_gpu, rng, p, t, (0.0, 0.1, 1.0, 2.0))
    a = R.check(torch_gpu, p, q, qv, t)
    assert torch_gpu.equal(a, R.run(torch_gpu, p, q, t))  # the same bits again
