"""Attention over the paged 4-bit cache on the GPU against float64 numpy
(cache_oracle), within the bound that its roundings give (attend_tolerance)."""
from __future__ import annotations

import math

import numpy as np
import pytest

import cache_oracle as O
from test_gpu_cache import Pool, draw16, ints

pytestmark = pytest.mark.gpu


def run(torch, p, q, out_type, causal=True, scale=None, sa=None, ws=None):
    import spl_sage as S

    sa = sa or S.SageAttention(torch.cuda.current_stream(), p.d)
    ws = ws or sa.cache_workspace(p.shape)
    out = torch.full(q.shape, 3.0, dtype=torch.bfloat16 if out_type == "bf16" else torch.float16, device="cuda")
    sa.cache_attend(ws, p.cache, p.index, S.Tensor(q), S.TensorMut(out), scale, causal)
    return out


def check(torch, p, q, qv, out_type, causal=True, scale=None):
    out = run(torch, p, q, out_type, causal, scale)
    s = 1 / math.sqrt(p.d) if scale is None else scale
    want, size, reach = O.attend(qv[0], p.values("k"), p.values("v"), p.starts, p.lengths, p.table, p.page, causal, s,
                                 np.full(qv[0].shape, 3.0), p.shape.max_new)
    got = out[0].double().cpu().numpy()
    assert (np.isnan(got) == np.isnan(want)).all(), np.argwhere(np.isnan(got) != np.isnan(want))[:4]
    tol = O.attend_tolerance(want, size, reach, p.d, out_type)
    bad = (np.abs(got - want) > tol) & ~np.isnan(want)
    assert not bad.any(), (int(bad.sum()), bad.size, np.argwhere(bad)[:4], got[bad][:4], want[bad][:4], tol[bad][:4])
    return out


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("t", ["bf16", "f16"])
@pytest.mark.parametrize("kv,group", [(1, 1), (2, 3), (1, 8), (2, 16), (1, 17)])
def test_single_tokens(torch_gpu, d, t, kv, group):
    """A decoding step over lengths around every tile's edge."""
    rng = np.random.default_rng(d + kv + group)
    lengths = [1, 2, 15, 16, 17, 63, 64, 65, 255, 256, 257, 511, 600, 0]
    starts = list(range(len(lengths) + 1))
    for page in (16, 256):
        p = Pool(torch_gpu, d, starts, lengths, kv, page, kv * group, seed=group)
        q, qv = draw16(torch_gpu, rng, (1, len(lengths), kv * group, d), t)
        check(torch_gpu, p, q, qv, t)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("t,out_t", [("bf16", "bf16"), ("bf16", "f16"), ("f16", "f16"), ("f16", "bf16")])
@pytest.mark.parametrize("kv,group", [(2, 1), (1, 5), (1, 8)])
def test_chunks(torch_gpu, d, causal, t, out_t, kv, group):
    """Several new rows a sequence: none, a few, more than a tile; the first of them the sequence's first tokens; rows
    behind the last sequence stay."""
    rng = np.random.default_rng(d + group)
    news, past = [3, 0, 40, 1, 130, 17], [0, 9, 100, 300, 0, 64]
    starts = np.concatenate([[0], np.cumsum(news)]).tolist()
    lengths = [a + b for a, b in zip(news, past)]
    if not causal:
        lengths = [33, 0, 129, 1, 64, 0]
    p = Pool(torch_gpu, d, starts, lengths, kv, 32, kv * group, starts[-1] + 5, seed=group)
    q, qv = draw16(torch_gpu, rng, (1, starts[-1] + 5, kv * group, d), t)
    out = check(torch_gpu, p, q, qv, out_t, causal)
    assert (out[0, starts[-1]:] == 3.0).all()


@pytest.mark.parametrize("d", [64, 128])
def test_long_sequences(torch_gpu, d):
    """Keys split over many workgroups, of sequences of very different lengths."""
    rng = np.random.default_rng(d)
    lengths = [9001, 3, 2048, 513, 0, 4097]
    p = Pool(torch_gpu, d, list(range(7)), lengths, 2, 64, 8, seed=1)
    q, qv = draw16(torch_gpu, rng, (1, 6, 8, d), "bf16", 2.0)
    a = check(torch_gpu, p, q, qv, "bf16")
    assert torch_gpu.equal(a, run(torch_gpu, p, q, "bf16"))  # the same bits again


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("batch", [63, 64, 65, 200])
def test_many_sequences(torch_gpu, d, batch):
    """Sequences without rows or tokens among others of up to 1500: the shares of the work begin and end everywhere."""
    rng = np.random.default_rng(batch)
    news = rng.integers(0, 3, batch)
    news[:2] = 0
    starts = np.concatenate([[0], np.cumsum(news)]).tolist()
    lengths = np.where(rng.random(batch) < 0.3, rng.integers(0, 4, batch), rng.integers(0, 1500, batch)).tolist()
    lengths[5] = 1500
    p = Pool(torch_gpu, d, starts, lengths, 2, 64, 4, seed=batch)
    q, qv = draw16(torch_gpu, rng, (1, starts[-1], 4, d), "bf16")
    a = check(torch_gpu, p, q, qv, "bf16")
    assert torch_gpu.equal(a, run(torch_gpu, p, q, "bf16"))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("t", ["bf16", "f16"])
@pytest.mark.parametrize("batch", [128, 130])
def test_short_sequences(torch_gpu, d, t, batch):
    """Up to 1000 tokens, a workgroup a unit: 256 units, and a few more than the chip has CUs."""
    rng = np.random.default_rng(batch)
    lengths = rng.integers(1, 1000, batch)
    lengths[:6] = [1000, 256, 257, 512, 513, 0]
    p = Pool(torch_gpu, d, list(range(batch + 1)), lengths.tolist(), 2, 16, 6, extra_cols=0, seed=batch)
    q, qv = draw16(torch_gpu, rng, (1, batch, 6, d), t)
    check(torch_gpu, p, q, qv, t)


@pytest.mark.parametrize("d", [64, 128])
def test_a_long_prefix_under_a_few_rows(torch_gpu, d):
    """Chunks whose keys are split over workgroups, and more rows than a workgroup's columns."""
    rng = np.random.default_rng(d)
    p = Pool(torch_gpu, d, [0, 33, 34, 200], [6001, 700, 1500], 1, 128, 3, seed=1)
    q, qv = draw16(torch_gpu, rng, (1, 200, 3, d), "f16", 2.0)
    a = check(torch_gpu, p, q, qv, "f16")
    assert torch_gpu.equal(a, run(torch_gpu, p, q, "f16"))


@pytest.mark.parametrize("scale", [0.0, -0.3, 3.0])
def test_softmax_scale(torch_gpu, scale):
    rng = np.random.default_rng(2)
    for more in (0, 60):  # few columns, and a chunk
        p = Pool(torch_gpu, 128, [0, 3 + more, 5 + more], [70, 200], 2, 16, 4, seed=1)
        q, qv = draw16(torch_gpu, rng, (1, 5 + more, 4, 128), "f16")
        check(torch_gpu, p, q, qv, "f16", scale=scale)


def test_views_in_place_and_types(torch_gpu):
    """Queries inside fused rows, head-major outputs, the output over the queries, each type with each."""
    import spl_sage as S

    torch, d, heads = torch_gpu, 64, 6
    rng = np.random.default_rng(2)
    p = Pool(torch, d, [0, 3, 40], [70, 900], 2, 16, heads, seed=1)
    sa = S.SageAttention(torch.cuda.current_stream(), d)
    ws = sa.cache_workspace(p.shape)
    for t in ("bf16", "f16"):
        fused, fv = draw16(torch, rng, (1, 40, heads + 4, d), t)
        q, qv = fused[:, :, 2:2 + heads], fv[:, :, 2:2 + heads]
        for ot in ("bf16", "f16"):
            want = check(torch, p, q, qv, ot)
        want = run(torch, p, q, t)
        out = torch.zeros(1, heads, 40, d, dtype=q.dtype, device="cuda")
        sa.cache_attend(ws, p.cache, p.index, S.Tensor(q), S.TensorMut(out, S.Strides.bhtd(40, heads, d)))
        assert torch.equal(out.transpose(1, 2), want)
        keep = fused.clone()
        sa.cache_attend(ws, p.cache, p.index, S.Tensor(q), S.TensorMut(q))
        assert torch.equal(q, want)
        assert torch.equal(fused[:, :, :2], keep[:, :, :2]) and torch.equal(fused[:, :, 8:], keep[:, :, 8:])


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("new", [1, 40])
def test_nan_and_infinity_stay_where_they_are_seen(torch_gpu, d, new):
    """NaN blocks in K and V, of tokens that some rows, all rows or no row sees, and behind every length."""
    rng = np.random.default_rng(d)
    lengths = [100, 300, 90, 64]
    starts = [0, new, 2 * new, 3 * new, 4 * new]
    p = Pool(torch_gpu, d, starts, lengths, 2, 16, 6, seed=5)

    def mark(b, slot, side, head, block):
        p.host[side + "_scales"][p.table[b, slot // 16], head, slot % 16, block] = 255

    for b, n in enumerate(lengths):  # everything behind the lengths
        for slot in range(n, p.table.shape[1] * 16):
            for side in "kv":
                p.host[side + "_scales"][p.table[b, slot // 16], :, slot % 16] = 255
    mark(0, 99, "v", 1, 1)        # only the last row sees it
    mark(0, 95, "k", 0, 0)
    mark(1, 10, "v", 0, d // 32 - 1)
    mark(2, 80, "v", 1, 0)
    p.upload()
    q, qv = draw16(torch_gpu, rng, (1, 4 * new, 6, d), "bf16")
    q[0, -1, 2, 3] = math.inf
    q[0, 0, 1, 0] = math.nan
    qv = q.double().cpu().numpy()
    out = check(torch_gpu, p, q, qv, "bf16")
    assert 0 < torch_gpu.isnan(out).sum() < out.numel() // 2


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("new", [1, 40])
def test_scales_past_the_range(torch_gpu, d, new):
    """V blocks of 2^126 and 2^127, whose values can be infinities: nothing where they are masked (memory that was never
    written holds them), NaN to the rows that see them."""
    rng = np.random.default_rng(d)
    lengths = [100, 300, 90]
    p = Pool(torch_gpu, d, [0, new, 2 * new, 3 * new], lengths, 2, 16, 6, seed=5)
    for b, n in enumerate(lengths):
        for slot in range(n, p.table.shape[1] * 16):
            for side in "kv":
                block = p.host[side + "_scales"][p.table[b, slot // 16], :, slot % 16]
                block[:] = rng.integers(253, 255, block.shape)
    p.host["v_scales"][p.table[0, 99 // 16], 1, 99 % 16, 1] = 254  # only the last row sees it
    p.upload()
    q, qv = draw16(torch_gpu, rng, (1, 3 * new, 6, d), "bf16")
    out = run(torch_gpu, p, q, "bf16")
    p.host["v_scales"][p.host["v_scales"] >= 253] = 255
    p.upload()
    want = check(torch_gpu, p, q, qv, "bf16")
    assert torch_gpu.equal(torch_gpu.isnan(out), torch_gpu.isnan(want)) and 0 < torch_gpu.isnan(out).sum() <= 3 * 32
    assert torch_gpu.equal(out.nan_to_num(7.0), want.nan_to_num(7.0))


def test_pages_that_the_pool_does_not_have(torch_gpu):
    """Their tokens are not attended to; a sequence with no other page gives zeros."""
    rng = np.random.default_rng(1)
    p = Pool(torch_gpu, 128, [0, 2, 4, 5], [400, 40, 200], 1, 16, 4, seed=1)
    p.table[0, 3:7] = -1
    p.table[0, 20] = p.pages
    p.table[1, :] = 2 ** 31 - 1
    p.table[2, 0] = -2 ** 31
    p.lengths[2] = p.table.shape[1] * 16 + 50  # and slots past the page table
    p.upload()
    q, qv = draw16(torch_gpu, rng, (1, 5, 4, 128), "bf16")
    out = check(torch_gpu, p, q, qv, "bf16", causal=False)
    assert (out[0, 2:4] == 0).all()
    check(torch_gpu, p, q, qv, "bf16")


def test_rows_past_max_new_and_odd_starts(torch_gpu):
    """Rows past max_new, sequences past the packed rows, lengths below the new rows (their first rows see nothing)."""
    rng = np.random.default_rng(1)
    p = Pool(torch_gpu, 64, [2, 12, 12, 30], [6, 50, 33], 2, 32, 2, rows=25, seed=1, max_new=8)
    q, qv = draw16(torch_gpu, rng, (1, 25, 2, 64), "f16")
    out = check(torch_gpu, p, q, qv, "f16")
    assert (out[0, :2] == 3.0).all() and (out[0, 10:12] == 3.0).all() and (out[0, 2:6] == 0).all()


def test_offset_channels(torch_gpu):
    """Keys with a large offset in some channels, which the softmax cancels: differences of logits survive."""
    rng = np.random.default_rng(3)
    d, n = 128, 700
    p = Pool(torch_gpu, d, [0, 4], [n], 1, 64, 4, seed=1)
    x = rng.standard_normal((p.pages, 1, 64, d)) + np.where(np.arange(d) % 32 == 5, 200.0, 0.0)
    p.host["k_codes"], p.host["k_scales"], _ = O.quantise(x)
    p.upload()
    q, qv = draw16(torch_gpu, rng, (1, 4, 4, d), "bf16")
    check(torch_gpu, p, q, qv, "bf16")


def test_offsets_past_31_bits(torch_gpu):
    """A pool of more than 2^31 code bytes: its last pages."""
    torch, d = torch_gpu, 128
    from spl_sage import cache as C
    import spl_sage as S

    pages, kv, page = 17000, 8, 256  # 17000 * 8 * 256 * 64 bytes = 2.23e9
    shape = C.CacheShape(1, 2, 2, 8, kv, pages, page, 2)
    cache = C.PagedCache.new(shape, d)
    sa = S.SageAttention(torch.cuda.current_stream(), d)
    rng = np.random.default_rng(0)
    table = np.array([[pages - 1, pages - 2]], np.int32)
    index = C.CacheIndex(ints(torch, [0, 2]), ints(torch, [300]), ints(torch, table))
    fill = C.CacheShape(1, 300, 300, 8, kv, pages, page, 2)
    k, kv_ = draw16(torch, rng, (1, 300, kv, d), "bf16")
    v, vv_ = draw16(torch, rng, (1, 300, kv, d), "bf16")
    whole = C.CacheIndex(ints(torch, [0, 300]), ints(torch, [300]), ints(torch, table))
    sa.cache_append(cache.with_shape(fill), whole, S.Tensor(k), S.Tensor(v))
    kb, vb = torch.empty_like(k), torch.empty_like(v)
    sa.cache_read(cache.with_shape(fill), whole, S.TensorMut(kb), S.TensorMut(vb))
    kq, vq = O.quantise(kv_[0])[2], O.quantise(vv_[0])[2]
    assert (kb[0].double().cpu().numpy() == kq).all() and (vb[0].double().cpu().numpy() == vq).all()
    q, qv = draw16(torch, rng, (1, 2, 8, d), "bf16")
    out = torch.empty_like(q)
    sa.cache_attend(sa.cache_workspace(shape), cache, index, S.Tensor(q), S.TensorMut(out))
    pad = lambda x: np.concatenate([x, np.zeros((212, kv, d))]).reshape(2, page, kv, d).transpose(0, 2, 1, 3)  # noqa: E731
    want, size, reach = O.attend(qv[0], pad(kq), pad(vq), [0, 2], [300], np.array([[0, 1]]), page, True, 1 / math.sqrt(d),
                                 np.zeros((2, 8, d)))
    assert (np.abs(out[0].double().cpu().numpy() - want) <= O.attend_tolerance(want, size, reach, d, "bf16")).all()
    assert not cache.k_codes[:pages - 2].any()
