"""Attention over the paged cache in float64 with a bound for every row of its
own (cache_oracle has the definitions), and pools whose softmax spreads over
many tokens, so that an error in any part of a sum shows."""
from __future__ import annotations

import math

import numpy as np

import cache_oracle as O
from cache_plans import plan
from test_gpu_cache import Pool, draw16

def attend(p, qv, causal, scale, out):
    """float64 attention of every row and head of the pool's sequences, into out [rows][heads][dim] where a row has
    one. Returns (out, sum p |v|, the largest sum |q k| scale of the row, its visible tokens, the largest |v|)."""
    rows, heads, _ = qv.shape
    kv, vv = p.values("k"), p.values("v")
    size, reach, count, top = np.zeros_like(out), np.zeros((rows, heads)), np.zeros((rows, heads)), np.zeros_like(out)
    group = heads // p.kv
    for b, length in enumerate(p.lengths):
        n = p.starts[b + 1] - p.starts[b]
        k, there = O.sequence(kv, p.table[b], length, p.page)
        v, _ = O.sequence(vv, p.table[b], length, p.page)
        slot = np.arange(len(k))
        for j in range(min(n, p.shape.max_new)):
            row = p.starts[b] + j
            if not 0 <= row < rows:
                continue
            seen = there & (slot <= (length - n + j if causal else length))
            if not seen.any():
                out[row] = 0
                continue
            for g in range(p.kv):
                h = slice(g * group, (g + 1) * group)
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


def tolerance(want, size, reach, count, top, d, out_type, fp16_weights):
    """How far an element may be. A logit is an fp32 sum of d exact products (whatever its order: d roundings, two a
    product of an fp16 query, of twice half a step in the MFMA) times a rounded factor, less the reference, into exp2.
    Its error is the weight's, and the weights' sum's. Either sum adds at most every second visible token in a row
    (a lane of the chunk kernel), and then the parts. For the second product a weight is rounded to two bf16 parts, or
    (fp16_weights) to fp16, 2^7 times as large: by half of 2^-24 where it is subnormal. The output is rounded once."""
    weight = O.HALF_STEP["f16"] if fp16_weights else O.HALF_STEP["bf16"] ** 2
    logit = (d + 6) * 2.0 ** -23 * reach
    sums = (count / 2 + 64) * 2.0 ** -24
    rel = (weight + 2 * logit + 2 * sums + 2.0 ** -20)[..., None]
    err = rel * size
    if fp16_weights:
        err = err + (count * 2.0 ** -32)[..., None] * top
    least = 2.0 ** -24 if out_type == "f16" else 0.0  # half an fp16 subnormal's step
    return err + O.HALF_STEP[out_type] * (np.abs(want) + err) + least + 1e-37


def spread(p, rng, v_shift=0, positive=False):
    """Keys whose logits are of the queries' size, and values whose tokens have sizes of their own and a mean, so that
    sums do not cancel (positive: none does). v_shift: more of V's exponents, an integer a block of a row."""
    dims = p.host["k_codes"].shape[:3]
    codes = lambda: rng.integers(0, 256, dims + (p.d // 2,)).astype(np.uint8)  # noqa: E731
    blocks = dims + (p.d // O.BLOCK,)
    p.host["k_codes"] = codes()
    p.host["k_scales"] = rng.integers(125, 127, blocks).astype(np.uint8)
    p.host["v_codes"] = codes() & (0x77 if positive else codes() | 0x77)  # half of the negative ones turned
    p.host["v_scales"] = (rng.integers(124, 128, dims + (1,)) + np.broadcast_to(v_shift, blocks)).astype(np.uint8)
    p.upload()


# A batch for each kernel and way through it: new rows, lengths, tokens a page, columns of the table, most new rows.
WAYS = {
    "whole": ([1, 5, 0, 2], [200, 33, 7, 100], 16, 16, None),
    "wide": ([1, 3, 0, 2], [900, 257, 0, 530], 64, 16, None),
    "shares": ([1, 2, 0, 3], [2900, 5, 77, 700], 256, 16, None),
    "chunk": ([40, 3, 0, 70], [1500, 3, 100, 330], 64, 48, 1100),  # tiles that the shape allows fill the chip: one split
    "splits": ([37, 3, 0, 70], [2500, 3, 100, 600], 128, 32, None),
}


def batch(torch, way, d, kv=2, group=4, seed=0, rows_behind=0, causal=True):
    """The way's batch; not causal: lengths of their own."""
    news, lengths, page, cols, most = WAYS[way]
    if not causal:
        lengths = [max(x - 7, 0) for x in lengths]
    starts = np.concatenate([[0], np.cumsum(news)]).tolist()
    width = -(-max(lengths) // page)
    p = Pool(torch, d, starts, lengths, kv, page, kv * group, starts[-1] + rows_behind, extra_cols=cols - width, seed=seed,
             max_new=most)
    assert plan(p.shape, d).kind == way
    return p


def queries(torch, rng, p, t, sizes=(0.0, 0.5, 1.0, 4.0)):
    """Queries [1][rows][heads][d] whose heads have sizes of their own: weights from all alike to one token's."""
    heads = p.shape.heads
    x, _ = draw16(torch, rng, (1, p.rows, heads, p.d), t)
    x *= torch.tensor([sizes[h % len(sizes)] for h in range(heads)], dtype=x.dtype, device="cuda")[:, None]
    return x, x.double().cpu().numpy()


def run(torch, p, q, out_type, causal=True, scale=None, out=None):
    import spl_sage as S

    sa = S.SageAttention(torch.cuda.current_stream(), p.d)
    if out is None:
        out = torch.full(q.shape, 3.0, dtype=torch.bfloat16 if out_type == "bf16" else torch.float16, device="cuda")
    ws = sa.cache_workspace(p.shape)
    sa.cache_attend(ws, p.cache, p.index, S.Tensor(q), S.TensorMut(out), scale, causal)
    torch.cuda.synchronize()  # the workspace lives to the end of the call's work
    return out


def check(torch, p, q, qv, out_type, causal=True, scale=None, out=None):
    """The call against float64 on every element; rows of no sequence keep their 3.0."""
    out = run(torch, p, q, out_type, causal, scale, out)
    s = 1 / math.sqrt(p.d) if scale is None else scale
    want, size, reach, count, top = attend(p, qv[0], causal, s, np.full(qv[0].shape, 3.0))
    got = out[0].double().cpu().numpy()
    assert (np.isnan(got) == np.isnan(want)).all(), np.argwhere(np.isnan(got) != np.isnan(want))[:4]
    with np.errstate(invalid="ignore"):
        tol = tolerance(want, size, reach, count, top, p.d, out_type, out_type == "bf16" and plan(p.shape, p.d).chunks)
        bad = ~(np.abs(got - want) <= tol) & ~np.isnan(want)
    assert not bad.any(), (int(bad.sum()), bad.size, np.argwhere(bad)[:4], got[bad][:4], want[bad][:4], tol[bad][:4])
    return out
