"""Plain forms of the rotary and paged-cache operators in float64 numpy: the
oracle of their tests. Everything is computed from the definitions in
include/sage_hip.h, one sequence at a time."""
from __future__ import annotations

import math

import numpy as np

LEVELS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
BLOCK = 32
# Half a step of each type, relative to the value: torch.finfo(t).eps / 2.
HALF_STEP = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}


def rotate(x, cos_sin, positions, rot, pairs, transpose=False):
    """x [rows][heads][dim] float64; cos_sin [positions][rot/2][2]; the rotated channels of rows whose position is
    outside become NaN."""
    y = np.array(x, np.float64)
    pos = np.asarray(positions)
    ok = (pos >= 0) & (pos < len(cos_sin))
    cs = np.asarray(cos_sin, np.float64)[np.where(ok, pos, 0)]
    c, s = np.where(ok[:, None], cs[..., 0], np.nan)[:, None], np.where(ok[:, None], cs[..., 1], np.nan)[:, None]
    s = -s if transpose else s
    i0 = np.arange(0, rot, 2) if pairs else np.arange(rot // 2)
    i1 = i0 + 1 if pairs else i0 + rot // 2
    a, b = y[..., i0].copy(), y[..., i1].copy()
    y[..., i0], y[..., i1] = a * c - b * s, b * c + a * s
    return y


def angles(rot, positions, base=10000.0, kind="none", factor=1.0, original=0.0, fast=32.0, slow=1.0):
    """[positions][rot/2] angles, from the definitions."""
    i = np.arange(rot // 2)
    if kind == "ntk":
        base = base * factor ** (rot / (rot - 2))
    w = base ** (-2.0 * i / rot)
    if kind == "linear":
        w = w / factor
    if kind == "yarn":
        turns = original * w / (2 * math.pi)
        g = np.clip((turns - slow) / (fast - slow), 0, 1)
        w = g * w + (1 - g) * w / factor
    return np.arange(positions)[:, None] * w


def quantise(x):
    """x [..., dim] -> (code bytes, scale bytes, values). 64-bit throughout."""
    y = np.asarray(x, np.float64)
    y = y.reshape(*y.shape[:-1], -1, BLOCK)
    with np.errstate(invalid="ignore", over="ignore"):
        bad = ~np.isfinite(y).all(-1)
        z = np.where(bad[..., None], 0.0, y)
        top = np.abs(z).max(-1)
        m, e = np.frexp(top)  # top = m 2^e; top <= 6 2^k <=> m 2^(e - k) <= 6
        k = np.where(m <= 0.75, e - 3, e - 2)
        k = np.where(top > 0, np.maximum(k, -126), -126)
        u = np.abs(z) / np.exp2(k)[..., None]
    d = np.abs(u[..., None] - LEVELS)
    near = d.min(-1, keepdims=True)
    tie = d == near  # one or two neighbours: the even code
    idx = np.arange(8)
    code = np.where(tie & (idx % 2 == 0), idx, -1).max(-1)
    code = np.where(tie.sum(-1) == 2, code, tie.argmax(-1))
    code = np.where(np.signbit(z), code + 8, code)
    code = np.where(bad[..., None], 0, code).astype(np.uint8)
    scale = np.where(bad, 255, k + 127).astype(np.uint8)
    flat = code.reshape(*code.shape[:-2], -1)
    codes = (flat[..., 0::2] | (flat[..., 1::2] << 4)).astype(np.uint8)
    return codes, scale, values(codes, scale)


def values(codes, scales):
    n = np.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], -1)
    v = np.where(n >= 8, -LEVELS[n & 7], LEVELS[n & 7])
    s = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    return v * np.repeat(s, BLOCK, -1)


def cells(starts, lengths, page_table, page_tokens, pages, rows):
    """(row, page, token in it) of every row of every sequence that has a place in the pool; page -1: none."""
    out = []
    for b in range(len(lengths)):
        n = starts[b + 1] - starts[b]
        for j in range(n):
            row, slot = starts[b] + j, lengths[b] - n + j
            if not 0 <= row < rows:
                continue
            page = -1
            if 0 <= slot < page_table.shape[1] * page_tokens:
                page = int(page_table[b, slot // page_tokens])
                page = page if 0 <= page < pages else -1
            out.append((row, page, slot % page_tokens, slot))
    return out


def sequence(cache_values, page_table_row, length, page_tokens):
    """[slots][kv_heads][dim] of a sequence's tokens and which of them exist. cache_values [pages][kv][page_tokens][dim]."""
    pages = cache_values.shape[0]
    length = max(0, min(length, len(page_table_row) * page_tokens))
    t = np.arange(length)
    p = page_table_row[t // page_tokens]
    there = (p >= 0) & (p < pages)
    return cache_values[np.where(there, p, 0), :, t % page_tokens], there


def attend(q, kv, vv, starts, lengths, page_table, page_tokens, causal, scale, out, max_new=1 << 30):
    """float64 attention. q [rows][heads][dim]; kv, vv [pages][kv_heads][page_tokens][dim]; out is filled where a row
    belongs to a sequence. Returns (out, bound on sum p |v| / l, the largest sum |q k| scale)."""
    rows, heads, d = q.shape
    kvh = kv.shape[1]
    size, reach = np.zeros_like(out), 0.0
    for b in range(len(lengths)):
        n = starts[b + 1] - starts[b]
        k, there = sequence(kv, page_table[b], lengths[b], page_tokens)
        v, _ = sequence(vv, page_table[b], lengths[b], page_tokens)
        for j in range(min(n, max_new)):
            row = starts[b] + j
            if not 0 <= row < rows:
                continue
            last = lengths[b] - n + j if causal else lengths[b]
            seen = there & (np.arange(len(k)) <= last)
            for h in range(heads):
                g = h // (heads // kvh)
                if not seen.any():
                    out[row, h] = 0
                    continue
                with np.errstate(invalid="ignore", over="ignore"):
                    kk, vs = k[seen, g], v[seen, g]
                    x = (kk @ q[row, h]) * scale
                    p = np.exp(x - x.max())
                    p = p / p.sum()
                    out[row, h] = p @ vs
                    size[row, h] = p @ np.abs(vs)
                    r = np.abs(kk) @ np.abs(q[row, h]) * abs(scale)
                    reach = max(reach, float(np.nanmax(r))) if np.isfinite(r).any() else reach
    return out, size, reach


def attend_tolerance(want, size, reach, d, out_type):
    """How far an element may be: each probability is rounded to bf16 once (half a step of it; the sum of the
    probabilities is not), for an fp16 output to two bf16 parts (half a step of half a step), each logit is an fp32 sum of d products (and of a second part of the query) in base 2, the
    output is an fp32 sum and is rounded once to its type."""
    logit = 4 * d * 2.0 ** -24 * reach  # absolute error of a logit; p is off by its exponential, and so is their sum
    p = (HALF_STEP["bf16"] if out_type == "bf16" else HALF_STEP["bf16"] ** 2) + 2 * logit + 2.0 ** -20
    least = 2.0 ** -24 if out_type == "f16" else 0.0  # half an fp16 subnormal's step
    return p * size + HALF_STEP[out_type] * (np.abs(want) + p * size) + least + 1e-30
