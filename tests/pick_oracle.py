"""Plain forms, in numpy and 64 bits, of a step's index, rotary axes, page bounds, picked pages and the attention over
them: the oracle of their tests, from the definitions in include/sage_hip.h, one request, page or row at a time."""
from __future__ import annotations

import math

import numpy as np

import cache_oracle as O


# ------------------------------------------------------------------ a step's index


def tables(news, past, ring, state, page_table, page_tokens, rows, pages_there=1 << 31):
    """What sage_cache_tables leaves: a dict of its outputs, the ring and the page table among them."""
    cap, cols = len(ring), page_table.shape[1]
    ring, table = list(ring), page_table.copy()
    head, count = int(state[0]) % (1 << 32) % cap, min(max(int(state[1]), 0), cap)
    pages = lambda n: -(-n // page_tokens)  # noqa: E731
    past = [max(int(p), 0) for p in past]
    fresh = [0 if n < 0 else pages(p + n) - pages(p) for n, p in zip(news, past)]
    over = [0 if n < 0 else max(0, pages(p + n) - cols) for n, p in zip(news, past)]
    missing = max(0, sum(fresh) - count) + sum(over)
    more = max(0, sum(max(n, 0) for n in news) - rows)
    good = not missing and not more
    out = {"positions": [0] * rows, "slots": [-1] * rows, "sequences": [-1] * rows}
    starts, lengths, given = [0], [], []
    for b, (n, p) in enumerate(zip(news, past)):
        if n < 0:
            given += [int(x) for x in page_table[b, :min(pages(p), cols)]]
            lengths.append(0)
            starts.append(starts[-1])
            continue
        n = n if good else 0
        for t in range(p, p + n):
            if t // page_tokens >= pages(p) and t % page_tokens == 0:  # the first token of a new page
                table[b, t // page_tokens] = ring[(head + sum(fresh[:b]) + t // page_tokens - pages(p)) % cap]
            row = starts[-1] + t - p
            out["positions"][row], out["sequences"][row] = t, b
            page = int(table[b, t // page_tokens])
            if 0 <= page < pages_there:
                out["slots"][row] = page * page_tokens + t % page_tokens
        lengths.append(p + n)
        starts.append(starts[-1] + n)
    given = given[:cap - count]
    for i, x in enumerate(given):
        ring[(head + count + i) % cap] = x
    taken = sum(fresh) if good else 0
    return {"starts": starts, "lengths": lengths, "page_table": table.tolist(), "ring": ring,
            "state": [(head + taken) % cap, count - taken + len(given), min(missing, 2 ** 31 - 1), min(more, 2 ** 31 - 1)], **out}


# ------------------------------------------------------------------ rotary axes


def axis_of(sections, dealt):
    """(axis, place among the axis's pairs) of each pair."""
    if not dealt:
        return [(a, j) for a, n in enumerate(sections) for j in range(n)]
    out, got = [], [0] * len(sections)
    while len(out) < sum(sections):
        for a, n in enumerate(sections):
            if got[a] < n:
                out.append((a, got[a]))
                got[a] += 1
    return out


def channels(sections, layout):
    """The two channels of each pair: layout "Half", "Pairs" or "AxisHalf"."""
    n = sum(sections)
    if layout == "Half":
        return np.arange(n), np.arange(n) + n
    if layout == "Pairs":
        return 2 * np.arange(n), 2 * np.arange(n) + 1
    first = [2 * sum(sections[:a]) + j for a, s in enumerate(sections) for j in range(s)]
    return np.array(first), np.array([c + s for c, s in zip(first, np.repeat(sections, sections))])


def rotate_axes(x, cos_sin, positions, sections, layout, dealt, transpose=False):
    """x [rows][heads][dim] float64, cos_sin [positions][pairs][2], positions [axes][rows]; the channels of an axis whose
    position the table does not hold become NaN."""
    y = np.array(x, np.float64)
    axis = np.array([a for a, _ in axis_of(sections, dealt)])
    pos = np.asarray(positions)[axis]  # [pair][row]
    ok = (pos >= 0) & (pos < len(cos_sin))
    cs = np.asarray(cos_sin, np.float64)[np.where(ok, pos, 0), np.arange(len(axis))[:, None]]
    cs = np.where(ok[..., None], cs, np.nan).transpose(1, 0, 2)[:, None]
    c, s = cs[..., 0], -cs[..., 1] if transpose else cs[..., 1]
    i, j = channels(sections, layout)
    a, b = y[..., i].copy(), y[..., j].copy()
    y[..., i], y[..., j] = a * c - b * s, b * c + a * s
    return y


# ------------------------------------------------------------------ bounds and picks


def page_bounds(codes, scales):
    """(hi, lo [dim], E) of one page's tokens of one KV head: codes [tokens][dim/2], scales [tokens][dim/32]."""
    whole = scales != 255
    top = max(1, int(scales[whole].max())) if whole.any() else 1
    with np.errstate(invalid="ignore"):
        x = O.values(codes, np.where(whole, scales, 127)) * 16
        x = np.where(np.repeat(whole, O.BLOCK, -1), x * 2.0 ** (127.0 - top), np.nan)
    bad = np.isnan(x).any(0)
    hi, lo = np.ceil(np.where(bad, 0, x.max(0))), np.floor(np.where(bad, 0, x.min(0)))
    return np.where(bad, 127, hi).astype(np.int8), np.where(bad, -127, lo).astype(np.int8), top


def touched(starts, lengths, page_tokens, cols, max_new):
    """(sequence, column, tokens held) of the pages that hold a row of the step."""
    for b, length in enumerate(lengths):
        n = starts[b + 1] - starts[b]
        slots = [t for t in range(length - n, length - n + min(n, max_new)) if 0 <= t < cols * page_tokens]
        for col in sorted({t // page_tokens for t in slots}):
            yield b, col, min(min(length, cols * page_tokens) - col * page_tokens, page_tokens)


def query_codes(q):
    """A group's queries [heads][dim] as whole numbers."""
    if not np.isfinite(q).all() or not np.abs(q).max():
        return np.zeros_like(q)
    e = 126
    while e > -126 and np.abs(q).max() * 2.0 ** e > 127:
        e -= 1
    return np.rint(q * 2.0 ** e)


def pick(q, hi, lo, scales, starts, lengths, page_table, page_tokens, pages, top, first, last, causal, out, max_new):
    """The picked columns, into out [rows][kv_heads][top] where a row has them. q [rows][heads][dim]; hi, lo
    [pages][kv_heads][dim], scales [pages][kv_heads]."""
    rows, heads, _ = q.shape
    kv, cols = hi.shape[1], page_table.shape[1]
    group = heads // kv
    for b, length in enumerate(lengths):
        n = starts[b + 1] - starts[b]
        length = max(0, min(length, cols * page_tokens))
        for j in range(min(n, max_new)):
            row = starts[b] + j
            if not 0 <= row < rows:
                continue
            limit = max(0, min(length, lengths[b] - n + j + 1)) if causal else length
            count = -(-limit // page_tokens)
            for g in range(kv):
                u = query_codes(q[row, g * group:(g + 1) * group])
                score = []
                for col in range(count):
                    p = int(page_table[b, col])
                    if col < first or col >= count - last:
                        score.append(math.inf)
                    elif not 0 <= p < pages:
                        score.append(-math.inf)
                    else:
                        s = np.where(u > 0, u * hi[p, g].astype(float), u * lo[p, g].astype(float)).sum(-1).max()
                        score.append(s * 2.0 ** (max(1, min(int(scales[p, g]), 228)) - 127))
                best = sorted(sorted(range(count), key=lambda col: -score[col])[:top])
                out[row, g] = best + [-1] * (top - len(best))
    return out


def scores(q, hi, lo, scales, table, pages):
    """Scores of some rows' queries [rows][heads][dim] for the pages of a sequence's table [columns]: [rows][kv_heads]
    [columns], -inf where there is no page. All at once, in 32 bits, which hold them exactly."""
    rows, kv = len(q), hi.shape[1]
    x = q.reshape(rows, kv, -1, q.shape[2])
    top = np.abs(x).max((2, 3), keepdims=True)
    with np.errstate(divide="ignore"):
        e = np.clip(np.floor(np.log2(127 / top)) + 1, -126, 126)
    for _ in range(2):
        e = np.where((top * 2.0 ** e > 127) & (e > -126), e - 1, e)
    u = np.rint(x * 2.0 ** e).astype(np.float32)
    there = (table >= 0) & (table < pages)
    at = np.where(there, table, 0)
    out = np.empty((rows, kv, len(table)))
    for g in range(kv):
        s = np.maximum(u[:, g], 0) @ hi[at, g].T.astype(np.float32) + np.minimum(u[:, g], 0) @ lo[at, g].T.astype(np.float32)
        out[:, g] = s.max(1).astype(float) * 2.0 ** (np.clip(scales[at, g].astype(int), 1, 228) - 127.0)
    return np.where(there, out, -np.inf)


def greatest(score, top, first, last):
    """The list of one row and KV head from the scores of the pages that it sees."""
    col = np.arange(len(score))
    score = np.where((col < first) | (col >= len(score) - last), np.inf, score)
    best = np.sort(np.argsort(-score, kind="stable")[:top])
    return np.concatenate([best, np.full(top - len(best), -1)])


def seen_by(picked, limit, page_tokens, slots):
    """Which of `slots` slots a row sees under its picked columns."""
    seen = np.zeros(slots, bool)
    for col in map(int, picked):
        if 0 <= col and col * page_tokens < min(slots, limit):
            seen[col * page_tokens:min((col + 1) * page_tokens, limit)] = True
    return seen
