"""The rotary and cache operators as a serving program runs them together:
prompts in chunks and single tokens against one float64 attention over the
whole sequences, a cached prefix read back for sage_forward, steps captured
into graphs, and calls on several streams."""
from __future__ import annotations

import math
import subprocess
from pathlib import Path

import numpy as np
import pytest

import cache_oracle as O
from test_gpu_cache import Pool, draw16, ints

pytestmark = pytest.mark.gpu


class Model:
    """One attention layer's projections of a batch of sequences, in full, and what the cache makes of them."""

    def __init__(self, torch, d, heads, kv, lengths, t="bf16", seed=0, rot=None):
        from spl_sage import rotary as R

        self.torch, self.d, self.heads, self.kv, self.t = torch, d, heads, kv, t
        self.rot = rot or d
        rng = np.random.default_rng(seed)
        self.rows = [draw16(torch, rng, (n, heads + 2 * kv, d), t) for n in lengths]
        self.table = R.RotaryTable.new(self.rot, max(lengths) + 1)
        self.device_table = self.table.upload()
        self.want = []
        for x, xv in self.rows:
            pos = np.arange(len(xv))
            qk = O.rotate(xv[:, :heads + kv], self.table.cos_sin, pos, self.rot, False)
            qk = torch.from_numpy(qk).to(x.dtype).double().numpy()  # rotated rows are 16-bit rows
            k, v = O.quantise(qk[:, heads:])[2], O.quantise(xv[:, heads + kv:])[2]
            n = len(xv)
            pad = -n % 16
            page = lambda y: np.concatenate([y, np.zeros((pad, kv, d))]).reshape(-1, 16, kv, d).transpose(0, 2, 1, 3)  # noqa: E731
            tab = np.arange((n + pad) // 16)[None]
            self.want.append(O.attend(qk[:, :heads], page(k), page(v), [0, n], [n], tab, 16, True, 1 / math.sqrt(d),
                                      np.zeros((n, heads, d))))


def step_rows(m, begin, end):
    """The packed fused rows of tokens begin[b] .. end[b] of every sequence, and the rows' starts."""
    parts = [x[b:e] for (x, _), b, e in zip(m.rows, begin, end)]
    return m.torch.cat(parts), np.concatenate([[0], np.cumsum([len(p) for p in parts])]).tolist()


@pytest.mark.parametrize("d,heads,kv,t", [(128, 8, 2, "bf16"), (64, 6, 6, "f16")])
def test_prompts_then_tokens(torch_gpu, d, heads, kv, t):
    """Prompts of odd lengths go in as two chunks, then token by token; every row's output is the causal attention of its
    whole sequence over the cached values."""
    import spl_sage as S
    from spl_sage import cache as C
    from spl_sage import rotary as R

    torch = torch_gpu
    lengths = [150, 33, 97]
    m = Model(torch, d, heads, kv, lengths, t)
    sa = S.SageAttention(torch.cuda.current_stream(), d)
    page = 32
    cols = -(-max(lengths) // page)
    pages = len(lengths) * cols + 2
    table = np.random.default_rng(1).permutation(pages)[:len(lengths) * cols].reshape(len(lengths), cols)
    table = ints(torch, table)
    at = [0, 0, 0]
    ends = [[100, 0, 61], [140, 25, 90]] + [[min(140 + i, 150), min(25 + i, 33), min(90 + i, 97)] for i in range(1, 11)]
    pool = C.PagedCache.new(C.CacheShape(3, 1, 1, heads, kv, pages, page, cols), d)
    for end in ends:
        fused, starts = step_rows(m, at, end)
        rows = starts[-1]
        shape = C.CacheShape(3, rows, max(e - b for b, e in zip(at, end)), heads, kv, pages, page, cols)
        cache = pool.with_shape(shape)
        index = C.CacheIndex(ints(torch, starts), ints(torch, end), table)
        x = fused[None]
        q, k, v = x[:, :, :heads], x[:, :, heads:heads + kv], x[:, :, heads + kv:]
        qr, out = torch.empty(1, rows, heads, d, dtype=x.dtype, device="cuda"), torch.empty(1, rows, heads, d, dtype=x.dtype, device="cuda")
        sa.cache_append(cache, index, S.Tensor(k), S.Tensor(v), R.Rotary(m.device_table, m.rot), S.Tensor(q), S.TensorMut(qr))
        sa.cache_attend(sa.cache_workspace(shape), cache, index, S.Tensor(qr), S.TensorMut(out))
        got = out[0].double().cpu().numpy()
        for b in range(3):
            want, size, reach = m.want[b]
            w, s = want[at[b]:end[b]], size[at[b]:end[b]]
            tol = O.attend_tolerance(w, s, reach, d, t)
            bad = np.abs(got[starts[b]:starts[b + 1]] - w) > tol
            assert not bad.any(), (b, at[b], end[b], int(bad.sum()))
        at = end


def test_a_cached_prefix_feeds_sage_forward(torch_gpu):
    """Cached keys and values read back are the operands of the INT8 / FP8 forward: bit for bit the call on the values
    that the codes stand for."""
    import spl_sage as S

    torch, d, n, heads, kv = torch_gpu, 128, 512, 8, 2
    rng = np.random.default_rng(3)
    sa = S.SageAttention(torch.cuda.current_stream(), d)
    p = Pool(torch, d, [0, n], [n], kv, 64, heads, seed=3)
    q, _ = draw16(torch, rng, (1, n, heads, d), "bf16")
    k, kv_ = draw16(torch, rng, (1, n, kv, d), "bf16")
    v, vv_ = draw16(torch, rng, (1, n, kv, d), "bf16")
    sa.cache_append(p.cache, p.index, S.Tensor(k), S.Tensor(v))
    kb, vb = torch.empty_like(k), torch.empty_like(k)
    sa.cache_read(p.cache, p.index, S.TensorMut(kb), S.TensorMut(vb))
    values = [torch.from_numpy(O.quantise(x)[2]).to(torch.bfloat16).cuda() for x in (kv_, vv_)]
    ws = sa.workspace(S.Shape(1, heads, n, kv))
    outs = []
    for kk, vv in ((kb, vb), values):
        outs.append(torch.empty_like(q))
        sa.forward(ws, S.Tensor(q), S.Tensor(kk), S.Tensor(vv), S.TensorMut(outs[-1]), S.Options(causal=True))
    assert torch.equal(*outs)


def steps_of(torch, d, seed, lengths, heads, kv, page, new, cols, pages):
    """Inputs of one step at these lengths (device tensors)."""
    rng = np.random.default_rng(seed)
    table = rng.permutation(pages)[:len(lengths) * cols].reshape(len(lengths), cols)
    rows = len(lengths) * new
    x, _ = draw16(torch, rng, (1, rows, heads + 2 * kv, d), "bf16")
    return {"x": x, "lengths": ints(torch, lengths), "table": ints(torch, table),
            "starts": ints(torch, np.arange(len(lengths) + 1) * new)}


@pytest.mark.parametrize("new,tokens", [(1, 4096), (1, 512), (40, 4096)])
def test_a_captured_step_serves_every_step(torch_gpu, new, tokens):
    """append (queries rotated) and attend captured once; replays with other lengths, pages, starts and rows equal the
    eager calls bit for bit, with eager work in between, and two graphs that share a workspace in order."""
    import spl_sage as S
    from spl_sage import cache as C
    from spl_sage import rotary as R

    torch, d, heads, kv, page = torch_gpu, 128, 8, 2, 64
    cols, batch = tokens // page, 3
    pages = batch * cols + 1
    shape = C.CacheShape(batch, batch * new, new, heads, kv, pages, page, cols)
    table = R.RotaryTable.new(d, tokens).upload()
    s = torch.cuda.Stream()
    sa = S.SageAttention(s, d)
    ws = sa.cache_workspace(shape)
    eager = S.SageAttention(torch.cuda.current_stream(), d)
    eager_ws = eager.cache_workspace(shape)
    pool, pool2 = C.PagedCache.new(shape, d), C.PagedCache.new(shape, d)
    for name in ("k_codes", "v_codes", "k_scales", "v_scales"):
        fill = torch.randint(0, 256, getattr(pool, name).shape, dtype=torch.uint8, device="cuda") if "codes" in name else \
            torch.randint(118, 130, getattr(pool, name).shape, device="cuda").to(torch.uint8)
        getattr(pool, name).copy_(fill)
        getattr(pool2, name).copy_(fill)

    def call(ctx, w, cache, i, out):
        x = i["x"]
        q, k, v = x[:, :, :heads], x[:, :, heads:heads + kv], x[:, :, heads + kv:]
        index = C.CacheIndex(i["starts"], i["lengths"], i["table"])
        ctx.cache_append(cache, index, S.Tensor(k), S.Tensor(v), R.Rotary(table, d), S.Tensor(q), S.TensorMut(out))
        ctx.cache_attend(w, cache, index, S.Tensor(out), S.TensorMut(out))

    hold = steps_of(torch, d, 0, [tokens, tokens // 2, new], heads, kv, page, new, cols, pages)
    out = torch.zeros(1, batch * new, heads, d, dtype=torch.bfloat16, device="cuda")
    graphs = []
    torch.cuda.synchronize()
    for _ in range(2):  # two graphs over one workspace
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            call(sa, ws, pool, hold, out)
        graphs.append(g)
    for n, lengths in enumerate([[tokens, 700 % tokens + new, new], [new, new, new], [tokens, tokens, tokens],
                                 [new + 1, tokens - 3, 333], [tokens, tokens // 2, new]]):
        i = steps_of(torch, d, n + 1, lengths, heads, kv, page, new, cols, pages)
        want = torch.zeros_like(out)
        call(eager, eager_ws, pool2, i, want)
        for k in hold:
            hold[k].copy_(i[k])
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            graphs[n % 2].replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), n
        for name in ("k_codes", "v_codes", "k_scales", "v_scales"):
            assert torch.equal(getattr(pool, name), getattr(pool2, name))


def test_calls_on_two_streams(torch_gpu):
    """Two contexts with workspaces of their own on two streams at once, over one pool: each gives what it gives alone."""
    import spl_sage as S

    torch = torch_gpu
    rng = np.random.default_rng(1)
    p = Pool(torch, 64, [0, 1, 2, 3], [5000, 40, 3000], 4, 64, 8, seed=1)
    p2 = Pool(torch, 64, [0, 30, 31], [2500, 900], 4, 64, 8, seed=1)
    jobs = []
    for pool, t in ((p, "bf16"), (p2, "f16")):
        q, _ = draw16(torch, rng, (1, pool.rows, 8, 64), t)
        s = torch.cuda.Stream()
        sa = S.SageAttention(s, 64)
        jobs.append((pool, q, s, sa, sa.cache_workspace(pool.shape)))
    alone = []
    torch.cuda.synchronize()
    for pool, q, s, sa, ws in jobs:
        out = torch.empty_like(q)
        sa.cache_attend(ws, pool.cache, pool.index, S.Tensor(q), S.TensorMut(out))
        torch.cuda.synchronize()
        alone.append(out)
    outs = [[torch.empty_like(q) for _ in range(8)] for _, q, *_ in jobs]
    torch.cuda.synchronize()
    for r in range(8):
        for (pool, q, s, sa, ws), o in zip(jobs, outs):
            sa.cache_attend(ws, pool.cache, pool.index, S.Tensor(q), S.TensorMut(o[r]))
    torch.cuda.synchronize()
    for want, o in zip(alone, outs):
        assert all(torch.equal(x, want) for x in o)


def test_more_sequences_than_shares(torch_gpu):
    """600 sequences of up to 1500 tokens, some without rows: whole units."""
    from test_gpu_cache_attend import check

    torch = torch_gpu
    rng = np.random.default_rng(2)
    news = rng.integers(0, 2, 600)
    starts = np.concatenate([[0], np.cumsum(news)]).tolist()
    lengths = rng.integers(0, 60, 600).tolist()
    lengths[::97] = [1500] * len(lengths[::97])
    p = Pool(torch, 64, starts, lengths, 1, 256, 2, seed=2)
    q, qv = draw16(torch, rng, (1, starts[-1], 2, 64), "bf16")
    check(torch, p, q, qv, "bf16")


def test_refused_on_the_gpu(torch_gpu):
    """A refusal leaves the outputs as they were, and the next call works."""
    import spl_sage as S

    torch = torch_gpu
    rng = np.random.default_rng(2)
    p = Pool(torch, 64, [0, 2], [30], 1, 16, 2, seed=2)
    q, _ = draw16(torch, rng, (1, 2, 2, 64), "bf16")
    sa, other = S.SageAttention(torch.cuda.current_stream(), 64), S.SageAttention(torch.cuda.current_stream(), 128)
    ws = sa.cache_workspace(p.shape)
    out = torch.full_like(q, 3.0)
    with pytest.raises(S.SageError, match="made for head dim 64"):
        other.cache_attend(ws, p.cache, p.index, S.Tensor(q), S.TensorMut(out))
    with pytest.raises(S.SageError, match="output: buffer holds"):
        sa.cache_attend(ws, p.cache, p.index, S.Tensor(q), S.TensorMut(out[:, :1].clone()))
    with pytest.raises(S.SageError, match="bf16 or fp16"):
        sa.cache_attend(ws, p.cache, p.index, S.Tensor(q.float()), S.TensorMut(out))
    from spl_sage import cache as C

    host = C.CacheIndex(p.index.starts.cpu(), p.index.lengths.cpu(), p.index.page_table.cpu())
    with pytest.raises(S.SageError, match="in host memory"):
        sa.cache_attend(ws, p.cache, host, S.Tensor(q), S.TensorMut(out))
    with pytest.raises(S.SageError, match="in host memory"):
        sa.cache_attend(ws, p.cache, p.index, S.Tensor(q.cpu()), S.TensorMut(out))
    torch.cuda.synchronize()
    assert (out == 3.0).all()
    sa.cache_attend(ws, p.cache, p.index, S.Tensor(q), S.TensorMut(out))
    assert (out != 3.0).any(-1).all()  # every row is written


def test_cpp_calls(torch_gpu):
    """The same calls through include/spl_sage.hpp (tests/cpp/gpu_cache.cpp)."""
    exe = Path(__file__).resolve().parent / "cpp" / "bin" / "gpu_cache"
    assert exe.exists(), f"{exe} is not built; run `python __graft_entry__.py` (build)"
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and "0 failure(s)" in r.stdout, r.stdout + r.stderr


@pytest.mark.parametrize("d,heads,kv", [(64, 6, 6), (128, 8, 2)])
def test_an_encoder_s_states_beside_a_decoder_s_steps(torch_gpu, d, heads, kv):
    """A decoder whose layer attends to its own cached tokens and to an encoder's cached states, in one pool: a prompt of
    more rows than a tile (the chunk kernel, under a wide page table), then single tokens."""
    import spl_sage as S
    from cache_plans import plan
    from spl_sage import cache as C
    from spl_sage import rotary as R

    torch, t, page, cols = torch_gpu, "bf16", 64, 40
    rng = np.random.default_rng(4)
    states, prompts = [301, 64, 7], [130, 20, 77]
    m = Model(torch, d, heads, kv, [n + 3 for n in prompts], t, seed=4)
    sa = S.SageAttention(torch.cuda.current_stream(), d)
    pages = 6 * cols
    tables = np.random.default_rng(5).permutation(pages).reshape(2, 3, cols)
    own, other = ints(torch, tables[0]), ints(torch, tables[1])
    # The encoder's states, once: no positions.
    x, xv = draw16(torch, rng, (sum(states), 2 * kv, d), t)
    at = np.concatenate([[0], np.cumsum(states)]).tolist()
    pool = C.PagedCache.new(C.CacheShape(3, at[-1], max(states), heads, kv, pages, page, cols), d)
    sa.cache_append(pool, C.CacheIndex(ints(torch, at), ints(torch, states), other), S.Tensor(x[None, :, :kv]),
                    S.Tensor(x[None, :, kv:]))
    keys, values = O.quantise(xv[:, :kv])[2], O.quantise(xv[:, kv:])[2]
    kinds, begin = set(), [0, 0, 0]
    for step in range(4):
        end = [n + step for n in prompts]
        fused, starts = step_rows(m, begin, end)
        rows = starts[-1]
        shape = C.CacheShape(3, rows, max(e - b for b, e in zip(begin, end)), heads, kv, pages, page, cols)
        kinds.add(plan(shape, d).chunks)
        cache, index, f = pool.with_shape(shape), C.CacheIndex(ints(torch, starts), ints(torch, end), own), fused[None]
        q, k, v = f[:, :, :heads], f[:, :, heads:heads + kv], f[:, :, heads + kv:]
        qr, out, cross = (torch.empty(1, rows, heads, d, dtype=f.dtype, device="cuda") for _ in range(3))
        sa.cache_append(cache, index, S.Tensor(k), S.Tensor(v), R.Rotary(m.device_table, m.rot), S.Tensor(q), S.TensorMut(qr))
        ws = sa.cache_workspace(shape)
        sa.cache_attend(ws, cache, index, S.Tensor(qr), S.TensorMut(out))
        sa.cache_attend(ws, cache, C.CacheIndex(ints(torch, starts), ints(torch, states), other), S.Tensor(q),
                        S.TensorMut(cross), causal=False)
        got, got_cross, qv = (y[0].double().cpu().numpy() for y in (out, cross, q))
        for b in range(3):
            want, size, reach = m.want[b]
            s = slice(starts[b], starts[b + 1])
            w, z = want[begin[b]:end[b]], size[begin[b]:end[b]]
            assert (np.abs(got[s] - w) <= O.attend_tolerance(w, z, reach, d, t)).all(), (step, b)
            pad = -states[b] % 16
            one = lambda y: np.concatenate([y[at[b]:at[b + 1]], np.zeros((pad, kv, d))]).reshape(-1, 16, kv, d).transpose(0, 2, 1, 3)  # noqa: E731
            n = starts[b + 1] - starts[b]
            w, z, reach = O.attend(qv[s], one(keys), one(values), [0, n], [states[b]], np.arange((states[b] + pad) // 16)[None],
                                   16, False, 1 / math.sqrt(d), np.zeros((n, heads, d)))
            assert (np.abs(got_cross[s] - w) <= O.attend_tolerance(w, z, reach, d, t)).all(), (step, b)
        begin = end
    assert kinds == {True, False}
