"""A step's index, rotary axes, the append, bounds, picks and the attention over
them as one program runs them: requests that come, grow and end, eagerly, captured
and replayed, on two streams, and graphs that share a workspace."""
from __future__ import annotations

import subprocess
from pathlib import Path

import numpy as np
import pytest

import cache_oracle as O
import pick_oracle as P
from test_gpu_cache import draw16, ints
from test_gpu_pick import check_attend, check_pick

pytestmark = pytest.mark.gpu
SECTIONS = (8, 12, 12)


class Server:
    """One layer's cache, and a step of it: index, append with rotary axes, bounds, pick, attention."""

    def __init__(self, torch, rows, batch=4, heads=6, kv=2, d=64, page=16, cols=12, pages=40, top=4, stream=None):
        import spl_sage as S
        from spl_sage import cache as C
        from spl_sage import rotary as R

        self.torch, self.S, self.C, self.d, self.page, self.kv, self.top = torch, S, C, d, page, kv, top
        self.sa = S.SageAttention(stream or torch.cuda.current_stream(), d)
        self.shape = C.CacheShape(batch, rows, rows, heads, kv, pages, page, cols)
        self.free = C.FreePages.new(pages)
        self.tables = C.CacheTables.new(self.shape, state=self.free.state)
        self.index = self.tables.index()
        self.pool, self.bounds = C.PagedCache.new(self.shape, d), C.PageBounds.new(self.shape, d)
        self.news = torch.zeros(batch, dtype=torch.int32, device="cuda")
        x = lambda n: torch.zeros(1, rows, n, d, dtype=torch.bfloat16, device="cuda")  # noqa: E731
        self.fused, self.q, self.out = x(heads + 2 * kv), x(heads), x(heads)
        self.positions = torch.zeros(3, rows, dtype=torch.int32, device="cuda")
        self.rotary = R.AxesRotary(R.RotaryTable.axes(SECTIONS, 400).upload(), SECTIONS, self.positions)
        self.picked = C.Picked(torch.full((rows, kv, top), -9, dtype=torch.int32, device="cuda"))
        self.ws = self.sa.cache_pick_workspace(self.shape, top)

    def step(self):
        S, sa, h = self.S, self.sa, self.shape.heads
        f = self.fused
        sa.cache_tables(self.tables, self.news, self.tables.lengths, self.free)
        self.positions.copy_(self.tables.positions.expand(3, -1))
        sa.cache_append(self.pool, self.index, S.Tensor(f[:, :, h:h + self.kv]), S.Tensor(f[:, :, h + self.kv:]), self.rotary,
                        S.Tensor(f[:, :, :h]), S.TensorMut(self.q))
        sa.cache_bounds(self.pool, self.index, self.bounds)
        sa.cache_pick(self.ws, self.bounds, self.index, S.Tensor(self.q), self.picked, first=1, last=1)
        sa.cache_attend_picked(self.ws, self.pool, self.index, self.picked, S.Tensor(self.q), S.TensorMut(self.out))

    def feed(self, rng, news):
        self.news.copy_(ints(self.torch, news))
        self.fused.copy_(draw16(self.torch, rng, self.fused.shape, "bf16")[0])

    def state(self):
        return {"out": self.out.clone(), "picked": self.picked.columns.clone(), "lengths": self.tables.lengths.clone(),
                "table": self.tables.page_table.clone(), "bounds": self.bounds.codes.clone(), "k": self.pool.k_codes.clone(),
                "ring": self.free.pages.clone(), "free": self.free.state.clone()}


NEWS = [[30, 0, 70, 1], [1, 50, 1, 1], [1, 1, 1, -1], [1, 1, -1, 90], [1, 1, 0, 1], [-1, 1, 20, 1], [44, 1, 1, 1]]


class Seen:
    """The server's host copies in the form that the tests of single calls take."""

    def __init__(self, s):
        host = lambda x: x.cpu().numpy()  # noqa: E731
        self.starts, self.lengths, self.table = s.tables.starts.tolist(), s.tables.lengths.tolist(), host(s.tables.page_table)
        self.rows, self.kv, self.d, self.page, self.pages, self.shape = s.shape.rows, s.kv, s.d, s.page, s.shape.pages, s.shape
        self.cache, self.index = s.pool, s.index
        self.host = {n: host(getattr(s.pool, n)) for n in ("k_codes", "k_scales", "v_codes", "v_scales")}

    def values(self, side):
        return O.values(self.host[side + "_codes"], self.host[side + "_scales"])


def test_steps_against_the_oracle(torch_gpu):
    """After every step: the cached keys are the rotated ones of all tokens so far, bounds are those of every cached page,
    the picks are the oracle's of these bounds, and the outputs attend to them."""
    torch = torch_gpu
    rng = np.random.default_rng(0)
    s = Server(torch, 130)
    tokens = [[] for _ in range(4)]  # rotated keys of each request, in float64
    for news in NEWS:
        s.feed(rng, news)
        s.step()
        torch.cuda.synchronize()
        p = Seen(s)
        assert s.tables.state.tolist()[2:] == [0, 0]
        x = s.fused[0, :, 6:8].double().cpu().numpy()
        pos = s.tables.positions.cpu().numpy()
        turned = P.rotate_axes(x, _table(), np.stack([pos] * 3), SECTIONS, "Half", False)
        turned = torch.from_numpy(turned).to(torch.bfloat16).double().numpy()
        for b, n in enumerate(news):
            tokens[b] = [] if n < 0 else tokens[b] + list(turned[p.starts[b]:p.starts[b + 1]])
            assert p.lengths[b] == len(tokens[b])
            if tokens[b]:
                k, there = O.sequence(p.values("k"), p.table[b], p.lengths[b], p.page)
                # The fp32 rotation may round a key to the other 16-bit neighbour: almost all codes are the same.
                assert there.all() and (k == O.quantise(np.array(tokens[b]))[2]).mean() > 0.99
        codes, scales = s.bounds.codes.cpu().numpy(), s.bounds.scales.cpu().numpy()
        for b, length in enumerate(p.lengths):
            for col in range(-(-length // p.page)):
                page, held = p.table[b, col], min(p.page, length - col * p.page)
                for g in range(2):
                    hi, lo, top = P.page_bounds(p.host["k_codes"][page, g, :held], p.host["k_scales"][page, g, :held])
                    assert (codes[page, g, 0] == hi).all() and (codes[page, g, 1] == lo).all() and scales[page, g] == top
        qv = s.q.double().cpu().numpy()
        picked = check_pick(torch, p, s.q, qv, s.bounds, codes, scales, 4, 1, 1, True)
        rows = p.starts[-1]
        assert torch.equal(picked[:rows], s.picked.columns[:rows])
        out = check_attend(torch, p, s.q, qv, s.picked.columns.cpu().numpy(), "bf16")
        assert torch.equal(out[0, :rows], s.out[0, :rows])


def _table():
    from spl_sage import rotary as R

    return R.RotaryTable.axes(SECTIONS, 400).cos_sin


def test_a_captured_step_serves_every_later_one(torch_gpu):
    """The whole step replayed from one graph, the program's own work between the replays, against the eager steps."""
    torch = torch_gpu
    eager = Server(torch, 130)
    want, rng = [], np.random.default_rng(1)
    for news in NEWS:
        eager.feed(rng, news)
        eager.step()
        want.append(eager.state())
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        s = Server(torch, 130, stream=stream)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            s.step()
        rng = np.random.default_rng(1)
        for i, news in enumerate(NEWS):
            s.feed(rng, news)
            graph.replay()
            for name, x in s.state().items():
                assert torch.equal(x, want[i][name]), (i, name)
            torch.cuda.synchronize()


def test_two_graphs_share_a_workspace_in_order(torch_gpu):
    """A pick's and an attention's graphs of one stream, each replayed in turns with eager calls."""
    torch = torch_gpu
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        s = Server(torch, 130, stream=stream)
        rng = np.random.default_rng(2)
        for news in NEWS[:2]:
            s.feed(rng, news)
            s.step()
        want = s.state()
        T, M = s.S.Tensor, s.S.TensorMut
        pick = lambda: s.sa.cache_pick(s.ws, s.bounds, s.index, T(s.q), s.picked, first=1, last=1)  # noqa: E731
        attend = lambda: s.sa.cache_attend_picked(s.ws, s.pool, s.index, s.picked, T(s.q), M(s.out))  # noqa: E731
        graphs = []
        for call in (pick, attend):
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1], stream=stream):
                call()
        for _ in range(4):
            s.picked.columns.fill_(-5), s.out.zero_()
            graphs[0].replay()
            graphs[1].replay()
            rows = s.tables.starts[-1].item()
            assert torch.equal(s.out[0, :rows], want["out"][0, :rows])
            assert torch.equal(s.picked.columns[:rows], want["picked"][:rows])
            pick()
            attend()
            assert torch.equal(s.out[0, :rows], want["out"][0, :rows])


def test_two_streams(torch_gpu):
    """Two programs' steps, enqueued in turns on streams of their own, give what each gives alone."""
    torch = torch_gpu

    def steps(servers, streams):
        rngs = [np.random.default_rng(3 + i) for i in range(len(servers))]
        got = [[] for _ in servers]
        for news in NEWS:
            for i, (s, stream) in enumerate(zip(servers, streams)):
                with torch.cuda.stream(stream):
                    s.feed(rngs[i], news)
            for s, stream in zip(servers, streams):
                with torch.cuda.stream(stream):
                    s.step()
            for i, (s, stream) in enumerate(zip(servers, streams)):
                with torch.cuda.stream(stream):
                    got[i].append(s.state())
        torch.cuda.synchronize()
        return got

    streams = [torch.cuda.Stream() for _ in range(2)]
    both = []
    for stream in streams:
        with torch.cuda.stream(stream):
            both.append(Server(torch, 130, stream=stream))
    got = steps(both, streams)
    main = torch.cuda.current_stream()
    alone = steps([Server(torch, 130), Server(torch, 130)], [main, main])
    for a, b in zip(got, alone):
        for x, y in zip(a, b):
            for name in x:
                assert torch.equal(x[name], y[name]), name


def test_a_void_step_leaves_everything(torch_gpu):
    """A step that the pages do not suffice for changes no cached byte and no bound, and the next one goes on."""
    torch = torch_gpu
    rng = np.random.default_rng(4)
    s = Server(torch, 130, pages=9)
    s.feed(rng, [30, 40, 0, 0])
    s.step()
    before = s.state()
    s.feed(rng, [1, 60, 60, 0])
    s.step()
    assert s.tables.state.tolist()[2] > 0
    after = s.state()
    for name in ("k", "bounds", "lengths", "table", "ring", "picked", "out"):
        assert torch.equal(before[name], after[name]), name
    assert after["free"][:2].tolist() == before["free"][:2].tolist()
    s.feed(rng, [1, 5, 30, -1])
    s.step()
    assert s.tables.state.tolist()[2:] == [0, 0] and s.tables.lengths.tolist() == [31, 45, 30, 0]


def test_cpp_api(torch_gpu):
    """The same calls through include/spl_sage.hpp (tests/cpp/gpu_pick.cpp)."""
    exe = Path(__file__).resolve().parent / "cpp" / "bin" / "gpu_pick"
    assert exe.exists(), f"{exe} is not built; run `python __graft_entry__.py` (build)"
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and "0 failure(s)" in r.stdout, r.stdout + r.stderr
