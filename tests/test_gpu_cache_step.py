"""A step's index built on the GPU from its requests' lengths, against pick_oracle:
every output equal, in one launch and in two, void steps, ended requests, rings that
wrap, numbers that make no sense, and steps that follow each other in place."""
from __future__ import annotations

import numpy as np
import pytest

import pick_oracle as P
from test_gpu_cache import ints

pytestmark = pytest.mark.gpu
NAMES = ("starts", "lengths", "page_table", "positions", "slots", "sequences", "state")


def step(torch, news, past, ring, state, table, page, rows, pages=None, drop=(), times=1):
    """The outputs of the call by name, the ring among them; every buffer has guards behind it."""
    import spl_sage as S
    from spl_sage import cache as C

    b, cols = table.shape
    pages = len(ring) if pages is None else pages
    shape = C.CacheShape(b, rows, 1, 2, 1, pages, page, cols)
    bufs = {}

    def buf(name, n, dtype=torch.int32):
        bufs[name] = torch.full((n + 8,), 77, dtype=dtype, device="cuda")
        return bufs[name][:n]

    t = buf("page_table", b * cols).view(b, cols)
    t.copy_(ints(torch, table))
    r = buf("ring", len(ring))
    r.copy_(ints(torch, ring))
    made = dict(starts=buf("starts", b + 1), lengths=buf("lengths", b), page_table=t, positions=buf("positions", rows),
                slots=buf("slots", rows, torch.int64), sequences=buf("sequences", rows), state=buf("state", 4),
                scratch=buf("scratch", 2 * b))
    tables = C.CacheTables(shape, **{k: None if k in drop else v for k, v in made.items()})
    sa = S.SageAttention(torch.cuda.current_stream(), 64)
    for _ in range(times):
        sa.cache_tables(tables, ints(torch, news), ints(torch, past), C.FreePages(r, ints(torch, state)))
    torch.cuda.synchronize()
    for name, x in bufs.items():
        assert (x[-8:] == 77).all(), name
        if name in drop:
            assert (x == 77).all(), name
    return {k: (made[k] if k != "ring" else r).cpu().numpy() for k in (*NAMES, "ring")}


def check(torch, news, past, ring, state, table, page, rows, pages=None, drop=(), **more):
    got = step(torch, news, past, ring, state, table, page, rows, pages, drop, **more)
    want = P.tables(news, past, ring, state, table, page, rows, len(ring) if pages is None else pages)
    for k in (*NAMES, "ring"):
        if k not in drop:
            w = np.asarray(want[k])
            bad = got[k] != w
            assert not bad.any(), (k, int(bad.sum()), np.argwhere(bad)[:4], got[k][bad][:4], w[bad][:4])
    return want


def batch(rng, news, past, page, spare=3, cols=None, head=None):
    """(ring, state, table): the pages that the requests hold, and the free ones behind a random place of the ring."""
    held = [-(-max(p, 0) // page) for p in past]
    want = [h if n < 0 else -(-(max(p, 0) + n) // page) for n, p, h in zip(news, past, held)]
    cols = max(1, max(want, default=1)) + 1 if cols is None else cols
    need = sum(w - h for w, h in zip(want, held))
    cap = sum(held) + need + max(spare, 0) + 2
    order = rng.permutation(cap)
    table = rng.integers(-3, cap, (len(news), cols))  # stale columns
    for b, h in enumerate(held):
        h = min(h, cols)
        table[b, :h], order = order[:h], order[h:]
    count = max(0, need + spare)
    head = int(rng.integers(0, cap)) if head is None else head
    ring = rng.integers(-5, cap, cap)
    ring[(head + np.arange(count)) % cap] = order[:count]
    return ring.tolist(), [head, count], table


CASES = {
    "one token": ([1], [0]),
    "one page full": ([1], [16]),
    "nothing": ([0, 0], [5, 0]),
    "steps": ([1] * 9, [0, 1, 15, 16, 17, 31, 32, 500, 3]),
    "prompts": ([100, 0, 33, 1, 16, 17], [7, 9, 0, 0, 16, 1000]),
    "ended": ([-1, 5, -7, 1, -1], [100, 3, 0, 16, 17]),
    "all ended": ([-1, -1, -1], [40, 0, 16]),
    "below 0": ([3, 1], [-9, -1]),
    "long": ([9000, 1, 5000], [11, 70000, 3]),
}


@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("name", CASES)
def test_steps(torch_gpu, name, page):
    rng = np.random.default_rng(page)
    news, past = CASES[name]
    ring, state, table = batch(rng, news, past, page)
    rows = sum(max(n, 0) for n in news)
    for pad in (0, 1, 6):
        want = check(torch_gpu, news, past, ring, state, table, page, rows + pad)
        assert want["state"][2:] == [0, 0] and want["starts"][-1] == rows


@pytest.mark.parametrize("n,rows_each,cols", [(1023, 3, None), (1024, 9, None), (1025, 2, None), (2047, 5, None), (2048, 5, None),
                                              (5000, 3, None), (65535, 1, 3), (300, 60, 1200)])
def test_many_requests(torch_gpu, n, rows_each, cols):
    """More requests than threads, than a workgroup's LDS holds starts, more rows than one workgroup sees to, wide tables."""
    rng = np.random.default_rng(n)
    news = rng.integers(-1, 2 * rows_each, n).tolist()
    past = rng.integers(0, 40, n).tolist()
    ring, state, table = batch(rng, news, past, 16, cols=cols)
    check(torch_gpu, news, past, ring, state, table, 16, sum(max(x, 0) for x in news) + 3)


def test_the_ring_goes_over_its_end(torch_gpu):
    """Wherever it begins, for pages taken and pages given back; exactly as many as there are."""
    rng = np.random.default_rng(0)
    news, past = [40, -1, 1, -1, 90], [3, 50, 32, 1, 0]
    for spare in (0, 3):
        for head in range(0, 26):
            ring, state, table = batch(rng, news, past, 16, spare=spare, head=head % 17)
            want = check(torch_gpu, news, past, ring, state, table, 16, 140)
            assert want["state"][2] == 0


@pytest.mark.parametrize("large", [False, True])
def test_void_steps(torch_gpu, large):
    """A page too few, tokens past the table, rows past the shape: no rows, the old lengths, what ended is given back."""
    rng = np.random.default_rng(1)
    news, past = [20, -1, 3, 0], [17, 33, 0, 64]
    if large:
        news, past = news * 400, past * 400
    rows = sum(max(n, 0) for n in news)
    for spare, cols, room, which in ((-1, None, rows, 2), (3, 4, rows, None), (3, 2, rows, 2), (3, None, rows - 1, 3), (-2, 1, 5, 2)):
        ring, state, table = batch(rng, news, past, 16, spare=spare, cols=cols)
        want = check(torch_gpu, news, past, ring, state, table, 16, room)
        assert which is None or want["state"][which] > 0
        if which is not None:
            assert want["starts"][-1] == 0 and want["lengths"][:4] == [17, 0, 0, 64]


def test_numbers_that_make_no_sense_stay_in_bounds(torch_gpu):
    """States past the ring, ids that are no pages', lengths past 31 bits together, a ring of one place."""
    rng = np.random.default_rng(2)
    big = 2 ** 31 - 1
    news, past = [5, -1, 2], [30, 40, 16]
    ring, _, table = batch(rng, news, past, 16)
    for state in ([-1, 4], [-2 ** 31, big], [big, -5], [len(ring) + 3, len(ring) + 9], [3, 0]):
        check(torch_gpu, news, past, ring, state, table, 16, 9)
    check(torch_gpu, news, past, [-7, 2 ** 30, 3, 99, -1, 5, 6, 7], [0, 8], table, 16, 9, pages=7)
    check(torch_gpu, [big, big, -big], [big, 5, big], ring, [0, 3], table, 16, 9)
    check(torch_gpu, [0, big, 0], [0, 0, big], ring, [0, 3], table, 16, 9)
    check(torch_gpu, [3], [0], [0], [0, 1], np.array([[5, 6]]), 16, 3)
    check(torch_gpu, [-1], [20], [4], [0, 0], np.array([[5, 6]]), 16, 3)


def test_outputs_that_are_not_asked_for(torch_gpu):
    rng = np.random.default_rng(3)
    for news, past in (([4, 1, -1], [30, 16, 5]), ([4000, 5000, -1], [30, 16, 5])):
        ring, state, table = batch(rng, news, past, 16)
        rows = sum(max(n, 0) for n in news) + 2
        for drop in (("positions",), ("slots",), ("sequences",), ("positions", "slots", "sequences")):
            check(torch_gpu, news, past, ring, state, table, 16, rows, drop=drop)


def test_a_step_called_again_is_the_same(torch_gpu):
    """Inputs that are not outputs stay as they are: the call gives the same again."""
    rng = np.random.default_rng(4)
    news, past = [40, -1, 1, 0], [3, 50, 32, 9]
    ring, state, table = batch(rng, news, past, 16)
    check(torch_gpu, news, past, ring, state, table, 16, 45, times=3)


def test_no_requests(torch_gpu):
    import spl_sage as S
    from spl_sage import cache as C

    torch = torch_gpu
    shape = C.CacheShape(0, 5, 1, 2, 1, 4, 16, 2)
    t, free = C.CacheTables.new(shape), C.FreePages.new(4)
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    S.SageAttention(torch.cuda.current_stream(), 64).cache_tables(t, none, none, free)
    assert t.starts.tolist() == [0] and t.state.tolist() == [0, 4, 0, 0] and t.slots.tolist() == [-1] * 5


def serve(torch, sa, rng, batch_size, page, cols, pages, steps, max_rows, run):
    """Random requests for `steps` steps in place: past is the step's lengths, the ring's state the step's. run(news)
    enqueues a step; the host follows with the oracle."""
    from spl_sage import cache as C

    shape = C.CacheShape(batch_size, max_rows, max_rows, 2, 1, pages, page, cols)
    free = C.FreePages.new(pages)
    tables = C.CacheTables.new(shape, state=free.state)
    news = torch.zeros(batch_size, dtype=torch.int32, device="cuda")
    call = run(lambda: sa.cache_tables(tables, news, tables.lengths, free))
    past, ring, state, table = [0] * batch_size, list(range(pages)), [0, pages], np.zeros((batch_size, cols), int)
    live = [False] * batch_size
    for _ in range(steps):
        n = [0] * batch_size
        for b in range(batch_size):
            if live[b] and (rng.random() < 0.15 or past[b] + 2 > cols * page):
                n[b] = -1
            elif live[b]:
                n[b] = 1
            elif rng.random() < 0.4:
                n[b] = int(rng.integers(1, cols * page // 2))
        news.copy_(ints(torch, n))
        call()
        want = P.tables(n, past, ring, state, table, page, max_rows, pages)
        for k in NAMES:
            got = getattr(tables, k).cpu().numpy()
            assert (got == np.asarray(want[k])).all(), k
        assert (free.pages.cpu().numpy() == np.asarray(want["ring"])).all()
        good = not want["state"][2] and not want["state"][3]
        live = [x >= 0 and (x > 0 and good or live[b]) for b, x in enumerate(n)]
        past, ring, state, table = want["lengths"], want["ring"], want["state"], np.array(want["page_table"])
        held = [table[b, :-(-p // page)].tolist() for b, p in enumerate(past)]
        owned = sum(held, []) + [ring[(state[0] + i) % pages] for i in range(state[1])]
        assert sorted(owned) == list(range(pages))  # every page has one owner, or is free


@pytest.mark.parametrize("batch_size,cols,pages,rows", [(7, 6, 24, 200), (1500, 3, 3600, 20000)])
def test_steps_in_place(torch_gpu, batch_size, cols, pages, rows):
    import spl_sage as S

    torch = torch_gpu
    sa = S.SageAttention(torch.cuda.current_stream(), 64)
    serve(torch, sa, np.random.default_rng(5), batch_size, 16, cols, pages, 40 if batch_size < 100 else 6, rows,
                  lambda call: call)


@pytest.mark.parametrize("batch_size,cols,pages,rows", [(7, 6, 24, 200), (1500, 3, 3600, 20000)])
def test_steps_captured(torch_gpu, batch_size, cols, pages, rows):
    """A step captured once and replayed for every later one."""
    import spl_sage as S

    torch = torch_gpu
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        sa = S.SageAttention(stream, 64)

        def run(call):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                call()
            return graph.replay

        serve(torch, sa, np.random.default_rng(6), batch_size, 16, cols, pages, 25 if batch_size < 100 else 5, rows, run)
