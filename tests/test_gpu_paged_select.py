"""Bounds of pages and the selection of blocks: equal to the definition (paged_reference.py), bit for bit."""
import numpy as np
import pytest
import torch

from helpers import dev, empty, host
from paged_reference import HD, World, bounds, scores, select

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def qe():
    import qe_amd
    return qe_amd


def _bounds(qe, w, cache=None):
    b, s = empty((w.num_pages, w.nkv, 2 * HD), torch.int8).fill_(99), empty((w.num_pages, w.nkv), torch.float32).fill_(-7)
    qe.launch_paged_key_bounds(*(cache or w.device(qe)), b, s)
    return host(b), host(s)


def _select(qe, w, q, b, s, num, sinks, recent, cache=None):
    out = empty((w.rows, w.nkv, num), torch.int32).fill_(-77)
    ws = empty(max(4, qe.paged_select_workspace_bytes(w.rows, w.nkv, w.max_pages)), torch.uint8).fill_(255)
    qe.launch_paged_select(dev(q), *(cache or w.device(qe)), dev(b), dev(s), out, ws, num_q_heads=w.nq, num_selected=num,
                           sinks=sinks, recent=recent)
    return host(out)


def _check_selection(w, q, b, s, num, sinks, recent, got):
    live = np.zeros(w.rows, bool)
    for row, seq, pos in w.tokens():
        live[row] = True
        own = pos // w.page
        n = min(own + 1, w.max_pages)
        page = w.table[seq, :n]
        there = (page >= 0) & (page < w.num_pages)
        page = np.where(there, page, 0)
        for h in range(w.nkv):
            score = scores(q[row, h * w.group:(h + 1) * w.group], b[page, h], s[page, h])
            want = select(score, there, own, num, sinks, recent)
            assert np.array_equal(got[row, h], want), (row, h, got[row, h], want)
    assert np.all(got[~live] == -77)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("nkv", [1, 2, 5])
def test_bounds(qe, page, nkv):
    """Pages that new tokens reach, full and partly filled; others stay as they are."""
    rng = np.random.default_rng(page + nkv)
    w = World(rng, [(0, 1), (page - 1, 2), (5 * page + 3, 1), (2 * page, 3 * page + 5), (-1, 4), (7, page)], page, nkv, nkv,
              joint=nkv == 2, pad_rows=2, single=False)
    w.k[0][0] = 0  # a page of zeros
    w.k[1][-1, :, 3] = np.float16(-60000)
    w.k[2][:, -1] = np.float16(6e-8)  # subnormal
    for s in range(3):
        w.store(s)
    got, steps = _bounds(qe, w)
    touched = np.zeros(w.num_pages, bool)
    for s, (a, n) in enumerate(w.lens):
        if a < 0 or n == 0:
            continue
        for blk in range(a // page, (a + n - 1) // page + 1):
            at = w.table[s, blk]
            touched[at] = True
            want, m = bounds(w.k_pages[at], min(page, a + n - blk * page))
            assert np.array_equal(got[at], want) and np.array_equal(steps[at], m.astype(np.float32))
    assert np.all(got[~touched] == 99) and np.all(steps[~touched] == -7)


def test_bounds_of_every_pair_of_values(qe):
    """127 x / m for many pairs of fp16 values: the bytes of exact whole-number arithmetic."""
    rng = np.random.default_rng(1)
    w = World(rng, [(0, 16 * 400)], 16, 1, 1, single=False)
    bits = rng.integers(0, 0x7C00, w.k[0].shape).astype(np.uint16)
    k = bits.view(np.float16).copy()
    k[0, 16 * 200:] = rng.integers(1, 300, k[0, 16 * 200:].shape) * 2.0 ** -6  # near-even quotients, exact ones among them
    w.k[0] = np.where(rng.random(k.shape) < 0.5, -k, k)
    w.store(0)
    got, steps = _bounds(qe, w)
    for blk in range(400):
        x = w.k[0][0, 16 * blk:16 * blk + 16].astype(np.float64)
        whole = np.rint(x * 2.0 ** 24).astype(object)  # fp16 values are multiples of 2^-24
        m = max(abs(v) for v in whole.reshape(-1))
        high = [-((-127 * max(c)) // m) for c in whole.T]
        low = [(127 * min(c)) // m for c in whole.T]
        assert got[w.table[0, blk], 0].tolist() == [int(v) for v in high + low]


def test_bounds_of_pages_that_are_not_finite(qe):
    w = World(np.random.default_rng(2), [(0, 48)], 16, 2, 2, single=False)
    w.k[0][0, 5, 7], w.k[0][1, 20, 0], w.k[0][0, 47, 127] = np.inf, np.nan, -np.inf
    w.store(0)
    got, steps = _bounds(qe, w)
    for blk in range(3):
        want, m = bounds(w.k[0][:, 16 * blk:16 * blk + 16], 16)
        assert np.array_equal(got[w.table[0, blk]], want) and np.array_equal(steps[w.table[0, blk]], m.astype(np.float32))
    assert np.isinf(steps).sum() == 3


def test_bounds_without_pages(qe):
    w = World(np.random.default_rng(3), [(0, 40), (60, 3)], 16, 2, 2, single=False, spare=0, holes=[(0, 1)])
    w.table = np.ascontiguousarray(w.table[:, :3])
    w.max_pages = 3
    got, steps = _bounds(qe, w)
    assert (steps != -7).any(1).sum() == 2  # blocks 0 and 2 of the first sequence


@pytest.mark.parametrize("lens,page,nq,nkv,num,sinks,recent", [
    ([(0, 1)], 16, 12, 2, 4, 1, 1),
    ([(999, 1)], 16, 12, 2, 8, 1, 2),
    ([(4000, 1), (100, 1), (-1, 1), (31, 1)], 32, 12, 2, 16, 0, 1),
    ([(5000, 1), (3, 1)], 64, 5, 5, 1, 0, 0),
    ([(5000, 1), (300, 1)], 16, 34, 2, 33, 3, 30),
    ([(3000, 40), (0, 70), (-1, 3), (500, 1)], 16, 12, 2, 9, 2, 3),
    ([(2000, 21)], 128, 7, 1, 5, 0, 0),
    ([(600, 37), (17, 2)], 16, 64, 1, 20, 4, 0),
    ([(600, 37), (17, 2)], 16, 3, 3, 20, 0, 20),
    ([(1000, 5)], 256, 16, 1, 3, 1, 1),
])
def test_selection(qe, lens, page, nq, nkv, num, sinks, recent):
    rng = np.random.default_rng(page + nq + num)
    w = World(rng, lens, page, nq, nkv, pad_rows=2, single=False, k_level=0.2) if any(n > 1 for _, n in lens) else \
        World(rng, lens, page, nq, nkv, k_level=0.2)
    b = rng.integers(-127, 128, (w.num_pages, nkv, 2, HD)).astype(np.int8)
    b = np.sort(b, 2)[:, :, ::-1].reshape(w.num_pages, nkv, 2 * HD)
    s = (rng.random((w.num_pages, nkv)) * 5).astype(np.float16).astype(np.float32)
    q = w.queries()
    _check_selection(w, q, b, s, num, sinks, recent, _select(qe, w, q, b, s, num, sinks, recent))


def test_selection_with_the_bounds_of_the_keys(qe):
    """The two launches after one another: every key's score is within its block's bound."""
    rng = np.random.default_rng(5)
    w = World(rng, [(0, 700), (0, 33)], 16, 12, 2, single=False)
    cache = w.device(qe)
    b, s = _bounds(qe, w, cache)
    q = w.queries()
    got = _select(qe, w, q, b, s, 6, 1, 1, cache)
    _check_selection(w, q, b, s, 6, 1, 1, got)
    qn = q[-1, 0].astype(np.float64)
    m = np.abs(qn).max()
    n = np.rint(127 * qn / m)
    for blk in range(2):
        page = w.table[1, blk]
        top = np.maximum(n * b[page, 0, :HD], n * b[page, 0, HD:]).sum() * s[page, 0] / 127
        keys = w.k[1][0, 16 * blk:16 * blk + 16].astype(np.float64)
        assert np.all(keys @ n <= top + 1e-6 * abs(top))


def test_ties_and_a_table_of_thousands_of_blocks(qe):
    """Thousands of blocks on a few pages: hundreds of equal scores, the lower blocks first.  Lists of up to 2048, 16384 and
    more blocks are selected by different kernels."""
    rng = np.random.default_rng(6)
    for blocks in (2048, 2049, 9000, 16384, 17000):
        w = World(rng, [(20, 1)], 16, 12, 2)
        w.lens = [(16 * blocks - 5, 1)]
        w.context = np.array([16 * blocks - 5], np.int32)
        w.max_pages = blocks
        w.table = rng.integers(0, w.num_pages, (1, blocks)).astype(np.int32)
        w.table[0, rng.random(blocks) < 0.1] = -1
        b = np.sort(rng.integers(-127, 128, (w.num_pages, 2, 2, HD)).astype(np.int8), 2)[:, :, ::-1].reshape(w.num_pages, 2, 2 * HD)
        s = np.ones((w.num_pages, 2), np.float32)
        q = w.queries()
        for num, sinks, recent in ((300, 1, 4), (2500, 0, 0), (blocks, 0, 1), (1, 0, 0)):
            _check_selection(w, q, b, s, num, sinks, recent, _select(qe, w, q, b, s, num, sinks, recent))


def test_values_that_are_not_finite_and_zeros(qe):
    rng = np.random.default_rng(7)
    w = World(rng, [(800, 3)], 16, 12, 2, single=False, holes=[(0, 7)])
    b = np.sort(rng.integers(-127, 128, (w.num_pages, 2, 2, HD)).astype(np.int8), 2)[:, :, ::-1].reshape(w.num_pages, 2, 2 * HD)
    s = rng.random((w.num_pages, 2)).astype(np.float16).astype(np.float32)
    s[w.table[0, 20]], s[w.table[0, 33]], s[w.table[0, 40]] = np.inf, np.inf, 0
    b[w.table[0, 20]], b[w.table[0, 33]], b[w.table[0, 40]] = 0, 0, 0
    q = w.queries()
    q[0, 2, 5], q[1, :6], q[2, 9, 100], q[2, 8, 1] = np.inf, 0, np.nan, -np.inf
    got = _select(qe, w, q, b, s, 6, 1, 1)
    _check_selection(w, q, b, s, 6, 1, 1, got)
    assert {20, 33} <= set(got[0, 0])


def test_recorded_selection(qe):
    rng = np.random.default_rng(8)
    worlds = [World(rng, [(a, 1), (c, 1)], 16, 12, 2, spare=0) for a, c in ((500, 30), (1000, -1), (0, 700))]
    pages, total = max(w.max_pages for w in worlds), max(w.num_pages for w in worlds)
    k, v = (empty((total, 2, 16, HD), torch.float16) for _ in range(2))
    table, context, q = empty((2, pages), torch.int32), empty((2,), torch.int32), empty((2, 12, HD), torch.float16)
    b, s = empty((total, 2, 2 * HD), torch.int8).zero_(), empty((total, 2), torch.float32).zero_()
    sel, ws = empty((2, 2, 5), torch.int32), empty(qe.paged_select_workspace_bytes(2, 2, pages), torch.uint8)
    cache, batch = qe.paged_cache(k, v), qe.paged_batch(table, context)

    def put(w, x):
        table.fill_(-1)
        table[:, :w.max_pages].copy_(dev(w.table))
        context.copy_(dev(w.context))
        k[:w.num_pages].copy_(dev(w.k_pages))
        q.copy_(dev(x))
        sel.fill_(-77)

    xs = [w.queries() for w in worlds]
    put(worlds[0], xs[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        qe.launch_paged_key_bounds(cache, batch, b, s)
        qe.launch_paged_select(q, cache, batch, b, s, sel, ws, num_selected=5, sinks=1, recent=1)
    for w, x in list(zip(worlds, xs)) * 2:
        put(w, x)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        full = World.__new__(World)
        full.__dict__.update(w.__dict__, max_pages=pages, table=host(table))
        _check_selection(full, x, host(b), host(s), 5, 1, 1, host(sel))
        for row, seq, pos in w.tokens():
            page = w.table[seq, pos // 16]
            want, m = bounds(w.k_pages[page], pos % 16 + 1)
            assert np.array_equal(host(b)[page], want) and np.array_equal(host(s)[page], m.astype(np.float32))
