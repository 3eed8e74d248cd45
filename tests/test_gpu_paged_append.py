"""Append to the paged cache: bias, norm of each head, rotation, pages (definition in 64 bits)."""
import numpy as np
import pytest
import torch

from helpers import dev, empty, host
from paged_reference import HD, World

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def qe():
    import qe_amd
    return qe_amd


class Inputs:
    def __init__(self, w, bias=True, norm=True, rot=128, interleaved=False, scale=1.0, theta=1e6, gap=0):
        rng, self.w, self.rot, self.interleaved, self.scale = w.rng, w, rot, interleaved, scale
        self.q, self.k, self.v = (rng.standard_normal((w.rows, n, HD)).astype(np.float16) for n in (w.nq, w.nkv, w.nkv))
        self.bias = [(rng.standard_normal((n, HD)) * 2).astype(np.float16) if bias else None for n in (w.nq, w.nkv, w.nkv)]
        self.norm = [(1 + 0.3 * rng.standard_normal(HD)).astype(np.float16) if norm else None for _ in range(2)]
        self.turns = theta ** (-2.0 * np.arange(rot // 2) / rot) / (2 * np.pi) if rot else None
        self.gap = gap

    def run(self, qe, cache, batch, q_out=None, eps=1e-6, stream=None):
        up = lambda a: None if a is None else dev(a.reshape(-1) if a.ndim == 2 and a.shape[1] == HD else a)  # noqa: E731
        w = self.w
        if self.gap:  # q, k and v in the rows of one projection, with something behind
            width = (w.nq + 2 * w.nkv) * HD + self.gap
            rows = np.full((w.rows, width), np.nan, np.float16)
            rows[:, :w.nq * HD] = self.q.reshape(w.rows, -1)
            rows[:, w.nq * HD:(w.nq + w.nkv) * HD] = self.k.reshape(w.rows, -1)
            rows[:, (w.nq + w.nkv) * HD:width - self.gap] = self.v.reshape(w.rows, -1)
            rows = dev(rows)
            q, k, v = rows, rows[:, w.nq * HD:], rows[:, (w.nq + w.nkv) * HD:]
            strides = {"q_stride": width, "kv_stride": width}
        else:
            q, k, v, strides = dev(self.q), dev(self.k), dev(self.v), {}
        out = empty((w.rows, w.nq, HD), torch.float16).fill_(-7) if q_out is None else q if q_out == "q" else q_out
        rope = qe.rope(dev(self.turns), self.scale, self.interleaved) if self.rot else None
        qe.launch_qkv_norm_rope_paged_append(q, out, k, v, *[up(b) for b in self.bias], *[up(g) for g in self.norm], rope,
                                             cache, batch, num_q_heads=w.nq, norm_eps=eps, stream=stream, **strides)
        return out

    def want(self, eps=1e-6):
        """(q, k, v) in 64 bits and the tolerance of each: one rounding to fp16 (2^-11), and before it the bias (2^-24
        of the sum), the norm (129 roundings in its sum, halved by the root, and five more: 2^-17 relative) and the rotation
        (two products, a sum, the angle's sine and cosine off by 2^-21: 2^-20 of |x0| + |x1|)."""
        w = self.w
        out = []
        pos = np.zeros(w.rows)
        for row, _, p in w.tokens():
            pos[row] = p
        for x, b, g in ((self.q, self.bias[0], self.norm[0]), (self.k, self.bias[1], self.norm[1]), (self.v, self.bias[2], None)):
            y = x.astype(np.float64) + (b.astype(np.float64) if b is not None else 0.0)
            if x is not self.v:
                if g is not None:
                    y = y / np.sqrt((y * y).mean(-1, keepdims=True) + eps) * g.astype(np.float64)
                size = np.abs(y)
                if self.rot:
                    half = self.rot // 2
                    first = np.arange(0, self.rot, 2) if self.interleaved else np.arange(half)
                    second = first + 1 if self.interleaved else first + half
                    a = 2 * np.pi * np.mod(pos[:, None] * self.turns, 1.0)[:, None]
                    x0, x1 = y[..., first].copy(), y[..., second].copy()
                    y[..., first] = self.scale * (x0 * np.cos(a) - x1 * np.sin(a))
                    y[..., second] = self.scale * (x0 * np.sin(a) + x1 * np.cos(a))
                    size[..., first] = size[..., second] = self.scale * (np.abs(x0) + np.abs(x1))
                tol = 2.0 ** -11 * np.abs(y) + (2.0 ** -17 + 2.0 ** -20) * size + 2.0 ** -25
            else:
                tol = 2.0 ** -11 * np.abs(y) + 2.0 ** -23 * np.abs(y) + 2.0 ** -25
            out.append((y, tol))
        return out


def _check(w, inputs, q_out, k_pages, v_pages, spoilt=()):
    """q, the stored rows, and everything else as it was."""
    want = inputs.want()
    q = host(q_out).reshape(w.rows, w.nq, HD).astype(np.float64)
    before = [w.k_pages.copy(), w.v_pages.copy()]
    rows = [row for row, _, _ in w.tokens()]
    idle = np.setdiff1d(np.arange(w.rows), rows)
    assert np.all(np.abs(q[rows] - want[0][0][rows]) <= want[0][1][rows])
    got = [host(k_pages), host(v_pages)]
    for row, s, pos in w.tokens():
        if not w.has_page(s, pos):
            continue
        page, r = w.table[s, pos // w.page], pos % w.page
        for i in range(2):
            for h in range(w.nkv):
                x = got[i][page, h, r].astype(np.float64)
                if (row, h) in spoilt:
                    assert np.all(np.isnan(x)) if i == 0 else np.all(x == 0)
                else:
                    y, tol = want[1 + i][0][row, h], want[1 + i][1][row, h]
                    assert np.all(np.abs(x - y) <= tol), (row, s, pos, i, h)
            before[i][page, :, r] = got[i][page, :, r]
    for i in range(2):
        assert np.array_equal(before[i].view(np.uint16), got[i].view(np.uint16))
    return idle, q


@pytest.mark.parametrize("lens,page,nq,nkv,opts", [
    ([(0, 1)], 16, 12, 2, {}),
    ([(1000, 1)], 64, 12, 2, {"norm": False}),
    ([(15, 1), (16, 1), (0, 1), (31, 1)], 16, 4, 4, {"bias": False}),
    ([(0, 40), (7, 1), (30, 17), (63, 2)], 32, 6, 2, {"interleaved": True}),
    ([(120000, 3), (5, 20)], 128, 8, 1, {"rot": 64, "scale": 1.2079441}),
    ([(250, 10)], 256, 7, 7, {"rot": 16, "interleaved": True}),
    ([(3, 5), (900000000, 2)], 16, 3, 1, {"rot": 80}),  # the second one's positions have no page
    ([(100, 6)], 16, 17, 1, {"rot": 0, "norm": False, "bias": False}),
    ([(40, 9)], 64, 64, 1, {"gap": 24}),
    ([(2, 3), (-1, 4), (8, 2)], 16, 12, 2, {"gap": 8, "interleaved": True, "rot": 32}),
])
@pytest.mark.parametrize("joint", [False, True])
def test_append(qe, lens, page, nq, nkv, opts, joint):
    rng = np.random.default_rng(len(lens) * 100 + page + nq)
    far = [s for s, (a, _) in enumerate(lens) if a > 10**6]
    small = [(a if s not in far else 0, n) for s, (a, n) in enumerate(lens)]
    w = World(rng, small, page, nq, nkv, joint=joint, pad_rows=3, known=0, single=False, first_row=2)
    for s in far:
        w.lens = lens
        w.context[s] = lens[s][0]
    x = Inputs(w, **opts)
    cache, batch = w.device(qe)
    idle, q = _check(w, x, x.run(qe, cache, batch), *w.tensors)
    assert np.all(q[idle] == -7)


def test_single_tokens_and_sequences_that_take_no_part(qe):
    rng = np.random.default_rng(5)
    w = World(rng, [(5, 1), (-1, 1), (100, 1), (-2**31, 1), (16, 1)], 16, known=0)
    assert w.single
    x = Inputs(w)
    cache, batch = w.device(qe)
    idle, q = _check(w, x, x.run(qe, cache, batch), *w.tensors)
    assert list(idle) == [1, 3] and np.all(q[idle] == -7)


def test_q_in_place(qe):
    for interleaved in (False, True):
        w = World(np.random.default_rng(6), [(5, 30), (60, 1)], 16, known=0)
        x = Inputs(w, interleaved=interleaved)
        apart = x.run(qe, *w.device(qe))
        same = x.run(qe, *w.device(qe), q_out="q")
        assert torch.equal(apart, same)
        _check(w, x, same, *w.tensors)


def test_missing_pages_and_positions_behind_the_table(qe):
    rng = np.random.default_rng(7)
    w = World(rng, [(10, 60), (0, 5)], 16, known=0, spare=0, holes=[(0, 1), (0, 3)])
    w.table = np.ascontiguousarray(w.table[:, :4])  # positions 64 .. 69 have no entry
    w.max_pages = 4
    x = Inputs(w)
    _check(w, x, x.run(qe, *w.device(qe)), *w.tensors)


def test_values_that_fp16_cannot_hold(qe):
    rng = np.random.default_rng(8)
    w = World(rng, [(3, 6), (20, 2)], 16, known=0)
    x = Inputs(w, bias=False, norm=False)
    x.v[1, 0, 5] = np.inf
    x.v[4, 1, 127] = np.nan
    x.v[6, 0, 0] = -np.inf
    x.v[6, 1, 64] = 65504
    _check(w, x, x.run(qe, *w.device(qe)), *w.tensors, spoilt={(1, 0), (4, 1), (6, 0)})
    y = Inputs(w, norm=False)  # the sum with the bias
    y.v[2, 1, 9], y.bias[2][1, 9] = 65504, 32
    _check(w, y, y.run(qe, *w.device(qe)), *w.tensors, spoilt={(2, 1)})


def test_a_norm_of_zeros_and_of_large_values(qe):
    w = World(np.random.default_rng(9), [(0, 4)], 16, known=0)
    x = Inputs(w, bias=False)
    x.q[0], x.k[0], x.q[1] = 0, 0, 60000
    _check(w, x, x.run(qe, *w.device(qe)), *w.tensors)


def test_many_sequences(qe):
    """More than one round of the search for a row's sequence; empty ones between."""
    rng = np.random.default_rng(10)
    lens = [(int(a), int(n)) for a, n in zip(rng.integers(0, 20, 5000), rng.integers(0, 3, 5000))]
    w = World(rng, lens, 16, 2, 1, known=0, pad_rows=7, single=False)
    x = Inputs(w)
    idle, q = _check(w, x, x.run(qe, *w.device(qe)), *w.tensors)
    assert idle.size == 7 and np.all(q[idle] == -7)


def test_pages_behind_four_gigabytes(qe):
    """(Row offsets of more than 32 bits: 60 pages, 80 MB apart in each pool.)"""
    w = World(np.random.default_rng(11), [(300, 40), (450, 7)], 16, known=0, stride_pages=10000)
    x = Inputs(w)
    _check(w, x, x.run(qe, *w.device(qe)), *w.tensors)


def test_no_rows(qe):
    w = World(np.random.default_rng(12), [(3, 0), (0, 0)], 16, known=0, single=False)
    cache, batch = w.device(qe)
    qe.launch_qkv_norm_rope_paged_append(None, None, None, None, None, None, None, None, None, None, cache, batch)
    k, v = (host(t) for t in w.tensors)
    assert np.array_equal(k.view(np.uint16), w.k_pages.view(np.uint16))
    assert np.array_equal(v.view(np.uint16), w.v_pages.view(np.uint16))


def test_recorded_launch_reads_the_batch_at_replay(qe):
    rng = np.random.default_rng(13)
    steps = [World(rng, [(a, 1), (b, 1), (c, 1)], 16, known=0, spare=0) for a, b, c in ((5, 100, 33), (80, -1, 111), (0, 7, 96))]
    pages = max(w.max_pages for w in steps)
    k, v = empty((64, 2, 16, HD), torch.float16), empty((64, 2, 16, HD), torch.float16)
    table, context = empty((3, pages), torch.int32), empty((3,), torch.int32)
    q, kk, vv = (empty((3, n * HD), torch.float16) for n in (12, 2, 2))
    out = empty((3, 12 * HD), torch.float16)
    x = [Inputs(w, bias=False, norm=False) for w in steps]
    rope = qe.rope(dev(x[0].turns))
    cache, batch = qe.paged_cache(k, v), qe.paged_batch(table, context)

    def put(w, y):
        table.fill_(-1)
        table[:, :w.max_pages].copy_(dev(w.table))
        context.copy_(dev(w.context))
        for t, a in ((q, y.q), (kk, y.k), (vv, y.v)):
            t.copy_(dev(a).reshape(3, -1))
        k[:w.num_pages].copy_(dev(w.k_pages))
        v[:w.num_pages].copy_(dev(w.v_pages))
        out.fill_(-7)

    put(steps[0], x[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        qe.launch_qkv_norm_rope_paged_append(q, out, kk, vv, None, None, None, None, None, rope, cache, batch)
    for w, y in list(zip(steps, x)) * 2:
        put(w, y)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        idle, got = _check(w, y, out, k[:w.num_pages], v[:w.num_pages])
        assert np.all(got[idle] == -7)
