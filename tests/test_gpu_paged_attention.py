"""Attention on the paged cache: single tokens, chunks, selected blocks (definition and tolerances: paged_reference.py)."""
import numpy as np
import pytest
import torch

from helpers import dev, empty, host
from paged_reference import HD, World, check

pytestmark = pytest.mark.gpu
FORMS = ("decode", "prefill", "sparse")


@pytest.fixture(scope="module")
def qe():
    import qe_amd
    return qe_amd


def everything(w):
    """Every block of every row, as a list that sparse attention takes."""
    s = np.full((w.rows, w.nkv, w.max_pages), -1, np.int32)
    for row, _, pos in w.tokens():
        n = min(pos // w.page + 1, w.max_pages)
        s[row, :, :n] = np.arange(n)
    return s


def workspace(qe, form, w):
    size = (qe.paged_prefill_workspace_bytes if form == "prefill" else qe.paged_decode_workspace_bytes)(w.rows, w.nq, w.nkv)
    return empty(size, torch.uint8).fill_(255)


def attend(qe, form, w, q, cache=None, window=0, selected=None, stream=None, ws=None):
    cache, batch = cache or w.device(qe)
    out, lse = empty((w.rows, w.nq, HD), torch.float16).fill_(-7), empty((w.rows, w.nq), torch.float32).fill_(-7)
    ws = workspace(qe, form, w) if ws is None else ws
    args = {"num_q_heads": w.nq, "row_lse": lse, "stream": stream}
    if form == "sparse":
        selected = everything(w) if selected is None else selected
        qe.launch_attention_gqa_paged_sparse(dev(q), cache, batch, dev(selected), ws, out, num_selected=selected.shape[2], **args)
    else:
        f = qe.launch_attention_gqa_paged_decode if form == "decode" else qe.launch_attention_gqa_paged_prefill
        f(dev(q), cache, batch, ws, out, window=window, **args)
    return host(out), host(lse)


def _try(qe, form, w, window=0, selected=None, q=None):
    q = w.queries(1.5) if q is None else q
    out, lse = attend(qe, form, w, q, window=window, selected=selected)
    check(out, lse, w.attention(q, window, selected), -7)
    return out, lse


SINGLE = [
    ([(0, 1)], 16, 12, 2, 0),
    ([(299, 1)], 64, 12, 2, 0),
    ([(5000, 1)], 16, 12, 2, 0),
    ([(31, 1), (32, 1), (33, 1), (15, 1), (16, 1)], 16, 2, 2, 0),
    ([(63, 1), (64, 1), (127, 1), (128, 1)], 128, 7, 1, 0),
    ([(700, 1), (-1, 1), (3, 1), (255, 1), (256, 1)], 256, 16, 1, 0),
    ([(100, 1), (1000, 1)], 32, 17, 1, 0),
    ([(90, 1), (777, 1)], 32, 128, 2, 0),
    ([(1500, 1), (2, 1), (40, 1)], 16, 5, 5, 1),
    ([(1500, 1), (2, 1), (40, 1), (39, 1)], 64, 12, 2, 40),
    ([(3001, 1)], 16, 8, 4, 1700),
]


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("lens,page,nq,nkv,window", SINGLE)
def test_single_tokens(qe, form, lens, page, nq, nkv, window):
    window = 0 if form == "sparse" else window  # (selected blocks have none)
    _try(qe, form, World(np.random.default_rng(page + nq), lens, page, nq, nkv, joint=nq == 12), window)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("lens,page,nq,nkv,window", SINGLE[:8])
def test_single_tokens_on_a_wide_table(qe, form, lens, page, nq, nkv, window):
    """Tables for more keys than there are: the work is divided by the lengths, where narrow ones have a block for each row."""
    _try(qe, form, World(np.random.default_rng(page + nq), lens, page, nq, nkv, spare=2200 // page, joint=nq == 12), window)


@pytest.mark.parametrize("lens", [300, 190, [(2000, 1)] + 200 * [(3, 1)]])
def test_many_sequences_on_a_wide_table(qe, lens):
    rng = np.random.default_rng(6)
    lens = [(int(a), 1) for a in rng.integers(-1, 400, lens)] if isinstance(lens, int) else lens
    for page in (16, 64):
        for window in (0, 100):
            _try(qe, "decode", World(rng, lens, page, 3, 1, spare=2200 // page), window)


CHUNKS = [
    ([(0, 2)], 16, 12, 2, 0),
    ([(0, 200)], 64, 12, 2, 0),
    ([(1200, 17)], 16, 12, 2, 0),
    ([(63, 64), (64, 65)], 32, 1, 1, 0),
    ([(0, 1), (500, 1), (3, 33), (0, 129), (130, 1), (7, 2)], 16, 4, 4, 0),
    ([(100, 50), (-1, 20), (0, 3), (12, 0), (900, 1)], 128, 7, 1, 0),
    ([(2000, 40)], 256, 64, 1, 0),
    ([(0, 90), (777, 10)], 16, 34, 2, 0),
    ([(0, 300)], 64, 3, 3, 1),
    ([(5, 150), (700, 30)], 16, 12, 2, 64),
    ([(1000, 70), (0, 5)], 32, 8, 1, 333),
    ([(4000, 3)], 64, 12, 2, 3000),
]


@pytest.mark.parametrize("form", ("prefill", "sparse"))
@pytest.mark.parametrize("lens,page,nq,nkv,window", CHUNKS)
def test_chunks(qe, form, lens, page, nq, nkv, window):
    window = 0 if form == "sparse" else window  # (selected blocks have none)
    w = World(np.random.default_rng(page + nq + window), lens, page, nq, nkv, joint=nq == 12, pad_rows=3, single=False,
              first_row=1 if window else 0)
    _try(qe, form, w, window)


FEW_ROWS = [
    ([(1500, 4), (2222, 5), (31, 3), (0, 4), (777, 1)], 16, 8, 2, 0),
    ([(1500, 2), (2222, 5), (31, 3), (0, 1), (777, 16)], 64, 3, 3, 50),
    ([(3000, 2), (1777, 600)], 32, 4, 2, 0),
    ([(2500, 2), (900, 600)], 16, 4, 2, 700),
    ([(5000, 2)], 32, 6, 1, 0),
    ([(640, 16), (639, 15)], 128, 2, 2, 0),
]


@pytest.mark.parametrize("lens,page,nq,nkv,window", FEW_ROWS)
def test_few_rows_beside_chunks(qe, lens, page, nq, nkv, window):
    """Sequences of up to 16 rows of a kv head (15, 16, 17, ...), alone and beside longer ones."""
    w = World(np.random.default_rng(page + nq + window), lens, page, nq, nkv, pad_rows=2, single=False)
    _try(qe, "prefill", w, window)


@pytest.mark.parametrize("form", FORMS)
def test_many_short_sequences(qe, form):
    """Several segments a block, and more than one round of the search for a row's sequence."""
    rng = np.random.default_rng(3)
    lens = [(int(a), 1) for a in rng.integers(-1, 70, 700)]
    _try(qe, form, World(rng, lens, 16, 4, 2))


def test_many_sequences_of_chunks(qe):
    rng = np.random.default_rng(4)
    lens = [(int(a), int(n)) for a, n in zip(rng.integers(-1, 60, 600), rng.integers(0, 7, 600))]
    w = World(rng, lens, 32, 3, 1, pad_rows=2, single=False)
    for form in ("prefill", "sparse"):
        _try(qe, form, w)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("page", [16, 32, 64])
def test_missing_pages(qe, form, page):
    """Holes in the table, a sequence with nothing at all, positions behind the table's last column."""
    rng = np.random.default_rng(page)
    n = 1 if form == "decode" else 5
    lens = [(9 * page, n), (page - n, n), (400, n), (20 * page, n)]
    w = World(rng, lens, page, 6, 2, holes=[(0, 0), (0, 3), (0, 4), (1, 0), (2, 400 // page)], pad_rows=0)
    w.table = np.ascontiguousarray(w.table[:, :15])
    w.max_pages = 15
    out, lse = _try(qe, form, w)
    nothing = np.isneginf(lse[n:2 * n])
    assert nothing.all() and np.all(out[n:2 * n] == 0)
    if form != "sparse":
        out, lse = _try(qe, form, w, window=page + 3)
        assert np.isneginf(lse[3 * n:]).all()  # the window of the last one lies behind the table


@pytest.mark.parametrize("n", [40, 200])
@pytest.mark.parametrize("page", [16, 32, 128])
def test_missing_pages_before_many_rows(qe, page, n):
    """The same for chunks that fill tiles: holes at the first, a middle and the last page of a sequence and of a row."""
    lens = [(9 * page, n), (0, n), (400, n), (20 * page, n)]
    last = (400 + n - 1) // page
    w = World(np.random.default_rng(page + n), lens, page, 6, 2, holes=[(0, 0), (0, 3), (0, 4), (0, 9), (1, 0), (2, 400 // page), (2, last)],
              pad_rows=2)
    w.table = np.ascontiguousarray(w.table[:, :max(15, last + 1)])
    w.max_pages = w.table.shape[1]
    for window in (0, page + 3, 150):
        _try(qe, "prefill", w, window)


@pytest.mark.parametrize("form", FORMS)
def test_positions_far_behind_the_table(qe, form):
    n = 1 if form == "decode" else 4
    w = World(np.random.default_rng(2), [(100, n), (50, n)], 16, 12, 2)
    w.lens = [(2**31 - 1, n), (50, n)]  # nearer: the last position is below 2^31
    w.context = np.array([2**31 - 1, 50], np.int32)
    q = w.queries()
    out, lse = attend(qe, form, w, q, selected=everything(World(np.random.default_rng(2), [(100, n), (50, n)], 16, 12, 2)))
    # every position of the table is in sight, and the last page's rows behind what was stored hold NaN
    assert np.all(np.isnan(out[:n]))
    full = World(np.random.default_rng(2), [(100, n), (50, n)], 16, 12, 2)
    check(out[n:], lse[n:], tuple(x[n:] for x in full.attention(q)), -7)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("context", [128, 1000, 2**30, 2**31 - 100])
def test_rows_behind_a_full_table(qe, form, context):
    """They attend to every position that has a row."""
    n = 1 if form == "decode" else 6
    w = World(np.random.default_rng(3), [(128 - n, n), (50, n)], 16, 12, 2, spare=0)
    sel = everything(w)
    w.lens = [(context, n), (50, n)]
    w.context = np.array([context, 50], np.int32)
    q = w.queries()
    out, lse = attend(qe, form, w, q, selected=sel)
    check(out, lse, w.attention(q), -7)
    if form != "sparse":  # the window of the first one lies behind the table
        out, lse = attend(qe, form, w, q, window=n)
        check(out, lse, w.attention(q, n), -7)


@pytest.mark.parametrize("form", FORMS)
def test_infinities_and_nan_reach_only_who_attends(qe, form):
    """As append stores what fp16 cannot hold (a K row of NaN, a V row of zeros), and an infinite key."""
    rng = np.random.default_rng(21)
    lens = [(150, 1), (90, 1)] if form == "decode" else [(100, 60), (0, 90)]
    w = World(rng, lens, 16, 12, 2)
    clean = w.queries(0.5)
    for s, head, at in ((0, 1, 130), (1, 0, 40)):
        w.k[s][head, at], w.v[s][head, at] = np.nan, 0
        w.store(s)
    out, lse = attend(qe, form, w, clean)
    for row, s, pos in w.tokens():
        for h in range(2):
            hit = (s, h) in ((0, 1), (1, 0)) and pos >= (130 if s == 0 else 40)
            assert np.isnan(out[row, 6 * h:6 * h + 6]).all() == hit and np.isnan(lse[row, 6 * h:6 * h + 6]).all() == hit
            assert hit or np.isfinite(out[row, 6 * h:6 * h + 6]).all()
    for s in range(2):
        w.k[s], w.v[s] = (np.nan_to_num(x) for x in (w.k[s], w.v[s]))
        w.store(s)
    want = w.attention(clean)
    fine = np.isfinite(out).all((1, 2))
    check(out[fine], lse[fine], tuple(x[fine] for x in want), -7)


@pytest.mark.parametrize("form", FORMS)
def test_every_score_minus_infinity(qe, form):
    rng = np.random.default_rng(22)
    lens = [(700, 1)] if form == "decode" else [(690, 11)]
    w = World(rng, lens, 16, 12, 2)
    w.k[0] = np.abs(w.k[0]) + np.float16(0.1)
    w.store(0)
    q = w.queries()
    q[-1, 4, 9] = -np.inf
    out, lse = attend(qe, form, w, q)
    assert np.isnan(out[-1, 4]).all() and lse[-1, 4] == -np.inf
    q[-1, 4, 9] = 0
    want = w.attention(q)
    out[-1, 4], lse[-1, 4] = want[0][-1, 4], want[2][-1, 4]
    check(out, lse, want, -7)


@pytest.mark.parametrize("form", ("decode", "prefill"))
@pytest.mark.parametrize("nq", [2, 40])
def test_the_only_key_scores_minus_infinity(qe, form, nq):
    """A window of one key, wherever it lies among the lanes: NaN, as for any row whose every score is -inf."""
    w = World(np.random.default_rng(24), [(i, 1) for i in range(40)], 16, nq, 1, pad_rows=0)
    for s in range(40):
        w.k[s] = np.abs(w.k[s]) + np.float16(0.1)
        w.store(s)
    q = w.queries()
    q[:, :, 9] = -np.inf
    out, lse = attend(qe, form, w, q, window=1)
    assert np.isnan(out).all() and np.isneginf(lse).all()


@pytest.mark.parametrize("form,lens,nq", [("decode", [(i, 1) for i in range(40)], 12), ("prefill", [(9, 3), (700, 60), (0, 1)], 12),
                                          ("prefill", [(333, 300)], 12), ("prefill", [(1000, 5)], 1)])
def test_one_key_gives_its_value(qe, form, lens, nq):
    """A window of one key: rows of V, bit for bit (a weight and the sum it is divided by are one number, off by 2^-22 at
    most, and a step of fp16 is 2^-11)."""
    nkv = 1 if nq == 1 else 2
    w = World(np.random.default_rng(25), lens, 16, nq, nkv, single=form == "decode")
    out, lse = attend(qe, form, w, w.queries(2.0), window=1)
    for row, s, pos in w.tokens():
        assert np.array_equal(out[row].reshape(nkv, -1, HD), np.repeat(w.v[s][:, pos][:, None], nq // nkv, 1)), (row, s, pos)


@pytest.mark.parametrize("form", FORMS)
def test_large_scores_and_rising_ones(qe, form):
    """Weights that underflow, a maximum that comes last, scores of a few hundred."""
    rng = np.random.default_rng(23)
    lens = [(1500, 1)] if form == "decode" else [(1490, 11)]
    w = World(rng, lens, 64, 12, 2)
    w.k[0] *= np.linspace(0.1, 4, w.k[0].shape[1])[None, :, None].astype(np.float16)
    w.store(0)
    _try(qe, form, w, q=w.queries(8.0))


@pytest.mark.parametrize("form", FORMS)
def test_pages_behind_four_gigabytes(qe, form):
    lens = [(300, 1), (450, 1)] if form == "decode" else [(300, 40), (450, 7)]
    _try(qe, form, World(np.random.default_rng(24), lens, 16, 4, 2, stride_pages=10000))


@pytest.mark.parametrize("form", FORMS)
def test_shared_pages(qe, form):
    """Two sequences with the same beginning in the same pages."""
    n = 1 if form == "decode" else 20
    w = World(np.random.default_rng(25), [(200, n), (210, n)], 16, 12, 2)
    w.table[1, :10] = w.table[0, :10]
    for x in (w.k, w.v):
        x[1][:, :160] = x[0][:, :160]
    _try(qe, form, w)


def test_selected_blocks(qe):
    rng = np.random.default_rng(26)
    for page, num in ((16, 7), (32, 5), (64, 3), (256, 2), (16, 1)):
        w = World(rng, [(900, 3), (40, 2), (-1, 1), (1500, 1), (16, 1)], page, 12, 2, pad_rows=1, single=False,
                  holes=[(0, 2)])
        sel = rng.integers(-3, w.max_pages + 3, (w.rows, 2, num)).astype(np.int32)  # any order, the same ones, ones behind
        sel[0, 0, 0], sel[1, 1, -1] = 2**31 - 1, -2**31
        sel[2, 0] = -5  # none at all
        _try(qe, "sparse", w, selected=sel)


def test_a_long_list(qe):
    """Lists longer than 64 blocks, cut over many blocks of the launch, and an odd number of 16-token pages."""
    rng = np.random.default_rng(27)
    w = World(rng, [(4000, 2)], 16, 12, 2, single=False)
    sel = np.stack([[rng.permutation(w.max_pages)[:201] for _ in range(2)] for _ in range(2)]).astype(np.int32)
    _try(qe, "sparse", w, selected=sel)


@pytest.mark.parametrize("form", FORMS)
def test_without_log_sums_and_again(qe, form):
    """The same call twice gives the same bits, whatever the workspace held; row_lse may be left out."""
    lens = [(3000, 1), (20, 1)] if form == "decode" else [(3000, 30), (20, 1)]
    w = World(np.random.default_rng(28), lens, 64, 12, 2, single=form == "decode")
    q = w.queries()
    first, _ = attend(qe, form, w, q)
    cache, batch = w.device(qe)
    ws, out = empty(workspace(qe, form, w).numel(), torch.uint8).fill_(1), empty((w.rows, 12 * HD), torch.float16)
    if form == "sparse":
        sel = everything(w)
        qe.launch_attention_gqa_paged_sparse(dev(q), cache, batch, dev(sel), ws, out, num_selected=sel.shape[2])
    else:
        f = qe.launch_attention_gqa_paged_decode if form == "decode" else qe.launch_attention_gqa_paged_prefill
        f(dev(q), cache, batch, ws, out)
    assert np.array_equal(host(out).reshape(first.shape).view(np.uint16), first.view(np.uint16))


@pytest.mark.parametrize("form", FORMS)
def test_two_streams(qe, form):
    """Calls on two streams at once, each with a workspace of its own."""
    rng = np.random.default_rng(29)
    new = 1 if form == "decode" else 40
    worlds = [World(rng, [(2000 + 500 * i, new), (70, new)], 16, 12, 2) for i in range(2)]
    qs = [w.queries() for w in worlds]
    want = [attend(qe, form, w, q) for w, q in zip(worlds, qs)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    caches, wss = [w.device(qe) for w in worlds], [workspace(qe, form, w) for w in worlds]
    sel = [dev(everything(w)) for w in worlds]
    outs = [empty((w.rows, 12, HD), torch.float16) for w in worlds]
    qd = [dev(q) for q in qs]
    torch.cuda.synchronize()
    for _ in range(5):
        for i, s in enumerate(streams):
            if form == "sparse":
                qe.launch_attention_gqa_paged_sparse(qd[i], *caches[i], sel[i], wss[i], outs[i], num_selected=sel[i].shape[2], stream=s)
            else:
                f = qe.launch_attention_gqa_paged_decode if form == "decode" else qe.launch_attention_gqa_paged_prefill
                f(qd[i], *caches[i], wss[i], outs[i], stream=s)
    for o, (x, _) in zip(outs, want):
        assert np.array_equal(host(o).view(np.uint16), x.view(np.uint16))


@pytest.mark.parametrize("form", FORMS)
def test_recorded_launch_reads_the_batch_at_replay(qe, form):
    """One recorded call for batches of other lengths, every replay against the definition and the eager call."""
    rng = np.random.default_rng(30)
    if form == "decode":
        batches = [[(50, 1), (1200, 1), (-1, 1)], [(3000, 1), (0, 1), (17, 1)], [(5, 1), (-1, 1), (-1, 1)]]
    else:
        batches = [[(50, 9), (1200, 1), (0, 20)], [(3000, 1), (0, 29), (17, 0)], [(5, 3), (-1, 1), (60, 2)]]
    rows = 3 if form == "decode" else 30
    worlds = [World(rng, b, 16, 12, 2, spare=0, single=form == "decode", pad_rows=rows - sum(n for _, n in b)) for b in batches]
    pages, total = max(w.max_pages for w in worlds), max(w.num_pages for w in worlds)
    k, v = (empty((total, 2, 16, HD), torch.float16) for _ in range(2))
    table, context, starts = empty((3, pages), torch.int32), empty((3,), torch.int32), empty((4,), torch.int32)
    q, out, lse = empty((rows, 12, HD), torch.float16), empty((rows, 12, HD), torch.float16), empty((rows, 12), torch.float32)
    selected = empty((rows, 2, pages), torch.int32)
    cache, batch = qe.paged_cache(k, v), qe.paged_batch(table, context, None if form == "decode" else starts, rows)
    ws = workspace(qe, form, worlds[0])

    def call():
        if form == "sparse":
            qe.launch_attention_gqa_paged_sparse(q, cache, batch, selected, ws, out, num_selected=pages, row_lse=lse)
        else:
            f = qe.launch_attention_gqa_paged_decode if form == "decode" else qe.launch_attention_gqa_paged_prefill
            f(q, cache, batch, ws, out, row_lse=lse)

    def put(w, x):
        table.fill_(-1)
        table[:, :w.max_pages].copy_(dev(w.table))
        context.copy_(dev(w.context))
        starts.copy_(dev(w.starts))
        k[:w.num_pages].copy_(dev(w.k_pages))
        v[:w.num_pages].copy_(dev(w.v_pages))
        selected.fill_(-1)
        selected[:, :, :w.max_pages].copy_(dev(everything(w)))
        q.copy_(dev(x))
        out.fill_(-7)
        lse.fill_(-7)

    xs = [w.queries() for w in worlds]
    put(worlds[0], xs[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for w, x in list(zip(worlds, xs)) * 2:
        put(w, x)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = host(out).copy()
        check(got, host(lse).copy(), w.attention(x), -7)
        put(w, x)
        call()
        assert np.array_equal(host(out).view(np.uint16), got.view(np.uint16))


def test_a_conversation(qe):
    """Two prompts appended and read in chunks, tokens appended and answered, one of them from selected blocks: every
    step against the definition on the rows that append stored."""
    import test_gpu_paged_append as app
    rng = np.random.default_rng(31)
    page, total = 16, 60
    pool = [empty((total, 2, page, HD), torch.float16).fill_(float("nan")) for _ in range(2)]
    order = rng.permutation(total)
    bounds, steps = empty((total, 2, 2 * HD), torch.int8), empty((total, 2), torch.float32)
    done = [0, 0]
    for new in ((70, 200), (300, 1), (1, 1), (1, 1), (33, 4)):
        lens = list(zip(done, new))
        w = World(rng, lens, page, 12, 2, known=0, single=all(n == 1 for n in new))
        w.max_pages, w.num_pages = 30, total
        w.table = np.ascontiguousarray(order.reshape(2, 30).astype(np.int32))
        x = app.Inputs(w, scale=1.1)
        cache = qe.paged_cache(*pool)
        batch = qe.paged_batch(dev(w.table), dev(w.context), None if w.single else dev(w.starts), w.rows)
        q = x.run(qe, cache, batch)
        stored = [host(p) for p in pool]
        for s, (a, n) in enumerate(lens):
            pos = np.arange(a + n)
            w.k[s], w.v[s] = (p[w.table[s, pos // page], :, pos % page].transpose(1, 0, 2).copy() for p in stored)
            for row in range(n):  # what append stored is what the definition stores
                y, tol = (y[w.starts[s] + row] for y in x.want()[1])
                assert np.all(np.abs(w.k[s][:, a + row].astype(np.float64) - y) <= tol)
        form = "decode" if w.single else "prefill"
        out, lse = attend(qe, form, w, host(q), cache=(cache, batch))
        check(out, lse, w.attention(host(q)), -7)
        qe.launch_paged_key_bounds(cache, batch, bounds, steps)
        sel = empty((w.rows, 2, 8), torch.int32)
        qe.launch_paged_select(q, cache, batch, bounds, steps, sel, empty(qe.paged_select_workspace_bytes(w.rows, 2, 30), torch.uint8),
                               num_selected=8, sinks=1, recent=2)
        chosen = host(sel)
        out, lse = attend(qe, "sparse", w, host(q), cache=(cache, batch), selected=chosen)
        check(out, lse, w.attention(host(q), selected=chosen), -7)
        done = [a + n for a, n in lens]
