"""Attention with tables for so many positions that the line's weights are shortened to stay below 2^30: few keys, wide tables."""
import numpy as np
import pytest

from paged_reference import World
from test_gpu_paged_attention import _try, qe  # noqa: F401 (qe: a fixture)

pytestmark = pytest.mark.gpu


def shortened_by(segments, most, floor=0):
    """By how many bits the launchers shorten weights of at most `most` (and `floor` beside them)."""
    bits = 0
    while segments * ((most >> bits) + floor) >= 2**30:
        bits += 1
    return bits


def _chunks(lens, page, nq, nkv, max_pages, seed):
    w = World(np.random.default_rng(seed), lens, page, nq, nkv, pad_rows=1, single=False)
    wide = np.full((len(lens), max_pages), -1, np.int32)
    wide[:, :w.max_pages] = w.table
    w.table, w.max_pages = wide, max_pages
    tile = 256 if w.rows * w.group >= 512 * len(lens) else 128
    tiles = w.rows * w.group // tile + len(lens)
    return w, tile, shortened_by(tiles * nkv, w.group * (max_pages * page + 256), 1)


@pytest.mark.parametrize("window", [0, 70])
@pytest.mark.parametrize("max_pages,bits", [(8192, 1), (2**19, 7)])
def test_chunks_of_64_sequences(qe, window, max_pages, bits):  # noqa: F811
    """The weights of row tiles grow by 128 keys each, shortened to 64 and to 1."""
    rng = np.random.default_rng(bits)
    lens = [(int(a), int(n)) for a, n in zip(rng.integers(-1, 400, 64), rng.integers(0, 45, 64))] + [(100, 300)]
    w, tile, short = _chunks(lens, 16, 64, 8, max_pages, bits)
    assert tile == 128 and short == bits
    _try(qe, "prefill", w, window)


@pytest.mark.parametrize("lens,tile,max_pages,bits", [([(900, 300), (10, 300)], 256, 2**16, 9), ([(900, 300), (10, 300)], 256, 2**22, 15),
                                                      ([(300, 6), (0, 1), (700, 7), (-1, 3), (90, 4)], 128, 2**21, 11)])
def test_row_tiles_of_equal_weights(qe, lens, tile, max_pages, bits):  # noqa: F811
    """Shortened by more bits than a row tile's own keys have."""
    w, rows, short = _chunks(lens, 256, 128, 2, max_pages, bits)
    assert rows == tile and short == bits and 2**bits > tile
    _try(qe, "prefill", w)


@pytest.mark.parametrize("window", [0, 2100])
def test_single_tokens(qe, window):  # noqa: F811
    rng = np.random.default_rng(5)
    w = World(rng, [(int(a), 1) for a in rng.integers(-1, 500, 72)], 256, 32, 32)
    wide = np.full((72, 2**16), -1, np.int32)
    wide[:, :w.max_pages] = w.table
    w.table, w.max_pages = wide, 2**16
    assert shortened_by(72 * 32, 2**24 // 32 + 1, 4) == 1
    _try(qe, "decode", w, window)
