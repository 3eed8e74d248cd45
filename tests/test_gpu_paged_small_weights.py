"""Attention on the paged cache with a few keys far above all others: small softmax weights keep their bits."""
import numpy as np
import pytest

from paged_levels import FP16, OCTAVE, TWO_FP16, Levels, check, far_below
from test_gpu_paged_attention import attend, qe  # noqa: F401 (qe: a fixture)

pytestmark = pytest.mark.gpu

# form, new tokens, bits of a weight; 12 q heads over 2: 12 rows of a kv head, 54 (blocks of four waves), 600 (of eight)
FORMS = [("decode", 1, TWO_FP16), ("sparse", 1, TWO_FP16), ("prefill", 2, TWO_FP16), ("prefill", 9, FP16), ("prefill", 100, FP16)]


@pytest.mark.parametrize("form,new,weight", FORMS)
@pytest.mark.parametrize("n", [100, 1000, 5001])
@pytest.mark.parametrize("depth", [4.3, 11.0, 15.87, 18.4, 20.6, 23.0, 25.2])
def test_one_key_of_32_far_above_the_others(qe, form, new, weight, n, depth):  # noqa: F811
    """depth: octaves of the weights."""
    w = Levels(*far_below(n, depth), new=new)
    q = w.levels(16)
    out, lse = attend(qe, form, w, q)
    check(out, lse, w.attention_within(q, weight), 1)


@pytest.mark.parametrize("form,new,weight", FORMS[:4])
@pytest.mark.parametrize("depth", [15.87, 20.6, 21.5])
def test_the_first_key_far_above_30000(qe, form, new, weight, depth):  # noqa: F811
    """As long texts have it: the others together weigh a few hundredths of the first, or half of it.  300 sequences, so
    that a block takes whole ones."""
    w = Levels(*far_below(30000, depth, every=30000), new=new, copies=300)
    w.v[0][:] = np.where(w.v[0] != 0, w.v[0] / np.float16(20000), 0)
    w.store(0)
    q = w.levels(16)
    out, lse = attend(qe, form, w, q)
    check(out, lse, w.attention_within(q, weight), 300)


@pytest.mark.parametrize("form,new,weight", FORMS)
@pytest.mark.parametrize("copies", [1, 300])
@pytest.mark.parametrize("depth", [12.1, 18.1, 20.1, 24.1])
def test_a_key_far_above_the_ones_just_weighed(qe, form, new, weight, copies, depth):  # noqa: F811
    """Keys 0 to 31 set a reference value, those of 32 to 63 lie as far above it as they may, and key 70 is `depth` octaves
    above them: what was weighed before counts that much less."""
    if new == 100 and copies > 1:
        copies = 40
    level, value = far_below(300, depth + 7.8, every=300)
    level[0], value[0] = level[1], value[1]
    level[32:64] = -depth / (16 * OCTAVE)
    level[70], value[70] = 0, 0
    w = Levels(level, value, new=new, copies=copies)
    q = w.levels(16)
    out, lse = attend(qe, form, w, q)
    check(out, lse, w.attention_within(q, weight), copies)
