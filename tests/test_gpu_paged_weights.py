"""In how many bits attention on the paged cache holds softmax weights: scores are exact and the values nearly cancel, so what
the weights are rounded to shows (test_paged_levels.py: one fp16 number in place of two does)."""
import numpy as np
import pytest

from paged_levels import FP16, TWO_FP16, Levels, cancelling, check, odd_weights
from test_gpu_paged_attention import attend, qe  # noqa: F401 (qe: a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("form,new,weight", [("decode", 1, TWO_FP16), ("sparse", 1, TWO_FP16), ("sparse", 7, TWO_FP16), ("prefill", 2, TWO_FP16),
                                             ("prefill", 9, FP16), ("prefill", 100, FP16)])
@pytest.mark.parametrize("n,page,copies", [(1, 16, 1), (64, 16, 3), (700, 64, 1), (700, 16, 40), (1501, 128, 2)])
def test_weights(qe, form, new, weight, n, page, copies):  # noqa: F811
    n = max(n, new)
    q0 = odd_weights(6)
    w = Levels(*cancelling(n, q0), new=new, page=page, copies=copies)
    q = w.levels(np.tile(q0, 2))
    out, lse = attend(qe, form, w, q)
    check(out, lse, w.attention_within(q, weight), copies)


@pytest.mark.parametrize("copies,pad,weight", [(1, 0, TWO_FP16), (1, 3, FP16), (2, 3, TWO_FP16)])
def test_weights_in_a_padded_batch(qe, copies, pad, weight):  # noqa: F811
    """Two tokens and 12 rows of a kv head each: a lone sequence counts the rows behind it, several do not."""
    q0 = odd_weights(6)
    w = Levels(*cancelling(700, q0), new=2, copies=copies)
    q = np.pad(w.levels(np.tile(q0, 2)), ((0, pad), (0, 0), (0, 0)))
    w.rows += pad
    out, lse = attend(qe, "prefill", w, q)
    live = 2 * copies
    assert np.all(out[live:] == -7) and np.all(lse[live:] == -7)
    check(out[:live], lse[:live], w.attention_within(q, weight), copies)
