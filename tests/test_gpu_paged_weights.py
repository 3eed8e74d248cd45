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
