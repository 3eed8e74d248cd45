"""Calls on the paged cache with no sequences or no rows, whose arrays are empty: nothing to do, whatever the addresses."""
import pytest

import test_paged_refusals as refusals
from test_paged_refusals import P, _at, _batch, _cache, qe  # noqa: F401 (qe: a fixture)


@pytest.mark.parametrize("name", ["append", "decode", "prefill", "bounds", "select", "sparse"])
def test_no_sequences_without_arrays(qe, name):  # noqa: F811
    call = refusals._calls(qe)[name]
    empty = {"seqs": 0, "table": None, "context": None}
    assert call(_at(_cache(qe)), _at(_batch(qe, tokens=0, **empty))) == 0
    if name != "decode":  # rows of no sequence
        assert call(_at(_cache(qe)), _at(_batch(qe, tokens=5, starts=4 * P, **empty))) == 0
    refusals._says(qe, call(_at(_cache(qe, k=None)), _at(_batch(qe, tokens=0, **empty))), "NULL")


@pytest.mark.parametrize("batch", [{"seqs": 0, "tokens": 0}, {"seqs": 4, "tokens": 0, "starts": 4 * P}])
def test_lists_without_rows(qe, batch):  # noqa: F811
    """Empty tensors for everything that has rows."""
    f = qe.lib().qe_launch_attention_gqa_paged_sparse
    assert f(None, _at(_cache(qe)), _at(_batch(qe, **batch)), None, None, None, None, None, 12, 4) == 0


@pytest.mark.gpu
def test_no_sequences_from_python(qe):  # noqa: F811
    """Tensors without elements have no address."""
    import torch
    f16 = lambda *s: torch.zeros(s, dtype=torch.float16, device="cuda")  # noqa: E731
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
    k, v = f16(4, 2, 16, 128), f16(4, 2, 16, 128)
    cache = qe.paged_cache(k, v)
    q, kk = f16(0, 12, 128), f16(0, 2, 128)
    bounds, steps = torch.zeros((4, 2, 256), dtype=torch.int8, device="cuda"), torch.zeros((4, 2), device="cuda")
    ws = torch.zeros(max(qe.paged_decode_workspace_bytes(0), qe.paged_prefill_workspace_bytes(0)), dtype=torch.uint8, device="cuda")
    for batch, single in ((qe.paged_batch(i32(0, 8), i32(0)), True), (qe.paged_batch(i32(0, 8), i32(0), i32(1), 0), False)):
        qe.launch_qkv_norm_rope_paged_append(q, q, kk, kk, None, None, None, None, None, None, cache, batch)
        if single:
            qe.launch_attention_gqa_paged_decode(q, cache, batch, ws, q)
        qe.launch_attention_gqa_paged_prefill(q, cache, batch, ws, q)
        qe.launch_paged_key_bounds(cache, batch, bounds, steps)
        qe.launch_paged_select(q, cache, batch, bounds, steps, i32(0, 2, 4), i32(0), num_selected=4)
        qe.launch_attention_gqa_paged_sparse(q, cache, batch, i32(0, 2, 4), ws, q, num_selected=4)
    torch.cuda.synchronize()
    assert not k.any() and not v.any()
