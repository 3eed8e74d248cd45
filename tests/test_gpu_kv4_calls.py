"""Calls of the 4-bit cache kernels that their documentation allows and that reach other
code than the usual ones (definition and tolerances: kv4_reference.py)."""
import numpy as np
import pytest
import torch

import kv4_reference as ref
from helpers import dev, empty, host
from test_gpu_kv4 import _cache, _check, _ctl, _decode, _prefill, qe, workspace

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,base", [(1, 700), (40, 1200), (600, 300)])
def test_outputs_in_the_place_of_q(qe, workspace, T, base):
    rng = np.random.default_rng(T)
    nq, nkv, ms = 12, 2, 2048
    kv = _cache(rng, nkv, ms, base + T)
    q = rng.standard_normal((T, nq * 128)).astype(np.float16)
    apart, _ = _prefill(qe, kv, q, T, nq, base, None, ms)
    x = dev(q)
    qe.launch_attention_gqa_prefill_kv4(x, dev(kv[0]), dev(kv[1]), x, _ctl(base), None, T, num_q_heads=nq,
                                        num_kv_heads=nkv, max_seq_len=ms, hidden_size=nq * 128)
    assert np.array_equal(host(x).view(np.uint16), apart.view(np.uint16))
    _check(qe, kv, q, T, nq, base, [0] * nkv, ms, apart)
    one, ws = dev(q[-1]), empty(qe.kv4_decode_workspace_bytes(nq, ms), torch.uint8)
    qe.launch_attention_gqa_flash_decode_kv4(one, dev(kv[0]), dev(kv[1]), ws, one, _ctl(base + T - 1), None, None, nq, nkv,
                                             max_seq_len=ms)
    assert np.array_equal(host(one), _decode(qe, kv, q[-1], nq, base + T - 1, None, ms))
