"""The engine on a 4-bit cache, every layer of it: its launches made one by one with a cache of its own for each layer
give the same caches, hidden rows and logits bit for bit, and the attention of every layer is the definition's over the
rows that the engine's own caches hold (kv4_reference.py)."""
import numpy as np
import pytest
import torch

from helpers import dev, empty, host
from test_gpu_engine_kv4 import _engine, qe
from test_gpu_kv4 import _check

pytestmark = pytest.mark.gpu
HID, INTER, NQ, NKV, VOCAB, LAYERS = 768, 1024, 6, 2, 4096, 3


class OneByOne:
    """The engine's sequence of launches on copies of its weights."""

    def __init__(self, qe, e, max_seq):
        self.qe, self.ms = qe, max_seq
        f16, u32 = np.float16, np.uint32

        def mat(name, rows, k):
            return dev(e.read(name + "_w", u32, rows * k // 8)), dev(e.read(name + "_s", f16, rows * (k // 128)))
        self.embed = mat("embed", VOCAB, HID)
        self.final_norm = dev(e.read("final_norm", f16, HID))
        self.layers = []
        for i in range(LAYERS):
            at = f"layer{i}."
            t = {n: mat(at + n, rows, k) for n, rows, k in (("q", NQ * 128, HID), ("k", NKV * 128, HID), ("v", NKV * 128, HID),
                                                            ("o", HID, NQ * 128), ("gate_up", 2 * INTER, HID),
                                                            ("down", HID, INTER))}
            for n, size in (("ln1", HID), ("ln2", HID), ("q_bias", NQ * 128), ("k_bias", NKV * 128), ("v_bias", NKV * 128)):
                t[n] = dev(e.read(at + n, f16, size))
            t["kc"], t["vc"] = qe.kv4_cache(NKV, max_seq), qe.kv4_cache(NKV, max_seq)
            self.layers.append(t)
        self.ws = empty(qe.kv4_decode_workspace_bytes(NQ, max_seq), torch.uint8)
        self.q8 = empty(INTER, torch.int8), empty(INTER // 128, torch.float32), empty(INTER // 8, torch.int32)
        self.seen = []  # (position, q, out) of every layer of the last pass

    def _ctl(self, pos, token=0):
        raw = np.zeros(64, np.int32)
        raw[0], raw[1] = token, pos
        return dev(raw)

    def _qkv(self, t, T):
        out = [empty((T, n * 128), torch.float16) for n in (NQ, NKV, NKV)]
        return out, self.qe.make_qkv_view(*t["q"], out[0], *t["k"], out[1], *t["v"], out[2])

    def _append(self, t, qkv, ctl, T):
        q, k, v = qkv
        self.qe.launch_qkv_bias_rope_kv4_append(q, q, k, v, t["q_bias"], t["k_bias"], t["v_bias"], t["kc"], t["vc"], ctl,
                                                None, T, None, NQ, NKV, max_seq_len=self.ms, rotary_dim=128)

    def chunk(self, tokens, pos):
        qe, T = self.qe, len(tokens)
        ctl, x, y, mlp = self._ctl(pos), empty((T, HID), torch.float16), empty((T, HID), torch.float16), empty((T, INTER), torch.float16)
        qe.launch_embed_lookup_w4a16(*self.embed, dev(np.array(tokens, np.int32)), x, None, T, hidden_size=HID)
        self.seen = []
        for t in self.layers:
            qe.launch_rmsnorm_fp16(x, t["ln1"], y, T, hidden_size=HID)
            qkv, view = self._qkv(t, T)
            qe.launch_gemm_prefill_qkv_w4a16(view, y, T, None, HID, NQ, NKV)
            self._append(t, qkv, ctl, T)
            out = empty((T, NQ * 128), torch.float16)
            qe.launch_attention_gqa_prefill_kv4(qkv[0], t["kc"], t["vc"], out, ctl, None, T, None, NQ, NKV,
                                                max_seq_len=self.ms, hidden_size=NQ * 128)
            self.seen.append((pos, host(qkv[0]), host(out)))
            qe.launch_gemm_prefill_w4a16(*t["o"], out, x, x, T, HID, NQ * 128)
            qe.launch_rmsnorm_fp16(x, t["ln2"], y, T, hidden_size=HID)
            qe.launch_gemm_prefill_dual_gate_up_swiglu_w4a16(*t["gate_up"], y, mlp, T, None, HID, INTER)
            qe.launch_gemm_prefill_w4a16(*t["down"], mlp, x, x, T, HID, INTER)
        return x

    def token(self, token, pos):
        qe, q8 = self.qe, self.q8
        ctl, x, mlp = self._ctl(pos, token), empty(HID, torch.float16), empty(INTER, torch.float16)
        qe.launch_embed_lookup_w4a16(*self.embed, None, x, ctl, 1, hidden_size=HID)
        self.seen = []
        for t in self.layers:
            qe.launch_rmsnorm_q8_1(x, t["ln1"], None, *q8, hidden_size=HID)
            qkv, view = self._qkv(t, 1)
            qe.launch_gemv_qkv_w4a8(view, *q8, None, HID, NQ, NKV)
            self._append(t, qkv, ctl, 1)
            out = empty((1, NQ * 128), torch.float16)
            qe.launch_attention_gqa_flash_decode_kv4(qkv[0], t["kc"], t["vc"], self.ws, out, ctl, None, None, NQ, NKV,
                                                     max_seq_len=self.ms, out_q8=q8[0], out_scale=q8[1], out_sum8=q8[2])
            self.seen.append((pos, host(qkv[0]), host(out)))
            qe.launch_gemv_w4a8(*t["o"], *q8, x, x, HID, NQ * 128)
            qe.launch_rmsnorm_q8_1(x, t["ln2"], None, *q8, hidden_size=HID)
            qe.launch_gemv_dual_gate_up_swiglu_w4a8(*t["gate_up"], *q8, mlp, HID, INTER)
            qe.launch_quantize_fp16_to_q8_1(mlp, *q8, INTER)
            qe.launch_gemv_w4a8(*t["down"], *q8, x, x, HID, INTER)
        return x

    def logits(self, row):
        out = empty(VOCAB, torch.float16)
        self.qe.launch_rmsnorm_q8_1(row, self.final_norm, None, *self.q8, hidden_size=HID)
        self.qe.launch_gemv_w4a8(*self.embed, *self.q8, None, out, VOCAB, HID)
        return host(out).view(np.uint16)


@pytest.mark.parametrize("max_seq,chunk,n", [(256, 64, 150), (2048, 512, 1300)])
def test_every_layer(qe, max_seq, chunk, n):
    prompt, steps = [(i * 37 % 3000) + 100 for i in range(n)], 5
    qe.set_tuning("engine_tiled_prefill", 0)  # prefill GEMMs on the layout that the weights are read back in
    try:
        e = _engine(qe, 1, chunk=chunk, fused=0, max_seq=max_seq)
    finally:
        qe.set_tuning("engine_tiled_prefill", 1)
    qe.gemm_reserve_workspace()  # as the engine's stream has one
    try:
        one = OneByOne(qe, e, max_seq)

        def caches_agree(T):
            size = LAYERS * NKV * max_seq * 80
            kv = [e.read(name, np.uint8, size).reshape(LAYERS, NKV, max_seq, 80) for name in ("kcache", "vcache")]
            for i, t in enumerate(one.layers):
                assert np.array_equal(kv[0][i], host(t["kc"])) and np.array_equal(kv[1][i], host(t["vc"])), f"layer {i}"
                pos, q, out = one.seen[i]
                _check(qe, np.stack([kv[0][i], kv[1][i]]), q, T, NQ, pos, [0] * NKV, max_seq, out, what=f"layer {i}")

        first = e.prefill(prompt)
        for start in range(0, n, chunk):
            x = one.chunk(prompt[start:start + chunk], start)
        last = n - start
        assert np.array_equal(e.read("hidden", np.uint16, last * HID), host(x).view(np.uint16).reshape(-1)[:last * HID])
        caches_agree(last)
        assert np.array_equal(e.logits().view(np.uint16), one.logits(x[last - 1]))
        tokens = [first] + e.decode(steps)
        for i in range(steps):
            x = one.token(tokens[i], n + i)
        caches_agree(1)
        assert np.array_equal(e.hidden_row0().view(np.uint16), host(x).view(np.uint16))
        assert np.array_equal(e.logits().view(np.uint16), one.logits(x))
    finally:
        qe.gemm_release_workspace()
        e.close()
