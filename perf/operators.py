"""Performance cases of a bounded 4-bit key/value cache and of scoring: what a long session of the engine does.

Five operators, each through the launcher API (qe_amd.launch_*):

  append    the K and V rows of new tokens, biased and rotated, stored in 4 bits; the q rows rotated
  decode    attention of one token over the 4-bit cache, with or without the accumulated weight of every cache row
  prefill   causal attention of the rows of a chunk over the 4-bit cache, with or without the accumulated weights
  evict     the cache rows with the least accumulated weight leave; the rest move up, in their order
  logprobs  log probabilities of given tokens, the entropy and the most likely alternatives, from rows of logits

A cache row of one head holds 128 values in 80 bytes: sixteen 32-bit words of eight nibbles (element 8 w + j of word w
at bit 16 * (j % 2) + 4 * (j // 2)), then four pairs (scale, low), fp16, one for every 32 elements.  A nibble n stands
for the fp16 value n * scale + low.  The row of position p is p - evicted, `evicted` being a count per key/value head.

Sizes are those of the engine's default configuration (12 query and 2 key/value heads of 128, vocabulary 151936);
drawn cases also take other head counts the launchers accept.
"""
from __future__ import annotations

import math
import os
import sys

import numpy as np
import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_PKG = os.path.join(_ROOT, "qwen-engine_amd")

NQ, NKV, HD, V = 12, 2, 128, 151936
ROW = 80  # bytes of a cache row of one head
THETA = 1000000.0
DEV = "cuda"


def listed():
    return [
        # every generated token, in every layer: launching it is what it costs
        {"name": "append_1", "kind": "append", "tokens": 1, "pos": 1000, "evicted": 0, "nq": NQ, "nkv": NKV,
         "max_seq": 4096, "bias": True, "rot": 128},
        # a pasted page late in a session whose cache is kept short: positions far beyond the rows
        {"name": "append_1000_far", "kind": "append", "tokens": 1000, "pos": 90000, "evicted": 87000, "nq": NQ,
         "nkv": NKV, "max_seq": 4096, "bias": True, "rot": 128},
        # a token early in a conversation
        {"name": "decode_300", "kind": "decode", "pos": 299, "evicted": 0, "nq": NQ, "nkv": NKV, "max_seq": 4096,
         "weights": False},
        # a token deep in a conversation that keeps count of what it looks at
        {"name": "decode_16k_weights", "kind": "decode", "pos": 16000, "evicted": 0, "nq": NQ, "nkv": NKV,
         "max_seq": 32768, "weights": True},
        # a token after a book: reading the cache is all there is
        {"name": "decode_131k", "kind": "decode", "pos": 130999, "evicted": 0, "nq": NQ, "nkv": NKV,
         "max_seq": 131072, "weights": False},
        # a short user turn on top of a longer history
        {"name": "prefill_17_at_1200", "kind": "prefill", "tokens": 17, "pos": 1200, "evicted": 0, "nq": NQ,
         "nkv": NKV, "max_seq": 4096, "weights": False},
        # a page read into a bounded cache, counting
        {"name": "prefill_1000_weights", "kind": "prefill", "tokens": 1000, "pos": 20000, "evicted": 17100, "nq": NQ,
         "nkv": NKV, "max_seq": 4096, "weights": True},
        # one chunk late in a long document
        {"name": "prefill_2048_at_14k", "kind": "prefill", "tokens": 2048, "pos": 14000, "evicted": 0, "nq": NQ,
         "nkv": NKV, "max_seq": 32768, "weights": False},
        # a full cache of the default engine is halved
        {"name": "evict_4k", "kind": "evict", "rows": 4096, "keep": 2048, "sinks": 4, "recent": 512, "nkv": NKV,
         "max_seq": 4096},
        # a long cache with many heads down to a quarter
        {"name": "evict_32k", "kind": "evict", "rows": 32000, "keep": 8000, "sinks": 4, "recent": 1000, "nkv": 8,
         "max_seq": 32768},
        # the alternatives shown beside one generated token
        {"name": "logprobs_1", "kind": "logprobs", "rows": 1, "vocab": V, "stride": V, "top": 20},
        # perplexity of a prefill chunk
        {"name": "logprobs_1024", "kind": "logprobs", "rows": 1024, "vocab": V, "stride": V, "top": 5},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "decode", "decode", "prefill", "prefill", "evict", "logprobs"])
    nkv = rng.choice([NKV, NKV, 1, 3, 4, 8])
    nq = nkv * rng.choice([6, 6, 1, 2, 4, 5, 7, 8])
    if kind == "append":
        tokens, past = _log_int(rng, 1, 2048), _log_int(rng, 1, 30000)
        evicted = rng.choice([0, _log_int(rng, 10, 200000)])
        return {"kind": kind, "tokens": tokens, "pos": past + evicted, "evicted": evicted, "nq": nq, "nkv": nkv,
                "max_seq": tokens + past + rng.randint(0, 1000), "bias": rng.random() < 0.5,
                "rot": rng.choice([128, 128, 64])}
    if kind == "decode":
        past = _log_int(rng, 1, 131000)
        while nkv * past > 2 * 131000:
            past //= 2
        evicted = rng.choice([0, _log_int(rng, 10, 200000)])
        return {"kind": kind, "pos": past + evicted, "evicted": evicted, "nq": nq, "nkv": nkv,
                "max_seq": past + rng.randint(1, 5000), "weights": rng.random() < 0.5}
    if kind == "prefill":
        tokens, past = _log_int(rng, 2, 2048), rng.choice([0, _log_int(rng, 1, 15000)])
        while nq * tokens * (past + tokens) > 12 * 2048 * 16048:
            tokens = (tokens + 1) // 2
        evicted = rng.choice([0, _log_int(rng, 10, 200000)])
        return {"kind": kind, "tokens": tokens, "pos": past + evicted, "evicted": evicted, "nq": nq, "nkv": nkv,
                "max_seq": tokens + past + rng.randint(0, 5000), "weights": rng.random() < 0.5}
    if kind == "evict":
        rows = _log_int(rng, 100, 60000)
        keep = rng.randint(rows // 10 + 1, rows)
        recent = rng.randint(0, keep)
        return {"kind": kind, "rows": rows, "keep": keep, "sinks": rng.randint(0, min(8, keep - recent)),
                "recent": recent, "nkv": nkv, "max_seq": rows + rng.randint(0, 1000)}
    vocab = rng.choice([V, _log_int(rng, 1000, 200000)])
    return {"kind": kind, "rows": _log_int(rng, 1, 700), "vocab": vocab, "stride": vocab + rng.choice([0, 0, 1, 64]),
            "top": rng.choice([0, 1, 5, 8, 20, 32])}


# ---- inputs ------------------------------------------------------------------------------------------------------
class _Rand:
    def __init__(self, seed):
        self.gen = torch.Generator(device=DEV)
        self.gen.manual_seed(seed)

    def normal(self, *shape, std=1.0, mean=0.0):
        return torch.randn(shape, device=DEV, generator=self.gen) * std + mean

    def uniform(self, *shape):
        return torch.rand(shape, device=DEV, generator=self.gen)

    def ints(self, lo, hi, *shape):
        return torch.randint(lo, hi, shape, device=DEV, generator=self.gen)


_SHIFTS = [0, 16, 4, 20, 8, 24, 12, 28]


def _quantize(x):
    """Rows of 128 values (fp32) as cache rows: [..., 128] -> uint8 [..., 80]."""
    g = x.reshape(*x.shape[:-1], 4, 32)
    low = g.amin(-1).half()
    scale = ((g.amax(-1) - low.float()) / 15.0).half()
    n = (g - low.float()[..., None]) / scale.float()[..., None]
    n = torch.where(scale[..., None] > 0, torch.round(n).clamp(0, 15), torch.zeros_like(n))
    shifts = torch.tensor(_SHIFTS, dtype=torch.int64, device=x.device)
    words = (n.to(torch.int64).reshape(*x.shape[:-1], 16, 8) << shifts).sum(-1)
    words = torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32)
    return torch.cat([words.contiguous().view(torch.uint8).reshape(*x.shape[:-1], 64),
                      torch.stack([scale, low], -1).contiguous().view(torch.uint8).reshape(*x.shape[:-1], 16)], -1)


def _dequantize(rows):
    """The values that cache rows stand for: uint8 [..., 80] -> fp16 [..., 128]."""
    words = rows[..., :64].contiguous().view(torch.int32)
    shifts = torch.tensor(_SHIFTS, dtype=torch.int32, device=rows.device)
    n = ((words[..., None] >> shifts) & 15).float().reshape(*rows.shape[:-1], 4, 32)
    params = rows[..., 64:].contiguous().view(torch.float16).reshape(*rows.shape[:-1], 4, 2).float()
    return (n * params[..., :1] + params[..., 1:]).half().reshape(*rows.shape[:-1], HD)


def _cache(r, nkv, max_seq, live):
    """A K and a V cache with `live` rows: K with the offsets between channels that keys have; the rest is rubbish."""
    k = torch.randint(0, 256, (nkv, max_seq, ROW), dtype=torch.uint8, device=DEV, generator=r.gen)
    v = torch.randint(0, 256, (nkv, max_seq, ROW), dtype=torch.uint8, device=DEV, generator=r.gen)
    k[:, :live] = _quantize(r.normal(nkv, live, HD) + r.normal(nkv, 1, HD, std=2.0))
    v[:, :live] = _quantize(r.normal(nkv, live, HD))
    return k, v


def _control(pos):
    c = torch.zeros(64, dtype=torch.int32, device=DEV)
    c[1] = pos
    return c


def prepare(case, seed):
    c, r = dict(case), _Rand(seed)
    s = {"case": c, "keep": {}}
    kind = c["kind"]
    if kind == "logprobs":
        x = r.normal(c["rows"], c["stride"], std=3.0).half()
        x[r.uniform(c["rows"], c["stride"]) < 0.01] = float("-inf")  # banned tokens
        s["logits"] = x[:, :c["vocab"]]
        best = s["logits"].argmax(-1)
        other = r.ints(0, c["vocab"], c["rows"])
        s["ids"] = torch.where(r.uniform(c["rows"]) < 0.5, best, other).to(torch.int32)
        s["logprob"], s["entropy"] = (torch.empty(c["rows"], device=DEV) for _ in range(2))
        s["top_logprob"] = torch.empty((c["rows"], c["top"]), device=DEV)
        s["top_ids"] = torch.empty((c["rows"], c["top"]), dtype=torch.int32, device=DEV)
        return s
    nkv, ms = c["nkv"], c["max_seq"]
    if kind == "evict":
        n, keep = c["rows"], c["keep"]
        s["k"], s["v"] = _cache(r, nkv, ms, n)
        s["control"] = _control(n + 7)
        s["evicted"] = torch.full((nkv,), 7, dtype=torch.int32, device=DEV)
        w = torch.exp(r.normal(nkv, ms, std=2.0))
        s["weights"] = torch.where(r.uniform(nkv, ms) < 0.1, torch.zeros_like(w), w)  # some rows nobody looked at
        s["k_out"], s["v_out"] = torch.empty_like(s["k"]), torch.empty_like(s["v"])
        s["weights_out"], s["evicted_out"] = torch.zeros_like(s["weights"]), torch.empty_like(s["evicted"])
        s["kept"] = torch.empty((nkv, keep), dtype=torch.int32, device=DEV)
        s["k16"], s["v16"] = (torch.empty((nkv, keep, HD), dtype=torch.float16, device=DEV) for _ in range(2))
        return s
    nq, t = c["nq"], c.get("tokens", 1)
    row0 = c["pos"] - c["evicted"]
    s["control"] = _control(c["pos"])
    s["evicted"] = torch.full((nkv,), c["evicted"], dtype=torch.int32, device=DEV)
    if kind == "append":
        s["q"], s["k_in"], s["v_in"] = (r.normal(t, n * HD).half() for n in (nq, nkv, nkv))
        s["bias"] = [r.normal(n * HD, std=sd).half() if c["bias"] else None
                     for n, sd in ((nq, 1.0), (nkv, 4.0), (nkv, 0.2))]
        s["k"], s["v"] = (torch.zeros((nkv, ms, ROW), dtype=torch.uint8, device=DEV) for _ in range(2))
        s["q_out"] = torch.empty_like(s["q"])
        s["k16"], s["v16"] = (torch.empty((nkv, t, HD), dtype=torch.float16, device=DEV) for _ in range(2))
        return s
    s["k"], s["v"] = _cache(r, nkv, ms, row0 + t)
    s["q"] = r.normal(t, nq * HD, std=1.5).half()
    s["out"] = torch.empty_like(s["q"])
    if c["weights"]:
        s["weights"] = torch.exp(r.normal(nkv, ms))
        s["weights_out"] = torch.empty_like(s["weights"])
        s["lse"] = torch.empty((t, nq), device=DEV)
    return s


# ---- plain forms ---------------------------------------------------------------------------------------------------
def _rope(x, pos, rot):
    """Rotates [T, heads, 128] (fp32) by the angles of positions pos, pos + 1, ...: angles in 64 bits."""
    i = torch.arange(rot // 2, dtype=torch.float64, device=x.device)
    p = torch.arange(pos, pos + x.shape[0], dtype=torch.float64, device=x.device)
    a = p[:, None] * THETA ** (-2.0 * i / rot)
    cs, sn = torch.cos(a).float()[:, None], torch.sin(a).float()[:, None]
    x0, x1 = x[..., :rot // 2], x[..., rot // 2:rot]
    return torch.cat([x0 * cs - x1 * sn, x1 * cs + x0 * sn, x[..., rot:]], -1)


def _plain_append(s):
    c = s["case"]
    q, k, v = (x.float().reshape(c["tokens"], -1, HD) for x in (s["q"], s["k_in"], s["v_in"]))
    if c["bias"]:
        q, k, v = (x + b.float().reshape(-1, HD) for x, b in zip((q, k, v), s["bias"]))
    row0 = c["pos"] - c["evicted"]
    q, k = _rope(q, c["pos"], c["rot"]), _rope(k, c["pos"], c["rot"])
    s["k"][:, row0:row0 + c["tokens"]] = _quantize(k).transpose(0, 1)
    s["v"][:, row0:row0 + c["tokens"]] = _quantize(v).transpose(0, 1)
    return {"q": q.half().reshape(c["tokens"], -1), "k": _dequantize(s["k"][:, row0:row0 + c["tokens"]]),
            "v": _dequantize(s["v"][:, row0:row0 + c["tokens"]])}


def _plain_attention(s):
    c = s["case"]
    t, nkv, group, row0 = c.get("tokens", 1), c["nkv"], c["nq"] // c["nkv"], c["pos"] - c["evicted"]
    live = row0 + t
    k, v = _dequantize(s["k"][:, :live]).float(), _dequantize(s["v"][:, :live]).float()
    q = s["q"].float().reshape(t, nkv, group, HD).permute(1, 0, 2, 3).reshape(nkv, t * group, HD)
    x = torch.matmul(q, k.transpose(1, 2)) / math.sqrt(HD)
    last = row0 + torch.arange(t, device=x.device).repeat_interleave(group)
    x = x.masked_fill(torch.arange(live, device=x.device) > last[:, None], float("-inf"))
    x = x - x.amax(-1, keepdim=True)
    p = torch.exp(x)
    p = p / p.sum(-1, keepdim=True)
    o = torch.matmul(p, v).reshape(nkv, t, group, HD).permute(1, 0, 2, 3).reshape(t, -1)
    out = {"out": o.half()}
    if c["weights"]:
        seen = s["weights"][:, :live].clone()
        seen[:, row0:] = 0  # the rows of these tokens are new
        s["weights_out"][:, :live] = seen + p.sum(1)
        out["weights"] = s["weights_out"][:, :live]
    return out


def _plain_evict(s):
    c = s["case"]
    n, keep = c["rows"], c["keep"]
    m = min(n, keep)
    w = s["weights"][:, :n]
    at = torch.arange(n, device=w.device)
    safe = (at < c["sinks"]) | (at >= n - c["recent"])
    order = torch.argsort(torch.where(safe, torch.full_like(w, float("inf")), w), dim=1, descending=True, stable=True)
    kept = torch.sort(order[:, :m], dim=1).values
    k = torch.gather(s["k"], 1, kept[..., None].expand(-1, -1, ROW))
    v = torch.gather(s["v"], 1, kept[..., None].expand(-1, -1, ROW))
    s["k_out"][:, :m], s["v_out"][:, :m] = k, v
    s["weights_out"][:, :m] = torch.gather(w, 1, kept)
    s["weights_out"][:, m:n] = 0
    s["kept"][:, :m] = kept.to(torch.int32)
    s["kept"][:, m:] = -1
    torch.add(s["evicted"], n - m, out=s["evicted_out"])
    return {"kept": s["kept"], "evicted": s["evicted_out"], "weights": s["weights_out"][:, :n], "k": _dequantize(k),
            "v": _dequantize(v)}


def _plain_logprobs(s):
    c = s["case"]
    x = s["logits"].float()
    m = x.amax(-1, keepdim=True)
    d = x - m
    e = torch.exp(d)
    total = e.sum(-1, keepdim=True)
    log_total = torch.log(total)
    ids = s["ids"].long()[:, None]
    entropy = log_total - torch.where(e > 0, e * d, torch.zeros_like(e)).sum(-1, keepdim=True) / total
    out = {"logprob": (d.gather(1, ids) - log_total)[:, 0], "entropy": entropy[:, 0]}
    if c["top"]:
        # one whole number for a (logit, index), the lowest index the largest: ties are settled
        b = s["logits"].contiguous().view(torch.int16).to(torch.int64)
        b = torch.where(b < 0, -(b & 0x7FFF), b)
        key = b * (1 << 32) + ((1 << 31) - torch.arange(c["vocab"], device=b.device))
        at = (1 << 31) - (torch.topk(key, c["top"], dim=1).values & 0xFFFFFFFF)
        out["top_logprob"] = d.gather(1, at) - log_total
        out["top_ids"] = at.to(torch.int32)
    return out


# ---- the framework's calls --------------------------------------------------------------------------------------------
def _lib():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import qe_amd
    return qe_amd


def _workspace(s, nbytes):
    """The program's workspace for a call, kept between calls."""
    if "ws" not in s["keep"]:
        s["keep"]["ws"] = torch.empty(max(nbytes, 16), dtype=torch.uint8, device=DEV)
    return s["keep"]["ws"]


def _own_run(s):
    qe, c = _lib(), s["case"]
    kind = c["kind"]
    if kind == "append":
        b = s["bias"]
        qe.launch_qkv_bias_rope_kv4_append(s["q"], s["q_out"], s["k_in"], s["v_in"], b[0], b[1], b[2], s["k"], s["v"],
                                           s["control"], s["evicted"], c["tokens"], num_q_heads=c["nq"],
                                           num_kv_heads=c["nkv"], max_seq_len=c["max_seq"], rotary_dim=c["rot"],
                                           rope_theta=THETA)
        qe.launch_kv4_unpack(s["k"], s["v"], s["k16"], s["v16"], c["pos"] - c["evicted"], c["tokens"],
                             num_kv_heads=c["nkv"], max_seq_len=c["max_seq"])
        return {"q": s["q_out"], "k": s["k16"], "v": s["v16"]}
    if kind == "decode":
        ws = _workspace(s, qe.kv4_decode_workspace_bytes(c["nq"], c["max_seq"], c["weights"]))
        w = {"key_weights_in": s["weights"], "key_weights_out": s["weights_out"]} if c["weights"] else {}
        qe.launch_attention_gqa_flash_decode_kv4(s["q"], s["k"], s["v"], ws, s["out"], s["control"], s["evicted"],
                                                 num_q_heads=c["nq"], num_kv_heads=c["nkv"], max_seq_len=c["max_seq"],
                                                 **w)
        live = c["pos"] - c["evicted"] + 1
        return {"out": s["out"], "weights": s["weights_out"][:, :live]} if c["weights"] else {"out": s["out"]}
    if kind == "prefill":
        if not s["keep"]:
            qe.gemm_reserve_workspace()
            s["keep"]["reserved"] = True
        w = {"key_weights_in": s["weights"], "key_weights_out": s["weights_out"], "row_lse": s["lse"]} \
            if c["weights"] else {}
        qe.launch_attention_gqa_prefill_kv4(s["q"], s["k"], s["v"], s["out"], s["control"], s["evicted"], c["tokens"],
                                            num_q_heads=c["nq"], num_kv_heads=c["nkv"], max_seq_len=c["max_seq"],
                                            hidden_size=c["nq"] * HD, **w)
        live = c["pos"] - c["evicted"] + c["tokens"]
        return {"out": s["out"], "weights": s["weights_out"][:, :live]} if c["weights"] else {"out": s["out"]}
    if kind == "evict":
        m = min(c["rows"], c["keep"])
        qe.launch_kv4_evict(s["k"], s["v"], s["weights"], s["evicted"], s["k_out"], s["v_out"], s["weights_out"],
                            s["evicted_out"], s["kept"], s["control"], c["keep"], sinks=c["sinks"],
                            recent=c["recent"], num_kv_heads=c["nkv"], max_seq_len=c["max_seq"])
        qe.launch_kv4_unpack(s["k_out"], s["v_out"], s["k16"], s["v16"], 0, m, num_kv_heads=c["nkv"],
                             max_seq_len=c["max_seq"])
        return {"kept": s["kept"], "evicted": s["evicted_out"], "weights": s["weights_out"][:, :c["rows"]],
                "k": s["k16"], "v": s["v16"]}
    ws = _workspace(s, qe.token_logprobs_workspace_bytes(c["rows"], c["vocab"], c["top"]))
    out = {"logprob": s["logprob"], "entropy": s["entropy"]}
    if c["top"]:
        out |= {"top_logprob": s["top_logprob"], "top_ids": s["top_ids"]}
    qe.launch_token_logprobs(s["logits"], s["ids"], s["logprob"], s["entropy"], out.get("top_logprob"),
                             out.get("top_ids"), ws, c["rows"], vocab_size=c["vocab"], row_stride=c["stride"],
                             top_k=c["top"])
    return out


_PLAIN = {"append": _plain_append, "decode": _plain_attention, "prefill": _plain_attention, "evict": _plain_evict,
          "logprobs": _plain_logprobs}


def run(state):
    if own:
        return _own_run(state)
    return _PLAIN[state["case"]["kind"]](state)


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------
def _values(rows):
    """What cache rows stand for, byte by byte: uint8 array [..., 80] -> fp16 values as float64."""
    b = rows[..., :64].reshape(*rows.shape[:-1], 16, 4).astype(np.float64)
    lo, hi = np.mod(b, 16), np.floor(b / 16)
    # byte 0: elements 0, 2; byte 1: 4, 6; byte 2: 1, 3; byte 3: 5, 7
    n = np.stack([lo[..., 0], lo[..., 2], hi[..., 0], hi[..., 2], lo[..., 1], lo[..., 3], hi[..., 1], hi[..., 3]], -1)
    par = np.ascontiguousarray(rows[..., 64:]).view(np.float16).astype(np.float64)
    n = n.reshape(*rows.shape[:-1], 4, 32)
    return (n * par[..., 0::2, None] + par[..., 1::2, None]).astype(np.float16).astype(np.float64) \
        .reshape(*rows.shape[:-1], HD)


def _stored(x):
    """What float64 rows of 128 stand for once they are stored in 4 bits."""
    g = x.reshape(*x.shape[:-1], 4, 32)
    low = g.min(-1, keepdims=True).astype(np.float16).astype(np.float64)
    step = ((g.max(-1, keepdims=True) - low) / 15).astype(np.float16).astype(np.float64)
    n = np.clip(np.rint((g - low) / np.where(step > 0, step, 1)), 0, 15) * (step > 0)
    return (n * step + low).astype(np.float16).astype(np.float64).reshape(x.shape)


def _np(t):
    return t.cpu().numpy()


def exact(case, seed):
    c, s = dict(case), prepare(case, seed)
    kind = c["kind"]
    if kind == "append":
        rows = []
        for x, b, turn in zip((s["q"], s["k_in"], s["v_in"]), s["bias"], (True, True, False)):
            y = _np(x).astype(np.float64) + (_np(b).astype(np.float64) if b is not None else 0.0)
            y = y.reshape(c["tokens"], -1, HD)
            if turn:
                half = c["rot"] // 2
                angle = np.arange(c["pos"], c["pos"] + c["tokens"])[:, None] * np.power(THETA, -np.arange(half) / half)
                z = (y[..., :half] + 1j * y[..., half:2 * half]) * np.exp(1j * angle)[:, None]
                y = np.concatenate([z.real, z.imag, y[..., c["rot"]:]], -1)
            rows.append(y)
        return {"q": rows[0].reshape(c["tokens"], -1), "k": _stored(rows[1].transpose(1, 0, 2)),
                "v": _stored(rows[2].transpose(1, 0, 2))}
    if kind in ("decode", "prefill"):
        t, nkv, group = c.get("tokens", 1), c["nkv"], c["nq"] // c["nkv"]
        row0 = c["pos"] - c["evicted"]
        outs, seen = [], []
        for h in range(nkv):
            k, v = (torch.from_numpy(_values(_np(s[x][h, :row0 + t]))).to(DEV) for x in "kv")
            q = s["q"].double().reshape(t, nkv, group, HD)[:, h].reshape(t * group, HD)
            x = q @ k.T * HD ** -0.5
            x = torch.where(torch.arange(row0 + t, device=DEV)[None] <= row0 + torch.arange(t * group, device=DEV)[:, None]
                            // group, x, -torch.inf)
            p = torch.softmax(x, -1)
            outs.append((p @ v).reshape(t, group * HD))
            if c["weights"]:
                w = s["weights"][h, :row0 + t].double()
                w[row0:] = 0.0
                seen.append(w + p.sum(0))
        out = {"out": torch.cat(outs, 1)}
        return out | {"weights": torch.stack(seen)} if c["weights"] else out
    if kind == "evict":
        n, m = c["rows"], min(c["rows"], c["keep"])
        w = _np(s["weights"])[:, :n].astype(np.float64)
        rank = w.copy()
        rank[:, :c["sinks"]] = np.inf
        rank[:, n - c["recent"]:] = np.inf
        kept = np.stack([np.sort(np.lexsort((np.arange(n), -r))[:m]) for r in rank])
        moved = np.zeros_like(w)
        moved[:, :m] = np.take_along_axis(w, kept, 1)
        k, v = (np.stack([_values(_np(s[x][h])[kept[h]]) for h in range(c["nkv"])]) for x in "kv")
        return {"kept": None, "evicted": None, "weights": moved, "k": k, "v": v}
    x = s["logits"].double()
    lp = torch.log_softmax(x, -1)
    out = {"logprob": torch.gather(lp, 1, s["ids"].long()[:, None])[:, 0],
           "entropy": -torch.special.xlogy(lp.exp(), lp.exp()).sum(-1)}
    if c["top"]:
        out |= {"top_logprob": torch.sort(lp, -1, descending=True).values[:, :c["top"]], "top_ids": None}
    return out


# ---- work ----------------------------------------------------------------------------------------------------------
def work(case):
    c = case
    kind = c["kind"]
    if kind == "logprobs":
        n = c["rows"] * c["vocab"]
        return {"bytes": 2 * n + c["rows"] * (12 + 8 * c["top"]), "flops": 4 * n}
    nkv = c["nkv"]
    if kind == "evict":
        m = min(c["rows"], c["keep"])
        # every weight read, every kept row read, moved and read out again as fp16
        return {"bytes": nkv * (4 * c["rows"] + m * (2 * 2 * ROW + 4 + 4) + 4 * c["rows"] + m * 2 * 2 * HD),
                "flops": nkv * c["rows"]}
    t, nq = c.get("tokens", 1), c["nq"]
    if kind == "append":
        return {"bytes": t * (2 * 2 * nq * HD + 2 * 2 * nkv * HD + 2 * nkv * ROW + 2 * 2 * nkv * HD),
                "flops": t * HD * (4 * nq + 8 * nkv)}
    live = c["pos"] - c["evicted"] + t
    pairs = nq * (t * (live - t) + t * (t + 1) // 2)
    extra = 8 * nkv * live if c["weights"] else 0
    return {"bytes": 2 * nkv * live * ROW + 2 * 2 * t * nq * HD + extra,
            "flops": (4 + (2 if c["weights"] and t > 1 else 0)) * HD * pairs}
