"""Performance cases of a paged key/value cache that many conversations share, and of attention to selected blocks of it.

Four operators, each through the launcher API (qe_amd.launch_*):

  append    the q, k and v rows of new tokens: bias, a norm for each head, rotation; K and V stored in pages
  decode    attention of one token of each sequence over its pages
  prefill   causal attention of the rows of chunks (and of single tokens among them) over their pages
  sparse    one step of block-sparse attention: the bounds of the pages that got new keys, the blocks that each row and
            key/value head selects by them, and attention to those blocks

A page holds `page` tokens of every key/value head: fp16 [key/value head][page][128].  Position p of sequence s is row
p % page of page block_table[s][p // page]; entries that are no page stand for positions nobody attends to.  The bounds
of a page and head are 128 highs and 128 lows in whole steps of m / 127, m being its largest absolute key value:
high = ceil(127 max / m), low = floor(127 min / m).  With qn = rint(127 q / m_h) for each q head, m_h its largest
absolute value, a block's score is m * max over the heads of m_h * sum max(qn high, qn low): whole numbers and two
products rounded to 32 bits, so that everyone selects the same blocks.

Head counts are those of the engine's default configuration (12 query and 2 key/value heads of 128); drawn cases also
take others.  Lengths are written "before+new", one for each sequence.
"""
from __future__ import annotations

import math
import os
import random
import sys

import numpy as np
import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_PKG = os.path.join(_ROOT, "qwen-engine_amd")

NQ, NKV, HD = 12, 2, 128
THETA = 1000000.0
EPS = 1e-6
DEV = "cuda"


def _spread(seed, count, low, high, new=1):
    """Lengths of `count` sequences, any between two bounds."""
    rng = random.Random(seed)
    return " ".join(f"{rng.randint(low, high)}+{new}" for _ in range(count))


def listed():
    heads = {"nq": NQ, "nkv": NKV}
    return [
        # one conversation, one token: launching it is what it costs
        {"name": "append_1", "kind": "append", "lens": "1000+1", "page": 64, "bias": True, "norm": False, "rot": 128,
         "inter": False, "far": 1.0, "joint": False, "pad": 0, **heads},
        # a token of each of 64 conversations far beyond the trained length, heads normed, in a batch padded to 72
        {"name": "append_64_far", "kind": "append", "lens": _spread(1, 64, 100, 120000), "page": 16, "bias": False,
         "norm": True, "rot": 128, "inter": False, "far": 4.0, "joint": True, "pad": 8, **heads},
        # prompts of several users read at once
        {"name": "append_6150", "kind": "append", "lens": "0+2500 700+1300 0+333 12000+2000 5+17", "page": 64,
         "bias": True, "norm": True, "rot": 64, "inter": True, "far": 1.0, "joint": False, "pad": 0, **heads},
        # a token early in the only conversation
        {"name": "decode_1_at_300", "kind": "decode", "lens": "299+1", "page": 64, "window": 0, "joint": False,
         "pad": 0, **heads},
        # a batch of 48 conversations, short and long ones
        {"name": "decode_48", "kind": "decode", "lens": _spread(2, 48, 200, 12000), "page": 16, "window": 0,
         "joint": True, "pad": 0, **heads},
        # one token after a book: reading the cache is all there is
        {"name": "decode_1_at_131k", "kind": "decode", "lens": "130999+1", "page": 64, "window": 0, "joint": False,
         "pad": 0, **heads},
        # a short user turn on top of a longer history
        {"name": "prefill_17_at_1200", "kind": "prefill", "lens": "1200+17", "page": 16, "window": 0, "joint": False,
         "pad": 0, **heads},
        # a scheduler's step: 40 conversations one token further, three prompts read beside them
        {"name": "prefill_mixed", "kind": "prefill", "lens": _spread(3, 40, 200, 6000) + " 0+700 0+1111 3000+300",
         "page": 32, "window": 0, "joint": True, "pad": 5, **heads},
        # one chunk late in a long document
        {"name": "prefill_2048_at_14k", "kind": "prefill", "lens": "14000+2048", "page": 64, "window": 0,
         "joint": False, "pad": 0, **heads},
        # one token after a book that looks at a sixty-fourth of it
        {"name": "sparse_1_at_131k", "kind": "sparse", "lens": "130999+1", "page": 64, "select": 32, "sinks": 1,
         "recent": 4, "joint": False, "pad": 0, **heads},
        # 32 long conversations
        {"name": "sparse_32_at_33k", "kind": "sparse", "lens": _spread(4, 32, 20000, 33000), "page": 64, "select": 32,
         "sinks": 1, "recent": 2, "joint": True, "pad": 0, **heads},
        # a question of 200 tokens about a long document
        {"name": "sparse_200_at_50k", "kind": "sparse", "lens": "50000+200", "page": 32, "select": 64, "sinks": 2,
         "recent": 4, "joint": False, "pad": 0, **heads},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _text(lens):
    return " ".join(f"{a}+{b}" for a, b in lens)


def draw(rng):
    kind = rng.choice(["append", "decode", "decode", "prefill", "prefill", "sparse", "sparse"])
    nkv = rng.choice([NKV, NKV, 1, 3, 4, 8])
    nq = nkv * rng.choice([6, 6, 1, 2, 4, 5, 7, 8, 16])
    c = {"kind": kind, "page": rng.choice([16, 32, 64, 64, 128, 256]), "joint": rng.random() < 0.5,
         "pad": rng.choice([0, 0, rng.randint(1, 9)]), "nq": nq, "nkv": nkv}
    if kind == "append":
        lens = [(rng.choice([0, _log_int(rng, 1, 120000)]), rng.choice([1, _log_int(rng, 1, 1500)]))
                for _ in range(_log_int(rng, 1, 64))]
        while sum(n for _, n in lens) * (nq + 2 * nkv) > 6150 * 16:
            lens.pop()
        if not lens:
            lens = [(_log_int(rng, 1, 30000), _log_int(rng, 1, 200))]
        far = rng.choice([1.0, 1.0, 4.0, rng.uniform(1.5, 16.0)])
        return {**c, "lens": _text(lens), "bias": rng.random() < 0.5, "norm": rng.random() < 0.5,
                "rot": rng.choice([128, 128, 64, 32, 80]), "inter": rng.random() < 0.3, "far": far}
    if kind == "decode":
        longest = _log_int(rng, 1, 131000)
        lens = [(rng.randint(longest // 8, longest), 1) for _ in range(_log_int(rng, 1, 64))]
        while nkv * sum(a for a, _ in lens) > 2 * 280000 and len(lens) > 1:
            lens.pop()
        while nkv * lens[0][0] > 2 * 280000:
            lens[0] = (lens[0][0] // 2, 1)
        return {**c, "lens": _text(lens), "window": rng.choice([0, 0, 0, _log_int(rng, 1, 8000)])}
    if kind == "prefill":
        lens = [(rng.choice([0, _log_int(rng, 1, 15000)]), rng.choice([1, _log_int(rng, 2, 2048), _log_int(rng, 2, 300)]))
                for _ in range(_log_int(rng, 1, 24))]

        def cost():
            return nq * sum(n * (a + n) for a, n in lens), nkv * sum(a + n for a, n in lens)
        while len(lens) > 1 and (cost()[0] > 6 * 2048 * 16048 or cost()[1] > 2 * 200000):
            lens.pop()
        while cost()[0] > 6 * 2048 * 16048:
            lens[0] = (lens[0][0] // 2, (lens[0][1] + 1) // 2)
        return {**c, "lens": _text(lens), "window": rng.choice([0, 0, 0, _log_int(rng, 1, 8000)])}
    select = rng.randint(1, 4096 // c["page"])
    recent = rng.randint(1, max(1, select // 4))
    c |= {"select": select, "recent": recent, "sinks": rng.randint(0, min(4, select - recent))}
    if rng.random() < 0.5:
        longest = _log_int(rng, 1000, 131000)
        lens = [(rng.randint(longest // 8, longest), 1) for _ in range(_log_int(rng, 1, 32))]
        while len(lens) > 1 and nkv * sum(a for a, _ in lens) > 2 * 280000:
            lens.pop()
        while nkv * lens[0][0] > 2 * 280000:
            lens[0] = (lens[0][0] // 2, 1)
    else:
        lens = [(_log_int(rng, 1000, 40000), _log_int(rng, 2, 200))]
        while nkv * lens[0][1] * select * c["page"] > 2 * 200 * 2048 and lens[0][1] > 1:
            lens[0] = (lens[0][0], lens[0][1] // 2)
    return {**c, "lens": _text(lens)}


# ---- inputs ------------------------------------------------------------------------------------------------------
class _Rand:
    def __init__(self, seed):
        self.gen = torch.Generator(device=DEV)
        self.gen.manual_seed(seed)

    def normal(self, *shape, std=1.0):
        return torch.randn(shape, device=DEV, generator=self.gen) * std

    def order(self, n):
        return torch.randperm(n, device=DEV, generator=self.gen)


def _lens(c):
    return [tuple(int(x) for x in w.split("+")) for w in c["lens"].split()]


def _rows(c):
    return sum(n for _, n in _lens(c)) + c["pad"]


def _turns(rot, far):
    """Turns a position for each rotated pair, and the factor on the rotated values.  For texts `far` times as long as
    the 32768 positions trained on: pairs that turn less than once in them are slowed down by `far`, those of more
    than 32 turns keep their pace, the ones between change over evenly; values grow by 0.1 ln(far) + 1."""
    i = np.arange(rot // 2, dtype=np.float64)
    turns = THETA ** (-2.0 * i / rot) / (2.0 * np.pi)
    if far <= 1.0:
        return turns, 1.0

    def at(n):  # the pair that turns n times
        return rot * np.log(32768.0 / (n * 2.0 * np.pi)) / (2.0 * np.log(THETA))
    first, last = max(np.floor(at(32.0)), 0.0), min(np.ceil(at(1.0)), rot - 1.0)
    slow = np.clip((i - first) / max(last - first, 0.001), 0.0, 1.0)
    return turns * (1.0 - slow) + turns / far * slow, 0.1 * math.log(far) + 1.0


def _pages(c, r, behind):
    """K and V pages, the table of every sequence.  Pages lie in any order; `behind` is what lies in rows in no use."""
    ps, nkv, lens = c["page"], c["nkv"], _lens(c)
    if c["kind"] == "append":  # the pages that the new tokens reach alone
        spans = [(a // ps, (a + n - 1) // ps + 1) for a, n in lens]
    else:
        spans = [(0, (a + n - 1) // ps + 1) for a, n in lens]
    total = sum(hi - lo for lo, hi in spans) + 3
    at = r.order(total).to(torch.int32)
    table = torch.full((len(lens) + c["pad"], max(hi for _, hi in spans) + 2), -1, dtype=torch.int32, device=DEV)
    used, rows = 0, torch.zeros((total, ps), dtype=torch.bool, device=DEV)
    for s, ((a, n), (lo, hi)) in enumerate(zip(lens, spans)):
        mine = at[used:used + hi - lo]
        used += hi - lo
        table[s, lo:hi] = mine
        full = torch.zeros((hi - lo) * ps, dtype=torch.bool, device=DEV)
        full[:a + n - lo * ps] = True
        rows[mine.long()] = full.reshape(-1, ps)
    pool = torch.empty((total, 2, nkv, ps, HD) if c["joint"] else (2, total, nkv, ps, HD), dtype=torch.float16, device=DEV)
    k, v = (pool[:, 0], pool[:, 1]) if c["joint"] else (pool[0], pool[1])
    level = r.normal(nkv, 1, HD, std=2.0)  # keys differ in level from channel to channel
    for i in range(0, total, 512):
        n = min(512, total - i)
        for x, lift in ((k, level), (v, 0.0)):
            y = (r.normal(n, nkv, ps, HD) + lift).half()
            y.masked_fill_(~rows[i:i + n, None, :, None], behind)
            x[i:i + n] = y
    return k, v, table


def prepare(case, seed):
    c, r = dict(case), _Rand(seed)
    lens, nq, nkv = _lens(c), c["nq"], c["nkv"]
    rows, seqs = _rows(c), len(lens) + c["pad"]
    s = {"case": c, "keep": {}}
    s["context"] = torch.tensor([a for a, _ in lens] + [-1] * c["pad"], dtype=torch.int32, device=DEV)
    starts = [0]
    for _, n in lens:
        starts.append(starts[-1] + n)
    s["starts"] = torch.tensor(starts + [starts[-1]] * c["pad"], dtype=torch.int32, device=DEV)
    # rows of no sequence lie behind the last one
    s["single"] = all(n == 1 for _, n in lens)
    s["seqs"], s["rows"] = seqs, rows
    s["k"], s["v"], s["table"] = _pages(c, r, 0.0 if c["kind"] == "append" else float("nan"))
    s["q"] = r.normal(rows, nq * HD, std=1.5).half()
    s["q_out"] = torch.zeros_like(s["q"])
    if c["kind"] == "append":
        s["k_in"], s["v_in"] = r.normal(rows, nkv * HD).half(), r.normal(rows, nkv * HD).half()
        s["bias"] = [r.normal(n * HD, std=sd).half() if c["bias"] else None
                     for n, sd in ((nq, 1.0), (nkv, 4.0), (nkv, 0.2))]
        s["norm"] = [(1.0 + r.normal(HD, std=0.3)).half() if c["norm"] else None for _ in range(2)]
        turns, s["scale"] = _turns(c["rot"], c["far"])
        s["turns"] = torch.from_numpy(turns).to(DEV)
        return s
    s["lse"] = torch.zeros((rows, nq), device=DEV)
    if c["kind"] == "sparse":
        total = s["k"].shape[0]
        s["bounds"] = torch.zeros((total, nkv, 2 * HD), dtype=torch.int8, device=DEV)
        s["step"] = torch.zeros((total, nkv), device=DEV)
        for i, (a, n) in enumerate(lens):  # pages that were full before
            ps = c["page"]
            pages = s["table"][i, :a // ps].long()
            for j in range(0, pages.numel(), 512):
                _bound_pages(s, pages[j:j + 512], None)
        s["selected"] = torch.zeros((rows, nkv, c["select"]), dtype=torch.int32, device=DEV)
    return s


# ---- plain forms ---------------------------------------------------------------------------------------------------
def _bound_pages(s, pages, live):
    """The bounds of some pages, of which `live` rows each are in use (None: all)."""
    x = s["k"][pages].float()
    if live is None:
        high, low = x.amax(2), x.amin(2)
    else:
        dead = (torch.arange(x.shape[2], device=DEV) >= live[:, None])[:, None, :, None]
        high = x.masked_fill(dead, float("-inf")).amax(2)
        low = x.masked_fill(dead, float("inf")).amin(2)
    m = torch.maximum(high.abs(), low.abs()).amax(-1)
    d = torch.where(m > 0, m, torch.ones_like(m))[..., None]
    s["bounds"][pages, :, :HD] = torch.ceil(high * 127.0 / d).to(torch.int8)
    s["bounds"][pages, :, HD:] = torch.floor(low * 127.0 / d).to(torch.int8)
    s["step"][pages] = m


def _plain_append(s):
    c = s["case"]
    rot, ps = c["rot"], c["page"]
    at = 0
    for i, (a, n) in enumerate(_lens(c)):
        rows = slice(at, at + n)
        at += n
        q, k, v = (x[rows].float().reshape(n, -1, HD) for x in (s["q"], s["k_in"], s["v_in"]))
        if c["bias"]:
            q, k, v = (x + b.float().reshape(-1, HD) for x, b in zip((q, k, v), s["bias"]))
        pos = torch.arange(a, a + n, device=DEV)
        angle = 2.0 * math.pi * torch.remainder(pos.double()[:, None] * s["turns"], 1.0)
        cs, sn = (s["scale"] * torch.cos(angle)).float()[:, None], (s["scale"] * torch.sin(angle)).float()[:, None]
        out = []
        for x, g in ((q, s["norm"][0]), (k, s["norm"][1])):
            if g is not None:
                x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * g.float()
            x0, x1 = (x[..., 0:rot:2], x[..., 1:rot:2]) if c["inter"] else (x[..., :rot // 2], x[..., rot // 2:rot])
            y = [x0 * cs - x1 * sn, x1 * cs + x0 * sn]
            y = torch.stack(y, -1).flatten(-2) if c["inter"] else torch.cat(y, -1)
            out.append(torch.cat([y, x[..., rot:]], -1))
        s["q_out"][rows] = out[0].half().reshape(n, -1)
        page = s["table"][i].long()[pos // ps]
        s["k"][page, :, pos % ps] = out[1].half()
        s["v"][page, :, pos % ps] = v.half()
    return {"q": s["q_out"], "k": s["k"], "v": s["v"]}


def _softmax(x, v):
    """Outputs and log sums of rows of scores."""
    m = x.amax(-1, keepdim=True)
    p = torch.exp(x - m)
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p / total, v), (m + torch.log(total))[..., 0]


def _plain_attention(s):
    c = s["case"]
    nkv, group, ps = c["nkv"], c["nq"] // c["nkv"], c["page"]
    at = 0
    for i, (a, n) in enumerate(_lens(c)):
        rows = slice(at, at + n)
        at += n
        first = max(0, a - c["window"] + 1) if c["window"] else 0
        first -= first % ps
        page = s["table"][i, first // ps:(a + n - 1) // ps + 1].long()
        k, v = (x[page].transpose(0, 1).reshape(nkv, -1, HD)[:, :a + n - first].float() for x in (s["k"], s["v"]))
        q = s["q"][rows].float().reshape(n, nkv, group, HD).permute(1, 0, 2, 3).reshape(nkv, n * group, HD)
        x = torch.matmul(q, k.transpose(1, 2).contiguous()) / math.sqrt(HD)
        own_pos = torch.arange(a, a + n, device=DEV).repeat_interleave(group)[:, None]
        pos = torch.arange(first, a + n, device=DEV)
        x = x.masked_fill(pos > own_pos, float("-inf"))
        if c["window"]:
            x = x.masked_fill(pos <= own_pos - c["window"], float("-inf"))
        o, lse = _softmax(x, v)
        s["q_out"][rows] = o.half().reshape(nkv, n, group, HD).permute(1, 0, 2, 3).reshape(n, -1)
        s["lse"][rows] = lse.reshape(nkv, n, group).permute(1, 0, 2).reshape(n, -1)
    return {"out": s["q_out"], "lse": s["lse"]}


def _plain_sparse(s):
    c = s["case"]
    nkv, group, ps, select = c["nkv"], c["nq"] // c["nkv"], c["page"], c["select"]
    at = 0
    for i, (a, n) in enumerate(_lens(c)):
        rows = slice(at, at + n)
        at += n
        nb = (a + n - 1) // ps + 1
        table = s["table"][i, :nb].long()
        new = torch.arange(a // ps, nb, device=DEV)
        _bound_pages(s, table[new], (a + n - new * ps).clamp(max=ps))
        q = s["q"][rows].float().reshape(n, nkv, group, HD).permute(1, 0, 2, 3)  # [kv head, row, q head, 128]
        m = q.abs().amax(-1)
        qn = torch.round(q * 127.0 / torch.where(m > 0, m, torch.ones_like(m))[..., None])
        qn = torch.cat([qn.clamp(min=0), qn.clamp(max=0)], -1).reshape(nkv, n * group, 2 * HD)
        b = s["bounds"][table].float().permute(1, 2, 0).contiguous()  # [kv head, 256, block]
        score = torch.matmul(qn, b).reshape(nkv, n, group, nb) * m[..., None]
        score = score.amax(2) * s["step"][table].T[:, None]  # [kv head, row, block]
        own_block = (torch.arange(a, a + n, device=DEV) // ps)[:, None]
        block = torch.arange(nb, device=DEV)
        score = score.masked_fill((block < c["sinks"]) | (block > own_block - c["recent"]), float("inf"))
        score = score.masked_fill(block > own_block, float("-inf"))
        best = torch.sort(score, dim=-1, descending=True, stable=True)
        ids = torch.where(best.values > float("-inf"), best.indices, nb)[..., :select]
        if nb < select:
            ids = torch.cat([ids, torch.full((nkv, n, select - nb), nb, device=DEV)], -1)
        ids = torch.sort(ids, dim=-1).values
        page = table[ids.clamp(max=nb - 1)]
        head = torch.arange(nkv, device=DEV)[:, None, None]
        k, v = (x[page, head].reshape(nkv, n, select * ps, HD).float() for x in (s["k"], s["v"]))
        pos = (ids[..., None] * ps + torch.arange(ps, device=DEV)).reshape(nkv, n, 1, select * ps)
        seen = (pos <= torch.arange(a, a + n, device=DEV)[:, None, None]) & (pos < nb * ps)
        v = torch.where(seen[:, :, 0, :, None], v, torch.zeros((), device=DEV))
        x = torch.matmul(q, k.transpose(2, 3).contiguous()) / math.sqrt(HD)
        x = torch.where(seen, x, torch.full((), float("-inf"), device=DEV))
        o, lse = _softmax(x, v)
        s["selected"][rows] = torch.where(ids < nb, ids, -1).permute(1, 0, 2).to(torch.int32)
        s["q_out"][rows] = o.half().permute(1, 0, 2, 3).reshape(n, -1)
        s["lse"][rows] = lse.permute(1, 0, 2).reshape(n, -1)
    return {"bounds": s["bounds"], "step": s["step"], "selected": s["selected"], "out": s["q_out"], "lse": s["lse"]}


# ---- the framework's calls --------------------------------------------------------------------------------------------
def _lib():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import qe_amd
    return qe_amd


def _handles(s):
    """What a program keeps between calls: the descriptions of cache and batch, the rotation, the workspaces."""
    keep, c = s["keep"], s["case"]
    if not keep:
        qe = _lib()
        keep["cache"] = qe.paged_cache(s["k"], s["v"])
        keep["batch"] = qe.paged_batch(s["table"], s["context"], None if s["single"] else s["starts"], s["rows"])
        size = 0
        if c["kind"] == "append":
            keep["rope"] = qe.rope(s["turns"], s["scale"], interleaved=c["inter"])
        elif c["kind"] == "prefill":
            size = qe.paged_prefill_workspace_bytes(s["rows"], c["nq"], c["nkv"])
        else:
            size = qe.paged_decode_workspace_bytes(s["rows"], c["nq"], c["nkv"])
        keep["ws"] = torch.empty(max(size, 16), dtype=torch.uint8, device=DEV)
        if c["kind"] == "sparse":
            size = qe.paged_select_workspace_bytes(s["rows"], c["nkv"], s["table"].shape[1])
            keep["select_ws"] = torch.empty(max(size, 16), dtype=torch.uint8, device=DEV)
    return keep


def _own_run(s):
    qe, c, h = _lib(), s["case"], _handles(s)
    kind, nq = c["kind"], c["nq"]
    if kind == "append":
        b, g = s["bias"], s["norm"]
        qe.launch_qkv_norm_rope_paged_append(s["q"], s["q_out"], s["k_in"], s["v_in"], b[0], b[1], b[2], g[0], g[1],
                                             h["rope"], h["cache"], h["batch"], num_q_heads=nq, norm_eps=EPS)
        return {"q": s["q_out"], "k": s["k"], "v": s["v"]}
    if kind == "decode":
        qe.launch_attention_gqa_paged_decode(s["q"], h["cache"], h["batch"], h["ws"], s["q_out"], num_q_heads=nq,
                                             window=c["window"], row_lse=s["lse"])
        return {"out": s["q_out"], "lse": s["lse"]}
    if kind == "prefill":
        qe.launch_attention_gqa_paged_prefill(s["q"], h["cache"], h["batch"], h["ws"], s["q_out"], num_q_heads=nq,
                                              window=c["window"], row_lse=s["lse"])
        return {"out": s["q_out"], "lse": s["lse"]}
    qe.launch_paged_key_bounds(h["cache"], h["batch"], s["bounds"], s["step"])
    qe.launch_paged_select(s["q"], h["cache"], h["batch"], s["bounds"], s["step"], s["selected"], h["select_ws"],
                           num_selected=c["select"], sinks=c["sinks"], recent=c["recent"], num_q_heads=nq)
    qe.launch_attention_gqa_paged_sparse(s["q"], h["cache"], h["batch"], s["selected"], h["ws"], s["q_out"],
                                         num_selected=c["select"], num_q_heads=nq, row_lse=s["lse"])
    return {"bounds": s["bounds"], "step": s["step"], "selected": s["selected"], "out": s["q_out"], "lse": s["lse"]}


_PLAIN = {"append": _plain_append, "decode": _plain_attention, "prefill": _plain_attention, "sparse": _plain_sparse}


def run(state):
    if own:
        return _own_run(state)
    return _PLAIN[state["case"]["kind"]](state)


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------
def _exact_append(s):
    c = s["case"]
    table, ps, rot = s["table"].cpu().numpy(), c["page"], c["rot"]
    half = rot // 2
    turns, scale = _turns(rot, c["far"])
    k_out, v_out = s["k"].double().cpu().numpy(), s["v"].double().cpu().numpy()
    q_out = np.zeros((s["rows"], c["nq"] * HD))
    pos = np.concatenate([np.arange(a, a + n) for a, n in _lens(c)])
    seq = np.concatenate([np.full(n, i) for i, (_, n) in enumerate(_lens(c))])
    page, row = table[seq, pos // ps], pos % ps
    first = list(range(0, rot, 2)) if c["inter"] else list(range(half))
    second = [i + 1 for i in first] if c["inter"] else [i + half for i in first]
    wheel = scale * np.exp(2j * np.pi * np.mod(pos[:, None] * turns, 1.0))[:, None]
    for name, b, g in (("q", 0, 0), ("k_in", 1, 1), ("v_in", 2, None)):
        y = s[name][:pos.size].double().cpu().numpy()
        if s["bias"][b] is not None:
            y = y + s["bias"][b].double().cpu().numpy()
        y = y.reshape(pos.size, -1, HD)
        if g is not None:
            if s["norm"][g] is not None:
                y = y / np.sqrt(np.square(y).sum(-1, keepdims=True) / HD + EPS) * s["norm"][g].double().cpu().numpy()
            z = (y[..., first] + 1j * y[..., second]) * wheel
            y[..., first], y[..., second] = z.real, z.imag
        if name == "q":
            q_out[:pos.size] = y.reshape(pos.size, -1)
        else:
            (k_out if name == "k_in" else v_out)[page, :, row] = y
    return {"q": q_out, "k": k_out, "v": v_out}


def _chosen(s, i, a, n, h, first):
    """Which blocks the rows of one sequence select in one head: truth values [rows, blocks]."""
    c = s["case"]
    ps, group = c["page"], c["nq"] // c["nkv"]
    nb = (a + n + ps - 1) // ps
    pages = s["table"][i, :nb].cpu().numpy()
    keys = s["k"][:, h][s["table"][i, :nb].long()].double()
    keys = keys.reshape(nb * ps, HD)
    high, low = keys.clone(), keys.clone()
    high[a + n:], low[a + n:] = -torch.inf, torch.inf
    high = high.reshape(nb, ps, HD).amax(1).cpu().numpy()
    low = low.reshape(nb, ps, HD).amin(1).cpu().numpy()
    m = np.maximum(np.abs(high), np.abs(low)).max(-1)
    high, low = np.ceil(127 * high / m[:, None]), np.floor(127 * low / m[:, None])
    q = s["q"][first:first + n].double().cpu().numpy().reshape(n, -1, group, HD)[:, h]
    mq = np.abs(q).max(-1)
    qn = np.rint(127 * q / mq[..., None])
    best = np.full((n, nb), -np.inf, np.float32)
    for j in range(group):
        dot = np.where(qn[:, j] > 0, qn[:, j], 0) @ high.T + np.where(qn[:, j] < 0, qn[:, j], 0) @ low.T
        best = np.maximum(best, dot.astype(np.float32) * mq[:, j, None].astype(np.float32))
    score = best * m.astype(np.float32)
    took = np.zeros((n, nb), bool)
    for t in range(n):
        own_block = (a + t) // ps
        live = np.arange(own_block + 1)
        sure = (live < c["sinks"]) | (live > own_block - c["recent"])
        order = np.lexsort((live, -score[t, :own_block + 1], ~sure))
        took[t, order[:c["select"]]] = True
    return took, pages


def _exact_attention(s):
    c = s["case"]
    group, ps = c["nq"] // c["nkv"], c["page"]
    out = torch.zeros((s["rows"], c["nq"], HD), dtype=torch.float64, device=DEV)
    lse = torch.zeros((s["rows"], c["nq"]), dtype=torch.float64, device=DEV)
    first = 0
    for i, (a, n) in enumerate(_lens(c)):
        nb = (a + n + ps - 1) // ps
        for h in range(c["nkv"]):
            k, v = (s[x][:, h][s["table"][i, :nb].long()].reshape(nb * ps, HD)[:a + n].double() for x in "kv")
            own_pos = (a + torch.arange(n, device=DEV))[:, None]
            pos = torch.arange(a + n, device=DEV)[None]
            allowed = pos <= own_pos
            if c.get("window"):
                allowed = allowed & (own_pos - pos < c["window"])
            if c["kind"] == "sparse":
                took, _ = _chosen(s, i, a, n, h, first)
                allowed = allowed & torch.from_numpy(took).to(DEV).repeat_interleave(ps, 1)[:, :a + n]
            for j in range(group):
                q = s["q"][first:first + n].double().reshape(n, -1, HD)[:, h * group + j]
                x = torch.where(allowed, q @ k.T * HD ** -0.5, -torch.inf)
                lse[first:first + n, h * group + j] = torch.logsumexp(x, -1)
                out[first:first + n, h * group + j] = torch.softmax(x, -1) @ v
        first += n
    return {"out": out.reshape(s["rows"], -1), "lse": lse}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "append":
        return _exact_append(s)
    out = _exact_attention(s)
    if case["kind"] != "sparse":
        return out
    step = s["step"].double()
    for i, (a, n) in enumerate(_lens(case)):
        ps = case["page"]
        for b in range(a // ps, (a + n - 1) // ps + 1):
            page = int(s["table"][i, b])
            step[page] = s["k"][page][:, :min(ps, a + n - b * ps)].double().abs().amax((1, 2))
    return {"bounds": None, "step": step, "selected": None, **out}


# ---- work ----------------------------------------------------------------------------------------------------------
def work(case):
    c = case
    nq, nkv, ps, lens = c["nq"], c["nkv"], c["page"], _lens(c)
    tokens = sum(n for _, n in lens)
    if c["kind"] == "append":
        return {"bytes": tokens * 2 * 2 * HD * (nq + 2 * nkv), "flops": tokens * HD * (8 * nq + 9 * nkv)}
    nbytes, pairs = tokens * nq * (2 * 2 * HD + 4), 0
    flops = 0
    for a, n in lens:
        if c["kind"] == "sparse":
            nb = (a + n - 1) // ps + 1
            new = nb - a // ps
            keys = min(a + n, n * c["select"] * ps)
            nbytes += nkv * (nb * (2 * HD + 4) + new * (ps * 2 * HD + 2 * HD + 4) + 4 * n * c["select"])
            nbytes += nkv * keys * 2 * 2 * HD
            pairs += nq * n * min(a + n, c["select"] * ps)
            flops += nq * n * nb * 4 * HD
            continue
        w = c["window"] or a + n
        nbytes += nkv * 2 * 2 * HD * min(a + n, w - 1 + n)
        # row t sees min(a + t + 1, w) keys
        short = max(0, min(n, w - a))  # rows that see all before them
        pairs += nq * (short * a + short * (short + 1) // 2 + (n - short) * w)
    return {"bytes": nbytes, "flops": flops + 4 * HD * pairs}
