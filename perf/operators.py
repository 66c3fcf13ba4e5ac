"""Serving several sequences at once, as timed cases: the paged KV cache, the attention that reads it, and what is done to
the logits before a token is chosen.

Kinds:

  store   RoPE of the new tokens' queries and keys, keys and values into the pages of their sequences as f32, f16 or Q8,
          and what the cache then holds for them read back
  read    whole sequences of a paged cache read back as f32 rows (a prefix handed to another cache)
  attend  attention of each sequence's new tokens (one while decoding, a chunk of a prompt) over its pages, causal, with
          an optional sliding window and first positions that stay visible
  logits  penalties for tokens of the history, biases and grammar masks on rows of logits, and the greedy choice

A page holds `page` positions of every KV head: keys as [head][position][dim], values as [head][dim][position], and for Q8
the scales of the 32-wide blocks of each position as [head][block][position].
"""
import importlib
import math
import random

import torch

own = False

TYPES = {"f32": 0, "f16": 1, "q8": 2}
BYTES = {"f32": 4.0, "f16": 2.0, "q8": 1.125}


def listed():
    return [
        # a decode step of 48 conversations on the 0.5B shape: one new token each into a Q8 cache
        {"name": "store-decode", "kind": "store", "type": "q8", "heads": 14, "kv": 2, "head_dim": 64, "page": 64,
         "seqs": 48, "chunks": 0, "new": 1, "length": 2000},
        # prompts of four users in one batch at the 1.5B shape's heads
        {"name": "store-chunk", "kind": "store", "type": "f16", "heads": 12, "kv": 2, "head_dim": 128, "page": 32,
         "seqs": 4, "chunks": 4, "new": 700, "length": 1900},
        # a shared prefix out of the pages into a contiguous cache
        {"name": "read-prefix", "kind": "read", "type": "f16", "heads": 14, "kv": 2, "head_dim": 64, "page": 64,
         "seqs": 1, "length": 1501},
        # eight long Q8 sequences read back
        {"name": "read-long", "kind": "read", "type": "q8", "heads": 32, "kv": 8, "head_dim": 128, "page": 128,
         "seqs": 8, "length": 8100},
        # one conversation's decode step early in its context: latency
        {"name": "attend-one", "kind": "attend", "type": "f32", "heads": 14, "kv": 2, "head_dim": 64, "page": 32,
         "seqs": 1, "chunks": 0, "new": 1, "length": 131, "window": 0, "sinks": 0},
        # a decode step of 32 conversations of ragged lengths
        {"name": "attend-decode", "kind": "attend", "type": "q8", "heads": 12, "kv": 2, "head_dim": 128, "page": 64,
         "seqs": 32, "chunks": 0, "new": 1, "length": 4090, "window": 0, "sinks": 0},
        # a decode step over long documents
        {"name": "attend-long", "kind": "attend", "type": "f16", "heads": 32, "kv": 8, "head_dim": 128, "page": 128,
         "seqs": 16, "chunks": 0, "new": 1, "length": 16384, "window": 0, "sinks": 0},
        # decoding far past a window of 1024 with the first four positions kept
        {"name": "attend-sinks", "kind": "attend", "type": "f16", "heads": 32, "kv": 4, "head_dim": 64, "page": 16,
         "seqs": 8, "chunks": 0, "new": 1, "length": 20011, "window": 1024, "sinks": 4},
        # one prompt's chunk beside seven conversations that decode
        {"name": "attend-mixed", "kind": "attend", "type": "q8", "heads": 14, "kv": 2, "head_dim": 64, "page": 64,
         "seqs": 8, "chunks": 1, "new": 500, "length": 3900, "window": 0, "sinks": 0},
        # two long prompts into empty caches
        {"name": "attend-prompt", "kind": "attend", "type": "f16", "heads": 32, "kv": 8, "head_dim": 64, "page": 64,
         "seqs": 2, "chunks": 2, "new": 2048, "length": 2048, "window": 0, "sinks": 0},
        # one row of the 0.5B shape's vocabulary under a grammar
        {"name": "logits-one", "kind": "logits", "vocab": 151936, "rows": 1, "history": 600, "bias": 20, "masks": 1},
        # the rows of 64 conversations, a third of them under grammars
        {"name": "logits-batch", "kind": "logits", "vocab": 151936, "rows": 64, "history": 2000, "bias": 50, "masks": 21},
    ]


SHAPES = ((14, 2, 64), (12, 2, 128), (32, 8, 64), (32, 8, 128), (9, 3, 64), (8, 8, 96), (16, 2, 80), (32, 4, 64))


def _log(rng, lo, hi):
    """A whole number of [lo, hi], uniform in its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("store", "read", "attend", "attend", "attend", "logits"))
    if kind == "logits":
        rows = _log(rng, 1, 64)
        return {"kind": kind, "vocab": _log(rng, 999, 151936), "rows": rows, "history": _log(rng, 1, 4000),
                "bias": rng.choice((0, 1, _log(rng, 2, 300))), "masks": rng.randint(0, rows)}
    heads, kv, head_dim = rng.choice(SHAPES)
    c = {"kind": kind, "type": rng.choice(("f32", "f16", "q8", "q8")), "heads": heads, "kv": kv, "head_dim": head_dim,
         "page": rng.choice((16, 32, 64, 128, 256))}
    if kind == "read":
        c.update(seqs=_log(rng, 1, 8), length=_log(rng, 1, 6000))
        return _within(c)
    if rng.random() < 0.5:  # every sequence decodes
        c.update(seqs=_log(rng, 1, 64), chunks=0, new=1, length=_log(rng, 1, 12000))
    else:
        new = _log(rng, 2, 1500)
        c.update(seqs=_log(rng, 1, 8), new=new, length=new + _log(rng, 1, 2500) - 1)
        c["chunks"] = rng.randint(1, c["seqs"])
    if kind == "attend":
        c["window"] = rng.choice((0, 0, _log(rng, 1, 2000)))
        c["sinks"] = rng.choice((0, 4, _log(rng, 1, 100))) if c["window"] else 0
    return _within(c)


def _within(c):
    """The case with fewer sequences, then shorter ones, until it is no more work than the largest listed one."""
    most = [work(x) for x in listed()]
    while any(work(c)[k] > max(m[k] for m in most) for k in ("bytes", "flops")):
        if c["seqs"] > 1:
            c["seqs"] //= 2
            if c.get("chunks"):
                c["chunks"] = min(c["chunks"], c["seqs"])
        else:
            c["length"] = (c["length"] + 1) // 2
            c["new"] = min(c.get("new", 1), c["length"])
    return c


# ---- inputs ---------------------------------------------------------------

def _batch(c):
    """(new tokens, positions) of each sequence; the first is the longest. `chunks` of them bring many tokens."""
    rng = random.Random("%(seqs)d %(length)d" % c)
    length = [c["length"]] + [rng.randint((c["length"] + 1) // 2, c["length"]) for _ in range(c["seqs"] - 1)]
    if c["kind"] == "read":
        return length, length
    new = [rng.randint((2 * c["new"] + 2) // 3, c["new"]) if 0 < s < c["chunks"] else c["new"] if s < c["chunks"] else 1
           for s in range(c["seqs"])]
    return [min(n, m) for n, m in zip(new, length)], length


def _histories(c):
    """Tokens in each row's history; the first is the longest."""
    rng = random.Random("%(rows)d %(history)d" % c)
    return [c["history"]] + [rng.randint(c["history"] // 2, c["history"]) for _ in range(c["rows"] - 1)]


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, *shape, sigma=1.0):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * sigma


def _ints(values, dtype=torch.int32):
    return torch.tensor(list(values), dtype=dtype, device="cuda")


def _blocks(c):
    return (c["head_dim"] + 31) // 32


def _pool(g, c, pages):
    """Pages full of earlier sequences' keys and values: a dict of keys, values and, for Q8, their scales."""
    kv, hd, p = c["kv"], c["head_dim"], c["page"]
    if c["type"] != "q8":
        t = torch.float32 if c["type"] == "f32" else torch.float16
        return {"keys": _normal(g, pages, kv, p, hd).to(t), "values": _normal(g, pages, kv, hd, p).to(t)}

    def codes(*shape):
        return torch.randint(-127, 128, shape, generator=g, device="cuda", dtype=torch.int8)

    def scales():
        return 0.01 + 0.02 * torch.rand((pages, kv, _blocks(c), p), generator=g, device="cuda")

    return {"keys": codes(pages, kv, p, hd), "values": codes(pages, kv, hd, p), "key_scales": scales(),
            "value_scales": scales()}


def _cache(g, c, length):
    """The pool and each sequence's page ids, in an order of no meaning; -1 where a sequence has no page."""
    need = [-(-n // c["page"]) for n in length]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(length), max(need)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    return _pool(g, c, pages), table, pages


def prepare(case, seed):
    c, g = case, _generator(seed)
    s = {"case": c}
    if c["kind"] == "logits":
        s.update(_logit_inputs(c, seed))
        s["out"] = torch.empty_like(s["logits"])
        s["token"] = torch.zeros(c["rows"], dtype=torch.int32, device="cuda")
    else:
        new, length = _batch(c)
        tokens, pairs = sum(new), c["head_dim"] // 2
        begin = [sum(new[:i]) for i in range(len(new) + 1)]
        s["new"], s["tokens"], s["context"] = new, tokens, c["length"]
        s["begin"], s["length"] = _ints(begin), _ints(length)
        s["pool"], s["table"], s["pages"] = _cache(g, c, length)
        # the row, sequence and position of every new token
        seq = torch.repeat_interleave(torch.arange(len(new), device="cuda"), _ints(new, torch.int64))
        s["seq"] = seq
        s["pos"] = (torch.arange(tokens, device="cuda") - s["begin"].long()[seq] + (s["length"].long() - _ints(new))[seq])
        qd, kd = c["heads"] * c["head_dim"], c["kv"] * c["head_dim"]
        if c["kind"] == "store":
            s["q"], s["k"], s["v"] = _normal(g, tokens, qd), _normal(g, tokens, kd), _normal(g, tokens, kd)
            angle = _angles(c)
            s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        elif c["kind"] == "attend":
            s["q"] = _normal(g, tokens, qd, sigma=1.5)
        s["out"] = {"store": lambda: [torch.zeros(tokens, n, device="cuda") for n in (qd, kd, kd)],
                    "read": lambda: [torch.zeros(tokens, kd, device="cuda") for _ in range(2)],
                    "attend": lambda: torch.zeros(tokens, qd, device="cuda")}[c["kind"]]()
    if own:
        _handles(s)
    return s


def _angles(c):
    half = torch.arange(0, c["head_dim"], 2, dtype=torch.float64, device="cuda") / c["head_dim"]
    return torch.arange(c["length"], dtype=torch.float64, device="cuda")[:, None] * 1e6 ** -half


def _logit_inputs(c, seed):
    g = _generator(seed)
    rows, vocab = c["rows"], c["vocab"]
    seen = _histories(c)
    # tokens repeat as in text: few ids often, many once
    u = torch.rand(sum(seen), generator=g, device="cuda", dtype=torch.float64)
    history = (vocab ** u - 1).long().clamp(0, vocab - 1)
    few = min(c["bias"], vocab)
    ids = torch.stack([torch.randperm(vocab, generator=g, device="cuda")[:few] for _ in range(rows)])
    words = (vocab + 31) // 32
    # a grammar leaves one id in sixteen
    bits = [torch.randint(0, 1 << 32, (max(1, c["masks"]), words), generator=g, device="cuda") for _ in range(4)]
    allowed = bits[0] & bits[1] & bits[2] & bits[3]
    allowed = torch.where(allowed >= 1 << 31, allowed - (1 << 32), allowed).to(torch.int32)
    penalty = torch.stack([1 + 0.3 * torch.rand(rows, generator=g, device="cuda"),
                           0.5 * torch.rand(rows, generator=g, device="cuda"),
                           0.2 * torch.rand(rows, generator=g, device="cuda")], 1).contiguous()
    return {"logits": _normal(g, rows, vocab, sigma=3.0), "history": history.to(torch.int32),
            "history_begin": _ints(sum(seen[:i]) for i in range(rows + 1)), "penalty": penalty,
            "history_row": torch.repeat_interleave(torch.arange(rows, device="cuda"), _ints(seen, torch.int64)),
            "bias_ids": ids.reshape(-1).to(torch.int32), "bias": _normal(g, rows * few, sigma=2.0),
            "bias_begin": _ints(i * few for i in range(rows + 1)), "allowed": allowed,
            "mask_row": _ints(i if i < c["masks"] else -1 for i in range(rows))}


def _handles(s):
    """The library's descriptors of these buffers (addresses and sizes, host side) and its workspace."""
    smq = s["smq"] = importlib.import_module("smolmoe-c99_amd")
    smq.init(0)
    c = s["case"]
    if c["kind"] == "logits":
        s["rules"] = smq.logit_rules(history=s["history"].data_ptr(), history_begin=s["history_begin"].data_ptr(),
                                     history_count=s["history"].numel(), penalty=s["penalty"].data_ptr(),
                                     bias_ids=s["bias_ids"].data_ptr(), bias=s["bias"].data_ptr(),
                                     bias_begin=s["bias_begin"].data_ptr(), bias_count=s["bias"].numel(),
                                     allowed=s["allowed"].data_ptr(), allowed_rows=s["allowed"].shape[0],
                                     mask_row=s["mask_row"].data_ptr())
        need = smq.logits_workspace(c["rows"], c["vocab"])
    else:
        p = {k: v.data_ptr() for k, v in s["pool"].items()}
        s["kv"] = smq.paged_kv(p["keys"], p["values"], p.get("key_scales"), p.get("value_scales"), TYPES[c["type"]],
                               c["page"], s["pages"])
        s["batch"] = smq.paged_batch(s["begin"].data_ptr(), s["length"].data_ptr(), s["table"].data_ptr(), c["seqs"],
                                     s["tokens"], s["table"].shape[1])
        s["shape"] = smq.attn_shape(c["heads"], c["kv"], c["head_dim"], c["head_dim"] // 2, c.get("window", 0),
                                    s["context"])
        need = smq.paged_attention_workspace(s["batch"], s["shape"])
    s["workspace"] = torch.empty(max(1, need), dtype=torch.uint8, device="cuda")


# ---- one pass -------------------------------------------------------------

def run(state):
    s = state
    kind = s["case"]["kind"]
    if own:
        return _run_own(s, kind)
    if kind == "store":
        return _store(s)
    if kind == "read":
        return _rows(s)
    return _attend(s) if kind == "attend" else _logits(s)


def _run_own(s, kind):
    smq, ptr = s["smq"], torch.Tensor.data_ptr
    if kind == "logits":
        smq.logits_adjust(ptr(s["logits"]), s["case"]["rows"], s["case"]["vocab"], s["rules"], ptr(s["out"]),
                          ptr(s["token"]), ptr(s["workspace"]), s["workspace"].numel())
        return [s["out"], s["token"]]
    if kind == "attend":
        smq.paged_attention(ptr(s["q"]), ptr(s["out"]), s["batch"], s["shape"], s["case"]["sinks"], s["kv"],
                            ptr(s["workspace"]), s["workspace"].numel())
        return s["out"]
    if kind == "store":
        smq.paged_rope_kv(ptr(s["q"]), ptr(s["out"][0]), ptr(s["k"]), ptr(s["v"]), s["batch"], s["shape"], ptr(s["cos"]),
                          ptr(s["sin"]), s["kv"])
    smq.paged_read(s["batch"], s["shape"], s["kv"], ptr(s["out"][-2]), ptr(s["out"][-1]))
    return s["out"]


def _slots(s):
    """Page and slot of every new token."""
    page = s["case"]["page"]
    return s["table"][s["seq"], s["pos"] // page].long(), s["pos"] % page


def _rotate(x, cos, sin, heads):
    x = x.reshape(x.shape[0], heads, -1, 2)
    a, b, cos, sin = x[..., 0], x[..., 1], cos[:, None], sin[:, None]
    return torch.stack([a * cos - b * sin, a * sin + b * cos], -1).reshape(x.shape[0], heads, -1)


def _q8(x):
    """Scales and codes of the 32-wide blocks of [tokens, heads, dims]."""
    pad = -x.shape[-1] % 32
    b = torch.nn.functional.pad(x, (0, pad)).reshape(*x.shape[:-1], -1, 32)
    scale = b.abs().amax(-1) / torch.full((1,), 127.0, device=x.device)
    inv = torch.where(scale >= torch.finfo(torch.float32).tiny, torch.ones_like(scale) / scale, torch.zeros_like(scale))
    code = torch.round(b * inv[..., None]).clamp(-127, 127)
    return scale, code.reshape(*x.shape[:-1], -1)[..., :x.shape[-1]].to(torch.int8)


def _store(s):
    c, pool = s["case"], s["pool"]
    cos, sin = s["cos"][s["pos"]], s["sin"][s["pos"]]
    q = _rotate(s["q"], cos, sin, c["heads"])
    k, v = _rotate(s["k"], cos, sin, c["kv"]), s["v"].reshape(s["tokens"], c["kv"], -1)
    page, slot = _slots(s)
    if c["type"] == "q8":
        (ks, k), (vs, v) = _q8(k), _q8(v)
        pool["key_scales"][page, :, :, slot] = ks
        pool["value_scales"][page, :, :, slot] = vs
    pool["keys"][page, :, slot] = k.to(pool["keys"].dtype)
    pool["values"][page, :, :, slot] = v.to(pool["values"].dtype)
    return [q.reshape(s["tokens"], -1)] + _rows(s)


def _rows(s):
    """The new tokens' keys and values as the cache holds them."""
    c, pool = s["case"], s["pool"]
    page, slot = _slots(s)
    k, v = pool["keys"][page, :, slot].float(), pool["values"][page, :, :, slot].float()
    if c["type"] == "q8":
        ks, vs = (pool[n][page, :, :, slot].repeat_interleave(32, -1)[..., :c["head_dim"]]
                  for n in ("key_scales", "value_scales"))
        k, v = k * ks, v * vs
    return [k.reshape(s["tokens"], -1), v.reshape(s["tokens"], -1)]


def _dense(s, dtype):
    """Keys and values of every sequence's pages, [sequence, KV head, position, dim]."""
    c, pool, ids = s["case"], s["pool"], s["table"].long().clamp(min=0)
    k = pool["keys"][ids].to(dtype)
    v = pool["values"][ids].to(dtype).transpose(-1, -2)
    if c["type"] == "q8":
        k, v = (x * pool[n][ids].to(dtype).repeat_interleave(32, 3)[:, :, :, :c["head_dim"]].transpose(-1, -2)
                for x, n in ((k, "key_scales"), (v, "value_scales")))
    return [x.transpose(1, 2).reshape(c["seqs"], c["kv"], -1, c["head_dim"]) for x in (k, v)]


def _attend(s):
    c = s["case"]
    seqs, kv, hd, grp, most = c["seqs"], c["kv"], c["head_dim"], c["heads"] // c["kv"], max(s["new"])
    k, v = _dense(s, torch.float32)
    place = torch.arange(s["tokens"], device="cuda") - s["begin"].long()[s["seq"]]
    q = torch.zeros(seqs, most, kv, grp, hd, device="cuda")
    q[s["seq"], place] = s["q"].reshape(-1, kv, grp, hd)
    q = q.permute(0, 2, 3, 1, 4).reshape(seqs, kv, grp * most, hd)
    score = (torch.matmul(q, k.transpose(2, 3).contiguous()) / math.sqrt(hd)).reshape(seqs, kv, grp, most, -1)
    first = s["length"].long() - (s["begin"][1:] - s["begin"][:-1]).long()
    p = (first[:, None] + torch.arange(most, device="cuda"))[:, :, None]
    j = torch.arange(k.shape[2], device="cuda")[None, None]
    seen = j <= p
    if c["window"]:
        seen &= (j > p - c["window"]) | (j < c["sinks"])
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    e = torch.exp(score - score.amax(-1, keepdim=True))
    e = e / e.sum(-1, keepdim=True)
    v = torch.where((j <= (s["length"].long() - 1)[:, None, None])[:, :, :, None], v, torch.zeros_like(v))
    out = torch.matmul(e.reshape(seqs, kv, grp * most, -1), v).reshape(seqs, kv, grp, most, hd)
    return out.permute(0, 3, 1, 2, 4)[s["seq"], place].reshape(s["tokens"], -1)


def _bits(s, vocab):
    """Which ids each row may take."""
    bit = (s["allowed"][..., None] >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1
    bit = bit.reshape(bit.shape[0], -1)[:, :vocab] != 0
    row = s["mask_row"].long()
    return bit[row.clamp(min=0)] | (row < 0)[:, None]


def _logits(s):
    c = s["case"]
    rows, vocab = c["rows"], c["vocab"]
    count = torch.zeros(rows, vocab, device="cuda")
    count.index_put_((s["history_row"], s["history"].long()), torch.ones((), device="cuda"), accumulate=True)
    rep, presence, frequency = (x[:, None] for x in s["penalty"].unbind(1))
    l = s["logits"]
    seen = torch.where(l > 0, l / rep, l * rep) - (count * frequency + presence)
    l = torch.where(count > 0, seen, l)
    per_row = s["bias"].numel() // rows
    if per_row:
        l = l.scatter_add(1, s["bias_ids"].long().reshape(rows, per_row), s["bias"].reshape(rows, per_row))
    may = _bits(s, vocab)
    l = l.masked_fill(~may, -math.inf)
    best = l.amax(1, keepdim=True)
    ids = torch.arange(vocab, device="cuda", dtype=torch.int32)
    return [l, torch.where(may & (l == best), ids, vocab).amin(1).to(torch.int32)]


# ---- what a pass cannot do without ----------------------------------------

def work(case):
    c = case
    if c["kind"] == "logits":
        words = (c["vocab"] + 31) // 32
        return {"bytes": c["rows"] * (8 * c["vocab"] + 8 * c["bias"]) + 4 * sum(_histories(c)) + 4 * c["masks"] * words,
                "flops": 4.0 * c["rows"] * c["vocab"]}
    new, length = _batch(c)
    qd, kd = c["heads"] * c["head_dim"], c["kv"] * c["head_dim"]
    row = 2 * kd * BYTES[c["type"]]
    if c["kind"] == "read":
        return {"bytes": sum(new) * (row + 8 * kd), "flops": 0}
    if c["kind"] == "store":  # read q, k, v; write q and the cache; read it back as f32 rows
        return {"bytes": sum(new) * (8 * qd + 8 * kd + 2 * row + 8 * kd), "flops": 3.0 * sum(new) * (qd + kd)}
    seen = union = 0
    for n, m in zip(new, length):
        w, k = c["window"] or m, c["sinks"]
        low = max(0, m - n + 1 - w)  # the first position that the first new token's window holds
        union += m - low + min(k, low)
        for p in range(m - n, m):
            low = max(0, p + 1 - w)
            seen += p + 1 - low + min(k, low)
    return {"bytes": union * row + 8 * sum(new) * qd, "flops": 4.0 * qd * seen}


# ---- the results in 64 bits -------------------------------------------------

def exact(case, seed):
    c = case
    s = prepare(c, seed)
    if c["kind"] == "read":
        page, slot = s["table"][s["seq"], s["pos"] // c["page"]].long(), s["pos"] % c["page"]
        out = []
        for n, x in (("key_scales", s["pool"]["keys"][page, :, slot].double()),
                     ("value_scales", s["pool"]["values"][page, :, :, slot].double())):
            if c["type"] == "q8":
                block = torch.arange(c["head_dim"], device="cuda") // 32
                x = x * s["pool"][n].double()[page, :, :, slot][..., block]
            out.append(x.reshape(s["tokens"], -1))
        return out
    if c["kind"] == "store":
        turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), _angles(c)[s["pos"]])[:, None]

        def rotated(x, heads):
            pairs = torch.view_as_complex(x.double().reshape(s["tokens"], heads, -1, 2)) * turn
            return torch.view_as_real(pairs).reshape(s["tokens"], -1)

        if c["type"] == "f32":
            return [rotated(s["q"], c["heads"]), rotated(s["k"], c["kv"]), s["v"].double()]
        return [rotated(s["q"], c["heads"]), None, None]  # f16 and Q8 values are rounded from the f32 rotation
    if c["kind"] == "logits":
        return _logits64(c, s)
    grp, hd, at, out = c["heads"] // c["kv"], c["head_dim"], 0, []
    for i, n in enumerate(s["new"]):
        m = int(s["length"][i])
        ids = s["table"][i, :-(-m // c["page"])].long()
        k, v = s["pool"]["keys"][ids].double(), s["pool"]["values"][ids].double().transpose(-1, -2)
        if c["type"] == "q8":
            block = torch.arange(hd, device="cuda") // 32
            k = k * s["pool"]["key_scales"][ids].double()[:, :, block].transpose(-1, -2)
            v = v * s["pool"]["value_scales"][ids].double()[:, :, block].transpose(-1, -2)
        k, v = (x.transpose(0, 1).reshape(c["kv"], -1, hd)[:, :m] for x in (k, v))
        q = s["q"][at:at + n].double().reshape(n, c["kv"], grp, hd)
        back = torch.arange(m - n, m, device="cuda")[:, None] - torch.arange(m, device="cuda")[None]
        hidden = back < 0
        if c["window"]:
            hidden |= (back >= c["window"]) & (torch.arange(m, device="cuda") >= c["sinks"])
        heads = []
        for h in range(c["heads"]):
            w = q[:, h // grp, h % grp] @ k[h // grp].T / math.sqrt(hd)
            heads.append(torch.softmax(w.masked_fill(hidden, -math.inf), -1) @ v[h // grp])
        out.append(torch.cat(heads, 1))
        at += n
    return torch.cat(out)


def _logits64(c, s):
    out = []
    for r in range(c["rows"]):
        l = s["logits"][r].double()
        rep, presence, frequency = s["penalty"][r].double().tolist()
        a, b = int(s["history_begin"][r]), int(s["history_begin"][r + 1])
        ids, times = torch.unique(s["history"][a:b].long(), return_counts=True)
        x = l[ids]
        l[ids] = torch.where(x > 0, x / rep, x * rep) - presence - frequency * times
        a, b = int(s["bias_begin"][r]), int(s["bias_begin"][r + 1])
        l[s["bias_ids"][a:b].long()] += s["bias"][a:b].double()
        if int(s["mask_row"][r]) >= 0:
            words = s["allowed"][int(s["mask_row"][r])].long()
            ids = torch.arange(c["vocab"], device="cuda")
            l[(words[ids // 32] >> (ids % 32)) & 1 == 0] = -math.inf
        out.append(l)
    return [torch.stack(out), None]
