"""Drafted tokens and beams over the paged KV cache, as timed cases.

Kinds:

  norm     RMSNorm of each query and key head, the rotation by each token's own position, keys and values into the pages
           of their sequences as f32, f16 or Q8, and what the cache then holds for them read back
  tree     drafted tokens that form a tree (each has a parent before it, or hangs on the context): which of them each one
           sees, and their attention over the context and their ancestors
  fork     the sequences' next page tables from parents: full pages shared, a last page that others hold copied, pages for
           the positions to come, the rest freed; and the copied positions of every layer
  compact  the accepted path of each sequence's draft moved to the front of its drafted tokens, in every layer
  beam     the best continuations of each group's beams over the vocabulary, and their histories

A page holds `page` positions of every KV head: keys as [head][position][dim], values as [head][dim][position], and for Q8
the scales of the 32-wide blocks of each position as [head][block][position].
"""
import importlib
import math
import random

import numpy as np
import torch

own = False

TYPES = {"f32": 0, "f16": 1, "q8": 2}
BYTES = {"f32": 4.0, "f16": 2.0, "q8": 1.125}
EPS = float(np.float32(1e-6))


def listed():
    return [
        # the drafts of 32 conversations on the 0.5B shape's heads into a Q8 cache, out of one row of q, k and v each
        {"name": "norm-drafts", "kind": "norm", "type": "q8", "heads": 14, "kv": 2, "head_dim": 64, "page": 64,
         "seqs": 32, "chunks": 32, "new": 8, "length": 2000, "tree": True, "packed": True},
        # four prompts in one batch
        {"name": "norm-chunk", "kind": "norm", "type": "f16", "heads": 32, "kv": 8, "head_dim": 128, "page": 64,
         "seqs": 4, "chunks": 4, "new": 1500, "length": 1900, "tree": False, "packed": False},
        # one conversation's draft: latency
        {"name": "tree-one", "kind": "tree", "type": "f16", "heads": 14, "kv": 2, "head_dim": 64, "page": 32,
         "seqs": 1, "chunks": 1, "new": 13, "length": 613, "window": 0, "sinks": 0},
        # the drafts of 24 conversations of ragged lengths
        {"name": "tree-batch", "kind": "tree", "type": "q8", "heads": 12, "kv": 2, "head_dim": 128, "page": 64,
         "seqs": 24, "chunks": 24, "new": 40, "length": 3001, "window": 0, "sinks": 0},
        # drafts over long documents
        {"name": "tree-long", "kind": "tree", "type": "f16", "heads": 32, "kv": 8, "head_dim": 128, "page": 128,
         "seqs": 8, "chunks": 8, "new": 63, "length": 16384, "window": 0, "sinks": 0},
        # one prompt's four beams go on, 24 layers
        {"name": "fork-beams", "kind": "fork", "type": "q8", "kv": 2, "head_dim": 64, "page": 64, "layers": 24,
         "groups": 1, "beams": 4, "prompt": 500, "length": 717},
        # eight prompts of eight beams, 12 layers
        {"name": "fork-batch", "kind": "fork", "type": "f16", "kv": 2, "head_dim": 128, "page": 128, "layers": 12,
         "groups": 8, "beams": 8, "prompt": 1500, "length": 1801},
        # the tables of 256 long conversations, some of which end while others begin: no page is copied
        {"name": "fork-tables", "kind": "fork", "type": "f16", "kv": 1, "head_dim": 16, "page": 16, "layers": 0,
         "groups": 256, "beams": 1, "prompt": 0, "length": 30000},
        # paths of eight drafts accepted, 24 layers
        {"name": "compact-drafts", "kind": "compact", "type": "q8", "heads": 14, "kv": 2, "head_dim": 64, "page": 64,
         "seqs": 8, "chunks": 8, "new": 16, "length": 300, "accept": 5, "layers": 24},
        # paths of 64 large drafts accepted, four layers
        {"name": "compact-batch", "kind": "compact", "type": "f16", "heads": 32, "kv": 8, "head_dim": 128, "page": 32,
         "seqs": 64, "chunks": 64, "new": 60, "length": 90, "accept": 12, "layers": 4},
        # four beams of one prompt over the 0.5B shape's vocabulary, eight continuations
        {"name": "beam-one", "kind": "beam", "groups": 1, "beams": 4, "select": 8, "vocab": 151936, "history": 700},
        # 16 prompts of eight beams
        {"name": "beam-batch", "kind": "beam", "groups": 16, "beams": 8, "select": 16, "vocab": 151936, "history": 500},
    ]


SHAPES = ((14, 2, 64), (12, 2, 128), (32, 8, 64), (32, 8, 128), (9, 3, 64), (8, 8, 96), (16, 2, 80), (32, 4, 64))


def _log(rng, lo, hi):
    """A whole number of [lo, hi], uniform in its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("norm", "tree", "tree", "fork", "compact", "beam"))
    if kind == "beam":
        beams = _log(rng, 1, 32)
        return _within({"kind": kind, "groups": _log(rng, 1, max(1, 128 // beams)), "beams": beams,
                        "select": rng.choice((beams, 2 * beams, _log(rng, 1, 16))), "vocab": _log(rng, 999, 151936),
                        "history": _log(rng, 1, 2000)})
    heads, kv, head_dim = rng.choice(SHAPES)
    c = {"kind": kind, "type": rng.choice(("f32", "f16", "q8", "q8")), "kv": kv, "head_dim": head_dim,
         "page": rng.choice((16, 32, 64, 128, 256))}
    if kind == "fork":
        prompt, beams = _log(rng, 1, 2000), rng.choice((1, 4, _log(rng, 2, 12)))
        c.update(layers=rng.choice((0, 1, 4)), groups=_log(rng, 1, 8), beams=beams, prompt=prompt,
                 length=prompt + _log(rng, 1, 400))
        if beams == 1:
            c.update(layers=0, groups=_log(rng, 1, 256), length=_log(rng, 1, 30000), prompt=0)
        return _within(c)
    c["heads"] = heads
    if kind == "compact":
        new = _log(rng, 1, 100)
        c.update(seqs=_log(rng, 1, 32), new=new, length=new + _log(rng, 1, 200) - 1, accept=min(new, _log(rng, 1, 16)),
                 layers=rng.choice((1, 4)))
        c["chunks"] = c["seqs"]
        return _within(c)
    if kind == "norm":
        new = rng.choice((1, _log(rng, 1, 1500)))
        c.update(seqs=_log(rng, 1, 32), new=new, length=new + _log(rng, 1, 2500) - 1, tree=new > 1 and rng.random() < 0.5,
                 packed=rng.random() < 0.5)
    else:
        new = _log(rng, 1, 200)
        c.update(seqs=_log(rng, 1, 32), new=new, length=new + _log(rng, 1, 10000) - 1)
        c["window"] = rng.choice((0, 0, _log(rng, 1, 2000)))
        c["sinks"] = rng.choice((0, 4, _log(rng, 1, 100))) if c["window"] else 0
    c["chunks"] = rng.randint(1, c["seqs"])
    return _within(c)


def _within(c):
    """The case with fewer sequences or groups, then shorter ones, until it is no more work than the largest listed one."""
    most = [work(x) for x in listed() if x["kind"] == c["kind"]]
    while any(work(c)[k] > max(m[k] for m in most) for k in ("bytes", "flops")):
        n = "seqs" if "seqs" in c else "groups"
        if c[n] > 1:
            c[n] //= 2
            if "chunks" in c:
                c["chunks"] = min(c["chunks"], c[n])
        elif c["kind"] == "beam":
            c["vocab"] = (c["vocab"] + 1) // 2
        elif c.get("layers", 0) > 1:
            c["layers"] //= 2
        else:
            c["length"] = (c["length"] + 1) // 2
            for k in ("new", "prompt", "accept"):
                if k in c:
                    c[k] = min(c[k], c["length"] if k != "accept" else c["new"])
    return c


# ---- the structure of a case: sizes, trees, parents ------------------------

def _batch(c):
    """(new tokens, positions) of each sequence; the first is the longest. `chunks` of them bring many tokens."""
    rng = random.Random("%(seqs)d %(length)d" % c)
    length = [c["length"]] + [rng.randint((c["length"] + 1) // 2, c["length"]) for _ in range(c["seqs"] - 1)]
    new = [rng.randint((2 * c["new"] + 2) // 3, c["new"]) if 0 < s < c["chunks"] else c["new"] if s < c["chunks"] else 1
           for s in range(c["seqs"])]
    return [min(n, m) for n, m in zip(new, length)], length


def _trees(c):
    """Of each sequence's new tokens: the parents (-1: the context), as a draft model's best guesses spread out."""
    rng = random.Random("%(seqs)d %(new)d %(length)d" % c)
    return [[-1 if i == 0 or rng.random() < 0.5 / n else rng.randint((i - 1) // 3, i - 1) for i in range(n)]
            for n in _batch(c)[0]]


def _depths(parents):
    d = []
    for p in parents:
        d.append(d[p] + 1 if p >= 0 else 0)
    return d


def _paths(c):
    """Of each sequence the accepted drafts, ascending: `accept` of the first, fewer of others. A token already at its place
    stays; one that moves comes from behind the path's places, so that a pass leaves the next one's input as it is."""
    rng = random.Random("%(seqs)d %(accept)d %(new)d" % c)
    paths = []
    for s, n in enumerate(_batch(c)[0]):
        m = min(n, c["accept"] if s == 0 else rng.randint(0, c["accept"]))
        stay = rng.randint(0, m)
        while stay < m and n - m < m - stay:
            stay += 1
        paths.append(list(range(stay)) + sorted(rng.sample(range(m, n), m - stay)))
    return paths


def _rows(c):
    """Of each new row: its old row (-1: none), the positions it keeps and the positions it needs pages for; and the
    positions of each old row."""
    rng = random.Random("%(groups)d %(beams)d %(length)d %(page)d" % c)
    b = c["beams"]
    if b > 1:  # every beam of a group has the group's length
        length = [rng.randint((c["prompt"] + c["length"]) // 2, c["length"]) for _ in range(c["groups"])]
        held = [length[r // b] for r in range(c["groups"] * b)]
        parent = [g * b + rng.randrange(b) for g in range(c["groups"]) for _ in range(b)]
        keep = [held[p] for p in parent]
        return parent, keep, [k + 1 for k in keep], held
    held = [rng.randint((c["length"] + 1) // 2, c["length"]) for _ in range(c["groups"])]
    parent = [r if rng.random() < 0.9 else -1 for r in range(c["groups"])]
    # drafts that were not accepted are given back; room for the next ones
    keep = [max(0, held[p] - rng.randint(0, 8)) if p >= 0 else 0 for p in parent]
    return parent, keep, [min(c["length"] + 16, k + 8) if p >= 0 else rng.randint((c["length"] + 1) // 2, c["length"])
                          for p, k in zip(parent, keep)], held


def _shared(c):
    """Full pages of a group's prompt, which its beams share."""
    return c["prompt"] // c["page"] if c["beams"] > 1 else 0


def _ceil(a, b):
    return -(-a // b)


# ---- inputs ---------------------------------------------------------------

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


def _pool(g, c, pages, layers=1):
    """Pages full of earlier sequences' keys and values, [layer, page, ...]: a dict of keys, values and, for Q8, scales."""
    kv, hd, p = c["kv"], c["head_dim"], c["page"]
    if c["type"] != "q8":
        t = torch.float32 if c["type"] == "f32" else torch.float16
        return {"keys": _normal(g, layers, pages, kv, p, hd).to(t), "values": _normal(g, layers, pages, kv, hd, p).to(t)}

    def codes(*shape):
        return torch.randint(-127, 128, shape, generator=g, device="cuda", dtype=torch.int8)

    def scales():
        return 0.01 + 0.02 * torch.rand((layers, pages, kv, _blocks(c), p), generator=g, device="cuda")

    return {"keys": codes(layers, pages, kv, p, hd), "values": codes(layers, pages, kv, hd, p), "key_scales": scales(),
            "value_scales": scales()}


def _table(g, c, length):
    """Each sequence's page ids, in an order of no meaning; -1 where a sequence has no page."""
    need = [_ceil(n, c["page"]) for n in length]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(length), max(need)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    return table, pages


def prepare(case, seed):
    c, g = case, _generator(seed)
    s = {"case": c}
    if c["kind"] == "beam":
        _beam_inputs(s, g)
    elif c["kind"] == "fork":
        _fork_inputs(s, g, seed)
    else:
        _batch_inputs(s, g)
    if own:
        _handles(s)
    return s


def _batch_inputs(s, g):
    c = s["case"]
    new, length = _batch(c)
    tokens, pairs = sum(new), c["head_dim"] // 2
    begin = [sum(new[:i]) for i in range(len(new) + 1)]
    s["new"], s["tokens"], s["most"] = new, tokens, max(new)
    s["begin"], s["length"] = _ints(begin), _ints(length)
    s["table"], s["pages"] = _table(g, c, length)
    s["pool"] = _pool(g, c, s["pages"], c.get("layers", 1))
    # the row, sequence and position of every new token
    seq = torch.repeat_interleave(torch.arange(len(new), device="cuda"), _ints(new, torch.int64))
    s["seq"], s["place"] = seq, torch.arange(tokens, device="cuda") - s["begin"].long()[seq]
    s["first"] = s["length"].long() - _ints(new, torch.int64)
    s["pos"] = s["first"][seq] + s["place"]
    qd, kd = c["heads"] * c["head_dim"], c["kv"] * c["head_dim"]
    if c["kind"] == "compact":
        paths = _paths(c)
        s["stride"] = max(1, max(len(p) for p in paths))
        s["accepted"] = _ints((p + [0] * (s["stride"] - len(p)) for p in paths)).reshape(len(paths), -1).contiguous()
        s["count"] = _ints(len(p) for p in paths)
        s["length_out"] = torch.zeros_like(s["length"])
        return
    if c["kind"] == "tree" or c["tree"]:
        trees = _trees(c)
        s["parent"] = _ints(p for t in trees for p in t)
        s["depth"] = _ints(d for t in trees for d in _depths(t))
    if c["kind"] == "tree":
        s["words"] = (s["most"] + 31) // 32
        s["depth"] = torch.zeros(tokens, dtype=torch.int32, device="cuda")  # the pass works them out
        s["mask"] = torch.zeros(tokens, s["words"], dtype=torch.int32, device="cuda")
        s["q"] = _normal(g, tokens, qd, sigma=1.5)
        s["out"] = torch.zeros(tokens, qd, device="cuda")
        return
    if c["packed"]:
        qkv = _normal(g, tokens, qd + 2 * kd, sigma=3.0)
        s["q"], s["k"], s["v"] = qkv[:, :qd], qkv[:, qd:qd + kd], qkv[:, qd + kd:]
    else:
        s["q"], s["k"], s["v"] = _normal(g, tokens, qd, sigma=3.0), _normal(g, tokens, kd, sigma=3.0), _normal(g, tokens, kd)
    s["q_norm"], s["k_norm"] = (1 + _normal(g, c["head_dim"], sigma=0.3) for _ in range(2))
    angle = _angles(c)
    s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
    s["out"] = [torch.zeros(tokens, n, device="cuda") for n in (qd, kd, kd)]


def _angles(c):
    half = torch.arange(0, c["head_dim"], 2, dtype=torch.float64, device="cuda") / c["head_dim"]
    return torch.arange(c["length"], dtype=torch.float64, device="cuda")[:, None] * 1e6 ** -half


def _fork_inputs(s, g, seed):
    c = s["case"]
    parent, keep, room, held = _rows(c)
    page, rows, shared = c["page"], len(held), _shared(c)
    need = [_ceil(n, page) for n in held]
    width = max(max(need), max(_ceil(n, page) for n in room))
    # ids in an order of no meaning: each group's shared pages, then the rows' own
    own_pages = sum(n - shared for n in need) + shared * c["groups"]
    pages = own_pages + sum(2 if p >= 0 else _ceil(n, page) for p, n in zip(parent, room)) + 5
    order = np.random.default_rng(seed).permutation(pages).astype(np.int32)
    table, at = np.full((rows, width), -1, np.int32), shared * c["groups"]
    for r, n in enumerate(need):
        group = r // c["beams"]
        table[r, :shared] = order[group * shared:(group + 1) * shared]
        table[r, shared:n] = order[at:at + n - shared]
        at += n - shared
    refs = np.bincount(table[table >= 0], minlength=pages).astype(np.int32)
    refs[order[:shared * c["groups"]]] += 1  # a store of prompts holds those too
    s["rows"], s["pages"], s["width"] = rows, pages, width
    s["table"], s["refs"] = torch.from_numpy(table).cuda(), torch.from_numpy(refs).cuda()
    s["held"], s["parent"], s["keep"], s["room"] = _ints(need), _ints(parent), _ints(keep), _ints(room)
    s["pool"] = _pool(g, c, pages, c["layers"]) if c["layers"] else {}
    s["out"] = {"table": torch.zeros_like(s["table"]), "held": torch.zeros_like(s["held"]),
                "refs": torch.zeros_like(s["refs"]), "copies": torch.zeros(rows, 3, dtype=torch.int32, device="cuda"),
                "free": torch.zeros(1, dtype=torch.int32, device="cuda")}


def _beam_inputs(s, g):
    c = s["case"]
    rows, n, out = c["groups"] * c["beams"], c["history"], c["groups"] * c["select"]
    rng = random.Random("%(groups)d %(beams)d %(history)d" % c)
    s["logits"] = _normal(g, rows, c["vocab"], sigma=3.0)
    s["score"] = _normal(g, rows, sigma=2.0) - n
    s["done"] = _ints((rng.random() < 0.1 for _ in range(rows)), torch.uint8)
    s["stride"] = n + 20
    length = [rng.randint((n + 1) // 2, n) for _ in range(rows)]
    ids = torch.randint(0, c["vocab"], (rows, s["stride"]), generator=g, device="cuda", dtype=torch.int32)
    s["lengths"] = _ints(length)
    ids[torch.arange(s["stride"], device="cuda")[None] >= s["lengths"][:, None]] = -1
    s["history"], s["pad"], s["eos"] = ids, 1, 2
    s["out"] = {"parent": torch.zeros(out, dtype=torch.int32, device="cuda"),
                "token": torch.zeros(out, dtype=torch.int32, device="cuda"), "score": torch.zeros(out, device="cuda"),
                "done": torch.zeros(out, dtype=torch.uint8, device="cuda"),
                "length": torch.zeros(out, dtype=torch.int32, device="cuda"),
                "history": torch.zeros(out, s["stride"], dtype=torch.int32, device="cuda")}


def _handles(s):
    """The library's descriptors of these buffers (addresses and sizes, host side) and its workspace."""
    smq = s["smq"] = importlib.import_module("smolmoe-c99_amd")
    smq.init(0)
    c, ptr = s["case"], torch.Tensor.data_ptr
    need = 0
    if c["kind"] == "beam":
        o = s["out"]
        s["step"] = smq.beam_step(ptr(s["logits"]), c["vocab"], c["groups"], c["beams"], c["vocab"], c["select"],
                                  ptr(s["score"]), ptr(o["parent"]), ptr(o["token"]), ptr(o["score"]), done=ptr(s["done"]),
                                  pad=s["pad"], eos=s["eos"], done_out=ptr(o["done"]), history=ptr(s["history"]),
                                  history_out=ptr(o["history"]), history_stride=s["stride"], length=ptr(s["lengths"]),
                                  length_out=ptr(o["length"]))
        need = smq.beam_select_workspace(s["step"])
    elif c["kind"] == "fork":
        o = s["out"]
        s["fork"] = smq.page_fork(ptr(s["table"]), ptr(s["held"]), ptr(s["refs"]), s["rows"], s["rows"], s["width"],
                                  c["page"], s["pages"], ptr(s["parent"]), ptr(s["keep"]), ptr(s["room"]),
                                  ptr(o["table"]), ptr(o["held"]), ptr(o["refs"]), ptr(o["copies"]), ptr(o["free"]))
        need = smq.paged_fork_workspace(s["fork"])
        s["shape"] = smq.attn_shape(c["kv"], c["kv"], c["head_dim"], 0, 0, c["length"])
    else:
        s["batch"] = smq.paged_batch(ptr(s["begin"]), ptr(s["length"]), ptr(s["table"]), c["seqs"], s["tokens"],
                                     s["table"].shape[1])
        s["shape"] = smq.attn_shape(c["heads"], c["kv"], c["head_dim"], c["head_dim"] // 2, c.get("window", 0), c["length"])
        if c["kind"] == "tree":
            need = smq.paged_tree_attention_workspace(s["batch"], s["shape"])
        elif c["kind"] == "norm":
            s["qkv"] = smq.paged_rows(ptr(s["q"]), ptr(s["out"][0]), ptr(s["k"]), ptr(s["v"]), ptr(s["q_norm"]),
                                      ptr(s["k_norm"]), EPS, ptr(s["depth"]) if c["tree"] else None,
                                      s["q"].stride(0), s["out"][0].stride(0), s["k"].stride(0), s["v"].stride(0))
    if c["kind"] != "beam" and s["pool"]:
        layers = range(c.get("layers", 1))
        s["kv"] = [smq.paged_kv(*(ptr(s["pool"][n][i]) if n in s["pool"] else None
                                  for n in ("keys", "values", "key_scales", "value_scales")), TYPES[c["type"]], c["page"],
                                s["pages"]) for i in layers]
        s["pools"] = smq.paged_pools(s["kv"])
    s["workspace"] = torch.empty(max(1, need), dtype=torch.uint8, device="cuda")


# ---- one pass -------------------------------------------------------------

def run(state):
    kind = state["case"]["kind"]
    if own:
        return _run_own(state, kind)
    return {"norm": _norm, "tree": _tree, "fork": _fork, "compact": _compact, "beam": _beam}[kind](state)


def _run_own(s, kind):
    smq, ptr, c = s["smq"], torch.Tensor.data_ptr, s["case"]
    ws, n = ptr(s["workspace"]), s["workspace"].numel()
    if kind == "beam":
        smq.beam_select(s["step"], ws, n)
        return s["out"]
    if kind == "fork":
        smq.paged_fork(s["fork"], ws, n)
        if c["layers"]:
            smq.paged_copy(ptr(s["out"]["copies"]), s["rows"], s["shape"], s["pools"])
        return [s["out"], s["pool"]]
    if kind == "compact":
        smq.paged_compact(s["batch"], s["shape"], ptr(s["accepted"]), s["stride"], ptr(s["count"]), s["pools"],
                          ptr(s["length_out"]))
        return [s["length_out"], s["pool"]]
    if kind == "tree":
        smq.draft_masks(ptr(s["parent"]), s["batch"], ptr(s["depth"]), ptr(s["mask"]), s["words"])
        smq.paged_tree_attention(ptr(s["q"]), ptr(s["out"]), s["batch"], s["shape"], c["sinks"], ptr(s["depth"]),
                                 ptr(s["mask"]), s["words"], s["kv"][0], ws, n)
        return [s["depth"], s["mask"], s["out"]]
    smq.paged_norm_rope_kv(s["qkv"], s["batch"], s["shape"], ptr(s["cos"]), ptr(s["sin"]), s["kv"][0])
    smq.paged_read(s["batch"], s["shape"], s["kv"][0], ptr(s["out"][1]), ptr(s["out"][2]))
    return s["out"]


def _slots(s):
    """Page and slot of every new token."""
    page = s["case"]["page"]
    return s["table"][s["seq"], s["pos"] // page].long(), s["pos"] % page


def _normed(x, w, heads):
    """Each head's RMSNorm: mean and root in 64 bits (values next to a step of the cache's type follow), rounded once."""
    x = x.reshape(x.shape[0], heads, -1)
    inv = (1 / torch.sqrt(x.double().square().mean(-1, keepdim=True) + EPS)).float()
    return x * inv * w


def _rotate(x, cos, sin):
    x = x.reshape(*x.shape[:2], -1, 2)
    a, b, cos, sin = x[..., 0], x[..., 1], cos[:, None], sin[:, None]
    return torch.stack([a * cos - b * sin, a * sin + b * cos], -1).reshape(*x.shape[:2], -1)


def _q8(x):
    """Scales and codes of the 32-wide blocks of [tokens, heads, dims]."""
    pad = -x.shape[-1] % 32
    b = torch.nn.functional.pad(x, (0, pad)).reshape(*x.shape[:-1], -1, 32)
    scale = b.abs().amax(-1) / torch.full((1,), 127.0, device=x.device)
    inv = torch.where(scale >= torch.finfo(torch.float32).tiny, torch.ones_like(scale) / scale, torch.zeros_like(scale))
    code = torch.round(b * inv[..., None]).clamp(-127, 127)
    return scale, code.reshape(*x.shape[:-1], -1)[..., :x.shape[-1]].to(torch.int8)


def _norm(s):
    c, pool = s["case"], {n: x[0] for n, x in s["pool"].items()}
    at = s["first"][s["seq"]] + s["depth"] if c["tree"] else s["pos"]
    cos, sin = s["cos"][at], s["sin"][at]
    q = _rotate(_normed(s["q"], s["q_norm"], c["heads"]), cos, sin)
    k = _rotate(_normed(s["k"], s["k_norm"], c["kv"]), cos, sin)
    v = s["v"].reshape(s["tokens"], c["kv"], -1)
    page, slot = _slots(s)
    if c["type"] == "q8":
        (ks, k), (vs, v) = _q8(k), _q8(v)
        pool["key_scales"][page, :, :, slot] = ks
        pool["value_scales"][page, :, :, slot] = vs
    pool["keys"][page, :, slot] = k.to(pool["keys"].dtype)
    pool["values"][page, :, :, slot] = v.to(pool["values"].dtype)
    k, v = pool["keys"][page, :, slot].float(), pool["values"][page, :, :, slot].float()
    if c["type"] == "q8":
        ks, vs = (pool[n][page, :, :, slot].repeat_interleave(32, -1)[..., :c["head_dim"]]
                  for n in ("key_scales", "value_scales"))
        k, v = k * ks, v * vs
    return [q.reshape(s["tokens"], -1), k.reshape(s["tokens"], -1), v.reshape(s["tokens"], -1)]


def _ancestors(s):
    """Depths, and [token, n] whether a token sees the n-th new token of its sequence: itself and its ancestors."""
    parent, base = s["parent"].long(), s["begin"].long()[s["seq"]]
    seen = torch.zeros(s["tokens"], s["most"], dtype=torch.bool, device="cuda")
    rows = torch.arange(s["tokens"], device="cuda")
    depth, at = torch.full_like(parent, -1), s["place"]
    for _ in range(s["most"]):
        on = at >= 0
        seen[rows, at.clamp(min=0)] |= on
        depth += on
        at = torch.where(on, parent[base + at.clamp(min=0)], at)
    return depth, seen


def _bits(seen, words):
    """Truth values of [rows, n] as words of 32 bits."""
    b = torch.nn.functional.pad(seen, (0, 32 * words - seen.shape[1])).reshape(seen.shape[0], words, 32).long()
    w = (b << torch.arange(32, device="cuda")).sum(-1)
    return torch.where(w >= 1 << 31, w - (1 << 32), w).to(torch.int32)


def _dense(s):
    """Keys and values of every sequence's pages, [sequence, KV head, position, dim]."""
    c, pool, ids = s["case"], s["pool"], s["table"].long().clamp(min=0)
    k = pool["keys"][0][ids].float()
    v = pool["values"][0][ids].float().transpose(-1, -2)
    if c["type"] == "q8":
        k, v = (x * pool[n][0][ids].repeat_interleave(32, 3)[:, :, :, :c["head_dim"]].transpose(-1, -2)
                for x, n in ((k, "key_scales"), (v, "value_scales")))
    return [x.transpose(1, 2).reshape(c["seqs"], c["kv"], -1, c["head_dim"]) for x in (k, v)]


def _tree(s):
    c = s["case"]
    seqs, kv, hd, grp, most = c["seqs"], c["kv"], c["head_dim"], c["heads"] // c["kv"], s["most"]
    depth, sees = _ancestors(s)
    k, v = _dense(s)
    seq, place = s["seq"], s["place"]
    q = torch.zeros(seqs, most, kv, grp, hd, device="cuda")
    q[seq, place] = s["q"].reshape(-1, kv, grp, hd)
    q = q.permute(0, 2, 3, 1, 4).reshape(seqs, kv, grp * most, hd)
    score = (torch.matmul(q, k.transpose(2, 3).contiguous()) / math.sqrt(hd)).reshape(seqs, kv, grp, most, -1)
    first = s["first"][:, None, None]
    p = torch.zeros(seqs, most, dtype=torch.int64, device="cuda")
    p[seq, place] = s["first"][seq] + depth
    j = torch.arange(k.shape[2], device="cuda")[None, None]
    seen = (j < first).expand(-1, most, -1)
    if c["window"]:
        seen = seen & ((j > p[:, :, None] - c["window"]) | (j < c["sinks"]))
    new = torch.zeros(seqs, most, most, dtype=torch.bool, device="cuda")
    new[seq, place] = sees
    at = (j - first).expand(-1, most, -1)
    seen = seen | ((at >= 0) & (at < most) & new.gather(2, at.clamp(0, most - 1)))
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    e = torch.exp(score - score.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min))
    e = e / e.sum(-1, keepdim=True)
    v = torch.where((j < s["length"].long()[:, None, None])[:, :, :, None], v, torch.zeros_like(v))
    out = torch.matmul(e.reshape(seqs, kv, grp * most, -1), v).reshape(seqs, kv, grp, most, hd)
    return [depth.to(torch.int32), _bits(sees, s["words"]), out.permute(0, 3, 1, 2, 4)[seq, place].reshape(s["tokens"], -1)]


def _fork(s):
    c, page, width = s["case"], s["case"]["page"], s["width"]
    x = torch.arange(width, device="cuda")[None]
    parent, keep, room = s["parent"].long(), s["keep"].long(), s["room"].long()
    old = s["table"].long()
    refs = s["refs"].long() - torch.bincount(old[x < s["held"][:, None]], minlength=s["pages"])
    full, part = keep // page, keep % page
    take = old[parent.clamp(min=0)]
    refs = refs + torch.bincount(take[x < full[:, None]], minlength=s["pages"])
    # the last page of a row, if it is not full, is the row's own when no other holds it: of several rows the first one's
    last = take.gather(1, full[:, None].clamp(max=width - 1))[:, 0]
    rows = torch.arange(s["rows"], device="cuda")
    lower = (last[:, None] == last[None]) & (part[None] > 0) & (rows[None] < rows[:, None])
    mine = (part > 0) & (refs[last] == 0) & ~lower.any(1)
    refs = refs.index_put((last[mine],), torch.ones_like(last[mine]))
    # pages for the rest, the lowest free ids in the order of rows and entries
    held = (room + page - 1) // page
    keeps = full + mine
    fresh = (x >= keeps[:, None]) & (x < held[:, None])
    free = torch.nonzero(refs == 0)[:, 0]
    need = int(fresh.sum())
    table = torch.where(x < keeps[:, None], take, torch.full_like(take, -1))
    table[fresh] = free[:need]
    refs = refs.index_put((free[:need],), torch.ones_like(free[:need]))
    copied = (part > 0) & ~mine
    none = torch.full_like(last, -1)
    to = table.gather(1, full[:, None].clamp(max=width - 1))[:, 0]
    copies = torch.stack([torch.where(copied, last, none), torch.where(copied, to, none), part * copied], 1)
    if c["layers"]:
        f, t, n = (y[copied] for y in (last, to, part))
        for name, y in s["pool"].items():
            slot = torch.arange(page, device="cuda")
            slot = slot[:, None] if name == "keys" else slot[None]  # positions are the last axis but of keys
            within = slot < n[:, None, None, None]
            y[:, t] = torch.where(within, y[:, f], y[:, t])
    out = {"table": table, "held": held, "refs": refs, "copies": copies, "free": (free.shape[0] - need) * torch.ones_like(held[:1])}
    return [{k: v.to(torch.int32) for k, v in out.items()}, s["pool"]]


def _compact(s):
    c, page = s["case"], s["case"]["page"]
    k = torch.arange(s["stride"], device="cuda")[None]
    count, first = s["count"].long()[:, None], s["first"][:, None]
    seq, at = torch.nonzero(k < count, as_tuple=True)
    to, frm = s["first"][seq] + at, s["first"][seq] + s["accepted"].long()[seq, at]
    (fp, fs), (tp, ts) = ((s["table"][seq, p // page].long(), p % page) for p in (frm, to))
    for name, y in s["pool"].items():
        if name == "keys":
            y[:, tp, :, ts] = y[:, fp, :, fs]
        else:
            y[:, tp, :, :, ts] = y[:, fp, :, :, fs]
    return [(first + count)[:, 0].to(torch.int32), s["pool"]]


def _beam(s):
    c = s["case"]
    groups, beams, vocab, select = c["groups"], c["beams"], c["vocab"], c["select"]
    l, score, done = s["logits"].double(), s["score"].double(), s["done"] != 0
    top = l.amax(1, keepdim=True)
    cand = score[:, None] + (l - (top + torch.log(torch.exp(l - top).sum(1, keepdim=True))))
    cand = cand.masked_fill(done[:, None], -math.inf)
    cand[:, s["pad"]] = torch.where(done, score, cand[:, s["pad"]])
    cand = cand.reshape(groups, beams * vocab)
    best, at, ids = [], [], torch.arange(beams * vocab, device="cuda")
    for _ in range(select):
        m = cand.amax(1, keepdim=True)
        i = torch.where(cand == m, ids, beams * vocab).amin(1, keepdim=True)
        cand.scatter_(1, i, -math.inf)
        best.append(m)
        at.append(i)
    best, at = torch.cat(best, 1).reshape(-1), torch.cat(at, 1)
    row = (at // vocab + beams * torch.arange(groups, device="cuda")[:, None]).reshape(-1)
    token = (at % vocab).reshape(-1)
    length, over = s["lengths"].long()[row], done[row]
    history = s["history"][row]
    more = ~over & (length < s["stride"])
    spot = length.clamp(max=s["stride"] - 1)[:, None]
    history = history.scatter(1, spot, torch.where(more[:, None], token[:, None].to(torch.int32), history.gather(1, spot)))
    return {"parent": row.to(torch.int32), "token": token.to(torch.int32), "score": best.float(),
            "done": (over | (token == s["eos"])).to(torch.uint8), "length": (length + more).to(torch.int32),
            "history": history}


# ---- what a pass cannot do without ----------------------------------------

def _context(c, first, p):
    """Positions of the context that a token at position p sees, behind `first` positions of it."""
    low = max(0, p + 1 - c["window"]) if c["window"] else 0
    low = min(low, first)
    return first - low + min(c["sinks"], low), low


def work(case):
    c = case
    if c["kind"] == "beam":
        rows, out = c["groups"] * c["beams"], c["groups"] * c["select"]
        return {"bytes": 4.0 * rows * c["vocab"] + 8 * out * (c["history"] + 20), "flops": 4.0 * rows * c["vocab"]}
    if c["kind"] == "fork":
        parent, keep, room, held = _rows(c)
        page, seen, copied = c["page"], set(), 0
        for p, k in zip(parent, keep):
            if k % page:
                copied += k % page if (p, k // page) in seen else 0
                seen.add((p, k // page))
        tables = sum(_ceil(n, page) for n in held) + sum(_ceil(n, page) for n in room)
        pages = sum(_ceil(n, page) - _shared(c) for n in held) + _shared(c) * c["groups"]
        return {"bytes": 4.0 * tables + 8 * pages + 4 * c["layers"] * copied * c["kv"] * c["head_dim"] * BYTES[c["type"]],
                "flops": 0}
    new, length = _batch(c)
    kd = c["kv"] * c["head_dim"]
    row = 2 * kd * BYTES[c["type"]]
    if c["kind"] == "compact":
        moved = sum(sum(i != k for k, i in enumerate(p)) for p in _paths(c))
        return {"bytes": 2.0 * c["layers"] * moved * row + 4 * sum(map(len, _paths(c))), "flops": 0}
    qd = c["heads"] * c["head_dim"]
    if c["kind"] == "norm":  # read q, k, v; write q and the cache; read it back as f32 rows
        return {"bytes": sum(new) * (8 * qd + 8 * kd + 2 * row + 8 * kd), "flops": 7.0 * sum(new) * (qd + kd)}
    seen = union = 0
    for n, m, t in zip(new, length, _trees(c)):
        first, depths, low = m - n, _depths(t), m - n
        for d in depths:
            x, at = _context(c, first, first + d)
            seen += x + d + 1
            low = min(low, at)
        union += n + first - low + min(c["sinks"], low)
    return {"bytes": union * row + 8 * sum(new) * qd, "flops": 4.0 * qd * seen}


# ---- the results in 64 bits -------------------------------------------------

def exact(case, seed):
    c = case
    s = prepare(c, seed)
    if c["kind"] in ("fork", "compact"):
        return None  # whole numbers, and values that are moved as they are
    if c["kind"] == "beam":
        if c["groups"] * c["beams"] * c["vocab"] > 30e6:
            return None
        best = []
        for g in range(c["groups"]):
            r = slice(g * c["beams"], (g + 1) * c["beams"])
            x = torch.log_softmax(s["logits"][r].double(), 1) + s["score"][r].double()[:, None]
            over = s["done"][r] != 0
            x = torch.cat([x[~over].reshape(-1), s["score"][r].double()[over]])
            best.append(torch.sort(x, descending=True).values[:c["select"]])
        return {"parent": None, "token": None, "score": torch.cat(best), "done": None, "length": None, "history": None}
    if c["kind"] == "norm":
        where = s["pos"] if not c["tree"] else s["pos"] - s["place"] + s["depth"]
        turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), _angles(c)[where])[:, None]

        def turned(x, w):
            x = x.double().reshape(s["tokens"], -1, c["head_dim"])
            x = x * torch.rsqrt((x * x).sum(-1, keepdim=True) / c["head_dim"] + EPS) * w.double()
            x = torch.view_as_complex(x.reshape(s["tokens"], -1, c["head_dim"] // 2, 2).contiguous()) * turn
            return torch.view_as_real(x).reshape(s["tokens"], -1)

        q = turned(s["q"], s["q_norm"])
        if c["type"] == "f32":
            return [q, turned(s["k"], s["k_norm"]), s["v"].double()]
        return [q, None, None]  # f16 and Q8 values are rounded from the f32 rotation
    grp, hd, at, out = c["heads"] // c["kv"], c["head_dim"], 0, []
    for i, (n, t) in enumerate(zip(s["new"], _trees(c))):
        m = int(s["length"][i])
        ids = s["table"][i, :_ceil(m, c["page"])].long()
        k, v = s["pool"]["keys"][0][ids].double(), s["pool"]["values"][0][ids].double().transpose(-1, -2)
        if c["type"] == "q8":
            block = torch.arange(hd, device="cuda") // 32
            k = k * s["pool"]["key_scales"][0][ids].double()[:, :, block].transpose(-1, -2)
            v = v * s["pool"]["value_scales"][0][ids].double()[:, :, block].transpose(-1, -2)
        k, v = (x.transpose(0, 1).reshape(c["kv"], -1, hd)[:, :m] for x in (k, v))
        q = s["q"][at:at + n].double().reshape(n, c["kv"], grp, hd)
        hidden = np.ones((n, m), bool)
        for r, d in enumerate(_depths(t)):
            low = max(0, m - n + d + 1 - c["window"]) if c["window"] else 0
            hidden[r, min(low, m - n):m - n] = False
            hidden[r, :min(c["sinks"], m - n)] = False
            a = r
            while a >= 0:
                hidden[r, m - n + a] = False
                a = t[a]
        hidden, heads = torch.from_numpy(hidden).cuda(), []
        for h in range(c["heads"]):
            w = q[:, h // grp, h % grp] @ k[h // grp].T / math.sqrt(hd)
            heads.append(torch.softmax(w.masked_fill(hidden, -math.inf), -1) @ v[h // grp])
        out.append(torch.cat(heads, 1))
        at += n
    return [None, None, torch.cat(out)]
