"""Cases of tests/test_drafts_host.py, each in a process of its own: drafts_host_cases.py FAKE_HIP_LIBRARY CASE. Refusals and
empty calls of the operators of drafts and beams over the recording runtime of tests/fake_hip.cpp, without a GPU."""
import itertools
import os
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, HERE)
import paged_host_cases as base  # noqa: E402
from paged_host_cases import RANGE, Paged, launches, refused  # noqa: E402

smq = fake = None
TOP = 0xFFFFFFFF


class Drafts(Paged):
    """The arguments of valid calls on a batch; keyword arguments change descriptors or buffer sizes."""

    def __init__(self, pools=1, words=2, stride=5, qs=0, os_=0, ks=0, vs=0, norms=True, depth=True, eps=1e-6, short=None, **kw):
        own = ("q_norm", "k_norm", "depth", "parent", "mask", "accepted", "count", "out", "copies", "sq", "so", "sk", "sv")
        super().__init__(short=None if short in own else short, **kw)
        o = self.o
        wide = lambda n, width, s: 4 * ((n - 1) * (s or width) + width) if n else 4  # noqa: E731
        qd, kd, n = o["heads"] * o["hd"], o["kv"] * o["hd"], o["tokens"]
        size = {"q_norm": 4 * o["hd"], "k_norm": 4 * o["hd"], "depth": 4 * n, "parent": 4 * n, "mask": 4 * n * words,
                "accepted": 4 * o["seqs"] * stride, "count": 4 * o["seqs"], "out": 4 * o["seqs"], "copies": 12 * 3,
                "sq": wide(n, qd, qs), "so": wide(n, qd, os_), "sk": wide(n, kd, ks), "sv": wide(n, kd, vs)}
        if short in size:
            size[short] -= 1
        self.b.update({k: smq.DeviceBuffer(max(1, s)) for k, s in size.items()})
        self.words, self.stride = words, stride
        b = self.b
        self.rows = smq.paged_rows(b["sq"], b["so"], b["sk"], b["sv"], b["q_norm"] if norms else None,
                                   b["k_norm"] if norms else None, eps, b["depth"] if depth else None, qs, os_, ks, vs)
        self.pools = smq.paged_pools([self.kv] * pools)
        need = smq.load().smq_paged_tree_attention_workspace(self.batch, self.shape)
        smq.load().smq_clear_error()
        self.tws = smq.DeviceBuffer(need + 16)

    def norm(self):
        smq.paged_norm_rope_kv(self.rows, self.batch, self.shape, self.b["cos"], self.b["sin"], self.kv)

    def masks(self):
        smq.draft_masks(self.b["parent"], self.batch, self.b["depth"], self.b["mask"], self.words)

    def tree(self, ws=None, n=0, **kw):
        b = dict(self.b, **kw)
        smq.paged_tree_attention(b["q"], b["att"], self.batch, self.shape, 0, b["depth"], b["mask"], self.words, self.kv,
                                 ws or self.tws, n)

    def compact(self, **kw):
        b = dict(self.b, **kw)
        smq.paged_compact(self.batch, self.shape, b["accepted"], self.stride, b["count"], self.pools, b["out"])

    def copy(self, rows=3):
        smq.paged_copy(self.b["copies"], rows, self.shape, self.pools)


ON_BATCHES = ("norm", "masks", "tree", "compact")


def valid_calls():
    for kv_type in (0, 1, 2):
        for hd in (16, 64, 80, 256):
            for page in (16, 256):
                p = Drafts(type=kv_type, hd=hd, pairs=hd // 2, page=page, pools=3)
                for f in (p.norm, p.masks, p.tree, p.compact, p.copy):
                    fake.fake_clear()
                    f()
                    assert launches() >= 1, f
    p = Drafts(norms=False, depth=False)
    p.norm()
    p.rows.q = p.rows.q_out = None
    p.norm()
    p.tree(depth=None)
    p = Drafts(qs=300, os_=256, ks=130, vs=777)
    p.norm()
    p.rows.q_out, p.rows.q_out_stride = p.rows.q, 300  # in place
    p.norm()
    smq.paged_tree_attention(p.b["q"], p.b["att"], p.batch, p.shape, 0, None, p.b["mask"], 2, p.kv)  # no workspace
    # more pools than a launch holds, and a grid that several launches share
    p = Drafts(pools=100)
    fake.fake_clear()
    p.copy()
    assert launches() == 3
    p.compact()
    assert launches() == 3
    big = Drafts(seqs=1000, tokens=1, kv=512, heads=512, hd=16, pairs=0, page=16, pages=1, stride=1, type=1, pools=20)
    fake.fake_clear()
    big.compact()
    g = [int(line.split(" grid ")[1].split()[0]) for line in fake.fake_log().decode().splitlines()]
    assert len(g) == 3 and max(g) <= 1 << 23 and sum(g) == 20 * 512 * 1000
    fake.fake_clear()


def empty_batches():
    for kw in (dict(seqs=0), dict(tokens=0), dict(seqs=0, tokens=0)):
        p = Drafts(**kw)
        fake.fake_clear()
        p.norm()
        p.masks()
        p.tree()
        assert launches() == 0
    p = Drafts(seqs=0)
    p.compact()
    p.copy(0)
    assert launches() == 0
    none = smq.paged_batch(None, None, None, 0, 0, 0)
    smq.paged_tree_attention(None, None, none, p.shape, 0, None, None, 1, p.kv)
    smq.draft_masks(None, none, None, None, 1)
    smq.paged_copy(None, 0, p.shape, p.pools)
    assert launches() == 0
    # sequences without new tokens have nothing accepted, and a length
    p = Drafts(tokens=0)
    p.compact()
    assert launches() == 1


def shapes():
    for kw in (dict(hd=8, pairs=4), dict(hd=24, pairs=12), dict(hd=272, pairs=8), dict(heads=5), dict(context=0, pairs=0),
               dict(page=8), dict(page=48), dict(page=512), dict(type=3), dict(pages=0)):
        p = Drafts(**kw)
        for f in (p.norm, p.tree, p.compact, p.copy):
            refused(f)
    for field, value in (("seqs", (1 << 20) + 1), ("tokens", (1 << 24) + 1)):
        p = Drafts()
        setattr(p.batch, field, value)
        for f in ON_BATCHES:
            refused(getattr(p, f), words="unsupported batch")
    for words in (0, 129, TOP):
        p = Drafts()
        p.words = words
        refused(p.masks, words="mask rows")
        refused(p.tree, words="mask rows")
    p = Drafts(window=7)
    p.tree()
    refused(lambda: p.tree(depth=None), words="a window without depths")
    for eps in (-1e-6, float("nan"), float("inf")):
        refused(Drafts(eps=eps).norm, words="eps")
    for stride in (0, (1 << 22) + 1):
        p = Drafts()
        p.stride = stride
        refused(p.compact, words="accepted_stride")
    p = Drafts()
    p.batch.seqs = 1 << 20
    p.shape.kv_heads = p.shape.heads = 8
    p.batch.tokens = 1
    refused(p.compact, words="KV heads exceed")
    refused(lambda: p.copy(1 << 20), words="KV heads exceed")


def buffers():
    for name, calls in {"sq": "n", "so": "n", "sk": "n", "sv": "n", "q_norm": "n", "k_norm": "n", "depth": "nmt", "cos": "n",
                        "sin": "n", "keys": "ntcy", "values": "ntcy", "ks": "ntcy", "vs": "ntcy", "begin": "nmtc",
                        "length": "ntc", "table": "ntc", "parent": "m", "mask": "mt", "q": "t", "att": "t", "accepted": "c",
                        "count": "c", "out": "c", "copies": "y"}.items():
        p = Drafts(short=name)
        for c in calls:
            refused({"n": p.norm, "m": p.masks, "t": p.tree, "c": p.compact, "y": p.copy}[c], words="exceed its allocation")
    for strides in (dict(qs=300), dict(os_=300), dict(ks=130), dict(vs=130)):
        for short in ("sq", "so", "sk", "sv"):
            refused(Drafts(short=short, **strides).norm, words="exceed its allocation")
    for field in ("begin", "length", "table"):
        p = Drafts()
        setattr(p.batch, field, None)
        for f in (p.norm, p.tree, p.compact) + ((p.masks,) if field == "begin" else ()):
            refused(f, words="NULL")
    for field in ("k", "v"):
        p = Drafts()
        setattr(p.rows, field, None)
        refused(p.norm, words="NULL")
    p = Drafts()
    p.rows.q = None
    refused(p.norm, words="q_out without q")
    p = Drafts()
    p.rows.q_out = None
    refused(p.norm, words="q without q_out")
    p = Drafts(qs=300)
    p.rows.q_out = p.rows.q
    refused(p.norm, words="in place with another stride")
    for field in ("q_stride", "q_out_stride", "k_stride", "v_stride"):
        for value in (1, 127, 1 << 62, (1 << 64) - 1):
            p = Drafts()
            setattr(p.rows, field, value)
            refused(p.norm, words="a row stride")
        p = Drafts()
        setattr(p.rows, field, 1 << 56)
        refused(p.norm, words="exceed its allocation")
    p = Drafts()
    refused(lambda: smq.draft_masks(p.b["parent"], p.batch, p.b["parent"], p.b["mask"], 2), words="overlap")
    refused(lambda: smq.draft_masks(p.b["parent"], p.batch, p.b["mask"], p.b["mask"], 2), words="overlap")
    refused(lambda: p.tree(p.tws.at(4), 16), words="aligned")
    refused(lambda: p.tree(p.tws.at(0), p.tws.nbytes + 16), words="exceed its allocation")
    refused(lambda: p.tree(mask=None), words="NULL")
    refused(lambda: p.compact(out=p.b["length"]), words="overlaps")
    refused(lambda: p.compact(out=p.b["count"]), words="overlaps")
    refused(lambda: p.compact(out=p.b["accepted"]), words="overlaps")
    # pools of layers: alike, all there, not too many
    for field, value in (("type", 1), ("page_size", 64), ("pages", 19)):
        p = Drafts(pools=3)
        setattr(p.pools[2], field, value)
        refused(p.copy, words="pool 2")
        refused(p.compact, words="pool 2")
    p = Drafts(pools=3)
    p.pools[1].values = None
    refused(p.copy, words="NULL")
    p = Drafts(pools=1025)
    refused(p.copy, words="pools")
    lib = smq.load()
    p = Drafts()
    for call in (lambda: lib.smq_paged_norm_rope_kv(None, p.batch, p.shape, None, None, p.kv),
                 lambda: lib.smq_paged_norm_rope_kv(p.rows, None, p.shape, None, None, p.kv),
                 lambda: lib.smq_paged_norm_rope_kv(p.rows, p.batch, p.shape, None, None, None),
                 lambda: lib.smq_draft_masks(None, None, None, None, 1),
                 lambda: lib.smq_paged_tree_attention(None, None, p.batch, p.shape, 0, None, None, 1, None, None, 0),
                 lambda: lib.smq_paged_tree_attention(None, None, None, p.shape, 0, None, None, 1, p.kv, None, 0),
                 lambda: lib.smq_paged_compact(p.batch, p.shape, None, 1, None, None, 0, None),
                 lambda: lib.smq_paged_compact(p.batch, None, None, 1, None, p.pools, 1, None),
                 lambda: lib.smq_paged_copy(None, 1, p.shape, None, 1),
                 lambda: lib.smq_paged_copy(None, 1, None, p.pools, 1),
                 lambda: lib.smq_paged_copy(None, 1, p.shape, p.pools, 0),
                 lambda: lib.smq_paged_fork(None, None, 0), lambda: lib.smq_beam_select(None, None, 0)):
        assert call() == RANGE
        lib.smq_clear_error()
    assert lib.smq_paged_tree_attention_workspace(None, p.shape) == 0
    assert lib.smq_paged_fork_workspace(None) == lib.smq_beam_select_workspace(None) == 0
    lib.smq_clear_error()


def results_over_descriptors():
    """What a call writes shares no byte with what its other workgroups read."""
    p = Drafts()
    for name in ("begin", "length", "table", "accepted", "count"):
        for at in (p.b[name].ptr, p.b[name].ptr + p.b[name].nbytes - 12):
            refused(lambda: p.compact(out=at), words="length_out overlaps " + name)
    b, mask = p.b, p.b["mask"]
    for out, args in (("depth", lambda at: (at, mask)), ("mask", lambda at: (b["depth"], at))):
        big = smq.DeviceBuffer(4096)
        p.batch.begin = big.at(12)
        refused(lambda: smq.draft_masks(b["parent"], p.batch, *args(big), 2), words=out + " overlaps begin")
    p = Drafts()
    for name in ("q", "depth", "mask"):
        refused(lambda: p.tree(**{name: p.b["att"].at(0 if name == "q" else 16)}), words="att overlaps " + name)


def pools_that_share_memory():
    """Refused, whichever kinds of arrays share a byte, in any order; a pool that is named again is not."""
    for kv_type, codes in ((0, 4), (1, 2), (2, 1)):
        p = Drafts(type=kv_type)
        k, w = 20 * 32 * 2 * 64 * codes, 20 * 32 * 2 * 2 * 4  # bytes of keys, of their scales
        room = smq.DeviceBuffer(40 * (k + w))
        at = lambda i: [room.ptr + i * 2 * (k + w) + x for x in (0, k, 2 * k, 2 * k + w)]  # noqa: E731

        def call(*arrays):
            p.pools = smq.paged_pools([smq.paged_kv(*x, kv_type, 32, 20) for x in arrays])
            fake.fake_clear()
            p.copy()
            p.compact()
            assert launches() == 2

        layers = [at(i) for i in range(12)]
        call(*layers)
        call(*layers[::-1])
        call(*(layers[i] for i in (5, 0, 11, 2, 7, 3)))
        call(*(layers[i] for i in (5, 0, 5, 11, 0, 0, 5)))
        call(*([x[1], x[0], x[3], x[2]] if i % 2 else x for i, x in enumerate(layers)))
        every = range(4 if kv_type == 2 else 2)
        for i in every:
            for j in every:
                for off in (0, 16, -16):
                    bad = [list(x) for x in layers]
                    bad[9][i] = bad[4][j] + off
                    if i != j or off:
                        for f in (p.copy, p.compact):
                            for order in (bad, bad[::-1]):
                                p.pools = smq.paged_pools([smq.paged_kv(*x, kv_type, 32, 20) for x in order])
                                refused(f, words="pools overlap")
        for i in every:  # the keys of another pool, but not its values
            bad = [list(x) for x in layers]
            bad[9] = list(bad[4])
            bad[9][i] = layers[9][i]
            p.pools = smq.paged_pools([smq.paged_kv(*x, kv_type, 32, 20) for x in bad])
            refused(p.compact, words="pools overlap")
        # a run of layers for each kind
        begin = [0, 12 * k, 24 * k, 24 * k + 12 * w]
        run = lambda i, moved=-1, by=0: [room.ptr + 4096 + b + (by if n == moved else 0) + i * x  # noqa: E731
                                         for n, (b, x) in enumerate(zip(begin, (k, k, w, w)))]
        call(*(run(i) for i in range(12)))
        for i in every:
            for by in (16, -16):
                if 0 <= i + (by > 0) - (by < 0) < len(every):  # into the next kind's run
                    p.pools = smq.paged_pools([smq.paged_kv(*run(x, i, by), kv_type, 32, 20) for x in range(12)])
                    refused(p.compact, words="pools overlap")
            for n in (1, 11):
                p.pools = smq.paged_pools([smq.paged_kv(*run(x, i if x == n else -1, -16), kv_type, 32, 20) for x in range(12)])
                refused(p.compact, words="pools overlap")
        if kv_type < 2:  # scales are not looked at
            for x in layers:
                x[2:] = layers[0][:2]
            call(*layers)


def fork(short=None, **kw):
    o = dict(old=5, seqs=7, stride=9, page=32, pages=60)
    o.update({k: v for k, v in kw.items() if k in o})
    size = dict(table=4 * o["old"] * o["stride"], held=4 * o["old"], refs=4 * o["pages"], parent=4 * o["seqs"],
                keep=4 * o["seqs"], room=4 * o["seqs"], table_out=4 * o["seqs"] * o["stride"], held_out=4 * o["seqs"],
                refs_out=4 * o["pages"], copies=12 * o["seqs"], free_out=4)
    b = {k: smq.DeviceBuffer(max(1, n - (k == short))) for k, n in size.items()}
    b.update({k: v(b) if callable(v) else v for k, v in kw.items() if k in b})
    f = smq.page_fork(b["table"], b["held"], b["refs"], o["old"], o["seqs"], o["stride"], o["page"], o["pages"], b["parent"],
                      b["keep"], b["room"], b["table_out"], b["held_out"], b["refs_out"], b["copies"], b["free_out"])
    for k, v in kw.items():
        if k.startswith("set_"):
            setattr(f, k[4:], v)
    need = smq.load().smq_paged_fork_workspace(f)
    smq.load().smq_clear_error()
    ws = smq.DeviceBuffer(need + 16)
    fake.fake_clear()
    smq.paged_fork(f, kw.get("ws", lambda w: w)(ws), max(1, need + kw.get("more", 0)))
    return launches()


def forks():
    assert fork() == 1 and fork(seqs=0) == 1 and fork(old=0) == 1  # in one workgroup
    assert fork(pages=8193) == 4 and fork(old=257) == 4 and fork(seqs=257) == 4 and fork(stride=4000) == 4
    assert fork(pages=9000, seqs=0) == 4 and fork(pages=9000, seqs=0, old=0) == 3
    for name in ("table", "held", "refs", "parent", "keep", "room", "table_out", "held_out", "refs_out", "copies", "free_out"):
        refused(fork, name, words="exceed its allocation")
        refused(lambda: fork(**{name: None}), words="NULL")
    for out in ("table_out", "held_out", "refs_out", "copies", "free_out"):
        for old in ("table", "held", "refs", "parent", "keep", "room"):
            buf = smq.DeviceBuffer(4096)
            refused(lambda: fork(**{out: buf, old: buf}), words=out + " overlaps " + old)
    outs = ("table_out", "held_out", "refs_out", "copies", "free_out")
    for i, out in enumerate(outs):
        for other in outs[:i]:
            buf = smq.DeviceBuffer(4096)
            refused(lambda: fork(**{out: buf, other: buf}), words=out + " overlaps " + other)
    for kw in (dict(page=8), dict(page=48), dict(page=512), dict(page=0), dict(stride=0), dict(pages=0), dict(set_old_seqs=65536),
               dict(set_seqs=65536), dict(set_table_stride=(1 << 20) + 1), dict(set_pages=(1 << 24) + 1)):
        refused(lambda: fork(**kw), words="unsupported tables")
    refused(lambda: fork(more=-1), words="workspace")
    refused(lambda: fork(ws=lambda w: w.at(4)), words="aligned")
    assert fork(ws=lambda w: w.at(16)) == 1


def beam(short=None, **kw):
    o = dict(groups=3, beams=4, vocab=999, select=5, stride=1003, hs=20)
    o.update({k: v for k, v in kw.items() if k in o})
    rows, n = o["groups"] * o["beams"], o["groups"] * o["select"]
    size = dict(logits=4 * ((max(rows, 1) - 1) * o["stride"] + o["vocab"]), score=4 * rows, done=rows, parent=4 * n, token=4 * n,
                score_out=4 * n, done_out=n, history=4 * rows * o["hs"], history_out=4 * n * o["hs"], length=4 * rows,
                length_out=4 * n)
    b = {k: smq.DeviceBuffer(max(1, x - (k == short))) for k, x in size.items()}
    b.update({k: v for k, v in kw.items() if k in b})
    s = smq.beam_step(b["logits"], o["stride"], o["groups"], o["beams"], o["vocab"], o["select"], b["score"], b["parent"],
                      b["token"], b["score_out"], done=b["done"], done_out=b["done_out"], history=b["history"],
                      history_out=b["history_out"], history_stride=o["hs"], length=b["length"], length_out=b["length_out"])
    for k, v in kw.items():
        if k.startswith("set_"):
            setattr(s, k[4:], v)
    need = smq.load().smq_beam_select_workspace(s)
    smq.load().smq_clear_error()
    ws = smq.DeviceBuffer(need + 16)
    fake.fake_clear()
    smq.beam_select(s, kw.get("ws", lambda w: w)(ws), max(1, need + kw.get("more", 0)))
    return launches()


def beams():
    assert beam() == 3 and beam(groups=0) == 0
    assert beam(done=None) == beam(done_out=None) == beam(history=None, history_out=None, length=None, length_out=None) == 3
    assert beam(beams=64, select=64, groups=1) == 3 and beam(vocab=1, stride=1) == 3
    for name in ("logits", "score", "done", "parent", "token", "score_out", "done_out", "history", "history_out", "length",
                 "length_out"):
        refused(beam, name, words="exceed its allocation")
        if name not in ("done", "done_out", "history"):
            refused(lambda: beam(**{name: None}), words="NULL")
    for out in ("parent", "token", "score_out", "done_out", "history_out", "length_out"):
        for old in ("logits", "score", "done", "history", "length"):
            buf = smq.DeviceBuffer(1 << 17)
            refused(lambda: beam(**{out: buf, old: buf.at(4)}), words=out + " overlaps " + old)
    buf = smq.DeviceBuffer(1 << 17)
    refused(lambda: beam(token=buf, score_out=buf), words="score_out overlaps token")
    for kw in (dict(set_beams=0), dict(set_beams=65), dict(set_select=0), dict(set_select=65), dict(set_vocab=0),
               dict(set_vocab=(1 << 20) + 1), dict(set_groups=16384), dict(set_groups=TOP)):
        refused(lambda: beam(**kw), words="unsupported step")
    refused(lambda: beam(set_stride=998), words="a row stride")
    refused(lambda: beam(set_stride=1 << 62), words="a row stride")
    refused(lambda: beam(set_stride=(1 << 64) - 1), words="a row stride")
    refused(lambda: beam(set_history_stride=0), words="history_stride")
    refused(lambda: beam(set_history_stride=1 << 31), words="history_stride")
    refused(lambda: beam(more=-1), words="workspace")
    refused(lambda: beam(ws=lambda w: w.at(4)), words="aligned")
    # of one row the stride is not looked at
    assert beam(groups=1, beams=1, set_stride=0) == 3


def beam_workspace_of_the_largest_step():
    """A workspace for the most rows, ids and choices serves every call of fewer."""
    lib = smq.load()

    def need(groups, beams_, vocab, select):
        s = smq.beam_step(None, vocab, groups, beams_, vocab, select, None, None, None, None)
        return lib.smq_beam_select_workspace(s)

    for groups, b, vocab, select in ((16, 8, 151936, 16), (4, 4, 151936, 8), (1, 13, 151936, 3), (100, 64, 999, 64)):
        have = need(groups, b, vocab, select)
        for g in {1, groups // 2 or 1, groups}:
            for k in {1, b // 2 or 1, b}:
                for v in {1, vocab // 3, vocab - 1, vocab}:
                    for n in {1, select // 2 or 1, select}:
                        assert 0 < need(g, k, v, n) <= have


def captures():
    """Every call may be captured and allocates nothing there."""
    p = Drafts(pools=3)
    before = fake.fake_errors()
    f = smq.page_fork(*[smq.DeviceBuffer(4096) for _ in range(3)], 5, 5, 9, 32, 60, *[smq.DeviceBuffer(4096) for _ in range(8)])
    ws = smq.DeviceBuffer(smq.paged_fork_workspace(f))
    b = smq.beam_step(smq.DeviceBuffer(4 * 999 * 4), 999, 1, 4, 999, 5, *[smq.DeviceBuffer(64) for _ in range(4)])
    bws = smq.DeviceBuffer(smq.beam_select_workspace(b))
    g = smq.capture(lambda: (p.norm(), p.masks(), p.tree(), p.compact(), p.copy(), smq.paged_fork(f, ws), smq.beam_select(b, bws)))
    fake.fake_clear()
    g.launch()
    assert launches() >= 9 and fake.fake_errors() == before == b""
    g.destroy()


def widest_split():
    """The bytes that the query of tree attention gives make the launches that boundless ones would, whatever sinks and table the
    call brings."""
    cut = 0
    for kv_type, (heads, kv, hd, seqs, new, window, context) in itertools.product((0, 1, 2), (
            (32, 4, 64, 8, 1, 64, 5000), (32, 8, 128, 1, 16, 512, 131072), (14, 2, 64, 3, 9, 1000, 32768),
            (4, 1, 64, 1, 1, 16, 1 << 20), (8, 2, 128, 2, 300, 200, 9000), (32, 8, 128, 6, 64, 33, 60000),
            (8, 2, 256, 1, 100, 0, 4000), (4, 1, 64, 1, 1, 0, 1 << 20), (14, 2, 64, 1, 13, 0, 3000), (12, 2, 128, 24, 40, 0, 3001),
            (14, 2, 64, 8, 16, 100, 2000))):
        p = Drafts(heads=heads, kv=kv, hd=hd, pairs=0, type=kv_type, page=64, pages=1, seqs=seqs, tokens=seqs * new,
                   stride=-(-context // 64), window=window, context=context, words=16)
        p.batch.table_stride = table = -(-context // 64)
        p.b["table"] = smq.DeviceBuffer(4 * seqs * table)
        p.batch.table = p.b["table"].ptr
        need = smq.load().smq_paged_tree_attention_workspace(p.batch, p.shape)
        large = smq.DeviceBuffer(max(4 * need, 1 << 28))
        for sinks in (0, 1, 100, 4000, context - 500, context, TOP):
            for t in (table, table - 1, table // 2 + 1):
                p.batch.table_stride = t
                got = []
                for n in (large.nbytes, need):
                    fake.fake_clear()
                    smq.paged_tree_attention(p.b["q"], p.b["att"], p.batch, p.shape, sinks, p.b["depth"], p.b["mask"], 16, p.kv,
                                             large.at(0), n)
                    got.append(base.grids())
                assert got[0] == got[1], (kv_type, heads, kv, hd, seqs, new, window, context, sinks, t, need, got)
                cut += len(got[0]) == 2
    assert cut > 150


def widest_split_of_many_tiles():
    """The same where tiles of 64 rows number 512 to 767, whole for one type of cache and cut for another."""
    cut = set()
    for kv_type, (heads, kv, hd, seqs, new, window, context) in itertools.product((0, 1, 2), (
            (32, 8, 128, 64, 8, 0, 4096), (32, 8, 128, 80, 8, 0, 8192), (32, 8, 128, 72, 16, 0, 3001), (32, 8, 128, 70, 16, 0, 16384),
            (28, 4, 128, 128, 8, 0, 4096), (32, 8, 64, 16, 63, 0, 8192), (12, 2, 128, 300, 8, 0, 4000), (24, 8, 112, 70, 16, 3000, 9000),
            (24, 8, 96, 72, 20, 0, 8000), (16, 8, 256, 70, 30, 0, 8000))):
        p = Drafts(heads=heads, kv=kv, hd=hd, pairs=0, type=kv_type, page=64, pages=1, seqs=seqs, tokens=seqs * new,
                   window=window, context=context, words=2)
        p.batch.table_stride = -(-context // 64)
        p.b["table"] = smq.DeviceBuffer(4 * seqs * p.batch.table_stride)
        p.batch.table = p.b["table"].ptr
        need = smq.load().smq_paged_tree_attention_workspace(p.batch, p.shape)
        large = smq.DeviceBuffer(1 << 31)
        for sinks in (0, 100, TOP):
            got = []
            for n in (large.nbytes, need):
                fake.fake_clear()
                smq.paged_tree_attention(p.b["q"], p.b["att"], p.batch, p.shape, sinks, p.b["depth"], p.b["mask"], 2, p.kv,
                                         large.at(0) if n else None, n)
                got.append(base.grids())
            assert got[0] == got[1], (kv_type, heads, kv, hd, seqs, new, window, context, sinks, need, got)
            if len(got[0]) == 2:
                cut.add((kv_type, heads, kv, seqs, new))
        large.free()
    assert {(2, 32, 8, 64, 8), (2, 32, 8, 80, 8), (2, 28, 4, 128, 8), (2, 12, 2, 300, 8), (0, 24, 8, 72, 20)} <= cut, cut


CASES = [valid_calls, empty_batches, shapes, buffers, forks, beams, beam_workspace_of_the_largest_step, captures, widest_split,
         widest_split_of_many_tiles, pools_that_share_memory,
         results_over_descriptors]

if __name__ == "__main__":
    base.load(sys.argv[1])
    smq, fake = base.smq, base.fake
    {f.__name__: f for f in CASES}[sys.argv[2]]()
    print("ok")
