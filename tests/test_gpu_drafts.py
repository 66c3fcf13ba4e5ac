"""Drafted tokens and beams over the paged cache on the GPU: whole numbers, pools and normed rows bit for bit against numpy,
attention against 64 bits within the bound beside tree64, scores of beams against 64 bits."""
import numpy as np
import pytest
import torch

import drafts_ref as ref
from checks import assert_same_f32, say
from paged_ref import F16, F32, Q8, Batch, Cache, attend64, rotate, tables
from smq_pkg import smq, synth

pytestmark = pytest.mark.gpu
dev = smq.DeviceBuffer.from_array
TYPES = {F32: "f32", F16: "f16", Q8: "q8"}
NONE = ref.NONE


@pytest.fixture(scope="module", autouse=True)
def gpu():
    assert smq.init(0) == "gfx950"
    yield


def same(got, want):
    got, want = np.ascontiguousarray(got), np.ascontiguousarray(want)
    if want.dtype == np.float16:
        got, want = got.view(np.uint16), want.view(np.uint16)
    elif want.dtype == np.float32:
        return assert_same_f32(got, want)
    assert np.array_equal(got, want), np.argwhere(got != want)[:5]


def flagged():
    try:
        smq.numeric_check()
    except smq.SmqError as e:
        assert e.status == smq.SM_ERR_NUMERIC
        return True
    return False


def close(got, want, tol, what=""):
    d = np.abs(got.astype(np.float64) - want)
    bad = ~(d <= tol)
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} off, worst {np.nanmax(d / np.maximum(tol, 1e-30)):.3g} of the " \
                          f"bound at {np.argwhere(bad)[0]}: {got[bad][0]} for {want[bad][0]}"


def pool_same(cache):
    for got, want in zip(cache.download(), (cache.k, cache.v, cache.ks, cache.vs)):
        same(got, want)


# ---- norms, rotation, store -------------------------------------------------

NORMS = [  # type, heads, kv, hd, pairs, page, lengths, new, packed, tree
    (Q8, 14, 2, 64, 32, 64, [200, 1, 65, 130], [8, 1, 1, 16], True, True),
    (F16, 12, 2, 128, 64, 32, [133, 70, 40], [133, 5, 0], False, False),
    (F32, 9, 3, 64, 16, 16, [17, 40], [17, 3], True, False),
    (Q8, 16, 2, 80, 40, 256, [300, 257], [290, 257], False, True),
    (Q8, 4, 4, 16, 8, 16, [33], [20], True, True),
    (F16, 2, 1, 256, 0, 128, [129, 3], [2, 2], False, False),
    (F32, 8, 8, 96, 48, 64, [64, 63, 65], [64, 63, 65], True, True),
    (F16, 32, 8, 48, 24, 128, [50], [1], False, False),
    (Q8, 5, 1, 112, 30, 32, [70, 90], [1, 33], True, True),
]


@pytest.mark.parametrize("norms", ["both", "q", "none"])
@pytest.mark.parametrize("kv_type,heads,kv,hd,pairs,page,lengths,new,packed,tree", NORMS)
def test_norm_rope_store(kv_type, heads, kv, hd, pairs, page, lengths, new, packed, tree, norms):
    say("paged norm", TYPES[kv_type], heads, kv, hd, pairs, page, lengths, new, packed, tree, norms)
    rng = np.random.default_rng(5)
    cache = Cache(kv_type, kv, hd, page, lengths).upload()
    batch = Batch(cache, new, padding=3)
    context, n, eps = max(lengths) + 5, batch.tokens, 1e-5
    shape = smq.attn_shape(heads, kv, hd, pairs, 0, context)
    cos, sin = tables(context, pairs)
    if not pairs:
        cos = sin = np.zeros(1, np.float32)
    qd, kd, gap = heads * hd, kv * hd, 7
    row = synth.normal(70, n * (qd + 2 * kd + gap), 3.0).reshape(n, -1)
    row[0, qd:qd + hd] *= 1e-30
    row[-4, :hd] *= 1e25  # squares past f32
    q, k, v = (np.ascontiguousarray(row[:, a:b]).reshape(n, -1, hd) for a, b in ((0, qd), (qd, qd + kd), (qd + kd, qd + 2 * kd)))
    w = [(1 + 0.3 * rng.standard_normal(hd)).astype(np.float32) for _ in range(2)]
    qw, kw = (w[0] if norms != "none" else None), (w[1] if norms == "both" else None)
    depth = np.full(n, 10 ** 6, np.int32)  # of padding: never read
    at, places = 0, []
    for s, pos in batch.where():
        if len(pos):
            depth[at:at + len(pos)] = ref.masks(ref.random_tree(rng, len(pos)))[0]
            places += list(pos[0] + depth[at:at + len(pos)] if tree else pos)
            at += len(pos)
    with np.errstate(over="ignore"):
        qn, kn = ref.normed(q, qw, eps), ref.normed(k, kw, eps)
    want_q, at = np.full_like(q, 7.0), 0
    for s, pos in batch.where():
        rows, turn = slice(at, at + len(pos)), np.array(places[at:at + len(pos)], int)
        if len(pos):
            want_q[rows] = rotate(qn[rows], cos[turn], sin[turn], pairs) if pairs else qn[rows]
            cache.put(s, pos, rotate(kn[rows], cos[turn], sin[turn], pairs) if pairs else kn[rows], v[rows])
        at += len(pos)
    norm_bufs = [None if x is None else dev(x) for x in (qw, kw)]
    db, cb, sb = dev(depth) if tree else None, dev(cos), dev(sin)
    wide = qd + 2 * kd + gap
    if packed:
        buf = dev(row)
        args = (buf, buf.at(4 * qd), buf.at(4 * (qd + kd)))
        strides = dict(q_stride=wide, k_stride=wide, v_stride=wide)
    else:
        args, strides = (dev(q), dev(k), dev(v)), {}
    out = dev(np.full((n, qd + gap), 7.0, np.float32))

    def store(q_in, q_out, **kw):
        r = smq.paged_rows(q_in, q_out, args[1], args[2], *norm_bufs, eps, db, **{**strides, **kw})
        smq.paged_norm_rope_kv(r, batch.desc, shape, cb, sb, cache.desc)

    store(args[0], out, q_out_stride=qd + gap)
    if kv_type == F16 or not kv_type:
        assert not flagged()
    else:
        smq.numeric_check()
    got = out.download(np.float32).reshape(n, -1)
    same(got[:, :qd].reshape(q.shape), want_q)
    assert (got[:, qd:] == 7.0).all()
    pool_same(cache)
    store(None, None)
    pool_same(cache)
    store(args[0], args[0], q_out_stride=wide if packed else 0)  # in place
    want_q[at:] = q[at:]
    got = args[0].download(np.float32).reshape(n, -1)
    same(got[:, :qd].reshape(q.shape), want_q)
    if packed:
        same(got[:, qd:], row[:, qd:])
    smq.numeric_check()


def test_norm_without_norms_is_rope_kv():
    """No norms, no depths: smq_paged_rope_kv's bits."""
    for kv_type in (F32, F16, Q8):
        caches = [Cache(kv_type, 2, 80, 32, [70, 33]).upload() for _ in range(2)]
        batch = [Batch(c, [40, 1]) for c in caches]
        shape = smq.attn_shape(6, 2, 80, 33, 0, 70)
        cos, sin = (dev(x) for x in tables(70, 33))
        q, k, v = (dev(synth.normal(20 + i, 41 * w)) for i, w in enumerate((480, 160, 160)))
        outs = [smq.DeviceBuffer(41 * 480 * 4) for _ in range(2)]
        smq.paged_rope_kv(q, outs[0], k, v, batch[0].desc, shape, cos, sin, caches[0].desc)
        smq.paged_norm_rope_kv(smq.paged_rows(q, outs[1], k, v), batch[1].desc, shape, cos, sin, caches[1].desc)
        same(outs[1].download(np.float32), outs[0].download(np.float32))
        for a, b in zip(caches[0].download(), caches[1].download()):
            same(a, b)
    smq.numeric_check()


@pytest.mark.parametrize("kv_type", [F32, F16, Q8])
def test_norm_of_special_rows(kv_type):
    """Zeros with and without eps, infinities, depths outside the tables: stored as documented, flagged; neighbours as ever."""
    hd, n = 64, 6
    cache = Cache(kv_type, 1, hd, 16, [40]).upload()
    batch = Batch(cache, [n])
    shape = smq.attn_shape(1, 1, hd, 32, 0, 48)
    cos, sin = tables(48, 32)
    w = (1 + 0.2 * synth.normal(31, hd)).astype(np.float32)
    k, v = (synth.normal(32 + i, n * hd).reshape(n, 1, hd) for i in range(2))
    k[2] = 0.0
    depth = np.array([0, 1, 1, 2, 3, 13], np.int32)
    out = dev(np.full((n, hd), 7.0, np.float32))

    def store(eps=1e-6):
        r = smq.paged_rows(dev(k), out, dev(k), dev(v), dev(w), dev(w), eps, dev(depth))
        smq.paged_norm_rope_kv(r, batch.desc, shape, dev(cos), dev(sin), cache.desc)
        return flagged()

    def check(eps, bad=()):
        y = ref.normed(k, w, eps)
        fine = [i for i in range(n) if i not in bad]
        turn = 34 + depth[fine]
        y[fine] = rotate(y[fine], cos[turn], sin[turn], 32)
        cache.put(0, 34 + np.array(fine), y[fine], v[fine])
        if bad:  # values are stored whatever the depth
            before = [x.copy() for x in (cache.k, cache.ks) if x is not None]
            cache.put(0, 34 + np.array(bad), y[list(bad)], v[list(bad)])
            cache.k[...] = before[0]
            if kv_type == Q8:
                cache.ks[...] = before[1]
        got = out.download(np.float32).reshape(n, 1, hd)
        nan = np.isnan(y)
        assert np.array_equal(np.isnan(got[fine]), nan[fine])
        same(np.where(nan[fine], 0, got[fine]), np.where(nan[fine], 0, y[fine]))
        for a, b in zip(cache.download(), (cache.k, cache.v, cache.ks, cache.vs)):
            nan = np.isnan(b.astype(np.float32))
            assert np.array_equal(np.isnan(a.astype(np.float32)), nan)
            same(np.where(nan, 0, a).astype(b.dtype), np.where(nan, 0, b).astype(b.dtype))

    assert not store()
    check(1e-6)
    assert store(0.0)  # 0 / 0
    check(0.0)
    k[2] = 1.0
    k[4, 0, 7] = np.inf
    assert store()
    check(1e-6)
    k[4, 0, 7] = 1.0
    for d in (14, -35, 2 ** 31 - 1, -2 ** 31):  # 48 or past it, below 0
        depth[3] = d
        out.upload(np.full((n, hd), 7.0, np.float32))
        assert store()
        assert (out.download(np.float32).reshape(n, hd)[3] == 7.0).all()
        check(1e-6, bad=(3,))


# ---- trees -------------------------------------------------------------------

class Trees:
    """Random trees (or masks of no shape, rows of nothing among them) for a batch, on the device."""

    def __init__(self, batch, seed=3, kind="tree", stride=None, fill=0):
        rng = np.random.default_rng(seed)
        self.parents = [ref.random_tree(rng, n) for n in batch.new]
        both = [ref.masks(p) for p in self.parents]
        self.seen = [b[1] for b in both]
        if kind == "any":
            self.seen = [rng.random(x.shape) < 0.4 for x in self.seen]
            for x in self.seen:
                x[rng.random(x.shape[0]) < 0.3] = False
        self.stride = stride or max(1, max(-(-n // 32) for n in batch.new))
        self.depth = np.full(batch.tokens, fill, np.int32)
        self.words = np.full((batch.tokens, self.stride), fill, np.uint32)
        self.parent = np.full(batch.tokens, 77, np.int32)
        for s, n in enumerate(batch.new):
            r = slice(batch.begin[s], batch.begin[s + 1])
            self.depth[r], self.parent[r] = both[s][0], self.parents[s]
            self.words[r] = ref.words(self.seen[s], self.stride)

    def upload(self):
        self.db, self.wb, self.pb = dev(self.depth), dev(self.words), dev(self.parent)
        return self


@pytest.mark.parametrize("new,stride", [([1], 1), ([13, 0, 32, 33], 2), ([64, 1, 5], 3), ([200, 31], 128), ([4096], 128)])
def test_draft_masks(new, stride):
    cache = Cache(F16, 1, 16, 256, [n + 5 for n in new], spare=0).upload()
    batch = Batch(cache, new, padding=3)
    t = Trees(batch, stride=stride, fill=9).upload()
    d, m = dev(np.full(batch.tokens, 9, np.int32)), dev(np.full((batch.tokens, stride), 9, np.uint32))
    smq.draft_masks(t.pb, batch.desc, d, m, stride)
    same(d.download(np.int32), t.depth)
    same(m.download(np.uint32).reshape(t.words.shape), t.words)
    smq.numeric_check()


def test_draft_masks_of_a_chain_and_bad_parents():
    cache = Cache(F16, 1, 16, 256, [100, 40, 9, 3]).upload()
    batch = Batch(cache, [90, 40, 9, 0])
    parent = np.concatenate([np.arange(-1, 89), np.full(40, -1), [-5, 0, 2, 7, 2 ** 31 - 1, -2 ** 31, 5, 7, 7]]).astype(np.int32)
    d, m = dev(np.full(139, 9, np.int32)), dev(np.full((139, 3), 9, np.uint32))
    smq.draft_masks(dev(parent), batch.desc, d, m, 3)
    assert flagged()  # parents 2, 7 and 2^31 - 1 of tokens 2, 3 and 4
    trees = [list(range(-1, 89)), [-1] * 40, [-1, 0, -1, -1, -1, -1, 5, -1, 7]]
    want = [ref.masks(t) for t in trees]
    same(d.download(np.int32), np.concatenate([w[0] for w in want]))
    same(m.download(np.uint32).reshape(139, 3), np.concatenate([ref.words(w[1], 3) for w in want]))
    # more new tokens than the words' bits: left as they are, the others done
    d, m = dev(np.full(139, 9, np.int32)), dev(np.full((139, 2), 9, np.uint32))
    parent[130:] = -1
    smq.draft_masks(dev(parent), batch.desc, d, m, 2)
    assert flagged()
    got = m.download(np.uint32).reshape(139, 2)
    assert (got[:90] == 9).all() and (d.download(np.int32)[:90] == 9).all()
    same(got[90:130], ref.words(want[1][1], 2))


def tree_attend(cache, batch, q, heads, trees, window=0, sinks=0, context=None, split=True, fill=9.0, depth=True):
    shape = smq.attn_shape(heads, cache.kv, cache.hd, cache.hd // 2, window, context or int(max(batch.length.max(), 1)))
    qb, att = dev(q), dev(np.full(q.shape, fill, np.float32))
    need = smq.paged_tree_attention_workspace(batch.desc, shape)
    ws = smq.DeviceBuffer(need) if split and need else None
    if ws:
        ws.fill(0xFF)
    smq.paged_tree_attention(qb, att, batch.desc, shape, sinks, trees.db if depth else None, trees.wb, trees.stride, cache.desc,
                             ws)
    return att.download(np.float32).reshape(q.shape)


TREES = [  # heads, kv, hd, page, lengths, new, window, sinks
    (14, 2, 64, 32, [1], [1], 0, 0),                                  # one token, no context
    (14, 2, 64, 64, [131, 1, 64, 65, 33], [8, 1, 1, 16, 33], 0, 0),   # no context in the last
    (12, 2, 128, 16, [15, 16, 17, 200], [3, 16, 1, 40], 0, 0),
    (32, 4, 64, 128, [1030], [13], 100, 4),
    (8, 8, 96, 256, [70, 300], [70, 33], 20, 3),                      # windows that end among the new tokens
    (16, 2, 80, 64, [150, 90], [37, 90], 0, 0),
    (9, 3, 64, 32, [100, 37], [64, 0], 1, 0),                         # no context seen
    (4, 4, 16, 16, [50], [31], 7, 50),
    (17, 1, 32, 64, [129], [5], 64, 1),
    (2, 1, 256, 64, [400], [20], 0, 0),
    (6, 2, 112, 32, [95], [64], 33, 2),
    (40, 1, 48, 32, [77, 35], [9, 35], 0, 0),
    (8, 2, 64, 64, [300, 200], [130, 97], 150, 9),
]


@pytest.mark.parametrize("kind", ["tree", "any"])
@pytest.mark.parametrize("kv_type", [F32, F16, Q8])
@pytest.mark.parametrize("heads,kv,hd,page,lengths,new,window,sinks", TREES)
def test_tree_attention(kv_type, heads, kv, hd, page, lengths, new, window, sinks, kind):
    say("tree attention", TYPES[kv_type], heads, kv, hd, page, lengths, new, window, sinks, kind)
    cache = Cache(kv_type, kv, hd, page, lengths, stale="nan")
    for s, (m, n) in enumerate(zip(lengths, new)):  # context that no row sees is poisoned too
        low = m - n + 1 - window if window and n else 0
        if low > sinks:
            cache.spoil_positions(s, np.arange(min(sinks, low), min(low, m - n)))
    batch = Batch(cache.upload(), new, padding=2)
    trees = Trees(batch, kind=kind)
    if kind == "any":  # new tokens that no row sees as well, and bits behind the last token
        for s, (m, n) in enumerate(zip(lengths, new)):
            unseen = np.nonzero(~trees.seen[s].any(0))[0]
            if len(unseen):
                cache.spoil_positions(s, m - n + unseen)
            for i in range(n):
                w = trees.words[batch.begin[s] + i].astype(np.uint64)
                bits = ref.words((np.arange(32 * trees.stride) >= n)[None], trees.stride)[0]
                trees.words[batch.begin[s] + i] = w | bits
        cache.upload()
        batch = Batch(cache, new, padding=2)
    trees.upload()
    q = synth.normal(90, batch.tokens * heads * hd, 1.5).reshape(-1, heads, hd)
    want, tol = ref.tree64(cache, batch, q, heads, trees.depth, trees.seen, window, sinks)
    n = int(batch.begin[-1])
    first = tree_attend(cache, batch, q, heads, trees, window, sinks)
    close(first[:n], want[:n], tol[:n])
    assert (first[n:] == 9.0).all()
    smq.numeric_check()
    same(tree_attend(cache, batch, q, heads, trees, window, sinks), first)
    close(tree_attend(cache, batch, q, heads, trees, window, sinks, split=False)[:n], want[:n], tol[:n], "without a workspace")
    close(tree_attend(cache, batch, q, heads, trees, window, sinks, context=9000)[:n], want[:n], tol[:n], "wide context")
    if not window:
        close(tree_attend(cache, batch, q, heads, trees, depth=False)[:n], want[:n], tol[:n], "without depths")
    smq.numeric_check()


@pytest.mark.parametrize("kv_type", [F32, F16, Q8])
@pytest.mark.parametrize("lengths,new", [([5000, 3001, 64, 4097], [7, 1, 5, 12]), ([4500, 700], [30, 130])])
def test_tree_attention_long(kv_type, lengths, new):
    """Sequences that are split over workgroups, with and without room for it."""
    heads, kv, hd = 8, 2, 64
    cache = Cache(kv_type, kv, hd, 64, lengths, stale="nan").upload()
    batch = Batch(cache, new)
    trees = Trees(batch).upload()
    q = synth.normal(91, batch.tokens * heads * hd, 1.5).reshape(-1, heads, hd)
    want, tol = ref.tree64(cache, batch, q, heads, trees.depth, trees.seen)
    close(tree_attend(cache, batch, q, heads, trees), want, tol)
    close(tree_attend(cache, batch, q, heads, trees, split=False), want, tol)
    shape = smq.attn_shape(heads, kv, hd, 32, 0, 5000)
    need = smq.paged_tree_attention_workspace(batch.desc, shape)
    for part in (need // 2, need // 3, 64):
        ws, att, qb = smq.DeviceBuffer(max(part, 64) + 64), dev(np.zeros_like(q)), dev(q)
        ws.upload(np.full(ws.nbytes, 0xAB, np.uint8))
        smq.paged_tree_attention(qb, att, batch.desc, shape, 0, trees.db, trees.wb, trees.stride, cache.desc, ws,
                                 part // 16 * 16)
        close(att.download(np.float32).reshape(q.shape), want, tol, f"{part} bytes")
        assert (ws.download(np.uint8)[part // 16 * 16:] == 0xAB).all()
    smq.numeric_check()


@pytest.mark.parametrize("kv_type", [F32, F16, Q8])
def test_tree_attention_of_many(kv_type):
    """More sequences than a wave has lanes, cut into pieces; then so many tiles that none is."""
    heads, kv, hd = 2, 1, 64
    lengths = [1500, 4, 33] + [1300 + 3 * s for s in range(66)]
    cache = Cache(kv_type, kv, hd, 64, lengths, stale="nan").upload()
    batch = Batch(cache, [4, 0] + [1 + s % 5 for s in range(67)])
    trees = Trees(batch).upload()
    q = synth.normal(98, batch.tokens * heads * hd, 1.5).reshape(-1, heads, hd)
    want, tol = ref.tree64(cache, batch, q, heads, trees.depth, trees.seen)
    close(tree_attend(cache, batch, q, heads, trees), want, tol)
    heads, kv, hd = 16, 8, 128
    lengths = [64 + s % 7 for s in range(66)]
    cache = Cache(kv_type, kv, hd, 32, lengths, stale="nan").upload()
    batch = Batch(cache, [64 - s % 5 for s in range(66)])
    trees = Trees(batch, kind="any").upload()
    q = synth.normal(99, batch.tokens * heads * hd, 1.5).reshape(-1, heads, hd)
    want, tol = ref.tree64(cache, batch, q, heads, trees.depth, trees.seen)
    close(tree_attend(cache, batch, q, heads, trees), want, tol)
    smq.numeric_check()


@pytest.mark.parametrize("kv_type", [F32, F16, Q8])
@pytest.mark.parametrize("heads,hd,page,window,sinks", [(6, 128, 64, 0, 0), (12, 96, 16, 0, 0), (6, 64, 32, 0, 0), (6, 128, 16, 900, 5),
                                                       (12, 128, 16, 2500, 5)])
def test_tree_attention_of_ragged_drafts(kv_type, heads, hd, page, window, sinks):
    """Tiles that waves own, cut into pieces, with sequences of a token or two between those of many: last tiles of few rows."""
    kv = 1
    new = [40, 1, 2, 33, 16, 0, 24, 3, 40, 1, 17, 30]
    cache = Cache(kv_type, kv, hd, page, [3001 - 97 * s for s in range(12)], stale="nan").upload()
    batch = Batch(cache, new, padding=1)
    trees = Trees(batch).upload()
    q = synth.normal(97, batch.tokens * heads * hd, 1.5).reshape(-1, heads, hd)
    want, tol = ref.tree64(cache, batch, q, heads, trees.depth, trees.seen, window, sinks)
    n = int(batch.begin[-1])
    got = tree_attend(cache, batch, q, heads, trees, window, sinks)
    close(got[:n], want[:n], tol[:n])
    assert (got[n:] == 9.0).all()
    same(tree_attend(cache, batch, q, heads, trees, window, sinks), got)
    close(tree_attend(cache, batch, q, heads, trees, window, sinks, split=False)[:n], want[:n], tol[:n])
    smq.numeric_check()


@pytest.mark.parametrize("kv_type", [F32, F16, Q8])
@pytest.mark.parametrize("length,new,page,kind", [(1107, 1100, 16, "tree"), (640, 640, 64, "any")])
def test_tree_attention_of_many_drafts(kv_type, length, new, page, kind):
    """Masks of many words, which steps of 32 positions meet anywhere; a context shorter than a step, and none."""
    heads, kv, hd = 2, 1, 48
    cache = Cache(kv_type, kv, hd, page, [length, 40], stale="nan").upload()
    batch = Batch(cache, [new, 40])
    trees = Trees(batch, kind=kind).upload()
    q = synth.normal(96, batch.tokens * heads * hd, 1.5).reshape(-1, heads, hd)
    want, tol = ref.tree64(cache, batch, q, heads, trees.depth, trees.seen)
    close(tree_attend(cache, batch, q, heads, trees), want, tol)
    close(tree_attend(cache, batch, q, heads, trees, split=False), want, tol)
    smq.numeric_check()


def test_tree_attention_of_a_causal_mask():
    """A chain is causal: smq_paged_attention's results, within both bounds; with its window, whose positions are the same."""
    heads, kv, hd = 8, 2, 64
    cache = Cache(F16, kv, hd, 32, [300, 90], stale="nan").upload()
    batch = Batch(cache, [40, 90])
    trees = Trees(batch)
    trees.seen = [np.tril(np.ones((n, n), bool)) for n in batch.new]
    trees.depth = np.concatenate([np.arange(n) for n in batch.new]).astype(np.int32)
    trees.words = np.concatenate([ref.words(x, trees.stride) for x in trees.seen])
    trees.upload()
    q = synth.normal(92, batch.tokens * heads * hd, 1.5).reshape(-1, heads, hd)
    for window, sinks in ((0, 0), (2 ** 32 - 1, 2 ** 32 - 1)):
        _, tol = ref.tree64(cache, batch, q, heads, trees.depth, trees.seen)
        got = tree_attend(cache, batch, q, heads, trees, window, sinks)
        shape = smq.attn_shape(heads, kv, hd, 32, window, 300)
        att = smq.DeviceBuffer(q.nbytes)
        smq.paged_attention(dev(q), att, batch.desc, shape, sinks, cache.desc)
        close(got, att.download(np.float32).reshape(q.shape), 2 * tol)
    smq.numeric_check()


@pytest.mark.parametrize("kv_type", [F32, F16, Q8])
@pytest.mark.parametrize("window,sinks", [(16, 4), (1, 0), (20, 70)])
def test_tree_attention_of_chains_deeper_than_the_window(kv_type, window, sinks):
    """A window does not clear the mask's bits: where those of the ancestors that it leaves behind are cleared, but for sinks, a
    chain's attention is smq_paged_attention's with that window."""
    heads, kv, hd = 8, 2, 64
    cache = Cache(kv_type, kv, hd, 32, [300, 90, 45]).upload()
    batch = Batch(cache, [40, 90, 45])
    trees = Trees(batch)
    trees.depth = np.concatenate([np.arange(n) for n in batch.new]).astype(np.int32)
    chain = [np.tril(np.ones((n, n), bool)) for n in batch.new]
    q = synth.normal(93, batch.tokens * heads * hd, 1.5).reshape(-1, heads, hd)
    causal, causal_tol = attend64(cache, batch, q, heads, window, sinks)
    for cleared in (True, False):
        trees.seen = [x & ((np.subtract.outer(np.arange(n), np.arange(n)) < window) | (m - n + np.arange(n) < sinks)) if cleared else x
                      for x, n, m in zip(chain, batch.new, cache.lengths)]
        trees.words = np.concatenate([ref.words(x, trees.stride) for x in trees.seen])
        got = tree_attend(cache, batch, q, heads, trees.upload(), window, sinks)
        want, tol = ref.tree64(cache, batch, q, heads, trees.depth, trees.seen, window, sinks)
        close(got, want, tol)
        if cleared:
            close(got, causal, causal_tol)
    smq.numeric_check()


@pytest.mark.parametrize("kv_type", [F32, F16, Q8])
def test_tree_rows_that_are_refused_on_the_device(kv_type):
    """Depths outside, sequences of more tokens than the mask, rows without a place, pages that are none: flagged, 0, the
    neighbours as ever."""
    heads, kv, hd = 4, 2, 64
    cache = Cache(kv_type, kv, hd, 32, [80, 70, 40], stale="nan").upload()
    batch = Batch(cache, [10, 40, 3], padding=1)
    trees = Trees(batch)
    q = synth.normal(93, batch.tokens * heads * hd, 1.5).reshape(-1, heads, hd)
    want, tol = ref.tree64(cache, batch, q, heads, trees.depth, trees.seen)
    last = int(batch.begin[-1])

    def check(zero, **kw):
        got = tree_attend(cache, batch, q, heads, trees.upload(), **kw)
        assert flagged() == bool(len(zero))
        w, t = want.copy(), tol.copy()
        w[zero], t[zero] = 0, 0
        close(got[:last], w[:last], t[:last])
        assert (got[last:] == 9.0).all()

    check([])
    keep = trees.depth.copy()
    for d in (-1, 10, 2 ** 31 - 1, -2 ** 31):  # 70 + 10 is the context
        trees.depth[3] = d
        check([3], window=1000)
        check([3], window=1000, split=False)
        check([])  # without a window depths are not read
    trees.depth = keep
    trees.words, trees.stride = trees.words[:, :1].copy(), 1
    check(list(range(10, 50)))
    # a position past the table
    trees = Trees(batch)
    batch.lb.upload(np.array([80, 97, 40], np.int32))
    got = tree_attend(cache, batch, q, heads, trees.upload(), context=200)
    assert flagged()
    close(got[:10], want[:10], tol[:10])
    close(got[50:last], want[50:last], tol[50:last])
    assert (got[10 + 39] == 0).all()  # position 96 of 3 pages of 32
    batch.lb.upload(batch.length)
    # a page that the context needs, and none beyond
    table = cache.table.copy()
    table[1, 0] = cache.pages
    cache.tb.upload(table)
    got = tree_attend(cache, batch, q, heads, trees)
    assert flagged()
    close(got[:10], want[:10], tol[:10])
    cache.tb.upload(cache.table)
    # begins that do not ascend: flagged, in range
    batch.bb.upload(np.array([0, 60, 50, 53], np.int32))
    tree_attend(cache, batch, q, heads, trees)
    assert flagged()


@pytest.mark.parametrize("kv_type", [F32, F16, Q8])
@pytest.mark.parametrize("page", [16, 64])
def test_tree_of_more_tokens_than_positions_without_pages(kv_type, page):
    """New tokens that begin before position 0, and no page for those that have a place: nothing is seen, and the other
    sequence is as ever."""
    heads, kv, hd = 4, 2, 64
    cache = Cache(kv_type, kv, hd, page, [64, 40]).upload()
    table = cache.table.copy()
    for new in (60, 20):  # owned and shared tiles
        batch = Batch(cache, [new, 7], lengths=[12, 40])
        trees = Trees(batch)
        q = synth.normal(95, batch.tokens * heads * hd, 1.5).reshape(-1, heads, hd)
        first = Batch(cache, [0, 7], lengths=[12, 40])
        want, tol = ref.tree64(cache, first, q[new:], heads, trees.depth[new:], [np.zeros((0, 0), bool), trees.seen[1]])
        trees.words[:new] = 0xFFFFFFFF
        table[0] = -1
        cache.tb.upload(table)
        got = tree_attend(cache, batch, q, heads, trees.upload(), context=64)
        assert flagged()
        assert (got[:new] == 0).all()
        close(got[new:], want, tol)


@pytest.mark.parametrize("kv_type", [F32, F16, Q8])
@pytest.mark.parametrize("page,length,new,limit", [(32, 44, 12, 40), (64, 200, 90, 150), (16, 60, 30, 48)])
def test_tree_tokens_without_a_place_are_not_seen(kv_type, page, length, new, limit):
    """New tokens past the context, or past a table whose last page ends inside a step: no row sees them, whatever its mask and
    whatever their slots hold."""
    heads, kv, hd = 4, 2, 64
    cache = Cache(kv_type, kv, hd, page, [length, 20])
    cache.spoil_positions(0, np.arange(limit, length))
    cache.upload()
    batch = Batch(cache, [new, 7])
    short = Batch(cache, [new - (length - limit), 7], lengths=[limit, 20])
    trees, there = Trees(batch), np.concatenate([np.arange(short.new[0]), np.arange(new, new + 7)])
    trees.words[:new] = 0xFFFFFFFF
    q = synth.normal(96, batch.tokens * heads * hd, 1.5).reshape(-1, heads, hd)
    want, tol = ref.tree64(cache, short, q[there], heads, trees.depth[there], [np.ones((short.new[0],) * 2, bool), trees.seen[1]])
    if page == 16:  # the table's last page is the third
        cache.table = np.ascontiguousarray(cache.table[:, :3])
        cache.tb, cache.stride = dev(cache.table), 3
        batch = Batch(cache, [new, 7])
    got = tree_attend(cache, batch, q, heads, trees.upload(), context=limit if page != 16 else 64)
    assert flagged()
    close(got[there], want, tol)
    assert (got[short.new[0]:new] == 0).all()


@pytest.mark.parametrize("kv_type", [F32, F16, Q8])
def test_tree_values_that_are_not_finite_stay_where_they_are_seen(kv_type):
    """A drafted token's NaN value reaches its descendants and nobody else."""
    heads, kv, hd = 4, 2, 64
    for new in ([12], [70]):  # shared and owned tiles
        cache = Cache(kv_type, kv, hd, 32, [150], stale="nan")
        batch = Batch(cache.upload(), new)
        trees = Trees(batch).upload()
        t = new[0] // 3
        q = synth.normal(94, batch.tokens * heads * hd, 1.5).reshape(-1, heads, hd)
        want, tol = ref.tree64(cache, batch, q, heads, trees.depth, trees.seen)
        cache.spoil_positions(0, np.array([150 - new[0] + t]))
        batch = Batch(cache.upload(), new)
        got = tree_attend(cache, batch, q, heads, trees)
        blind = ~trees.seen[0][:, t]
        close(got[blind], want[blind], tol[blind])


# ---- pages --------------------------------------------------------------------

class Forked:
    """Tables with shared pages and other holders, and what a fork makes of them."""

    def __init__(self, rng, groups, beams, lengths, page, spare=10, held_more=0, stride=None):
        self.page, rows = page, groups * beams
        self.length = np.repeat(np.asarray(lengths), beams)
        need = -(-self.length // page) + held_more
        shared = np.repeat([int(rng.integers(0, n // page + 1)) if beams > 1 else 0 for n in lengths], beams)
        self.stride = stride or int(need.max()) + 2
        total = int(sum(need - shared) + sum(shared[::beams]))
        self.pages = total + spare
        order, at = rng.permutation(self.pages).astype(np.int32), 0
        self.table = np.full((rows, self.stride), -1, np.int32)
        self.refs = np.zeros(self.pages, np.int32)
        for r in range(rows):
            if r % beams == 0:
                common = order[at:at + shared[r]]
                at += shared[r]
                self.refs[common] += rng.integers(0, 2)
            self.table[r, :shared[r]] = common
            self.table[r, shared[r]:need[r]] = order[at:at + need[r] - shared[r]]
            at += need[r] - shared[r]
        self.held = need.astype(np.int32)
        self.refs += np.bincount(self.table[self.table >= 0], minlength=self.pages).astype(np.int32)

    def call(self, parent, keep, room, workspace_fill=0xFF):
        rows = len(parent)
        bufs = [dev(np.ascontiguousarray(x, np.int32)) if len(x) else smq.DeviceBuffer(4)
                for x in (self.table, self.held, self.refs, parent, keep, room)]
        outs = [smq.DeviceBuffer(max(4, 4 * n)) for n in (rows * self.stride, rows, self.pages, rows * 3, 1)]
        for o in outs:
            o.fill(0x5A)
        f = smq.page_fork(bufs[0], bufs[1], bufs[2], self.table.shape[0], rows, self.stride, self.page, self.pages, *bufs[3:],
                          *outs)
        ws = smq.DeviceBuffer(smq.paged_fork_workspace(f))
        ws.fill(workspace_fill)
        smq.paged_fork(f, ws)
        got = [o.download(np.int32) for o in outs]
        for b, x in zip(bufs, (self.table, self.held, self.refs)):
            if len(x):
                same(b.download(np.int32).reshape(x.shape), x)
        return got[0][:rows * self.stride].reshape(rows, self.stride), got[1][:rows], got[2], got[3][:3 * rows].reshape(rows, 3), got[4][0]

    def check(self, parent, keep, room):
        got = self.call(parent, keep, room)
        want = ref.fork(self.table, self.held, self.refs, parent, keep, room, self.page)
        for g, w in zip(got, want):
            same(g, np.asarray(w))
        return got


FORKS = [  # groups, beams, longest, page, spare
    (1, 1, 1, 16, 3), (1, 4, 100, 16, 20), (3, 8, 300, 32, 60), (8, 1, 700, 64, 300), (40, 5, 200, 16, 500), (64, 1, 4000, 16, 20000),
    (2, 4, 90, 256, 40000), (300, 1, 2500, 16, 5000),
]


@pytest.mark.parametrize("groups,beams,longest,page,spare", FORKS)
def test_fork(groups, beams, longest, page, spare):
    say("paged fork", groups, beams, longest, page, spare)
    rng = np.random.default_rng(groups + beams)
    lengths = [longest] + [int(rng.integers(1, longest + 1)) for _ in range(groups - 1)]
    f = Forked(rng, groups, beams, lengths, page, spare)
    rows = groups * beams
    most = f.stride * page
    # the beams go on; one more token
    parent = [g * beams + int(rng.integers(0, beams)) for g in range(groups) for _ in range(beams)]
    keep = [int(f.length[p]) for p in parent]
    f.check(parent, keep, [k + 1 for k in keep])
    # nothing happens
    f.check(list(range(rows)), list(f.length), list(f.length))
    # rows end, begin, are cut and extended, in another order and number
    n = max(1, rows // 2)
    parent = [int(rng.integers(-1, rows)) for _ in range(n)]
    keep = [int(rng.integers(0, f.length[p] + 1)) if p >= 0 else 0 for p in parent]
    room = [min(most, k + int(rng.integers(0, 3 * page))) for k in keep]
    f.check(parent, keep, room)
    # everything ends
    f.check([-1] * rows, [0] * rows, [0] * rows)
    # one row becomes all
    f.check([rows - 1] * rows, [int(f.length[rows - 1])] * rows, [int(f.length[rows - 1])] * rows)
    assert not flagged()


def test_fork_of_pages_in_part_and_whole():
    """A page that one row takes whole and others in part: all of those copy. Held beside the tables: every one copies."""
    rng = np.random.default_rng(2)
    f = Forked(rng, 1, 1, [64], 16, 30)
    got = f.check([0, 0, 0, 0], [64, 40, 40, 16], [65, 41, 48, 16])
    assert (got[3][:, 2] == [0, 8, 8, 0]).all()
    got = f.check([0, 0, 0], [40, 40, 33], [41, 41, 34])
    assert (got[3][:, 2] == [0, 8, 1]).all()
    f.refs[f.table[0, 2]] += 1
    got = f.check([0, 0, 0], [40, 40, 33], [41, 41, 34])
    assert (got[3][:, 2] == [8, 8, 1]).all()
    assert not flagged()


def test_fork_from_nothing_and_to_nothing():
    f = Forked(np.random.default_rng(3), 1, 1, [64], 16, 30)
    full = f.refs.copy()
    got = f.check([], [], [])
    assert (got[2][f.table[0, :4]] == 0).all()
    f.table, f.held, f.refs = np.zeros((0, f.stride), np.int32), np.zeros(0, np.int32), 0 * full
    got = f.check([-1, -1], [0, 0], [20, 33])
    assert list(got[0][0, :3]) == [0, 1, -1] and list(got[0][1, :4]) == [2, 3, 4, -1]
    assert not flagged()


@pytest.mark.parametrize("big", [False, True])
def test_fork_without_enough_pages(big):
    """Entries past the free pages are -1, what is missing comes back, the flag is raised; the old arrays serve again."""
    rng = np.random.default_rng(4)
    f = Forked(rng, 4, 1, [64, 50, 33, 20], 16, 40000 if big else 3, stride=16)
    if big:
        f.refs[f.refs == 0] = 1  # held elsewhere
        f.refs[[5, 39999, 17000]] = 0 * f.refs[[5, 39999, 17000]] + (np.isin([5, 39999, 17000], f.table))
    parent, keep = [0, 0, 1, 3], [64, 50, 50, 20]
    got = f.check(parent, keep, [100, 100, 100, 30])
    assert got[4] < 0 and flagged()
    f.check(parent, keep, [65, 50, 50, 20])
    assert not flagged()


@pytest.mark.parametrize("rows", [2100, 4200])
def test_fork_that_needs_more_pages_than_32_bits_count(rows):
    """2^31 and 2^32 entries without a page: as many as are free go to the first row, none is given twice."""
    stride, page, pages = 1 << 20, 16, 9000
    say("paged fork", rows, "rows of", stride)
    top = stride * page
    held, refs = dev(np.zeros(1, np.int32)), np.zeros(pages, np.int32)
    refs[::3] = 1  # a store of prompts
    bufs = [dev(np.full(stride, -1, np.int32)), held, dev(refs)] + [
        dev(np.full(rows, x, np.int32)) for x in (-1, 0, top)]
    outs = [smq.DeviceBuffer(4 * n) for n in (rows * stride, rows, pages, rows * 3, 1)]
    f = smq.page_fork(*bufs[:3], 1, rows, stride, page, pages, *bufs[3:], *outs)
    smq.paged_fork(f, smq.DeviceBuffer(smq.paged_fork_workspace(f)))
    assert flagged()
    free = np.nonzero(refs == 0)[0]
    assert outs[4].download(np.int32)[0] == max(len(free) - rows * stride, -2 ** 31)
    same(outs[2].download(np.int32), np.ones(pages, np.int32))
    same(outs[1].download(np.int32), np.full(rows, stride, np.int32))
    none = np.full(stride, -1, np.int32)
    for r in (0, 1, 2047, 2048, 2049, 4095, 4096, 4097, rows - 1):
        if r < rows:
            want = none.copy()
            if r == 0:
                want[:len(free)] = free
            same(outs[0].download(np.int32, stride, 4 * r * stride), want)
    for b in outs:
        b.free()


def test_fork_of_what_is_not_valid():
    """Flagged and cut; every index stays in range, and the neighbours are as ever."""
    f = Forked(np.random.default_rng(5), 3, 1, [64, 50, 33], 16, 200, stride=8)
    top = 2 ** 31 - 1
    cut = [([0, 7, 2], [64, 10, 33], [70, 20, 40], [0, -1, 2], [64, 0, 33], [70, 20, 40]),
           ([0, -2, 2], [64, 10, 33], [70, 20, 40], [0, -1, 2], [64, 0, 33], [70, 20, 40]),
           ([0, 1, 2], [64, 70, 33], [70, 80, 40], [0, 1, 2], [64, 64, 33], [70, 80, 40]),
           ([0, 1, 2], [64, top, 33], [70, top, 40], [0, 1, 2], [64, 64, 33], [70, 128, 40]),
           ([0, 1, 2], [-5, 50, 33], [70, 20, 40], [0, 1, 2], [0, 50, 33], [70, 50, 40]),
           ([0, 1, 2], [64, 50, -top - 1], [70, 50, -top - 1], [0, 1, 2], [64, 50, 0], [70, 50, 0])]
    for parent, keep, room, p, k, r in cut:
        got = f.call(parent, keep, room)
        assert flagged()
        for g, w in zip(got, ref.fork(f.table, f.held, f.refs, p, k, r, 16)):
            same(g, np.asarray(w))
    for held in (-1, 9, top):
        keep = f.held[1]
        f.held[1] = held
        f.call([0, 1, 2], [64, 0, 33], [64, 16, 33])
        assert flagged()
        f.held[1] = keep
    f.table[1, 1] = f.pages  # no page: stays none
    got = f.call([0, 1, 2], [64, 50, 33], [64, 50, 33])
    assert flagged() and got[0][1, 1] == -1 and got[0][1, 0] == f.table[1, 0]
    f.table[1, 1] = 0
    f.refs[:] = 0  # fewer holders than entries
    f.call([0, 1, 2], [64, 50, 33], [64, 50, 33])
    assert flagged()


@pytest.mark.parametrize("kv_type,kv,hd,page,layers", [(F32, 2, 64, 16, 1), (F16, 3, 80, 64, 3), (Q8, 2, 96, 32, 2), (Q8, 1, 16, 256, 1),
                                                       (F16, 1, 256, 128, 1), (Q8, 1, 48, 16, 50)])
def test_copy(kv_type, kv, hd, page, layers):
    """The first positions of pages, nothing else; rows that are none skipped, bad ones flagged and skipped."""
    caches = [Cache(kv_type, kv, hd, page, [page * 8], seed=i + 1).upload() for i in range(layers)]
    counts = [1, page, page // 2 + 1, page - 1, 0, 3]
    copies = np.array([[i, 9 - i, n] for i, n in zip((0, 1, 2, 3, 4, 4), counts)], np.int32)
    copies[5] = -1, -1, 0
    shape = smq.attn_shape(kv * 2, kv, hd, 0, 0, 64)
    pools = smq.paged_pools([c.desc for c in caches])
    for c in caches:
        ref.copy(c, copies[:5])
    smq.paged_copy(dev(copies), 6, shape, pools)
    for c in caches:
        pool_same(c)
    assert not flagged()
    bad = np.array([[0, 10, 1], [-1, 5, 1], [0, 5, page + 1], [0, 5, -1], [2 ** 31 - 1, 5, 3], [3, 4, 7]], np.int32)
    for c in caches:
        ref.copy(c, bad[5:])
    smq.paged_copy(dev(bad), 6, shape, pools)
    assert flagged()
    for c in caches:
        pool_same(c)


PATHS = [  # type, kv, hd, page, lengths, new, layers
    (F32, 2, 64, 16, [40, 33, 20], [20, 33, 1], 1),
    (F16, 2, 80, 32, [100, 70, 64, 9], [64, 40, 1, 0], 3),
    (Q8, 3, 96, 64, [130, 200], [60, 150], 2),
    (Q8, 1, 16, 16, [90], [90], 50),
    (F16, 1, 256, 128, [300], [200], 1),
]


@pytest.mark.parametrize("kind", ["random", "dense", "all"])
@pytest.mark.parametrize("kv_type,kv,hd,page,lengths,new,layers", PATHS)
def test_compact(kv_type, kv, hd, page, lengths, new, layers, kind):
    """Paths of any length, those whose places are other tokens of the path among them, in every pool."""
    say("compact", TYPES[kv_type], kv, hd, page, lengths, new, layers, kind)
    rng = np.random.default_rng(6)
    caches = [Cache(kv_type, kv, hd, page, lengths, seed=4) for i in range(layers)]
    for i, c in enumerate(caches):  # one table, other contents
        for x, _ in ref.pool_parts(c):
            x[...] = np.roll(x, i, 0)
        c.upload()
    batch = Batch(caches[0], new)
    paths = [[] if not n else list(range(n)) if kind == "all" else
             sorted(rng.choice(n, min(n, rng.integers(1, 9) if kind == "random" else n * 3 // 4), replace=False)) for n in new]
    stride = max(map(len, paths)) + 2
    acc = np.full((len(new), stride), -7, np.int32)
    for s, p in enumerate(paths):
        acc[s, :len(p)] = p
        for c in caches:
            ref.compact(c, s, lengths[s] - new[s], p)
    out = smq.DeviceBuffer(4 * len(new))
    shape = smq.attn_shape(kv, kv, hd, 0, 0, max(lengths))
    smq.paged_compact(batch.desc, shape, dev(acc), stride, dev(np.array([len(p) for p in paths], np.int32)),
                      smq.paged_pools([c.desc for c in caches]), out)
    same(out.download(np.int32), np.array([m - n + len(p) for m, n, p in zip(lengths, new, paths)], np.int32))
    for c in caches:
        pool_same(c)
    assert not flagged()


@pytest.mark.parametrize("kv_type", [F32, F16, Q8])
def test_pools_named_again_count_once(kv_type):
    """Paths move, and pages are copied, once in a pool that is named several times, in one launch or two."""
    caches = [Cache(kv_type, 2, 64, 32, [100, 70], seed=4) for _ in range(3)]
    for i, c in enumerate(caches):
        for x, _ in ref.pool_parts(c):
            x[...] = np.roll(x, i, 0)
        c.upload()
    names = [0, 1, 0, 2, 2, 0] + [1] * 50 + [2, 0]
    pools = smq.paged_pools([caches[i].desc for i in names])
    batch = Batch(caches[0], [60, 50])
    paths = [list(range(1, 60, 2)), [1, 2, 3, 5, 8, 13, 21, 34, 49]]
    acc, out = np.zeros((2, 30), np.int32), smq.DeviceBuffer(8)
    for s, p in enumerate(paths):
        acc[s, :len(p)] = p
        for c in caches:
            ref.compact(c, s, (40, 20)[s], p)
    shape = smq.attn_shape(2, 2, 64, 0, 0, 100)
    smq.paged_compact(batch.desc, shape, dev(acc), 30, dev(np.array([30, 9], np.int32)), pools, out)
    assert list(out.download(np.int32)) == [70, 29]
    copies = np.array([[0, 5, 32], [1, 6, 17]], np.int32)
    for c in caches:
        ref.copy(c, copies)
    smq.paged_copy(dev(copies), 2, shape, pools)
    for c in caches:
        pool_same(c)
    assert not flagged()


def test_compact_of_what_is_not_valid():
    """Lists that do not ascend, leave the draft or are too long: the sequence stays, the others are done."""
    for path, count in (([3, 3], 2), ([4, 2], 2), ([0, 20], 2), ([-1, 2], 2), ([1, 2], 4), ([1, 2], -1), ([1, 2], 2 ** 31 - 1)):
        cache = Cache(F16, 2, 64, 32, [100, 70]).upload()
        batch = Batch(cache, [20, 20])
        acc = np.array([path + [9], [5, 7, 19]], np.int32)
        ref.compact(cache, 1, 50, [5, 7, 19])
        out = smq.DeviceBuffer(8)
        smq.paged_compact(batch.desc, smq.attn_shape(2, 2, 64, 0, 0, 100), dev(acc), 3, dev(np.array([count, 3], np.int32)),
                          smq.paged_pools([cache.desc]), out)
        assert flagged()
        assert list(out.download(np.int32)) == [100, 53]
        pool_same(cache)
    # a page that is none: those tokens stay
    cache = Cache(F16, 2, 64, 32, [100, 70]).upload()
    table = cache.table.copy()
    table[1, 2] = -1
    cache.tb.upload(table)
    ref.compact(cache, 1, 50, [5])
    smq.paged_compact(Batch(cache, [20, 20]).desc, smq.attn_shape(2, 2, 64, 0, 0, 100), dev(np.array([[0], [5]], np.int32)), 1,
                      dev(np.array([0, 1], np.int32)), smq.paged_pools([cache.desc]), out)
    assert not flagged()
    smq.paged_compact(Batch(cache, [20, 20]).desc, smq.attn_shape(2, 2, 64, 0, 0, 100), dev(np.array([[0, 0], [1, 19]], np.int32)), 2,
                      dev(np.array([0, 2], np.int32)), smq.paged_pools([cache.desc]), out)
    ref.compact(cache, 1, 50, [1])
    assert flagged()
    pool_same(cache)


# ---- beams ----------------------------------------------------------------------

def beam_call(logits, score, groups, beams, select, done=None, pad=0, eos=NONE, history=None, length=None, stride=None, shift=0):
    rows, vocab, n = groups * beams, logits.shape[1], groups * select
    stride = stride or vocab
    wide = np.full((rows, stride), 1e30, np.float32)
    wide[:, :vocab] = logits
    lb = smq.DeviceBuffer(wide.nbytes + 16)
    lb.upload(wide, 4 * shift)
    outs = [smq.DeviceBuffer(4 * n) for _ in range(3)] + [smq.DeviceBuffer(n)]
    kw = {}
    if history is not None:
        kw = dict(history=dev(history), history_out=smq.DeviceBuffer(4 * n * history.shape[1]), history_stride=history.shape[1],
                  length=dev(length), length_out=smq.DeviceBuffer(4 * n))
    b = smq.beam_step(lb.at(4 * shift), stride, groups, beams, vocab, select, dev(score), *outs[:3], done=None if done is None else dev(done),
                      pad=pad, eos=eos, done_out=outs[3], **kw)
    need = smq.beam_select_workspace(b)
    ws = smq.DeviceBuffer(need + 64)
    ws.fill(0xFF)
    smq.beam_select(b, ws, need)
    got = [outs[0].download(np.int32), outs[1].download(np.uint32), outs[2].download(np.float32), outs[3].download(np.uint8)]
    assert (ws.download(np.uint8)[need:] == 0xFF).all()
    if history is not None:
        got += [kw["history_out"].download(np.uint32).reshape(n, -1), kw["length_out"].download(np.int32)]
    return got


def beam_check(logits, score, groups, beams, select, **kw):
    """Ids and parents as in 64 bits, scores within half a step of the value and 2^-40 of what sums of 64 bits may be off."""
    got = beam_call(logits, score, groups, beams, select, **kw)
    want = ref.beam(logits, score, groups, beams, select, kw.get("done"), kw.get("pad", 0), kw.get("eos", NONE))
    same(got[0], want[0].astype(np.int32))
    same(got[1], want[1].astype(np.uint32))
    fine = want[0] >= 0
    assert (got[2][~fine] == -np.inf).all()
    assert (np.abs(got[2][fine] - want[2][fine]) <= np.abs(want[2][fine]) * 2.0 ** -24 + 2.0 ** -40).all()
    same(got[3], want[3].astype(np.uint8))
    return got


BEAMS = [  # groups, beams, select, vocab
    (1, 1, 1, 1), (1, 4, 8, 151936), (3, 8, 16, 5000), (2, 64, 64, 3001), (5, 3, 7, 999), (1, 2, 64, 40), (7, 1, 5, 2049),
    (1, 32, 64, 20000), (2, 2, 4, 300001), (40, 2, 2, 1500), (16, 8, 16, 4097),
]


@pytest.mark.parametrize("groups,beams,select,vocab", BEAMS)
def test_beam_select(groups, beams, select, vocab):
    say("beam", groups, beams, select, vocab)
    rng = np.random.default_rng(vocab + beams)
    rows = groups * beams
    logits = synth.normal(40, rows * vocab, 3.0).reshape(rows, vocab)
    score = (-20 + 2 * rng.standard_normal(rows)).astype(np.float32)
    beam_check(logits, score, groups, beams, select)
    beam_check(logits, score, groups, beams, select, stride=vocab + 3, shift=1)
    # masked ids, dead and finished rows, the end
    logits[rng.random(logits.shape) < 0.9] = -np.inf
    done = (rng.random(rows) < 0.3).astype(np.uint8)
    score[rng.random(rows) < 0.2] = -np.inf
    logits[rows // 2] = -np.inf
    n = 9
    history, length = rng.integers(0, vocab, (rows, n)).astype(np.uint32), rng.integers(0, n, rows).astype(np.int32)
    eos = int(np.argmax(logits[0]))
    got = beam_check(logits, score, groups, beams, select, done=done, pad=5, eos=eos, history=history, length=length)
    for parent, token, h, m in zip(got[0], got[1], got[4], got[5]):
        want = [] if parent < 0 else list(history[parent, :length[parent]]) + ([] if done[parent] else [token])
        assert m == len(want) and list(h) == want + [NONE] * (n - len(want))
    assert not flagged()


def test_beam_ties():
    """Equal logits: lower ids; equal values: lower rows; a zero is a zero whatever its sign."""
    logits = np.zeros((4, 5000), np.float32)
    logits[:, 1::2] = -0.0
    score = np.full(4, -1.0, np.float32)
    got = beam_check(logits, score, 1, 4, 64)
    assert (got[0] == 0).all() and list(got[1]) == list(range(64))
    logits = np.full((2, 100000), -3.0, np.float32)
    logits[:, [99999, 17, 2048, 2047, 60000]] = 2.0
    got = beam_check(logits, score[:2], 1, 2, 12)
    assert list(got[0]) == [0] * 5 + [1] * 5 + [0] * 2 and list(got[1]) == [17, 2047, 2048, 60000, 99999] * 2 + [0, 1]
    # one workgroup's ids descend by their place, so that each span's best are its last
    logits = np.tile(np.arange(70000, dtype=np.float32) / 7e4, (3, 1))
    beam_check(logits, score[:3], 1, 3, 64)
    beam_check(logits[:, ::-1].copy(), score[:3], 1, 3, 64)


def test_beam_of_what_is_not_finite():
    """NaN and +inf flag their row, which has no continuation; the other rows and groups go on."""
    base = synth.normal(41, 4 * 6000, 3.0).reshape(4, 6000)
    score = np.array([-1, -2, -3, -4], np.float32)
    for row, x in ((0, np.nan), (3, np.inf)):
        logits = base.copy()
        logits[row, 4500] = x
        dead = score.copy()
        dead[row] = -np.inf
        clean = base.copy()
        got = beam_call(logits, score, 2, 2, 6)
        assert flagged()
        want = ref.beam(clean, dead, 2, 2, 6)
        same(got[0], want[0].astype(np.int32))
        same(got[1], want[1].astype(np.uint32))
        # a row that is done is not looked at
        done = np.zeros(4, np.uint8)
        done[row] = 1
        beam_call(logits, score, 2, 2, 6, done=done)
        assert not flagged()
    for x in (np.nan, np.inf):
        bad = score.copy()
        bad[1] = x
        dead = score.copy()
        dead[1] = -np.inf
        for done in (None, np.array([0, 1, 0, 0], np.uint8)):
            got = beam_call(base, bad, 2, 2, 6, done=done)
            assert flagged()
            want = ref.beam(base, dead, 2, 2, 6, done)
            same(got[0], want[0].astype(np.int32))
            same(got[1], want[1].astype(np.uint32))
    # large and tiny logits
    logits = base * np.float32(1e36)
    beam_check(logits, score, 2, 2, 6)
    beam_check(base * np.float32(1e-42), score, 2, 2, 6)


@pytest.mark.parametrize("d", [-0.4326171875, -1.65625])
def test_beam_sums_are_within_their_bound(d):
    """A row whose sum of exponentials is mostly one term, at a distance d from the largest of its 256 ids, which is at d from the
    row's: where the exponential is furthest off. Each is within 1e-12 of its size, so that the sum's logarithm is within 1e-12;
    64-bit sums and logarithms of this size add less than 1e-14, and the result, near 0, half an f32 step."""
    vocab = 50000
    logits = np.full((1, vocab), 2 * d, np.float32)
    logits[0, ::256] = d
    logits[0, :256] = -np.inf
    logits[0, 0] = 0
    lse = np.log(np.exp(logits[0].astype(np.longdouble)).sum())
    score = np.array([lse], np.float32)
    got = beam_call(logits, score, 1, 1, 1)
    want = float(np.longdouble(score[0]) - lse)
    assert got[0][0] == 0 and got[1][0] == 0 and abs(want) < 1e-6
    assert abs(float(got[2][0]) - want) <= 1e-12 + 1e-14 + abs(want) * 2.0 ** -24
    assert not flagged()


def test_beam_histories_that_are_full():
    logits = synth.normal(42, 2 * 500, 3.0).reshape(2, 500)
    history = np.arange(20, dtype=np.uint32).reshape(2, 10)
    for length in ([10, 10], [11, 2 ** 31 - 1], [-1, -2 ** 31]):
        got = beam_call(logits, np.zeros(2, np.float32), 1, 2, 3, history=history, length=np.array(length, np.int32))
        assert flagged()
        for parent, token, h, m in zip(got[0], got[1], got[4], got[5]):
            want = list(history[parent]) if length[0] > 0 else [token] + [NONE] * 9
            assert list(h) == want and m == (10 if length[0] > 0 else 1)


# ---- together -----------------------------------------------------------------

@pytest.mark.parametrize("kv_type", [F32, F16, Q8])
def test_drafts_together(kv_type):
    """Drafting on a shared pool: trees stored, attended, an accepted path kept, the rest given back, new pages, for several
    steps. Another cache gets the accepted tokens one after another: its rows are the same bits, and causal attention over it
    gives the accepted tokens' results."""
    heads, kv, hd, page, context = 6, 2, 64, 16, 256
    rng = np.random.default_rng(8)
    lengths = np.array([70, 33, 16], np.int32)
    cache = Cache(kv_type, kv, hd, page, list(lengths), spare=60, stride=16).upload()
    plain = Cache(kv_type, kv, hd, page, [context - 16] * 3, spare=0, stride=16, stale="nan")
    for s, m in enumerate(lengths):
        for a, b in zip(ref.pool_parts(plain), ref.pool_parts(cache)):
            pg, sl = plain.slots(s, np.arange(m))
            cg, cl = cache.slots(s, np.arange(m))
            if a[1] == 2:
                a[0][pg, :, sl] = b[0][cg, :, cl]
            else:
                a[0][pg, :, :, sl] = b[0][cg, :, :, cl]
    plain.upload()
    shape = smq.attn_shape(heads, kv, hd, hd // 2, 0, context)
    cb, sb = (dev(x) for x in tables(context, hd // 2))
    w = [dev((1 + 0.2 * synth.normal(300 + i, hd)).astype(np.float32)) for i in range(2)]
    held = np.array([-(-m // page) for m in lengths], np.int32)
    refs = np.zeros(cache.pages, np.int32)
    for s in range(3):
        refs[cache.table[s, :held[s]]] += 1
    words = 1
    for step in range(4):
        new = [int(rng.integers(1, 20)), 12, 1 if step % 2 else 9]
        # room for the drafts: every row goes on
        grown = lengths + np.array(new, np.int32)
        bufs = [dev(x) for x in (cache.table, held, refs, np.arange(3, dtype=np.int32), lengths, grown)]
        outs = [smq.DeviceBuffer(4 * n) for n in (3 * 16, 3, cache.pages, 9, 1)]
        f = smq.page_fork(*bufs[:3], 3, 3, 16, page, cache.pages, *bufs[3:], *outs)
        smq.paged_fork(f, smq.DeviceBuffer(smq.paged_fork_workspace(f)))
        assert (outs[3].download(np.int32).reshape(3, 3)[:, 2] == 0).all()  # alone in its last page
        cache.table, held, refs = outs[0].download(np.int32).reshape(3, 16), outs[1].download(np.int32), outs[2].download(np.int32)
        assert (held == -(-grown // page)).all() and refs.sum() == held.sum() and refs.max() == 1
        cache.tb = outs[0]
        batch = Batch(cache, new, lengths=grown)
        n = batch.tokens
        trees = Trees(batch, seed=step, stride=words).upload()
        q, k, v = (synth.normal(310 + 3 * step + i, n * x * hd, 2.0).reshape(n, x, hd) for i, x in enumerate((heads, kv, kv)))
        d, m, rot, att, out = (smq.DeviceBuffer(x) for x in (4 * n, 4 * n * words, q.nbytes, q.nbytes, 12))
        smq.draft_masks(trees.pb, batch.desc, d, m, words)
        smq.paged_norm_rope_kv(smq.paged_rows(dev(q), rot, dev(k), dev(v), *w, 1e-6, d), batch.desc, shape, cb, sb, cache.desc)
        ws = smq.DeviceBuffer(max(16, smq.paged_tree_attention_workspace(batch.desc, shape)))
        smq.paged_tree_attention(rot, att, batch.desc, shape, 0, d, m, words, cache.desc, ws)
        # the path of each sequence's deepest token
        paths = []
        for s in range(3):
            t = int(np.argmax(trees.depth[batch.begin[s]:batch.begin[s + 1]]))
            paths.append([int(x) for x in np.nonzero(trees.seen[s][t])[0]])
        stride = max(map(len, paths))
        acc = np.array([p + [0] * (stride - len(p)) for p in paths], np.int32)
        count = np.array([len(p) for p in paths], np.int32)
        smq.paged_compact(batch.desc, shape, dev(acc), stride, dev(count), smq.paged_pools([cache.desc]), out)
        first, lengths = lengths, out.download(np.int32)
        same(lengths, first + count)
        # the same tokens, one path each
        at = np.concatenate([batch.begin[s] + np.array(paths[s], int) for s in range(3)])
        one = Batch(plain, list(count), lengths=lengths)
        prot, patt = (smq.DeviceBuffer(4 * len(at) * heads * hd) for _ in range(2))
        smq.paged_norm_rope_kv(smq.paged_rows(dev(q[at]), prot, dev(k[at]), dev(v[at]), *w), one.desc, shape, cb, sb, plain.desc)
        smq.paged_attention(prot, patt, one.desc, shape, 0, plain.desc)
        same(rot.download(np.float32).reshape(q.shape)[at], prot.download(np.float32).reshape(-1, heads, hd))
        both = []
        for c in (cache, plain):
            whole = Batch(c, list(lengths), lengths=lengths)
            rk, rv = (smq.DeviceBuffer(4 * whole.tokens * kv * hd) for _ in range(2))
            smq.paged_read(whole.desc, smq.attn_shape(heads, kv, hd, 0, 0, context), c.desc, rk, rv)
            both.append((rk.download(np.float32), rv.download(np.float32)))
        for a, b in zip(*both):
            same(a, b)
        got, want = att.download(np.float32).reshape(q.shape)[at], patt.download(np.float32).reshape(-1, heads, hd)
        top = np.abs(both[1][1]).max()
        # both within an f32 calculation's error of the same value: scores off by (hd + 8) 2^-24 of sum |q k| each, see tree64
        size = max(np.abs(both[1][0]).max() * np.abs(prot.download(np.float32)).max() * np.sqrt(hd), 1.0)
        limit = 2 * top * (4 * size * (hd + 8) + 4 * (size + 2) + lengths.max() / 8 + 64) * 2.0 ** -24
        assert np.abs(got - want).max() <= limit
        assert not flagged()


@pytest.mark.parametrize("kv_type", [F32, F16, Q8])
def test_drafts_on_a_shared_prompt(kv_type):
    """Three sequences draft on one prompt that a store holds too: its last page, which they take in part, is copied to each
    one's own before their tokens are stored, and stays what it was."""
    heads, kv, hd, page, stride, keep, new = 6, 2, 64, 16, 6, 37, [9, 20, 1]
    cache = Cache(kv_type, kv, hd, page, [keep], spare=40, stride=stride, stale="nan").upload()
    refs = np.zeros(cache.pages, np.int32)
    refs[cache.table[0, :3]] = 2  # the table's row and the store
    room = np.array([keep + n for n in new], np.int32)
    parent, kept = np.zeros(3, np.int32), np.full(3, keep, np.int32)
    want = ref.fork(cache.table, [3], refs, parent, kept, room, page)
    assert (want[3][:, 2] == 5).all() and want[2][cache.table[0, 2]] == 1
    bufs = [dev(x) for x in (cache.table, np.array([3], np.int32), refs, parent, kept, room)]
    outs = [smq.DeviceBuffer(4 * n) for n in (3 * stride, 3, cache.pages, 9, 1)]
    f = smq.page_fork(*bufs[:3], 1, 3, stride, page, cache.pages, *bufs[3:], *outs)
    smq.paged_fork(f, smq.DeviceBuffer(smq.paged_fork_workspace(f)))
    for got, w in zip(outs, want[:4]):
        same(got.download(np.int32), np.ravel(w))
    shape = smq.attn_shape(heads, kv, hd, hd // 2, 0, 64)
    smq.paged_copy(outs[3], 3, shape, smq.paged_pools([cache.desc]))
    ref.copy(cache, want[3])
    cache.table, cache.tb = want[0], outs[0]
    batch = Batch(cache, new, lengths=room)
    trees = Trees(batch).upload()
    cos, sin = tables(64, hd // 2)
    q, k, v = (synth.normal(400 + i, batch.tokens * x * hd, 1.5).reshape(-1, x, hd) for i, x in enumerate((heads, kv, kv)))
    w = (1 + 0.2 * synth.normal(410, hd)).astype(np.float32)
    rot = smq.DeviceBuffer(q.nbytes)
    smq.paged_norm_rope_kv(smq.paged_rows(dev(q), rot, dev(k), dev(v), dev(w), dev(w), depth=trees.db), batch.desc, shape, dev(cos),
                           dev(sin), cache.desc)
    turn = keep + trees.depth
    k = rotate(ref.normed(k, w, 1e-6), cos[turn], sin[turn], 32)
    for s in range(3):
        r = slice(batch.begin[s], batch.begin[s + 1])
        cache.put(s, np.arange(keep, room[s]), k[r], v[r])
    pool_same(cache)
    q = rotate(ref.normed(q, w, 1e-6), cos[turn], sin[turn], 32)
    same(rot.download(np.float32).reshape(q.shape), q)
    want, tol = ref.tree64(cache, batch, q, heads, trees.depth, trees.seen)
    close(tree_attend(cache, batch, q, heads, trees), want, tol)
    assert not flagged()


def test_beams_together():
    """A beam search of three prompts' beams over one pool: choice, fork, copy, store and attention of every step against a
    search that keeps each beam's tokens and works its attention out from them in 64 bits."""
    heads, kv, hd, page, beams, groups, vocab, layers = 4, 2, 32, 16, 4, 3, 300, 2
    rng = np.random.default_rng(9)
    rows, stride, context = groups * beams, 8, 128
    pages = rows * 6
    embed = [(rng.standard_normal((vocab, x * hd))).astype(np.float32) for x in (heads, kv, kv)]
    head = rng.standard_normal((heads * hd, vocab)) * 0.5
    shape = smq.attn_shape(heads, kv, hd, hd // 2, 0, context)
    cos, sin = tables(context, hd // 2)
    cb, sb = dev(cos), dev(sin)
    pools = [Cache(F32, kv, hd, page, [page * pages], spare=0).upload() for _ in range(layers)]
    descs = smq.paged_pools([p.desc for p in pools])
    prompts = [list(rng.integers(3, vocab, n)) for n in (37, 16, 5)]

    def logits_of(tokens):
        pos = np.arange(len(tokens))
        q = rotate(embed[0][tokens[-1:]].reshape(1, heads, hd), cos[pos[-1:]], sin[pos[-1:]], hd // 2)[0].astype(np.float64)
        k = rotate(embed[1][tokens].reshape(-1, kv, hd), cos[pos], sin[pos], hd // 2).astype(np.float64)
        v = embed[2][tokens].reshape(-1, kv, hd).astype(np.float64)
        out = []
        for h in range(heads):
            x = k[:, h // 2] @ q[h] / np.sqrt(hd)
            p = np.exp(x - x.max())
            out.append(p @ v[:, h // 2] / p.sum())
        return (np.concatenate(out) @ head).astype(np.float32)

    # old rows: one per prompt, its pages shared by the beams from the first fork on
    table = np.full((groups, stride), -1, np.int32)
    order, at = rng.permutation(pages).astype(np.int32), 0
    held = np.array([-(-len(p) // page) for p in prompts], np.int32)
    for g, n in enumerate(held):
        table[g, :n] = order[at:at + n]
        at += n
    refs = np.bincount(table[table >= 0], minlength=pages).astype(np.int32)
    tb, hb, rb = dev(table), dev(held), dev(refs)

    def store(tb, n_rows, new, lengths, tokens):
        begin = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        total = int(begin[-1])
        batch = smq.paged_batch(dev(begin), dev(np.asarray(lengths, np.int32)), tb, n_rows, total, stride)
        q, k, v = (dev(np.ascontiguousarray(e[tokens])) for e in embed)
        rot, att = smq.DeviceBuffer(4 * total * heads * hd), smq.DeviceBuffer(4 * total * heads * hd)
        for p in pools:
            smq.paged_norm_rope_kv(smq.paged_rows(q, rot, k, v), batch, shape, cb, sb, p.desc)
        ws = smq.DeviceBuffer(max(16, smq.paged_attention_workspace(batch, shape)))
        smq.paged_attention(rot, att, batch, shape, 0, pools[-1].desc, ws)
        return att.download(np.float32).reshape(total, -1)[begin[1:] - 1] @ head

    first = store(tb, groups, [len(p) for p in prompts], [len(p) for p in prompts], [t for p in prompts for t in p])
    live = [[(list(p), 0.0, False)] for p in prompts]
    logits, score, done = first.astype(np.float32), np.zeros(groups, np.float32), np.zeros(groups, np.uint8)
    width, ends, eos = 1, 0, NONE
    history = np.full((groups, 64), NONE, np.uint32)
    for g, p in enumerate(prompts):
        history[g, :len(p)] = p
    hist, length = dev(history), dev(np.array([len(p) for p in prompts], np.int32))
    old = groups
    for step in range(9):
        n = groups * beams
        # the search on tokens
        nxt = []
        for g in range(groups):
            cand = []
            for i, (tokens, s, over) in enumerate(live[g]):
                if over:
                    cand.append((-s, i, 0, tokens, True))
                    continue
                l = logits_of(tokens).astype(np.float64)
                l -= l.max() + np.log(np.exp(l - l.max()).sum())
                cand += [(-(s + l[v]), i, int(v), tokens + [int(v)], False) for v in np.argsort(-l, kind="stable")[:beams]]
            cand.sort(key=lambda c: c[:3])
            nxt.append([(c[3], -c[0], c[4]) for c in cand[:beams]])
        if step == 2:
            eos = nxt[0][1][0][-1]  # one that some beam ends with
        nxt = [[(tokens, s, over or tokens[-1] == eos) for tokens, s, over in x] for x in nxt]
        lb, sc, dn = dev(np.ascontiguousarray(logits, np.float32)), dev(score), dev(done)
        outs = [smq.DeviceBuffer(4 * n) for _ in range(3)] + [smq.DeviceBuffer(n), smq.DeviceBuffer(4 * n * 64), smq.DeviceBuffer(4 * n)]
        b = smq.beam_step(lb, vocab, groups, width, vocab, beams, sc, *outs[:3], done=dn, pad=0, eos=eos, done_out=outs[3],
                          history=hist, history_out=outs[4], history_stride=64, length=length, length_out=outs[5])
        smq.beam_select(b, smq.DeviceBuffer(smq.beam_select_workspace(b)))
        parent, token, score, done = (o.download(t) for o, t in zip(outs, (np.int32, np.uint32, np.float32, np.uint8)))
        live = nxt
        hist, length, lens = outs[4], outs[5], outs[5].download(np.int32)
        rows_of = hist.download(np.uint32).reshape(n, 64)
        for i in range(n):
            tokens, s, over = live[i // beams][i % beams]
            assert list(rows_of[i, :lens[i]]) == tokens and bool(done[i]) == over, (step, i)
            assert abs(score[i] - s) < 1e-4 * max(1.0, abs(s))  # of nine steps' f32 attention and logits
            ends += over
        # pages: each beam keeps its parent's positions and gets room for its last token (done ones: the same as before)
        kept = (lens - 1).astype(np.int32)
        no = [smq.DeviceBuffer(4 * x) for x in (n * stride, n, pages, n * 3, 1)]
        f = smq.page_fork(tb, hb, rb, old, n, stride, page, pages, outs[0], dev(kept), dev(lens.astype(np.int32)), *no)
        smq.paged_fork(f, smq.DeviceBuffer(smq.paged_fork_workspace(f)))
        smq.paged_copy(no[3], n, shape, descs)
        tb, hb, rb, old, width = no[0], no[1], no[2], n, beams
        assert no[4].download(np.int32)[0] >= 0
        now, counts = tb.download(np.int32).reshape(n, stride), rb.download(np.int32)
        same(np.bincount(now[now >= 0], minlength=pages).astype(np.int32), counts)
        logits = store(tb, n, [1] * n, lens, [int(r[m - 1]) for r, m in zip(rows_of, lens)])
        assert not flagged()
    assert ends
    now, lens = tb.download(np.int32).reshape(n, stride), length.download(np.int32)
    keys = [p.kb.download(np.float32).reshape(pages, kv, page, hd) for p in pools]
    for row in range(n):  # every layer went the same way
        for pos in range(lens[row]):
            pg, sl = now[row, pos // page], pos % page
            a, b = (x[pg, :, sl] for x in keys)
            same(a, b)
            same(a[0], rotate(embed[1][rows_of[row, pos]].reshape(1, kv, hd), cos[pos:pos + 1], sin[pos:pos + 1], hd // 2)[0, 0])


def test_replays_of_all():
    """Each operator captured into one graph and replayed with other contents beside eager work on buffers of its own, and on
    another stream; two graphs at the same time have workspaces of their own."""
    heads, kv, hd, page, words = 8, 2, 64, 32, 2
    lengths, new = [700, 190, 64], [20, 33, 1]
    cos, sin = (dev(x) for x in tables(800, hd // 2))
    shape = smq.attn_shape(heads, kv, hd, hd // 2, 0, 800)
    n, groups, beams, select, vocab = sum(new), 3, 2, 3, 3000

    class Side:
        """The same calls on buffers of its own."""

        def __init__(self):
            self.cache = Cache(Q8, kv, hd, page, lengths, seed=12, spare=20).upload()
            c = self.cache
            self.batch = Batch(c, new)
            buf = smq.DeviceBuffer
            self.q, self.k, self.v = (buf(4 * n * x * hd) for x in (heads, kv, kv))
            self.norm, self.parent, self.depth, self.mask = buf(4 * hd), buf(4 * n), buf(4 * n), buf(4 * n * words)
            self.rot, self.att, self.acc, self.count, self.out = buf(4 * n * heads * hd), buf(4 * n * heads * hd), buf(36), buf(12), buf(12)
            self.rows = smq.paged_rows(self.q, self.rot, self.k, self.v, self.norm, self.norm, 1e-6, self.depth)
            self.pools = smq.paged_pools([c.desc])
            held = np.array([-(-m // page) for m in lengths], np.int32)
            refs = np.bincount(c.table[c.table >= 0], minlength=c.pages).astype(np.int32)
            self.old = [dev(x) for x in (held, refs)]
            self.plan = [buf(12) for _ in range(3)]
            self.no = [buf(4 * x) for x in (3 * c.stride, 3, c.pages, 9, 1)]
            self.fork = smq.page_fork(c.tb, *self.old, 3, 3, c.stride, page, c.pages, *self.plan, *self.no)
            self.logits, self.score = buf(4 * groups * beams * vocab), buf(4 * groups * beams)
            self.res = [buf(4 * groups * select) for _ in range(3)]
            self.step = smq.beam_step(self.logits, vocab, groups, beams, vocab, select, self.score, *self.res)
            self.ws = [buf(max(16, x)) for x in (smq.paged_tree_attention_workspace(self.batch.desc, shape),
                                                 smq.paged_fork_workspace(self.fork), smq.beam_select_workspace(self.step))]

        def run(self):
            c = self.cache.desc
            smq.draft_masks(self.parent, self.batch.desc, self.depth, self.mask, words)
            smq.paged_norm_rope_kv(self.rows, self.batch.desc, shape, cos, sin, c)
            smq.paged_tree_attention(self.rot, self.att, self.batch.desc, shape, 0, self.depth, self.mask, words, c, self.ws[0])
            smq.paged_compact(self.batch.desc, shape, self.acc, 3, self.count, self.pools, self.out)
            smq.paged_fork(self.fork, self.ws[1])
            smq.paged_copy(self.no[3], 3, shape, self.pools)
            smq.beam_select(self.step, self.ws[2])

        def fill(self, t):
            rng = np.random.default_rng(500 + t)
            f32 = lambda m: rng.standard_normal(m).astype(np.float32)  # noqa: E731
            for b in (self.q, self.k, self.v, self.norm, self.score):
                b.upload(f32(b.nbytes // 4))
            self.logits.upload(3 * f32(groups * beams * vocab))
            self.parent.upload(np.concatenate([ref.random_tree(rng, m) for m in new]).astype(np.int32))
            self.acc.upload(np.array([sorted(rng.choice(m, 3, replace=False)) if m > 3 else [0, 0, 0] for m in new], np.int32))
            self.count.upload(np.array([3, 2, 1], np.int32))
            keep = [int(rng.integers(0, m)) for m in lengths]
            for b, x in zip(self.plan, ([0, 0, 2], [keep[0], keep[0], keep[2]], [keep[0] + 9, keep[0] + 40, keep[2]])):
                b.upload(np.array(x, np.int32))

        def results(self):
            bufs = [self.depth, self.mask, self.rot, self.att, self.out, *self.no, *self.res]
            return [b.download(np.uint32) for b in bufs] + [x.view(np.uint8) for x in map(np.ascontiguousarray, self.cache.download())]

    sides = [Side() for _ in range(3)]
    graphs = [smq.capture(s.run) for s in sides[:2]]
    side = torch.cuda.Stream()
    for t in range(4):
        for s in sides:
            s.fill(t)
        smq.synchronize()
        smq.load().smq_set_stream(side.cuda_stream)
        try:
            graphs[1].launch()
        finally:
            smq.load().smq_set_stream(None)
        graphs[0].launch()
        sides[2].run()
        smq.synchronize()
        side.synchronize()
        assert not flagged()
        want = sides[2].results()
        for s in sides[:2]:
            for a, b in zip(s.results(), want):
                assert np.array_equal(a, b)
    for g in graphs:
        g.destroy()


def test_offsets_past_32_bits_of_all():
    """A Q8 pool of more than 2^32 codes, pages at its end: stored, attended, copied and moved there."""
    heads, kv, hd, page = 4, 4, 128, 256
    pages = (1 << 32) // (kv * hd * page) + 12
    shape = smq.attn_shape(heads, kv, hd, 0, 0, 600)
    small = Cache(Q8, kv, hd, page, [600], spare=5, seed=2)  # the same pages at the end of a large pool
    k, v = (smq.DeviceBuffer(pages * kv * hd * page) for _ in range(2))
    ks, vs = (smq.DeviceBuffer(pages * kv * 4 * page * 4) for _ in range(2))
    low = pages - small.pages
    for b, x, one in ((k, small.k, kv * hd * page), (v, small.values_layout(small.v), kv * hd * page),
                      (ks, small.ks, kv * 16 * page), (vs, small.vs, kv * 16 * page)):
        b.upload(x, low * one)
    small.upload()
    big = smq.paged_kv(k, v, ks, vs, Q8, page, pages)
    small.tb.upload(np.where(small.table >= 0, small.table + low, -1).astype(np.int32))
    pools = smq.paged_pools([big])
    batch = Batch(small, [40])
    trees = Trees(batch).upload()
    rows = [synth.normal(97 + i, 40 * kv * hd).reshape(40, kv, hd) for i in range(2)]
    q = synth.normal(99, 40 * heads * hd).reshape(40, heads, hd)
    w = (1 + 0.2 * synth.normal(31, hd)).astype(np.float32)
    z = dev(np.zeros(1, np.float32))
    rot, att, out = smq.DeviceBuffer(q.nbytes), smq.DeviceBuffer(q.nbytes), smq.DeviceBuffer(4)
    smq.paged_norm_rope_kv(smq.paged_rows(dev(q), rot, dev(rows[0]), dev(rows[1]), dev(w), dev(w)), batch.desc, shape, z, z, big)
    small.put(0, np.arange(560, 600), ref.normed(rows[0], w, 1e-6), rows[1])
    want, tol = ref.tree64(small, batch, ref.normed(q, w, 1e-6), heads, trees.depth, trees.seen)
    smq.paged_tree_attention(rot, att, batch.desc, shape, 0, trees.db, trees.wb, trees.stride, big)
    close(att.download(np.float32).reshape(q.shape), want, tol)
    path = [1, 2, 9, 30, 39]
    smq.paged_compact(batch.desc, shape, dev(np.array(path, np.int32)), 5, dev(np.array([5], np.int32)), pools, out)
    ref.compact(small, 0, 560, path)
    free = [p for p in range(small.pages) if p not in small.table]
    copies = np.array([[small.table[0, 1], free[0], 200], [small.table[0, 2], free[1], 53]], np.int32)
    smq.paged_copy(dev((copies + [low, low, 0]).astype(np.int32)), 2, shape, pools)
    ref.copy(small, copies)
    for b, x, one, t in ((k, small.k, kv * hd * page, np.int8), (v, small.values_layout(small.v), kv * hd * page, np.int8),
                         (ks, small.ks, kv * 4 * page, np.float32), (vs, small.vs, kv * 4 * page, np.float32)):
        same(b.download(t, x.size, low * one * x.itemsize).reshape(x.shape), x)
    assert not flagged()


def test_unaligned_rows_of_drafts():
    """q, k, v, norms and outputs at 4-byte addresses."""
    heads, kv, hd, n = 6, 2, 64, 21
    cache = Cache(F16, kv, hd, 32, [70], stale="nan").upload()
    batch = Batch(cache, [n])
    trees = Trees(batch).upload()
    shape = smq.attn_shape(heads, kv, hd, 32, 0, 70)
    cos, sin = tables(70, 32)
    q, k, v = (synth.normal(101 + i, n * w).reshape(n, -1, hd) for i, w in enumerate((heads * hd, kv * hd, kv * hd)))
    w = (1 + 0.2 * synth.normal(31, hd)).astype(np.float32)

    def off(x):
        b = smq.DeviceBuffer(x.nbytes + 4)
        b.upload(x, 4)
        return b

    qb, kb, vb, wb, cb, sb = (off(x) for x in (q, k, v, w, cos, sin))
    att = smq.DeviceBuffer(q.nbytes + 4)
    r = smq.paged_rows(qb.at(4), qb.at(4), kb.at(4), vb.at(4), wb.at(4), wb.at(4), 1e-6, trees.db)
    smq.paged_norm_rope_kv(r, batch.desc, shape, cb.at(4), sb.at(4), cache.desc)
    smq.paged_tree_attention(qb.at(4), att.at(4), batch.desc, shape, 0, trees.db, trees.wb, trees.stride, cache.desc)
    turn = 49 + trees.depth
    cache.put(0, np.arange(49, 70), rotate(ref.normed(k, w, 1e-6), cos[turn], sin[turn], 32), v)
    qr = rotate(ref.normed(q, w, 1e-6), cos[turn], sin[turn], 32)
    same(qb.download(np.float32, offset=4).reshape(q.shape), qr)
    want, tol = ref.tree64(cache, batch, qr, heads, trees.depth, trees.seen)
    close(att.download(np.float32, offset=4).reshape(q.shape), want, tol)
