"""The paged KV cache and its attention on the GPU: the store and the rows read back bit for bit against numpy, whole pools
compared; the attention against 64 bits within a bound derived beside attend64."""
import numpy as np
import pytest
import torch

from checks import assert_same_f32, say
from paged_ref import F16, F32, Q8, Batch, Cache, attend64, rotate, tables
from paged_ref import visible
from smq_pkg import smq, synth

pytestmark = pytest.mark.gpu
dev = smq.DeviceBuffer.from_array
TYPES = {F32: "f32", F16: "f16", Q8: "q8"}


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
    assert np.array_equal(got, want)


def flagged():
    try:
        smq.numeric_check()
    except smq.SmqError as e:
        assert e.status == smq.SM_ERR_NUMERIC
        return True
    return False


STORES = [  # type, heads, kv, hd, rotary pairs, page, lengths, new
    (Q8, 14, 2, 64, 32, 64, [200, 1, 65, 130], [1, 1, 1, 1]),      # a decode step; a first token; a first slot of a page
    (F16, 12, 2, 128, 64, 32, [133, 70, 40], [133, 5, 0]),         # a whole prompt, a ragged chunk, no token at all
    (F32, 9, 3, 64, 16, 16, [17, 40], [17, 3]),                    # partial rotary, the smallest page
    (Q8, 16, 2, 80, 40, 256, [300, 257], [290, 257]),              # a last block of 16 dims
    (Q8, 4, 4, 16, 8, 16, [33], [20]),                             # one half block
    (F16, 2, 1, 256, 0, 128, [129, 3], [2, 2]),                    # no rotation, the widest head
    (F32, 8, 8, 96, 48, 64, [64, 63, 65], [64, 63, 65]),
    (Q8, 32, 8, 128, 64, 128, [500], [500]),
]


@pytest.mark.parametrize("kv_type,heads,kv,hd,pairs,page,lengths,new", STORES)
def test_store_and_read(kv_type, heads, kv, hd, pairs, page, lengths, new):
    say("paged store", TYPES[kv_type], heads, kv, hd, pairs, page, lengths, new)
    cache = Cache(kv_type, kv, hd, page, lengths).upload()
    batch = Batch(cache, new, padding=3)
    context, n = max(lengths) + 5, batch.tokens
    shape = smq.attn_shape(heads, kv, hd, pairs, 0, context)
    cos, sin = tables(context, pairs)
    if not pairs:
        cos = sin = np.zeros(1, np.float32)
    q, k, v = (synth.normal(70 + i, n * w).reshape(n, -1, hd) for i, w in enumerate((heads * hd, kv * hd, kv * hd)))
    k[0] *= 1e-30  # tiny scales
    v[-4] *= 300.0
    qb, kb, vb = dev(q), dev(k), dev(v)
    want_q, rot_k = np.full_like(q, 7.0), np.zeros_like(k)
    at = 0
    for s, pos in batch.where():
        rows = slice(at, at + len(pos))
        want_q[rows] = rotate(q[rows], cos[pos], sin[pos], pairs) if pairs else q[rows]
        rot_k[rows] = rotate(k[rows], cos[pos], sin[pos], pairs) if pairs else k[rows]
        if len(pos):
            cache.put(s, pos, rot_k[rows], v[rows])
        at += len(pos)
    out = dev(np.full_like(q, 7.0))
    smq.paged_rope_kv(qb, out, kb, vb, batch.desc, shape, dev(cos), dev(sin), cache.desc)
    smq.numeric_check()
    same(out.download(np.float32).reshape(q.shape), want_q)
    same(kb.download(np.float32).reshape(k.shape), k)
    wants = (cache.k, cache.v) + ((cache.ks, cache.vs) if kv_type == Q8 else ())
    for got, want in zip(cache.download(), wants):
        same(got, want)
    # in place, and without q
    smq.paged_rope_kv(qb, qb, kb, vb, batch.desc, shape, dev(cos), dev(sin), cache.desc)
    want_q[at:] = q[at:]
    same(qb.download(np.float32).reshape(q.shape), want_q)
    smq.paged_rope_kv(None, None, kb, vb, batch.desc, shape, dev(cos), dev(sin), cache.desc)
    for got, want in zip(cache.download(), wants):
        same(got, want)
    # the rows back, padding untouched
    rk, rv = (dev(np.full((n, kv, hd), 5.0, np.float32)) for _ in range(2))
    smq.paged_read(batch.desc, shape, cache.desc, rk, rv)
    wk, wv = (np.full((n, kv, hd), 5.0, np.float32) for _ in range(2))
    at = 0
    for s, pos in batch.where():
        if len(pos):
            wk[at:at + len(pos)], wv[at:at + len(pos)] = cache.rows(s, pos)
        at += len(pos)
    same(rk.download(np.float32).reshape(wk.shape), wk)
    same(rv.download(np.float32).reshape(wv.shape), wv)
    smq.numeric_check()


@pytest.mark.parametrize("kv_type", [F32, F16, Q8])
def test_read_whole_sequences(kv_type):
    """Whole sequences, from one position to many pages, at an unaligned destination."""
    lengths = [1, 700, 64, 129]
    cache = Cache(kv_type, 2, 80, 32, lengths).upload()
    batch = Batch(cache, lengths)
    shape = smq.attn_shape(4, 2, 80, 40, 0, 700)
    n = batch.tokens * 160
    kb, vb = smq.DeviceBuffer(4 * n + 4), smq.DeviceBuffer(4 * n + 4)
    smq.paged_read(batch.desc, shape, cache.desc, kb.at(4), vb.at(4))
    want = [np.concatenate(x) for x in zip(*(cache.rows(s, pos) for s, pos in batch.where()))]
    for b, w in zip((kb, vb), want):
        same(b.download(np.float32, offset=4).reshape(w.shape), w)
    smq.numeric_check()


@pytest.mark.parametrize("kv_type", [F32, F16, Q8])
def test_store_of_values_that_do_not_fit(kv_type):
    """NaN, infinities and (f16) values past 65504: stored as documented, flagged; their neighbours as ever."""
    cache = Cache(kv_type, 2, 64, 16, [20]).upload()
    batch = Batch(cache, [4])
    shape = smq.attn_shape(2, 2, 64, 0, 0, 64)
    k, v = (synth.normal(80 + i, 4 * 128).reshape(4, 2, 64) for i in range(2))
    z = dev(np.zeros(1, np.float32))

    def store():
        smq.paged_rope_kv(None, None, dev(k), dev(v), batch.desc, shape, z, z, cache.desc)
        return flagged()

    assert not store()
    for row, head, dim, x in ((1, 0, 3, np.nan), (2, 1, 40, np.inf), (3, 0, 63, 7e4)):
        v[row, head, dim] = x
        assert store() == (kv_type == F16 or not np.isfinite(x) or row > 1)
        cache.put(0, np.arange(16, 20), k, v)
        for got, want in zip(cache.download(), (cache.k, cache.v, cache.ks, cache.vs)):
            nan = np.isnan(want.astype(np.float32))
            assert np.array_equal(np.isnan(got.astype(np.float32)), nan)
            same(np.where(nan, 0, got).astype(want.dtype), np.where(nan, 0, want).astype(want.dtype))


def attend(cache, batch, q, heads, kv, hd, window=0, sinks=0, context=None, split=True, fill=9.0):
    shape = smq.attn_shape(heads, kv, hd, hd // 2, window, context or int(max(batch.length.max(), 1)))
    qb, att = dev(q), dev(np.full(q.shape, fill, np.float32))
    need = smq.paged_attention_workspace(batch.desc, shape)
    ws = smq.DeviceBuffer(need) if split and need else None
    if ws:
        ws.fill(0xFF)
    smq.paged_attention(qb, att, batch.desc, shape, sinks, cache.desc, ws)
    return att.download(np.float32).reshape(q.shape)


def close(got, want, tol, rows=slice(None), what=""):
    d = np.abs(got[rows].astype(np.float64) - want[rows])
    bad = ~(d <= tol[rows])
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} off, worst {np.nanmax(d / np.maximum(tol[rows], 1e-30)):.3g} " \
                          f"of the bound at {np.argwhere(bad)[0]}: {got[rows][bad][0]} for {want[rows][bad][0]}"


ATTENDS = [  # heads, kv, hd, page, lengths, new, window, sinks
    (14, 2, 64, 32, [1], [1], 0, 0),                                        # one position
    (14, 2, 64, 64, [131, 1, 64, 65, 33], [1, 1, 1, 1, 1], 0, 0),           # a ragged decode step
    (12, 2, 128, 16, [15, 16, 17, 200], [3, 16, 1, 40], 0, 0),              # ragged chunks over the smallest pages
    (32, 4, 64, 128, [1030], [1], 100, 4),                                  # window and sinks far apart
    (8, 8, 96, 256, [70, 300], [70, 33], 20, 3),                            # no shared heads; a window inside a chunk
    (16, 2, 80, 64, [150, 90], [37, 90], 0, 0),                             # a head that is no multiple of 32
    (9, 3, 64, 32, [100, 37], [64, 0], 1, 0),                               # each row sees itself alone; no new token
    (4, 4, 16, 16, [50], [50], 7, 50),                                      # sinks past the window: all visible
    (17, 1, 32, 64, [129], [5], 64, 1),                                     # 17 heads on one KV head
    (2, 1, 256, 64, [400], [2], 0, 0),                                      # the widest head
    (6, 2, 112, 32, [95], [95], 33, 2),
    (40, 1, 48, 32, [77, 5], [9, 5], 0, 0),                                 # 40 heads on one KV head
]


@pytest.mark.parametrize("kv_type", [F32, F16, Q8])
@pytest.mark.parametrize("heads,kv,hd,page,lengths,new,window,sinks", ATTENDS)
def test_attention(kv_type, heads, kv, hd, page, lengths, new, window, sinks):
    say("paged attention", TYPES[kv_type], heads, kv, hd, page, lengths, new, window, sinks)
    cache = Cache(kv_type, kv, hd, page, lengths, stale="nan")
    for s, (m, n) in enumerate(zip(lengths, new)):  # what no row of the batch sees is poisoned too
        if window and n:
            low = m - n + 1 - window
            cache.spoil_positions(s, np.arange(min(sinks, low), low) if low > sinks else np.zeros(0, int))
    cache.upload()
    batch = Batch(cache, new, padding=2)
    q = synth.normal(90, batch.tokens * heads * hd, 1.5).reshape(-1, heads, hd)
    want, tol = attend64(cache, batch, q, heads, window, sinks)
    n = int(batch.begin[-1])
    first = attend(cache, batch, q, heads, kv, hd, window, sinks)
    close(first, want, tol, slice(0, n))
    assert (first[n:] == 9.0).all()
    smq.numeric_check()
    again = attend(cache, batch, q, heads, kv, hd, window, sinks)
    same(again, first)
    whole = attend(cache, batch, q, heads, kv, hd, window, sinks, split=False)
    close(whole, want, tol, slice(0, n), "without a workspace")
    # a context far past the lengths (as a captured step has it)
    wide = attend(cache, batch, q, heads, kv, hd, window, sinks, context=9000)
    close(wide, want, tol, slice(0, n), "wide context")


@pytest.mark.parametrize("kv_type", [F32, F16, Q8])
@pytest.mark.parametrize("lengths,new", [([5000, 3001, 64, 4097], [1, 1, 1, 1]), ([4500, 700], [3, 130])])
def test_attention_long(kv_type, lengths, new):
    """Sequences that are split over workgroups, with and without room for it."""
    heads, kv, hd = 8, 2, 64
    cache = Cache(kv_type, kv, hd, 64, lengths, stale="nan").upload()
    batch = Batch(cache, new)
    q = synth.normal(91, batch.tokens * heads * hd, 1.5).reshape(-1, heads, hd)
    want, tol = attend64(cache, batch, q, heads)
    close(attend(cache, batch, q, heads, kv, hd), want, tol)
    close(attend(cache, batch, q, heads, kv, hd, split=False), want, tol)
    shape = smq.attn_shape(heads, kv, hd, 32, 0, 5000)
    need = smq.paged_attention_workspace(batch.desc, shape)
    for part in (need // 2, need // 3, 64):  # less room than the widest split
        ws, att, qb = smq.DeviceBuffer(max(part, 64) + 64), dev(np.zeros_like(q)), dev(q)
        guard = np.full(ws.nbytes, 0xAB, np.uint8)
        ws.upload(guard)
        smq.paged_attention(qb, att, batch.desc, shape, 0, cache.desc, ws, part // 16 * 16)
        close(att.download(np.float32).reshape(q.shape), want, tol, what=f"{part} bytes")
        assert (ws.download(np.uint8)[part // 16 * 16:] == 0xAB).all()
    smq.numeric_check()


@pytest.mark.parametrize("kv_type", [F32, F16, Q8])
def test_attention_of_many(kv_type):
    """More sequences than a wave has lanes, cut into pieces; then so many tiles of chunks that none is."""
    heads, kv, hd = 2, 1, 64
    lengths = [1500, 1, 33] + [1300 + 3 * s for s in range(66)]
    cache = Cache(kv_type, kv, hd, 64, lengths, stale="nan").upload()
    batch = Batch(cache, [1, 0] + [1] * 67)
    assert smq.paged_attention_workspace(batch.desc, smq.attn_shape(heads, kv, hd, 0, 0, 1500)) > 0
    q = synth.normal(98, batch.tokens * heads * hd, 1.5).reshape(-1, heads, hd)
    want, tol = attend64(cache, batch, q, heads)
    close(attend(cache, batch, q, heads, kv, hd), want, tol)
    heads, kv, hd = 32, 8, 128
    lengths = [64 + s % 7 for s in range(34)]
    cache = Cache(kv_type, kv, hd, 32, lengths, stale="nan").upload()
    batch = Batch(cache, [64 - s % 5 for s in range(34)])
    assert batch.tokens >= 2048  # 512 tiles of 128 rows of four 32-wide steps
    q = synth.normal(99, batch.tokens * heads * hd, 1.5).reshape(-1, heads, hd)
    want, tol = attend64(cache, batch, q, heads)
    close(attend(cache, batch, q, heads, kv, hd), want, tol)
    smq.numeric_check()


@pytest.mark.parametrize("new", [[1, 1, 1], [2, 1, 400]])
def test_the_longest_context(new):
    """Tables and a context of 1,048,576 positions, lengths far below: the host plans for the first, the device cuts the
    second. With windows, whose steps are few, too."""
    heads, kv, hd = 6, 2, 64
    cache = Cache(F16, kv, hd, 64, [3001, 1, 700], stale="nan", stride=1 << 14).upload()
    batch = Batch(cache, new, padding=3)
    q = synth.normal(100, batch.tokens * heads * hd, 1.5).reshape(-1, heads, hd)
    n = int(batch.begin[-1])
    for window, sinks in ((0, 0), (129, 5), (0xFFFFFFFF, 0xFFFFFFFF)):
        want, tol = attend64(cache, batch, q, heads, window if window < 1 << 20 else 0, sinks if window < 1 << 20 else 0)
        for split in (True, False):
            got = attend(cache, batch, q, heads, kv, hd, window, sinks, context=1 << 20, split=split)
            close(got, want, tol, slice(0, n))
            assert (got[n:] == 9.0).all()
    smq.numeric_check()


def test_scores_of_every_size():
    """Rows whose softmax is one position, whose scores are all equal, tiny or past f16's range."""
    heads, kv, hd, n = 4, 2, 64, 90
    for kv_type in (F32, F16, Q8):
        for size in (1e-20, 1e-3, 30.0, 3000.0):
            cache = Cache(kv_type, kv, hd, 32, [n], stale="nan")
            if kv_type == Q8:
                cache.vs *= np.float32(1e6 if size > 1 else 1e-12)
                cache.vs[:, :, :, ::3] *= np.float32(1e-9)  # scales far apart within a page
            cache.upload()
            batch = Batch(cache, [7])
            q = (synth.normal(93, 7 * heads * hd) * size).astype(np.float32).reshape(-1, heads, hd)
            q[3] = 0.0
            want, tol = attend64(cache, batch, q, heads)
            got = attend(cache, batch, q, heads, kv, hd)
            # a block scale far below its tile's largest rounds at the tile's size: 2^-22 of the largest |v|
            _, v = cache.rows(0, np.arange(n), np.float64)
            close(got, want, tol + 2.0 ** -22 * np.abs(v).max(), what=f"{TYPES[kv_type]} {size}")


def test_values_that_are_not_finite_stay_where_they_are_seen():
    """An infinite value in a chunk's last tokens changes no earlier row, one outside a later row's window not that row."""
    heads, kv, hd = 4, 2, 64
    for kv_type in (F32, F16, Q8):
        cache = Cache(kv_type, kv, hd, 32, [100], stale="nan")
        cache.spoil_positions(0, np.array([70, 98, 99]))
        cache.upload()
        batch = Batch(cache, [60])  # positions 40 .. 99
        q = synth.normal(94, 60 * heads * hd, 1.0).reshape(-1, heads, hd)
        with np.errstate(all="ignore"):
            want, tol = attend64(cache, batch, q, heads, 10, 2)
        got = attend(cache, batch, q, heads, kv, hd, 10, 2)
        fine = np.isfinite(want).all((1, 2))
        assert fine.sum() == 60 - 10 - 2  # rows 70 .. 79, 98 and 99 see one
        close(got, want, tol, fine, TYPES[kv_type])


def test_rows_without_a_place():
    """More new tokens than positions, lengths past the table and the context, page ids of no page: flagged, nothing else
    touched, and what has a place is right."""
    heads, kv, hd = 4, 2, 64
    cache = Cache(F16, kv, hd, 32, [40, 96, 64], stale="nan").upload()
    q = synth.normal(95, 9 * heads * hd).reshape(-1, heads, hd)
    good = Batch(cache, [3, 3, 3])
    want, tol = attend64(cache, good, q, heads)
    close(attend(cache, good, q, heads, kv, hd), want, tol)
    assert not flagged()
    cases = [([2, 96, 64], slice(3, 9)), ([40, 97, 64], slice(0, 3)), ([40, 96, -1], slice(0, 6))]
    z = dev(np.zeros(9 * kv * hd, np.float32))
    for lengths, rows in cases:
        batch = Batch(cache, [3, 3, 3], lengths=lengths)
        got = attend(cache, batch, q, heads, kv, hd, context=96)
        close(got, want, tol, rows)
        assert np.isfinite(got[rows]).all()
        assert flagged()
    # positions before 0 and past the context: no store, no read, zeros
    batch = Batch(cache, [3, 0, 0], lengths=[2, 96, 64])
    got = attend(cache, batch, q[:3], heads, kv, hd, context=96)
    assert (got[0] == 0).all() and (got[1:3] != 0).any(-1).all() and flagged()
    shape = smq.attn_shape(heads, kv, hd, 0, 0, 96)
    before = cache.download()
    batch = Batch(cache, [1, 1, 0], lengths=[0, 97, 64])
    smq.paged_rope_kv(None, None, z, z, batch.desc, shape, z, z, cache.desc)
    assert flagged()
    for a, b in zip(before, cache.download()):
        same(a, b)
    rk, rv = (dev(np.full(2 * kv * hd, 5.0, np.float32)) for _ in range(2))
    smq.paged_read(batch.desc, shape, cache.desc, rk, rv)
    assert flagged() and (rk.download(np.float32) == 5.0).all() and (rv.download(np.float32) == 5.0).all()
    # page ids of no page: those positions are not seen, nothing is stored or read there
    table = cache.table.copy()
    table[1, 0], table[2, 1] = cache.pages, -7
    cache.tb.upload(table)
    got = attend(cache, good, q, heads, kv, hd)
    assert flagged()
    close(got, want, tol, slice(0, 3))
    assert np.isfinite(got).all()
    for r in range(3, 6):  # sequence 1 without its first page: the others alone
        k, v = cache.rows(1, np.arange(32, good.length[1] - 3 + (r - 3) + 1), np.float64)
        for h in range(heads):
            x = k[:, h // 2] @ q[r, h].astype(np.float64) / 8
            w = np.exp(x - x.max())
            assert np.abs(got[r, h] - w @ v[:, h // 2] / w.sum()).max() < 1e-4
    batch = Batch(cache, [0, 0, 2])  # positions 62, 63: the page that is none
    smq.paged_rope_kv(None, None, z, z, batch.desc, shape, z, z, cache.desc)
    assert flagged()
    for a, b in zip(before, cache.download()):
        same(a, b)
    smq.paged_read(batch.desc, shape, cache.desc, rk, rv)
    assert flagged() and (rk.download(np.float32) == 5.0).all()
    # a table whose every page is none: a row that sees nothing is 0
    cache.tb.upload(np.full_like(table, -1))
    assert (attend(cache, good, q, heads, kv, hd) == 0).all() and flagged()
    # pages that no row sees may have any id
    table[:] = cache.table
    table[1, 0] = 1 << 30
    cache.tb.upload(table)
    got = attend(cache, good, q, heads, kv, hd, window=20)
    want, tol = attend64(cache, good, q, heads, 20)
    close(got, want, tol)
    assert not flagged()


def test_begins_that_do_not_ascend():
    """A begin array of nonsense: flagged, nothing outside the rows touched."""
    heads, kv, hd = 4, 2, 64
    cache = Cache(F32, kv, hd, 32, [64, 64], stale="nan").upload()
    q = synth.normal(96, 6 * heads * hd).reshape(-1, heads, hd)
    for begin in ([0, 5, 3], [-4, 2, 6], [0, 3, 1 << 30], [3, 1, 2], [0, -1, 6]):
        batch = Batch(cache, [3, 3])
        batch.bb.upload(np.array(begin, np.int32))
        got = attend(cache, batch, q, heads, kv, hd)
        assert np.isfinite(got).all() and flagged()


def test_sequences_that_overlap():
    """Sequences of the same rows, many more tiles than the batch's tokens can have, where tiles are cut: flagged, results
    finite, rows behind left as they were, and the next call with the same workspace is right."""
    heads, kv, hd, seqs = 4, 2, 64, 12
    cache = Cache(F16, kv, hd, 64, [1300] * seqs).upload()
    q = synth.normal(97, 6 * heads * hd).reshape(-1, heads, hd)
    batch = Batch(cache, [1] * 6 + [0] * (seqs - 6))
    assert smq.paged_attention_workspace(batch.desc, smq.attn_shape(heads, kv, hd, 0, 0, 1300)) > 0
    want, tol = attend64(cache, batch, q, heads)
    close(attend(cache, batch, q, heads, kv, hd), want, tol)
    good = batch.begin.copy()
    batch.bb.upload(np.array([0, 6] * (seqs // 2) + [0], np.int32))
    assert np.isfinite(attend(cache, batch, q, heads, kv, hd)).all() and flagged()
    z = dev(np.zeros(6 * kv * hd, np.float32))
    smq.paged_read(batch.desc, smq.attn_shape(heads, kv, hd, 0, 0, 1300), cache.desc, z, z)
    assert flagged()
    batch.bb.upload(np.asarray(good, np.int32))
    close(attend(cache, batch, q, heads, kv, hd), want, tol)
    assert not flagged()


@pytest.mark.parametrize("kv_type", [F32, F16, Q8])
def test_replays(kv_type):
    """A captured decode step (store, attention) replayed at successive positions beside eager work, two graphs with
    workspaces of their own at once, and the same calls on another stream."""
    heads, kv, hd, steps = 8, 2, 64, 6
    lengths = [700, 2000]
    cache = Cache(kv_type, kv, hd, 64, [n + steps for n in lengths], stale="nan").upload()
    context = 2048
    cos, sin = tables(context, hd // 2)
    cb, sb = dev(cos), dev(sin)
    shape = smq.attn_shape(heads, kv, hd, hd // 2, 0, context)
    batch = Batch(cache, [1, 1], lengths=lengths)
    q = dev(np.zeros(2 * heads * hd, np.float32))
    k, v = (dev(np.zeros(2 * kv * hd, np.float32)) for _ in range(2))
    rot = smq.DeviceBuffer(q.nbytes)
    need = smq.paged_attention_workspace(batch.desc, shape)
    att, ws = ([smq.DeviceBuffer(q.nbytes) for _ in range(3)], [smq.DeviceBuffer(max(16, need)) for _ in range(3)])

    def step(i):
        smq.paged_rope_kv(q, rot, k, v, batch.desc, shape, cb, sb, cache.desc)
        smq.paged_attention(rot, att[i], batch.desc, shape, 0, cache.desc, ws[i])

    graphs = [smq.capture(lambda i=i: step(i)) for i in range(2)]
    side = torch.cuda.Stream()
    for t in range(steps):
        now = np.array([n + t + 1 for n in lengths], np.int32)
        batch.lb.upload(now)
        rows = [synth.normal(200 + 3 * t + i, 2 * w).reshape(2, -1, hd) for i, w in enumerate((heads * hd, kv * hd, kv * hd))]
        for b, x in zip((q, k, v), rows):
            b.upload(x)
        batch.length = now
        for s in range(2):
            cache.put(s, now[s:s + 1] - 1, rotate(rows[1][s:s + 1], cos[now[s:s + 1] - 1], sin[now[s:s + 1] - 1], hd // 2),
                      rows[2][s:s + 1])
        want, tol = attend64(cache, batch, rotate(rows[0], cos[now - 1], sin[now - 1], hd // 2), heads)
        smq.synchronize()
        graphs[0].launch()
        step(2)
        smq.synchronize()
        smq.load().smq_set_stream(side.cuda_stream)
        try:
            graphs[1].launch()
        finally:
            smq.load().smq_set_stream(None)
        graphs[0].launch()
        side.synchronize()
        smq.numeric_check()
        for i in range(3):
            got = att[i].download(np.float32).reshape(want.shape)
            close(got, want, tol, what=f"step {t}, {i}")
            same(got, att[2].download(np.float32).reshape(want.shape))
    smq.load().smq_set_stream(side.cuda_stream)
    try:
        step(1)
        smq.synchronize()
    finally:
        smq.load().smq_set_stream(None)
    same(att[1].download(np.float32), att[2].download(np.float32))
    for g in graphs:
        g.destroy()


def test_offsets_past_32_bits():
    """A Q8 pool of more than 2^32 codes, pages at its end."""
    heads, kv, hd, page = 4, 4, 128, 256
    pages = (1 << 32) // (kv * hd * page) + 8
    shape = smq.attn_shape(heads, kv, hd, 0, 0, 600)
    small = Cache(Q8, kv, hd, page, [600], spare=0)  # the same pages at the end of a large pool
    small.upload()
    k, v = (smq.DeviceBuffer(pages * kv * hd * page) for _ in range(2))
    ks, vs = (smq.DeviceBuffer(pages * kv * 4 * page * 4) for _ in range(2))
    big = smq.paged_kv(k, v, ks, vs, Q8, page, pages)
    small.tb.upload(small.table + pages - 3)
    batch = Batch(small, [600])
    rows = [synth.normal(97 + i, 600 * kv * hd).reshape(600, kv, hd) for i in range(2)]
    small.put(0, np.arange(600), *rows)
    z = dev(np.zeros(1, np.float32))
    smq.paged_rope_kv(None, None, dev(rows[0]), dev(rows[1]), batch.desc, shape, z, z, big)
    rk, rv = (smq.DeviceBuffer(600 * kv * hd * 4) for _ in range(2))
    smq.paged_read(batch.desc, shape, big, rk, rv)
    for b, w in zip((rk, rv), small.rows(0, np.arange(600))):
        same(b.download(np.float32).reshape(w.shape), w)
    one = Batch(small, [2])
    q = synth.normal(99, 2 * heads * hd).reshape(2, heads, hd)
    want, tol = attend64(small, one, q, heads)
    att = smq.DeviceBuffer(q.nbytes)
    smq.paged_attention(dev(q), att, one.desc, shape, 0, big)
    close(att.download(np.float32).reshape(q.shape), want, tol)
    smq.numeric_check()


def test_unaligned_rows():
    """q, k, v and the outputs at 4-byte addresses."""
    heads, kv, hd = 6, 2, 64
    cache = Cache(F16, kv, hd, 32, [70], stale="nan").upload()
    batch = Batch(cache, [21])
    shape = smq.attn_shape(heads, kv, hd, 32, 0, 70)
    cos, sin = tables(70, 32)
    q, k, v = (synth.normal(101 + i, 21 * w).reshape(21, -1, hd) for i, w in enumerate((heads * hd, kv * hd, kv * hd)))
    pos = np.arange(49, 70)
    cache.put(0, pos, rotate(k, cos[pos], sin[pos], 32), v)

    def off(x):
        b = smq.DeviceBuffer(x.nbytes + 4)
        b.upload(x, 4)
        return b

    qb, kb, vb, cb, sb = (off(x) for x in (q, k, v, cos, sin))
    att = smq.DeviceBuffer(q.nbytes + 4)
    smq.paged_rope_kv(qb.at(4), qb.at(4), kb.at(4), vb.at(4), batch.desc, shape, cb.at(4), sb.at(4), cache.desc)
    smq.paged_attention(qb.at(4), att.at(4), batch.desc, shape, 0, cache.desc)
    want, tol = attend64(cache, batch, rotate(q, cos[pos], sin[pos], 32), heads)
    close(att.download(np.float32, offset=4).reshape(q.shape), want, tol)


def test_serving_together():
    """Three conversations through prompt chunks and decode steps: the paged operators against the contiguous cache's
    (smq_rope_kv, smq_attention) with the same tokens, then the rules and the choice on a projection of the result."""
    heads, kv, hd, context, vocab = 6, 2, 64, 160, 500
    plan = [(40, 1, 0), (30, 17, 64), (1, 1, 3), (1, 1, 1), (1, 0, 1)]  # new tokens of each conversation per step
    shape = smq.attn_shape(heads, kv, hd, hd // 2, 0, context)
    total = [sum(p[s] for p in plan) for s in range(3)]
    cos, sin = tables(context, hd // 2)
    cb, sb = dev(cos), dev(sin)
    caches = {t: Cache(t, kv, hd, 16, total, stale="nan").upload() for t in (F32, F16, Q8)}
    flat = [[smq.DeviceBuffer(context * kv * hd * 4) for _ in range(2)] for _ in range(3)]
    head = synth.normal(300, vocab * heads * hd, 0.1).reshape(vocab, heads * hd)
    done, history = [0, 0, 0], [[], [], []]
    for t, new in enumerate(plan):
        n = sum(new)
        q, k, v = (synth.normal(301 + 3 * t + i, n * w).reshape(n, w) for i, w in enumerate((heads * hd, kv * hd, kv * hd)))
        done = [d + x for d, x in zip(done, new)]
        at, want = 0, np.zeros((n, heads * hd), np.float32)
        for s, x in enumerate(new):
            if x:
                qb, kb, vb, ab = dev(q[at:at + x]), dev(k[at:at + x]), dev(v[at:at + x]), smq.DeviceBuffer(x * heads * hd * 4)
                smq.rope_kv(qb, kb, vb, x, shape, cb, sb, *flat[s], pos0=done[s] - x)
                smq.attention(qb, *flat[s], ab, x, shape, pos0=done[s] - x)
                want[at:at + x] = ab.download(np.float32).reshape(x, -1)
            at += x
        for kv_type, cache in caches.items():
            batch = Batch(cache, new, lengths=done)
            qb, att = dev(q), smq.DeviceBuffer(q.nbytes)
            smq.paged_rope_kv(qb, qb, dev(k), dev(v), batch.desc, shape, cb, sb, cache.desc)
            ws = smq.DeviceBuffer(max(16, smq.paged_attention_workspace(batch.desc, shape)))
            smq.paged_attention(qb, att, batch.desc, shape, 0, cache.desc, ws)
            got = att.download(np.float32).reshape(n, -1)
            # f32: both within f32 sums; f16: half a step of 2^-11 of keys and values; Q8: half a step of 1/127 of a
            # block's largest (about 2.5 sigma), scores off by that times |q| sqrt(hd) / sqrt(hd)
            limit = {F32: 2e-5, F16: 4e-3, Q8: 0.1}[kv_type]
            assert np.abs(got - want).max() < limit, (t, TYPES[kv_type], np.abs(got - want).max())
            if kv_type == F32:
                last = [int(x) - 1 for x, m in zip(batch.begin[1:], new)]
                logits = (got[last] @ head.T).astype(np.float32)
        begins = np.concatenate([[0], np.cumsum([len(h) for h in history])]).astype(np.int32)
        flat_ids = np.array([i for h in history for i in h] or [0], np.uint32)
        rules = smq.logit_rules(history=dev(flat_ids), history_begin=dev(begins), history_count=flat_ids.size,
                                penalty=dev(np.tile(np.array([1.5, 0.5, 0.25], np.float32), (3, 1))))
        lb, out, token = dev(logits), smq.DeviceBuffer(logits.nbytes), smq.DeviceBuffer(12)
        smq.logits_adjust(lb, 3, vocab, rules, out, token, smq.DeviceBuffer(smq.logits_workspace(3, vocab)))
        from paged_ref import logits_rules
        for s in range(3):
            w, pick = logits_rules(logits[s], history[s], (1.5, 0.5, 0.25))
            same(out.download(np.float32).reshape(3, vocab)[s], w)
            assert token.download(np.uint32)[s] == pick
            history[s].append(pick)
    smq.numeric_check()


def rows_in_bound(cache, new, heads, window=0, sinks=0, rows=None, padding=0, seed=110, size=1.0):
    """Attention of the batch, cut into pieces and whole, within attend64's own bound in the rows of a mask (all)."""
    batch = Batch(cache, new, padding=padding)
    q = synth.normal(seed, batch.tokens * heads * cache.hd, size).reshape(-1, heads, cache.hd)
    want, tol = attend64(cache, batch, q, heads, window, sinks)
    rows = slice(0, int(batch.begin[-1])) if rows is None else rows
    for split in (True, False):
        got = attend(cache, batch, q, heads, cache.kv, cache.hd, window, sinks, split=split)
        close(got, want, tol, rows, f"split {split}")
    return batch, got, want, tol


Q8_FORMS = [  # heads, kv, hd, page, new of 200 positions
    (8, 2, 64, 32, 1),       # decode
    (4, 2, 96, 16, 3),
    (8, 2, 128, 64, 150),    # rows owned by waves
    (2, 2, 64, 16, 150),
    (6, 1, 160, 64, 40),
]


@pytest.mark.parametrize("heads,kv,hd,page,new", Q8_FORMS)
@pytest.mark.parametrize("scale", [1e-6, 1e-8, 1e-10, 1e-20])
def test_q8_values_after_a_block_of_zeros(heads, kv, hd, page, new, scale):
    """A step whose values are all zero in one block of 32 dims says nothing of that block's size: neither before its first
    values nor between them, while the other blocks have ordinary ones."""
    say("q8 zeros", heads, kv, hd, page, new, scale)
    for zeros in (slice(0, 32), slice(0, 64), slice(64, 96)):
        cache = Cache(Q8, kv, hd, page, [200], stale="nan")
        pg, sl = cache.slots(0, np.arange(200))
        cache.vs[pg, :, 1, sl] *= np.float32(scale)
        pg, sl = cache.slots(0, np.arange(200)[zeros])
        cache.vs[pg, :, 1, sl] = 0.0
        rows_in_bound(cache.upload(), [new], heads)
    smq.numeric_check()


@pytest.mark.parametrize("heads,kv,hd,page,new", Q8_FORMS[2:] + [(16, 1, 32, 128, 2), (3, 1, 256, 32, 50)])
@pytest.mark.parametrize("ratio", [1e6, 2.0 ** 40, 1e30, 3e38])
def test_q8_scales_that_a_row_does_not_see(heads, kv, hd, page, new, ratio):
    """Values of a chunk's last token, and of a position that the window has left, far larger than all others: the rows
    that do not see them keep their own accuracy, and the rows that do are off by no more than the documented rounding."""
    say("q8 unseen scales", heads, kv, hd, page, new, ratio)
    n, first = 200, 200 - new
    for window, sinks, large in ((0, 0, [n - 1]), (0, 0, [n - 2, n - 1]), (20, 0, [first - 10]), (20, 3, [first - 19, n - 1]),
                                 (40, 2, [first - 5, first + new // 2])):
        cache = Cache(Q8, kv, hd, page, [n], stale="nan")
        pg, sl = cache.slots(0, large)
        cache.vs[pg, 0, 1 % cache.nb, sl] = np.float32(min(ratio * 0.01, 3e38))
        cache.upload()
        pos = np.arange(first, n)
        sees = np.array([np.isin(large, visible(p, window, sinks)).any() for p in pos])
        batch, got, want, tol = rows_in_bound(cache, [new], heads, window, sinks, ~sees)
        if ratio > 1e38:  # a code of 2 is past f32 there
            continue
        # half a step of f16's subnormals, 2^-25, per weight of at most twice the largest scale's power of two; 127 is the
        # largest code but one, the row's largest weight at least 2^6
        v = float(cache.vs[pg, 0, 1 % cache.nb, sl].max())
        close(got, want, tol + n * 2.0 ** -25 * 2 * v * 128 / 2 ** 6, sees)
    smq.numeric_check()


LARGE = [  # heads, kv, hd, page, lengths, new, window, sinks
    (4, 2, 64, 32, [1, 2, 40], [1, 1, 1], 0, 0),
    (8, 2, 64, 64, [5000, 3001, 64], [1, 1, 1], 0, 0),       # cut into pieces
    (4, 2, 128, 16, [150], [150], 0, 0),                     # rows owned by waves
    (4, 1, 48, 64, [1500, 90], [1, 90], 33, 2),
    (2, 1, 256, 32, [100], [60], 0, 0),
]


@pytest.mark.parametrize("kv_type", [F32, Q8])
@pytest.mark.parametrize("size", [3e38, 1e36, 1e33, 1e-30])
@pytest.mark.parametrize("heads,kv,hd,page,lengths,new,window,sinks", LARGE)
def test_values_near_the_ends_of_f32(kv_type, size, heads, kv, hd, page, lengths, new, window, sinks):
    """Finite values give finite results: averages of values up to f32's largest, and of tiny ones."""
    say("paged values", TYPES[kv_type], size, heads, kv, hd, page, lengths, new, window, sinks)
    cache = Cache(kv_type, kv, hd, page, lengths, stale=None)
    rng = np.random.default_rng(7)
    if kv_type == Q8:
        cache.v = np.clip(cache.v, -127, 127)
        cache.vs = (size / 127 * rng.uniform(0.25, 1, cache.vs.shape)).astype(np.float32)
    else:
        cache.v = (size * rng.uniform(-1, 1, cache.v.shape)).astype(np.float32)
    rows_in_bound(cache.upload(), new, heads, window, sinks, seed=111, size=0.3)
    smq.numeric_check()


@pytest.mark.parametrize("kv_type", [F32, Q8])
def test_values_of_one_sign_near_the_largest(kv_type):
    """All values alike: the average is the value, however many positions and pieces."""
    heads, kv, hd = 8, 2, 64
    for lengths, new in (([4000, 1, 130], [1, 1, 1]), ([300], [150])):
        cache = Cache(kv_type, kv, hd, 64, lengths, stale=None)
        if kv_type == Q8:
            cache.v[:] = 127
            cache.vs[:] = np.float32(3.3e38 / 127)
        else:
            cache.v[:] = np.float32(-3.3e38)
        rows_in_bound(cache.upload(), new, heads, seed=112, size=0.3)


WIDE_CHUNKS = [  # heads, kv, hd, page, lengths, new, window, sinks
    (4, 2, 256, 16, [90, 64], [90, 33], 0, 0),
    (4, 1, 256, 64, [300], [70], 0, 0),
    (8, 2, 144, 16, [100, 40], [64, 40], 0, 0),
    (8, 2, 144, 128, [150], [100], 31, 2),
    (2, 2, 192, 32, [130, 77], [130, 50], 0, 0),
    (6, 2, 208, 16, [200], [90], 50, 3),
    (3, 1, 240, 256, [280], [40], 0, 0),
    (4, 4, 256, 32, [5000, 40], [40, 40], 0, 0),             # cut into pieces
]


@pytest.mark.parametrize("kv_type", [F32, F16, Q8])
@pytest.mark.parametrize("heads,kv,hd,page,lengths,new,window,sinks", WIDE_CHUNKS)
def test_chunks_of_wide_heads(kv_type, heads, kv, hd, page, lengths, new, window, sinks):
    """Heads above 128 where waves own rows (more than 32 rows a sequence and KV head), over pages of 16 and larger ones."""
    say("paged attention, wide heads", TYPES[kv_type], heads, kv, hd, page, lengths, new, window, sinks)
    assert sum(new) * heads // kv > 32 * len(new)
    cache = Cache(kv_type, kv, hd, page, lengths, stale="nan")
    for s, (m, n) in enumerate(zip(lengths, new)):
        if window:
            low = m - n + 1 - window
            cache.spoil_positions(s, np.arange(min(sinks, low), low) if low > sinks else np.zeros(0, int))
    batch, got, _, _ = rows_in_bound(cache.upload(), new, heads, window, sinks, padding=2, seed=113, size=1.5)
    assert (got[int(batch.begin[-1]):] == 9.0).all()
    smq.numeric_check()


@pytest.mark.parametrize("kv_type", [F32, F16, Q8])
@pytest.mark.parametrize("hd", [144, 176, 208, 240])
def test_decode_of_wide_heads(kv_type, hd):
    """Head sizes between 128 and 256 whose last block or last 32 dims are not whole."""
    for page in (16, 64):
        cache = Cache(kv_type, 2, hd, page, [700, 33, 1], stale="nan").upload()
        rows_in_bound(cache, [1, 3, 1], 6, seed=114, size=1.5)
    smq.numeric_check()


@pytest.mark.parametrize("kv_type", [F32, F16, Q8])
@pytest.mark.parametrize("heads,kv,hd,page,new", Q8_FORMS)
def test_weights_far_below_the_largest(kv_type, heads, kv, hd, page, new):
    """A first position that takes nearly the whole weight and whose values are 0: what the others leave is off by f32's
    rounding and, where the cache is not f32, by 2^-31 of the largest weight for each of them (half a step of f16, 2^-25, in
    units where the largest is above 2^6)."""
    say("weights far apart", TYPES[kv_type], heads, kv, hd, page, new)
    n = 200
    for power in (4.0, 9.0, 14.0):  # the others' weights, about 2^-power of the first one's
        cache = Cache(kv_type, kv, hd, page, [n], stale="nan")
        pg, sl = cache.slots(0, [0])
        cache.k[pg, :, sl] = 127 if kv_type == Q8 else 1
        cache.v[pg, :, sl] = 0
        if kv_type == Q8:
            cache.ks[pg, :, :, sl] = 1 / 127
        cache.upload()
        batch = Batch(cache, [new])
        q = synth.normal(115, new * heads * hd, 0.3).reshape(-1, heads, hd)
        q += np.float32(power * np.log(2) / np.sqrt(hd))  # q . 1 / sqrt(hd): power in units of log 2, beside the rest
        want, tol = attend64(cache, batch, q, heads)
        if kv_type != F32:
            for i, p in enumerate(range(n - new, n)):
                _, v = cache.rows(0, np.arange(p + 1), np.float64)
                big = np.abs(v).max(0)
                if kv_type == Q8:  # 127 codes of the block's largest scale
                    pg, sl = cache.slots(0, np.arange(p + 1))
                    big = np.repeat(cache.vs[pg, :, :, sl].max(0).astype(np.float64), 32, -1)[:, :hd] * 128
                tol[i] += (p + 1) * 2.0 ** -31 * np.repeat(big, heads // kv, 0)
        for split in (True, False):
            close(attend(cache, batch, q, heads, kv, hd, split=split), want, tol, what=f"2^-{power}")
    smq.numeric_check()
