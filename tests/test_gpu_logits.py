"""Penalties, biases, masks and the choice on rows of logits, bit for bit against numpy (tests/paged_ref.py)."""
import numpy as np
import pytest
import torch

from checks import assert_same_f32, say
from paged_ref import logits_rules
from smq_pkg import smq, synth

pytestmark = pytest.mark.gpu
dev = smq.DeviceBuffer.from_array


@pytest.fixture(scope="module", autouse=True)
def gpu():
    assert smq.init(0) == "gfx950"
    yield


def pack(masks):
    """[rows, vocab] bool -> words."""
    rows, vocab = masks.shape
    bits = np.zeros((rows, (vocab + 31) // 32 * 32), np.uint64)
    bits[:, :vocab] = masks
    return (bits.reshape(rows, -1, 32) << np.arange(32, dtype=np.uint64)).sum(-1).astype(np.uint32)


class Rules:
    """Lists per row (history ids, (bias ids, values), mask or None) in device memory."""

    def __init__(self, vocab, history=None, penalty=None, bias=None, masks=None):
        kw = {}
        if history is not None:
            flat = np.concatenate([np.asarray(h, np.uint32) for h in history] + [np.zeros(1, np.uint32)])
            begin = np.concatenate([[0], np.cumsum([len(h) for h in history])]).astype(np.int32)
            kw.update(history=dev(flat), history_begin=dev(begin), history_count=int(begin[-1]),
                      penalty=dev(np.asarray(penalty, np.float32)))
        if bias is not None:
            ids = np.concatenate([np.asarray(b[0], np.uint32) for b in bias] + [np.zeros(1, np.uint32)])
            val = np.concatenate([np.asarray(b[1], np.float32) for b in bias] + [np.zeros(1, np.float32)])
            begin = np.concatenate([[0], np.cumsum([len(b[0]) for b in bias])]).astype(np.int32)
            kw.update(bias_ids=dev(ids), bias=dev(val), bias_begin=dev(begin), bias_count=int(begin[-1]))
        if masks is not None:
            have = [m for m in masks if m is not None]
            index = np.cumsum([m is not None for m in masks]) - 1
            index = np.where([m is not None for m in masks], index, -1).astype(np.int32)
            kw.update(allowed=dev(pack(np.stack(have)) if have else np.zeros(1, np.uint32)), allowed_rows=len(have),
                      mask_row=dev(index))
        self.c = smq.logit_rules(**kw)


def check(logits, rules, wants, stride=None, in_place=False, offset=0):
    rows, vocab = logits.shape
    stride = stride or vocab
    host = np.full(rows * stride + offset // 4, 3.0, np.float32)
    at = offset // 4
    for r in range(rows):
        host[at + r * stride:at + r * stride + vocab] = logits[r]
    lb = dev(host)
    out = lb if in_place else dev(np.full(host.size, 3.0, np.float32))
    token = dev(np.full(rows + 1, 77, np.uint32))
    ws = smq.DeviceBuffer(smq.logits_workspace(rows, vocab))
    ws.fill(0xFF)
    smq.logits_adjust(lb.at(offset), rows, vocab, rules.c if rules else None, out.at(offset), token, ws, ws.nbytes,
                      stride=stride, out_stride=stride)
    got, tok = out.download(np.float32), token.download(np.uint32)
    want = np.full(host.size, 3.0, np.float32)
    for r, (w, _) in enumerate(wants):
        want[at + r * stride:at + r * stride + vocab] = w
    assert_same_f32(got, want)
    assert list(tok) == [t for _, t in wants] + [77]
    if not in_place:
        assert_same_f32(lb.download(np.float32), host)
        # the tokens alone
        only = dev(np.zeros(rows, np.uint32))
        smq.logits_adjust(lb.at(offset), rows, vocab, rules.c if rules else None, None, only, ws, ws.nbytes, stride=stride)
        assert list(only.download(np.uint32)) == [t for _, t in wants]


@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 33), (2, 1000), (5, 1023), (4, 1024), (3, 1025), (2, 4099), (9, 32000),
                                        (1, 151936), (7, 20000), (70, 5001),
                                        (260, 4099)])  # the last one in spans of 4096 ids
def test_all_rules(rows, vocab):
    say("logits", rows, vocab)
    rng = np.random.default_rng(rows * vocab)
    logits = synth.normal(400, rows * vocab, 4.0).reshape(rows, vocab)
    history = [rng.integers(0, vocab, n) for n in rng.integers(0, 3000, rows)]
    history[0] = np.concatenate([history[0], np.full(300, vocab - 1), [vocab, 0xFFFFFFFF, vocab + 7]])  # ids of no token
    penalty = np.stack([rng.uniform(0.7, 1.6, rows), rng.uniform(-1, 1, rows), rng.uniform(-0.2, 0.5, rows)], 1)
    bias = [(rng.integers(0, vocab + 1, n), rng.standard_normal(n) * 3) for n in rng.integers(0, 40, rows)]
    masks = [None if r % 3 == 1 else rng.random(vocab) < 0.1 for r in range(rows)]
    if rows > 3:
        masks[3] = np.zeros(vocab, bool)  # nothing may be taken
    wants = [logits_rules(logits[r], history[r], penalty[r], bias[r], masks[r]) for r in range(rows)]
    rules = Rules(vocab, history, penalty, bias, masks)
    check(logits, rules, wants)
    check(logits, rules, wants, stride=vocab + 3, offset=4)  # rows at 4-byte addresses
    check(logits, rules, wants, stride=(vocab + 3) // 4 * 4, in_place=True)
    smq.numeric_check()
    check(logits, None, [logits_rules(logits[r]) for r in range(rows)])
    for part in ({"history": history, "penalty": penalty}, {"bias": bias}, {"masks": masks}):
        want = [logits_rules(logits[r], *[part[k][r] if k in part else None for k in ("history", "penalty", "bias", "masks")])
                for r in range(rows)]
        check(logits, Rules(vocab, **part), want)


def test_the_same_id_many_times():
    """Thousands of history entries and biases on few ids, sums in the order of the list, the same on every run."""
    vocab = 3000
    logits = synth.normal(401, vocab).reshape(1, vocab)
    rng = np.random.default_rng(3)
    ids, vals = rng.integers(0, 5, 1500) * 511, rng.standard_normal(1500).astype(np.float32)
    history = np.concatenate([np.full(70000, 2), np.full(5, 2044), np.full(1, 999)])
    want = logits_rules(logits[0], history, (1.1, 0.1, 1e-4), (ids, vals))
    for _ in range(3):
        check(logits, Rules(vocab, [history], [(1.1, 0.1, 1e-4)], [(ids, vals)]), [want])


def test_ties_nan_and_infinities():
    vocab = 5000
    rows = np.zeros((8, vocab), np.float32)
    rows[0, [4000, 900]] = 5.0                 # a tie: the lowest id
    rows[1, 0] = np.nan                        # a NaN first candidate wins
    rows[2, [1, 4999]] = np.nan                # a later one never does
    rows[3] = -np.inf                          # all the same: the first
    rows[4] = np.nan
    rows[5, 77] = np.inf
    rows[6] = -0.0
    rows[6, 3000] = 0.0                        # equal: not strictly greater
    rows[7, :] = -np.inf
    rows[7, 0:2000] = np.nan
    masks = [None] * 8
    masks[7] = np.arange(vocab) >= 1500        # the first that may be taken is a NaN
    check(rows, Rules(vocab, masks=masks), [logits_rules(rows[r], masks=masks[r]) for r in range(8)])
    # penalties on infinities and zeros, a bias that bans
    h = [[0, 1, 4999]] * 8
    p = [(1.3, 0.2, 0.1)] * 8
    b = [([900, 0], [-np.inf, 1.0])] * 8
    check(rows, Rules(vocab, h, p, b), [logits_rules(rows[r], h[r], p[r], b[r]) for r in range(8)])


def test_mask_rows_out_of_range_and_lists_past_their_end():
    vocab = 100
    logits = synth.normal(402, 3 * vocab).reshape(3, vocab)
    rules = Rules(vocab, masks=[np.arange(vocab) % 2 == 0, None, None])
    keep = dev(np.array([0, 1, -5], np.int32))
    rules.c.mask_row = keep.ptr
    check_rows = [logits_rules(logits[0], masks=np.arange(vocab) % 2 == 0), logits_rules(logits[1], masks=np.zeros(vocab, bool)),
                  logits_rules(logits[2])]
    check(logits, rules, check_rows)
    with pytest.raises(smq.SmqError) as e:
        smq.numeric_check()
    assert e.value.status == smq.SM_ERR_NUMERIC
    # begins past the lists, descending and negative: cut to the lists
    hist = Rules(vocab, [[1, 2, 3], [4], [5, 6]], [(2.0, 0.0, 0.0)] * 3)
    begin = dev(np.array([-7, 2, 1, 1 << 30], np.int32))
    hist.c.history_begin = begin.ptr
    wants = [logits_rules(logits[0], [1, 2], (2.0, 0, 0)), logits_rules(logits[1]),
             logits_rules(logits[2], [2, 3, 4, 5, 6], (2.0, 0, 0))]
    check(logits, hist, wants)
    smq.numeric_check()


def test_replays_and_streams():
    vocab, rows = 30000, 4
    rng = np.random.default_rng(9)
    logits = [synth.normal(410 + i, rows * vocab, 3.0).reshape(rows, vocab) for i in range(3)]
    history = [rng.integers(0, vocab, 500) for _ in range(rows)]
    rules = Rules(vocab, history, [(1.2, 0.3, 0.1)] * rows)
    bufs = [(dev(l), smq.DeviceBuffer(l.nbytes), smq.DeviceBuffer(4 * rows), smq.DeviceBuffer(smq.logits_workspace(rows, vocab)))
            for l in logits]
    wants = [[logits_rules(l[r], history[r], (1.2, 0.3, 0.1)) for r in range(rows)] for l in logits]

    def run(i):
        lb, out, token, ws = bufs[i]
        smq.logits_adjust(lb, rows, vocab, rules.c, out, token, ws)

    graphs = [smq.capture(lambda i=i: run(i)) for i in range(2)]
    side = torch.cuda.Stream()
    for _ in range(5):
        for b in bufs:
            b[1].fill(0)
            b[2].fill(0)
        smq.synchronize()
        graphs[0].launch()
        run(2)
        smq.load().smq_set_stream(side.cuda_stream)
        try:
            graphs[1].launch()
        finally:
            smq.load().smq_set_stream(None)
        side.synchronize()
        smq.synchronize()
        for b, want in zip(bufs, wants):
            assert_same_f32(b[1].download(np.float32), np.concatenate([w for w, _ in want]))
            assert list(b[2].download(np.uint32)) == [t for _, t in want]
    for g in graphs:
        g.destroy()


@pytest.mark.parametrize("rows,vocab", [(341, 4099), (342, 4099), (64, 32769), (512, 2049), (1030, 5)])
def test_all_rules_on_both_sides_of_the_span_rule(rows, vocab):
    """Spans of 2048 ids from 1024 workgroups on, of 1024 below (341 x 3 spans are 1023, and the largest batch of
    test_all_rules has 780): rows of several spans, of one and a bit, and of less than one, aligned, at 4-byte addresses
    and in place."""
    say("logits, spans", rows, vocab)
    test_all_rules(rows, vocab)


def test_special_values_and_long_lists_in_spans_of_2048():
    """Ties over threads, waves and spans, NaN and infinities, thousands of entries on few ids, in 352 rows of three spans."""
    vocab, rows = 5000, 352
    logits = np.zeros((rows, vocab), np.float32)
    logits[0::8, 4500] = logits[0::8, 2100] = logits[0::8, 2047] = 5.0
    logits[1::8, 0] = np.nan
    logits[2::8, 1] = logits[2::8, 4999] = np.nan
    logits[3::8] = -np.inf
    logits[4::8] = np.nan
    logits[5::8, 4097] = np.inf
    logits[6::8] = -0.0
    logits[6::8, 3000] = 0.0
    logits[7::8] = -np.inf
    logits[7::8, :3000] = np.nan
    masks = [np.arange(vocab) >= 2500 if r % 8 == 7 else None for r in range(rows)]
    plain = [logits_rules(logits[r], masks=masks[r]) for r in range(8)]
    check(logits, Rules(vocab, masks=masks), [plain[r % 8] for r in range(rows)])
    rng = np.random.default_rng(5)
    ids, vals = rng.integers(0, 5, 900) * 1020, rng.standard_normal(900).astype(np.float32)
    h, p = np.concatenate([np.full(6000, 2047), np.full(5, 2048), [0, 1, 4999]]), (1.3, 0.2, 0.001)
    want = [logits_rules(logits[r], h, p, (ids, vals), masks[r]) for r in range(8)]
    check(logits, Rules(vocab, [h] * rows, [p] * rows, [(ids, vals)] * rows, masks), [want[r % 8] for r in range(rows)])
