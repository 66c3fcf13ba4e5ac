"""Cases of tests/test_paged_host.py, each in a process of its own: paged_host_cases.py FAKE_HIP_LIBRARY CASE. Refusals and
empty calls of the paged cache and the logits' rules over the recording runtime of tests/fake_hip.cpp, without a GPU."""
import ctypes
import os
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, HERE)
fake = smq = None
RANGE = 4


def load(path):
    global fake, smq
    fake = ctypes.CDLL(path, mode=ctypes.RTLD_GLOBAL)
    fake.fake_log.restype = fake.fake_errors.restype = ctypes.c_char_p
    from smq_pkg import smq as package
    smq = package
    smq.init(0)


def launches():
    n = len(fake.fake_log().decode().splitlines())
    fake.fake_clear()
    return n


def refused(f, *args, words=""):
    fake.fake_clear()
    try:
        f(*args)
    except smq.SmqError as e:
        assert e.status == RANGE and words in str(e), e
        assert launches() == 0
        return
    raise AssertionError(("not refused", f.__name__, words))


class Paged:
    """A valid call's arguments; keyword arguments change descriptors or buffer sizes."""

    def __init__(self, **kw):
        self.o = dict(heads=4, kv=2, hd=64, pairs=32, window=0, context=256, type=2, page=32, pages=20, seqs=3, tokens=9,
                      stride=8, short=None)
        self.o.update(kw)
        o, short = self.o, kw.get("short")
        one = {0: 4, 1: 2, 2: 1}.get(o["type"], 4)
        positions, nb = o["pages"] * o["page"], (o["hd"] + 31) // 32
        size = {"keys": positions * o["kv"] * o["hd"] * one, "ks": positions * o["kv"] * nb * 4,
                "begin": 4 * (o["seqs"] + 1), "length": 4 * o["seqs"], "table": 4 * o["seqs"] * o["stride"],
                "q": 4 * o["tokens"] * o["heads"] * o["hd"], "k": 4 * o["tokens"] * o["kv"] * o["hd"],
                "cos": 4 * o["context"] * o["pairs"]}
        size.update(values=size["keys"], vs=size["ks"], q_out=size["q"], v=size["k"], sin=size["cos"], att=size["q"],
                    rk=size["k"], rv=size["k"])
        if short:
            size[short] -= 1
        self.b = {n: smq.DeviceBuffer(max(1, s)) for n, s in size.items()}
        self.shape = smq.attn_shape(o["heads"], o["kv"], o["hd"], o["pairs"], o["window"], o["context"])
        self.batch = smq.paged_batch(self.b["begin"], self.b["length"], self.b["table"], o["seqs"], o["tokens"], o["stride"])
        self.kv = smq.paged_kv(self.b["keys"], self.b["values"], self.b["ks"], self.b["vs"], o["type"], o["page"], o["pages"])
        need = smq.load().smq_paged_attention_workspace(self.batch, self.shape)
        smq.load().smq_clear_error()
        self.ws = smq.DeviceBuffer(need + 16)

    def store(self, **kw):
        b = dict(self.b, **kw)
        smq.paged_rope_kv(b["q"], b["q_out"], b["k"], b["v"], self.batch, self.shape, b["cos"], b["sin"], self.kv)

    def read(self):
        smq.paged_read(self.batch, self.shape, self.kv, self.b["rk"], self.b["rv"])

    def attend(self, ws=None, n=0):
        smq.paged_attention(self.b["q"], self.b["att"], self.batch, self.shape, 0, self.kv, ws or self.ws, n or 0)


def valid_calls():
    for kv_type in (0, 1, 2):
        for hd in (16, 64, 80, 256):
            for page in (16, 32, 64, 128, 256):
                p = Paged(type=kv_type, hd=hd, pairs=hd // 2, page=page)
                for f in (p.store, p.read, p.attend):
                    fake.fake_clear()
                    f()
                    assert launches() >= 1
    p = Paged()
    p.store(q=None, q_out=None)
    smq.paged_attention(p.b["q"], p.b["att"], p.batch, p.shape, 0, p.kv)  # no workspace


def empty_batches():
    for kw in (dict(seqs=0), dict(tokens=0), dict(seqs=0, tokens=0, stride=0)):
        p = Paged(**kw)
        fake.fake_clear()
        p.store()
        p.read()
        p.attend()
        assert launches() == 0
    # nothing of an empty batch is looked at
    empty = smq.paged_batch(None, None, None, 0, 0, 0)
    smq.paged_attention(None, None, empty, p.shape, 0, p.kv)
    assert launches() == 0


def shapes():
    for kw in (dict(hd=8, pairs=4), dict(hd=24, pairs=12), dict(hd=272, pairs=8), dict(hd=0, pairs=0), dict(heads=0),
               dict(heads=5), dict(kv=0), dict(pairs=33), dict(context=0, pairs=0), dict(context=(1 << 20) + 1, pairs=0),
               dict(page=8), dict(page=48), dict(page=512), dict(page=0), dict(type=3), dict(pages=0), dict(stride=0)):
        p = Paged(**kw)
        for f in (p.store, p.read, p.attend):
            refused(f)
    p = Paged()
    for field, value in (("seqs", (1 << 20) + 1), ("tokens", (1 << 24) + 1), ("table_stride", (1 << 20) + 1)):
        q = Paged()
        setattr(q.batch, field, value)
        for f in (q.store, q.read, q.attend):
            refused(f, words="unsupported batch")
    p.kv.pages = 0xFFFFFFFF
    refused(p.attend, words="unsupported cache")
    # as many tokens times heads as fit, one more, and pools past the address space
    p = Paged()
    p.batch.tokens = (1 << 20) + 1
    for f in (p.store, p.read, p.attend):
        refused(f, words="unsupported batch")
    p.batch.tokens = 1 << 20
    refused(p.attend, words="q")
    p = Paged(heads=65535, kv=65535, hd=256, pairs=0, type=0, page=16, pages=1, seqs=1, tokens=1, stride=1, context=16)
    p.kv.pages, p.kv.page_size = 0x7FFFFFFF, 256
    for f in (p.store, p.read, p.attend):
        refused(f, words="past the address space")


def buffers():
    for name, calls in {"keys": "sra", "values": "sra", "ks": "sra", "vs": "sra", "begin": "sra", "length": "sra",
                        "table": "sra", "q": "sa", "q_out": "s", "k": "s", "v": "s", "cos": "s", "sin": "s", "att": "a",
                        "rk": "r", "rv": "r"}.items():
        p = Paged(short=name)
        for c in calls:
            refused({"s": p.store, "r": p.read, "a": p.attend}[c], words="exceed its allocation")
    for field in ("begin", "length", "table"):
        p = Paged()
        setattr(p.batch, field, None)
        for f in (p.store, p.read, p.attend):
            refused(f, words="NULL")
    for field in ("keys", "values", "key_scales", "value_scales"):
        p = Paged()
        setattr(p.kv, field, None)
        refused(p.attend, words="NULL")
        q = Paged(pages=30)
        setattr(q.kv, field, getattr(q.kv, field) + 4)
        q.kv.pages = 20
        refused(q.attend, words="aligned")
    Paged(type=1).attend()
    p = Paged(type=1)
    p.kv.key_scales = p.kv.value_scales = None  # only Q8 has them
    p.attend()
    p = Paged()
    refused(lambda: p.store(q=None), words="q_out without q")
    refused(lambda: p.store(q_out=None), words="q without q_out")
    refused(lambda: p.store(k=None), words="NULL")
    refused(lambda: p.attend(p.ws.at(4), 16), words="aligned")
    refused(lambda: p.attend(p.ws.at(0), p.ws.nbytes + 16), words="exceed its allocation")
    lib = smq.load()
    for call in (lambda: lib.smq_paged_rope_kv(None, None, None, None, None, p.shape, None, None, p.kv),
                 lambda: lib.smq_paged_read(p.batch, None, p.kv, None, None),
                 lambda: lib.smq_paged_read(p.batch, p.shape, None, None, None),
                 lambda: lib.smq_paged_attention(None, None, p.batch, p.shape, 0, None, None, 0)):
        assert call() == RANGE
        lib.smq_clear_error()
    assert lib.smq_paged_attention_workspace(None, p.shape) == 0
    lib.smq_clear_error()


def captures():
    """Every call may be captured and allocates nothing there."""
    p = Paged()
    before = fake.fake_errors()
    g = smq.capture(lambda: (p.store(), p.read(), p.attend()))
    fake.fake_clear()
    g.launch()
    assert launches() >= 3 and fake.fake_errors() == before == b""
    g.destroy()


def logits():
    rows, vocab = 5, 4099
    words = (vocab + 31) // 32
    size = dict(logits=rows * vocab * 4, out=rows * vocab * 4, token=rows * 4, history=400, history_begin=24, penalty=60,
                bias_ids=80, bias=80, bias_begin=24, allowed=3 * words * 4, mask_row=20,
                ws=smq.logits_workspace(rows, vocab))
    assert 0 < size["ws"] < 1 << 20

    def call(short=None, stride=None, out_stride=None, out=True, token=True, n=rows, v=vocab, ws_bytes=None, **kw):
        b = {k: smq.DeviceBuffer(x - (k == short)) for k, x in size.items()}
        r = smq.logit_rules(b["history"], b["history_begin"], 100, b["penalty"], b["bias_ids"], b["bias"], b["bias_begin"], 20,
                            b["allowed"], 3, b["mask_row"])
        for k, x in kw.items():
            setattr(r, k, x)
        fake.fake_clear()
        smq.logits_adjust(b["logits"], n, v, r, b["out"] if out else None, b["token"] if token else None, b["ws"],
                          size["ws"] if ws_bytes is None else ws_bytes, stride, out_stride)
        return launches()

    assert call() >= 1
    assert call(out=False) >= 1 and call(token=False, ws_bytes=0) >= 1
    assert call(n=0) == 0
    for name in size:
        refused(call, name, words="exceed its allocation")
    for kw in (dict(history_begin=None), dict(penalty=None), dict(bias=None), dict(bias_begin=None)):
        refused(lambda: call(**kw), words="NULL")
    refused(lambda: call(mask_row=None), words="3 masks for 5 rows")
    refused(lambda: call(out=False, token=False), words="neither")
    refused(lambda: call(v=0), words="vocabulary")
    refused(lambda: call(v=(1 << 30) + 1), words="vocabulary")
    refused(lambda: call(n=65536), words="rows")
    refused(lambda: call(stride=vocab - 1), words="strides")
    refused(lambda: call(out_stride=vocab - 1), words="strides")
    refused(lambda: call(ws_bytes=size["ws"] - 1), words="workspace")
    b = smq.DeviceBuffer(rows * (vocab + 1) * 4)
    ws = smq.DeviceBuffer(size["ws"] + 16)
    refused(lambda: smq.logits_adjust(b, rows, vocab, None, b, None, stride=vocab, out_stride=vocab + 1), words="in place")
    refused(lambda: smq.logits_adjust(b, rows, vocab, None, b, smq.DeviceBuffer(20), ws.at(4), size["ws"]), words="aligned")
    refused(lambda: smq.logits_adjust(None, rows, vocab, None, b, None), words="NULL")


CASES = [f for f in (valid_calls, empty_batches, shapes, buffers, captures, logits)]


def grids():
    g = [line.split(" grid ")[1].split()[0] for line in fake.fake_log().decode().splitlines()]
    fake.fake_clear()
    return g


def widest_split():
    """The bytes that the workspace query gives make the launches that boundless ones would, whatever sinks and table the call
    brings: the query knows neither."""
    cut = 0
    for heads, kv, hd, seqs, new, window, context in (
            (32, 4, 64, 8, 1, 64, 5000), (32, 8, 128, 1, 1, 512, 131072), (14, 2, 64, 3, 1, 1000, 32768),
            (4, 1, 64, 1, 1, 16, 1 << 20), (8, 2, 128, 2, 300, 200, 9000), (32, 8, 128, 6, 64, 33, 60000),
            (8, 2, 256, 1, 100, 0, 4000), (4, 1, 64, 1, 1, 0, 1 << 20)):
        p = Paged(heads=heads, kv=kv, hd=hd, pairs=0, type=1, page=64, pages=1, seqs=seqs, tokens=seqs * new,
                  stride=-(-context // 64), window=window, context=context)
        need = smq.load().smq_paged_attention_workspace(p.batch, p.shape)
        large = smq.DeviceBuffer(max(4 * need, 1 << 28))
        for sinks in (0, 1, 100, 4000, context - 500, context, 0xFFFFFFFF):
            for stride in (p.o["stride"], p.o["stride"] - 1, p.o["stride"] // 2 + 1):
                p.batch.table_stride = stride
                got = []
                for n in (large.nbytes, need):
                    fake.fake_clear()
                    smq.paged_attention(p.b["q"], p.b["att"], p.batch, p.shape, sinks, p.kv, large.at(0), n)
                    got.append(grids())
                assert got[0] == got[1], (heads, kv, hd, seqs, new, window, context, sinks, stride, need, got)
                cut += len(got[0]) == 2
    assert cut > 50


def logits_past_the_address_space():
    """Row strides whose product with the rows wraps around: refused, not taken for a few bytes."""
    rows, vocab = 3, 1000
    logits, out, token, ws = (smq.DeviceBuffer(n) for n in (rows * vocab * 4, rows * vocab * 4, rows * 4,
                                                            smq.logits_workspace(rows, vocab)))

    def call(stride, out_stride, to=out):
        smq.logits_adjust(logits, rows, vocab, None, to, token, ws, ws.nbytes, stride, out_stride)

    call(vocab, vocab)
    for stride in (1 << 61, (1 << 61) + vocab, 1 << 62, (1 << 63) + 1, (1 << 64) - 1):
        refused(lambda: call(stride, vocab), words="address space")
        refused(lambda: call(vocab, stride), words="address space")
        refused(lambda: call(stride, vocab, None), words="address space")
        refused(lambda: call(stride, stride, logits), words="address space")
    refused(lambda: call(1 << 60, vocab), words="exceed its allocation")
    # of one row the stride is not looked at
    fake.fake_clear()
    smq.logits_adjust(logits, 1, vocab, None, out, token, ws, ws.nbytes, (1 << 64) - 1, 1 << 62)
    assert launches() >= 1


def logits_workspace_of_the_largest_batch():
    """A workspace for the most rows and ids serves every call of fewer: a batch that shrinks is not refused."""
    for rows, vocab in ((64, 151936), (16, 151936), (14, 151936), (13, 151936), (342, 4099), (341, 4099), (1, 3_000_000)):
        have = smq.logits_workspace(rows, vocab)
        b, token = smq.DeviceBuffer(rows * vocab * 4), smq.DeviceBuffer(rows * 4)
        ws = smq.DeviceBuffer(have)
        for n in sorted({1, rows // 2, rows - 3, rows - 1, rows, 13, 14} & set(range(1, rows + 1))):
            for v in sorted({vocab, vocab - 1, vocab * 9 // 10, vocab // 2, 2049, 1024, 5} & set(range(1, vocab + 1))):
                assert smq.logits_workspace(n, v) <= have, (rows, vocab, n, v)
                smq.logits_adjust(b, n, v, None, b, token, ws, have)


CASES += [widest_split, logits_past_the_address_space, logits_workspace_of_the_largest_batch]

if __name__ == "__main__":
    load(sys.argv[1])
    {f.__name__: f for f in CASES}[sys.argv[2]]()
    print("ok")
