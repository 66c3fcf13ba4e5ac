"""Plain numpy restatement of the paged KV cache, its attention (64 bits) and the logits' rules, and a paged cache in
device memory with its numpy image."""
import numpy as np

from smq_pkg import smq

F32, F16, Q8 = 0, 1, 2
NP = {F32: np.float32, F16: np.float16, Q8: np.int8}


def tables(context, pairs, seed=5):
    ang = np.arange(context)[:, None] * (1e4 ** -(np.arange(pairs) / max(1, pairs)))[None]
    return np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)


def rotate(x, cos, sin, pairs):
    """x [rows, heads, hd] f32, cos and sin [rows, pairs]: each product rounded, then the sum."""
    y = x.copy()
    a, b = x[..., 0:2 * pairs:2], x[..., 1:2 * pairs:2]
    c, s = cos[:, None], sin[:, None]
    y[..., 0:2 * pairs:2] = a * c - b * s
    y[..., 1:2 * pairs:2] = a * s + b * c
    return y


def q8(x):
    """(scales [..., nb], codes [..., hd]) of the last dimension's 32-wide blocks, as the activation quantizer."""
    hd = x.shape[-1]
    nb = (hd + 31) // 32
    pad = np.zeros(x.shape[:-1] + (nb * 32,), np.float32)
    pad[..., :hd] = x
    b = pad.reshape(x.shape[:-1] + (nb, 32))
    with np.errstate(all="ignore"):
        scale = (np.abs(b).max(-1) / np.float32(127)).astype(np.float32)
        inv = np.where(scale >= np.finfo(np.float32).tiny, np.float32(1) / scale, np.float32(0)).astype(np.float32)
        code = np.clip(np.rint(b * inv[..., None]), -127, 127)
    bad = ~np.isfinite(b).all(-1)
    scale[bad] = np.nan
    code[bad] = 0
    return scale, code.astype(np.int8).reshape(x.shape[:-1] + (nb * 32,))[..., :hd]


class Cache:
    """A pool in device memory and its numpy image; pages of the sequences in a shuffled order."""

    def __init__(self, kv_type, kv, hd, page, lengths, seed=1, spare=2, stale="random", stride=None):
        rng = np.random.default_rng(seed)
        self.type, self.kv, self.hd, self.page, self.nb = kv_type, kv, hd, page, (hd + 31) // 32
        self.lengths = list(lengths)
        need = [-(-n // page) for n in lengths]
        self.pages = sum(need) + spare
        self.stride = stride or max(need + [1])
        self.table = np.full((len(lengths), self.stride), -1, np.int32)
        order, at = rng.permutation(self.pages).astype(np.int32), 0
        for s, n in enumerate(need):
            self.table[s, :n] = order[at:at + n]
            at += n
        shape = (self.pages, kv, page, hd)
        if kv_type == Q8:
            self.k = rng.integers(-128, 128, shape).astype(np.int8)
            self.v = rng.integers(-128, 128, shape).astype(np.int8)
            self.ks = rng.uniform(0.005, 0.02, (self.pages, kv, self.nb, page)).astype(np.float32)
            self.vs = rng.uniform(0.005, 0.02, (self.pages, kv, self.nb, page)).astype(np.float32)
        else:
            self.k, self.v = (rng.standard_normal(shape).astype(NP[kv_type]) for _ in range(2))
            self.ks = self.vs = None
        if stale == "nan":  # every slot that no sequence holds
            self.spoil(~self.held())

    def held(self):
        m = np.zeros((self.pages, self.page), bool)
        for s, n in enumerate(self.lengths):
            for j in range(n):
                m[self.table[s, j // self.page], j % self.page] = True
        return m

    def spoil(self, mask):
        """NaN (Q8: a NaN scale; every second slot infinite) into the slots of mask [pages, page]."""
        pg, sl = np.nonzero(mask)
        bad = np.where(np.arange(pg.size) % 2, np.nan, np.inf)
        if self.type == Q8:
            self.ks[pg, :, :, sl] = bad[:, None, None]
            self.vs[pg, :, :, sl] = -bad[:, None, None]
        else:
            self.k[pg, :, sl] = bad[:, None, None]
            self.v[pg, :, sl] = -bad[:, None, None]

    def slots(self, s, pos):
        pos = np.asarray(pos)
        return self.table[s, pos // self.page], pos % self.page

    def spoil_positions(self, s, pos):
        m = np.zeros((self.pages, self.page), bool)
        m[self.slots(s, pos)] = True
        self.spoil(m)

    def values_layout(self, v):
        return np.ascontiguousarray(v.transpose(0, 1, 3, 2))

    def upload(self):
        self.kb, self.vb = smq.DeviceBuffer.from_array(self.k), smq.DeviceBuffer.from_array(self.values_layout(self.v))
        self.ksb = self.vsb = None
        if self.type == Q8:
            self.ksb, self.vsb = smq.DeviceBuffer.from_array(self.ks), smq.DeviceBuffer.from_array(self.vs)
        self.tb = smq.DeviceBuffer.from_array(self.table)
        self.desc = smq.paged_kv(self.kb, self.vb, self.ksb, self.vsb, self.type, self.page, self.pages)
        return self

    def download(self):
        dt = NP[self.type]
        k = self.kb.download(dt).reshape(self.k.shape)
        v = self.vb.download(dt).reshape(self.pages, self.kv, self.hd, self.page).transpose(0, 1, 3, 2)
        if self.type != Q8:
            return k, v
        return k, v, self.ksb.download(np.float32).reshape(self.ks.shape), self.vsb.download(np.float32).reshape(self.vs.shape)

    def put(self, s, pos, k, v):
        """The rows k, v [n, kv, hd] at positions pos of sequence s, into the numpy image."""
        pg, sl = self.slots(s, pos)
        if self.type == Q8:
            (ks, k), (vs, v) = q8(k), q8(v)
            self.ks[pg, :, :, sl], self.vs[pg, :, :, sl] = ks, vs
        with np.errstate(over="ignore"):
            self.k[pg, :, sl], self.v[pg, :, sl] = k.astype(NP[self.type]), v.astype(NP[self.type])

    def rows(self, s, pos, dtype=np.float32):
        """What the cache holds at positions pos of sequence s: keys and values [n, kv, hd]."""
        pg, sl = self.slots(s, pos)
        k, v = self.k[pg, :, sl].astype(dtype), self.v[pg, :, sl].astype(dtype)
        if self.type == Q8:
            with np.errstate(all="ignore"):
                k = k * np.repeat(self.ks[pg, :, :, sl].astype(dtype), 32, -1)[..., :self.hd]
                v = v * np.repeat(self.vs[pg, :, :, sl].astype(dtype), 32, -1)[..., :self.hd]
        return k, v


class Batch:
    def __init__(self, cache, new, lengths=None, padding=0):
        self.new = list(new)
        self.begin = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        self.length = np.array(cache.lengths if lengths is None else lengths, np.int32)
        self.tokens = int(self.begin[-1]) + padding
        self.bb, self.lb = smq.DeviceBuffer.from_array(self.begin), smq.DeviceBuffer.from_array(self.length)
        self.desc = smq.paged_batch(self.bb, self.lb, cache.tb, len(self.new), self.tokens, cache.stride)

    def where(self):
        """(sequence, positions) of each sequence's rows."""
        for s, n in enumerate(self.new):
            yield s, np.arange(self.length[s] - n, self.length[s])


def visible(p, window, sinks):
    j = np.arange(p + 1)
    return j[(j > p - window) | (j < sinks)] if window else j


def attend64(cache, batch, q, heads, window=0, sinks=0):
    """(attention [tokens, heads, hd] in 64 bits, bound of the error of a calculation in f32 of each coordinate).

    The bound: a score is a sum of hd products, each within (hd + 8) * 2^-24 of sum |q k| (operands to 22 bits or
    better, f32 sums); the softmax argument rounds at 2^-24 of the largest score, exp2 within 2 units; N terms add
    up in blocks of at least 8, (N / 8 + 64) * 2^-24. A weight's relative error counts twice (weight and sum)."""
    hd, grp = cache.hd, heads // cache.kv
    out = np.zeros((batch.tokens, heads, hd))
    tol = np.zeros((batch.tokens, heads, hd))
    eps = 2.0 ** -24
    r = 0
    for s, pos in batch.where():
        if not len(pos):
            continue
        k, v = cache.rows(s, np.arange(pos[-1] + 1), np.float64)
        for p in pos:
            j = visible(p, window, sinks)
            for h in range(heads):
                kk, vv, qq = k[j, h // grp], v[j, h // grp], q[r, h].astype(np.float64)
                x = kk @ qq / np.sqrt(hd)
                size = (np.abs(kk) @ np.abs(qq)).max() / np.sqrt(hd)
                w = np.exp(x - x.max())
                w /= w.sum()
                out[r, h] = w @ vv
                ds = size * (hd + 8) * eps
                tol[r, h] = w @ np.abs(vv) * (4 * ds + 4 * (np.abs(x).max() + 2) * eps + (len(j) / 8 + 64) * eps)
            r += 1
    return out, tol


def logits_rules(logits, history=None, penalty=None, bias=None, masks=None):
    """One row in f32 as the library rounds it: (adjusted, token). history: ids; bias: (ids, values); masks: bool [vocab]."""
    l, v = logits.astype(np.float32).copy(), logits.size
    with np.errstate(all="ignore"):
        if history is not None and len(history):
            ids, times = np.unique(np.asarray(history, np.uint32), return_counts=True)
            keep = ids < v
            ids, times = ids[keep], times[keep].astype(np.float32)
            rep, pres, freq = (np.float32(x) for x in penalty)
            x = l[ids]
            l[ids] = np.where(x > 0, x / rep, x * rep) - (times * freq + pres)
        if bias is not None and len(bias[0]):
            add = np.zeros(v, np.float32)
            for i, b in zip(*bias):
                if i < v:
                    add[i] += np.float32(b)
            l += add
    if masks is not None:
        l[~masks] = -np.inf
    may = np.arange(v) if masks is None else np.nonzero(masks)[0]
    if not may.size:
        return l, 0xFFFFFFFF
    if np.isnan(l[may[0]]):
        return l, int(may[0])
    x = np.where(np.isnan(l[may]), -np.inf, l[may])
    fine = ~np.isnan(l[may])
    best = x[fine].max()
    return l, int(may[fine][np.nonzero(x[fine] == best)[0][0]])
