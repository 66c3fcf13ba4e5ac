"""Plain numpy restatement of the operators of drafts and beams: normed and rotated rows, trees and their attention (64 bits),
page forks, copies, accepted paths, beam steps (64 bits)."""
import numpy as np

from paged_ref import Q8

NONE = 0xFFFFFFFF


def normed(x, w, eps):
    """x [rows, heads, hd] f32: mean, root and quotient in 64 bits, the quotient and both products rounded to f32."""
    if w is None:
        return x
    with np.errstate(all="ignore"):
        inv = (1.0 / np.sqrt((x.astype(np.float64) ** 2).sum(-1, keepdims=True) / x.shape[-1] + np.float64(np.float32(eps))))
        return (x * inv.astype(np.float32)).astype(np.float32) * w


def random_tree(rng, n, roots=0.1):
    return [-1 if i == 0 or rng.random() < roots else int(rng.integers(0, i)) for i in range(n)]


def masks(parents):
    """(depths, bool [n, n]) of one sequence's tree."""
    n = len(parents)
    depth, seen = np.zeros(n, np.int32), np.zeros((n, n), bool)
    for i, p in enumerate(parents):
        seen[i, i] = True
        if p >= 0:
            depth[i] = depth[p] + 1
            seen[i] |= seen[p]
    return depth, seen


def words(seen, stride):
    """bool [rows, n] as mask words [rows, stride]."""
    b = np.zeros((seen.shape[0], 32 * stride), np.uint64)
    b[:, :seen.shape[1]] = seen
    return (b.reshape(seen.shape[0], stride, 32) << np.arange(32, dtype=np.uint64)).sum(-1).astype(np.uint32)


def context_seen(first, p, window, sinks):
    j = np.arange(first)
    return j[(j > p - window) | (j < sinks)] if window else j


def tree64(cache, batch, q, heads, depth, seen, window=0, sinks=0):
    """(attention [tokens, heads, hd] in 64 bits, bound of an f32 calculation's error) as attend64 derives it; depth [tokens],
    seen: each sequence's bool [n, n]. Rows that see nothing are 0, exactly."""
    hd, grp, eps = cache.hd, heads // cache.kv, 2.0 ** -24
    out, tol = np.zeros((batch.tokens, heads, hd)), np.zeros((batch.tokens, heads, hd))
    r = 0
    for s, pos in batch.where():
        if not len(pos):
            continue
        first = int(pos[0])
        k, v = cache.rows(s, np.arange(pos[-1] + 1), np.float64)
        for i in range(len(pos)):
            j = np.concatenate([context_seen(first, first + int(depth[r]), window, sinks), first + np.nonzero(seen[s][i])[0]])
            for h in range(heads if len(j) else 0):
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


def fork(table, held, refs, parent, keep, room, page):
    """A valid call's results: table, held, refs, copies, free."""
    rows, stride = len(parent), table.shape[1]
    refs = refs.copy()
    for s, n in enumerate(held):
        for x in range(n):
            refs[table[s, x]] -= 1
    full, part = np.asarray(keep) // page, np.asarray(keep) % page
    for d in range(rows):
        for x in range(full[d]):
            refs[table[parent[d], x]] += 1
    out, copies = np.full((rows, stride), -1, np.int32), np.tile(np.array([-1, -1, 0], np.int32), (rows, 1))
    last = [int(table[parent[d], full[d]]) if part[d] else -1 for d in range(rows)]
    mine = [part[d] > 0 and refs[last[d]] == 0 and last[d] not in last[:d] for d in range(rows)]
    for d in range(rows):
        refs[last[d]] += mine[d]
    free = list(np.nonzero(refs == 0)[0])
    need, have, at = 0, len(free), 0
    new_held = -(-np.asarray(room) // page)
    for d in range(rows):
        if full[d] + mine[d]:
            out[d, :full[d] + mine[d]] = table[parent[d], :full[d] + mine[d]]
        for x in range(full[d] + mine[d], new_held[d]):
            need += 1
            if at < have:
                out[d, x] = free[at]
                refs[free[at]] = 1
                at += 1
        if part[d] and not mine[d] and out[d, full[d]] >= 0:
            copies[d] = last[d], out[d, full[d]], part[d]
    return out, new_held.astype(np.int32), refs.astype(np.int32), copies, have - need


def pool_parts(cache):
    """The cache's arrays with positions second to last (keys, values) or last (scales)."""
    return [(cache.k, 2), (cache.v, 2)] + ([(cache.ks, 3), (cache.vs, 3)] if cache.type == Q8 else [])


def copy(cache, copies):
    for a, b, n in copies:
        for x, axis in pool_parts(cache):
            if axis == 2:
                x[b, :, :n] = x[a, :, :n]
            else:
                x[b, :, :, :n] = x[a, :, :, :n]


def compact(cache, s, first, path):
    pg, sl = cache.slots(s, first + np.asarray(path, int))
    tp, ts = cache.slots(s, first + np.arange(len(path)))
    for x, axis in pool_parts(cache):
        if axis == 2:
            x[tp, :, ts] = x[pg, :, sl]
        else:
            x[tp, :, :, ts] = x[pg, :, :, sl]


def beam(logits, score, groups, beams, select, done=None, pad=0, eos=NONE):
    """(parent, token, score in 64 bits, done) of each group's best, by the rules of order."""
    out = []
    for g in range(groups):
        cand = []
        for r in range(g * beams, (g + 1) * beams):
            if score[r] == -np.inf:
                continue
            if done is not None and done[r]:
                cand.append((-float(score[r]), r, 0, 0, pad))
                continue
            l = logits[r].astype(np.float64)
            top = l.max()
            if top == -np.inf:
                continue
            lse = top + np.log(np.exp(l - top).sum())
            ids = np.lexsort((np.arange(l.size), -l))[:select]
            cand += [(-(float(score[r]) + (l[i] - lse)), r, k, 0, int(i)) for k, i in enumerate(ids) if l[i] > -np.inf]
        cand.sort()
        cand = cand[:select]
        for v, r, _, _, i in cand:
            over = bool(done is not None and done[r])
            out.append((r, i, -v, over or (eos != NONE and i == eos)))
        out += [(-1, NONE, -np.inf, True)] * (select - len(cand))
    return [np.array(x) for x in zip(*out)]
