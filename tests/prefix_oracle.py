"""Plain 64-bit forms of the operators for drafted tokens behind a shared prompt: rotary tables, rotation and append, attention over a shared prefix,
verification.  numpy only; every formula is written out for one row at a time."""
import math

import numpy as np


def frequencies(kind, dims, base, factor=1.0, original=0.0, low=0.0, high=1.0):
    f = []
    for i in range(dims // 2):
        b = base * factor ** (dims / (dims - 2)) if kind == 2 and dims > 2 else base
        v = b ** (-2.0 * i / dims)
        if kind == 1:
            v /= factor
        if kind == 3:
            kept = min(1.0, max(0.0, (original * v / math.tau - low) / (high - low)))
            v = kept * v + (1.0 - kept) * v / factor
        f.append(v)
    return np.array(f)


def rotate(x, cosine, sine, rot, pairs):
    """One head's vector."""
    y = x.astype(np.float64).copy()
    half = rot // 2
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if pairs else (i, i + half)
        c, s = float(cosine[i]), float(sine[i])
        y[a], y[b] = x[a] * c - x[b] * s, x[b] * c + x[a] * s
    return y


class Pages:
    """Pools [pages, kv_heads, page, dim] and a table of page numbers."""

    def __init__(self, key, value, table):
        self.key, self.value, self.table = key, value, table
        self.page = key.shape[2]

    def capacity(self):
        return self.table.shape[1] * self.page

    def row(self, pool, slot, position, head):
        page = self.table[slot, position // self.page]
        if not 0 <= page < len(pool):
            return np.zeros(pool.shape[3])
        return pool[page, head, position % self.page].astype(np.float64)

    def rows(self, pool, slot, count, head):
        return np.stack([self.row(pool, slot, i, head) for i in range(count)]) if count else np.zeros((0, pool.shape[3]))


def attention(query, heads, scale, cache, slots, first, lengths, prefix=None, group_first=(0,), group_prefix=(), prefix_length=()):
    """out, and the sums of w |v| and the largest sum of |scale q k| of every row and head, by which errors are bounded.  query [rows, heads, dim]."""
    rows, _, dim = query.shape
    kv_heads = cache.key.shape[1]
    group = heads // kv_heads
    out, mass, size = np.zeros((rows, heads, dim)), np.zeros((rows, heads, dim)), np.zeros((rows, heads))
    keys = np.zeros((rows,), dtype=np.int64)
    for s, slot in enumerate(slots):
        count = first[s + 1] - first[s]
        owner = [g for g in range(len(group_prefix)) if group_first[g] <= s < group_first[g + 1]]
        shared = group_prefix[owner[0]] if owner else -1
        if not (prefix is not None and 0 <= shared < len(prefix.table)):
            shared = -1
        shared_keys = min(max(0, prefix_length[shared]), prefix.capacity()) if shared >= 0 else 0
        own_slot = 0 <= slot < len(cache.table)
        for k in range(kv_heads):
            total = min(lengths[slot] + count, cache.capacity()) if own_slot else 0
            kp = prefix.rows(prefix.key, shared, shared_keys, k) if shared >= 0 else np.zeros((0, dim))
            vp = prefix.rows(prefix.value, shared, shared_keys, k) if shared >= 0 else np.zeros((0, dim))
            ko, vo = cache.rows(cache.key, slot, total, k), cache.rows(cache.value, slot, total, k)
            for t in range(count):
                r = first[s] + t
                seen = min(total, lengths[slot] + t + 1) if own_slot else 0
                kk, vv = np.concatenate([kp, ko[:seen]]), np.concatenate([vp, vo[:seen]])
                keys[r] = len(kk)
                if not len(kk):
                    continue
                for h in range(k * group, (k + 1) * group):
                    q = query[r, h].astype(np.float64)
                    score = kk @ q * scale
                    w = np.exp(score - score.max())
                    w /= w.sum()
                    out[r, h] = w @ vv
                    mass[r, h] = w @ np.abs(vv)
                    size[r, h] = (np.abs(kk) @ np.abs(q)).max() * abs(scale)
    return out, mass, size, keys


def weights(x, temperature):
    e = np.exp((x.astype(np.float64) - x.max()) / temperature)
    return e / e.sum()


def verify(logits, draft, ids, first, temperature, accept, draw):
    """accepted, next, and how far every decision was from its border."""
    accepted, chosen, margin = [], [], math.inf
    vocab = logits.shape[1]
    for s in range(len(first) - 1):
        begin, last = first[s], first[s + 1] - 1
        if last < begin:
            accepted.append(0)
            chosen.append(-1)
            continue
        row = begin
        while row < last:
            x = ids[row + 1]
            if temperature == 0:
                if x != argmax(logits[row]):
                    break
            else:
                if not finite(logits[row]) or not 0 <= x < vocab or (draft is not None and not finite(draft[row])):
                    break
                p, q = weights(logits[row], temperature)[x], weights(draft[row], temperature)[x] if draft is not None else 1.0
                margin = min(margin, abs(accept[row] * q - p) / max(p, q, 1e-300))
                if not accept[row] * q < p:
                    break
            row += 1
        accepted.append(row - begin)
        if temperature == 0 or not finite(logits[row]):
            chosen.append(argmax(logits[row]))
            continue
        left = weights(logits[row], temperature)
        x = ids[row + 1] if row < last else -1
        if 0 <= x < vocab:
            minus = weights(draft[row], temperature) if draft is not None and finite(draft[row]) else np.zeros(vocab)
            if draft is None:
                minus[x] = 1.0
            rest = np.maximum(left - minus, 0)
            left = rest if rest.sum() > 0 else left
        running = np.cumsum(left)
        at = int(np.searchsorted(running, draw[s] * running[-1], side="right"))
        chosen.append(at)
        margin = min(margin, *(np.abs(running[max(0, at - 1):at + 1] - draw[s] * running[-1]) / running[-1]))
    return np.array(accepted), np.array(chosen), margin


def finite(row):
    return not np.isnan(row).any() and not np.isposinf(row).any() and np.isfinite(row).any()


def argmax(row):
    nans = np.flatnonzero(np.isnan(row))
    return int(nans[0]) if len(nans) else int(np.argmax(row))
