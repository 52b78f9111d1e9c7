"""The operators of booster_b200.serve around drafted tokens and the 16-bit cache, in 64 bits and plain numpy: what the GPU tests hold them to."""
import math

import numpy as np


# ---- attention over the 16-bit cache -----------------------------------------------------------------------------------------
def attention(q, kv, held, first, window, sinks, scale, eps):
    """q [rows, heads, hd] float64; kv[s]: K, V [n_kv, positions, hd] float64 and present [positions]. Returns the result and the largest error that the kernels' roundings may make"""
    out, room = np.zeros(q.shape), np.zeros(q.shape)
    heads = q.shape[1]
    for s in range(len(first) - 1):
        K, V, present = kv[s]
        group = heads // K.shape[0]
        for r in range(first[s], first[s + 1]):
            p = held[s] + r - first[s]
            j = np.arange(min(p + 1, present.size))
            j = j[present[j] & ((j > p - window) | (j < sinks) if window else True)]
            if not j.size:
                continue
            for h in range(heads):
                k, v, x = K[h // group][j], V[h // group][j], q[r, h]
                y = scale * (k @ x)
                if np.isnan(y).any() or not np.isfinite(x).all():
                    out[r, h] = np.nan
                    continue
                w = np.exp(y - y.max())
                w /= w.sum()
                out[r, h] = w @ v
                # P is rounded once to the type (half a step of eps; of fp16 below 2^-14 half a step of 2^-24, the largest P being at least 1) and the sum of weights is that of P or of what it is
                # rounded to: both sides off by eps / 2. exp2 2^-20. A score is hd exact products summed by hd / 16 instructions, each off by 2^-22 of the largest sum at most, scaled with
                # 2^-23, and its distance from the largest is off by twice that
                score = abs(scale) * (2.0 ** -22 * x.size / 16 + 2.0 ** -22) * (np.abs(k) @ np.abs(x)).max()
                room[r, h] = (w @ np.abs(v)) * (eps + 2.0 ** -20 + 2 * score) + 2.0 ** -24 * np.abs(v).sum(0)
    return out, room


# ---- pages -------------------------------------------------------------------------------------------------------------------
def plan(table, held, refs, slots, counts, rows, page):
    """(first, positions, places, status), and table and refs as they become (lists, changed in place)"""
    P, n_pages, width = page, len(refs), len(table[0])
    first = [0]
    for c in counts:
        first.append(first[-1] + max(0, c))
    bad = first[-1] > rows or any(c < 0 for c in counts)
    first = [min(f, rows) for f in first]
    wanted = []
    for i, (s, c) in enumerate(zip(slots, counts)):
        if not 0 <= s < len(table) or s in slots[:i]:
            bad = True
            continue
        need = -(-(held[s] + max(0, c)) // P)
        if held[s] < 0 or need > width:
            bad = True
            continue
        f = min(held[s] // P, need)
        while f < need and table[s][f] >= 0:
            f += 1
        if any(p >= 0 for p in table[s][f:need]):
            bad = True
        wanted += [(s, i) for i in range(f, need)]
    free = [p for p in range(n_pages) if refs[p] <= 0]
    status = -1 if bad else max(0, len(wanted) - len(free))
    if status == 0:
        for (s, i), p in zip(wanted, free):
            table[s][i] = p
            refs[p] = 1
    positions, places = [-1] * rows, [-1] * rows
    for i, s in enumerate(slots):
        for r in range(first[i], first[i + 1]):
            if 0 <= s < len(table) and held[s] >= 0:
                pos = positions[r] = held[s] + r - first[i]
                p = table[s][pos // P] if pos // P < width else -1
                if 0 <= p < n_pages:
                    places[r] = p * P + pos % P
    return first, positions, places, status


def trim(table, held, refs, slots, page, window, sinks):
    for s in slots:
        if not 0 <= s < len(table):
            continue
        for i, p in enumerate(table[s]):
            h = max(0, held[s])
            seen = i * page < h and (not window or i * page < sinks or (i + 1) * page > h - window + 1)
            if p >= 0 and not seen:
                table[s][i] = -1
                if p < len(refs):
                    refs[p] -= 1


# ---- verification ------------------------------------------------------------------------------------------------------------
def shares(x, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """p of one row, and how near a filter's border is to a token; None where no logit is a number"""
    x = np.asarray(x, np.float64).copy()
    x[np.isnan(x)] = -np.inf
    top = x.max()
    if top == -np.inf:
        return None, 1.0
    out = np.zeros(x.size)
    if not temperature > 0:
        out[int(np.argmax(x))] = 1.0
        return out, 1.0
    d = np.where(x == top, 0.0, top - np.where(x == top, 0.0, x))
    order, near = np.lexsort((np.arange(x.size), d)), 1.0
    if 0 < top_k < x.size:
        order = order[:top_k]
    w = np.exp(-d[order])
    if top_p < 1:
        c = np.cumsum(w) / w.sum()
        n = 1 + int(np.searchsorted(c, top_p)) if top_p > 0 else 1
        near = np.abs(c - top_p).min()
        order, w = order[:n], w[:n]
    order = order[w >= min(min_p, 1.0)]
    out[order] = np.exp(np.where(d[order] == 0, 0.0, -d[order] / temperature))
    return out / out.sum(), near


def verify(logits, ids, first, u, accept, filters, probs):
    """(gained, tokens, logprobs, near): filters[r] are shares' arguments; near[i] is how near sequence i came to deciding otherwise"""
    rows, vocab = logits.shape
    gained, tokens, logprobs, near = [], [-1] * rows, [0.0] * rows, []
    for a, b in zip(first, first[1:]):
        n, nearest = 0, 1.0
        for r in range(a, b):
            p, border = shares(logits[r], **filters[r])
            nearest = min(nearest, border)
            n += 1
            greedy = not filters[r].get("temperature", 1.0) > 0
            if p is None:
                logprobs[r] = -math.inf
                break
            rest = p
            if r + 1 < b:
                x = ids[r + 1]
                q = np.zeros(vocab)
                if probs is not None:
                    q = np.where(probs[r] > 0, probs[r], 0.0).astype(np.float64)
                elif 0 <= x < vocab:
                    q[x] = 1.0
                if 0 <= x < vocab:
                    nearest = min(nearest, abs(accept[r] * q[x] - p[x]))
                    if accept[r] * q[x] < p[x]:
                        tokens[r], logprobs[r] = x, 0.0 if greedy else math.log(p[x])
                        continue
                rest = np.maximum(p - q, 0.0)
                rest[rest < 2.0 ** -41] = 0.0
                if rest.sum() == 0:
                    rest = p
            if greedy:
                tokens[r] = int(np.argmax(p))
                break
            c = np.cumsum(rest) / rest.sum()
            at = min(int(np.searchsorted(c, u[r], side="right")), int(np.flatnonzero(rest)[-1]))
            nearest = min(nearest, np.abs(c[:-1] - u[r]).min() if c.size > 1 else 1.0)
            tokens[r], logprobs[r] = at, math.log(p[at])
            break
        gained.append(n)
        near.append(nearest)
    return gained, tokens, logprobs, near
