"""The operators of booster_b200.serve in 64 bits and plain numpy, one place after the other: what the GPU tests hold them to."""
import math

import numpy as np
import torch


# ---- the 4-bit cache ---------------------------------------------------------------------------------------------------------
def quantize(x):
    """one head's row x [head_dim] -> codes 0 .. 15, scales of its blocks (exact values), ignoring rows that are not finite"""
    codes, scales = np.empty(x.size, np.int64), np.empty(x.size // 32)
    for b in range(x.size // 32):
        blk = x[32 * b:32 * b + 32].astype(np.float64)
        lo, hi = blk.min(), blk.max()
        d = min(8160.0, max(-8160.0, (lo if -lo >= hi else hi) / -8))
        d = float(torch.tensor(d, dtype=torch.float32).bfloat16().half().double())
        scales[b] = d if d else 0.0
        codes[32 * b:32 * b + 32] = 8 if d == 0 else np.clip(np.rint(blk / d), -8, 7) + 8
    return codes, scales


def held_rows(k, v):
    """what the cache holds of one token's key and value of a head: values in 64 bits"""
    if not (np.isfinite(k).all() and np.isfinite(v).all()):
        return np.full(k.size, np.nan), np.zeros(k.size)
    out = []
    for x in (k, v):
        c, d = quantize(x)
        out.append((c - 8) * np.repeat(d, 32))
    return out


def write_tile(tile, t, k, v):
    """puts token t of a tile's 16 into its bytes (uint8 [18 * head_dim])"""
    hd = k.size
    nb, c, i = hd // 32, t % 4, t // 4
    bad = not (np.isfinite(k).all() and np.isfinite(v).all())
    (kc, ks), (vc, vs) = (quantize(x) if not bad else (np.full(hd, 8), np.zeros(hd // 32)) for x in (k, v))
    for d in range(hd):
        word = (((i // 2) * 8 + 2 * c + i % 2) * 4 + d % 32 // 8) * nb + d // 32
        for at, shift, code in ((4 * word + d % 8 // 2, 4 * (d % 2), kc[d]),
                                (8 * hd + 2 * (((((d // 64) * 8 + d % 32 // 4) * 4 + c) * 2 + d // 32 % 2) * 4 + i) + d % 4 // 2, 4 * (d % 2), vc[d])):
            tile[at] = (int(tile[at]) & ~(15 << shift) & 255) | int(code) << shift
    halves = tile.view(np.float16)
    for b in range(nb):
        halves[8 * hd + ((c * 2 + i % 2) * 2 + i // 2) * nb + b] = np.nan if bad else ks[b]
        halves[8 * hd + hd // 2 + (c * nb + b) * 4 + i] = vs[b]


def rows_of(first, n_rows):
    """(sequence, row of the step, its number in the sequence)"""
    return [(s, r, r - first[s]) for s in range(len(first) - 1) for r in range(first[s], min(first[s + 1], n_rows))]


def page_of(table, slot, pos, page_tokens, n_pages):
    if not 0 <= slot < len(table) or not pos // page_tokens < len(table[slot]):
        return -1
    p = table[slot][pos // page_tokens]
    return p if 0 <= p < n_pages else -1


# ---- attention ---------------------------------------------------------------------------------------------------------------
def attention(q, kv, held, first, window, scale):
    """q [rows, heads, head_dim] float64 of values that the input type holds; kv[s]: (K, V) [n_kv, positions, head_dim] float64, NaN rows of K where a position is absent or poisoned and
    present[s] bool [positions]. Returns the result and the largest error that the kernel's roundings may make, see below"""
    out, room = np.zeros(q.shape), np.zeros(q.shape)
    heads, hd = q.shape[1:]
    for s in range(len(first) - 1):
        K, V, present = kv[s]
        group = heads // K.shape[0]
        for r in range(first[s], first[s + 1]):
            p = held[s] + r - first[s]
            j = np.arange(max(0, p - window + 1) if window else 0, min(p + 1, present.size))
            j = j[present[j]]
            if not j.size:
                continue
            for h in range(heads):
                k, v = K[h // group][j], V[h // group][j]
                x = scale * (k @ q[r, h])
                if np.isnan(x).any():
                    out[r, h] = np.nan
                    continue
                w = np.exp(x - x.max())
                w /= w.sum()
                out[r, h] = w @ v
                # P's rounding to fp16 (half a step, 2^-11; below 2^-14 half a step of 2^-24, the largest P being at least 1), exp2 (2^-20), and scores: 32 products of codes with
                # their offset (at most 1039 times an entry of q) are summed by two instructions with 2^-22 of the largest sum at most, then scaled
                big = np.abs(k).reshape(j.size, -1, 32).max(2) / 7 @ np.abs(q[r, h]).reshape(-1, 32).sum(1)
                score = abs(scale) * 1039 * 2.0 ** -22 * big.max()
                room[r, h] = (w @ np.abs(v)) * (2.0 ** -11 + 2.0 ** -20 + 2 * score) + 2.0 ** -25 * np.abs(v).sum(0)
    return out, room


# ---- sampling ----------------------------------------------------------------------------------------------------------------
def sample(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, log of its share, distance of u from the nearest border of the draw, distance of top-p's and min-p's borders) of one row x in 64 bits"""
    x = np.asarray(x, np.float64).copy()
    x[np.isnan(x)] = -np.inf
    top = x.max()
    if top == -np.inf:
        return -1, -np.inf, 1.0
    if not temperature > 0:
        return int(np.argmax(x)), 0.0, 1.0
    d = np.where(x == top, 0.0, top - np.where(x == top, 0.0, x))
    order = np.lexsort((np.arange(x.size), d))
    if 0 < top_k < x.size:
        order = order[:top_k]
    w = np.exp(-d[order])
    near = 1.0
    if top_p < 1:
        c = np.cumsum(w)
        share = c / c[-1]
        n = 1 + int(np.searchsorted(share, top_p)) if top_p > 0 else 1
        near = min(near, np.abs(share - top_p).min())
        order, w = order[:n], w[:n]
    m = min(min_p, 1.0)
    order = order[w >= m]
    order = np.sort(order)
    w = np.exp(np.where(d[order] == 0, 0.0, -d[order] / temperature))
    c = np.cumsum(w) / w.sum()
    at = min(int(np.searchsorted(c, u, side="right")), int(np.flatnonzero(w)[-1]))
    near = min(near, np.abs(c - u).min())
    return int(order[at]), math.log(w[at] / w.sum()), near
