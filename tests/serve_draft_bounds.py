"""Attention over the 16-bit cache in 64 bits, with the largest error that each form of the kernels may make. tests/serve_draft_oracle.py allows all forms a rounding of every weight to the type, which
is as large as the result's own: a form that keeps weights in two numbers of the type is held to that here."""
import math

import numpy as np

# columns (rows announced x query heads of a KV head) choose the form, and whether the table allows sequences of any length: (rows, query heads a KV head, whether it does, whether weights are rounded once)
FORMS = {"one launch, 8": (1, 4, False, False), "one launch, 16": (3, 5, False, False), "one launch, 32": (5, 4, False, False), "one launch, 64": (9, 7, False, False),
         "a line, 8": (2, 4, True, False), "a line, 16": (3, 5, True, False), "many, boxes": (40, 4, True, True), "many, gathered": (40, 5, True, True)}


def row(q, k, v, scale, bf16, once):
    """of one row and head: soft-max weights p, the result, and the largest error of a kernel's.

    A weight is 2^y, y = s - b in log2 units, with b the same for all. Off by: the score's sum, hd exact products added by hd / 16 instructions, each off by 2^-22 of the largest sum at most; its
    scaling, 2^-22; y's rounding, 2^-24 of |y|, which is the distance from the largest score and up to 46 (bfloat16: weights from 2^-38 to 2^-30) or 15 (fp16: 2^7 to 2^15); 2^y, 2^-22 (of many rows
    2^-18.5, the polynomial's). These are the same above and below the line of the quotient. What is multiplied with values is rounded to the type once (half a step) or in two numbers (half a step of
    half a step), of fp16 below 2^-14 by half a step of 2^-24, the largest weight being 2^7 at least. Sums of values take n / 8 instructions at most, sums of weights as many.
    The result is rounded to the type: of fp16 below 2^-14, whose steps are 2^-24 there, by 2^-25."""
    n, hd = k.shape
    s = scale * (k @ q)
    p = np.exp(s - s.max())
    p /= p.sum()
    r = p @ v
    far = (s.max() - s) / math.log(2)
    eps = 2.0 ** -7 if bf16 else 2.0 ** -10
    weight = abs(scale) * (np.abs(k) @ np.abs(q)) * 2.0 ** -22 * hd / 16 + np.abs(s) * 2.0 ** -22 + ((46 if bf16 else 15) + far) * math.log(2) * 2.0 ** -24 + (2.0 ** -18.5 if once else 2.0 ** -22)
    part = eps / 2 if once else (eps / 2) ** 2
    size = np.abs(v)
    room = (p * (weight + part)) @ size + np.abs(r) * (p @ weight) + (p @ size + np.abs(r)) * (n / 8 + 16) * 2.0 ** -22 + 2.0 ** -32 * size.sum(0)
    return p, r, room + eps / 2 * (np.abs(r) + room) + (0.0 if bf16 else 2.0 ** -25)


def seen(p, there, window, sinks):
    """the positions that a row at position p sees"""
    j = np.arange(min(p + 1, there.size))
    return j[there[j] & ((j > p - window) | (j < sinks) if window else True)]


def attention(q, kv, held, first, window, sinks, scale, bf16, once):
    """q [rows, heads, hd] float64; kv[s]: K, V [n_kv, positions, hd] float64 and which positions have a page. The result, and how far off it may be"""
    out, room = np.zeros(q.shape), np.zeros(q.shape)
    for s in range(len(first) - 1):
        K, V, there = kv[s]
        group = q.shape[1] // K.shape[0]
        for i in range(first[s], first[s + 1]):
            j = seen(held[s] + i - first[s], there, window, sinks)
            for h in range(q.shape[1] if j.size else 0):
                _, out[i, h], room[i, h] = row(q[i, h], K[h // group][j], V[h // group][j], scale, bf16, once)
    return out, room
