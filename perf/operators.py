"""The operators of a server that runs many sequences at once, as they are measured: attention over a paged cache held in 4 bits, the rows that are
written into it, forking, freeing and compacting its pages, and the draw of the next token.

Where `own` is true, `run` calls booster_b200.serve; otherwise it computes the same in elementary torch operations. The cache's layout, which both
sides read and write, is a tile of 16 tokens of one KV head (18 * head_dim bytes): K codes, V codes, K scales, V scales, see _pack. Pages stand
scattered over the pool, and the pool's other pages hold what earlier sequences left.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

TYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
# (query heads, KV heads, head_dim): layer shapes of the 8B, 70B and small models of this repository, and one KV head a query head
HEADS = {"8b": (32, 8, 128), "70b": (64, 8, 128), "tiny": (4, 1, 128), "half": (8, 2, 64), "each": (16, 16, 64)}


def listed():
    return [
        # one user alone, early in a chat: the latency of one layer's attention
        dict(name="attend-one-at-333", kind="attend", shape="8b", seqs=1, lo=333, hi=333, rows=1, page=16, window=0, dtype="bfloat16"),
        # a busy server: one new token of 48 conversations of very different length
        dict(name="attend-48-ragged", kind="attend", shape="8b", seqs=48, lo=90, hi=4090, rows=1, page=64, window=0, dtype="bfloat16"),
        # few long documents under a large model's heads: each sequence alone has to fill the card
        dict(name="attend-3-long", kind="attend", shape="70b", seqs=3, lo=21001, hi=32700, rows=1, page=128, window=0, dtype="float16"),
        # a sliding window over long sequences, heads of 64, an odd number of sequences
        dict(name="attend-21-window", kind="attend", shape="half", seqs=21, lo=5, hi=2100, rows=1, page=32, window=1000, dtype="float16"),
        # the next portion of a long prompt behind a conversation
        dict(name="attend-prompt-512-at-6000", kind="attend", shape="8b", seqs=1, lo=6000, hi=6000, rows=512, page=64, window=0, dtype="bfloat16"),
        # several prompts' portions in one pass, ragged
        dict(name="attend-prompts-ragged", kind="attend", shape="8b", seqs=5, lo=0, hi=1500, rows=1100, page=32, window=0, dtype="float16"),
        # the step's new rows of a batch of conversations
        dict(name="append-48", kind="append", shape="8b", seqs=48, lo=90, hi=4090, rows=1, page=64, dtype="bfloat16"),
        # a long prompt's rows
        dict(name="append-prompts-8192", kind="append", shape="8b", seqs=3, lo=7, hi=700, rows=2731, page=64, dtype="bfloat16"),
        # 24 second answers to prompts that are in the cache already
        dict(name="fork-24", kind="fork", shape="8b", layers=8, seqs=24, lo=200, hi=1500, page=64, pages=640),
        # a third of the conversations end, and the pool's end is cleared to give it back
        dict(name="free-and-compact", kind="compact", shape="8b", layers=8, seqs=36, lo=200, hi=1500, page=64, pages=900),
        # one user: one row of logits
        dict(name="sample-one", kind="sample", rows=1, vocab=128256, dtype="float32", truncated=True),
        # a busy server's rows, some of them cut off by top-k, some by top-p alone, some not at all
        dict(name="sample-160", kind="sample", rows=160, vocab=128256, dtype="float32", truncated=False),
    ]


def _spread(rng, lo, hi):
    """a whole number from lo to hi, spread over its logarithm"""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "prompt", "prompt", "append", "fork", "compact", "sample", "sample"])
    shape, page, dtype = rng.choice(sorted(HEADS)), rng.choice([16, 32, 64, 128]), rng.choice(["bfloat16", "float16"])
    heads, kv, hd = HEADS[shape]
    if kind == "attend":
        hi = _spread(rng, 1, 32000)
        seqs = _spread(rng, 1, max(1, min(200, 80000 * 1024 // (hi * kv * hd))))
        return dict(kind="attend", shape=shape, seqs=seqs, lo=rng.randrange(0, hi + 1), hi=hi, rows=rng.choice([1, 1, 1, 2, 5]), page=page,
                    window=rng.choice([0, 0, 0, _spread(rng, 1, 4000)]), dtype=dtype)
    if kind == "prompt":
        hi, seqs = _spread(rng, 1, 6000), rng.choice([1, 1, 2, 3])
        rows = _spread(rng, 6, max(12, min(1000, 32 * 128 * 512 * 6200 // (heads * hd * seqs * (hi + 1000)))))
        return dict(kind="attend", shape=shape, seqs=seqs, lo=rng.randrange(0, hi + 1), hi=hi, rows=rows, page=page,
                    window=rng.choice([0, 0, _spread(rng, 1, 4000)]), dtype=dtype)
    if kind == "append":
        seqs = _spread(rng, 1, 200)
        return dict(kind="append", shape=shape, seqs=seqs, lo=rng.randrange(0, 50), hi=rng.randrange(50, 2000), rows=_spread(rng, 1, max(1, 4000 // seqs)), page=page,
                    dtype=rng.choice(["bfloat16", "float16", "float32"]))
    if kind in ("fork", "compact"):
        seqs, hi = _spread(rng, 1, 24), _spread(rng, 20, 1200)
        return dict(kind=kind, shape=shape, layers=rng.randrange(1, 9), seqs=seqs, lo=rng.randrange(1, hi + 1), hi=hi, page=page, pages=2 * seqs * (-(-hi // page) + 1) + rng.randrange(1, 60))
    return dict(kind="sample", rows=_spread(rng, 1, 150), vocab=_spread(rng, 200, 128256), dtype=rng.choice(["float32", "bfloat16", "float16"]), truncated=rng.choice([True, False]))


# ---- sizes that a case stands for, the same for every seed ------------------------------------------------------------------
def _between(lo, hi, n, turn):
    return [lo + int((hi - lo + 1) * ((turn + 0.618034 * i) % 1.0)) for i in range(n)]


def _held(case):
    """tokens of each sequence before the step"""
    return [min(case["hi"], v) for v in _between(case["lo"], case["hi"], case["seqs"], 0.37)]


def _counts(case):
    """new rows of each sequence: all the same for single tokens, ragged around `rows` for portions of prompts"""
    r = case["rows"]
    if r <= 5 or case["seqs"] == 1:
        return [r] * case["seqs"]
    return [max(1, v) for v in _between(r // 3, r, case["seqs"], 0.81)]


def _seen(held, count, window):
    """(pairs of a row and a position that it sees, positions that some row sees)"""
    pairs = 0
    for i in range(count):
        p = held + i + 1
        pairs += min(p, window) if window else p
    last = held + count
    return pairs, last if not window else min(last, window + count - 1)


# ---- the cache's layout ------------------------------------------------------------------------------------------------------
def _quantized(x):
    """x [..., head_dim] -> codes (0..15, int32) and scales (float16 with 8 significant bits) of blocks of 32, before the rule for numbers that are not finite"""
    b = x.float().unflatten(-1, (-1, 32))
    lo, hi = b.amin(-1), b.amax(-1)
    d = (torch.where(-lo >= hi, lo, hi) / -8).clamp(-8160, 8160)
    d = torch.where(torch.isfinite(d), d, torch.zeros_like(d)).bfloat16().half()
    d = torch.where(d == 0, torch.zeros_like(d), d)
    f = d.double().unsqueeze(-1)
    c = torch.where(f == 0, torch.zeros_like(f), b.double() / torch.where(f == 0, torch.ones_like(f), f))
    c = torch.nan_to_num(c, nan=0.0).round().clamp(-8, 7).int() + 8
    return c.flatten(-2), d


def _codes(k, v):
    """rows [..., head_dim] -> (K codes, K scales, V codes, V scales). A token that holds an infinity or a NaN in a head: scales NaN and 0"""
    kc, kd = _quantized(k)
    vc, vd = _quantized(v)
    bad = ~(torch.isfinite(k).all(-1, keepdim=True) & torch.isfinite(v).all(-1, keepdim=True))
    return (torch.where(bad, 8, kc), torch.where(bad, torch.full_like(kd, float("nan")), kd), torch.where(bad, 8, vc), torch.where(bad, torch.zeros_like(vd), vd))


def _pack(k, v):
    """k, v [tiles..., 16, head_dim] -> bytes [tiles..., 18 * head_dim]. With token t = c + 4 i:
    K codes  [t / 8][c, i % 2][8 dims' group within a block (4)][block] words of 8 codes, lowest bits first
    V codes  [block / 2][4 dims' group within a block (8)][c][block % 2][i / 2][i % 2] 16-bit units of 4 codes
    K scales [c][i % 2][i / 2][block] float16
    V scales [c][block][i] float16"""
    kc, kd, vc, vd = _codes(k, v)
    lead, nb = k.shape[:-2], k.shape[-1] // 32
    n = math.prod(lead)
    # token axis 16 -> (i / 2, i % 2, c)
    kc = kc.reshape(n, 2, 2, 4, nb, 4, 8).permute(0, 1, 3, 2, 5, 4, 6)            # [j][c][e][dims' group][block][8]
    kb = (kc[..., 0::2] | kc[..., 1::2] << 4).to(torch.uint8).reshape(n, -1)
    vc = vc.reshape(n, 2, 2, 4, nb // 2, 2, 8, 4).permute(0, 4, 6, 3, 5, 1, 2, 7)  # [block / 2][dims' group][c][block % 2][i / 2][i % 2][4]
    vb = (vc[..., 0::2] | vc[..., 1::2] << 4).to(torch.uint8).reshape(n, -1)
    sc = [d.contiguous().view(torch.uint8).reshape(n, -1) for d in (kd.reshape(n, 2, 2, 4, nb).permute(0, 3, 2, 1, 4), vd.reshape(n, 4, 4, nb).permute(0, 2, 3, 1))]
    return torch.cat([kb, vb] + sc, 1).reshape(*lead, -1)


def _unpack(tiles):
    """bytes [tiles..., 18 * head_dim] -> K and V values in float32 [tiles..., 16, head_dim]"""
    lead, hd = tiles.shape[:-1], tiles.shape[-1] // 18
    nb, n = hd // 32, math.prod(lead)
    t = tiles.reshape(n, 18 * hd)
    kb, vb, ks, vs = t.split([8 * hd, 8 * hd, hd, hd], 1)
    kc = torch.stack([kb & 15, kb >> 4], -1).reshape(n, 2, 4, 2, 4, nb, 8).permute(0, 1, 3, 2, 5, 4, 6).reshape(n, 16, nb, 32)
    vc = torch.stack([vb & 15, vb >> 4], -1).reshape(n, nb // 2, 8, 4, 2, 2, 2, 4).permute(0, 5, 6, 3, 1, 4, 2, 7).reshape(n, 16, nb, 32)
    kd = ks.contiguous().view(torch.float16).reshape(n, 4, 2, 2, nb).permute(0, 3, 2, 1, 4).reshape(n, 16, nb, 1)
    vd = vs.contiguous().view(torch.float16).reshape(n, 4, nb, 4).permute(0, 3, 1, 2).reshape(n, 16, nb, 1)
    return [((c.float() - 8) * d.float()).reshape(*lead, 16, hd) for c, d in ((kc, kd), (vc, vd))]


def _values(gen, shape, device):
    """keys or values as a model makes them: some channels much larger than others"""
    x = torch.randn(shape, generator=gen, device=device)
    return x * torch.exp(0.7 * torch.randn(shape[-1], generator=gen, device=device))


def _filled_pool(gen, layers, pages, shape, page, device):
    _, kv, hd = HEADS[shape]
    pool = torch.empty(layers, pages, kv, page // 16, 18 * hd, dtype=torch.uint8, device=device)
    step = max(1, (1 << 25) // (kv * page * hd))
    for layer in range(layers):
        for p in range(0, pages, step):
            dims = (min(step, pages - p), kv, page // 16, 16, hd)
            pool[layer, p:p + step] = _pack(_values(gen, dims, device), _values(gen, dims, device))
    return pool


def _tables(seed, slots, counts, page, pages, free_rows=0):
    """a table of pages in no order: slot slots[s] holds counts[s] tokens; all in plain numbers"""
    r = random.Random(seed)
    order = list(range(pages))
    r.shuffle(order)
    width = max(1, max(-(-c // page) for c in counts))
    table = [[-1] * width for _ in range(max(slots) + 1 + free_rows)]
    for s, c in zip(slots, counts):
        for i in range(-(-c // page)):
            table[s][i] = order.pop()
    return table, width


# ---- inputs ------------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    device = "cuda"
    gen = torch.Generator(device=device).manual_seed(seed)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=device)  # noqa: E731
    if case["kind"] == "sample":
        rows, vocab, t = case["rows"], case["vocab"], TYPES[case["dtype"]]
        logits = torch.randn(rows, vocab, generator=gen, device=device) * 2.2
        peaks = torch.randint(0, vocab, (rows, 12), generator=gen, device=device)
        logits.scatter_add_(1, peaks, 6 + 3 * torch.randn(rows, 12, generator=gen, device=device))
        r = random.Random(seed)
        # a server's requests differ: the defaults (40, 0.95, 0.05), nucleus alone, min-p alone, nothing, the most likely token
        kinds = [(40, 0.95, 0.05, 0.8), (40, 0.95, 0.05, 0.8), (0, 0.9, 0.0, 1.0), (0, 1.0, 0.1, 1.3), (200, 1.0, 0.0, 1.0), (0, 1.0, 0.0, 0.7), (5, 0.5, 0.0, 0.0)]
        picks = [kinds[0] if case["truncated"] else r.choice(kinds) for _ in range(rows)]
        col = lambda i, t: torch.tensor([p[i] for p in picks], dtype=t, device=device)  # noqa: E731
        return dict(case=case, logits=logits.to(t), u=torch.rand(rows, generator=gen, device=device), top_k=col(0, torch.int32), top_p=col(1, torch.float32),
                    min_p=col(2, torch.float32), temperature=col(3, torch.float32))
    heads, kv, hd = HEADS[case["shape"]]
    held, page = _held(case), case["page"]
    if case["kind"] in ("fork", "compact"):
        n = case["seqs"]
        slots = list(range(2 * n))
        random.Random(seed + 1).shuffle(slots)
        table, _ = _tables(seed, slots[:n], held, page, case["pages"])
        table += [[-1] * len(table[0]) for _ in range(2 * n - len(table))]
        at, refs = [0] * (2 * n), [0] * case["pages"]
        for s, c in zip(slots, held):
            at[s] = c
        if case["kind"] == "compact":  # every third conversation has a second one that began with the same full pages
            for i in range(0, n, 3):
                full = held[i] // page
                table[slots[n + i]][:full], at[slots[n + i]] = table[slots[i]][:full], full * page
        for row in table:
            for p in row:
                if p >= 0:
                    refs[p] += 1
        return dict(case=case, pool=_filled_pool(gen, case["layers"], case["pages"], case["shape"], page, device), table=ints(table), held=ints(at), refs=ints(refs),
                    parents=ints(slots[:n]), children=ints(slots[n:]), ended=ints(slots[:n][: (n + 2) // 3]))
    counts = _counts(case)
    slots = list(range(case["seqs"]))
    random.Random(seed + 1).shuffle(slots)
    after = [h + c for h, c in zip(held, counts)]
    pages = sum(-(-a // page) for a in after) + 3
    table, _ = _tables(seed, slots, after, page, pages)
    at = [0] * len(slots)
    for s, h in zip(slots, held):
        at[s] = h
    first = [0]
    for c in counts:
        first.append(first[-1] + c)
    t = TYPES[case["dtype"]]
    state = dict(case=case, pool=_filled_pool(gen, 1, pages, case["shape"], page, device)[0], table=ints(table), held=ints(at), first=ints(first), slots=ints(slots),
                 max_rows=max(counts), longest=max(after))
    if case["kind"] == "append":
        # keys and values stand in the rows of one product, behind the queries
        qkv = _values(gen, (first[-1], (heads + 2 * kv) * hd), device).to(t)
        state["k"] = qkv[:, heads * hd:(heads + kv) * hd].unflatten(1, (kv, hd))
        state["v"] = qkv[:, (heads + kv) * hd:].unflatten(1, (kv, hd))
    else:
        state["q"] = (1.5 * torch.randn(first[-1], heads, hd, generator=gen, device=device)).to(t)
    return state


# ---- one pass ----------------------------------------------------------------------------------------------------------------
def run(state):
    return {"attend": _attend, "append": _append, "fork": _fork, "compact": _compact, "sample": _sample}[state["case"]["kind"]](state)


def _places(s):
    """for each row its sequence, its slot and its position"""
    rows = torch.arange((s["k"] if "k" in s else s["q"]).shape[0], device=s["first"].device)
    seq = torch.searchsorted(s["first"], rows, right=True) - 1
    slot = s["slots"][seq]
    return seq, slot, s["held"][slot] + rows - s["first"][seq]


def _attend(s):
    case = s["case"]
    if own:
        from booster_b200 import serve
        return serve.kv4_attention(s["q"], s["pool"], s["table"], s["held"], s["first"], slots=s["slots"], window=case["window"], max_rows=s["max_rows"])
    q, page, longest = s["q"].float(), case["page"], s["longest"]
    n, kv, hd = len(s["slots"]), s["pool"].shape[1], q.shape[-1]
    seq, _, pos = _places(s)
    pages = s["table"][s["slots"].long()][:, : -(-longest // page)]
    k, v = _unpack(s["pool"][pages.clamp_min(0).long()])                       # [n][pages][kv][tiles][16][hd]
    k, v = (x.transpose(1, 2).reshape(n, kv, -1, hd) for x in (k, v))
    j = torch.arange(k.shape[2], device=q.device)
    there = (pages >= 0).repeat_interleave(page, 1)
    # rows side by side, sequence by sequence, as [n][kv][group * max_rows]
    i = torch.arange(len(seq), device=q.device) - s["first"][seq]
    m = s["max_rows"]
    group = q.shape[1] // kv
    wide = q.new_zeros(n, m, kv, group, hd)
    wide[seq, i] = q.unflatten(1, (kv, group))
    p = torch.full((n, m), -1, dtype=torch.long, device=q.device)
    p[seq, i] = pos.long()
    p = p.unsqueeze(-1)
    sees = (j <= p) & there.unsqueeze(1)
    if case["window"]:
        sees &= j > p - case["window"]
    score = torch.einsum("nmkgd,nkjd->nkgmj", wide, k) * hd ** -0.5
    score = score.masked_fill(~sees[:, None, None], float("-inf"))
    top = score.amax(-1, keepdim=True).clamp_min(-1e30)
    w = torch.exp(score - top)
    out = torch.einsum("nkgmj,nkjd->nmkgd", w / w.sum(-1, keepdim=True).clamp_min(1e-30), v)
    return out[seq, i].reshape(s["q"].shape).to(s["q"].dtype)


def _append(s):
    if own:
        from booster_b200 import serve
        serve.kv4_append(s["pool"], s["table"], s["held"], s["first"], s["k"], s["v"], slots=s["slots"])
        return serve.kv4_read(s["pool"], s["table"], s["held"], s["first"], len(s["k"]), dtype=s["k"].dtype, slots=s["slots"])
    page, pool = s["case"]["page"], s["pool"]
    _, slot, pos = _places(s)
    pages, kv, tiles, _ = pool.shape
    hd, nb = s["k"].shape[-1], s["k"].shape[-1] // 32
    at = s["table"][slot.long(), (pos // page).long()].long()
    tile, t = (pos % page // 16).long(), (pos % 16).long()
    c, i = t % 4, t // 4
    kc, kd, vc, vd = _codes(s["k"], s["v"])
    lo = lambda x: (x[..., 0::2] | x[..., 1::2] << 4).to(torch.uint8)  # noqa: E731
    # each field of the tile as the array that _pack describes, and the new rows' places in it
    kf = pool[..., : 8 * hd].unflatten(-1, (2, 4, 2, 4, nb, 4))
    kf[at, :, tile, i // 2, c, i % 2] = lo(kc.unflatten(-1, (nb, 4, 8)).transpose(2, 3))
    vf = pool[..., 8 * hd:16 * hd].unflatten(-1, (nb // 2, 8, 4, 2, 2, 2, 2))
    vf.permute(0, 2, 5, 7, 8, 1, 3, 6, 4, 9)[at, tile, c, i // 2, i % 2] = lo(vc.unflatten(-1, (nb // 2, 2, 8, 4)))
    pool[..., 16 * hd:17 * hd].view(torch.float16).unflatten(-1, (4, 2, 2, nb)).permute(0, 2, 3, 4, 5, 1, 6)[at, tile, c, i % 2, i // 2] = kd
    pool[..., 17 * hd:].view(torch.float16).unflatten(-1, (4, nb, 4)).permute(0, 2, 3, 5, 1, 4)[at, tile, c, i] = vd
    k, v = _unpack(pool[at, :, tile])
    r = torch.arange(len(at), device=at.device)
    return k[r, :, t].to(s["k"].dtype), v[r, :, t].to(s["v"].dtype)


def _fork(s):
    table, held, refs = s["table"].clone(), s["held"].clone(), s["refs"].clone()
    if own:
        from booster_b200 import serve
        status = serve.pages_fork(s["pool"], table, held, refs, s["parents"], s["children"])
        return dict(pool=s["pool"], table=table, held=held, refs=refs, status=status)
    page, pool = s["case"]["page"], s["pool"]
    parents, children = s["parents"].long(), s["children"].long()
    tokens, rows = held[parents], table[parents]
    full = torch.arange(table.shape[1], device=table.device) < (tokens // page).unsqueeze(1)
    refs.scatter_add_(0, torch.where(full, rows, 0).long().flatten(), full.int().flatten())
    # a page that is part full is copied, as far as its tiles hold tokens, to the lowest free page
    rest = tokens % page
    part = rest > 0
    free = torch.argsort((refs != 0).int(), stable=True)[: len(parents)]
    order = torch.where(part, part.cumsum(0) - 1, part.sum() + (~part).cumsum(0) - 1)
    status = torch.zeros(1, dtype=torch.int32, device=table.device)
    got = free[order]
    where = (tokens // page).clamp_max(table.shape[1] - 1).long()
    source = rows.gather(1, where[:, None])[:, 0]
    new = torch.where(full, rows, -1)
    last = torch.where(part, got.int(), new.gather(1, where[:, None])[:, 0])
    new.scatter_(1, where[:, None], last[:, None])
    table[children], held[children] = new, tokens
    refs.scatter_add_(0, torch.where(part, got, 0), part.int())
    keep = torch.arange(page // 16, device=table.device) < ((rest + 15) // 16).unsqueeze(1)             # [n][tiles]
    copied = torch.where(keep[None, :, None, :, None], pool[:, source.clamp_min(0).long()], pool[:, got])
    pool[:, got] = torch.where(part[None, :, None, None, None], copied, pool[:, got])
    return dict(pool=pool, table=table, held=held, refs=refs, status=status)


def _compact(s):
    table, held, refs = s["table"].clone(), s["held"].clone(), s["refs"].clone()
    if own:
        from booster_b200 import serve
        serve.pages_free(table, held, refs, s["ended"])
        live = serve.pages_compact(s["pool"], table, refs)
        return dict(pool=s["pool"], table=table, held=held, refs=refs, live=live)
    pool, ended = s["pool"], s["ended"].long()
    gone = table[ended].flatten()
    refs.scatter_add_(0, gone.clamp_min(0).long(), -(gone >= 0).int())
    table[ended], held[ended] = -1, 0
    used = refs > 0
    live = used.sum(dtype=torch.int32)
    n = torch.arange(len(refs), device=refs.device)
    # the lowest free page takes the lowest page in use behind the live ones' number, and so on
    hole, moved = ~used & (n < live), used & (n >= live)
    movers = moved.nonzero()[:, 0]
    holes = hole.nonzero()[: len(movers), 0]
    to = n.clone()
    to[movers] = holes
    table = torch.where(table >= 0, to[table.clamp_min(0).long()].int(), table)
    refs[holes] = refs[movers]
    refs[movers] = 0
    pool[:, holes] = pool[:, movers]
    return dict(pool=pool, table=table, held=held, refs=refs, live=live.reshape(1))


def _sample(s):
    if own:
        from booster_b200 import serve
        return serve.sample(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])
    x = s["logits"].double()
    t, k = s["temperature"].double()[:, None], s["top_k"][:, None]
    top, order = torch.sort(x, dim=1, descending=True, stable=True)
    delta = top - top[:, :1]
    w = torch.exp(delta)
    rank = torch.arange(x.shape[1], device=x.device)
    w1 = torch.where((rank < k) | (k <= 0), w, 0)
    total, before = w1.sum(1, keepdim=True), torch.cumsum(w1, 1) - w1
    p, q = s["top_p"].double()[:, None], s["min_p"].double()[:, None]
    kept = (w1 > 0) & ((before < p * total) | (p >= 1)) & (w >= q)
    tempered = torch.where(kept, torch.exp(delta / torch.where(t > 0, t, 1.0)), 0)
    placed = torch.zeros_like(x).scatter_(1, order, tempered)
    run_ = torch.cumsum(placed, 1)
    sum_ = run_[:, -1:]
    token = (run_ <= s["u"].double()[:, None] * sum_).sum(1)
    token = torch.where(t[:, 0] > 0, token, order[:, 0])
    share = torch.log(placed.gather(1, token[:, None]) / sum_)[:, 0]
    return token.int(), torch.where(t[:, 0] > 0, share, 0.0).float()


# ---- what a pass cannot do without -------------------------------------------------------------------------------------------
def work(case):
    if case["kind"] == "sample":
        size = {"float32": 4, "bfloat16": 2, "float16": 2}[case["dtype"]]
        return {"bytes": case["rows"] * (case["vocab"] * size + 28), "flops": 2 * case["rows"] * case["vocab"]}
    heads, kv, hd = HEADS[case["shape"]]
    held, page = _held(case), case["page"]
    if case["kind"] == "fork":
        tiles = sum(-(-(h % page) // 16) for h in held)
        return {"bytes": 2 * case["layers"] * kv * tiles * 18 * hd, "flops": 0}
    if case["kind"] == "compact":
        # pages are in no order: of the live ones, the share that lies behind their number
        ended = (case["seqs"] + 2) // 3
        live = sum(-(-h // page) for h in held[ended:]) + sum(h // page for h in held[:ended:3])
        return {"bytes": 2 * case["layers"] * kv * (page // 16) * 18 * hd * live * (1 - live / case["pages"]) + 8 * case["pages"], "flops": 0}
    counts = _counts(case)
    size = {"float32": 4, "bfloat16": 2, "float16": 2}[case["dtype"]]
    if case["kind"] == "append":
        return {"bytes": sum(counts) * kv * hd * (4 * size + 2 * 1.125), "flops": 0}
    seen = [_seen(h, c, case["window"]) for h, c in zip(held, counts)]
    return {"bytes": 1.125 * hd * kv * sum(t for _, t in seen) + 2 * size * sum(counts) * heads * hd, "flops": 4 * hd * heads * sum(p for p, _ in seen)}


# ---- the same in 64 bits, from the definitions -------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "attend":
        return _exact_attend(case, s)
    if case["kind"] == "append":
        return [_exact_rows(s["k"], s["k"], s["v"], True), _exact_rows(s["v"], s["k"], s["v"], False)]
    if case["kind"] == "sample":
        return _exact_sample(s)
    return None


def _exact_rows(x, k, v, keys):
    b = x.double().reshape(*x.shape[:-1], -1, 32)
    low, high = b.min(-1).values, b.max(-1).values
    scale = torch.clamp(torch.where(low.abs() >= high, low, high) * -0.125, -8160.0, 8160.0).to(torch.bfloat16).to(torch.float16).double()[..., None]
    held = torch.clamp(torch.round(b / scale), -8, 7) * scale
    held = torch.where(scale == 0, torch.zeros_like(held), held).reshape(x.shape)
    whole = (torch.isfinite(k).all(-1) & torch.isfinite(v).all(-1))[..., None]
    return torch.where(whole, held, torch.full_like(held, float("nan") if keys else 0.0))


def _exact_tile(raw):
    """codes and scales of tiles [n, 18 * hd] -> K, V [n, 16, hd] in float64, place by place"""
    n, hd = raw.shape[0], raw.shape[1] // 18
    t, d = np.meshgrid(np.arange(16), np.arange(hd), indexing="ij")
    c, i, block, nb = t % 4, t // 4, d // 32, hd // 32
    word = (((i // 2) * 8 + 2 * c + i % 2) * 4 + d % 32 // 8) * nb + block
    kbyte, khigh = word * 4 + d % 8 // 2, d % 2
    unit = ((((block // 2) * 8 + d % 32 // 4) * 4 + c) * 2 + block % 2) * 4 + i
    vbyte, vhigh = 8 * hd + unit * 2 + d % 4 // 2, d % 2
    kscale, vscale = ((c * 2 + i % 2) * 2 + i // 2) * nb + block, (c * nb + block) * 4 + i
    out = []
    for byte, high, scale, begin in ((kbyte, khigh, kscale, 16 * hd), (vbyte, vhigh, vscale, 17 * hd)):
        b = raw[:, torch.from_numpy(byte).to(raw.device)].int()
        code = torch.where(torch.from_numpy(high).to(raw.device) > 0, b // 16, b % 16)
        f = raw[:, begin:begin + hd].contiguous().view(torch.float16).double()[:, torch.from_numpy(scale).to(raw.device)]
        out.append((code - 8).double() * f)
    return out


def _exact_attend(case, s):
    heads, kv, hd = HEADS[case["shape"]]
    page, group = case["page"], heads // kv
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    held, counts, table, slots = _held(case), _counts(case), s["table"].tolist(), s["slots"].tolist()
    row = 0
    for h, c, slot in zip(held, counts, slots):
        last = h + c
        raw = s["pool"][torch.tensor(table[slot][: -(-last // page)], device=out.device)]
        k, v = (x.reshape(raw.shape[0], kv, page // 16, 16, hd).permute(1, 0, 2, 3, 4).reshape(kv, -1, hd)[:, :last] for x in _exact_tile(raw.reshape(-1, 18 * hd)))
        for a in range(0, c, 64):
            b = min(c, a + 64)
            q = s["q"][row + a:row + b].double()
            p = torch.arange(h + a, h + b, device=out.device)[:, None]
            j = torch.arange(last, device=out.device)[None]
            hidden = (j > p) if not case["window"] else (j > p) | (j <= p - case["window"])
            for g in range(kv):
                logit = torch.matmul(q[:, g * group:(g + 1) * group].transpose(0, 1), k[g].T) / math.sqrt(hd)
                out[row + a:row + b, g * group:(g + 1) * group] = torch.matmul(torch.softmax(logit.masked_fill(hidden[None], -math.inf), -1), v[g]).transpose(0, 1)
        row += c
    return out


def _exact_sample(s):
    logits = s["logits"].double().cpu().numpy()
    u, temperature, top_p, min_p = (s[n].double().cpu().numpy() for n in ("u", "temperature", "top_p", "min_p"))
    shares = []
    for r, x in enumerate(logits):
        order = np.lexsort((np.arange(len(x)), -x))
        k = int(s["top_k"][r])
        order = order[:k] if k > 0 else order
        w = np.exp(x[order] - x[order[0]])
        if top_p[r] < 1:
            order = order[: 1 + int(np.searchsorted(np.cumsum(w), top_p[r] * w.sum()))]
        order = order[np.exp(x[order] - x[order[0]]) >= min_p[r]]
        if temperature[r] <= 0:
            shares.append(0.0)
            continue
        order = np.sort(order)
        w = np.exp((x[order] - x.max()) / temperature[r])
        c = np.cumsum(w)
        at = int(np.searchsorted(c, u[r] * c[-1], side="right"))
        shares.append(math.log(w[at] / c[-1]))
    return [None, np.array(shares)]
