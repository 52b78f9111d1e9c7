"""The operators of a server that drafts tokens ahead and keeps its cache in 16 bits, as they are measured: attention over a paged cache of 16-bit keys and values, under a sliding
window with first tokens that stay visible if asked; the rows that are written into it; the tables of a step (pages that nobody sees any more given back, pages and places for the
next rows made from their numbers); and the verification of drafted tokens against the target's logits.

Where `own` is true, `run` calls booster_b200.serve; otherwise it computes the same in elementary torch operations. A pool is [pages, 2 (keys, values), KV heads, page tokens, head_dim];
pages stand scattered over it, and the pool's other pages hold what earlier sequences left.
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
        dict(name="attend-one-at-333", kind="attend", shape="8b", seqs=1, lo=333, hi=333, rows=1, page=16, window=0, sinks=0, dtype="bfloat16"),
        # a busy server: one new token of 48 conversations of very different length
        dict(name="attend-48-ragged", kind="attend", shape="8b", seqs=48, lo=90, hi=4090, rows=1, page=64, window=0, sinks=0, dtype="bfloat16"),
        # endless conversations that see their last 1000 tokens and their first four, heads of 64, an odd number of them
        dict(name="attend-61-sinks", kind="attend", shape="half", seqs=61, lo=5, hi=12000, rows=1, page=32, window=1000, sinks=4, dtype="float16"),
        # five rows each (a token and four drafted ones) of few long documents, under a large model's heads
        dict(name="attend-drafts-6-long", kind="attend", shape="70b", seqs=6, lo=9001, hi=30000, rows=5, page=128, window=0, sinks=0, dtype="bfloat16"),
        # the next portion of a long prompt behind a conversation
        dict(name="attend-prompt-1000-at-5000", kind="attend", shape="8b", seqs=1, lo=5000, hi=5000, rows=1000, page=64, window=0, sinks=0, dtype="bfloat16"),
        # several prompts' portions in one pass, ragged, under a window with sinks
        dict(name="attend-prompts-window", kind="attend", shape="8b", seqs=5, lo=0, hi=1500, rows=1100, page=32, window=700, sinks=20, dtype="float16"),
        # the step's new rows of a batch of conversations
        dict(name="append-48", kind="append", shape="8b", seqs=48, lo=90, hi=1090, rows=1, page=64, dtype="bfloat16", source="bfloat16"),
        # long prompts' rows, from 32 bits
        dict(name="append-prompts-8193", kind="append", shape="8b", seqs=3, lo=7, hi=700, rows=2731, page=64, dtype="float16", source="float32"),
        # between two steps of 48 conversations with up to seven drafted tokens, some of which were refused
        dict(name="tables-48-drafts", kind="tables", seqs=48, lo=90, hi=4090, rows=5, page=64, pages=4096, window=0, sinks=0),
        # the same of 300 conversations under a window, and three prompts' portions among their rows
        dict(name="tables-300-window", kind="tables", seqs=300, lo=5, hi=9000, rows=900, page=32, pages=60000, window=2000, sinks=4),
        # one user, four tokens that were looked up in the text so far
        dict(name="verify-one", kind="verify", seqs=1, rows=5, vocab=128256, dtype="float32", drafter=False, truncated=True),
        # a busy server: up to five drafted tokens each and the distributions that they were drawn from, requests that filter in all ways
        dict(name="verify-48", kind="verify", seqs=48, rows=6, vocab=128256, dtype="float32", drafter=True, truncated=False),
    ]


def _spread(rng, lo, hi):
    """a whole number from lo to hi, spread over its logarithm"""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "prompt", "prompt", "append", "tables", "verify", "verify"])
    shape, page, dtype = rng.choice(sorted(HEADS)), rng.choice([16, 32, 64, 128]), rng.choice(["bfloat16", "float16"])
    heads, kv, hd = HEADS[shape]
    window = rng.choice([0, 0, _spread(rng, 1, 4000)])
    sinks = rng.choice([0, 4, _spread(rng, 1, 300)]) if window else 0
    if kind == "attend":
        hi = _spread(rng, 1, 32000)
        seqs = _spread(rng, 1, max(1, min(200, 80000 * 1024 // (hi * kv * hd))))
        return dict(kind="attend", shape=shape, seqs=seqs, lo=rng.randrange(0, hi + 1), hi=hi, rows=rng.choice([1, 1, 1, 2, 5, 8]), page=page, window=window, sinks=sinks, dtype=dtype)
    if kind == "prompt":
        hi, seqs = _spread(rng, 1, 6000), rng.choice([1, 1, 2, 3])
        rows = _spread(rng, 9, max(16, min(1000, 32 * 128 * 700 * 6000 // (heads * hd * seqs * (hi + 1000)))))
        return dict(kind="attend", shape=shape, seqs=seqs, lo=rng.randrange(0, hi + 1), hi=hi, rows=rows, page=page, window=window, sinks=sinks, dtype=dtype)
    if kind == "append":
        seqs = _spread(rng, 1, 200)
        return dict(kind="append", shape=shape, seqs=seqs, lo=rng.randrange(0, 50), hi=rng.randrange(50, 1000), rows=_spread(rng, 1, max(1, 3000 // seqs)), page=page, dtype=dtype,
                    source=rng.choice([dtype, dtype, "float32"]))
    if kind == "tables":
        seqs, hi, rows = _spread(rng, 1, 300), _spread(rng, 20, 9000), rng.choice([1, 5, 8, _spread(rng, 9, 900)])
        return dict(kind="tables", seqs=seqs, lo=rng.randrange(1, hi + 1), hi=hi, rows=rows, page=page, pages=seqs * ((hi + rows) // page + 3) + rng.randrange(0, 5000), window=window, sinks=sinks)
    return dict(kind="verify", seqs=_spread(rng, 1, 48), rows=rng.randrange(1, 6), vocab=_spread(rng, 200, 128256), dtype=rng.choice(["float32", "bfloat16", "float16"]),
                drafter=rng.choice([True, False]), truncated=rng.choice([True, False]))


# ---- sizes that a case stands for, the same for every seed ------------------------------------------------------------------
def _between(lo, hi, n, turn):
    return [lo + int((hi - lo + 1) * ((turn + 0.618034 * i) % 1.0)) for i in range(n)]


def _held(case):
    """tokens of each sequence before the step"""
    return [min(case["hi"], v) for v in _between(case["lo"], case["hi"], case["seqs"], 0.37)]


def _counts(case):
    """new rows of each sequence: a token and its drafts, ragged around `rows` for portions of prompts"""
    r, n = case["rows"], case["seqs"]
    if case["kind"] == "verify":
        return [min(r, v) for v in _between(1, r, n, 0.81)] if n > 1 else [r]
    if case["kind"] == "tables" and r > 8:  # three prompts among single tokens
        return [max(1, r - 17 * i) if i < 3 else 1 for i in range(n)]
    if r <= 8 or n == 1:
        return [r] * n
    return [max(1, v) for v in _between(r // 3, r, n, 0.81)]


def _seen(held, count, window, sinks):
    """(pairs of a row and a position that it sees, positions that some row sees)"""
    pairs = 0
    for i in range(count):
        p = held + i + 1
        pairs += min(p, window + min(sinks, max(0, p - window))) if window else p
    last = held + count
    if not window:
        return pairs, last
    own_ = min(last, window + count - 1)
    return pairs, own_ + min(sinks, last - own_)


# ---- inputs ------------------------------------------------------------------------------------------------------------------
def _values(gen, shape, device):
    """keys or values as a model makes them: some channels much larger than others"""
    x = torch.randn(shape, generator=gen, device=device)
    return x * torch.exp(0.7 * torch.randn(shape[-1], generator=gen, device=device))


def _filled_pool(gen, pages, shape, page, dtype, device):
    _, kv, hd = HEADS[shape]
    pool = torch.empty(pages, 2, kv, page, hd, dtype=dtype, device=device)
    step = max(1, (1 << 26) // (2 * kv * page * hd))
    for p in range(0, pages, step):
        pool[p:p + step] = _values(gen, pool[p:p + step].shape, device).to(dtype)
    return pool


def _tables(seed, slots, counts, page, pages):
    """a table of pages in no order: slot slots[s] holds counts[s] tokens; all in plain numbers"""
    r = random.Random(seed)
    order = list(range(pages))
    r.shuffle(order)
    width = max(1, max(-(-c // page) for c in counts))
    table = [[-1] * width for _ in range(max(slots) + 1)]
    for s, c in zip(slots, counts):
        for i in range(-(-c // page)):
            table[s][i] = order.pop()
    return table, width


def prepare(case, seed):
    device = "cuda"
    gen = torch.Generator(device=device).manual_seed(seed)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=device)  # noqa: E731
    counts = _counts(case)
    first = [0]
    for c in counts:
        first.append(first[-1] + c)
    if case["kind"] == "verify":
        rows, vocab, t = first[-1], case["vocab"], TYPES[case["dtype"]]
        logits = torch.randn(rows, vocab, generator=gen, device=device) * 2.2
        peaks = torch.randint(0, vocab, (rows, 12), generator=gen, device=device)
        logits.scatter_add_(1, peaks, 6 + 3 * torch.randn(rows, 12, generator=gen, device=device))
        # a drafter is a smaller model that mostly agrees; what is looked up in the text is the likeliest token or any
        drafter = logits + 0.8 * torch.randn(rows, vocab, generator=gen, device=device)
        probs = torch.softmax(drafter / 0.8, 1) if case["drafter"] else None
        if case["drafter"]:
            guess = torch.multinomial(probs, 1, generator=gen)[:, 0]
        else:
            guess = torch.where(torch.rand(rows, generator=gen, device=device) < 0.8, logits.argmax(1), peaks[:, 0])
        ids = torch.cat([torch.randint(0, vocab, (1,), generator=gen, device=device), guess[:-1]]).int()
        r = random.Random(seed)
        # requests differ: the defaults (40, 0.95, 0.05), nucleus alone, min-p alone, nothing, the most likely token
        kinds = [(40, 0.95, 0.05, 0.8), (40, 0.95, 0.05, 0.8), (0, 0.9, 0.0, 1.0), (0, 1.0, 0.1, 1.3), (200, 1.0, 0.0, 1.0), (0, 1.0, 0.0, 0.7), (5, 0.5, 0.0, 0.0)]
        picks = []
        for c in counts:
            picks += [kinds[0] if case["truncated"] else r.choice(kinds)] * c
        col = lambda i, t: torch.tensor([p[i] for p in picks], dtype=t, device=device)  # noqa: E731
        return dict(case=case, logits=logits.to(t), ids=ids, first=ints(first), u=torch.rand(rows, generator=gen, device=device), accept=torch.rand(rows, generator=gen, device=device),
                    temperature=col(3, torch.float32), top_k=col(0, torch.int32), top_p=col(1, torch.float32), min_p=col(2, torch.float32), probs=probs)
    held, page = _held(case), case["page"]
    slots = list(range(case["seqs"]))
    random.Random(seed + 1).shuffle(slots)
    at = [0] * len(slots)
    for s, h in zip(slots, held):
        at[s] = h
    if case["kind"] == "tables":
        # the pages of rows that were refused stand behind the tokens that are held, up to eight of them; a third of the first pages has a second holder
        r = random.Random(seed + 2)
        table, _ = _tables(seed, slots, [h + r.randrange(0, 9) for h in held], page, case["pages"])
        width = max(-(-(h + c) // page) for h, c in zip(held, counts))
        table = [row + [-1] * max(0, width - len(row)) for row in table]
        refs = [0] * case["pages"]
        for row in table:
            for p in row:
                if p >= 0:
                    refs[p] = 1
        for s in slots[::3]:
            refs[table[s][0]] = 2
        return dict(case=case, table=ints(table), held=ints(at), refs=ints(refs), slots=ints(slots), counts=ints(counts), rows=first[-1] + 7)
    after = [h + c for h, c in zip(held, counts)]
    pages = sum(-(-a // page) for a in after) + 3
    table, _ = _tables(seed, slots, after, page, pages)
    t = TYPES[case["dtype"]]
    state = dict(case=case, pool=_filled_pool(gen, pages, case["shape"], page, t, device), table=ints(table), held=ints(at), first=ints(first), slots=ints(slots), max_rows=max(counts),
                 longest=max(after))
    heads, kv, hd = HEADS[case["shape"]]
    if case["kind"] == "append":
        # keys and values stand in the rows of one product, behind the queries
        qkv = _values(gen, (first[-1], (heads + 2 * kv) * hd), device).to(TYPES[case["source"]])
        state["k"] = qkv[:, heads * hd:(heads + kv) * hd].unflatten(1, (kv, hd))
        state["v"] = qkv[:, (heads + kv) * hd:].unflatten(1, (kv, hd))
    else:
        state["q"] = (1.5 * torch.randn(first[-1], heads, hd, generator=gen, device=device)).to(t)
    return state


# ---- one pass ----------------------------------------------------------------------------------------------------------------
def run(state):
    return {"attend": _attend, "append": _append, "tables": _tables_of_a_step, "verify": _verify}[state["case"]["kind"]](state)


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
        return serve.kv16_attention(s["q"], s["pool"], s["table"], s["held"], s["first"], slots=s["slots"], window=case["window"], sinks=case["sinks"], max_rows=s["max_rows"])
    q, page, longest = s["q"].float(), case["page"], s["longest"]
    n, kv, hd = len(s["slots"]), s["pool"].shape[2], q.shape[-1]
    seq, _, pos = _places(s)
    pages = s["table"][s["slots"].long()][:, : -(-longest // page)]
    kv_all = s["pool"][pages.clamp_min(0).long()]                                # [n][pages][2][kv][page][hd]
    k, v = (kv_all[:, :, i].transpose(1, 2).reshape(n, kv, -1, hd).float() for i in (0, 1))
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
        sees &= (j > p - case["window"]) | (j < case["sinks"])
    score = torch.einsum("nmkgd,nkjd->nkgmj", wide, k) * hd ** -0.5
    score = score.masked_fill(~sees[:, None, None], float("-inf"))
    top = score.amax(-1, keepdim=True).clamp_min(-1e30)
    w = torch.exp(score - top)
    out = torch.einsum("nkgmj,nkjd->nmkgd", w / w.sum(-1, keepdim=True).clamp_min(1e-30), v)
    return out[seq, i].reshape(s["q"].shape).to(s["q"].dtype)


def _append(s):
    if own:
        from booster_b200 import serve
        serve.kv16_append(s["pool"], s["table"], s["held"], s["first"], s["k"], s["v"], slots=s["slots"])
        return s["pool"]
    page, pool = s["case"]["page"], s["pool"]
    _, slot, pos = _places(s)
    at = s["table"][slot.long(), (pos // page).long()].long()
    # a token that holds an infinity or a NaN in a head: its key NaN, its value 0
    k, v = s["k"].to(pool.dtype), s["v"].to(pool.dtype)
    fine = torch.isfinite(k).all(-1, keepdim=True) & torch.isfinite(v).all(-1, keepdim=True)
    pool[at, 0, :, (pos % page).long()] = torch.where(fine, k, float("nan"))
    pool[at, 1, :, (pos % page).long()] = torch.where(fine, v, 0.0)
    return pool


def _tables_of_a_step(s):
    """what stands behind the tokens that are held or in front of the window goes back; then pages, places and positions for the next rows"""
    case, slots, rows = s["case"], s["slots"], s["rows"]
    table, refs, held, page = s["table"].clone(), s["refs"].clone(), s["held"], s["case"]["page"]
    if own:
        from booster_b200 import serve
        serve.pages_trim(table, held, refs, page, slots, window=case["window"], sinks=case["sinks"])
        first, positions, places, status = serve.pages_plan(table, held, refs, s["counts"], page, rows, slots)
        return dict(table=table, refs=refs, first=first, positions=positions, places=places, status=status)
    at = slots.long()
    mine, h = table[at], held[at].unsqueeze(1)
    i = torch.arange(table.shape[1], device=table.device)
    keep = i < (h + page - 1) // page
    if case["window"]:
        keep &= (i * page < case["sinks"]) | ((i + 1) * page > h - case["window"] + 1)
    gone = ~keep & (mine >= 0)
    refs.scatter_add_(0, torch.where(gone, mine, 0).long().flatten(), -gone.int().flatten())
    mine = torch.where(keep, mine, -1)
    # pages for the new rows, the lowest free ones in order
    counts = s["counts"]
    after = h + counts.unsqueeze(1)
    wanted = (i >= (h + page - 1) // page) & (i < (after + page - 1) // page)
    order = torch.argsort((refs != 0).int(), stable=True).int()
    rank = wanted.flatten().cumsum(0).reshape(wanted.shape) - 1
    got = order[rank.clamp_min(0)]
    mine = torch.where(wanted, got, mine)
    refs.scatter_add_(0, torch.where(wanted, got, 0).long().flatten(), wanted.int().flatten())
    table[at] = mine
    first = torch.cat([counts.new_zeros(1), counts.cumsum(0, dtype=torch.int32)])
    r = torch.arange(rows, device=table.device)
    seq = torch.searchsorted(first, r, right=True) - 1
    inside = seq < len(slots)
    seq = seq.clamp_max(len(slots) - 1)
    positions = torch.where(inside, h[seq, 0] + r - first[seq], -1).int()
    p = mine[seq, (positions.clamp_min(0) // page).long()]
    places = torch.where(inside, p * page + positions % page, -1).int()
    return dict(table=table, refs=refs, first=first, positions=positions, places=places, status=first.new_zeros(1))


def _verify(s):
    if own:
        from booster_b200 import serve
        return serve.verify(s["logits"], s["ids"], s["first"], s["u"], s["accept"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"], draft_probs=s["probs"])
    # the target's distribution as a draw has it: top-k, top-p, min-p, temperature, in 64 bits since tokens are decided by sums
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
    tempered = torch.where(t > 0, tempered, (rank == 0).double())
    share = torch.zeros_like(x).scatter_(1, order, tempered)
    share = share / share.sum(1, keepdim=True)
    # each row's draft is the next row's token; a sequence's last row has none
    rows, first, device = len(x), s["first"].long(), x.device
    r = torch.arange(rows, device=device)
    seq = torch.searchsorted(first, r, right=True) - 1
    last = r == first[seq + 1] - 1
    draft = torch.cat([s["ids"][1:], s["ids"][:1]]).long()
    if s["probs"] is None:
        q_all = torch.zeros_like(x).scatter_(1, draft[:, None], 1.0)
    else:
        q_all = s["probs"].double()
    p_x, q_x = share.gather(1, draft[:, None])[:, 0], q_all.gather(1, draft[:, None])[:, 0]
    taken = ~last & (s["accept"].double() * q_x < p_x)
    # drawn where a draft is refused: from what the target has more of than the drafter; behind the last draft: from the target
    rest = (share - q_all).clamp_min(0)
    rest = torch.where(last[:, None] | (rest.sum(1, keepdim=True) == 0), share, rest)
    run_ = torch.cumsum(rest, 1)
    drawn = (run_ <= s["u"].double()[:, None] * run_[:, -1:]).sum(1)
    drawn = torch.where(t[:, 0] > 0, drawn, order[:, 0])
    # a sequence ends with the first row whose draft is not taken
    stops = torch.where(taken, rows, r)
    stop = torch.full((len(first) - 1,), rows, device=device).scatter_reduce_(0, seq, stops, "amin")
    new = (stop - first[:-1] + 1).int()
    token = torch.where(r < stop[seq], draft, torch.where(r == stop[seq], drawn, -1))
    logprob = torch.where(t[:, 0] > 0, torch.log(share.gather(1, token.clamp_min(0)[:, None])[:, 0]), 0.0)
    return new, token.int(), torch.where(r <= stop[seq], logprob, 0.0).float()


# ---- what a pass cannot do without -------------------------------------------------------------------------------------------
def work(case):
    counts = _counts(case)
    rows = sum(counts)
    if case["kind"] == "verify":
        size = {"float32": 4, "bfloat16": 2, "float16": 2}[case["dtype"]]
        # a drafter's whole distribution is read where a draft is refused: once a sequence that has drafts
        refused = sum(c > 1 for c in counts) if case["drafter"] else 0
        return {"bytes": rows * (case["vocab"] * size + 40) + refused * case["vocab"] * 4, "flops": 2 * rows * case["vocab"]}
    held, page = _held(case), case["page"]
    if case["kind"] == "tables":
        # the counts of pages, the sequences' rows of the table and the new rows' places
        width = max(-(-(h + c) // page) for h, c in zip(held, counts))
        return {"bytes": 4 * case["pages"] + 8 * case["seqs"] * width + 8 * rows + 16 * case["seqs"], "flops": 0}
    heads, kv, hd = HEADS[case["shape"]]
    if case["kind"] == "append":
        return {"bytes": rows * 2 * kv * hd * (2 + {"float32": 4, "bfloat16": 2, "float16": 2}[case["source"]]), "flops": 0}
    seen = [_seen(h, c, case["window"], case["sinks"]) for h, c in zip(held, counts)]
    return {"bytes": 4 * hd * kv * sum(t for _, t in seen) + 4 * rows * heads * hd, "flops": 4 * hd * heads * sum(p for p, _ in seen)}


# ---- the same in 64 bits, from the definitions -------------------------------------------------------------------------------
def exact(case, seed):
    if case["kind"] == "tables":
        return None
    s = prepare(case, seed)
    return {"attend": _exact_attend, "append": _exact_append, "verify": _exact_verify}[case["kind"]](case, s)


def _exact_attend(case, s):
    heads, kv, hd = HEADS[case["shape"]]
    group = heads // kv
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    held, counts, table, slots = _held(case), _counts(case), s["table"].tolist(), s["slots"].tolist()
    row = 0
    for h, c, slot in zip(held, counts, slots):
        last = h + c
        mine = s["pool"][torch.tensor(table[slot][: -(-last // case["page"])], device=out.device)]      # [pages][2][kv][page][hd]
        for g in range(kv):
            k, v = (mine[:, i, g].reshape(-1, hd)[:last].double() for i in (0, 1))
            for a in range(0, c, 64):
                b = min(c, a + 64)
                q = s["q"][row + a:row + b, g * group:(g + 1) * group].double().transpose(0, 1)
                at = torch.arange(h + a, h + b, device=out.device)[:, None]
                j = torch.arange(last, device=out.device)[None]
                hidden = j > at
                if case["window"]:
                    hidden = hidden | ((j <= at - case["window"]) & (j >= case["sinks"]))
                logit = torch.matmul(q, k.T) / math.sqrt(hd)
                out[row + a:row + b, g * group:(g + 1) * group] = torch.matmul(torch.softmax(logit.masked_fill(hidden[None], -math.inf), -1), v).transpose(0, 1)
        row += c
    return out


def _exact_append(case, s):
    pool, page = s["pool"].double(), case["page"]
    table, slots, row = s["table"].tolist(), s["slots"].tolist(), 0
    for h, c, slot in zip(_held(case), _counts(case), slots):
        for i in range(h // page, (h + c - 1) // page + 1):
            a, b = max(h, i * page), min(h + c, (i + 1) * page)
            for side, x in ((0, s["k"]), (1, s["v"])):
                pool[table[slot][i], side, :, a - i * page:b - i * page] = x[row + a - h:row + b - h].transpose(0, 1).double()
        row += c
    return pool


def _exact_verify(case, s):
    def listed_(name):
        return s[name].double().cpu().numpy()
    logits, u, accept, temperature, top_p, min_p = (listed_(n) for n in ("logits", "u", "accept", "temperature", "top_p", "min_p"))
    top_k, ids, first = s["top_k"].tolist(), s["ids"].tolist(), s["first"].tolist()
    out = np.zeros(len(ids))
    for a, b in zip(first, first[1:]):
        for r in range(a, b):
            x = logits[r]
            if temperature[r] <= 0:
                if r == b - 1 or ids[r + 1] != int(np.argmax(x)):
                    break
                continue
            order = np.lexsort((np.arange(len(x)), -x))
            order = order[:top_k[r]] if top_k[r] > 0 else order
            w = np.exp(x[order] - x[order[0]])
            if top_p[r] < 1:
                order = order[: 1 + int(np.searchsorted(np.cumsum(w), top_p[r] * w.sum()))]
            order = order[np.exp(x[order] - x[order[0]]) >= min_p[r]]
            share = np.zeros(len(x))
            share[order] = np.exp((x[order] - x.max()) / temperature[r])
            share /= share.sum()
            rest = share
            if r < b - 1:
                if s["probs"] is None:
                    q = np.zeros(len(x))
                    q[ids[r + 1]] = 1.0
                else:
                    q = s["probs"][r].double().cpu().numpy()
                if accept[r] * q[ids[r + 1]] < share[ids[r + 1]]:
                    out[r] = math.log(share[ids[r + 1]])
                    continue
                rest = np.maximum(share - q, 0.0)
            c = np.cumsum(rest)
            out[r] = math.log(share[int(np.searchsorted(c, u[r] * c[-1], side="right"))])
            break
    return [None, None, out]
