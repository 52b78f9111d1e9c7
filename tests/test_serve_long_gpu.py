"""Attention over the 4-bit cache through long pieces of work, where a warp or a block walks over many pages and many pieces are added, and each of its forms against a bound of its own: of what
the form rounds, in scores and in values."""
import random

import pytest
import torch

from booster_b200 import serve
from tests.test_serve_gpu import BF16, F16, F32, ints

pytestmark = pytest.mark.gpu

MANY = 4096                              # rows announced: always the form for many
# What a form's sums of scores lose, in steps of 2^-22 of (a block's scale) x (the sum of its |q|). One tile of columns: two instructions a block, of codes with their offset, 1039 at most. Two
# tiles: the same of codes less 8, and four additions of the blocks' sums in fp32. Many rows: eight instructions (of head_dim 128), 2^-23 of all blocks' sums each, of codes less 8
STEPS = {"one": 1039.0, "two": 10.0, "many": 36.0}


def check(q, k, v, present, held, window, scale, form, out):
    """out [rows, heads, head_dim] of a sequence's rows at positions held, held + 1, ...; k, v [positions, kv, head_dim] in 64 bits, as they are held"""
    rows, heads, hd = q.shape
    kv, group, T = k.shape[1], heads // k.shape[1], k.shape[0]
    qd = q.double().view(rows, kv, group, hd)
    s = scale * torch.einsum("rhgd,thd->rhgt", qd, k)
    pos = torch.arange(T, device="cuda")
    p = held + torch.arange(rows, device="cuda")
    sees = present & (pos <= p[:, None])
    if window:
        sees &= pos > p[:, None] - window
    w = torch.softmax(s.masked_fill(~sees[:, None, None], -torch.inf), -1)
    want = torch.einsum("rhgt,thd->rhgd", w, v)
    mean = torch.einsum("rhgt,thd->rhgd", w, v.abs())
    d = k.abs().view(T, kv, hd // 32, 32).amax(3) / 7
    lost = abs(scale) * STEPS[form] * 2.0 ** -22 * torch.einsum("rhgb,thb->rhgt", qd.abs().view(rows, kv, group, hd // 32, 32).sum(4), d).masked_fill(~sees[:, None, None], 0).amax(3)
    # P to fp16 and its exponential; scores; fp32 sums of 16 tokens a step, of values and of weights; what P leaves out of each weight, 2^-32 of the largest
    room = mean * (2.0 ** -11 + 2.0 ** -20 + 2 * lost[..., None] + T / 16 * 2.0 ** -22) + 2.0 ** -32 * v.abs().sum(0)[:, None]
    room = room + torch.finfo(q.dtype).eps / 2 * (want.abs() + room) + 2.0 ** -25
    off = (out.double().view(want.shape) - want).abs()
    assert (off <= room).all(), (form, (off / room).max().item())


class Long:
    """sequences of `lengths` positions, rows included, in pages that stand scattered; some pages are absent"""

    def __init__(self, lengths, kv, hd, seed, gone=(), page=16):
        r = random.Random(seed)
        self.lengths, self.kv, self.hd, n = lengths, kv, hd, len(lengths)
        need = [-(-t // page) for t in lengths]
        order = list(range(sum(need)))
        r.shuffle(order)
        table = torch.full((n, max(need)), -1, dtype=torch.int32)
        at = 0
        for s, m in enumerate(need):
            table[s, :m] = torch.tensor(order[at:at + m], dtype=torch.int32)
            at += m
        self.pool, self.table = serve.kv4_pool(sum(need), page, kv, hd)[0], table.cuda()
        first = [0]
        for t in lengths:
            first.append(first[-1] + t)
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.gen = gen
        k, v = (torch.randn(first[-1], kv, hd, generator=gen, device="cuda").half() for _ in range(2))
        serve.kv4_append(self.pool, self.table, ints([0] * n), ints(first), k, v)
        self.k, self.v = (x.double() for x in serve.kv4_read(self.pool, self.table, ints([0] * n), ints(first), first[-1], F32))
        self.first, self.present = first, torch.ones(first[-1], dtype=torch.bool, device="cuda")
        for s, i in gone:
            self.table[s, i] = -1
            self.present[first[s] + page * i:first[s] + page * (i + 1)] = False

    def attend(self, rows, heads, max_rows, form, window=0, dtype=F16, scale=0.125):
        n = len(self.lengths)
        q = torch.randn(n * rows, heads, self.hd, generator=self.gen, device="cuda").to(dtype)
        held = [t - rows for t in self.lengths]
        out = serve.kv4_attention(q, self.pool, self.table, ints(held), ints([rows * i for i in range(n + 1)]), scale=scale, window=window, max_rows=max_rows)
        for s in range(n):
            a, b = self.first[s], self.first[s + 1]
            check(q[rows * s:rows * (s + 1)], self.k[a:b], self.v[a:b], self.present[a:b], held[s], window, scale, form, out[rows * s:rows * (s + 1)])


@pytest.mark.parametrize("kv,heads,rows,max_rows,form", [(1, 4, 1, 1, "one"), (1, 16, 1, 1, "two"), (2, 8, 3, 3, "two"), (1, 4, 2, MANY, "many")])
def test_one_long_sequence(kv, heads, rows, max_rows, form):
    """more parts than a round of the join adds"""
    c = Long([20491], kv, 128, kv, gone=[(0, 5), (0, 700), (0, 701)])
    c.attend(rows, heads, max_rows, form)
    c.attend(rows, heads, max_rows, form, window=9000, dtype=BF16)


@pytest.mark.parametrize("heads,rows,max_rows,form", [(4, 1, 1, "one"), (20, 1, 1, "two"), (4, 3, 3, "one"), (4, 3, MANY, "many")])
def test_pieces_of_many_pages(heads, rows, max_rows, form):
    """140 sequences of about 4000 positions: a warp's piece has 40 pages, a block's over 400, which are looked up 32 at a time; some of the sequences lack pages inside"""
    r = random.Random(heads)
    lengths = [r.randrange(3600, 4400) for _ in range(140)]
    c = Long(lengths, 2, 64, heads, gone=[(s, r.randrange(1, 220)) for s in range(0, 140, 3) for _ in range(4)])
    c.attend(rows, heads, max_rows, form)
    c.attend(rows, heads, max_rows, form, window=3001)


@pytest.mark.parametrize("heads,max_rows,form", [(8, 1, "one"), (32, 1, "two"), (8, MANY, "many")])
@pytest.mark.parametrize("size", [1.0, 6.0, 30.0])
@pytest.mark.parametrize("hd", [64, 128])
def test_each_form_within_its_own_roundings(heads, max_rows, form, size, hd):
    """queries and some of the keys' dims with large entries, where sums of scores lose most"""
    gen = torch.Generator(device="cuda").manual_seed(int(size) + hd)
    T, kv = 500, 2
    k, v = (torch.randn(T, kv, hd, generator=gen, device="cuda") for _ in range(2))
    k[:, :, 5] *= 8
    k[:, :, hd - 1] *= 8
    pool, table = serve.kv4_pool(32, 16, kv, hd)[0], ints([list(range(32))])
    serve.kv4_append(pool, table, ints([0]), ints([0, T]), k, v)
    k, v = (x.double() for x in serve.kv4_read(pool, table, ints([0]), ints([0, T]), T, F32))
    n = 40
    q = (size * torch.randn(n, heads, hd, generator=gen, device="cuda")).half()
    out = serve.kv4_attention(q, pool, table.expand(n, 32).contiguous(), ints([T - 1] * n), ints(list(range(n + 1))), scale=0.0625, max_rows=max_rows)
    all_there = torch.ones(T, dtype=torch.bool, device="cuda")
    for i in range(n):
        check(q[i:i + 1], k, v, all_there, T - 1, 0, 0.0625, form, out[i:i + 1])


@pytest.mark.parametrize("kv,heads,rows,max_rows,form,page,hd", [(5, 35, 1, 1, "one", 1024, 64), (5, 35, 2, 2, "two", 512, 128), (5, 35, 7, MANY, "many", 1024, 128), (1, 300, 1, 1, "many", 32, 64),
                                                                 (1, 300, 3, 3, "many", 256, 128), (1024, 1024, 1, 1, "one", 16, 64), (256, 256, 2, MANY, "many", 16, 64), (3, 3, 300, MANY, "many", 128, 64)])
def test_odd_heads_and_pages(kv, heads, rows, max_rows, form, page, hd):
    """groups that do not divide a tile of columns, one head under hundreds, hundreds of heads, the longest pages"""
    c = Long([rows + x for x in (0, 1, 700, 1500)], kv, hd, heads, page=page)
    c.attend(rows, heads, max_rows, form, dtype=BF16)
    c.attend(rows, heads, max_rows, form, window=33)


@pytest.mark.parametrize("heads,max_rows,form", [(4, 1, "one"), (32, 1, "two"), (4, MANY, "many")])
def test_scales_of_any_sign(heads, max_rows, form):
    c = Long([1, 40, 333], 2, 64, heads)
    for scale in (-0.25, 0.0, 2.0 ** -60, -2.0 ** -130, 4.0):
        c.attend(1, heads, max_rows, form, scale=scale)
