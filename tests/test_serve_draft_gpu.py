"""The operators of booster_b200.serve around drafted tokens and the 16-bit cache on the GPU against tests/serve_draft_oracle.py, at the sizes, masks and tables where they can go wrong."""
import math
import random

import numpy as np
import pytest
import torch

from booster_b200 import serve
from tests import serve_draft_oracle as oracle

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


class Case:
    """a 16-bit pool with sequences in scattered pages: counts[i] new rows behind held[i] tokens of slot slots[i]"""

    def __init__(self, held, counts, page=16, kv=2, hd=64, seed=0, spare=2, layers=1, dtype=F16):
        r = random.Random(seed)
        n = len(held)
        self.page, self.kv, self.hd, self.held_l, self.counts, self.dtype = page, kv, hd, list(held), list(counts), dtype
        self.slots_l = r.sample(range(n + 2), n)
        need = [-(-(h + c) // page) for h, c in zip(held, counts)]
        self.pages = sum(need) + spare
        order = r.sample(range(self.pages), self.pages)
        width = max(need + [1]) + 1
        self.table_l = [[-1] * width for _ in range(n + 2)]
        at = [0] * (n + 2)
        for s, h, m in zip(self.slots_l, held, need):
            at[s] = h
            for i in range(m):
                self.table_l[s][i] = order.pop()
        self.first_l = [0]
        for c in counts:
            self.first_l.append(self.first_l[-1] + c)
        self.rows = self.first_l[-1]
        self.pool = serve.kv16_pool(self.pages, page, kv, hd, layers, dtype)
        self.gen = torch.Generator(device="cuda").manual_seed(seed)
        self.held, self.slots, self.first = ints(at), ints(self.slots_l), ints(self.first_l)

    def widened(self, tokens=100000):
        """the same under a table that allows sequences of more tokens: what is chosen by the longest possible one is another form"""
        self.table_l = [row + [-1] * (tokens // self.page) for row in self.table_l]
        return self

    @property
    def table(self):
        return ints(self.table_l)

    def args(self):
        return self.pool[0], self.table, self.held, self.first

    def randn(self, *shape):
        return torch.randn(*shape, generator=self.gen, device="cuda")

    def fill(self):
        """all places of the pool hold numbers, whether a sequence has them or not"""
        self.pool.copy_((self.randn(*self.pool.shape) * torch.exp(0.5 * self.randn(self.hd))).to(self.dtype))

    def seen(self):
        """what the oracle sees of each sequence: K, V [kv, positions, hd] and which positions have a page"""
        out, pool = [], self.pool[0].double().cpu().numpy()
        for s, h, c in zip(self.slots_l, self.held_l, self.counts):
            n = min(h + c, len(self.table_l[s]) * self.page)
            K, V, there = np.zeros((self.kv, n, self.hd)), np.zeros((self.kv, n, self.hd)), np.zeros(n, bool)
            for t in range(n):
                p = self.table_l[s][t // self.page]
                if 0 <= p < self.pages:
                    K[:, t], V[:, t], there[t] = pool[p, 0, :, t % self.page], pool[p, 1, :, t % self.page], True
            out.append((K, V, there))
        return out


def assert_attends(case, q, out, window=0, sinks=0, scale=None):
    scale = case.hd ** -0.5 if scale is None else scale
    eps = torch.finfo(q.dtype).eps
    want, room = oracle.attention(q.double().cpu().numpy(), case.seen(), case.held_l, case.first_l, window, sinks, scale, eps)
    got = out.double().cpu().numpy()
    nan = np.isnan(want)
    assert np.array_equal(nan, np.isnan(got)), f"{(nan != np.isnan(got)).sum()} of {nan.size} are no numbers where the other is one"
    over = np.abs(got - want)[~nan] - (room + eps / 2 * (np.abs(want) + room) + 2.0 ** -25)[~nan]
    assert over.size == 0 or over.max() <= 0, f"off by {over.max():.3g} more than the roundings allow"


# ---- rows into the cache -----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("source", [F32, BF16, F16])
@pytest.mark.parametrize("page,kv,held,counts", [(16, 3, [0, 3, 15, 16, 40], [1, 1, 1, 1, 1]), (32, 1, [7, 0, 31], [20, 0, 70]), (64, 5, [100, 1], [1, 33]), (128, 20, [2, 200], [900, 17])])
def test_append_rounds_once_and_writes_nothing_else(hd, dtype, source, page, kv, held, counts):
    c = Case(held, counts, page=page, kv=kv, hd=hd, seed=hd + page, dtype=dtype)
    c.fill()
    want = c.pool.clone()
    wide = c.randn(c.rows, 3 + 2 * kv, hd).to(source)                  # keys and values behind something else, in one tensor
    k, v = wide[:, 3:3 + kv], wide[:, 3 + kv:]
    serve.kv16_append(*c.args(), k, v, c.slots)
    for i, s in enumerate(c.slots_l):
        for r in range(c.first_l[i], c.first_l[i + 1]):
            pos = c.held_l[i] + r - c.first_l[i]
            p = c.table_l[s][pos // page]
            want[0, p, 0, :, pos % page], want[0, p, 1, :, pos % page] = k[r].to(dtype), v[r].to(dtype)
    assert torch.equal(c.pool.view(torch.int16), want.view(torch.int16))


@pytest.mark.parametrize("source", [F32, F16])
@pytest.mark.parametrize("shift", [1, 2, 3])
def test_append_takes_rows_on_any_alignment(source, shift):
    c = Case([5, 20], [3, 1], kv=1, hd=64, seed=shift)
    flat = c.randn(2, c.rows * 67 + 8).to(source)
    k, v = (flat[i, shift:shift + c.rows * 67].view(c.rows, 1, 67)[:, :, :64] for i in (0, 1))
    serve.kv16_append(*c.args(), k, v, c.slots)
    one = c.pool.clone()
    c.pool.zero_()
    serve.kv16_append(*c.args(), k.contiguous(), v.contiguous(), c.slots)
    assert torch.equal(one, c.pool) and one.any()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("hd", [64, 128])
def test_append_of_what_is_no_number(dtype, hd):
    c = Case([0], [9], kv=5, hd=hd, dtype=dtype)
    k, v = c.randn(9, 5, hd), c.randn(9, 5, hd)
    k[1, 2, 5], k[2, 0, hd - 1], v[3, 4, 0], v[4, 1, 7] = float("nan"), float("inf"), -float("inf"), float("nan")
    k[5, 3, 1] = 65519.0                                               # fp16's largest, 65504, is nearest
    v[6, 2, 9] = 65520.0                                               # half way to 65536: an infinity of fp16, a number of bfloat16
    v[7, 2, 9] = 3.4e38                                                # an infinity of both
    k[8] = 1e-9
    serve.kv16_append(*c.args(), k, v, c.slots)
    wk, wv = k.to(dtype), v.to(dtype)
    bad = ~(torch.isfinite(wk).all(-1, keepdim=True) & torch.isfinite(wv).all(-1, keepdim=True))
    assert bad.sum() == (6 if dtype == F16 else 5)
    page = c.pool[0, c.table_l[c.slots_l[0]][0]]
    assert torch.equal(page[0].transpose(0, 1)[:9].float().nan_to_num(123.0), torch.where(bad, 123.0, wk.float()))
    assert torch.equal(page[1].transpose(0, 1)[:9], torch.where(bad, 0.0, wv))


def test_append_drops_rows_without_a_place():
    c = Case([3, 0, 10], [4, 2, 3], kv=2, spare=0)
    c.fill()
    before = c.pool.clone()
    k, v = c.randn(12, 2, 64).half(), c.randn(12, 2, 64).half()         # three rows behind the last sequence
    table = c.table.clone()
    table[c.slots_l[0]] = -1
    table[c.slots_l[1], 0] = c.pages                                    # no such page
    held = c.held.clone()
    held[c.slots_l[2]] = table.shape[1] * 16 - 1                        # its second row lies beyond the table, its first where no page is
    serve.kv16_append(c.pool[0], table, held, c.first, k, v, c.slots)
    assert torch.equal(before, c.pool)
    serve.kv16_append(c.pool[0], c.table, c.held, c.first, k, v, ints([99, -1, 1 << 30]))
    assert torch.equal(before, c.pool)


# ---- attention ---------------------------------------------------------------------------------------------------------------
HELD = {"short": ([0, 1, 15, 16, 31, 32, 33, 100], [1] * 8), "drafts": ([0, 3, 40, 200, 31], [5, 2, 8, 1, 5]), "ragged": ([0, 700, 64, 5], [37, 3, 200, 0]), "one": ([333], [1]),
        "long": ([2600, 7], [1, 1]), "portion": ([130], [300])}


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("hd,heads,kv", [(64, 2, 2), (64, 6, 2), (64, 8, 1), (128, 8, 2), (128, 16, 1), (128, 5, 1), (128, 40, 1)])
@pytest.mark.parametrize("which,page", [("short", 16), ("short", 64), ("drafts", 16), ("drafts", 32), ("ragged", 16), ("ragged", 128), ("one", 16), ("one", 256), ("long", 64), ("portion", 32)])
def test_attention(dtype, hd, heads, kv, which, page):
    c = Case(*HELD[which], page=page, kv=kv, hd=hd, seed=hd + page, dtype=dtype)
    c.fill()
    q = (1.5 * c.randn(c.rows, heads, hd)).to(dtype)
    assert_attends(c, q, serve.kv16_attention(q, *c.args(), slots=c.slots))
    if max(c.counts) <= 8:
        assert_attends(c.widened(), q, serve.kv16_attention(q, *c.args(), slots=c.slots))


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 3), (16, 16), (17, 40), (64, 0), (100, 4), (100, 33), (128, 128), (300, 1000), (5000, 9), (2 ** 31 - 1, 2 ** 31 - 1)])
@pytest.mark.parametrize("dtype,hd,heads,kv,which,page", [(BF16, 128, 8, 2, "drafts", 16), (F16, 64, 4, 2, "ragged", 32), (BF16, 64, 16, 1, "long", 64), (F16, 128, 4, 1, "portion", 16),
                                                          (BF16, 128, 8, 1, "ragged", 256)])
def test_attention_under_a_window(window, sinks, dtype, hd, heads, kv, which, page):
    c = Case(*HELD[which], page=page, kv=kv, hd=hd, seed=window % 1000 + sinks % 100, dtype=dtype)
    c.fill()
    q = (1.5 * c.randn(c.rows, heads, hd)).to(dtype)
    assert_attends(c, q, serve.kv16_attention(q, *c.args(), slots=c.slots, window=window, sinks=sinks), window, sinks)
    assert_attends(c.widened(), q, serve.kv16_attention(q, *c.args(), slots=c.slots, window=window, sinks=sinks), window, sinks)


def test_sinks_count_under_a_window_alone():
    c = Case([300, 20], [2, 9], kv=1, hd=64)
    c.fill()
    q = c.randn(11, 4, 64).half()
    assert torch.equal(serve.kv16_attention(q, *c.args(), slots=c.slots, sinks=50), serve.kv16_attention(q, *c.args(), slots=c.slots))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rows", [1, 6, 150])
@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 5)])
@pytest.mark.parametrize("wide", [False, True])
def test_attention_over_absent_pages_and_slots(dtype, rows, window, sinks, wide):
    held = [0, 50, 100, 200, 64, 30, 500]
    c = Case(held, [rows] * 7, kv=2, hd=128, seed=rows, dtype=dtype)
    c.fill()
    q = c.randn(c.rows, 6, 128).to(dtype)
    c.table_l[c.slots_l[1]][0] = -1                                     # the first page is away
    c.table_l[c.slots_l[2]] = [-1] * len(c.table_l[0])                  # all are: nothing is seen
    c.table_l[c.slots_l[3]][2], c.table_l[c.slots_l[3]][5] = c.pages, 2 ** 31 - 1
    for i in range(2, (30 + rows) // 16 + 1):                           # nothing from position 32 on, under the window some rows see their first tokens alone
        c.table_l[c.slots_l[5]][i] = -2 ** 31
    slots = list(c.slots_l)
    slots[4] = 1000                                                     # no such slot
    c.table_l[c.slots_l[4]] = [-1] * len(c.table_l[0])                  # (as the oracle sees it)
    if wide:
        c.widened()
    out = serve.kv16_attention(q, *c.args(), slots=ints(slots), window=window, sinks=sinks)
    assert_attends(c, q, out, window, sinks)
    assert not out[2 * rows:3 * rows].any() and not out[4 * rows:5 * rows].any()


@pytest.mark.parametrize("rows", [1, 40])
def test_rows_beyond_the_table(rows):
    """a slot that holds as much as its table can: its new rows have no place, but see what there is"""
    c = Case([47 + 16], [rows], kv=1, hd=64, page=16)
    c.table_l = [r[:4] for r in c.table_l]
    c.fill()
    q = c.randn(rows, 2, 64).half()
    assert_attends(c, q, serve.kv16_attention(q, *c.args(), slots=c.slots))
    assert_attends(c, q, serve.kv16_attention(q, *c.args(), slots=c.slots, window=5, sinks=2), 5, 2)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rows", [1, 5, 90])
@pytest.mark.parametrize("wide", [False, True])
def test_tokens_and_queries_that_are_no_numbers(dtype, rows, wide):
    c = Case([40, 200, 10], [rows] * 3, kv=2, hd=64, seed=3, dtype=dtype)
    if wide:
        c.widened()
    k, v = (c.randn(250 + 3 * rows, 2, 64) for _ in range(2))
    k[5, 0, 3] = float("nan")                                           # of the first sequence, KV head 0
    v[40 + rows + 100, 1, 3] = float("inf")                             # of the second, KV head 1, position 100
    k[40 + rows + 200 + rows - 1, 0, 0] = -float("inf")                 # its last row's own, which no other row sees
    total = [0, 40 + rows, 240 + 2 * rows, 250 + 3 * rows]
    serve.kv16_append(c.pool[0], c.table, torch.zeros_like(c.held), ints(total), k, v, c.slots)
    q = c.randn(c.rows, 4, 64).to(dtype)
    q[2 * rows, 1, 7], q[2 * rows, 2, 9], q[3 * rows - 1, 3, 0] = float("inf"), float("nan"), -float("inf")
    out = serve.kv16_attention(q, *c.args(), slots=c.slots)
    assert_attends(c, q, out)
    assert out[0, :2].isnan().all() and not out[0, 2:].isnan().any() and out[2 * rows - 1, :2].isnan().all()
    if rows > 1:
        assert not out[2 * rows - 2, :2].isnan().any()
    out = serve.kv16_attention(q, *c.args(), slots=c.slots, window=30, sinks=5)
    assert_attends(c, q, out, 30, 5)
    assert not out[2 * rows - 1, 2:].isnan().any()                      # position 100 is out of sight
    out = serve.kv16_attention(q, *c.args(), slots=c.slots, window=30, sinks=6)
    assert out[rows - 1, :2].isnan().all()                              # position 5 is among the first six


@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("scale", [-0.2, 0.0, 3.0])
def test_scales_of_any_sign(rows, scale):
    c = Case([100, 300], [rows, rows], kv=2, hd=64, dtype=BF16)
    c.fill()
    q = c.randn(c.rows, 8, 64).bfloat16()
    assert_attends(c, q, serve.kv16_attention(q, *c.args(), slots=c.slots, scale=scale), scale=scale)
    assert_attends(c.widened(), q, serve.kv16_attention(q, *c.args(), slots=c.slots, scale=scale), scale=scale)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rows", [1, 3, 100])
def test_small_weights_behind_one_that_takes_most(dtype, rows):
    """values of 1 everywhere and one token with nearly all of the weight: the others keep theirs, and the weights sum to 1"""
    c = Case([4000], [rows], kv=1, hd=64, page=64, dtype=dtype)
    c.pool[0, :, 0], c.pool[0, :, 1] = 0.0, 1.0
    c.pool[0, c.table_l[c.slots_l[0]][10], 0, 0, 3, 0] = 40.0
    q = torch.zeros(rows, 2, 64, dtype=dtype, device="cuda")
    q[:, :, 0] = 1.0
    out = serve.kv16_attention(q, *c.args(), slots=c.slots, scale=0.4)
    assert torch.equal(out, torch.ones_like(out))
    c.pool[0, c.table_l[c.slots_l[0]][10], 1, 0, 3] = 0.0               # now the others alone: 4000 of e^-16 each
    out = serve.kv16_attention(q, *c.args(), slots=c.slots, scale=0.4)
    assert_attends(c, q, out, scale=0.4)
    want = 4000 * math.exp(-16.0)
    assert abs(float(out.float().mean()) / want - 1) < 0.02


@pytest.mark.parametrize("rows,heads", [(1, 4), (7, 8), (200, 2)])
def test_one_position_gives_its_value(rows, heads):
    c = Case([300] * 3, [rows] * 3, kv=1, hd=128, dtype=BF16)
    c.fill()
    q = c.randn(c.rows, heads, 128).bfloat16()
    out = serve.kv16_attention(q, *c.args(), slots=c.slots, window=1)
    for i, s in enumerate(c.slots_l):
        for r in range(rows):
            p = 300 + r
            v = c.pool[0, c.table_l[s][p // 16], 1, 0, p % 16]
            assert torch.equal(out[i * rows + r], v.expand(heads, 128))


def test_rows_of_no_sequence_and_layouts():
    """a padded step, queries with strides and off their alignment, a given out, layers of a pool, slots left out, a wide table"""
    for dtype, rows, shift in ((BF16, [1, 1, 0, 1], 0), (F16, [3, 60, 1, 0], 1), (BF16, [2, 2, 2, 2], 2)):
        c = Case([40, 3, 90, 16], rows, kv=2, hd=64, layers=3, seed=shift, dtype=dtype)
        c.fill()
        flat = c.randn((c.rows + 5) * 7 * 80 + 8).to(dtype)
        q = flat[shift:shift + (c.rows + 5) * 560].view(c.rows + 5, 7, 80)[:, 1:7, :64]
        out = torch.full((c.rows + 5, 6, 64), 7.0, dtype=dtype, device="cuda")
        wide = torch.full((c.table.shape[0], 50), 3, dtype=torch.int32, device="cuda")
        wide[:, :c.table.shape[1]] = c.table
        table = wide[:, :c.table.shape[1]]
        for layer in (2, 0):
            got = serve.kv16_attention(q, c.pool[layer], table, c.held, c.first, c.slots, out=out)
            assert got is out or got.data_ptr() == out.data_ptr()
            assert (out[c.rows:] == 7).all()
            one = c.pool[layer:layer + 1]
            keep, c.pool = c.pool, one
            assert_attends(c, q[:c.rows], out[:c.rows])
            c.pool = keep
        order = torch.argsort(c.slots)
        if all(x == rows[0] for x in rows):
            by_slot = torch.zeros(len(c.table_l), dtype=torch.int32, device="cuda")
            by_slot[c.slots.long()] = rows[0]
            first = torch.cat([by_slot.new_zeros(1), by_slot.cumsum(0, dtype=torch.int32)])
            qq = q[:c.rows].reshape(4, rows[0], 6, 64)[order].reshape(c.rows, 6, 64)
            a = serve.kv16_attention(qq, c.pool[0], table, c.held, first)
            assert torch.equal(a.reshape(4, rows[0], 6, 64), out[:c.rows].reshape(4, rows[0], 6, 64)[order])


@pytest.mark.parametrize("counts,max_rows", [([1, 1, 50, 1], None), ([1, 1, 50, 1], 1), ([1, 1, 50, 1], 500), ([2, 300, 1], 1), ([1, 1, 1], 400)])
def test_any_number_of_rows_is_right(counts, max_rows):
    c = Case([70 * i for i in range(len(counts))], counts, kv=2, hd=128, dtype=BF16)
    c.fill()
    q = c.randn(c.rows, 8, 128).bfloat16()
    assert_attends(c, q, serve.kv16_attention(q, *c.args(), slots=c.slots, max_rows=max_rows))
    assert_attends(c, q, serve.kv16_attention(q, *c.args(), slots=c.slots, max_rows=max_rows, window=33, sinks=5), 33, 5)
    assert_attends(c.widened(), q, serve.kv16_attention(q, *c.args(), slots=c.slots, max_rows=max_rows))


@pytest.mark.parametrize("hd", [64, 128])
def test_many_sequences(hd):
    n = 4096
    r = random.Random(5)
    c = Case([r.randrange(0, 40) for _ in range(n)], [1] * n, kv=1, hd=hd, dtype=BF16)
    c.fill()
    q = c.randn(n, 2, hd).bfloat16()
    assert_attends(c, q, serve.kv16_attention(q, *c.args(), slots=c.slots))
    assert_attends(c, q, serve.kv16_attention(q, *c.args(), slots=c.slots, max_rows=200, window=9, sinks=2), 9, 2)


def test_pools_whose_offsets_pass_32_bits():
    """a pool of over 4 GB whose last pages a sequence holds"""
    page, kv, hd = 1024, 8, 128
    pages = 1100                                                        # 4.2 MB each
    c = Case([1500], [1], page=page, kv=kv, hd=hd, dtype=BF16)
    c.pages = pages
    c.pool = torch.zeros(1, pages, 2, kv, page, hd, dtype=BF16, device="cuda")
    c.table_l[c.slots_l[0]][:2] = [pages - 1, pages - 2]
    c.pool[0, -2:] = c.randn(2, 2, kv, page, hd).bfloat16()
    k, v = c.randn(1, kv, hd).bfloat16(), c.randn(1, kv, hd).bfloat16()
    serve.kv16_append(*c.args(), k, v, c.slots)
    assert torch.equal(c.pool[0, -2, 0, :, 1500 - 1024], k[0]) and torch.equal(c.pool[0, -2, 1, :, 1500 - 1024], v[0])
    q = c.randn(1, 16, hd).bfloat16()
    want = [serve.kv16_attention(q, *c.args(), slots=c.slots), serve.kv16_attention(q, *c.args(), slots=c.slots, max_rows=100)]
    small = Case([1500], [1], page=page, kv=kv, hd=hd, dtype=BF16)
    small.pages = 2
    small.pool = c.pool[:, -2:].clone()
    small.table_l[small.slots_l[0]][:2] = [1, 0]
    for w, m in zip(want, (None, 100)):
        out = serve.kv16_attention(q, *small.args(), slots=small.slots, max_rows=m)
        assert torch.equal(out, w)
        assert_attends(small, q, out)


# ---- pages -------------------------------------------------------------------------------------------------------------------
def lists(table, held, refs):
    return table.tolist(), held.tolist(), refs.tolist()


def random_tables(seed, n_slots, width, page, n_pages, share=True):
    r = random.Random(seed)
    order = r.sample(range(n_pages), n_pages)
    table, held, refs = [[-1] * width for _ in range(n_slots)], [0] * n_slots, [0] * n_pages
    for s in range(n_slots):
        held[s] = r.randrange(0, width * page + 1)
        for i in range(-(-held[s] // page)):
            if share and s and i < held[s - 1] // page and r.random() < 0.3 and table[s - 1][i] >= 0:
                table[s][i] = table[s - 1][i]
            elif order:
                table[s][i] = order.pop()
        held[s] = min(held[s], page * next((i for i in range(width) if table[s][i] < 0), width))
        for p in table[s]:
            if p >= 0:
                refs[p] += 1
    return ints(table), ints(held), ints(refs)


def assert_plans(table, held, refs, slots, counts, rows, page):
    t, h, f = lists(table, held, refs)
    want = oracle.plan(t, h, f, slots if slots is not None else list(range(len(counts))), counts, rows, page)
    got = serve.pages_plan(table, held, refs, ints(counts), page, rows, None if slots is None else ints(slots))
    for name, a, b in zip(("first", "positions", "places", "status"), got, (*want[:3], [want[3]])):
        assert a.tolist() == b, name
    assert table.tolist() == t and refs.tolist() == f and held.tolist() == h
    return want[3]


@pytest.mark.parametrize("seed", range(12))
@pytest.mark.parametrize("page", [16, 128])
def test_plan_of_a_step(seed, page):
    r = random.Random(seed + 100)
    n_slots, width = r.choice([1, 3, 40]), r.choice([2, 9, 70])
    n_pages = r.choice([n_slots * width, n_slots * width * 2 // 3 + 1, 33, 1025])
    table, held, refs = random_tables(seed, n_slots, width, page, n_pages)
    n = r.randrange(0, n_slots + 1)
    slots = r.sample(range(n_slots), n)
    counts = [r.choice([0, 1, 5, page, 3 * page + 1]) for _ in range(n)]
    assert_plans(table, held, refs, slots, counts, sum(counts) + r.choice([0, 9]), page)


def test_plan_of_many_rows_and_sequences():
    table, held, refs = random_tables(1, 4096, 3, 16, 20000)
    held.clamp_(max=30)
    assert assert_plans(table, held, refs, None, [1 + i % 3 for i in range(4096)], 9000, 16) == 0
    table, held, refs = random_tables(2, 3, 200, 64, 1000)
    held.copy_(ints([100, 64, 0]))
    assert assert_plans(table, held, refs, [2, 0, 1], [4097, 5000, 1], 9100, 64) in (0, -1)
    table, held, refs = ints([[-1] * 400, [-1] * 400]), ints([0, 0]), ints([0] * 700)
    assert assert_plans(table, held, refs, [1, 0], [5000, 6000], 11000, 32) == 0
    assert assert_plans(table, ints([6000, 5000]), refs, [0, 1], [9000, 6000], 15000, 32) == -1     # the table ends
    assert assert_plans(table, ints([6000, 5000]), refs, [0, 1], [5000, 6000], 11000, 32) == 0
    assert assert_plans(ints([[-1] * 400]), ints([0]), ints([0] * 300), None, [10000], 10000, 32) == 13          # 13 pages are missing


@pytest.mark.parametrize("shift", [0, 1])
def test_plan_in_a_large_pool(shift):
    """free pages far behind the first 32 768, a few here and there, more than one chunk of them at once; counts off their alignment"""
    n_pages = 150001
    r = random.Random(shift)
    flat = torch.ones(n_pages + shift, dtype=torch.int32, device="cuda")
    refs = flat[shift:]
    refs[r.sample(range(70000), 500)] = 0
    refs[100000:] = 0
    table, held = ints([[-1] * 3000 for _ in range(4)]), ints([0] * 4)
    free = torch.nonzero(refs == 0)[:, 0].tolist()
    for counts, rows in (([16 * 100, 5, 0, 16 * 300], 6500), ([0, 16 * 2500, 16 * 900, 1], 60000)):
        t, h, f = lists(table, held, refs)
        want = oracle.plan(t, h, f, [2, 0, 1, 3], counts, rows, 16)
        assert want[3] == 0
        got = serve.pages_plan(table, held, refs, ints(counts), 16, rows, ints([2, 0, 1, 3]))
        for a, b in zip(got, (*want[:3], [0])):
            assert a.tolist() == b
        assert table.tolist() == t and refs.tolist() == f
        held[ints([2, 0, 1, 3]).long()] += ints(counts)
    assert sorted(p for row in table.tolist() for p in row if p >= 0) == free[:int((table >= 0).sum())]
    t, h, f = lists(table, held, refs)
    missing = int((refs == 0).sum()) // 2995 + 1
    big = ints([[-1] * 3000 for _ in range(missing)])
    got = serve.pages_plan(big, ints([0] * missing), refs, ints([16 * 3000] * missing), 16, 10)
    assert got[3].item() == -1                                          # more than 10 rows
    got = serve.pages_plan(big, ints([0] * missing), refs, ints([16 * 3000] * missing), 16, 16 * 3000 * missing)
    assert got[3].item() == 3000 * missing - f.count(0) and refs.tolist() == f and (big == -1).all()


def test_plans_that_cannot_be():
    base = lambda: (ints([[0, 1, -1, -1], [2, -1, -1, -1], [-1] * 4]), ints([20, 16, 0]), ints([1, 1, 1] + [0] * 9))  # noqa: E731
    for slots, counts, rows in (([0, 0], [1, 1], 4), ([0, 3], [1, 1], 4), ([0, -1], [1, 1], 4), ([0, 1], [1, -1], 4), ([0, 1], [3, 2], 4), ([0], [100], 200), ([0, 1], [2 ** 31 - 1, 2 ** 31 - 1], 7)):
        assert assert_plans(*base(), slots, counts, rows, 16) == -1
    t, h, f = base()
    h[1] = -5
    assert assert_plans(t, h, f, [1, 0], [1, 2], 3, 16) == -1
    t, h, f = base()
    t[1, 2] = 7                                                         # a page behind one that is missing
    assert assert_plans(t, h, f, [1], [20], 20, 16) == -1
    assert assert_plans(*base(), [], [], 0, 16) == 0
    assert assert_plans(*base(), [], [], 5, 16) == 0
    assert assert_plans(*base(), None, [0, 0, 0], 0, 16) == 0


@pytest.mark.parametrize("seed", range(10))
@pytest.mark.parametrize("window,sinks", [(0, 0), (0, 100), (1, 0), (16, 16), (33, 17), (100, 5), (1000, 40), (2 ** 31 - 1, 3), (5, 2 ** 31 - 1)])
def test_trim(seed, window, sinks):
    page = [16, 32][seed % 2]
    table, held, refs = random_tables(seed, 9, 80, page, 800)
    r = random.Random(seed)
    for s in range(9):                                                  # rows were refused
        held[s] = max(0, int(held[s]) - r.choice([0, 1, 5, page, 3 * page]))
    t, h, f = lists(table, held, refs)
    slots = r.sample(range(9), 6) + [99, -3]
    slots.append(slots[0])
    oracle.trim(t, h, f, slots, page, window, sinks)
    serve.pages_trim(table, held, refs, page, ints(slots), window, sinks)
    assert table.tolist() == t and refs.tolist() == f and held.tolist() == h


def test_slots_without_their_first_pages_fork():
    table, held, refs = ints([[9, -1, -1, 3, 4, -1], [-1] * 6, [-1, 5, -1, -1, -1, -1], [-1] * 6, [7, -1, -1, -1, -1, -1]]), ints([70, 0, 32, 0, 20]), ints([0, 0, 0, 1, 1, 1, 0, 1, 0, 1])
    pool = serve.kv16_pool(10, 16, 1, 64)
    pool.copy_(torch.randn(pool.shape, device="cuda"))
    want = pool.clone()
    assert serve.pages_fork(pool, table, held, refs, ints([0, 2]), ints([1, 3])).item() == 0
    want[:, 0] = want[:, 4]                                             # the part-full page's one tile of 16 tokens is a whole page here
    assert torch.equal(pool, want) and held.tolist() == [70, 70, 32, 32, 20]
    assert table.tolist() == [[9, -1, -1, 3, 4, -1], [9, -1, -1, 3, 0, -1], [-1, 5, -1, -1, -1, -1], [-1, 5, -1, -1, -1, -1], [7, -1, -1, -1, -1, -1]]
    assert refs.tolist() == [1, 0, 0, 2, 1, 2, 0, 1, 0, 2]
    before = [x.clone() for x in (table, held, refs)]
    serve.pages_free(table, held, refs, ints([1]))
    assert serve.pages_fork(pool, table, held, refs, ints([4]), ints([1])).item() == -1          # its last page, which is part full, is away
    assert table[1].tolist() == [-1] * 6 and torch.equal(table[[0, 2, 3, 4]], before[0][[0, 2, 3, 4]]) and torch.equal(pool, want)


def test_trim_of_odd_entries():
    table, held, refs = ints([[5, 99, -7, 2], [2, 3, -1, -1]]), ints([-4, 2 ** 31 - 1]), ints([0, 0, 2, 1, 0, 1])
    serve.pages_trim(table, held, refs, 16, ints([0, 1]))
    assert table.tolist() == [[-1, -1, -7, -1], [2, 3, -1, -1]] and refs.tolist() == [0, 0, 1, 1, 0, 0]


@pytest.mark.parametrize("hd,page,dtype", [(64, 16, F16), (128, 64, BF16)])
def test_pages_of_a_16_bit_pool_fork_copy_and_compact(hd, page, dtype):
    c = Case([3 * page + 5, page, 2 * page + 1], [0, 0, 0], page=page, kv=3, hd=hd, layers=2, spare=6, dtype=dtype)
    c.fill()
    table, held = c.table, c.held.clone()
    refs = torch.zeros(c.pages, dtype=torch.int32, device="cuda")
    for row in c.table_l:
        for p in row:
            if p >= 0:
                refs[p] += 1
    content = lambda s: [c.pool[:, int(table[s, t // page]), :, :, t % page].clone() for t in range(int(held[s]))]  # noqa: E731
    was = {s: content(s) for s in c.slots_l}
    free = [s for s in range(len(c.table_l)) if s not in c.slots_l]
    assert serve.pages_fork(c.pool, table, held, refs, ints(c.slots_l[:2]), ints(free)).item() == 0
    for a, b in zip(c.slots_l, free):
        assert int(held[b]) == int(held[a]) and all(torch.equal(x, y) for x, y in zip(was[a], content(b)))
    assert int(table[free[0], 3]) != int(table[c.slots_l[0], 3])       # the part-full page is its own
    serve.pages_free(table, held, refs, ints([c.slots_l[0]]))
    live = serve.pages_compact(c.pool, table, refs).item()
    assert live == int((refs > 0).sum()) and not refs[live:].any() and int(table.max()) < live
    assert all(torch.equal(x, y) for x, y in zip(was[c.slots_l[0]], content(free[0])))
    assert all(torch.equal(x, y) for s in c.slots_l[1:] for x, y in zip(was[s], content(s)))
    before = c.pool.clone()
    assert serve.pages_copy(c.pool, table, refs, ints([0]), ints([live])).item() == 0
    before[:, live] = before[:, 0]
    assert torch.equal(c.pool, before)


# ---- verification ------------------------------------------------------------------------------------------------------------
KINDS = [dict(), dict(temperature=0.0), dict(temperature=0.7, top_k=40, top_p=0.95, min_p=0.05), dict(top_p=0.9), dict(temperature=1.3, min_p=0.1), dict(top_k=700, temperature=2.0),
         dict(top_k=5, top_p=0.5, temperature=-1.0), dict(top_p=0.0), dict(top_k=3000, top_p=0.999, temperature=1.5), dict(top_k=1)]


def verified(logits, ids, first, u, accept, filters, probs):
    col = lambda name, t, none: torch.tensor([f.get(name, none) for f in filters], dtype=t, device="cuda")  # noqa: E731
    return serve.verify(logits, ints(ids), ints(first), u, accept, col("temperature", F32, 1.0), col("top_k", torch.int32, 0), col("top_p", F32, 1.0), col("min_p", F32, 0.0), probs)


def as_f32(filters):
    """filters as the device has them"""
    return [{k: float(np.float32(v)) if k != "top_k" else v for k, v in f.items()} for f in filters]


def assert_verifies(logits, ids, first, u, accept, filters, probs):
    got = [x.tolist() for x in verified(logits, ids, first, u, accept, filters, probs)]
    want = oracle.verify(logits.double().cpu().numpy(), ids, first, u.double().tolist(), accept.double().tolist(), as_f32(filters), None if probs is None else probs.double().cpu().numpy())
    for i, (a, b) in enumerate(zip(first, first[1:])):
        if want[3][i] < 1e-9:                                           # decided by less than the weights' step of 2^-40 and sums of doubles are sure of
            continue
        assert got[0][i] == want[0][i], i
        assert got[1][a:b] == want[1][a:b], i
        for x, y in zip(got[2][a:b], want[2][a:b]):
            assert x == y or abs(x - y) <= 1e-6 * abs(y) + 2e-6, (i, x, y)      # a share is off by half a step of 2^-40 at 2^-20 or more, its logarithm rounded to fp32
    return got


def step(seed, vocab, counts, dtype, kinds, drafter, sharp=2.2):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = random.Random(seed)
    rows = sum(counts)
    first = [0]
    for n in counts:
        first.append(first[-1] + n)
    logits = sharp * torch.randn(rows, vocab, generator=gen, device="cuda")
    near = logits + 0.7 * torch.randn(rows, vocab, generator=gen, device="cuda")
    probs = torch.softmax(near, 1)
    ids = [r.randrange(vocab)] + (torch.multinomial(probs, 1, generator=gen)[:-1, 0] if drafter or vocab < 50 else torch.where(torch.rand(rows, generator=gen, device="cuda") < 0.7, logits.argmax(1), near.argmax(1))[:-1]).tolist()
    u, accept = torch.rand(rows, generator=gen, device="cuda"), torch.rand(rows, generator=gen, device="cuda")
    filters = []
    for n in counts:
        filters += [r.choice(kinds)] * n
    return logits.to(dtype), ids, first, u, accept, filters, probs if drafter else None


@pytest.mark.parametrize("drafter", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("vocab,counts", [(1, [1, 2, 3]), (2, [2, 2, 5, 1, 0, 3]), (37, [4, 1, 6, 2, 2, 8, 3]), (1000, [5, 1, 2, 0, 7, 3]), (4099, [3, 5, 1, 4]), (32000, [2, 5, 1, 4, 4]), (128256, [5, 1, 4, 3])])
def test_verify(drafter, dtype, vocab, counts):
    for seed in range(4):
        assert_verifies(*step(seed * 100 + vocab % 97, vocab, counts, dtype, KINDS, drafter))


@pytest.mark.parametrize("drafter", [False, True])
@pytest.mark.parametrize("kind", range(len(KINDS)))
def test_verify_by_each_filter(drafter, kind):
    for seed, sharp in ((1, 2.2), (2, 0.3), (3, 6.0)):
        assert_verifies(*step(seed, 9001, [4, 3, 1, 6, 2, 5], F32, [KINDS[kind]], drafter, sharp))


def test_verify_of_many_equal_logits():
    """edges of filters among thousands of equal logits, whole numbers of a few values"""
    for vocab, kinds in ((9001, [dict(top_k=3000), dict(top_p=0.4), dict(top_k=5000, top_p=0.7, temperature=0.5), dict()]), (70000, [dict(top_k=2500), dict(top_p=0.6)])):
        for drafter in (False, True):
            logits, ids, first, u, accept, filters, probs = step(vocab, vocab, [3, 3, 2, 4], F32, kinds, drafter, 0.6)
            got = verified(logits.round(), ids, first, u, accept, filters, probs)
            want = oracle.verify(logits.round().double().cpu().numpy(), ids, first, u.double().tolist(), accept.double().tolist(), as_f32(filters), None if probs is None else probs.double().cpu().numpy())
            sure = [i for i in range(4) if want[3][i] > 1e-9]
            assert sure
            for i in sure:
                assert got[0].tolist()[i] == want[0][i] and got[1].tolist()[first[i]:first[i + 1]] == want[1][first[i]:first[i + 1]]


@pytest.mark.parametrize("vocab", [7, 9001, 128256])
def test_one_row_is_a_draw(vocab):
    logits, ids, first, u, accept, filters, _ = step(7, vocab, [1] * 40, BF16, KINDS, False)
    gained, tokens, logprobs = verified(logits, ids, first, u, accept, filters, None)
    col = lambda name, t, none: torch.tensor([f.get(name, none) for f in filters], dtype=t, device="cuda")  # noqa: E731
    a, b = serve.sample(logits, u, col("temperature", F32, 1.0), col("top_k", torch.int32, 0), col("top_p", F32, 1.0), col("min_p", F32, 0.0))
    assert torch.equal(tokens, a) and torch.equal(logprobs, b) and (gained == 1).all()


def test_drafts_and_distributions_that_are_odd():
    vocab, inf, nan = 1000, float("inf"), float("nan")
    for top_k in (0, 30, 600):
        kinds = [dict(top_k=top_k)]
        logits, ids, first, u, accept, filters, probs = step(3, vocab, [2] * 14, F32, kinds, True)
        ids[1], ids[3], ids[5] = -1, vocab, 2 ** 31 - 1                  # no token: never taken, and nothing comes off p
        for draft_probs in (probs, None):
            assert_verifies(logits, ids, first, u, accept, filters, draft_probs)
        p = torch.softmax(logits, 1)
        probs[6] = p[6]                                                  # the target's own: taken but for the last digits
        accept[6] = 0.999
        probs[8] = 0.0                                                   # nothing: whatever has weight is taken, and nothing comes off p
        probs[10] = -1.0
        probs[12] = nan
        probs[14] = inf                                                  # everything comes off: p
        probs[16, ids[17]], probs[18, ids[19]] = nan, inf
        accept[20] = 0.0
        logits[22] = nan                                                 # no logit at all
        logits[24, ::2], logits[26, 5] = -inf, inf
        ids[27] = 5
        got = assert_verifies(logits, ids, first, u, accept, filters, probs)
        assert got[1][22] == -1 and got[2][22] == -inf and got[0][11] == 1 and got[1][26] == 5


def test_rows_of_no_sequence_have_no_token():
    logits, ids, _, u, accept, filters, probs = step(4, 500, [9], F32, [dict()], True)
    first = [2, 4, 4, 7]
    gained, tokens, logprobs = verified(logits, ids, first, u, accept, filters, probs)
    assert tokens[:2].tolist() == [-1, -1] and tokens[7:].tolist() == [-1, -1] and not logprobs[:2].any() and not logprobs[7:].any() and gained[1] == 0
    want = oracle.verify(logits.double().cpu().numpy(), ids, first, u.double().tolist(), accept.double().tolist(), filters, probs.double().cpu().numpy())
    assert gained.tolist() == want[0] and tokens[2:7].tolist() == want[1][2:7]
    for n_seq in (0, 1):
        out = serve.verify(logits[:0], ints([]), ints([0] * (n_seq + 1)), u[:0], accept[:0])
        assert out[0].tolist() == [0] * n_seq and out[1].numel() == 0
    gained, tokens, _ = serve.verify(logits, ints(ids), ints([0]), u, accept)
    assert gained.numel() == 0 and (tokens == -1).all()
    gained, tokens, _ = serve.verify(logits, ints(ids), ints([-5, 3, 2 ** 31 - 1]), u, accept)       # bounded by the rows
    assert gained.min() >= 1 and gained.sum() <= 9


def test_long_sequences_of_drafts():
    """more drafts than a warp looks at in one go, all of them taken or not"""
    vocab, n = 50, 100
    logits = torch.zeros(2 * n, vocab, device="cuda")
    ids = [(7 * i) % vocab for i in range(2 * n)]
    for r in range(2 * n - 1):
        logits[r, ids[r + 1]] = 200.0
    u = torch.full((2 * n,), 0.5, device="cuda")
    gained, tokens, _ = serve.verify(logits, ints(ids), ints([0, n, 2 * n]), u, u)
    assert gained.tolist() == [n, n] and tokens[:n - 1].tolist() == ids[1:n] and tokens[n:-1].tolist() == ids[n + 1:]
    for stop in (0, 31, 32, 33, 64, 98):
        x = logits.clone()
        x[stop, ids[stop + 1]] = -200.0
        gained, tokens, logprobs = serve.verify(x, ints(ids), ints([0, n, 2 * n]), u, u)
        assert gained.tolist() == [stop + 1, n] and tokens[:stop].tolist() == ids[1:stop + 1] and tokens[stop] >= 0 and (tokens[stop + 1:n] == -1).all() and not logprobs[stop + 1:n].any()


@pytest.mark.parametrize("drafter", [False, True])
@pytest.mark.parametrize("vocab,n", [(300, 400), (9000, 130), (70000, 30)])
def test_more_rows_than_the_card_holds_at_once(vocab, n, drafter):
    """the later rows of sequences come last, and those behind the end of theirs are left; sequences without rows, of one and of many"""
    r = random.Random(vocab)
    counts = [r.choice([0, 1, 1, 2, 3, 5, 8]) for _ in range(n)] + [70, 0]
    kinds = KINDS if vocab < 70000 else KINDS[:3] + KINDS[4:7]
    logits, ids, first, u, accept, filters, probs = step(vocab, vocab, counts, F32, kinds, drafter)
    first_row = first[-1] - 70
    for i in range(60):                                                 # the long one takes 60 drafts
        logits[first_row + i, ids[first_row + i + 1]] += 60.0
    got = assert_verifies(logits, ids, first, u, accept, filters, probs)
    assert got[0][n] >= 60 and got[0][n + 1] == 0
    again = verified(logits, ids, first, u, accept, filters, probs)
    assert [x.tolist() for x in again] == got
    # rows in front of the first sequence and behind the last one; sequences that do not ascend are bounded by the rows, and others keep their tokens
    inner = [x + 3 for x in first[:-2]]
    rows = sum(counts)
    gained, tokens, logprobs = verified(logits, ids, inner, u, accept, filters, probs)
    assert (tokens[:3] == -1).all() and not logprobs[:3].any() and (tokens[min(rows, inner[-1]):] == -1).all()
    gained, tokens, _ = verified(logits, ids, [5, 50, 20, rows + 100, -4, 40], u, accept, filters, probs)
    assert 0 <= gained.min() and gained.max() <= rows


@pytest.mark.parametrize("drafter", [False, True])
def test_what_comes_out_has_the_target_s_distribution(drafter):
    """the first token of 2 x 10^5 sequences whose drafts come from another distribution: counts within five standard deviations of the target's"""
    vocab, n, rounds = 6, 4000, 50
    gen = torch.Generator(device="cuda").manual_seed(11)
    target, other = torch.randn(vocab, generator=gen, device="cuda"), torch.randn(vocab, generator=gen, device="cuda")
    q, p = torch.softmax(other, 0), torch.softmax(target, 0).cpu().double()
    counts = torch.zeros(vocab)
    for _ in range(rounds):
        draft = torch.multinomial(q.expand(n, -1), 1, generator=gen)[:, 0] if drafter else torch.randint(0, vocab, (n,), generator=gen, device="cuda")
        ids = torch.stack([torch.zeros_like(draft), draft], 1).flatten().int()
        rows = target.expand(2 * n, -1)
        u, accept = torch.rand(2 * n, generator=gen, device="cuda"), torch.rand(2 * n, generator=gen, device="cuda")
        first = torch.arange(0, 2 * n + 1, 2, device="cuda").int()
        _, tokens, _ = serve.verify(rows.contiguous(), ids, first, u, accept, draft_probs=q.expand(2 * n, -1).contiguous() if drafter else None)
        counts += torch.bincount(tokens[::2].long(), minlength=vocab).cpu()
    total = n * rounds
    assert ((counts.double() - total * p).abs() <= 5 * (total * p * (1 - p)).sqrt()).all(), (counts / total, p)


def test_verify_takes_rows_apart():
    """rows of logits and of drafts' distributions with strides, on any alignment"""
    logits, ids, first, u, accept, filters, probs = step(9, 5003, [3, 2, 4], F32, KINDS, True)
    want = verified(logits, ids, first, u, accept, filters, probs)
    for shift in (0, 1, 3):
        a, b = (torch.zeros(9, 5010, device="cuda")[:, shift:shift + 5003] for _ in range(2))
        a.copy_(logits)
        b.copy_(probs)
        assert all(torch.equal(x, y) for x, y in zip(want, verified(a, ids, first, u, accept, filters, b)))
