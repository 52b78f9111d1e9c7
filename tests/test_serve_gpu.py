"""booster_b200.serve on the GPU against tests/serve_oracle.py: the 4-bit cache, attention over it, its pages and the draw of tokens, at the sizes, masks and tables where they can go wrong."""
import math
import random

import numpy as np
import pytest
import torch

from booster_b200 import serve
from tests import serve_oracle as oracle

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


class Case:
    """a pool with sequences in scattered pages: counts[i] new rows behind held[i] tokens of slot slots[i]"""

    def __init__(self, held, counts, page=16, kv=2, hd=64, seed=0, spare=2, layers=1):
        r = random.Random(seed)
        n = len(held)
        self.page, self.kv, self.hd, self.held_l, self.counts = page, kv, hd, list(held), list(counts)
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
        self.pool = serve.kv4_pool(self.pages, page, kv, hd, layers)
        self.table, self.held, self.slots, self.first = ints(self.table_l), ints(at), ints(self.slots_l), ints(self.first_l)
        self.gen = torch.Generator(device="cuda").manual_seed(seed)

    def args(self):
        return self.pool[0], self.table, self.held, self.first

    def randn(self, *shape):
        return torch.randn(*shape, generator=self.gen, device="cuda")

    def fill(self, dtype=F16):
        """all tokens up to the step's last row are written; returns K and V [rows of all, kv, hd] of each sequence"""
        total = [h + c for h, c in zip(self.held_l, self.counts)]
        first = [0]
        for t in total:
            first.append(first[-1] + t)
        k, v = (self.randn(first[-1], self.kv, self.hd) * torch.exp(0.5 * self.randn(self.hd)) for _ in range(2))
        k, v = k.to(dtype), v.to(dtype)
        serve.kv4_append(self.pool[0], self.table, torch.zeros_like(self.held), ints(first), k, v, self.slots)
        self.k = [k[a:b].double().cpu().numpy() for a, b in zip(first, first[1:])]
        self.v = [v[a:b].double().cpu().numpy() for a, b in zip(first, first[1:])]

    def seen(self):
        """what the oracle sees of each sequence"""
        out = []
        for k, v in zip(self.k, self.v):
            rows = [[oracle.held_rows(k[t, h], v[t, h]) for t in range(len(k))] for h in range(self.kv)]
            K, V = (np.array([[rows[h][t][i] for t in range(len(k))] for h in range(self.kv)]).reshape(self.kv, len(k), self.hd) for i in (0, 1))
            out.append((K, V, np.ones(len(k), bool)))
        return out


def assert_attends(case, seen, q, out, window=0, scale=None):
    scale = case.hd ** -0.5 if scale is None else scale
    want, room = oracle.attention(q.double().cpu().numpy(), seen, case.held_l, case.first_l, window, scale)
    got = out.double().cpu().numpy()
    half = torch.finfo(q.dtype).eps / 2
    nan = np.isnan(want)
    assert np.array_equal(nan, np.isnan(got))
    over = np.abs(got - want)[~nan] - (room + half * (np.abs(want) + room) + 2.0 ** -25)[~nan]
    assert over.size == 0 or over.max() <= 0, f"off by {over.max():.3g} more than the roundings allow"


# ---- writing and reading -----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("page,held,counts", [(16, [0, 3, 15, 16, 40], [1, 1, 1, 1, 1]), (32, [7, 0, 31], [20, 1, 70]), (64, [100, 1], [1, 0]), (16, [2], [16]), (32, [5, 0, 16], [60, 1, 33]), (16, [15, 0], [50, 0])])
def test_append_writes_the_definition(hd, dtype, page, held, counts):
    c = Case(held, counts, page=page, kv=3, hd=hd, seed=hd + page)
    c.pool.copy_(torch.randint(0, 256, c.pool.shape, generator=c.gen, device="cuda", dtype=torch.uint8))
    before = c.pool[0].cpu().numpy()
    wide = c.randn(c.rows, 3 + 2 * 3, hd).to(dtype)                    # keys and values behind something else, in one tensor
    k, v = wide[:, 3:6], wide[:, 6:9]
    serve.kv4_append(*c.args(), k, v, c.slots)
    kn, vn = k.float().cpu().numpy(), v.float().cpu().numpy()
    for s, r, i in oracle.rows_of(c.first_l, c.rows):
        pos = c.held_l[s] + i
        p = oracle.page_of(c.table_l, c.slots_l[s], pos, page, c.pages)
        for h in range(3):
            oracle.write_tile(before[p, h, pos % page // 16], pos % 16, kn[r, h], vn[r, h])
    got = c.pool[0].cpu().numpy()
    assert np.array_equal(got, before), f"{(got != before).sum()} bytes differ"
    rk, rv = serve.kv4_read(*c.args(), c.rows, dtype, c.slots)
    want = [[oracle.held_rows(kn[r, h], vn[r, h]) for h in range(3)] for r in range(c.rows)]
    for i, x in enumerate((rk, rv)):
        w = torch.tensor(np.array([[want[r][h][i] for h in range(3)] for r in range(c.rows)])).reshape(c.rows, 3, hd).to(dtype)
        assert torch.equal(x.cpu(), w)


@pytest.mark.parametrize("shift", [1, 3])
def test_append_takes_rows_on_any_alignment(shift):
    c = Case([5, 20], [3, 1], kv=1, hd=64, seed=shift)
    flat = c.randn(2, c.rows * 67 + 8).to(F16)
    k, v = (flat[i, shift:shift + c.rows * 67].view(c.rows, 1, 67)[:, :, :64] for i in (0, 1))
    serve.kv4_append(*c.args(), k, v, c.slots)
    one = c.pool.clone()
    c.pool.zero_()
    serve.kv4_append(*c.args(), k.contiguous(), v.contiguous(), c.slots)
    assert torch.equal(one, c.pool)


def test_append_of_edge_values():
    c = Case([0], [12], kv=1, hd=64)
    k = c.randn(12, 1, 64)
    k[0] = 0
    k[1] = 1e-9                                                       # a scale below the smallest fp16: held as 0
    k[2] = 1e30                                                       # beyond 65280
    k[3, 0, :32] = torch.linspace(-1, 1, 32, device="cuda")           # both signs as large: the negative one is code 0
    k[4, 0, 5] = float("nan")
    k[5, 0, 40] = float("inf")
    k[6, 0, 0], k[6, 0, 1:32] = 1.0, torch.arange(31, device="cuda") / 16 - 0.9375      # quotients on halves
    k[7, 0, :32] = 3.0 * torch.arange(32, device="cuda") / 16
    k[8] = 2.0 ** -20 * c.randn(64)                                    # scales among fp16's subnormals
    v = c.randn(12, 1, 64)
    v[9, 0, 3] = -float("inf")
    serve.kv4_append(*c.args(), k, v, c.slots)
    got = [x.double().cpu().numpy()[:, 0] for x in serve.kv4_read(*c.args(), 12, F32, c.slots)]
    for r in range(12):
        for x, w in zip(got, oracle.held_rows(k[r, 0].cpu().numpy(), v[r, 0].cpu().numpy())):
            assert np.array_equal(x[r], w, equal_nan=True), r
    assert np.isnan(got[0][[4, 5, 9]]).all() and not got[1][[4, 5, 9]].any()


def test_rows_and_tables_that_do_not_exist():
    c = Case([3, 10, 4], [2, 2, 2], kv=1, hd=64)
    c.fill()
    whole = c.pool.clone()
    k = c.randn(c.rows + 3, 1, 64).half()
    slots = c.slots.clone()
    slots[1] = 99                                                     # no such slot
    table = c.table.clone()
    table[slots[2], 0] = c.pages                                       # no such page
    serve.kv4_append(c.pool[0], table, c.held, c.first, k, k, slots)
    page = c.table_l[c.slots_l[0]][0]
    changed = (c.pool[0] != whole[0]).flatten(1).any(1).nonzero().flatten().tolist()
    assert changed == [page]
    out = torch.full((c.rows + 3, 2, 64), 7.0, dtype=F16, device="cuda")
    serve.kv4_attention(k.expand(-1, 2, -1), c.pool[0], table, c.held, c.first, slots, out=out)
    assert (out[c.rows:] == 7).all() and not out[2:6].any() and torch.isfinite(out[:2]).all() and out[:2].any()
    rk, rv = torch.full((c.rows + 3, 1, 64), 7.0, dtype=F16, device="cuda"), torch.full((c.rows + 3, 1, 64), 7.0, dtype=F16, device="cuda")
    serve.kv4_read(c.pool[0], table, c.held, c.first, c.rows + 3, F16, slots, out=(rk, rv))
    assert (rk[c.rows:] == 7).all() and not rk[2:6].any() and (rv[c.rows:] == 7).all()


# ---- attention ---------------------------------------------------------------------------------------------------------------
LENGTHS = [0, 1, 15, 16, 17, 62, 63, 64, 200, 333]


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("heads,kv", [(4, 1), (4, 4), (8, 1), (6, 2), (16, 1)])
@pytest.mark.parametrize("page", [16, 64])
def test_attention_of_single_tokens(hd, heads, kv, page):
    c = Case(LENGTHS, [1] * len(LENGTHS), page=page, kv=kv, hd=hd, seed=heads)
    c.fill(BF16)
    q = (2 * c.randn(c.rows, heads, hd)).to(F16 if page == 16 else BF16)
    out = serve.kv4_attention(q, *c.args(), slots=c.slots, max_rows=1)
    assert_attends(c, c.seen(), q, out)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("heads,kv", [(4, 1), (2, 2), (10, 2)])
@pytest.mark.parametrize("held,counts", [([0, 30, 5], [3, 2, 1]), ([0], [70]), ([100, 0, 17], [40, 1, 33]), ([0, 250], [150, 0])])
@pytest.mark.parametrize("window", [0, 1, 20])
def test_attention_of_portions(hd, heads, kv, held, counts, window):
    c = Case(held, counts, page=32, kv=kv, hd=hd, seed=window)
    c.fill()
    q = (2 * c.randn(heads, c.rows, hd)).to(F16).transpose(0, 1)        # heads outside
    out = serve.kv4_attention(q, *c.args(), slots=c.slots, window=window, max_rows=max(counts), scale=0.2)
    assert_attends(c, c.seen(), q, out, window, 0.2)


@pytest.mark.parametrize("hd,heads,kv", [(64, 4, 2), (128, 8, 1)])
def test_attention_of_many_short_portions(hd, heads, kv):
    """blocks walk through many pieces of one and of two halves of columns, one after the other"""
    r = random.Random(hd)
    n = 260
    c = Case([r.randrange(0, 300) for _ in range(n)], [r.choice([17, 20, 33, 40, 64]) for _ in range(n)], kv=kv, hd=hd, seed=hd)
    c.fill()
    q = c.randn(c.rows, heads, hd).half()
    out = serve.kv4_attention(q, *c.args(), slots=c.slots, max_rows=64)
    # the same row by row, by the kernels of single tokens, which the tests above hold to the definition: both round P (2^-11) and the result
    one = torch.empty_like(out)
    for i in range(max(c.counts)):
        sel = [s for s in range(n) if i < c.counts[s]]
        rows = torch.tensor([c.first_l[s] + i for s in sel], device="cuda")
        held = c.held.clone()
        held[c.slots[sel].long()] += i
        one[rows] = serve.kv4_attention(q[rows], c.pool[0], c.table, held, ints(list(range(len(sel) + 1))), c.slots[sel], max_rows=1)
    assert torch.isfinite(out).all()
    big = max(np.abs(v).max() for v in c.v)
    assert (out.double() - one.double()).abs().max().item() <= big * (2 * 2.0 ** -11 + 2 * 2.0 ** -11 + 2.0 ** -14)


@pytest.mark.parametrize("rows,max_rows", [(70, 1), (70, 3), (3, 1000)])
def test_a_wrong_max_rows_changes_no_result(rows, max_rows):
    c = Case([20, 3], [rows, 2], kv=1, hd=64)
    c.fill()
    q = c.randn(c.rows, 4, 64).half()
    assert_attends(c, c.seen(), q, serve.kv4_attention(q, *c.args(), slots=c.slots, max_rows=max_rows))


def test_attention_over_large_and_small_numbers():
    c = Case([70] * 4, [1] * 4, kv=1, hd=64, seed=5)
    c.fill()
    for scale, dtype in ((3e4, BF16), (2e-5, BF16), (1e35, BF16), (6e3, F16)):
        q = (c.randn(4, 4, 64) * scale).to(dtype)
        out = serve.kv4_attention(q, *c.args(), slots=c.slots, scale=0.3 / scale)
        assert_attends(c, c.seen(), q, out, 0, float(np.float32(0.3 / scale)))


def test_scores_that_rise_and_fall():
    """the running maximum moves often, by more and by less than what the kernel lets pass"""
    for sign in (1, -1):
        c = Case([1000], [1], kv=1, hd=64, seed=6)
        c.fill(F32)
        k = torch.zeros(1001, 1, 64, device="cuda")
        k[:, 0, 0] = sign * torch.linspace(-60, 60, 1001, device="cuda")
        v = c.randn(1001, 1, 64)
        serve.kv4_append(c.pool[0], c.table, torch.zeros_like(c.held), ints([0, 1001]), k, v, c.slots)
        c.k, c.v = [k.double().cpu().numpy()], [v.double().cpu().numpy()]
        q = torch.zeros(1, 4, 64, device="cuda", dtype=F16)
        q[0, :, 0] = torch.tensor([0.1, 1.0, 3.0, -2.0])
        assert_attends(c, c.seen(), q, serve.kv4_attention(q, *c.args(), slots=c.slots, scale=1.0), 0, 1.0)


def test_nothing_is_seen_of_what_is_masked():
    """tokens that hold a NaN or an infinity: rows that see them answer NaN for that head, all others as if they were not there"""
    for rows in (8, 40):
        c = Case([20, 30], [rows, 2], kv=2, hd=64)
        c.fill()
        k = c.randn(rows + 2, 2, 64).half()
        v = c.randn(rows + 2, 2, 64).half()
        k[4, 0, 3], v[6, 1, 60], k[rows - 1, 1, 0] = float("nan"), float("inf"), -float("inf")
        serve.kv4_append(*c.args(), k, v, c.slots)
        for s, a in ((0, 0), (1, rows)):
            n = c.counts[s]
            c.k[s][c.held_l[s]:], c.v[s][c.held_l[s]:] = k[a:a + n].double().cpu().numpy(), v[a:a + n].double().cpu().numpy()
        q = c.randn(rows + 2, 4, 64).half()
        out = serve.kv4_attention(q, *c.args(), slots=c.slots, max_rows=rows)
        assert_attends(c, c.seen(), q, out)
        assert torch.isnan(out[4:rows, :2]).all() and torch.isfinite(out[:4]).all() and torch.isfinite(out[rows:]).all()
        # the window leaves the token behind
        out = serve.kv4_attention(q, *c.args(), slots=c.slots, max_rows=rows, window=2)
        assert torch.isfinite(out[6:rows - 1, :2]).all() and torch.isnan(out[4:6, :2]).all()


def test_absent_pages_are_not_seen():
    c = Case([100, 40], [1, 20], page=16, kv=1, hd=64)
    c.fill()
    table = c.table.clone()
    table[c.slots[0], 2], table[c.slots[1], 0] = -5, 10 ** 6
    q = c.randn(c.rows, 4, 64).half()
    seen = c.seen()
    seen[0][2][32:48] = False
    seen[1][2][0:16] = False
    assert_attends(c, seen, q, serve.kv4_attention(q, c.pool[0], table, c.held, c.first, c.slots))
    table.fill_(-1)
    assert not serve.kv4_attention(q, c.pool[0], table, c.held, c.first, c.slots).any()


def test_many_sequences_and_none():
    n = 700
    c = Case([(7 * i) % 40 for i in range(n)], [1 if i % 5 else 0 for i in range(n)], kv=1, hd=64, seed=1)
    c.fill()
    q = c.randn(c.rows, 2, 64).half()
    assert_attends(c, c.seen(), q, serve.kv4_attention(q, *c.args(), slots=c.slots, max_rows=1))
    empty = serve.kv4_attention(q[:0], c.pool[0], c.table, c.held, ints([0]), ints([]))
    assert empty.shape == (0, 2, 64)
    serve.kv4_append(c.pool[0], c.table, c.held, ints([0]), q[:0, :1], q[:0, :1], ints([]))
    assert serve.sample(torch.empty(0, 5, device="cuda"), torch.empty(0, device="cuda"))[0].shape == (0,)


def test_offsets_beyond_32_bits():
    """a pool of over 4 GB: pages at its end are written and read where they are"""
    page, kv, hd = 64, 8, 128
    size = kv * page // 16 * 18 * hd
    n = (1 << 32) // size + 10
    pool = serve.kv4_pool(n, page, kv, hd)
    table = ints([[n - 1, 3, n - 7]])
    k, v = (torch.randn(150, kv, hd, device="cuda", dtype=F16) for _ in range(2))
    serve.kv4_append(pool[0], table, ints([0]), ints([0, 150]), k, v)
    small = serve.kv4_pool(3, page, kv, hd)
    serve.kv4_append(small[0], ints([[0, 1, 2]]), ints([0]), ints([0, 150]), k, v)
    assert torch.equal(pool[0, [n - 1, 3, n - 7]], small[0])
    q = torch.randn(2, 16, hd, device="cuda", dtype=F16)
    a = serve.kv4_attention(q, pool[0], table, ints([148]), ints([0, 2]))
    assert torch.equal(a, serve.kv4_attention(q, small[0], ints([[0, 1, 2]]), ints([148]), ints([0, 2])))
    # whole layers apart, and copied there
    two = pool.view(-1)[: 2 * (n // 2) * size].view(2, n // 2, kv, page // 16, 18 * hd)
    two[1, n // 2 - 10].random_(0, 256)
    status = serve.pages_copy(two, ints([[0]]), ints([0] * (n // 2)), ints([n // 2 - 10]), ints([5]))
    assert status.item() == 0 and torch.equal(two[1, n // 2 - 10], two[1, 5]) and torch.equal(two[0, 5], two[0, n // 2 - 10])


@pytest.mark.parametrize("rows", [1, 40])
def test_graphs_streams_and_order(rows):
    """captured and replayed with other lengths; two graphs; another stream; the same call twice gives the same bits"""
    c = Case([90, 33, 0], [rows] * 3, page=16, kv=2, hd=128, seed=3)
    c.fill()
    q = c.randn(c.rows, 8, 128).half()
    held = c.held.clone()
    eager = [serve.kv4_attention(q, c.pool[0], c.table, held - d, c.first, c.slots, max_rows=rows) for d in (0, 0)]
    assert torch.equal(*eager)
    short = torch.clamp(held - 20, min=0)
    other = serve.kv4_attention(q, c.pool[0], c.table, short, c.first, c.slots, max_rows=rows)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    with torch.cuda.stream(stream):
        serve.kv4_attention(q, c.pool[0], c.table, held, c.first, c.slots, max_rows=rows)
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                outs.append(serve.kv4_attention(q, c.pool[0], c.table, held, c.first, c.slots, max_rows=rows))
            graphs.append(g)
        for lengths, want in ((c.held, eager[0]), (short, other), (c.held, eager[0])):
            held.copy_(lengths)
            for g in graphs:
                g.replay()
            stream.synchronize()
            assert torch.equal(outs[0], want) and torch.equal(outs[1], want)


# ---- pages -------------------------------------------------------------------------------------------------------------------
class Book:
    """the pages' life in plain numbers"""

    def __init__(self, n_pages, n_slots, width, page):
        self.table, self.held, self.refs, self.page = [[-1] * width for _ in range(n_slots)], [0] * n_slots, [0] * n_pages, page

    def free_pages(self):
        return [i for i, r in enumerate(self.refs) if r == 0]

    def reserve(self, slots, counts):
        free, todo = self.free_pages(), []
        if len(set(slots)) < len(slots) or any(not 0 <= s < len(self.table) or -(-(self.held[s] + c) // self.page) > len(self.table[0]) for s, c in zip(slots, counts)):
            return -1
        for s, c in zip(slots, counts):
            todo += [(s, i) for i in range(self.held[s] // self.page, -(-(self.held[s] + c) // self.page)) if self.table[s][i] < 0]
        if len(todo) > len(free):
            return len(todo) - len(free)
        for (s, i), p in zip(todo, free):
            self.table[s][i], self.refs[p] = p, 1
        return 0

    def fork(self, parents, children):
        n = len(self.table)
        if any(not 0 <= s < n for s in parents + children) or len(set(children)) < len(children) or set(parents) & set(children) or any(self.held[c] or self.table[c][0] >= 0 for c in children):
            return -1, []
        free, copies = self.free_pages(), []
        short = sum(self.held[a] % self.page != 0 for a in parents) - len(free)
        if short > 0:
            return short, []
        for a, c in zip(parents, children):
            full, rest = divmod(self.held[a], self.page)
            self.table[c] = self.table[a][:full] + [-1] * (len(self.table[a]) - full)
            for p in self.table[c][:full]:
                self.refs[p] += 1
            if rest:
                self.table[c][full] = free.pop(0)
                self.refs[self.table[c][full]] = 1
                copies.append((self.table[a][full], self.table[c][full], -(-rest // 16)))
            self.held[c] = self.held[a]
        return 0, copies

    def release(self, slots):
        for s in slots:
            if 0 <= s < len(self.table):
                for p in self.table[s]:
                    if p >= 0:
                        self.refs[p] -= 1
                self.table[s], self.held[s] = [-1] * len(self.table[s]), 0

    def compact(self):
        live = sum(r > 0 for r in self.refs)
        moved = dict(zip([i for i, r in enumerate(self.refs) if r > 0 and i >= live], [i for i, r in enumerate(self.refs) if r == 0 and i < live]))
        for a, b in moved.items():
            self.refs[b], self.refs[a] = self.refs[a], 0
        self.table = [[moved.get(p, p) for p in row] for row in self.table]
        return live, moved


@pytest.mark.parametrize("seed,n_pages,n_slots,width,page,layers,kv,hd", [(0, 40, 12, 6, 16, 2, 1, 64), (1, 3001, 64, 70, 32, 1, 2, 64), (2, 33, 9, 5, 64, 3, 2, 128), (3, 31, 5, 40, 16, 1, 1, 64)])
def test_pages_live_as_the_book_says(seed, n_pages, n_slots, width, page, layers, kv, hd):
    r = random.Random(seed)
    b = Book(n_pages, n_slots, width, page)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    pool = torch.randint(0, 256, (layers, n_pages, kv, page // 16, 18 * hd), generator=gen, device="cuda", dtype=torch.uint8)
    table, held, refs = ints(b.table), ints(b.held), ints(b.refs)
    seen = set()
    for step in range(60):
        want = pool.cpu()
        do = r.choice(["reserve", "reserve", "fork", "fork", "free", "compact", "copy"])
        if do == "reserve":
            slots = r.sample(range(n_slots), r.randrange(0, n_slots + 1)) + ([n_slots] if r.random() < 0.1 else []) + ([0, 0] if r.random() < 0.1 else [])
            counts = [r.randrange(0, page * width // 3) for _ in slots]
            first = [0]
            for c in counts:
                first.append(first[-1] + c)
            got, status = serve.pages_reserve(table, held, refs, ints(first), page, ints(slots)).item(), b.reserve(slots, counts)
            if status == 0:
                for s, c in zip(slots, counts):
                    b.held[s] += c
                held.copy_(ints(b.held))
        elif do == "fork":
            n = r.randrange(0, n_slots // 2 + 1)
            parents = [r.randrange(n_slots) for _ in range(n)]
            empty = [s for s in range(n_slots) if b.held[s] == 0 and b.table[s][0] < 0 and s not in parents]
            children = r.sample(empty, min(n, len(empty))) if r.random() < 0.9 else [r.randrange(-1, n_slots + 1) for _ in range(n)]
            parents = parents[:len(children)]
            got = serve.pages_fork(pool, table, held, refs, ints(parents), ints(children)).item()
            status, copies = b.fork(parents, children)
            for x, y, t in copies:
                want[:, y, :, :t] = want[:, x, :, :t]
        elif do == "free":
            slots = [r.randrange(-1, n_slots + 1) for _ in range(r.randrange(0, 5))]
            serve.pages_free(table, held, refs, ints(slots))
            b.release(slots)
            got = status = 0
        elif do == "compact":
            got, (status, moved) = serve.pages_compact(pool, table, refs).item(), b.compact()
            for x, y in moved.items():
                want[:, y] = want[:, x]
        else:
            n = r.randrange(0, min(6, n_pages // 2))
            pick = r.sample(range(n_pages), 2 * n)
            src, dst = [r.choice(pick[:n]) for _ in range(n)], pick[n:]
            fault = r.random()
            if n and fault < 0.1:
                dst[0] = src[-1]
            elif n > 1 and fault < 0.2:
                dst[0] = dst[1]
            elif n and fault < 0.3:
                src[0] = n_pages
            status = -1 if len(set(dst)) < n or set(src) & set(dst) or any(not 0 <= p < n_pages for p in src + dst) else 0
            got = serve.pages_copy(pool, table, refs, ints(src), ints(dst)).item()
            if status == 0:
                for x, y in zip(src, dst):
                    want[:, y] = want[:, x]
        seen.add((do, min(1, max(-1, status))))
        assert got == status, (step, do)
        assert table.tolist() == b.table and held.tolist() == b.held and refs.tolist() == b.refs, (step, do)
        assert torch.equal(pool.cpu(), want), (step, do)
    assert ("fork", 0) in seen and ("reserve", 0) in seen


def test_reserved_pages_are_not_reserved_again():
    table, held, refs = ints([[-1] * 4, [-1] * 4]), ints([0, 5]), ints([0] * 8)
    first = ints([0, 20, 30])
    for _ in range(2):
        assert serve.pages_reserve(table, held, refs, first, 16).item() == 0
        assert table.tolist() == [[0, 1, -1, -1], [2, -1, -1, -1]] and refs.tolist() == [1, 1, 1, 0, 0, 0, 0, 0]
    assert serve.pages_reserve(table, held, refs, ints([0, 64, 64]), 16).item() == 0 and serve.pages_reserve(table, held, refs, ints([0, 65, 65]), 16).item() == -1
    assert serve.pages_reserve(table, held, refs, ints([0, 0, 59]), 16).item() == 0 and refs.tolist() == [1] * 8
    held[0] = 64
    refs2 = refs.clone()
    assert serve.pages_reserve(ints([[-1] * 4]), ints([0]), refs, ints([0, 33]), 16).item() == 3 and torch.equal(refs, refs2)


# ---- sampling ----------------------------------------------------------------------------------------------------------------
def check_rows(logits, u, **p):
    n = len(logits)
    params = {k: torch.tensor(v, dtype=torch.int32 if k == "top_k" else F32, device="cuda") for k, v in p.items()}
    ids, lp = serve.sample(logits, u, **params)
    x, uu = logits.float().cpu().numpy(), u.double().cpu().numpy()
    for r in range(n):
        want, share, near = oracle.sample(x[r], uu[r], **{k: float(t[r].double()) if k != "top_k" else int(t[r]) for k, t in params.items()})
        if near > 1e-9:                                                # weights are multiples of 2^-40: closer to a border the sums of 64 bits do not decide either
            assert ids[r].item() == want, (r, {k: v[r] for k, v in p.items()}, ids[r].item(), want, near)
            # the log is rounded to float32 at the end; the sum holds the share to 2^-30
            assert lp[r].item() == share or abs(lp[r].item() - share) <= 2.0 ** -24 * abs(share) + 2.0 ** -30, (r, lp[r].item(), share)
    return ids, lp


SETTINGS = [dict(top_k=40, top_p=0.95, min_p=0.05, temperature=0.8), dict(top_p=0.9), dict(top_k=1), dict(min_p=0.1, temperature=1.5), dict(temperature=0.0), dict(), dict(top_k=200, top_p=0.3),
            dict(top_p=0.999), dict(top_p=0.0), dict(top_k=10 ** 6, top_p=0.5), dict(min_p=1.0), dict(temperature=0.01), dict(temperature=100.0, top_k=7), dict(top_k=-3, top_p=2.0)]


@pytest.mark.parametrize("vocab", [1, 2, 31, 1000, 4099, 32064, 128256])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_sample_follows_the_definition(vocab, dtype):
    gen = torch.Generator(device="cuda").manual_seed(vocab)
    n = 2 * len(SETTINGS)
    rows = torch.randn(n, vocab + 3, generator=gen, device="cuda")[:, :vocab] * torch.linspace(0.5, 5, n, device="cuda")[:, None]
    rows = rows.to(dtype)
    u = torch.rand(n, generator=gen, device="cuda")
    u[0], u[1] = 0.0, 1 - 2.0 ** -24
    p = {k: [(SETTINGS[r % len(SETTINGS)]).get(k, d) for r in range(n)] for k, d in (("top_k", 0), ("top_p", 1.0), ("min_p", 0.0), ("temperature", 1.0))}
    first = check_rows(rows, u, **p)
    again = check_rows(rows.clone(), u, **p)                           # rows on another alignment
    assert all(torch.equal(a, b) for a, b in zip(first, again))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_sample_among_equals(dtype):
    """ties at every border: constant rows, few distinct values, blocks of equals of thousands"""
    vocab = 20000
    gen = torch.Generator(device="cuda").manual_seed(2)
    i = torch.arange(vocab, device="cuda")
    rows = torch.stack([torch.zeros(vocab, device="cuda"), (i % 7).float(), -(i % 3).float() * 2, torch.where(i < 9000, 1.0, -4.0), torch.randint(0, 5, (vocab,), generator=gen, device="cuda") / 4.0,
                        torch.where(i % 2 == 0, 0.0, -0.0)]).to(dtype)
    for k, top_p, min_p in ((0, 0.5, 0.0), (5, 1.0, 0.0), (6000, 0.7, 0.0), (0, 0.123, 0.5), (5000, 1.0, 0.0), (0, 0.99, 0.0), (4097, 0.5, 0.9)):
        u = torch.rand(6, generator=gen, device="cuda")
        check_rows(rows, u, top_k=[k] * 6, top_p=[top_p] * 6, min_p=[min_p] * 6, temperature=[0.7] * 6)


def test_sample_of_values_that_are_not_finite():
    inf, nan = float("inf"), float("nan")
    rows = torch.tensor([[-inf] * 5, [nan] * 5, [1, nan, -inf, 2, 0], [inf, 1, inf, nan, -inf], [-inf, -inf, -3, -inf, -inf], [3e38, -3e38, 0, 3e38, 1]], device="cuda")
    u = torch.tensor([0.3, 0.3, 0.6, 0.7, 0.9, 0.2], device="cuda")
    for p in (dict(), dict(top_k=[2] * 6), dict(top_p=[0.8] * 6), dict(temperature=[0.0] * 6), dict(min_p=[0.5] * 6, temperature=[2.0] * 6), dict(top_k=[5] * 6, top_p=[0.9] * 6)):
        ids, lp = check_rows(rows, u, **p)
        assert ids[:2].tolist() == [-1, -1] and (lp[:2] == -inf).all() and ids[4].item() == 2


def test_sample_draws_by_weight():
    """the shares of 200 thousand draws from one row are its distribution's"""
    n = 200000
    gen = torch.Generator(device="cuda").manual_seed(9)
    x = torch.randn(1, 50, generator=gen, device="cuda")
    u = (torch.arange(n, device="cuda") + 0.5) / n                     # every 1 / n once: counts are off by one at most for each of a token's two borders, and one for u's rounding
    ids, lp = serve.sample(x.expand(n, 50).contiguous(), u)
    p = torch.softmax(x[0].double(), 0)
    counts = torch.bincount(ids.long(), minlength=50)
    assert (counts - n * p).abs().max() <= 3
    assert (lp.double() - torch.log(p)[ids.long()]).abs().max() < 1e-6


# ---- together ----------------------------------------------------------------------------------------------------------------
def test_a_server_of_them_together():
    """prompts, then tokens of several answers to each: reserve, append, attend, sample, advance; forks, ends and compactions between. At the end what each slot attends to is what its own
    tokens say, and all pages come back"""
    layers, heads, kv, hd, page, vocab, slots = 2, 4, 2, 64, 16, 300, 6
    r = random.Random(4)
    gen = torch.Generator(device="cuda").manual_seed(4)
    embed, wq = torch.randn(vocab, layers, (heads + 2 * kv) * hd, generator=gen, device="cuda").half(), torch.randn(heads * hd, vocab, generator=gen, device="cuda") / 12
    pool = serve.kv4_pool(60, page, kv, hd, layers)
    table, held, refs = ints([[-1] * 12] * slots), ints([0] * slots), ints([0] * 60)
    said = {}

    def step(new):
        ids, counts = list(new), [len(t) for t in new.values()]
        first = ints([sum(counts[:i]) for i in range(len(counts) + 1)])
        on, tokens = ints(ids), torch.tensor(sum(new.values(), []), device="cuda")
        assert serve.pages_reserve(table, held, refs, first, page, on).item() == 0
        x = torch.zeros(len(tokens), heads * hd, device="cuda")
        for layer in range(layers):
            row = embed[tokens, layer].view(len(tokens), -1, hd)
            serve.kv4_append(pool[layer], table, held, first, row[:, heads:heads + kv], row[:, heads + kv:], on)
            x += serve.kv4_attention(row[:, :heads], pool[layer], table, held, first, on, max_rows=max(counts)).flatten(1).float()
        held[on.long()] += first.diff()
        for s, t in new.items():
            said[s] = said.get(s, []) + t
        last = x[first[1:].long() - 1]
        picked, _ = serve.sample(last @ wq, torch.rand(len(ids), generator=gen, device="cuda"), top_k=ints([20] * len(ids)))
        return dict(zip(ids, picked.tolist())), dict(zip(ids, last))

    following, _ = step({0: [r.randrange(vocab) for _ in range(37)], 3: [r.randrange(vocab) for _ in range(16)]})
    for turn in range(40):
        following, last = step({s: [t] for s, t in following.items()})
        if turn in (3, 9, 20):
            empty = [s for s in range(slots) if s not in said][:2]
            parents = r.choices(sorted(said), k=len(empty))
            assert serve.pages_fork(pool, table, held, refs, ints(parents), ints(empty)).item() == 0
            for a, c in zip(parents, empty):
                said[c], following[c] = list(said[a]), r.randrange(vocab)
        if turn in (8, 19, 30):
            gone = r.sample(sorted(said), len(said) - 2)
            serve.pages_free(table, held, refs, ints(gone))
            for s in gone:
                del said[s], following[s]
            live = serve.pages_compact(pool, table, refs).item()
            assert live == (refs > 0).sum().item() and not refs[live:].any()
        assert all(held[s].item() == len(t) for s, t in said.items())
    for s in sorted(said):
        tokens = torch.tensor(said[s], device="cuda")
        want = np.zeros((1, heads * hd))
        room = np.zeros((1, heads * hd))
        for layer in range(layers):
            row = embed[tokens, layer].view(len(tokens), -1, hd).double().cpu().numpy()
            kvs = [[oracle.held_rows(row[t, heads + h], row[t, heads + kv + h]) for t in range(len(tokens))] for h in range(kv)]
            K, V = (np.array([[kvs[h][t][i] for t in range(len(tokens))] for h in range(kv)]) for i in (0, 1))
            o, e = oracle.attention(row[-1:, :heads], [(K, V, np.ones(len(tokens), bool))], [len(tokens) - 1], [0, 1], 0, hd ** -0.5)
            want += o.reshape(1, -1)
            room += (e + 2.0 ** -11 * (np.abs(o) + e)).reshape(1, -1) + 2.0 ** -23 * np.abs(want)
        if s in last:
            assert (np.abs(last[s].double().cpu().numpy() - want[0]) <= room[0]).all()
    serve.pages_free(table, held, refs, ints(sorted(said)))
    assert not refs.any() and (table == -1).all() and not held.any()
