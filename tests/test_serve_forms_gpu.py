"""Attention over the 4-bit cache by its form for many rows, which a call reaches by what it announces as the largest number of rows: the sizes, masks, tables and numbers at which the form
for few rows is tested give the definition here too. Bounds of the roundings: tests/serve_oracle.py."""
import numpy as np
import pytest
import torch

from booster_b200 import serve
from tests.test_serve_gpu import BF16, F16, F32, LENGTHS, Case, assert_attends, ints

pytestmark = pytest.mark.gpu

MANY = 4096                              # rows announced: always the form for many


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("heads,kv", [(4, 1), (8, 1), (6, 2), (2, 2)])
def test_single_tokens(hd, heads, kv):
    c = Case(LENGTHS, [1] * len(LENGTHS), page=64, kv=kv, hd=hd, seed=heads)
    c.fill(BF16)
    q = (2 * c.randn(c.rows, heads, hd)).to(BF16)
    assert_attends(c, c.seen(), q, serve.kv4_attention(q, *c.args(), slots=c.slots, max_rows=MANY))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("heads,kv", [(4, 1), (2, 2), (10, 2)])
@pytest.mark.parametrize("held,counts", [([0, 30, 5], [3, 2, 1]), ([0], [70]), ([100, 0, 17], [40, 1, 33]), ([0, 250], [150, 0]), ([600], [64])])
@pytest.mark.parametrize("window", [0, 1, 20])
def test_portions(hd, heads, kv, held, counts, window):
    c = Case(held, counts, page=32, kv=kv, hd=hd, seed=window)
    c.fill()
    q = (2 * c.randn(heads, c.rows, hd)).to(F16).transpose(0, 1)        # heads outside
    assert_attends(c, c.seen(), q, serve.kv4_attention(q, *c.args(), slots=c.slots, window=window, max_rows=MANY, scale=0.2), window, 0.2)


def test_queries_on_any_alignment_and_head_stride():
    c = Case([33], [20], kv=1, hd=64)
    c.fill()
    flat = c.randn(c.rows * 4 * 67 + 8).to(F16)
    for shift in (0, 1, 3):
        q = flat[shift:shift + c.rows * 4 * 67].view(c.rows, 4, 67)[:, :, :64]
        assert_attends(c, c.seen(), q, serve.kv4_attention(q, *c.args(), slots=c.slots, max_rows=MANY))


def test_large_and_small_numbers():
    c = Case([70] * 4, [1] * 4, kv=1, hd=64, seed=5)
    c.fill()
    for scale, dtype in ((3e4, BF16), (2e-5, BF16), (1e35, BF16), (6e3, F16)):
        q = (c.randn(4, 4, 64) * scale).to(dtype)
        out = serve.kv4_attention(q, *c.args(), slots=c.slots, scale=0.3 / scale, max_rows=MANY)
        assert_attends(c, c.seen(), q, out, 0, float(np.float32(0.3 / scale)))


def test_scores_that_rise_and_fall():
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
        assert_attends(c, c.seen(), q, serve.kv4_attention(q, *c.args(), slots=c.slots, scale=1.0, max_rows=MANY), 0, 1.0)


def test_nothing_is_seen_of_what_is_masked():
    rows = 40
    c = Case([20, 30], [rows, 2], kv=2, hd=64)
    c.fill()
    k, v = c.randn(rows + 2, 2, 64).half(), c.randn(rows + 2, 2, 64).half()
    k[4, 0, 3], v[6, 1, 60], k[rows - 1, 1, 0] = float("nan"), float("inf"), -float("inf")
    serve.kv4_append(*c.args(), k, v, c.slots)
    for s, a in ((0, 0), (1, rows)):
        n = c.counts[s]
        c.k[s][c.held_l[s]:], c.v[s][c.held_l[s]:] = k[a:a + n].double().cpu().numpy(), v[a:a + n].double().cpu().numpy()
    q = c.randn(rows + 2, 4, 64).half()
    out = serve.kv4_attention(q, *c.args(), slots=c.slots, max_rows=MANY)
    assert_attends(c, c.seen(), q, out)
    assert torch.isnan(out[4:rows, :2]).all() and torch.isfinite(out[:4]).all() and torch.isfinite(out[rows:]).all()
    out = serve.kv4_attention(q, *c.args(), slots=c.slots, max_rows=MANY, window=2)
    assert torch.isfinite(out[6:rows - 1, :2]).all() and torch.isnan(out[4:6, :2]).all()


def test_absent_pages_are_not_seen():
    c = Case([100, 40, 300], [1, 20, 30], page=16, kv=1, hd=64)
    c.fill()
    table = c.table.clone()
    table[c.slots[0], 2], table[c.slots[1], 0], table[c.slots[2], 5:9] = -5, 10 ** 6, -1
    q = c.randn(c.rows, 4, 64).half()
    seen = c.seen()
    seen[0][2][32:48] = False
    seen[1][2][0:16] = False
    seen[2][2][80:144] = False
    assert_attends(c, seen, q, serve.kv4_attention(q, c.pool[0], table, c.held, c.first, c.slots, max_rows=MANY))
    table.fill_(-1)
    assert not serve.kv4_attention(q, c.pool[0], table, c.held, c.first, c.slots, max_rows=MANY).any()


@pytest.mark.parametrize("max_rows", [1, MANY])
def test_rows_that_do_not_ascend_stay_within_bounds(max_rows):
    """`first` that goes up and down says nothing, but what it writes are rows of the step: those behind them, and what other calls answer, stay"""
    n = 64
    c = Case([40] * n, [3] * n, kv=1, hd=64)
    c.fill()
    rows = c.rows
    out = torch.full((rows + 4, 4, 64), 7.0, dtype=F16, device="cuda")
    q = c.randn(rows, 4, 64).half()
    right = serve.kv4_attention(q, *c.args(), slots=c.slots, max_rows=max_rows)
    first = ints([0 if i % 2 else rows for i in range(n + 1)])
    serve.kv4_attention(q, c.pool[0], c.table, c.held, first, c.slots, max_rows=max_rows, out=out[:rows])
    assert (out[rows:] == 7).all()
    assert torch.equal(right, serve.kv4_attention(q, *c.args(), slots=c.slots, max_rows=max_rows))


@pytest.mark.parametrize("n_pages,n_slots,offset", [(1 << 20, 1 << 18, 0), (5003, 40, 1), (70001, 300, 2)])
def test_reserving_in_large_and_odd_pools(n_pages, n_slots, offset):
    """thousands of pages by one call, counts on any alignment: the lowest free ones, in the order of the call's sequences"""
    g = torch.Generator().manual_seed(n_pages)
    refs_h = (torch.rand(n_pages, generator=g) < 0.3).int() * 3
    flat = torch.zeros(n_pages + 4, dtype=torch.int32, device="cuda")
    refs = flat[offset:offset + n_pages]
    refs.copy_(refs_h)
    n, width = 33, 120
    table = torch.full((n_slots, width), -1, dtype=torch.int32, device="cuda")
    held = torch.zeros(n_slots, dtype=torch.int32, device="cuda")
    slots = torch.randperm(n_slots, generator=g)[:n]
    counts = torch.randint(0, width + 1, (n,), generator=g)
    first = torch.cat([torch.zeros(1, dtype=torch.long), (counts * 16).cumsum(0)])
    free = (refs_h == 0).nonzero().flatten()
    assert serve.pages_reserve(table, held, refs, first.int().cuda(), 16, slots.int().cuda()).item() == 0
    at = 0
    want = torch.full((n_slots, width), -1, dtype=torch.int32)
    for s, c in zip(slots.tolist(), counts.tolist()):
        want[s, :c] = free[at:at + c].int()
        at += c
    refs_h[free[:at]] = 1
    assert at > 1000 and torch.equal(table.cpu(), want) and torch.equal(refs.cpu(), refs_h) and not flat[:offset].any() and not flat[offset + n_pages:].any()
    # and given back
    serve.pages_free(table, held, refs, slots.int().cuda())
    refs_h[free[:at]] = 0
    assert (table == -1).all() and torch.equal(refs.cpu(), refs_h)


@pytest.mark.parametrize("n", [2500, 4096])
def test_as_many_sequences_as_there_may_be(n):
    """both forms over thousands of sequences, some without rows, against the form for few rows on 500 of them at a time. All round P and the result to 2^-11"""
    c = Case([(7 * i) % 40 for i in range(n)], [(1, 1, 2, 0, 1)[i % 5] for i in range(n)], kv=1, hd=64, seed=1)
    c.fill()
    q = c.randn(c.rows, 2, 64).half()
    outs = [serve.kv4_attention(q, *c.args(), slots=c.slots, max_rows=m) for m in (2, MANY)]
    parts = []
    for s in range(0, n, 500):
        e = min(n, s + 500)
        a, b = c.first_l[s], c.first_l[e]
        parts.append(serve.kv4_attention(q[a:b], c.pool[0], c.table, c.held, c.first[s:e + 1] - a, c.slots[s:e], max_rows=2))
    want = torch.cat(parts).double()
    big = max(np.abs(v).max() for v in c.v if v.size)
    for out in outs:
        assert torch.isfinite(out).all() and (out.double() - want).abs().max().item() <= big * (2 * 2.0 ** -11 + 2 * 2.0 ** -11 + 2.0 ** -14)
    # the cache and the pages take as many: a further token each, reserved, written and read back
    refs = torch.zeros(c.pages, dtype=torch.int32, device="cuda")
    used = c.table[c.table >= 0].long()
    refs[used] = 1
    extra = serve.kv4_pool(c.pages + n, c.page, 1, 64)
    refs = torch.cat([refs, torch.zeros(n, dtype=torch.int32, device="cuda")])
    held = c.held.clone()
    held[c.slots.long()] += ints(c.counts)
    one = ints(range(n + 1))
    assert serve.pages_reserve(c.table, held, refs, one, c.page, c.slots).item() == 0
    k = c.randn(n, 1, 64).half()
    serve.kv4_append(extra[0], c.table, held, one, k, -k, c.slots)
    rk, rv = serve.kv4_read(extra[0], c.table, held, one, n, F16, c.slots)
    # half a step of a code, an eighth of the block's largest entry, and at the side that has no code 8 a whole one; d itself is rounded to 2^-8
    step = k.float().view(n, 1, 2, 32).abs().amax(-1, keepdim=True).expand(n, 1, 2, 32).reshape(n, 1, 64) / 8
    assert ((rk.float() - k.float()).abs() <= 1.05 * step).all() and ((rv.float() + k.float()).abs() <= 1.05 * step).all()
    assert (refs >= 0).all() and refs.max().item() == 1


@pytest.mark.parametrize("max_rows", [1, MANY])
@pytest.mark.parametrize("page", [128, 1024])
@pytest.mark.parametrize("window", [0, 33, 70])
def test_long_pages(max_rows, page, window):
    """sequences that end and windows that begin anywhere in a page"""
    c = Case([0, 127, 128, 700, 1023, 1024, 1500], [1, 2, 1, 3, 1, 1, 2], page=page, kv=2, hd=64, seed=page)
    c.fill()
    q = c.randn(c.rows, 4, 64).half()
    assert_attends(c, c.seen(), q, serve.kv4_attention(q, *c.args(), slots=c.slots, window=window, max_rows=max_rows), window)


@pytest.mark.parametrize("max_rows", [1, MANY])
@pytest.mark.parametrize("heads", [71, 128, 300])
def test_many_heads_on_one(max_rows, heads):
    c = Case([40, 0, 17], [1, 1, 2], kv=1, hd=64, seed=heads)
    c.fill()
    q = c.randn(c.rows, heads, 64).to(BF16)
    assert_attends(c, c.seen(), q, serve.kv4_attention(q, *c.args(), slots=c.slots, max_rows=max_rows))
