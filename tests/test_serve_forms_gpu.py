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
