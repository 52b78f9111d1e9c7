"""Attention over the 16-bit cache on the GPU, each of its forms by itself (tests/serve_draft_bounds.py): the bits that a form keeps, the edges of windows and first tokens at long contexts, values up
to the ends of the type's range, and waits that run out."""
import numpy as np
import pytest
import torch

from booster_b200 import _lib, serve
from tests import serve_draft_bounds as bounds
from tests.test_serve_draft_gpu import BF16, F16, Case

pytestmark = pytest.mark.gpu


def made(form, held, kv=2, hd=64, page=32, dtype=BF16, seed=0):
    """sequences of so many tokens with the rows of a form; its query heads a KV head; what a call of it gets"""
    rows, group, wide, once = bounds.FORMS[form]
    c = Case(held, [rows] * len(held), page=page, kv=kv, hd=hd, seed=seed, dtype=dtype)
    if wide:
        c.widened()
    return c, group, once


def attend(c, q, **more):
    return serve.kv16_attention(q, *c.args(), slots=c.slots, max_rows=max(c.counts), **more)


@pytest.mark.parametrize("form", bounds.FORMS)
@pytest.mark.parametrize("dtype,hd,window,sinks", [(BF16, 128, 0, 0), (BF16, 64, 50, 3), (F16, 64, 0, 0), (F16, 128, 50, 3)])
def test_bits_of_each_form(form, dtype, hd, window, sinks):
    c, group, once = made(form, [30, 190, 0], hd=hd, dtype=dtype, seed=hd)
    c.fill()
    q = (1.5 * c.randn(c.rows, 2 * group, hd)).to(dtype)
    out = attend(c, q, window=window, sinks=sinks).double().cpu().numpy()
    want, room = bounds.attention(q.double().cpu().numpy(), c.seen(), c.held_l, c.first_l, window, sinks, hd ** -0.5, dtype == BF16, once)
    over = np.abs(out - want) / room
    assert over.max() <= 1.0, f"off by {over.max():.3g} of what the form's roundings allow"


@pytest.mark.parametrize("form", bounds.FORMS)
@pytest.mark.parametrize("hd,page,window,sinks", [(64, 32, 1500, 4), (64, 16, 70, 33), (128, 256, 1203, 129), (128, 64, 0, 0), (64, 128, 1, 0), (64, 64, 33, 5000), (128, 16, 517, 31)])
def test_edges_of_windows_and_first_tokens(form, hd, page, window, sinks):
    """keys of 0 and values that are 1 at one dim each: results count, for each dim, the positions that are seen. What nobody may see is 100"""
    c, group, _ = made(form, [1903, 777, 5], hd=hd, page=page, dtype=BF16)
    c.pool[0, :, 0], c.pool[0, :, 1] = 0.0, 100.0
    eye = torch.eye(hd, dtype=BF16, device="cuda")
    for s, h, n in zip(c.slots_l, c.held_l, c.counts):
        for i in range(-(-(h + n) // page)):
            some = min(page, h + n - i * page)
            c.pool[0, c.table_l[s][i], 1, :, :some] = eye[torch.arange(i * page, i * page + some, device="cuda") % hd]
    q = c.randn(c.rows, 2 * group, hd).to(BF16)
    out = attend(c, q, window=window, sinks=sinks).double().cpu().numpy()
    for s, (h, n) in enumerate(zip(c.held_l, c.counts)):
        for r in range(n):
            j = bounds.seen(h + r, np.ones(h + n, bool), window, sinks)
            count = np.bincount(j % hd, minlength=hd)
            got = out[c.first_l[s] + r] * j.size
            assert (np.rint(got) == count).all()
            assert (np.abs(got - count) <= count * (2.0 ** -8 + 2.0 ** -12)).all()      # (weights are all the same: one rounding of the result)


@pytest.mark.parametrize("form", bounds.FORMS)
@pytest.mark.parametrize("hd", [64, 128])
def test_values_up_to_the_ends_of_bfloat16(form, hd):
    """a power of two on the values is one on the results: nothing on the way is larger than the largest value"""
    c, group, _ = made(form, [1500, 300, 0], hd=hd, page=64, seed=3)
    c.fill()
    c.pool[0, :, 1].clamp_(-7.96875, 7.96875)                           # below 2^3
    q = (1.5 * c.randn(c.rows, 2 * group, hd)).to(BF16)
    values = c.pool[0, :, 1].clone()
    right = attend(c, q)
    assert torch.isfinite(right).all()
    for k in (60, 100, 125):                                            # below 2^128
        c.pool[0, :, 1] = values * 2.0 ** k
        assert torch.equal(attend(c, q), right * 2.0 ** k)
    # small ones keep what the result's rounding keeps: weights of 2^-38 and more, of which those below 2^-26 of the largest may be lost with values of 2^-60
    c.pool[0, :, 1] = values * 2.0 ** -60
    small = attend(c, q).double() * 2.0 ** 60
    assert ((small - right.double()).abs() <= 2.0 ** -7 * right.double().abs() + 2.0 ** -20).all()


@pytest.mark.parametrize("form", bounds.FORMS)
def test_the_largest_number_as_it_stands(form):
    """one position seen gives its value, and a thousand that are the same give that one"""
    c, group, _ = made(form, [1000, 70], hd=128, page=16)
    c.fill()
    most = torch.finfo(BF16).max
    c.pool[0, :, 1] = torch.where(c.pool[0, :, 1] > 0, most, -most)
    q = c.randn(c.rows, 2 * group, 128).to(BF16)
    out = attend(c, q, window=1)
    for s, f, h, n in zip(c.slots_l, c.first_l, c.held_l, c.counts):
        for r in range(n):
            v = c.pool[0, c.table_l[s][(h + r) // 16], 1, :, (h + r) % 16]
            assert torch.equal(out[f + r], v.repeat_interleave(group, 0))
    assert torch.isfinite(attend(c, q)).all()
    c.pool[0, :, 0], c.pool[0, :, 1] = 0.0, most
    assert torch.equal(attend(c, q), torch.full_like(q, most))


@pytest.mark.parametrize("form", bounds.FORMS)
@pytest.mark.parametrize("hd", [64, 128])
def test_waits_that_run_out_in_each_form(form, hd):
    """what a wait is for never comes: the kernel gives up and ends, the next call says so and does nothing, and after it all is as before"""
    c, group, _ = made(form, [1000, 333, 0], hd=hd, page=16)
    c.fill()
    q = c.randn(c.rows, 2 * group, hd).to(BF16)
    right = attend(c, q)
    pool = c.pool.clone()
    serve.kv4_status()
    try:
        _lib.lib().b200_kv4_drill(64)
        attend(c, q)
        _lib.lib().b200_kv4_drill(0)
        torch.cuda.synchronize()
        with pytest.raises(_lib.B200Error, match="ran out"):
            attend(c, q)
        serve.kv4_status()
        assert torch.equal(c.pool, pool) and torch.equal(attend(c, q), right)
    finally:
        _lib.lib().b200_kv4_drill(0)


@pytest.mark.parametrize("rows,group,wide", [(1, 4, False), (3, 5, False), (5, 4, False), (9, 7, False), (2, 4, True), (3, 5, True), (5, 4, True), (37, 4, True), (9, 2, True), (40, 16, True), (7, 5, True)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_other_sequences_queries_change_nothing(rows, group, wide, dtype):
    """bit by bit: what stands beside a sequence's rows, behind its last one, or is written there by the same call (out is q) is nothing to them"""
    c = Case([300, 700, 20, 1000, 64, 411], [rows] * 6, page=16, dtype=dtype, seed=5)
    if wide:
        c.widened()
    c.fill()
    q = (2.0 * c.randn(c.rows, 2 * group, 64)).to(dtype)
    right = attend(c, q)
    mine = torch.zeros(c.rows, dtype=torch.bool, device="cuda")
    for s in (0, 2, 4):
        mine[c.first_l[s]:c.first_l[s + 1]] = True
    for other in (30.0, 0.0, float("nan"), float("inf")):
        p = q.clone()
        p[~mine] = p[~mine] * other if other < 100 else other
        assert torch.equal(attend(c, p)[mine], right[mine])
    for _ in range(20):
        p = q.clone()
        assert torch.equal(attend(c, p, out=p), right)


@pytest.mark.parametrize("hd,units", [(128, [1, 14, 15, 16, 18, 32, 33, 34, 37, 73, 74, 75, 147, 148, 149]), (64, [32, 33, 34, 37, 70, 71, 72, 74, 148, 149, 295, 296, 297])])
def test_as_many_units_as_the_card_just_holds(hd, units):
    """clusters of 8, 4 and 2 blocks a unit, up to and beyond what stands on the card at once"""
    for n in units:
        c = Case([(37 * i) % 90 for i in range(n)], [1 + i % 2 for i in range(n)], kv=1, hd=hd, page=16, dtype=BF16, seed=n)
        c.fill()
        q = (1.5 * c.randn(c.rows, 4, hd)).to(BF16)
        out = attend(c, q).double().cpu().numpy()
        want, room = bounds.attention(q.double().cpu().numpy(), c.seen(), c.held_l, c.first_l, 0, 0, hd ** -0.5, True, False)
        assert (np.abs(out - want) <= room).all(), n


def test_a_view_of_a_wide_table_is_a_narrow_one():
    c = Case([333, 90, 12], [1, 1, 1], kv=8, hd=128, page=16, dtype=BF16)
    c.fill()
    q = c.randn(3, 32, 128).to(BF16)
    narrow = attend(c, q)
    width = len(c.table_l[0])
    c.widened()
    out = serve.kv16_attention(q, c.pool[0], c.table[:, :width], c.held, c.first, c.slots, max_rows=1)
    assert torch.equal(out, narrow)
