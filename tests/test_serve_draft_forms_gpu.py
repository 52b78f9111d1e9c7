"""Attention over the 16-bit cache on the GPU, each of its forms by itself (tests/serve_draft_bounds.py): values up to the ends of the type's range."""
import pytest
import torch

from booster_b200 import serve
from tests import serve_draft_bounds as bounds
from tests.test_serve_draft_gpu import BF16, Case

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
