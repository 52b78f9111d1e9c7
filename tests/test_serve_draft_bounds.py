"""The bounds of tests/serve_draft_bounds.py, on the CPU: a result that is rounded once is within them, one whose weights are rounded to the type, or a mask that is off by one, is not."""
import numpy as np
import pytest
import torch

from tests import serve_draft_bounds as bounds


def rounded(x, dtype):
    return torch.from_numpy(np.asarray(x, np.float64)).to(dtype).double().numpy()


def made(rng, dtype, n, hd, much=1.5):
    spread = np.exp(0.5 * rng.standard_normal(hd))
    return (rounded(much * rng.standard_normal(hd), dtype), *(rounded(rng.standard_normal((n, hd)) * spread, dtype) for _ in range(2)))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n", [40, 200])
def test_weights_in_one_number_pass_the_bound_of_two(dtype, hd, n):
    rng, bf16 = np.random.default_rng(n + hd), dtype == torch.bfloat16
    within = beyond = 0.0
    for _ in range(40):
        q, k, v = made(rng, dtype, n, hd)
        p, r, room = bounds.row(q, k, v, hd ** -0.5, bf16, False)
        w = p / p.max() * 128.0
        hi = rounded(w, dtype)
        two = hi + rounded(w - hi, dtype)
        within = max(within, (np.abs(rounded(two @ v / w.sum(), dtype) - r) / room).max())
        once = np.abs(rounded(hi @ v / w.sum(), dtype) - r)
        beyond = max(beyond, (once / room).max())
        assert (once <= bounds.row(q, k, v, hd ** -0.5, bf16, True)[2]).all()
    assert within <= 1.0 < 2.0 < beyond


@pytest.mark.parametrize("rows,window,sinks", [(1900, 1500, 4), (900, 70, 33), (300, 0, 0), (40, 1, 0)])
def test_counts_tell_a_mask_that_is_off_by_one(rows, window, sinks):
    """keys of 0 and values that are 1 at one dim each: results count what is seen, whatever is rounded (a window of a multiple of the dims would count the same one position further on)"""
    there, hd = np.ones(rows, bool), 64
    p = rows - 2

    def result(j):
        return rounded(np.bincount(j % hd, minlength=hd) / j.size, torch.bfloat16)

    def counted(out, j):
        return np.array_equal(np.rint(out * j.size), np.bincount(j % hd, minlength=hd))

    j = bounds.seen(p, there, window, sinks)
    assert counted(result(j), j)
    others = [bounds.seen(p + 1, there, window, sinks)]
    if window:
        others += [bounds.seen(p, there, window + 1, sinks), bounds.seen(p, there, window, sinks + 1)]
        others += [bounds.seen(p, there, window - 1, sinks)] if window > 1 else []
        others += [bounds.seen(p, there, window, sinks - 1)] if sinks else []
    for other in others:
        assert not counted(result(other), j)
