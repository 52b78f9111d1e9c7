"""b200_verify on the GPU: a draft is taken where accept q < p, whatever makes p."""
import numpy as np
import pytest
import torch

from booster_b200 import serve
from tests import serve_draft_oracle as oracle
from tests.test_serve_draft_gpu import F32, ints

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab", [50, 70000])
@pytest.mark.parametrize("drafter", [False, True])
def test_one_token_that_has_everything(vocab, drafter):
    """p is 1 at the largest logit by a temperature of 0 and by top-k 1: both take and end alike, at accept and q up to their ends and beyond"""
    accepts, shares = [0.0, 0.5, 1.0, 1.5, float("nan")], [1.0, 0.25, 2.0, 0.0, float("nan")] if drafter else [1.0]
    pairs = [(a, s) for a in accepts for s in shares]
    n = len(pairs)
    gen = torch.Generator(device="cuda").manual_seed(vocab)
    logits = torch.randn(2 * n, vocab, generator=gen, device="cuda")
    best = logits.argmax(1).tolist()
    ids = [x for i in range(n) for x in (0, best[2 * i])]               # every draft is the largest
    first = list(range(0, 2 * n + 1, 2))
    u, accept = torch.rand(2 * n, generator=gen, device="cuda"), torch.full((2 * n,), 0.5, device="cuda")
    probs = torch.zeros(2 * n, vocab, device="cuda") if drafter else None
    for i, (a, s) in enumerate(pairs):
        accept[2 * i] = a
        if drafter:
            probs[2 * i, best[2 * i]] = s
    takes = [not np.isnan(a) and a * (s if s > 0 else 0.0) < 1.0 for a, s in pairs]
    for filters in (dict(temperature=0.0), dict(top_k=1)):
        col = {"temperature": torch.full((2 * n,), filters.get("temperature", 1.0), device="cuda"), "top_k": torch.full((2 * n,), filters.get("top_k", 0), dtype=torch.int32, device="cuda")}
        gained, tokens, _ = serve.verify(logits, ints(ids), ints(first), u, accept, draft_probs=probs, **col)
        want = oracle.verify(logits.double().cpu().numpy(), ids, first, u.double().tolist(), accept.double().tolist(), [filters] * (2 * n), None if probs is None else probs.double().cpu().numpy())
        assert want[0] == [2 if t else 1 for t in takes]
        assert gained.tolist() == want[0] and tokens.tolist() == want[1]
