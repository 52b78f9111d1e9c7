"""What the operators around drafted tokens and the 16-bit cache refuse, without a GPU: every check of arguments comes before the device is touched."""
import ctypes as C

import pytest
import torch

from booster_b200 import _lib, serve
from tests.test_serve import CACHE, FAKE, kv4, pages, refused

L = _lib.lib()


def kv16(**changes):
    return kv4(**{"page_stride": 2 * 2 * 16 * 64 * 2, **changes})


@pytest.mark.parametrize("changes,text", [c for c in CACHE if "page_stride" not in c[0]] + [(dict(page_stride=2 * 2 * 16 * 64 * 2 - 16), "page_stride"), (dict(page_stride=2 * 2 * 16 * 64 * 2 + 8), "page_stride")])
def test_descriptions_of_a_16_bit_cache(changes, text):
    c = kv16(**changes)
    refused(L.b200_kv16_append(C.byref(c), 1, 2, FAKE, 128, 64, FAKE, 128, 64), text)
    refused(L.b200_kv16_attention(C.byref(c), 2, FAKE, 256, 64, 4, 1.0, 0, 0, 1, FAKE, FAKE, 1 << 40), text)
    refused(L.b200_kv16_attention_workspace(C.byref(c), 4, 1), text)


def test_arguments_of_the_16_bit_cache_calls():
    c = kv16()
    refused(L.b200_kv16_append(None, 1, 2, FAKE, 128, 64, FAKE, 128, 64), "null")
    for args, text in (((0, 2, FAKE, 128, 64, FAKE, 128, 64), "dtype"), ((1, 3, FAKE, 128, 64, FAKE, 128, 64), "dtype"), ((1, 2, None, 128, 64, FAKE, 128, 64), "pointers"),
                       ((1, 0, FAKE + 2, 128, 64, FAKE, 128, 64), "whole entries")):
        refused(L.b200_kv16_append(C.byref(c), *args), text)
    good = [2, FAKE, 256, 64, 4, 1.0, 0, 0, 1, FAKE, FAKE, 1 << 40]
    for at, value, text in ((0, 0, "dtype"), (1, None, "q points"), (1, FAKE + 1, "q points"), (4, 3, "multiple of n_head_kv"), (4, 0, "multiple of n_head_kv"), (5, float("inf"), "scale"), (6, -1, "window"),
                            (7, -1, "sinks"), (8, 0, "max_rows"), (9, FAKE + 8, "out starts")):
        refused(L.b200_kv16_attention(C.byref(c), *[value if i == at else x for i, x in enumerate(good)]), text)


@pytest.mark.parametrize("changes,text", [(dict(page_tokens=40), "page_tokens"), (dict(n_pages=0), "2\\^20 pages"), (dict(n_slots=0), "slots"), (dict(max_pages=0), "one page"),
                                          (dict(table_stride=1), "table_stride"), (dict(table=None), "null"), (dict(held=None), "null"), (dict(refs=FAKE + 1), "4 bytes")])
def test_descriptions_of_pages_for_a_step(changes, text):
    p = pages(**changes)
    refused(L.b200_pages_plan(C.byref(p), FAKE, FAKE, 1, 4, FAKE, FAKE, FAKE, FAKE), text)
    refused(L.b200_pages_trim(C.byref(p), FAKE, 1, 0, 0), text)


def test_arguments_of_a_step_s_tables():
    p = pages()
    good = [FAKE, FAKE, 1, 4, FAKE, FAKE, FAKE, FAKE]
    for at, value, text in ((1, None, "null"), (2, -1, "sequences"), (2, 4097, "sequences"), (3, -1, "rows"), (3, (1 << 24) + 1, "rows"), (4, None, "null"), (5, None, "null"), (6, None, "null"), (7, None, "null")):
        refused(L.b200_pages_plan(C.byref(p), *[value if i == at else x for i, x in enumerate(good)]), text)
    refused(L.b200_pages_plan(C.byref(p), None, FAKE, 3, 4, FAKE, FAKE, FAKE, FAKE), "more sequences than slots")
    for args, text in (((None, 1, 0, 0), "null"), ((FAKE, -1, 0, 0), "slots"), ((FAKE, 1, -1, 0), "window"), ((FAKE, 1, 5, -2), "sinks")):
        refused(L.b200_pages_trim(C.byref(p), *args), text)


@pytest.mark.parametrize("changes,text", [(dict(head_dim=32 + 0x10000), "head_dim"), (dict(head_dim=64 + 0x20000), "head_dim"), (dict(page_stride=2 * 18 * 64, head_dim=64 + 0x10000), "strides")])
def test_descriptions_of_a_16_bit_pool(changes, text):
    p = pages(**changes)
    refused(L.b200_pages_fork(C.byref(p), FAKE, FAKE, 1, FAKE, FAKE, 1 << 40), text)
    refused(L.b200_pages_compact(C.byref(p), FAKE, FAKE, 1 << 40), text)
    refused(L.b200_pages_copy(C.byref(p), FAKE, FAKE, 1, FAKE, FAKE, 1 << 40), text)


def test_arguments_of_the_verification():
    good = [0, None, 0, FAKE, 100, 2, 100, FAKE, FAKE, 1, FAKE, FAKE, None, None, None, None, FAKE, 100, FAKE, FAKE, FAKE, FAKE, 16]
    assert L.b200_verify_workspace(-1) == -1 and L.b200_verify_workspace((1 << 20) + 1) == -1 and L.b200_verify_workspace(2) == 16
    for at, value, text in ((2, 5, "dtype"), (6, 0, "logits a row"), (6, (1 << 18) + 1, "logits a row"), (5, -1, "rows"), (5, (1 << 20) + 1, "rows"), (4, 99, "row_stride"), (17, 99, "draft_stride"),
                            (3, None, "null"), (3, FAKE + 2, "null"), (7, None, "null"), (8, None, "null"), (9, -1, "sequences"), (9, 4097, "sequences"), (10, None, "null"), (11, None, "null"),
                            (18, None, "null"), (19, None, "null"), (20, None, "null"), (21, None, "workspace"), (21, FAKE + 4, "workspace"), (22, 15, "workspace has 15")):
        refused(L.b200_verify(*[value if i == at else x for i, x in enumerate(good)]), text)


@pytest.mark.skipif(torch.cuda.is_available(), reason="only meaningful without a CUDA device")
def test_no_cpu_fallback_here_either():
    c, p = kv16(), pages()
    refused(L.b200_kv16_append(C.byref(c), 1, 2, FAKE, 128, 64, FAKE, 128, 64), "no CUDA device")
    refused(L.b200_kv16_attention(C.byref(c), 2, FAKE, 256, 64, 4, 1.0, 0, 0, 1, FAKE, FAKE, 1 << 40), "no CUDA device")
    refused(L.b200_pages_plan(C.byref(p), FAKE, FAKE, 1, 4, FAKE, FAKE, FAKE, FAKE), "no CUDA device")
    refused(L.b200_pages_trim(C.byref(p), FAKE, 1, 0, 0), "no CUDA device")
    refused(L.b200_verify(0, None, 0, FAKE, 100, 2, 100, FAKE, FAKE, 1, FAKE, FAKE, None, None, None, None, None, 0, FAKE, FAKE, FAKE, FAKE, 16), "no CUDA device")
    ints = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA device"):
        serve.verify(torch.zeros(2, 5), ints, ints, torch.zeros(2), torch.zeros(2))


def test_16_bit_tensors_that_do_not_fit():
    pool = serve.kv16_pool(4, 16, 2, 64, device="cpu", dtype=torch.half)
    assert pool.shape == (1, 4, 2, 2, 16, 64) and not pool.any()
    table, ints, first = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    k = torch.zeros(2, 2, 64, dtype=torch.half)
    for bad in (k[:, :1], k[:, :, :32], k[0], k.transpose(1, 2), k.double(), torch.zeros(2, 2, 128, dtype=torch.half)[:, :, ::2]):
        with pytest.raises(ValueError):
            serve.kv16_append(pool[0], table, ints, first, bad, bad)
    for q in (k.float(), k.bfloat16(), k[0], k[:, :, :32]):
        with pytest.raises(ValueError):
            serve.kv16_attention(q, pool[0], table, ints, first)
    for wrong in (pool, pool[0, 0], None, serve.kv4_pool(4, 16, 2, 64, device="cpu")[0]):
        with pytest.raises(ValueError):
            serve.kv16_append(wrong, table, ints, first, k, k)
    for bad in (dict(page_tokens=20), dict(head_dim=80), dict(dtype=torch.float32), dict(n_pages=0), dict(n_head_kv=0), dict(n_layer=0)):
        with pytest.raises(ValueError):
            serve.kv16_pool(**{**dict(n_pages=4, page_tokens=16, n_head_kv=2, head_dim=64, device="cpu"), **bad})
    with pytest.raises(ValueError, match="counts is a tensor"):
        serve.pages_plan(table, ints, ints, [1, 1], 16, 2)
    with pytest.raises(ValueError, match="whole number"):
        serve.pages_plan(table, ints, ints, ints, 16, "2")
    with pytest.raises(ValueError, match="logits"):
        serve.verify(torch.zeros(2, 5, dtype=torch.int32), ints, ints, ints, ints)
