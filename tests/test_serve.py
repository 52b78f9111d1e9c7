"""What booster_b200.serve and its C entry points refuse, without a GPU: every check of arguments comes before the device is touched."""
import ctypes as C
import re

import pytest
import torch

from booster_b200 import _lib, serve

FAKE = 1 << 20                                                        # a pointer that nothing reads: all calls here end in a check


def kv4(**changes):
    d = dict(device=0, n_pages=4, page_tokens=16, n_head_kv=2, head_dim=64, n_slots=2, max_pages=3, n_seq=2, n_rows=2, stream=None, pool=FAKE, page_stride=2 * 18 * 64, table_stride=3,
             table=FAKE, held=FAKE, slots=None, first=FAKE)
    d.update(changes)
    return _lib.Kv4(**d)


def pages(**changes):
    d = dict(device=0, n_pages=4, page_tokens=16, n_head_kv=2, head_dim=64, n_slots=2, max_pages=3, n_layer=2, stream=None, pool=FAKE, layer_stride=4 * 2 * 18 * 64, page_stride=2 * 18 * 64,
             table_stride=3, table=FAKE, held=FAKE, refs=FAKE)
    d.update(changes)
    return _lib.Pages(**d)


def refused(rc, text):
    message = _lib.last_error()
    assert rc not in (0, None) and re.search(text, message), (rc, message)


L = _lib.lib()
CACHE = [(dict(head_dim=96), "head_dim"), (dict(head_dim=0), "head_dim"), (dict(page_tokens=24), "page_tokens"), (dict(page_tokens=8), "page_tokens"), (dict(page_tokens=2048), "page_tokens"),
         (dict(n_head_kv=0), "n_head_kv"), (dict(n_pages=0), "pool of one page"), (dict(n_slots=0), "one slot"), (dict(max_pages=0), "one page"), (dict(max_pages=1 << 27), "2\\^30"),
         (dict(n_seq=-1), "sequences"), (dict(n_seq=5000), "sequences"), (dict(n_rows=-1), "rows"), (dict(page_stride=18 * 64), "page_stride"), (dict(page_stride=2 * 18 * 64 + 8), "page_stride"),
         (dict(table_stride=2), "table_stride"), (dict(pool=None), "null"), (dict(table=None), "null"), (dict(held=None), "null"), (dict(first=None), "null"), (dict(pool=FAKE + 8), "16 bytes"),
         (dict(held=FAKE + 2), "4 bytes")]


@pytest.mark.parametrize("changes,text", CACHE)
def test_descriptions_of_a_cache(changes, text):
    c = kv4(**changes)
    refused(L.b200_kv4_append(C.byref(c), 2, FAKE, 128, 64, FAKE, 128, 64), text)
    refused(L.b200_kv4_read(C.byref(c), 2, FAKE, FAKE), text)
    refused(L.b200_kv4_attention(C.byref(c), 2, FAKE, 256, 64, 4, 1.0, 0, 1, FAKE, FAKE, 1 << 40), text)
    assert L.b200_kv4_attention_workspace(C.byref(c), 4, 1) == -1 and re.search(text, _lib.last_error())


def test_arguments_of_the_cache_calls():
    c = kv4()
    refused(L.b200_kv4_append(None, 2, FAKE, 128, 64, FAKE, 128, 64), "null")
    refused(L.b200_kv4_append(C.byref(c), 3, FAKE, 128, 64, FAKE, 128, 64), "dtype")
    refused(L.b200_kv4_append(C.byref(c), 2, None, 128, 64, FAKE, 128, 64), "pointers")
    refused(L.b200_kv4_append(C.byref(c), 0, FAKE + 2, 128, 64, FAKE, 128, 64), "whole entries")
    refused(L.b200_kv4_read(C.byref(c), 2, FAKE + 8, FAKE), "16 bytes")
    for args, text in (((0, FAKE, 256, 64, 4, 1.0, 0, 1, FAKE, FAKE, 1 << 40), "dtype"), ((2, FAKE, 256, 64, 3, 1.0, 0, 1, FAKE, FAKE, 1 << 40), "multiple of n_head_kv"),
                       ((2, FAKE, 256, 64, 0, 1.0, 0, 1, FAKE, FAKE, 1 << 40), "multiple of n_head_kv"), ((2, FAKE, 256, 64, 4, float("nan"), 0, 1, FAKE, FAKE, 1 << 40), "scale"),
                       ((2, FAKE, 256, 64, 4, 1.0, -1, 1, FAKE, FAKE, 1 << 40), "window"), ((2, FAKE, 256, 64, 4, 1.0, 0, 0, FAKE, FAKE, 1 << 40), "max_rows"),
                       ((2, None, 256, 64, 4, 1.0, 0, 1, FAKE, FAKE, 1 << 40), "q points"), ((2, FAKE, 256, 64, 4, 1.0, 0, 1, FAKE + 4, FAKE, 1 << 40), "out starts")):
        refused(L.b200_kv4_attention(C.byref(c), *args), text)


@pytest.mark.parametrize("changes,text", [(dict(page_tokens=40), "page_tokens"), (dict(n_pages=0), "2\\^20 pages"), (dict(n_pages=(1 << 20) + 1), "2\\^20 pages"), (dict(n_slots=0), "slots"),
                                          (dict(n_slots=1 << 19), "slots"), (dict(max_pages=0), "one page"), (dict(table_stride=1), "table_stride"), (dict(table=None), "null"), (dict(refs=None), "null"),
                                          (dict(refs=FAKE + 1), "4 bytes")])
def test_descriptions_of_pages(changes, text):
    p = pages(**changes)
    refused(L.b200_pages_reserve(C.byref(p), FAKE, FAKE, 1, FAKE), text)
    refused(L.b200_pages_fork(C.byref(p), FAKE, FAKE, 1, FAKE, FAKE, 1 << 40), text)
    refused(L.b200_pages_free(C.byref(p), FAKE, 1), text)
    refused(L.b200_pages_compact(C.byref(p), FAKE, FAKE, 1 << 40), text)
    refused(L.b200_pages_copy(C.byref(p), FAKE, FAKE, 1, FAKE, FAKE, 1 << 40), text)


@pytest.mark.parametrize("changes,text", [(dict(head_dim=32), "head_dim"), (dict(n_layer=0), "n_layer"), (dict(pool=None), "16 bytes"), (dict(page_stride=16), "strides"), (dict(layer_stride=24), "strides")])
def test_descriptions_of_a_pool(changes, text):
    p = pages(**changes)
    refused(L.b200_pages_fork(C.byref(p), FAKE, FAKE, 1, FAKE, FAKE, 1 << 40), text)
    refused(L.b200_pages_compact(C.byref(p), FAKE, FAKE, 1 << 40), text)
    refused(L.b200_pages_copy(C.byref(p), FAKE, FAKE, 1, FAKE, FAKE, 1 << 40), text)


def test_arguments_of_the_page_calls():
    p = pages()
    refused(L.b200_pages_reserve(C.byref(p), None, FAKE, 3, FAKE), "more sequences than slots")
    refused(L.b200_pages_reserve(C.byref(p), FAKE, None, 1, FAKE), "null")
    refused(L.b200_pages_reserve(C.byref(p), FAKE, FAKE, -1, FAKE), "sequences")
    refused(L.b200_pages_fork(C.byref(p), FAKE, None, 1, FAKE, FAKE, 1 << 40), "null")
    refused(L.b200_pages_fork(C.byref(p), FAKE, FAKE, 1, FAKE, FAKE, 4), "workspace has 4 bytes")
    refused(L.b200_pages_fork(C.byref(p), FAKE, FAKE, 1, FAKE, FAKE + 4, 1 << 40), "16 bytes")
    refused(L.b200_pages_free(C.byref(p), None, 1), "null")
    refused(L.b200_pages_compact(C.byref(p), None, FAKE, 1 << 40), "null")
    refused(L.b200_pages_copy(C.byref(p), FAKE, FAKE, 5, FAKE, FAKE, 1 << 40), "pairs")
    assert L.b200_pages_workspace(C.byref(p), -1) == -1 and L.b200_pages_workspace(C.byref(p), 4) > 0


def test_arguments_of_the_draw():
    good = [0, None, 0, FAKE, 100, 2, 100, FAKE, None, None, None, None, FAKE, None]
    for at, value, text in ((2, 5, "dtype"), (6, 0, "logits a row"), (6, 1 << 19, "logits a row"), (5, -1, "rows"), (4, 99, "row_stride"), (3, None, "null"), (7, None, "null"), (12, None, "null")):
        refused(L.b200_sample(*[value if i == at else x for i, x in enumerate(good)]), text)


@pytest.mark.skipif(torch.cuda.is_available(), reason="only meaningful without a CUDA device")
def test_no_cpu_fallback():
    c, p = kv4(), pages()
    refused(L.b200_kv4_append(C.byref(c), 2, FAKE, 128, 64, FAKE, 128, 64), "no CUDA device")
    refused(L.b200_pages_free(C.byref(p), FAKE, 1), "no CUDA device")
    refused(L.b200_sample(0, None, 0, FAKE, 100, 2, 100, FAKE, None, None, None, None, FAKE, None), "no CUDA device")
    with pytest.raises(ValueError, match="CUDA device"):
        serve.sample(torch.zeros(1, 5), torch.zeros(1))


def test_tensors_that_do_not_fit():
    pool = serve.kv4_pool(4, 16, 2, 64, device="cpu")
    table, ints = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    k = torch.zeros(2, 2, 64, dtype=torch.half)
    for bad in (k[:, :1], k[:, :, :32], k[0], k.transpose(1, 2), k.double(), torch.zeros(2, 2, 128, dtype=torch.half)[:, :, ::2]):
        with pytest.raises(ValueError):
            serve.kv4_append(pool[0], table, ints, torch.zeros(3, dtype=torch.int32), bad, bad)
    with pytest.raises(ValueError):
        serve.kv4_attention(k.float(), pool[0], table, ints, torch.zeros(3, dtype=torch.int32))
    with pytest.raises(ValueError):
        serve.kv4_pool(4, 20, 2, 64, device="cpu")
    with pytest.raises(ValueError):
        serve.kv4_pool(4, 16, 2, 80, device="cpu")


def test_what_is_no_tensor_is_refused():
    pool = serve.kv4_pool(4, 16, 2, 64, device="cpu")
    x, k = torch.zeros(3, dtype=torch.int32), torch.zeros(2, 2, 64, dtype=torch.half)
    with pytest.raises(ValueError, match="pool is a tensor"):
        serve.kv4_append(None, x, x, x, k, k)
    with pytest.raises(ValueError, match="q is a tensor"):
        serve.kv4_attention([1.0], pool[0], x, x, x)
    with pytest.raises(ValueError, match="dtype"):
        serve.kv4_read(pool[0], x, x, x, 2, "bfloat16")
    with pytest.raises(ValueError, match="whole number"):
        serve.kv4_read(pool[0], x, x, x, 1 << 40)
    with pytest.raises(ValueError, match="refs is a tensor"):
        serve.pages_free(x, x, 3, x)
    with pytest.raises(ValueError, match="logits is a tensor"):
        serve.sample(7, x)
    with pytest.raises(TypeError):
        serve.sample(k[0], x, x, x, x, x, x)


def test_the_module_calls_the_library_that_is_loaded():
    """its functions come by address: without them it refuses, and it is the library's own class that its errors have"""
    module = serve._native()
    for bad in ((), (_lib.B200Error, 1), (_lib.B200Error,) + (0,) * 12):
        with pytest.raises((TypeError, ValueError)):
            module.bind(*bad)
    assert serve._native() is module
