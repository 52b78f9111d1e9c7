"""Device-level operators of a server that runs many sequences at once (include/booster_b200.h, b200_kv4_* / b200_pages_* / b200_sample), on torch tensors.

A layer's keys and values lie in 4 bits in pages of a pool; sequences hold pages through a table and may share them. A step of the server:

    status = pages_reserve(table, held, refs, first, page_tokens, slots)          # room for the step's rows
    for layer in ...:
        kv4_append(pool[layer], table, held, first, k, v, slots)                  # their keys and values
        out = kv4_attention(q, pool[layer], table, held, first, slots)            # what they see
    ids, logprobs = sample(logits, u, temperature, top_k, top_p, min_p)
    held[slots] += first.diff()                                                   # the step is over

and between steps pages_fork (several answers to one prompt), pages_free, pages_compact, pages_copy. Sequence i of a step is slot slots[i] (None: slot i) of
table [n_slots, max_pages] and held [n_slots], and has the rows first[i] .. first[i + 1] - 1 of the step's tensors. All calls enqueue on the tensors' device and
torch's current stream of it, wait for nothing and can be captured into a CUDA graph. Arguments that the host can see are checked (ValueError, B200Error); pages and
slots that a table names but that do not exist count as absent.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch

from . import _lib

_module = None


def _native():
    """booster_b200/csrc/serve_torch.cpp, which looks the tensors over and calls the library"""
    global _module
    if _module is None:
        try:
            from . import _serve
        except ImportError as e:
            raise ImportError("booster_b200/_serve.so is not built for this torch (run `make`): there is no other path") from e
        L = _lib.lib()
        _serve.bind(_lib.B200Error, *(ctypes.cast(getattr(L, "b200_" + name), ctypes.c_void_p).value for name in (
            "last_error", "kv4_append", "kv4_read", "kv4_attention_workspace", "kv4_attention", "pages_workspace", "pages_reserve", "pages_fork", "pages_free", "pages_compact", "pages_copy",
            "sample")))
        _module = _serve
    return _module


def kv4_pool(n_pages: int, page_tokens: int, n_head_kv: int, head_dim: int, n_layer: int = 1, device="cuda") -> torch.Tensor:
    """an empty pool: uint8 [n_layer, n_pages, n_head_kv, page_tokens / 16, 18 * head_dim], 4.5 bits a number"""
    if page_tokens not in (16, 32, 64, 128, 256, 512, 1024) or head_dim not in (64, 128):
        raise ValueError("kv4_pool: page_tokens is a power of two from 16 to 1024, head_dim 64 or 128")
    return torch.zeros(n_layer, n_pages, n_head_kv, page_tokens // 16, 18 * head_dim, dtype=torch.uint8, device=device)


def kv4_append(pool: torch.Tensor, table: torch.Tensor, held: torch.Tensor, first: torch.Tensor, k: torch.Tensor, v: torch.Tensor, slots: Optional[torch.Tensor] = None) -> None:
    """keys and values [rows, n_head_kv, head_dim] (any strides over rows and heads; float32, bfloat16 or float16) of the step's rows into one layer's pool"""
    _native().kv4_append(pool, table, held, first, k, v, slots)


def kv4_read(pool: torch.Tensor, table: torch.Tensor, held: torch.Tensor, first: torch.Tensor, rows: int, dtype: torch.dtype = torch.bfloat16, slots: Optional[torch.Tensor] = None,
             out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """the rows at positions held, held + 1, ... of each sequence, as kv4_append wrote them: k, v [rows, n_head_kv, head_dim]. Rows of no sequence are left as they are (in `out`)"""
    return _native().kv4_read(pool, table, held, first, rows, dtype, slots, out)


def kv4_attention(q: torch.Tensor, pool: torch.Tensor, table: torch.Tensor, held: torch.Tensor, first: torch.Tensor, slots: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                  window: int = 0, max_rows: Optional[int] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """attention of the step's rows q [rows, n_head, head_dim] (bfloat16 or float16, any strides over rows and heads) over the positions up to their own, kv4_append having put those into
    the pool; window > 0: over the last `window` of them. scale: 1 / sqrt(head_dim). max_rows: the largest number of rows of a sequence, if the program knows it. It chooses
    between kernels, whose results differ by their roundings, and any number is right; without it the mean is taken. Single tokens and a
    long portion are quickest as two calls (48 tokens at 3000 positions and 512 rows at 6000: 133 us, in one 254 to 395; 200 at 500 and 512 rows at 500: 79, in one 109 to 239).
    Rows of no sequence are left as they are (in `out`)"""
    return _native().kv4_attention(q, pool, table, held, first, slots, scale, window, max_rows, out)


def kv4_status(device: Optional[int] = None) -> None:
    """raises B200Error where a bounded wait inside an earlier kv4_attention on the device ran out, so that its results are worthless, and no call has told of it yet. The other calls here look by
    themselves; a program that replays graphs asks, behind a synchronisation"""
    _lib.check(_lib.lib().b200_kv4_status(torch.cuda.current_device() if device is None else device), "kv4_status")


def pages_reserve(table: torch.Tensor, held: torch.Tensor, refs: torch.Tensor, first: torch.Tensor, page_tokens: int, slots: Optional[torch.Tensor] = None) -> torch.Tensor:
    """pages for first[i + 1] - first[i] tokens more of each sequence, the lowest free ones, in order. Returns the status on the device, int32 [1]: 0, the number of pages that were
    missing, or -1 where slots or tables cannot be; then nothing has changed"""
    return _native().pages_reserve(table, held, refs, first, page_tokens, slots)


def pages_fork(pool: torch.Tensor, table: torch.Tensor, held: torch.Tensor, refs: torch.Tensor, parents: torch.Tensor, children: torch.Tensor) -> torch.Tensor:
    """slot children[i], which is empty, becomes what slot parents[i] is: full pages are shared, a last page that is part full is copied in every layer. Returns the status, see pages_reserve"""
    return _native().pages_fork(pool, table, held, refs, parents, children)


def pages_free(table: torch.Tensor, held: torch.Tensor, refs: torch.Tensor, slots: torch.Tensor) -> None:
    """the slots give their pages back and are empty"""
    _native().pages_free(table, held, refs, slots)


def pages_compact(pool: torch.Tensor, table: torch.Tensor, refs: torch.Tensor) -> torch.Tensor:
    """pages in use move to the lowest places and tables follow. Returns how many there are, int32 [1] on the device: no page from that one on is in use"""
    return _native().pages_compact(pool, table, refs)


def pages_copy(pool: torch.Tensor, table: torch.Tensor, refs: torch.Tensor, src: torch.Tensor, dst: torch.Tensor) -> torch.Tensor:
    """page dst[i] becomes page src[i] in every layer. Returns the status: -1, and nothing copied, where a page is written twice, or written and read, or does not exist"""
    return _native().pages_copy(pool, table, refs, src, dst)


def sample(logits: torch.Tensor, u: torch.Tensor, temperature: Optional[torch.Tensor] = None, top_k: Optional[torch.Tensor] = None, top_p: Optional[torch.Tensor] = None,
           min_p: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """one token a row of logits [rows, n_vocab] by the row's random number u (0 <= u < 1), temperature, top_k, top_p and min_p (tensors of an entry a row; None: 1, all, 1, 0), the filters in
    that order of b200_sample. Returns ids, int32 [rows], and the log of each drawn token's share of what the filters kept, float32 [rows]"""
    return _native().sample(logits, u, temperature, top_k, top_p, min_p)
