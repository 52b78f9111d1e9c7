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

import ctypes as C
from typing import Optional, Tuple

import torch

from . import _lib
from ._lib import Kv4, Pages, check

_TYPE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def kv4_pool(n_pages: int, page_tokens: int, n_head_kv: int, head_dim: int, n_layer: int = 1, device="cuda") -> torch.Tensor:
    """an empty pool: uint8 [n_layer, n_pages, n_head_kv, page_tokens / 16, 18 * head_dim], 4.5 bits a number"""
    if page_tokens % 16 or head_dim not in (64, 128):
        raise ValueError("kv4_pool: page_tokens is a power of two from 16 to 1024, head_dim 64 or 128")
    return torch.zeros(n_layer, n_pages, n_head_kv, page_tokens // 16, 18 * head_dim, dtype=torch.uint8, device=device)


def _need(ok, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _ints(name: str, t: torch.Tensor, device, dims: int, n: Optional[int] = None) -> int:
    if t.dtype != torch.int32 or t.device != device or t.dim() != dims or (dims == 1 and not t.is_contiguous()) or (n is not None and t.shape[0] != n):
        raise ValueError(f"{name} is a contiguous int32 tensor of {dims} dimension(s)" + (f" and {n} entries" if n is not None else "") + f" on {device}")
    return t.data_ptr()


def _table(table: torch.Tensor, device) -> int:
    p = _ints("table", table, device, 2)
    _need(table.stride(1) == 1 or table.shape[1] == 1, "table's rows are contiguous")
    return p


def _on(device):
    _need(device.type == "cuda", "tensors are on a CUDA device: booster_b200 has no CPU fallback")
    return device.index, torch.cuda.current_stream(device).cuda_stream


def _page_stride(pool: torch.Tensor) -> int:
    _, kv, tiles, size = pool.shape[-4:]
    st = pool.stride()
    _need(pool.dtype == torch.uint8 and size % 18 == 0, "pool is a uint8 tensor [..., n_pages, n_head_kv, page_tokens / 16, 18 * head_dim]")
    _need(st[-1] == 1 and (tiles == 1 or st[-2] == size) and (kv == 1 or st[-3] == tiles * size), "pool's pages are contiguous")
    return st[-4] if pool.shape[-4] > 1 else max(st[-4], kv * tiles * size)


def _step(pool, table, held, first, slots, n_rows: int) -> Kv4:
    device = pool.device
    index, stream = _on(device)
    _need(pool.dim() == 4, "pool is one layer's [n_pages, n_head_kv, page_tokens / 16, 18 * head_dim]")
    stride = _page_stride(pool)
    pages, kv, tiles, size = pool.shape
    n_seq = first.shape[0] - 1
    _need(n_seq >= 0, "first has one entry more than there are sequences")
    n_slots = table.shape[0]
    return Kv4(index, pages, 16 * tiles, kv, size // 18, n_slots, table.shape[1], n_seq, n_rows, stream, pool.data_ptr(), stride, table.stride(0) if n_slots > 1 else table.shape[1],
               _table(table, device), _ints("held", held, device, 1, n_slots), _ints("slots", slots, device, 1, n_seq) if slots is not None else _first_n(n_seq, n_slots),
               _ints("first", first, device, 1))


def _first_n(n_seq: int, n_slots: int) -> None:
    _need(n_seq <= n_slots, "without slots, sequence i is slot i: more sequences than slots")


def _rows(name: str, x: torch.Tensor, pool, heads: Optional[int]) -> None:
    if x.dim() != 3 or x.device != pool.device or x.shape[2] * 18 != pool.shape[3] or (heads is not None and x.shape[1] != heads):
        raise ValueError(f"{name} is a tensor [rows, heads, head_dim] that fits the pool, on its device")
    if x.stride(2) != 1:
        raise ValueError(f"{name}: the entries of a head are contiguous")


def kv4_append(pool: torch.Tensor, table: torch.Tensor, held: torch.Tensor, first: torch.Tensor, k: torch.Tensor, v: torch.Tensor, slots: Optional[torch.Tensor] = None) -> None:
    """keys and values [rows, n_head_kv, head_dim] (any strides over rows and heads; float32, bfloat16 or float16) of the step's rows into one layer's pool"""
    _rows("k", k, pool, pool.shape[1])
    _rows("v", v, pool, pool.shape[1])
    _need(k.dtype == v.dtype and k.dtype in _TYPE and k.shape == v.shape, "k and v are float32, bfloat16 or float16, and alike")
    c = _step(pool, table, held, first, slots, k.shape[0])
    check(_lib.lib().b200_kv4_append(C.byref(c), _TYPE[k.dtype], k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1)), "kv4_append")


def kv4_read(pool: torch.Tensor, table: torch.Tensor, held: torch.Tensor, first: torch.Tensor, rows: int, dtype: torch.dtype = torch.bfloat16, slots: Optional[torch.Tensor] = None,
             out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """the rows at positions held, held + 1, ... of each sequence, as kv4_append wrote them: k, v [rows, n_head_kv, head_dim]. Rows of no sequence are left as they are (in `out`)"""
    _need(dtype in _TYPE, "dtype is float32, bfloat16 or float16")
    c = _step(pool, table, held, first, slots, rows)
    shape = (rows, pool.shape[1], pool.shape[3] // 18)
    k, v = out if out is not None else (torch.empty(shape, dtype=dtype, device=pool.device), torch.empty(shape, dtype=dtype, device=pool.device))
    for x in (k, v):
        _need(x.shape == shape and x.dtype == dtype and x.device == pool.device and x.is_contiguous(), "out is a pair of contiguous tensors [rows, n_head_kv, head_dim] of dtype")
    check(_lib.lib().b200_kv4_read(C.byref(c), _TYPE[dtype], k.data_ptr(), v.data_ptr()), "kv4_read")
    return k, v


def kv4_attention(q: torch.Tensor, pool: torch.Tensor, table: torch.Tensor, held: torch.Tensor, first: torch.Tensor, slots: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                  window: int = 0, max_rows: Optional[int] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """attention of the step's rows q [rows, n_head, head_dim] (bfloat16 or float16, any strides over rows and heads) over the positions up to their own, kv4_append having put those into
    the pool; window > 0: over the last `window` of them. scale: 1 / sqrt(head_dim). max_rows: the largest number of rows of a sequence, if the program knows it (else: rows).
    Rows of no sequence are left as they are (in `out`)"""
    _rows("q", q, pool, None)
    _need(q.dtype in (torch.bfloat16, torch.float16), "q is bfloat16 or float16")
    rows, heads, hd = q.shape
    c = _step(pool, table, held, first, slots, rows)
    if out is None:
        out = torch.empty((rows, heads, hd), dtype=q.dtype, device=q.device)
    _need(out.shape == q.shape and out.dtype == q.dtype and out.device == q.device and out.is_contiguous(), "out is a contiguous tensor like q")
    most = max(1, rows if max_rows is None else max_rows)
    L = _lib.lib()
    size = L.b200_kv4_attention_workspace(C.byref(c), heads, most)
    check(size < 0, "kv4_attention")
    work = torch.empty(size, dtype=torch.uint8, device=q.device)
    check(L.b200_kv4_attention(C.byref(c), _TYPE[q.dtype], q.data_ptr(), q.stride(0), q.stride(1), heads, hd ** -0.5 if scale is None else scale, window, most, out.data_ptr(), work.data_ptr(), size),
          "kv4_attention")
    return out


def _pages(table, held, refs, page_tokens: int, pool=None) -> Pages:
    device = refs.device
    index, stream = _on(device)
    n_slots, most = table.shape
    p = Pages(index, refs.shape[0], page_tokens, 1, 64, n_slots, most, 1, stream, None, 0, 0, table.stride(0) if n_slots > 1 else most, _table(table, device),
              _ints("held", held, device, 1, n_slots) if held is not None else table.data_ptr(), _ints("refs", refs, device, 1))
    if pool is not None:
        _need(pool.dim() == 5 and pool.device == device and pool.shape[1] == refs.shape[0], "pool is [n_layer, n_pages, n_head_kv, page_tokens / 16, 18 * head_dim], refs has an entry a page")
        p.page_stride = _page_stride(pool)
        p.pool, p.n_layer, p.layer_stride, p.n_head_kv, p.head_dim = pool.data_ptr(), pool.shape[0], pool.stride(0), pool.shape[2], pool.shape[4] // 18
    return p


def _work(p: Pages, n: int, device) -> torch.Tensor:
    size = _lib.lib().b200_pages_workspace(C.byref(p), n)
    check(size < 0, "pages_workspace")
    return torch.empty(size, dtype=torch.uint8, device=device)


def pages_reserve(table: torch.Tensor, held: torch.Tensor, refs: torch.Tensor, first: torch.Tensor, page_tokens: int, slots: Optional[torch.Tensor] = None) -> torch.Tensor:
    """pages for first[i + 1] - first[i] tokens more of each sequence, the lowest free ones, in order. Returns the status on the device, int32 [1]: 0, the number of pages that were
    missing, or -1 where slots or tables cannot be; then nothing has changed"""
    n = first.shape[0] - 1
    _need(n >= 0, "first has one entry more than there are sequences")
    p = _pages(table, held, refs, page_tokens)
    status = torch.empty(1, dtype=torch.int32, device=refs.device)
    s = _ints("slots", slots, refs.device, 1, n) if slots is not None else _first_n(n, table.shape[0])
    check(_lib.lib().b200_pages_reserve(C.byref(p), s, _ints("first", first, refs.device, 1), n, status.data_ptr()), "pages_reserve")
    return status


def pages_fork(pool: torch.Tensor, table: torch.Tensor, held: torch.Tensor, refs: torch.Tensor, parents: torch.Tensor, children: torch.Tensor) -> torch.Tensor:
    """slot children[i], which is empty, becomes what slot parents[i] is: full pages are shared, a last page that is part full is copied in every layer. Returns the status, see pages_reserve"""
    n = parents.shape[0]
    p = _pages(table, held, refs, 16 * pool.shape[-2], pool)
    work, status = _work(p, n, refs.device), torch.empty(1, dtype=torch.int32, device=refs.device)
    check(_lib.lib().b200_pages_fork(C.byref(p), _ints("parents", parents, refs.device, 1), _ints("children", children, refs.device, 1, n), n, status.data_ptr(), work.data_ptr(), work.numel()),
          "pages_fork")
    return status


def pages_free(table: torch.Tensor, held: torch.Tensor, refs: torch.Tensor, slots: torch.Tensor) -> None:
    """the slots give their pages back and are empty"""
    p = _pages(table, held, refs, 16)
    check(_lib.lib().b200_pages_free(C.byref(p), _ints("slots", slots, refs.device, 1), slots.shape[0]), "pages_free")


def pages_compact(pool: torch.Tensor, table: torch.Tensor, refs: torch.Tensor) -> torch.Tensor:
    """pages in use move to the lowest places and tables follow. Returns how many there are, int32 [1] on the device: no page from that one on is in use"""
    p = _pages(table, None, refs, 16 * pool.shape[-2], pool)
    work, live = _work(p, refs.shape[0], refs.device), torch.empty(1, dtype=torch.int32, device=refs.device)
    check(_lib.lib().b200_pages_compact(C.byref(p), live.data_ptr(), work.data_ptr(), work.numel()), "pages_compact")
    return live


def pages_copy(pool: torch.Tensor, table: torch.Tensor, refs: torch.Tensor, src: torch.Tensor, dst: torch.Tensor) -> torch.Tensor:
    """page dst[i] becomes page src[i] in every layer. Returns the status: -1, and nothing copied, where a page is written twice, or written and read, or does not exist"""
    n = src.shape[0]
    p = _pages(table, None, refs, 16 * pool.shape[-2], pool)
    work, status = _work(p, n, refs.device), torch.empty(1, dtype=torch.int32, device=refs.device)
    check(_lib.lib().b200_pages_copy(C.byref(p), _ints("src", src, refs.device, 1), _ints("dst", dst, refs.device, 1, n), n, status.data_ptr(), work.data_ptr(), work.numel()), "pages_copy")
    return status


def sample(logits: torch.Tensor, u: torch.Tensor, temperature: Optional[torch.Tensor] = None, top_k: Optional[torch.Tensor] = None, top_p: Optional[torch.Tensor] = None,
           min_p: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """one token a row of logits [rows, n_vocab] by the row's random number u (0 <= u < 1), temperature, top_k, top_p and min_p (tensors of an entry a row; None: 1, all, 1, 0), the filters in
    that order of b200_sample. Returns ids, int32 [rows], and the log of each drawn token's share of what the filters kept, float32 [rows]"""
    device = logits.device
    index, stream = _on(device)
    _need(logits.dim() == 2 and logits.dtype in _TYPE and (logits.stride(1) == 1 or logits.shape[1] == 1), "logits is a float32, bfloat16 or float16 tensor [rows, n_vocab] of contiguous rows")
    rows, vocab = logits.shape
    given = []
    for name, t, dtype in (("u", u, torch.float32), ("temperature", temperature, torch.float32), ("top_k", top_k, torch.int32), ("top_p", top_p, torch.float32), ("min_p", min_p, torch.float32)):
        if t is not None and (t.dtype != dtype or t.shape != (rows,) or t.device != device or not t.is_contiguous()):
            raise ValueError(f"{name} is a contiguous {dtype} tensor of {rows} entries on {device}")
        given.append(t.data_ptr() if t is not None else None)
    ids, logprobs = torch.empty(rows, dtype=torch.int32, device=device), torch.empty(rows, dtype=torch.float32, device=device)
    check(_lib.lib().b200_sample(index, stream, _TYPE[logits.dtype], logits.data_ptr(), logits.stride(0) if rows > 1 else vocab, rows, vocab, *given, ids.data_ptr(), logprobs.data_ptr()), "sample")
    return ids, logprobs
