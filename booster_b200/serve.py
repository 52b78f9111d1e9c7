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

import struct
from typing import Dict, Optional, Tuple

import torch

from . import _lib
from ._lib import check

_TYPE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_KV4, _PAGES = struct.Struct("@9i2P2q4P"), struct.Struct("@8i2P3q3P")      # struct b200_kv4, struct b200_pages
_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else lambda index: torch.cuda.current_stream(index).cuda_stream
_I32 = torch.int32


def kv4_pool(n_pages: int, page_tokens: int, n_head_kv: int, head_dim: int, n_layer: int = 1, device="cuda") -> torch.Tensor:
    """an empty pool: uint8 [n_layer, n_pages, n_head_kv, page_tokens / 16, 18 * head_dim], 4.5 bits a number"""
    if page_tokens % 16 or head_dim not in (64, 128):
        raise ValueError("kv4_pool: page_tokens is a power of two from 16 to 1024, head_dim 64 or 128")
    return torch.zeros(n_layer, n_pages, n_head_kv, page_tokens // 16, 18 * head_dim, dtype=torch.uint8, device=device)


def _need(ok, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _ints(name: str, t: torch.Tensor, index: int, n: int = -1) -> int:
    """address of a contiguous int32 vector (of n entries) on device `index`"""
    if t.dtype is not _I32 or t.get_device() != index or t.dim() != 1 or not t.is_contiguous() or (n >= 0 and t.numel() != n):
        raise ValueError(f"{name} is a contiguous int32 tensor of 1 dimension" + (f" and {n} entries" if n >= 0 else "") + " on the device of the others")
    return t.data_ptr()


def _table(t: torch.Tensor, index: int) -> Tuple[int, int, int, int]:
    """address, slots, pages and stride of a slot"""
    if t.dtype is not _I32 or t.get_device() != index or t.dim() != 2 or (t.stride(1) != 1 and t.shape[1] != 1):
        raise ValueError("table is an int32 tensor [n_slots, max_pages] of contiguous rows on the device of the others")
    slots, most = t.shape
    return t.data_ptr(), slots, most, t.stride(0) if slots > 1 else most


def _on(t: torch.Tensor) -> int:
    index = t.get_device()
    _need(index >= 0, "tensors are on a CUDA device: booster_b200 has no CPU fallback")
    return index


def _page_stride(pool: torch.Tensor, shape) -> int:
    kv, tiles, size = shape[-3:]
    st = pool.stride()
    if pool.dtype is not torch.uint8 or size % 18 or st[-1] != 1 or (tiles != 1 and st[-2] != size) or (kv != 1 and st[-3] != tiles * size):
        raise ValueError("pool is a uint8 tensor [..., n_pages, n_head_kv, page_tokens / 16, 18 * head_dim] of contiguous pages")
    return st[-4] if shape[-4] > 1 else max(st[-4], kv * tiles * size)


def _step(pool, table, held, first, slots, n_rows: int) -> bytes:
    """struct b200_kv4 of one layer and a step"""
    index = _on(pool)
    shape = pool.shape
    _need(len(shape) == 4, "pool is one layer's [n_pages, n_head_kv, page_tokens / 16, 18 * head_dim]")
    pages, kv, tiles, size = shape
    n_seq = first.numel() - 1
    _need(n_seq >= 0, "first has one entry more than there are sequences")
    table_at, n_slots, most, stride = _table(table, index)
    if slots is None:
        _need(n_seq <= n_slots, "without slots, sequence i is slot i: more sequences than slots")
        slots_at = 0
    else:
        slots_at = _ints("slots", slots, index, n_seq)
    return _KV4.pack(index, pages, 16 * tiles, kv, size // 18, n_slots, most, n_seq, n_rows, _stream(index), pool.data_ptr(), _page_stride(pool, shape), stride, table_at,
                     _ints("held", held, index, n_slots), slots_at, _ints("first", first, index))


def _rows(name: str, x: torch.Tensor, pool, heads: int = -1) -> Tuple[int, int]:
    """strides of rows and heads"""
    if x.dim() != 3 or x.get_device() != pool.get_device() or x.shape[2] * 18 != pool.shape[-1] or (heads >= 0 and x.shape[1] != heads):
        raise ValueError(f"{name} is a tensor [rows, heads, head_dim] that fits the pool, on its device")
    row, head, one = x.stride()
    if one != 1:
        raise ValueError(f"{name}: the entries of a head are contiguous")
    return row, head


def kv4_append(pool: torch.Tensor, table: torch.Tensor, held: torch.Tensor, first: torch.Tensor, k: torch.Tensor, v: torch.Tensor, slots: Optional[torch.Tensor] = None) -> None:
    """keys and values [rows, n_head_kv, head_dim] (any strides over rows and heads; float32, bfloat16 or float16) of the step's rows into one layer's pool"""
    kv = pool.shape[1] if pool.dim() == 4 else -1
    k_row, k_head = _rows("k", k, pool, kv)
    v_row, v_head = _rows("v", v, pool, kv)
    dtype = _TYPE.get(k.dtype)
    _need(dtype is not None and k.dtype is v.dtype and k.shape == v.shape, "k and v are float32, bfloat16 or float16, and alike")
    check(_lib.lib().b200_kv4_append(_step(pool, table, held, first, slots, k.shape[0]), dtype, k.data_ptr(), k_row, k_head, v.data_ptr(), v_row, v_head), "kv4_append")


def kv4_read(pool: torch.Tensor, table: torch.Tensor, held: torch.Tensor, first: torch.Tensor, rows: int, dtype: torch.dtype = torch.bfloat16, slots: Optional[torch.Tensor] = None,
             out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """the rows at positions held, held + 1, ... of each sequence, as kv4_append wrote them: k, v [rows, n_head_kv, head_dim]. Rows of no sequence are left as they are (in `out`)"""
    _need(dtype in _TYPE, "dtype is float32, bfloat16 or float16")
    c = _step(pool, table, held, first, slots, rows)
    shape = (rows, pool.shape[1], pool.shape[3] // 18)
    if out is None:
        k, v = torch.empty(shape, dtype=dtype, device=pool.device), torch.empty(shape, dtype=dtype, device=pool.device)
    else:
        k, v = out
        for x in out:
            _need(x.shape == shape and x.dtype is dtype and x.device == pool.device and x.is_contiguous(), "out is a pair of contiguous tensors [rows, n_head_kv, head_dim] of dtype")
    check(_lib.lib().b200_kv4_read(c, _TYPE[dtype], k.data_ptr(), v.data_ptr()), "kv4_read")
    return k, v


def kv4_attention(q: torch.Tensor, pool: torch.Tensor, table: torch.Tensor, held: torch.Tensor, first: torch.Tensor, slots: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                  window: int = 0, max_rows: Optional[int] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """attention of the step's rows q [rows, n_head, head_dim] (bfloat16 or float16, any strides over rows and heads) over the positions up to their own, kv4_append having put those into
    the pool; window > 0: over the last `window` of them. scale: 1 / sqrt(head_dim). max_rows: the largest number of rows of a sequence, if the program knows it (it chooses kernels and
    changes no result; else the mean).
    Rows of no sequence are left as they are (in `out`)"""
    row, head = _rows("q", q, pool)
    dtype = _TYPE.get(q.dtype)
    _need(dtype, "q is bfloat16 or float16")
    rows, heads, hd = q.shape
    c = _step(pool, table, held, first, slots, rows)
    device = q.device
    if out is None:
        out = torch.empty((rows, heads, hd), dtype=q.dtype, device=device)
    else:
        _need(out.shape == q.shape and out.dtype is q.dtype and out.device == device and out.is_contiguous(), "out is a contiguous tensor like q")
    most = max(1, -(-rows // max(1, first.numel() - 1)) if max_rows is None else max_rows)
    L = _lib.lib()
    shape = (device.index, heads, pool.shape[1], hd, first.numel(), rows, most)
    size = _work_bytes.get(shape)
    if size is None:
        size = L.b200_kv4_attention_workspace(c, heads, most)
        check(size < 0, "kv4_attention")
        if len(_work_bytes) > 4096:
            _work_bytes.clear()
        _work_bytes[shape] = size
    work = torch.empty(size, dtype=torch.uint8, device=device)
    check(L.b200_kv4_attention(c, dtype, q.data_ptr(), row, head, heads, hd ** -0.5 if scale is None else scale, window, most, out.data_ptr(), work.data_ptr(), size), "kv4_attention")
    return out


_work_bytes: Dict[tuple, int] = {}       # sizes of workspaces by the shapes they are for


def _pages(table, held, refs, page_tokens: int, pool=None) -> bytes:
    """struct b200_pages"""
    index = _on(refs)
    at, n_slots, most, stride = _table(table, index)
    held_at = _ints("held", held, index, n_slots) if held is not None else at
    n = refs.numel()
    if pool is None:
        return _PAGES.pack(index, n, page_tokens, 1, 64, n_slots, most, 1, _stream(index), 0, 0, 0, stride, at, held_at, _ints("refs", refs, index))
    shape = pool.shape
    if len(shape) != 5 or pool.get_device() != index or shape[1] != n:
        raise ValueError("pool is [n_layer, n_pages, n_head_kv, page_tokens / 16, 18 * head_dim], refs has an entry a page")
    return _PAGES.pack(index, n, 16 * shape[3], shape[2], shape[4] // 18, n_slots, most, shape[0], _stream(index), pool.data_ptr(), pool.stride(0), _page_stride(pool, shape), stride, at, held_at,
                       _ints("refs", refs, index))


def _work(p: bytes, n: int, device) -> torch.Tensor:
    size = _lib.lib().b200_pages_workspace(p, n)
    check(size < 0, "pages_workspace")
    return torch.empty(size, dtype=torch.uint8, device=device)


def pages_reserve(table: torch.Tensor, held: torch.Tensor, refs: torch.Tensor, first: torch.Tensor, page_tokens: int, slots: Optional[torch.Tensor] = None) -> torch.Tensor:
    """pages for first[i + 1] - first[i] tokens more of each sequence, the lowest free ones, in order. Returns the status on the device, int32 [1]: 0, the number of pages that were
    missing, or -1 where slots or tables cannot be; then nothing has changed"""
    n = first.numel() - 1
    _need(n >= 0, "first has one entry more than there are sequences")
    p, index = _pages(table, held, refs, page_tokens), refs.get_device()
    if slots is None:
        _need(n <= table.shape[0], "without slots, sequence i is slot i: more sequences than slots")
    status = torch.empty(1, dtype=_I32, device=refs.device)
    check(_lib.lib().b200_pages_reserve(p, _ints("slots", slots, index, n) if slots is not None else None, _ints("first", first, index), n, status.data_ptr()), "pages_reserve")
    return status


def pages_fork(pool: torch.Tensor, table: torch.Tensor, held: torch.Tensor, refs: torch.Tensor, parents: torch.Tensor, children: torch.Tensor) -> torch.Tensor:
    """slot children[i], which is empty, becomes what slot parents[i] is: full pages are shared, a last page that is part full is copied in every layer. Returns the status, see pages_reserve"""
    p, n, index = _pages(table, held, refs, 0, pool), parents.numel(), refs.get_device()
    work, status = _work(p, n, refs.device), torch.empty(1, dtype=_I32, device=refs.device)
    check(_lib.lib().b200_pages_fork(p, _ints("parents", parents, index), _ints("children", children, index, n), n, status.data_ptr(), work.data_ptr(), work.numel()), "pages_fork")
    return status


def pages_free(table: torch.Tensor, held: torch.Tensor, refs: torch.Tensor, slots: torch.Tensor) -> None:
    """the slots give their pages back and are empty"""
    check(_lib.lib().b200_pages_free(_pages(table, held, refs, 16), _ints("slots", slots, refs.get_device()), slots.numel()), "pages_free")


def pages_compact(pool: torch.Tensor, table: torch.Tensor, refs: torch.Tensor) -> torch.Tensor:
    """pages in use move to the lowest places and tables follow. Returns how many there are, int32 [1] on the device: no page from that one on is in use"""
    p = _pages(table, None, refs, 0, pool)
    work, live = _work(p, refs.numel(), refs.device), torch.empty(1, dtype=_I32, device=refs.device)
    check(_lib.lib().b200_pages_compact(p, live.data_ptr(), work.data_ptr(), work.numel()), "pages_compact")
    return live


def pages_copy(pool: torch.Tensor, table: torch.Tensor, refs: torch.Tensor, src: torch.Tensor, dst: torch.Tensor) -> torch.Tensor:
    """page dst[i] becomes page src[i] in every layer. Returns the status: -1, and nothing copied, where a page is written twice, or written and read, or does not exist"""
    p, n, index = _pages(table, None, refs, 0, pool), src.numel(), refs.get_device()
    work, status = _work(p, n, refs.device), torch.empty(1, dtype=_I32, device=refs.device)
    check(_lib.lib().b200_pages_copy(p, _ints("src", src, index), _ints("dst", dst, index, n), n, status.data_ptr(), work.data_ptr(), work.numel()), "pages_copy")
    return status


def sample(logits: torch.Tensor, u: torch.Tensor, temperature: Optional[torch.Tensor] = None, top_k: Optional[torch.Tensor] = None, top_p: Optional[torch.Tensor] = None,
           min_p: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """one token a row of logits [rows, n_vocab] by the row's random number u (0 <= u < 1), temperature, top_k, top_p and min_p (tensors of an entry a row; None: 1, all, 1, 0), the filters in
    that order of b200_sample. Returns ids, int32 [rows], and the log of each drawn token's share of what the filters kept, float32 [rows]"""
    index = _on(logits)
    dtype, rows = _TYPE.get(logits.dtype), logits.shape[0]
    if logits.dim() != 2 or dtype is None or (logits.stride(1) != 1 and logits.shape[1] != 1):
        raise ValueError("logits is a float32, bfloat16 or float16 tensor [rows, n_vocab] of contiguous rows")
    vocab = logits.shape[1]
    f = torch.float32
    at = (_per_row("u", u, f, rows, index), _per_row("temperature", temperature, f, rows, index), _per_row("top_k", top_k, _I32, rows, index), _per_row("top_p", top_p, f, rows, index),
          _per_row("min_p", min_p, f, rows, index))
    device = logits.device
    ids, logprobs = torch.empty(rows, dtype=_I32, device=device), torch.empty(rows, dtype=f, device=device)
    check(_lib.lib().b200_sample(index, _stream(index), dtype, logits.data_ptr(), logits.stride(0) if rows > 1 else vocab, rows, vocab, *at, ids.data_ptr(), logprobs.data_ptr()), "sample")
    return ids, logprobs


def _per_row(name: str, t: Optional[torch.Tensor], dtype: torch.dtype, rows: int, index: int) -> Optional[int]:
    if t is None:
        return None
    if t.dtype is not dtype or t.dim() != 1 or t.numel() != rows or t.get_device() != index or not t.is_contiguous():
        raise ValueError(f"{name} is a contiguous {dtype} tensor of {rows} entries on the logits' device")
    return t.data_ptr()
