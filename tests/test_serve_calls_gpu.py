"""Calls of booster_b200.serve and of its C entry points that a program may make beside those of tests/test_serve_gpu.py."""
import ctypes as C
import math
import os
import subprocess
import sys

import pytest
import torch

from booster_b200 import _lib, serve
from tests.test_serve_gpu import BF16, F16, F32, Case, check_rows, ints

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
MANY = 4096                              # rows announced: always the form for many


def alone(program):
    """in a process of its own, where nothing was called before"""
    r = subprocess.run([sys.executable, "-c", program], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip().endswith("done"), (r.returncode, r.stdout[-2000:], r.stderr[-4000:])


@pytest.mark.parametrize("n_pages,n_slots", [(65024, 256), (65000, 300), (64416, 1)])
def test_the_first_pool_of_a_process(n_pages, n_slots):
    """the bitmaps of pages and slots take 8052 to 8192 bytes, the lists beside them 40 KB: more than a block has without leave"""
    alone(f"""
import torch
from booster_b200 import serve
ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
table, held, refs = torch.full(({n_slots}, 4), -1, dtype=torch.int32, device="cuda"), torch.zeros({n_slots}, dtype=torch.int32, device="cuda"), torch.zeros({n_pages}, dtype=torch.int32, device="cuda")
refs[:3] = 1
assert serve.pages_reserve(table, held, refs, ints([0, 20]), 16).item() == 0
assert table[0].tolist() == [3, 4, -1, -1] and refs.sum().item() == 5
print("done")
""")


def test_a_call_that_failed_leaves_no_error_behind():
    """a launch that CUDA refuses (the legacy stream, while a stream that waits for it is captured) is that call's error and no other's"""
    alone("""
import ctypes as C
import numpy as np, torch
from cuda.bindings import runtime as rt
from booster_b200 import _lib, serve
L = _lib.lib()
x = torch.randn(4, 1, 64, device="cuda", dtype=torch.float16)
pool = serve.kv4_pool(2, 16, 1, 64)[0]
table, held, first = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in ([[0, 1]], [0], [0, 4]))
c = _lib.Kv4(device=0, n_pages=2, page_tokens=16, n_head_kv=1, head_dim=64, n_slots=1, max_pages=2, n_seq=1, n_rows=4, stream=None, pool=pool.data_ptr(), page_stride=18 * 64, table_stride=2,
             table=table.data_ptr(), held=held.data_ptr(), slots=None, first=first.data_ptr())
append = lambda: L.b200_kv4_append(C.byref(c), 2, x.data_ptr(), 64, 64, x.data_ptr(), 64, 64)
assert append() == 0
torch.cuda.synchronize()
err, stream = rt.cudaStreamCreate()
assert int(err) == 0
assert int(rt.cudaStreamBeginCapture(stream, rt.cudaStreamCaptureMode.cudaStreamCaptureModeGlobal)[0]) == 0
assert append() != 0 and "launch" in _lib.last_error(), _lib.last_error()
rt.cudaStreamEndCapture(stream)
while int(rt.cudaGetLastError()[0]): pass
y, v = np.zeros(64, np.float32), np.ones(64, np.float32)
f = C.POINTER(C.c_float)
rc = L.b200_op_rms_norm(v.ctypes.data_as(f), None, 64, 1e-6, y.ctypes.data_as(f))
assert rc == 0, _lib.last_error()
assert append() == 0, _lib.last_error()
print("done")
""")


def test_threads_with_calls_of_different_sizes():
    """two host threads ask for different amounts of shared memory for the same kernels at the same time: each gets its own, and so does every call behind them"""
    alone("""
import ctypes as C, threading
import torch
from booster_b200 import _lib, serve
L = _lib.lib()
N = 4096
ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
pool, table, held, first = serve.kv4_pool(1, 16, 1, 64)[0], torch.zeros(N, 1, dtype=torch.int32, device="cuda"), ints([0] * N), ints([0] + [1] * N)
logits = torch.zeros(1, 1 << 18, device="cuda")
class Caller:
    def __init__(self, me):
        self.stream = torch.cuda.Stream()
        self.q, self.out = (torch.zeros(1, 1, 64, dtype=torch.float16, device="cuda") for _ in range(2))
        self.work = torch.empty(64 << 20, dtype=torch.uint8, device="cuda")
        self.u, self.ids = torch.zeros(1, device="cuda"), ints([0])
        self.steps = [_lib.Kv4(device=0, n_pages=1, page_tokens=16, n_head_kv=1, head_dim=64, n_slots=N, max_pages=1, n_seq=2 * i + me, n_rows=1, stream=self.stream.cuda_stream,
                               pool=pool.data_ptr(), page_stride=18 * 64, table_stride=1, table=table.data_ptr(), held=held.data_ptr(), slots=None, first=first.data_ptr()) for i in range(1, 2000)]
        # (the addresses are made ready: between two calls stands as little as can be)
        self.attends = [(C.byref(c), 2, self.q.data_ptr(), 64, 64, 1, 1.0, 0, 1, self.out.data_ptr(), self.work.data_ptr(), self.work.numel()) for c in self.steps]
        self.samples = [(0, self.stream.cuda_stream, 0, logits.data_ptr(), 1 << 18, 1, 128 * i + 64 * me, self.u.data_ptr(), None, None, None, None, self.ids.data_ptr(), None) for i in range(1, 2000)]
bad, gate = [], threading.Barrier(2)
def run(caller, call, all_args):
    gate.wait()
    for args in all_args:
        if call(*args): bad.append((call.__name__, args[6], _lib.last_error()))
callers = [Caller(0), Caller(1)]
torch.cuda.synchronize()
for call, name in ((L.b200_kv4_attention, "attends"), (L.b200_sample, "samples")):
    threads = [threading.Thread(target=run, args=(c, call, getattr(c, name))) for c in callers]
    [t.start() for t in threads]; [t.join() for t in threads]
for args in callers[0].attends[::3]:                                  # and one after the other
    if L.b200_kv4_attention(*args): bad.append(("later", args[6], _lib.last_error()))
torch.cuda.synchronize()
assert not bad, (len(bad), bad[:5])
print("done")
""")


def test_a_step_whose_rows_belong_to_no_sequence():
    """a captured step that idles: nothing is computed, but the kernels write their plan into the workspace, which is its owner's again behind the call"""
    n, rows = 4096, 5
    L = _lib.lib()
    pool, table, held, first = serve.kv4_pool(1, 16, 2, 64)[0], ints([[0]] * n), ints([0] * n), ints([0] * (n + 1))
    out = torch.full((rows, 64, 64), 7.0, dtype=F16, device="cuda")
    q = torch.randn(rows, 64, 64, device="cuda").half()
    for heads, max_rows in ((8, 1), (64, 1), (8, MANY)):
        c = _lib.Kv4(device=0, n_pages=1, page_tokens=16, n_head_kv=2, head_dim=64, n_slots=n, max_pages=1, n_seq=n, n_rows=rows, stream=torch.cuda.current_stream().cuda_stream, pool=pool.data_ptr(),
                     page_stride=2 * 18 * 64, table_stride=1, table=table.data_ptr(), held=held.data_ptr(), slots=None, first=first.data_ptr())
        work = torch.empty(L.b200_kv4_attention_workspace(C.byref(c), heads, max_rows), dtype=torch.uint8, device="cuda")
        for _ in range(50):
            assert L.b200_kv4_attention(C.byref(c), 2, q.data_ptr(), 64 * 64, 64, heads, 1.0, 0, max_rows, out.data_ptr(), work.data_ptr(), work.numel()) == 0, _lib.last_error()
            work.fill_(0x55)
            assert (work == 0x55).all()
    assert (out == 7).all()


def test_first_calls_inside_a_capture():
    """every operator for the first time in its process while a graph is captured; the graph then gives what calls give"""
    alone("""
import torch
from booster_b200 import serve
ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
gen = torch.Generator(device="cuda").manual_seed(0)
n, page = 3, 16
table, held, refs, first = torch.full((8, 6), -1, dtype=torch.int32, device="cuda"), torch.zeros(8, dtype=torch.int32, device="cuda"), torch.zeros(40, dtype=torch.int32, device="cuda"), ints([0, 20, 21, 60])
advance = torch.zeros(8, dtype=torch.int32, device="cuda")
advance[:3] = first.diff()
pool = serve.kv4_pool(40, page, 2, 64, 2)
k, v, q = (torch.randn(60, h, 64, generator=gen, device="cuda").half() for h in (2, 2, 8))
logits, u = torch.randn(3, 5000, generator=gen, device="cuda"), torch.rand(3, generator=gen, device="cuda")
gone, parents, children, src, dst, ks = ints([1]), ints([0, 2]), ints([4, 5]), ints([0]), ints([39]), ints([5, 0, 40])
def step():
    out = [serve.pages_reserve(table, held, refs, first, page)]
    for layer in pool:
        serve.kv4_append(layer, table, held, first, k, v)
        out += serve.kv4_read(layer, table, held, first, 60)
        out += [serve.kv4_attention(q, layer, table, held, first, max_rows=m) for m in (4096, 2, 12)]
    held.add_(advance)
    out.append(serve.pages_fork(pool, table, held, refs, parents, children))
    serve.pages_free(table, held, refs, gone)
    out.append(serve.pages_compact(pool, table, refs))
    out.append(serve.pages_copy(pool, table, refs, src, dst))
    out += serve.sample(logits, u, top_k=ks)
    return out
state = (table, held, refs, pool)
start = [x.clone() for x in state]
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    outs = step()
for x, y in zip(state, start): assert torch.equal(x, y)
graph.replay()
torch.cuda.synchronize()
ends = [x.clone() for x in state]
for x, y in zip(state, start): x.copy_(y)
eager = step()
for x, y in zip(state, ends): assert torch.equal(x, y)
for x, y in zip(outs, eager): assert torch.equal(x, y)
assert outs[0].item() == 0 and eager[-5].item() == 0 and outs[-3].item() == 0, [o.tolist() for o in outs[-5:-2]]
print("done")
""")


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_the_widest_vocabulary(dtype):
    """2^18 logits: as many parts and as long slices as there are; a row on its own and several"""
    vocab = 1 << 18
    gen = torch.Generator(device="cuda").manual_seed(5)
    rows = (3 * torch.randn(5, vocab, generator=gen, device="cuda")).to(dtype)
    rows[4, -1] = 40                                                     # the last token
    u = torch.rand(5, generator=gen, device="cuda")
    u[3] = 1 - 2.0 ** -24
    for p in (dict(), dict(top_k=[50] * 5), dict(top_p=[0.9] * 5), dict(top_k=[vocab] * 5, min_p=[0.01] * 5), dict(top_k=[5000] * 5, top_p=[0.99] * 5, temperature=[2.0] * 5)):
        check_rows(rows, u, **p)
        check_rows(rows[1:2], u[1:2], **{k: v[:1] for k, v in p.items()})


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads,max_rows", [(4, 1), (64, 1), (4, MANY)])
def test_weights_far_below_the_largest(heads, max_rows, dtype):
    """one position stands `above` over all others and has a value of 0, as the first token of a long text does: the result is what the others say, however small their weights. Pieces hold
    whole sequences here, so that all weights stand against that one. What is left out of P by its rounding is half a step of 2^-24 of weights whose largest is 2^7 or more; a thousand tokens'
    sums in fp32 add less than 1000 x 2^-23"""
    n, kv, hd, held = 600, 4, 64, 1999
    pool = serve.kv4_pool(125, 16, kv, hd)
    table = ints([list(range(125))]).expand(n, 125).contiguous()
    gen = torch.Generator(device="cuda").manual_seed(1)
    k = torch.zeros(held + 1, kv, hd, device="cuda")
    k[0, :, 0] = 8.0
    v = 0.25 + torch.rand(held + 1, kv, hd, generator=gen, device="cuda")
    v[0] = 0
    serve.kv4_append(pool[0], table, ints([0] * n), ints([0, held + 1]), k, v)
    k, v = (x.double() for x in serve.kv4_read(pool[0], table, ints([0] * n), ints([0, held + 1]), held + 1, F32))
    for above in (4.0, 9.0, 13.0, 17.5):
        q = torch.zeros(n, heads, hd, device="cuda", dtype=dtype)
        q[:, :, 0] = above / 8
        assert (q[0, 0, 0].item() * k[0, 0, 0].item()) == above
        out = serve.kv4_attention(q, pool[0], table, ints([held] * n), ints(list(range(n + 1))), scale=1.0, max_rows=max_rows).double()
        w = torch.softmax(k[:, 0, 0] * above / 8, 0)
        want = torch.einsum("t,thd->hd", w, v).repeat_interleave(heads // kv, 0)
        room = want * (2.0 ** -11 + 2.0 ** -13) + 2.0 ** -32 * v.abs().sum(0).repeat_interleave(heads // kv, 0)
        room = room + torch.finfo(dtype).eps / 2 * (want + room) + (2.0 ** -25 if dtype == F16 else 0.0)
        assert ((out - want).abs() <= room).all(), (above, ((out - want).abs() / want).max().item())


@pytest.mark.parametrize("heads,max_rows", [(2, 1), (32, 1), (2, MANY)])
def test_queries_that_are_not_finite(heads, max_rows):
    """a product with an infinity is an infinity or a NaN, and no soft-max of such scores is a number: the row's head answers NaN, and 0 where it sees nothing. Other rows do not notice"""
    c = Case([0, 40, 7], [1, 1, 1], kv=2, hd=64)
    c.fill()
    k = -torch.ones(c.rows, 2, 64, device="cuda").half()                # the first sequence sees one position; every score with a query of one infinity is an infinity of one sign
    v = c.randn(c.rows, 2, 64).half()
    serve.kv4_append(*c.args(), k, v, c.slots)
    q = c.randn(c.rows, heads, 64).half()
    right = serve.kv4_attention(q, *c.args(), slots=c.slots, max_rows=max_rows)
    for x in (float("inf"), -float("inf"), float("nan")):
        for row in range(c.rows):
            bad = q.clone()
            bad[row, 1] = 0
            bad[row, 1, 9] = x
            out = serve.kv4_attention(bad, *c.args(), slots=c.slots, max_rows=max_rows)
            assert torch.isnan(out[row, 1]).all(), (x, row)
            out[row, 1] = right[row, 1]
            assert torch.equal(out, right)
            none = torch.full_like(c.table, -1)
            assert not serve.kv4_attention(bad, c.pool[0], none, c.held, c.first, c.slots, max_rows=max_rows).any()


@pytest.mark.parametrize("hd", [64, 128])
def test_a_wait_that_runs_out_is_told(hd):
    """queries that never come: the kernel gives up, frees what it holds and says so, whichever call comes next; that call has done nothing, and after it all is as before"""
    L = _lib.lib()
    c = Case([300, 5], [64, 1], kv=2, hd=hd)
    c.fill()
    q = c.randn(c.rows, 8, hd).half()
    attend = lambda most=MANY: serve.kv4_attention(q, *c.args(), slots=c.slots, max_rows=most)
    right, few = attend(), attend(1)
    k = c.randn(c.rows, 2, hd).half()
    refs = torch.ones(c.pages, dtype=torch.int32, device="cuda")
    pool, one, none = c.pool.clone(), ints([1]), ints([])
    calls = [lambda: serve.kv4_append(*c.args(), k, k, c.slots), lambda: serve.kv4_read(*c.args(), c.rows, F16, c.slots), lambda: attend(1), attend,
             lambda: serve.pages_reserve(c.table, c.held, refs, ints([0, 1]), 16, c.slots[:1]), lambda: serve.pages_fork(c.pool, c.table, c.held, refs, none, none),
             lambda: serve.pages_free(c.table, c.held, refs, c.slots), lambda: serve.pages_compact(c.pool, c.table, refs), lambda: serve.pages_copy(c.pool, c.table, refs, none, none),
             lambda: serve.sample(torch.zeros(1, 10, device="cuda"), torch.zeros(1, device="cuda")), serve.kv4_status]
    table, held = c.table.clone(), c.held.clone()
    try:
        for call in calls:
            L.b200_kv4_drill(64)
            attend()
            L.b200_kv4_drill(0)
            torch.cuda.synchronize()
            with pytest.raises(_lib.B200Error, match="ran out"):
                call()
            assert torch.equal(c.pool, pool) and torch.equal(c.table, table) and torch.equal(c.held, held)
            serve.kv4_status()
            assert torch.equal(attend(), right) and torch.equal(attend(1), few)
        # a replayed graph makes no call that could look
        stream = torch.cuda.Stream()
        graph = torch.cuda.CUDAGraph()
        L.b200_kv4_drill(64)
        with torch.cuda.graph(graph, stream=stream):
            attend()
        L.b200_kv4_drill(0)
        graph.replay()
        torch.cuda.synchronize()
        with pytest.raises(_lib.B200Error, match="ran out"):
            serve.kv4_status(0)
        assert torch.equal(attend(), right)
    finally:
        L.b200_kv4_drill(0)


@pytest.mark.parametrize("hd", [64, 128])
def test_calls_one_behind_the_other_repeat_themselves(hd):
    """blocks of one call begin where those of another have just ended, with barriers and tiles in the same shared memory: every call gives the bits that it gave alone"""
    cases = [Case([300, 0, 77], [200, 65, 130], page=32, kv=2, hd=hd, seed=1), Case([2000], [40], page=16, kv=4, hd=hd, seed=2), Case([50] * 40, [1] * 40, page=16, kv=2, hd=hd, seed=3)]
    calls = []
    for c, most in zip(cases, (MANY, MANY, 1)):
        c.fill()
        q = c.randn(c.rows, 8, hd).half()
        calls.append(lambda c=c, q=q, most=most: serve.kv4_attention(q, *c.args(), slots=c.slots, max_rows=most))
    alone = []
    for call in calls:
        torch.cuda.synchronize()
        alone.append(call())
        torch.cuda.synchronize()
    outs = [[call() for call in calls] for _ in range(100)]
    for out in outs:
        assert all(torch.equal(x, y) for x, y in zip(out, alone))


def test_a_min_p_that_is_no_number_filters_nothing():
    """as a top_p that is none does"""
    gen = torch.Generator(device="cuda").manual_seed(3)
    rows, u = torch.randn(64, 1000, generator=gen, device="cuda"), torch.rand(64, generator=gen, device="cuda")
    nan = torch.full((64,), math.nan, device="cuda")
    for more in ({}, dict(top_k=ints([30] * 64)), dict(top_p=torch.full((64,), 0.9, device="cuda"))):
        want = serve.sample(rows, u, **more)
        for name in ("min_p", "top_p"):
            if name not in more:
                got = serve.sample(rows, u, **more, **{name: nan})
                assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), name
