"""Calls of the operators around drafted tokens and the 16-bit cache that a program makes in earnest: captured, on streams, from threads, one behind the other, and all of them together."""
import ctypes as C
import random

import numpy as np
import pytest
import torch

from booster_b200 import _lib, serve
from tests import serve_draft_oracle as oracle
from tests.test_serve_calls_gpu import alone
from tests.test_serve_draft_gpu import BF16, F16, Case, assert_attends, assert_verifies, ints, step as rows_to_verify

pytestmark = pytest.mark.gpu

# (held, counts, query heads, KV heads, wide table): few rows in one launch, with warps that share what is read, in a line of pieces, and rows for tcgen05
FORMS = {"unit": ([300, 5, 40], [1, 1, 1], 8, 2, False), "shared": ([300, 5, 40], [5, 2, 7], 8, 2, False), "line": ([3000, 5, 400], [1, 2, 1], 8, 2, True), "rows": ([300, 0, 77], [200, 65, 3], 8, 2, False)}


def made(form, hd=64, seed=0, dtype=BF16):
    held, counts, heads, kv, wide = FORMS[form]
    c = Case(held, counts, page=16, kv=kv, hd=hd, seed=seed, dtype=dtype)
    if wide:
        c.widened()
    c.fill()
    return c, c.randn(c.rows, heads, hd).to(dtype)


def test_first_calls_inside_a_capture():
    """every operator for the first time in its process while a graph is captured; the graph then gives what calls give"""
    alone("""
import torch
from booster_b200 import serve
ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
gen = torch.Generator(device="cuda").manual_seed(0)
page = 16
table, held, refs, counts = torch.full((8, 6), -1, dtype=torch.int32, device="cuda"), torch.zeros(8, dtype=torch.int32, device="cuda"), torch.zeros(400, dtype=torch.int32, device="cuda"), ints([20, 1, 39])
wide = torch.full((8, 4000), -1, dtype=torch.int32, device="cuda")
pool = serve.kv16_pool(400, page, 2, 64, 2)
k, v, q = (torch.randn(62, h, 64, generator=gen, device="cuda").bfloat16() for h in (2, 2, 8))
logits, u, accept, ids = torch.randn(62, 5000, generator=gen, device="cuda"), torch.rand(62, generator=gen, device="cuda"), torch.rand(62, generator=gen, device="cuda"), ints(list(range(62)))
probs, ks, slots = torch.softmax(logits + 1, 1), ints([5] * 30 + [0] * 32), ints([0, 1, 2])
def step():
    out = list(serve.pages_plan(table, held, refs, counts, page, 62))
    first = out[0]
    for layer in pool:
        serve.kv16_append(layer, table, held, first, k, v)
        out += [serve.kv16_attention(q, layer, table, held, first, max_rows=m, window=w, sinks=3) for m in (1, 5, 12, 4096) for w in (0, 9)]
        wide[:, :6] = table
        out += [serve.kv16_attention(q, layer, wide, held, first, max_rows=m) for m in (1, 4, 12)]
    new = serve.verify(logits, ids, first, u, accept, top_k=ks, draft_probs=probs)
    out += new
    held[:3] += new[0]
    serve.pages_trim(table, held, refs, page, slots, 20, 2)
    return out
state = (table, held, refs, pool, wide)
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
for x, y in zip(outs, eager): assert torch.equal(x[:60], y[:60])
assert outs[3].item() == 0 and outs[0].tolist() == [0, 20, 21, 60] and refs.sum().item() > 0
print("done")
""")


@pytest.mark.parametrize("form", FORMS)
def test_graphs_streams_and_order(form):
    """captured and replayed with other lengths and queries; two graphs in one pool of memory; another stream; the same call twice gives the same bits"""
    c, q = made(form)
    out = torch.zeros_like(q)
    table, held = c.table, c.held.clone()
    call = lambda: serve.kv16_attention(q, c.pool[0], table, held, c.first, c.slots, window=100, sinks=7, out=out)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    with torch.cuda.graph(graphs[0]):
        call()
    with torch.cuda.graph(graphs[1], pool=graphs[0].pool()):
        call()
    for turn in range(4):
        held.copy_(c.held - turn * (c.held > 10).int())
        q.copy_(c.randn(*q.shape))
        c2 = Case.__new__(Case)
        c2.__dict__.update(c.__dict__)
        c2.held_l = [held[s].item() for s in c.slots_l]
        out.zero_()
        graphs[turn % 2].replay()
        got = out.clone()
        assert_attends(c2, q, got, 100, 7)
        assert torch.equal(call(), got)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            again = serve.kv16_attention(q, c.pool[0], table, held, c.first, c.slots, window=100, sinks=7)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(again, got)


def test_calls_see_what_the_call_in_front_wrote():
    """a step's calls stand ready behind one another and behind other kernels, some of which let the next one begin early: with nothing waited for between them they give what they give one by one"""
    page, kv, hd, slots = 16, 2, 64, 6
    gen = torch.Generator(device="cuda").manual_seed(2)
    logits = 3 * torch.randn(40, 4000, generator=gen, device="cuda")
    wide = 2 * torch.randn(60, 70000, generator=gen, device="cuda")

    def state():
        return [ints([[-1] * 60] * slots), ints([0] * slots), ints([0] * 400), torch.zeros(1, 400, 2, kv, page, hd, dtype=BF16, device="cuda"), torch.zeros(400 * page, dtype=torch.int32, device="cuda")]

    def steps(sync):
        table, held, refs, pool, marks = state()
        r, g, seen = random.Random(1), torch.Generator(device="cuda").manual_seed(3), []
        done = torch.cuda.synchronize if sync else lambda: None
        for turn in range(25):
            counts = [r.choice([0, 1, 4, 6]) for _ in range(slots)] if turn % 5 else [r.choice([1, 30]) for _ in range(slots)]
            rows = sum(counts)
            n, ids = ints(counts), torch.randint(0, 4000, (rows,), generator=g, device="cuda", dtype=torch.int32)
            done()
            first, positions, places, status = serve.pages_plan(table, held, refs, n, page, rows)
            done()
            marks[places.long()] = ids
            k, v, q = (torch.randn(rows, h, hd, generator=g, device="cuda").bfloat16() for h in (kv, kv, 8))
            serve.kv16_append(pool[0], table, held, first, k, v)
            done()
            outs = [serve.kv16_attention(q, pool[0], table, held, first, max_rows=max(counts + [1]), window=200, sinks=3)]
            done()
            outs.append(serve.kv16_attention(q, pool[0], torch.cat([table, torch.full((slots, 5000), -1, dtype=torch.int32, device="cuda")], 1), held, first, max_rows=2))
            done()
            outs.append(serve.kv16_attention(q, pool[0], table, held, first, max_rows=100))
            done()
            u = torch.rand(max(rows, 60), generator=g, device="cuda")
            new = serve.verify(logits[:min(rows, 40)], ids[:40], first.clamp(max=min(rows, 40)), u[:min(rows, 40)], u[:min(rows, 40)])
            done()
            many = serve.verify(wide, ids.repeat(60)[:60] if rows else ints([0] * 60), torch.arange(0, 61, 2, device="cuda").int(), u[:60], u[:60])
            done()
            held += torch.maximum(new[0], torch.minimum(n, torch.full_like(n, 2)))
            held.copy_(torch.minimum(held, torch.full_like(held, 700)))
            serve.pages_trim(table, held, refs, page, torch.arange(slots, device="cuda").int(), 200, 3)
            done()
            seen += [first, positions, places, status, *outs, *new, *many, table.clone(), refs.clone()]
        return [x.clone() for x in seen] + [pool, marks]
    want = steps(True)
    for _ in range(3):
        got = steps(False)
        assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("call", [*FORMS, "append", "plan", "trim", "verify", "verify many"])
def test_what_another_stream_wrote(call, captured):
    """a call that stands ready behind a kernel of its own stream waits for another stream's event too: what that one wrote late is what the call sees"""
    c, q = made(call if call in FORMS else "unit")
    front, q_front = made("unit", seed=3)
    table, big = c.table, torch.zeros(1 << 24, device="cuda")
    refs = torch.zeros(c.pages, dtype=torch.int32, device="cuda")
    k = torch.randn(c.rows, 2, 64, device="cuda").bfloat16()
    logits = torch.randn(60, 70000 if call == "verify many" else 500, device="cuda")
    ids, u, ends = torch.arange(60, device="cuda").int(), torch.full((60,), 0.4, device="cuda"), torch.arange(0, 61, 4, device="cuda").int()
    counts = ints([1, 2, 3])
    late = {"append": (c.held,), "plan": (c.held, counts, refs), "trim": (c.held, table), "verify": (logits, ends), "verify many": (logits, ends)}.get(call, (c.held, c.first, q))
    right, side = [x.clone() for x in late], torch.cuda.Stream()
    t_front, pool = front.table, c.pool.clone()
    tables, counted = table.clone(), refs.clone()

    def run():
        if call == "append":
            serve.kv16_append(c.pool[0], table, c.held, c.first, k, k, c.slots)
            return [c.pool]
        if call == "plan":
            return [*serve.pages_plan(table, c.held, refs, counts, 16, 9, c.slots), table, refs]
        if call == "trim":
            serve.pages_trim(table, c.held, refs, 16, c.slots, 20, 3)
            return [table, refs]
        if call.startswith("verify"):
            return list(serve.verify(logits, ids, ends, u, u))
        return [serve.kv16_attention(q, c.pool[0], table, c.held, c.first, c.slots)]

    def reset(wrong):
        c.pool.copy_(pool), table.copy_(tables), refs.copy_(counted)
        for x, y in zip(late, right):
            x.zero_() if wrong else x.copy_(y)

    def work():
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(20):
                big.add_(1.0)
            for x, y in zip(late, right):
                x.copy_(y)
        serve.kv16_attention(q_front, front.pool[0], t_front, front.held, front.first, front.slots)
        torch.cuda.current_stream().wait_stream(side)
        return run()
    reset(False)
    torch.cuda.synchronize()
    want = [x.clone() for x in run()]
    reset(True)
    if captured:
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            got = work()
    for _ in range(5):
        reset(True)
        torch.cuda.synchronize()
        if captured:
            graph.replay()
        else:
            got = work()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("form", FORMS)
def test_results_in_the_queries_place(form, hd):
    """a query is read by those who work on its result alone, and before that is written"""
    c, q = made(form, hd)
    want = serve.kv16_attention(q, *c.args(), slots=c.slots)
    for _ in range(20):
        x = q.clone()
        assert serve.kv16_attention(x, *c.args(), slots=c.slots, out=x).data_ptr() == x.data_ptr()
        assert torch.equal(x, want)


@pytest.mark.parametrize("captured", [False, True])
def test_behind_the_operators_of_the_4_bit_cache(captured):
    """calls of both kinds of cache one behind the other, on tables that the call in front wrote"""
    page, kv, hd, slots, rows = 16, 2, 64, 5, 60
    gen = torch.Generator(device="cuda").manual_seed(4)
    k, v, q = (torch.randn(rows, h, hd, generator=gen, device="cuda").bfloat16() for h in (kv, kv, 8))
    logits, u = torch.randn(rows, 3000, generator=gen, device="cuda"), torch.rand(rows, generator=gen, device="cuda")
    table, held, refs = ints([[-1] * 40] * slots), ints([0] * slots), ints([0] * 250)
    four, wide = serve.kv4_pool(250, page, kv, hd), torch.zeros(1, 250, 2, kv, page, hd, dtype=BF16, device="cuda")
    counts, some = ints([12, 1, 30, 0, 17]), ints([3, 0, 4])
    own, far = torch.arange(slots, device="cuda").int(), ints([[-1] * 5000] * slots)

    def work(done=lambda: None):
        out = []
        for turn in range(6):
            first = torch.cat([ints_0, counts.cumsum(0).int()])
            for call in (lambda: serve.pages_reserve(table, held, refs, first, page), lambda: serve.kv4_append(four[0], table, held, first, k, v), lambda: serve.kv16_append(wide[0], table, held, first, k, v),
                         lambda: serve.kv4_attention(q, four[0], table, held, first), lambda: serve.kv16_attention(q, wide[0], table, held, first),
                         lambda: serve.kv4_attention(q, four[0], table, held, first, max_rows=1), lambda: serve.kv16_attention(q, wide[0], torch.cat([table, far], 1), held, first, max_rows=1),
                         lambda: serve.sample(logits, u)[0], lambda: serve.verify(logits, counts.repeat(12), first, u, u)[0]):
                out.append(call())
                done()
            held.add_(torch.maximum(out[-1], torch.minimum(counts, ones)))
            serve.pages_trim(table, held, refs, page, own)
            done()
            serve.pages_free(table, held, refs, some)
            done()
            out += serve.pages_plan(table, held, refs, counts, page, rows)
            done()
            serve.pages_compact(four, table, refs) if turn == 2 else serve.pages_trim(table, held, refs, page, own, 20, 3)
            done()
            out += [table.clone(), refs.clone(), held.clone()]
        return [x for x in out if x is not None]

    def fresh():
        table.fill_(-1); held.zero_(); refs.zero_(); wide.zero_(); four.zero_()
    ints_0, ones = ints([0]), ints([4] * slots)
    want = [x.clone() for x in work(torch.cuda.synchronize)]
    fresh()
    if captured:
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = work()
        for _ in range(3):
            fresh()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(got, want))
    else:
        for _ in range(3):
            got = work()
            assert all(torch.equal(x, y) for x, y in zip(got, want))
            fresh()


def test_captured_behind_what_is_no_kernel():
    """first in a graph, behind a memset, behind a copy, and where two streams meet"""
    c, q = made("unit")
    line, q_line = made("line")
    rows, q_rows = made("rows")
    table, out = c.table, torch.zeros_like(q)
    t_line, t_rows = line.table, rows.table
    k = torch.randn(3, 2, 64, device="cuda").bfloat16()
    src = c.held.clone()
    held, other = c.held.clone(), torch.zeros(1 << 20, device="cuda")
    refs = torch.ones(c.pages, dtype=torch.int32, device="cuda")
    logits, u = torch.randn(3, 500, device="cuda"), torch.full((3,), 0.5, device="cuda")
    side = torch.cuda.Stream()

    def work():
        a = [serve.kv16_attention(q, c.pool[0], table, held, c.first, c.slots)]
        held.zero_()
        serve.kv16_append(c.pool[0], table, held, c.first, k, k, c.slots)
        held.copy_(src, non_blocking=True)
        a.append(serve.kv16_attention(q, c.pool[0], table, held, c.first, c.slots))
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(20):
                other.add_(1.0)
            held.copy_(src)
        a.append(serve.kv16_attention(q_line, line.pool[0], t_line, line.held, line.first, line.slots))
        torch.cuda.current_stream().wait_stream(side)
        a.append(serve.kv16_attention(q_rows, rows.pool[0], t_rows, rows.held, rows.first, rows.slots))
        torch.cuda.current_stream().wait_stream(side)
        a += serve.verify(logits, ints_kept, c.first, u, u)
        other.zero_()
        serve.pages_trim(table, held, refs, 16, c.slots)
        a += serve.pages_plan(table, held, refs, counts, 16, 9, c.slots)
        return a
    ints_kept, counts = ints([1, 2, 3]), ints([1, 1, 1])
    pool = c.pool.clone()
    kept = table.clone()
    want = [x.clone() for x in work()]
    torch.cuda.synchronize()
    c.pool.copy_(pool); table.copy_(kept); held.copy_(src); refs.fill_(1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = work()
    for _ in range(3):
        c.pool.copy_(pool); table.copy_(kept); held.copy_(src); refs.fill_(1)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_captured_steps_of_tables_and_verification():
    """a graph of the step's small operators, replayed with other numbers in its inputs"""
    page, n = 16, 5
    logits, ids, first, u, accept, filters, probs = rows_to_verify(3, 900, [3, 1, 4, 2, 5], BF16, [dict(temperature=0.7, top_k=40), dict(top_p=0.8), dict()], True)
    table, held, refs = ints([[-1] * 30] * n), ints([0] * n), ints([0] * 90)
    counts, slots, ids_t = ints([3, 1, 4, 2, 5]), ints([4, 2, 0, 1, 3]), ints(ids)
    state = [table, held, refs]

    def step():
        plan = serve.pages_plan(table, held, refs, counts, page, 15, slots)
        new = serve.verify(logits, ids_t, plan[0], u, accept, draft_probs=probs)
        held.index_add_(0, slots.long(), new[0])
        serve.pages_trim(table, held, refs, page, slots, 33, 5)
        return [*plan, *new]
    step()
    for x, v in zip(state, (-1, 0, 0)):
        x.fill_(v)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    gen = torch.Generator(device="cuda").manual_seed(0)
    for turn in range(40):
        counts.copy_(ints([[3, 1, 4, 2, 5], [5, 5, 5, 0, 0], [1, 1, 1, 1, 1]][turn % 3]))
        u.copy_(torch.rand(15, generator=gen, device="cuda"))
        accept.copy_(torch.rand(15, generator=gen, device="cuda"))
        before = [x.clone() for x in state]
        graph.replay()
        got, after = [x.clone() for x in outs], [x.clone() for x in state]
        for x, y in zip(state, before):
            x.copy_(y)
        want = step()
        assert all(torch.equal(x, y) for x, y in zip(got, want)) and all(torch.equal(x, y) for x, y in zip(state, after))
        used = [p for row in table.tolist() for p in row if p >= 0]
        assert len(used) == len(set(used)) == int(refs.sum()) and got[3].item() == 0


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_calls_one_behind_the_other_repeat_themselves(hd, dtype):
    """blocks of one call begin where those of another have just ended, with barriers and tiles in the same shared memory: every call gives the bits that it gave alone"""
    calls = []
    for i, form in enumerate(FORMS):
        c, q = made(form, hd, i, dtype)
        calls.append(lambda c=c, q=q, t=c.table: serve.kv16_attention(q, c.pool[0], t, c.held, c.first, c.slots))
        c4 = serve.kv4_pool(c.pages, 16, 2, hd)
        calls.append(lambda c=c, q=q, t=c.table, p=c4: serve.kv4_attention(q, p[0], t, c.held, c.first, c.slots))
    first = []
    for call in calls:
        torch.cuda.synchronize()
        first.append(call())
        torch.cuda.synchronize()
    outs = [[call() for call in calls] for _ in range(60)]
    for out in outs:
        assert all(torch.equal(x, y) for x, y in zip(out, first))


def test_two_streams_at_once():
    """calls of all forms on two streams, their kernels side by side on the card: nothing is shared but the pools, which are read"""
    pairs = [made(form, 128, i) for i, form in enumerate(FORMS)]
    call = lambda c, q, t: serve.kv16_attention(q, c.pool[0], t, c.held, c.first, c.slots)  # noqa: E731
    tables = [c.table for c, _ in pairs]
    want = [call(c, q, t) for (c, q), t in zip(pairs, tables)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for turn in range(30):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                k = (turn + i) % len(pairs)
                got[i].append((k, call(*pairs[k], tables[k])))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[k]) for g in got for k, x in g)


def test_threads_with_calls_of_different_sizes():
    """host threads whose calls ask for different forms and sizes at the same time, for the first time in their process"""
    alone("""
import threading, torch
from booster_b200 import serve
ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
pool = serve.kv16_pool(40, 16, 2, 64)
pool.normal_()
table = torch.arange(40, dtype=torch.int32, device="cuda").reshape(2, 20)
held = ints([100, 37])
logits = torch.randn(64, 3000, device="cuda")
jobs = []
for rows in (1, 2, 5, 30, 100):
    q, first = torch.randn(2 * rows, 8, 64, device="cuda").bfloat16(), ints([0, rows, 2 * rows])
    jobs.append(lambda q=q, first=first, rows=rows: serve.kv16_attention(q, pool[0], table, held, first, max_rows=rows))
    n = min(64, 2 * rows)
    jobs.append(lambda n=n: serve.verify(logits[:n], ints(list(range(n))), ints([0, n]), torch.full((n,), 0.3, device="cuda"), torch.full((n,), 0.6, device="cuda"))[1])
bad, outs = [], [[], []]
gate = threading.Barrier(2)
def run(me):
    try:
        s = torch.cuda.Stream()
        gate.wait()
        with torch.cuda.stream(s):
            for turn in range(20):
                for i in range(len(jobs)): outs[me].append((i if not me else len(jobs) - 1 - i, jobs[i if not me else len(jobs) - 1 - i]()))
        s.synchronize()
    except Exception as e:
        bad.append(e)
torch.cuda.synchronize()
threads = [threading.Thread(target=run, args=(m,)) for m in (0, 1)]
[t.start() for t in threads]; [t.join() for t in threads]
torch.cuda.synchronize()
assert not bad, bad
want = [j() for j in jobs]
assert all(torch.equal(x, want[i]) for o in outs for i, x in o)
print("done")
""")


def test_a_workspace_is_its_owner_s_again_behind_the_call():
    """also where the step's rows belong to no sequence; one that is too small or off its alignment is refused, and none is needed where one launch does"""
    L = _lib.lib()
    for heads, kv, max_rows, max_pages, n in ((8, 2, 1, 60000, 4096), (64, 2, 1, 60000, 4096), (8, 2, 500, 2, 300), (8, 2, 1, 2, 2)):
        pool, table, held = serve.kv16_pool(1, 16, kv, 64, dtype=F16)[0], torch.zeros(1, max_pages, dtype=torch.int32, device="cuda").expand(n, -1), ints([0] * n)
        rows = 5
        q, out = torch.randn(rows, heads, 64, device="cuda").half(), torch.full((rows, heads, 64), 7.0, dtype=F16, device="cuda")
        slots, first = ints([0] * n), ints([0] * (n + 1))
        c = _lib.Kv4(device=0, n_pages=1, page_tokens=16, n_head_kv=kv, head_dim=64, n_slots=1, max_pages=max_pages, n_seq=n, n_rows=rows, stream=torch.cuda.current_stream().cuda_stream,
                     pool=pool.data_ptr(), page_stride=2 * kv * 16 * 64 * 2, table_stride=max_pages, table=table.data_ptr(), held=held.data_ptr(), slots=slots.data_ptr(), first=first.data_ptr())
        size = L.b200_kv16_attention_workspace(C.byref(c), heads, max_rows)
        assert (size == 0) == (n == 2)
        work = torch.empty(size + 32, dtype=torch.uint8, device="cuda")
        attend = lambda at, bytes_: L.b200_kv16_attention(C.byref(c), 2, q.data_ptr(), heads * 64, 64, heads, 1.0, 0, 0, max_rows, out.data_ptr(), at, bytes_)  # noqa: E731
        for _ in range(20):
            assert attend(work.data_ptr() if size else None, size) == 0, _lib.last_error()
            work.fill_(0x55)
            assert (work == 0x55).all()
        assert (out == 7).all()
        if size:
            assert attend(work.data_ptr(), size - 1) and "workspace" in _lib.last_error()
            assert attend(work.data_ptr() + 8, size) and "16 bytes" in _lib.last_error()
            assert attend(None, size) and "workspace" in _lib.last_error()


@pytest.mark.parametrize("group", [4, 5])
def test_a_wait_that_runs_out_is_told(group):
    """queries that never come, as boxes or gathered by warps: the kernel gives up, frees what it holds and says so, whichever call comes next; after it all is as before"""
    L = _lib.lib()
    c = Case([300, 5], [64, 1], kv=2, hd=128, dtype=BF16)
    c.fill()
    q = c.randn(c.rows, 2 * group, 128).bfloat16()
    attend = lambda most=64: serve.kv16_attention(q, *c.args(), slots=c.slots, max_rows=most)  # noqa: E731
    right, few = attend(), attend(1)
    k = c.randn(c.rows, 2, 128).bfloat16()
    refs, pool = torch.ones(c.pages, dtype=torch.int32, device="cuda"), c.pool.clone()
    one = torch.zeros(1, device="cuda")
    calls = [lambda: serve.kv16_append(*c.args(), k, k, c.slots), attend, lambda: attend(1), lambda: serve.pages_plan(c.table, c.held, refs, ints([1]), 16, 1, c.slots[:1]),
             lambda: serve.pages_trim(c.table, c.held, refs, 16, c.slots), lambda: serve.verify(torch.zeros(1, 10, device="cuda"), ints([0]), ints([0, 1]), one, one), serve.kv4_status]
    try:
        for call in calls:
            L.b200_kv4_drill(64)
            attend()
            L.b200_kv4_drill(0)
            torch.cuda.synchronize()
            with pytest.raises(_lib.B200Error, match="ran out"):
                call()
            assert torch.equal(c.pool, pool)
            serve.kv4_status()
            assert torch.equal(attend(), right) and torch.equal(attend(1), few)
    finally:
        L.b200_kv4_drill(0)


def test_a_server_that_drafts_ahead():
    """prompts, then tokens with drafts under a window with sinks, two answers to one prompt, conversations that end, pages moved between: the tokens of greedy requests are those that one token at a
    time would give, what each slot sees is what its own tokens say, and all pages come back"""
    heads, kv, hd, page, vocab, slots, window, sinks = 8, 2, 64, 16, 200, 5, 40, 5
    r = random.Random(7)
    gen = torch.Generator(device="cuda").manual_seed(7)
    embed = torch.randn(vocab, (heads + 2 * kv) * hd, generator=gen, device="cuda").bfloat16()
    wq = torch.randn(heads * hd, vocab, generator=gen, device="cuda")
    pool = serve.kv16_pool(80, page, kv, hd)
    table, held, refs = ints([[-1] * 40] * slots), ints([0] * slots), ints([0] * 80)
    said = {s: [] for s in range(slots)}                                # tokens that are certain, the last of them not in the cache yet

    def truth(tokens):
        """logits behind the last of `tokens`, in 64 bits, and how far off the step's may be"""
        row = embed[torch.tensor(tokens, device="cuda")].view(len(tokens), -1, hd).double().cpu().numpy()
        K, V = (row[:, heads + i * kv:heads + (i + 1) * kv].transpose(1, 0, 2) for i in (0, 1))
        o, e = oracle.attention(row[-1:, :heads], [(K, V, np.ones(len(tokens), bool))], [len(tokens) - 1], [0, 1], window, sinks, hd ** -0.5, 2.0 ** -7)
        e = e + 2.0 ** -8 * (np.abs(o) + e)
        w = wq.double().cpu().numpy()
        return o.reshape(-1) @ w, e.reshape(-1) @ np.abs(w) + 1e-4

    def advance(new):
        ids, counts = list(new), [len(t) for t in new.values()]
        on, tokens = ints(ids), torch.tensor(sum(new.values(), []), device="cuda", dtype=torch.int32)
        first, positions, places, status = serve.pages_plan(table, held, refs, ints(counts), page, len(tokens), on)
        assert status.item() == 0
        row = embed[tokens.long()].view(len(tokens), -1, hd)
        serve.kv16_append(pool[0], table, held, first, row[:, heads:heads + kv], row[:, heads + kv:], on)
        assert torch.equal(pool[0, places // page, 0, :, places % page], row[:, heads:heads + kv])
        x = serve.kv16_attention(row[:, :heads], pool[0], table, held, first, on, window=window, sinks=sinks, max_rows=max(counts))
        return on, tokens, first, x.flatten(1).float() @ wq

    for s, n in ((0, 80), (2, 30), (4, 3)):
        said[s] = [r.randrange(vocab) for _ in range(n)]
    on, tokens, first, logits = advance({s: said[s] for s in (0, 2, 4)})
    held[on.long()] += first.diff()
    for s, t in zip((0, 2, 4), logits[first[1:].long() - 1].argmax(1).tolist()):
        said[s].append(t)
    taken = 0
    for turn in range(30):
        live = [s for s in range(slots) if said[s]]
        new = {}
        for s in live:                                                  # what the likeliest following tokens are, sometimes another
            drafts = []
            for _ in range(r.randrange(0, 5)):
                best, _ = truth((said[s] + drafts)[-400:] if len(said[s]) < 400 else said[s] + drafts)
                drafts.append(int(np.argmax(best)) if r.random() < 0.7 else r.randrange(vocab))
            new[s] = [said[s][-1]] + drafts
        on, tokens, first, logits = advance(new)
        zeros = torch.zeros(len(tokens), device="cuda")
        u = torch.rand(len(tokens), generator=gen, device="cuda")
        gained, out, _ = serve.verify(logits, tokens, first, u, u, temperature=zeros)
        for i, s in enumerate(live):
            a, n = int(first[i]), int(gained[i])
            got = out[a:a + n].tolist()
            assert (out[a + n:int(first[i + 1])] == -1).all()
            for t in got:
                best, room = truth(said[s])
                assert best[t] + room[t] >= (best - room).max(), (turn, s)                # the largest, as far as roundings tell
                said[s].append(t)
            assert got[:-1] == new[s][1:n]
            taken += n - 1
        held.index_add_(0, on.long(), gained)
        serve.pages_trim(table, held, refs, page, on, window, sinks)
        assert all(held[s].item() == len(said[s]) - 1 for s in live)
        for s in live:                                                  # no more pages than the window, the sinks and their edges need
            assert int((table[s] >= 0).sum()) <= window // page + 2 + 1
        if turn == 2:                                                   # two answers to one conversation, whose first pages are away
            assert (table[0, 1:2] == -1).all() and serve.pages_fork(pool, table, held, refs, ints([0]), ints([1])).item() == 0
            said[1] = list(said[0])
        if turn in (9, 20):
            gone = {9: 2, 20: 1}[turn]
            serve.pages_free(table, held, refs, ints([gone]))
            said[gone] = []
            n = serve.pages_compact(pool, table, refs).item()
            assert n == int((refs > 0).sum()) and not refs[n:].any()
    assert taken > 30
    serve.pages_free(table, held, refs, ints(list(range(slots))))
    assert not refs.any() and (table == -1).all() and not held.any()


def test_a_wide_vocabulary_of_drafts():
    """2^18 logits, as many parts and as long slices as there are, with a drafter's distribution or without"""
    for drafter in (False, True):
        for kinds in ([dict()], [dict(top_k=50)], [dict(top_p=0.9)], [dict(top_k=5000, top_p=0.99, temperature=2.0)]):
            assert_verifies(*rows_to_verify(5, 1 << 18, [3, 2], BF16, kinds, drafter))
