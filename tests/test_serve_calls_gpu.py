"""Calls of booster_b200.serve and of its C entry points that a program may make beside those of tests/test_serve_gpu.py."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


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
