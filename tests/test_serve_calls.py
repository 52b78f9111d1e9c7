"""Calls of booster_b200.serve beside those of tests/test_serve.py that need no GPU."""
import re

import pytest

from booster_b200 import _lib, serve


def test_status_without_calls():
    """nothing has run out where nothing has run; a device that cannot be is refused"""
    L = _lib.lib()
    assert L.b200_kv4_status(0) == 0
    serve.kv4_status(0)
    for device in (-1, 64):
        assert L.b200_kv4_status(device) != 0 and re.search("no such device", _lib.last_error())
        with pytest.raises(_lib.B200Error, match="no such device"):
            serve.kv4_status(device)


def test_pools_that_no_call_would_take():
    for page_tokens, head_dim in ((48, 64), (0, 64), (8, 64), (2048, 128), (16, 32), (16, 96)):
        with pytest.raises(ValueError, match="kv4_pool"):
            serve.kv4_pool(2, page_tokens, 1, head_dim, device="cpu")
    assert serve.kv4_pool(2, 1024, 3, 128, device="cpu").shape == (1, 2, 3, 64, 2304)
