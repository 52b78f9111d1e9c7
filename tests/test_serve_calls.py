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
