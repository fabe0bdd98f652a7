"""charlotte_amd/batching.py's bounds, on the CPU: a request that cannot be served is refused
as it is added. In a process of its own, where torch is loaded before the library."""

import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
START = """
import collections
import types
import torch
from charlotte_amd import batching as ba
from charlotte_amd import speculative as sp

batch = object.__new__(ba.Batch)
batch.model = types.SimpleNamespace(config=sp.Config(vocabulary=100))
batch.longest, batch.page_tokens, batch.pages, batch.waiting = 128, 32, 4, collections.deque()
batch.add(ba.Request([0, 99], 1))
"""


@pytest.mark.parametrize("request_,word", [
    # nothing to generate, or nothing left: its first step would end it, whatever it had read
    ("ba.Request([1], 0)", "0 tokens"), ("ba.Request([1], -3)", "-3 tokens"), ("ba.Request([1], 2, taken=[5, 6])", "2 tokens"),
    # tokens that the table has no row for: their rows of the stream would be another step's
    ("ba.Request([1, 100], 1)", "vocabulary"), ("ba.Request([-1], 1)", "vocabulary")])
def test_requests_that_cannot_be_served(request_, word):
    body = f"""
try:
    batch.add({request_})
except ValueError as e:
    assert {word!r} in str(e), e
    assert len(batch.waiting) == 1
    print("refused")
"""
    run = subprocess.run([sys.executable, "-c", START + body], cwd=ROOT, capture_output=True, text=True, timeout=120)
    assert run.returncode == 0 and run.stdout == "refused\n", (run.stdout, run.stderr)
