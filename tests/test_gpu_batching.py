"""The operators of a step over several requests and the products run together:
a small model serving requests (charlotte_amd/batching.py), in a process of its
own, where torch and its HIP runtime are loaded before the library."""

import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("check", [["greedy", "Q8_0"], ["greedy", "Q4_0"], ["greedy", "F16"], ["drawn"], ["refusals"]],
                         ids=" ".join)
def test_batching(check):
    run = subprocess.run([sys.executable, "-u", "-m", "tests.support.batching_checks", *check], cwd=ROOT, timeout=100,
                         stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    print(run.stdout, flush=True)
    assert run.returncode == 0 and run.stdout.endswith("passed\n")


@pytest.mark.parametrize("cache", ["Q8_0", "Q4_0", "F16"])
def test_a_request_without_numbers(cache):
    test_batching(["spoilt", cache])
