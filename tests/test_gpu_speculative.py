"""The serving operators and the products run together: a small model's
speculative decoding (charlotte_amd/speculative.py), in a process of its own,
where torch and its HIP runtime are loaded before the library."""

import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("check", [["greedy", "Q8_0"], ["greedy", "Q4_0"], ["greedy", "F16"], ["itself"], ["prompts"]],
                         ids=" ".join)
def test_speculative_decoding(check):
    run = subprocess.run([sys.executable, "-u", "-m", "tests.support.speculative_checks", *check], cwd=ROOT, timeout=100,
                         stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    print(run.stdout, flush=True)
    assert run.returncode == 0 and run.stdout.endswith("passed\n")


def test_positions_past_the_default_tables():
    test_speculative_decoding(["long"])
