"""charlotte_amd/speculative.py's bounds, on the CPU: what does not fit is refused before
anything runs. In a process of its own, where torch is loaded before the library."""

import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
START = """
import types
import torch
from charlotte_amd import matmul as mm
from charlotte_amd import speculative as sp

def refused(call, word):
    try:
        call()
    except ValueError as e:
        assert word in str(e), e
        print("refused")

model = types.SimpleNamespace(ctx=None, config=sp.Config(), device="cpu", cosines=torch.zeros(100, 32), sines=torch.zeros(100, 32))
bare = object.__new__(sp.Decoder)
bare.model, bare.capacity, bare.most, bare.past = model, 100, 8, torch.tensor([40, 60])
bare.step = lambda *a, **k: print("a step")
"""


@pytest.mark.parametrize("body", [
    # slots whose positions the rotation's tables do not reach
    "refused(lambda: sp.Decoder(model, 1, 1, 101, 8, mm.TensorType.Q8_0), 'tables')",
    # a prompt behind what is there
    "refused(lambda: bare.read(torch.zeros((2, 41), dtype=torch.int32)), 'capacity')",
    # a prompt, and the tokens after it
    "refused(lambda: sp.decode(model, torch.zeros((1, 50), dtype=torch.int32), 52, capacity=100, block=8), 'capacity')",
    "pair = object.__new__(sp.Speculative); pair.target = pair.draft = bare; pair.sequences, pair.nodes = 2, 5; "
    "refused(lambda: pair.generate(torch.zeros((2, 97), dtype=torch.int32), 1), 'capacity')",
])
def test_what_does_not_fit_is_refused_before_a_step(body):
    run = subprocess.run([sys.executable, "-c", START + body], cwd=ROOT, timeout=300, stdout=subprocess.PIPE,
                         stderr=subprocess.PIPE, text=True)
    assert run.returncode == 0 and run.stdout == "refused\n", run.stdout + run.stderr[-2000:]


def test_a_prompt_that_fits_is_read():
    body = "bare.past = torch.tensor([40, 59]); bare.read(torch.zeros((2, 41), dtype=torch.int32)); print(bare.past.tolist())"
    run = subprocess.run([sys.executable, "-c", START + body], cwd=ROOT, timeout=300, stdout=subprocess.PIPE, text=True)
    assert run.stdout == "a step\n" * 6 + "[81, 100]\n"
