"""Checks of charlotte_amd/speculative.py, for a process that loads torch before
the library: python -m tests.support.speculative_checks NAME [arguments].
"""

import sys

import numpy as np
import torch

from charlotte_amd import matmul as mm
from charlotte_amd import speculative as sp

CONFIG = dict(vocabulary=1024, hidden=256, layers=3, draft_layers=1, heads=6, kv_heads=2, head_dim=64, feed_forward=512)


def _prompt(model, sequences, tokens, seed=0):
    rng = np.random.default_rng(seed)
    return torch.tensor(rng.integers(0, model.config.vocabulary, (sequences, tokens)), dtype=torch.int32,
                        device=model.device)


def greedy(ctx, cache):
    """At temperature zero drafts change no token."""
    model = sp.Model(ctx, sp.Config(**CONFIG), seed=4)
    for depth, width, sequences, prompt in ((3, 0, 1, 5), (4, 0, 2, 150), (2, 3, 1, 40), (3, 2, 2, 70), (2, 1, 1, 1)):
        print("greedy", cache, depth, width, sequences, prompt, flush=True)
        x = _prompt(model, sequences, prompt, seed=depth + width)
        pair = sp.Speculative(model, sequences, 512, depth, width, cache_type=mm.TensorType[cache])
        got, rounds = pair.generate(x, 40)
        pair.free()
        want = sp.decode(model, x, 40, cache_type=mm.TensorType[cache], capacity=512)
        assert [line[:40] for line in got] == want
        assert rounds <= 40


def itself(ctx):
    """A draft that is the target: every drafted token is accepted, but where f32's last bits part the two (the draft
    steps a token at a time, the target five)."""
    whole = sp.Model(ctx, sp.Config(**{**CONFIG, "draft_layers": CONFIG["layers"]}), seed=4)
    pair = sp.Speculative(whole, 2, 512, 4, temperature=0.9, seed=1)
    _, rounds = pair.generate(_prompt(whole, 2, 30, seed=9), 100)
    pair.free()
    print("itself", rounds, flush=True)
    assert rounds <= 22  # 20 with every token accepted


def prompts(ctx):
    """The logits after a prompt read token by token, in blocks and in one step."""
    model = sp.Model(ctx, sp.Config(**CONFIG), seed=4)
    x, logits = _prompt(model, 2, 130, seed=3), []
    for most in (1, 48, 130):
        decoder = sp.Decoder(model, model.config.layers, 2, 256, most, mm.TensorType.F16)
        for at in range(0, 130, most):
            block = x[:, at:at + most]
            last = decoder.step(block)[:, -1].clone()
            decoder.past += block.shape[1]
        logits.append(last)
        decoder.free()
        print("prompts", most, float((last - logits[0]).abs().max()), flush=True)
    size = logits[0].abs().max()
    # what a step adds in another order (1e-7 a layer) can turn the last bit of a binary16 key or value (2^-11)
    assert all(bool(torch.isfinite(y).all()) and (y - logits[0]).abs().max() <= 2e-3 * size for y in logits)


def long(ctx):
    """Positions past 4,096, up to the last slot; and one token more, refused."""
    capacity = 4200
    model = sp.Model(ctx, sp.Config(**CONFIG), seed=4, positions=capacity)
    x = _prompt(model, 1, capacity - 20, seed=5)
    want = sp.decode(model, x, 21, capacity=capacity)
    pair = sp.Speculative(model, 1, capacity, 2)
    got, _ = pair.generate(x, 18)  # a round of three tokens has to fit behind the last
    pair.free()
    print("long", want, got, flush=True)
    assert got[0][:18] == want[0][:18]
    decoder = sp.Decoder(model, model.config.layers, 1, capacity, 64, mm.TensorType.Q8_0)
    decoder.read(x)
    assert bool(torch.isfinite(decoder.step(x[:, -1:])).all())
    decoder.free()
    try:
        sp.decode(model, x, 22, capacity=capacity)
    except ValueError:
        return
    raise AssertionError("a step past the capacity")


if __name__ == "__main__":
    with mm.Context(0) as context:
        {"greedy": greedy, "itself": itself, "prompts": prompts, "long": long}[sys.argv[1]](context, *sys.argv[2:])
    print("passed")
