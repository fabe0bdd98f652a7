"""Checks of charlotte_amd/batching.py, for a process that loads torch before
the library: python -m tests.support.batching_checks NAME [arguments].
"""

import sys

import numpy as np
import torch

from charlotte_amd import batching as ba
from charlotte_amd import matmul as mm
from charlotte_amd import speculative as sp
from charlotte_amd import synthetic

CONFIG = dict(vocabulary=1024, hidden=256, layers=3, draft_layers=1, heads=6, kv_heads=2, head_dim=64, feed_forward=512)


def _requests(model, lengths, tokens, **settings):
    rng = np.random.default_rng(5)
    return [ba.Request(rng.integers(0, model.config.vocabulary, n).tolist(), tokens, seed=i, **settings)
            for i, n in enumerate(lengths)]


def _taken(batch, requests):
    batch.run(requests)
    assert all(r is None for r in batch.active) and not batch.waiting
    # every page has come back, once
    assert int(batch.free_count[0]) == batch.pages and not batch.held.any()
    assert sorted(batch.free_pages.tolist()) == list(range(batch.pages))
    return [r.taken for r in requests]


def greedy(ctx, cache):
    """At temperature zero each request's tokens are those that it has by itself over a contiguous cache."""
    model = sp.Model(ctx, sp.Config(**CONFIG), seed=4)
    lengths = [1, 70, 33, 200, 5, 32, 31, 150, 2, 64]
    batch = ba.Batch(model, together=4, pages=60, rows=96, longest=512, cache_type=mm.TensorType[cache])
    got = _taken(batch, _requests(model, lengths, 24))
    batch.free()
    for taken, request in zip(got, _requests(model, lengths, 24)):
        prompt = torch.tensor([request.prompt], dtype=torch.int32, device=model.device)
        want = sp.decode(model, prompt, 24, cache_type=mm.TensorType[cache], capacity=512)[0]
        print("greedy", cache, len(request.prompt), taken == want, flush=True)
        assert taken == want


def drawn(ctx):
    """Drawn tokens do not depend on what a request is served beside, nor on whether it had to wait for pages."""
    model = sp.Model(ctx, sp.Config(**CONFIG), seed=4)
    lengths, settings = [40, 3, 90, 17, 120, 60, 33, 8], dict(temperature=0.9, top_k=40, top_p=0.95, min_p=0.01)
    found = []
    for together, pages, rows, page_tokens in ((1, 40, 64, 32), (8, 60, 256, 32), (8, 8, 64, 32), (3, 4, 40, 64), (5, 20, 33, 96)):
        batch = ba.Batch(model, together, pages, page_tokens, rows, longest=256)
        requests = _requests(model, lengths, 40, **settings)
        found.append(_taken(batch, requests))
        assert all(0 < x <= 1 for r in requests for x in r.chances)
        print("drawn", together, pages, rows, page_tokens, batch.steps, flush=True)
        batch.free()
    assert all(len(x) == 40 for x in found[0])
    assert all(x == found[0] for x in found[1:])


def refusals(ctx):
    model = sp.Model(ctx, sp.Config(**CONFIG), seed=4)
    batch = ba.Batch(model, together=2, pages=3, rows=8, longest=128)
    for request in (ba.Request([1] * 100, 29), ba.Request([1] * 90, 20), ba.Request([], 3)):
        try:
            batch.add(request)
        except ValueError:
            continue
        raise AssertionError(request)
    batch.free()
    for together, rows, longest in ((4, 3, 128), (2, 8, 1 << 20)):
        try:
            ba.Batch(model, together=together, pages=3, rows=rows, longest=longest)
        except ValueError:
            continue
        raise AssertionError((together, rows, longest))


def spoilt(ctx, cache):
    """A request whose stream is not numbers ends as failed, without a token; those beside it are as they are without it."""
    c = sp.Config(**CONFIG)
    model = sp.Model(ctx, c, seed=4)
    rows = np.frombuffer(synthetic.weight(np.random.default_rng(4), int(c.weights), c.vocabulary, c.hidden), np.uint8).copy()
    blocks = rows.reshape(c.vocabulary, c.hidden // 32, -1)
    bad = 77
    blocks[bad, 3, :2] = np.array([0x7E00], "<u2").view(np.uint8)  # a block's scale, not a number
    model.table.free()
    model.table = mm.Weight(ctx, c.weights, c.vocabulary, c.hidden, rows.tobytes())
    found = []
    for with_it in (False, True):
        requests = _requests(model, [5, 90, 33, 64, 17, 2], 12, temperature=0.9, top_k=40)
        for r in requests:
            r.prompt = [bad + 1 if t == bad else t for t in r.prompt]
        requests.insert(3, ba.Request([5, 9, bad, 3] + [1] * 40, 12, temperature=0.9))
        requests.insert(1, ba.Request([bad], 12))
        fine = [r for r in requests if bad not in r.prompt]
        assert len(fine) == 6
        batch = ba.Batch(model, together=4, pages=14, rows=48, longest=256, cache_type=mm.TensorType[cache])
        _taken(batch, requests if with_it else fine)
        assert len(batch.finished) == (8 if with_it else 6)
        if with_it:
            assert all(r.failed and not r.taken and not r.chances for r in requests if bad in r.prompt)
        assert not any(r.failed for r in fine) and all(len(r.taken) == 12 for r in fine)
        found.append([r.taken for r in fine])
        batch.free()
    assert found[0] == found[1]


def main():
    name, arguments = sys.argv[1], sys.argv[2:]
    with mm.Context(0) as ctx:
        {"greedy": greedy, "drawn": drawn, "refusals": refusals, "spoilt": spoilt}[name](ctx, *arguments)
    print("passed")


if __name__ == "__main__":
    main()
