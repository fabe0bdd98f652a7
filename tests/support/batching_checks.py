"""Checks of charlotte_amd/batching.py, for a process that loads torch before
the library: python -m tests.support.batching_checks NAME [arguments].
"""

import sys

import numpy as np
import torch

from charlotte_amd import batching as ba
from charlotte_amd import matmul as mm
from charlotte_amd import speculative as sp

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


def main():
    name, arguments = sys.argv[1], sys.argv[2:]
    with mm.Context(0) as ctx:
        {"greedy": greedy, "drawn": drawn, "refusals": refusals}[name](ctx, *arguments)
    print("passed")


if __name__ == "__main__":
    main()
