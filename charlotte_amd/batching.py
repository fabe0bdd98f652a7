"""Requests of any lengths served together by a small synthetic model: the
products of charlotte_amd.matmul and, of charlotte_amd.serving, what runs
between them for a step of several requests, as a program would run them.

    python -m charlotte_amd.batching [--requests 40] [--together 16] [--pages 400] [--temperature 0.8] ...

A step has a token of every request that is generating and blocks of the
prompts of those that came last. page_plan gives the new tokens pages and every
row its slot and position; then, for each layer, queries, keys and values in one
product, their norms and rotation, the keys and values written into the pool's
pages, attention over them, and the products after it, the sums of the residual
stream and the norms before each product in one pass between them; then the head
for the requests whose prompt is read, and a token drawn for each by its own
settings. Requests end and others take their places between steps; where the
pool has no pages left, the request that came last gives its own back and waits for another's end.

torch holds the memory. It brings a HIP runtime of its own, so a process imports
torch (or this module) before the rest.
"""

import argparse
import collections
import time
from dataclasses import dataclass, field

import numpy as np
import torch

from charlotte_amd import matmul as mm
from charlotte_amd import serving as sv
from charlotte_amd import speculative as sp


@dataclass
class Request:
    prompt: list
    tokens: int                # to generate
    temperature: float = 0.0
    top_k: int = 0
    top_p: float = 1.0
    min_p: float = 0.0
    seed: int = 0
    taken: list = field(default_factory=list)
    chances: list = field(default_factory=list)
    failed: bool = False       # its logits had no number: it ended with the tokens before

    def __post_init__(self):
        self.random = np.random.default_rng(self.seed)

    def line(self):
        """All that the pool is to hold before the next token: what is read after a request had to wait."""
        return self.prompt + self.taken


class Batch:
    """Up to `together` requests at once over pools of `pages` pages, steps of up to `rows` tokens."""

    def __init__(self, model, together=16, pages=256, page_tokens=32, rows=256, longest=4096, cache_type=mm.TensorType.Q8_0):
        c, ctx, device = model.config, model.ctx, model.device
        if longest > model.cosines.shape[0]:
            raise ValueError(f"requests of {longest} tokens, past the rotation's tables of {model.cosines.shape[0]} positions")
        if rows < together:
            raise ValueError(f"steps of {rows} rows for {together} requests")
        self.model, self.ctx, self.together, self.rows, self.longest, self.page_tokens = model, ctx, together, rows, longest, page_tokens
        self.pages, self.device = pages, device
        self.waiting, self.active, self.finished = collections.deque(), [None] * together, []
        self.crowded = False                          # none is taken in until one ends
        self.read = np.zeros(together, np.int64)      # tokens of each that the pool holds
        self.came = np.zeros(together, np.int64)      # when each came
        self.steps = self.arrivals = 0

        def room(*shape, dtype=torch.float32):
            return torch.zeros(shape, dtype=dtype, device=device)

        stride = -(-longest // page_tokens)
        words = dict(dtype=torch.int32)
        self.past, self.counts, self.held, self.granted = (room(together, **words) for _ in range(4))
        self.table = room(together, stride, **words)
        self.free_pages, self.free_count = torch.arange(pages, device=device, **words), torch.tensor([pages], device=device, **words)
        self.starts = room(together + 1, **words)
        self.ids, self.slots, self.positions = (room(rows, **words) for _ in range(3))
        self.hidden, self.normed, self.product = (room(rows, c.hidden) for _ in range(3))
        self.q, self.k, self.v = (room(rows, n * c.head_dim) for n in (c.heads, c.kv_heads, c.kv_heads))
        self.mixed, self.gated = room(rows, c.heads * c.head_dim), room(rows, c.feed_forward)
        self.last, self.logits = room(together, c.hidden), room(together, c.vocabulary)
        self.tokens, self.chances = room(together, **words), room(together)
        self.settings = {n: room(together, dtype=torch.int32 if n == "top_ks" else torch.float32)
                         for n in ("temperatures", "top_ks", "top_ps", "min_ps", "uniforms")}
        self.pools = [sv.PagePool(ctx, cache_type, pages, page_tokens, c.kv_heads, c.head_dim) for _ in model.layers]
        need = max(sv.paged_attention_workspace_bytes(ctx, self.pools[0], c.heads, rows),
                   sv.sample_workspace_bytes(together, c.vocabulary))
        self.workspace = room(need, dtype=torch.uint8)
        work = {"workspace": self.workspace.data_ptr(), "workspace_bytes": need}

        M, p = mm.Member, torch.Tensor.data_ptr
        self.plan = sv.PagePlan(together, rows, pages, page_tokens, p(self.past), p(self.counts), p(self.table), stride, p(self.held),
                                p(self.held), p(self.free_pages), p(self.free_count), p(self.free_count), p(self.starts),
                                p(self.granted), p(self.slots), p(self.positions))
        norm = dict(residual=p(self.hidden), normed=p(self.normed), epsilon=c.epsilon)
        self.first = sv.ResidualNorm(c.hidden, weight=p(model.layers[0].before), **norm)
        self.calls = []
        for i, (layer, pool) in enumerate(zip(model.layers, self.pools)):
            following = model.layers[i + 1].before if i + 1 < len(model.layers) else model.final
            self.calls.append((
                mm.MatmulLaunch([M(layer.q), M(layer.k), M(layer.v)], p(self.normed), [p(self.q), p(self.k), p(self.v)],
                                epilogue=mm.Epilogue.QKV),
                sv.HeadNormRope([sv.Heads(p(self.q), p(self.q), c.heads, p(layer.q_norm)),
                                 sv.Heads(p(self.k), p(self.k), c.kv_heads, p(layer.k_norm))],
                                c.head_dim, c.epsilon, sv.Rope.Halves, cosines=p(model.cosines), sines=p(model.sines),
                                table_rows=model.cosines.shape[0], positions=p(self.positions)),
                pool,
                sv.PagedAttention(pool, p(self.q), p(self.mixed), c.heads, c.head_dim ** -0.5, together, rows, p(self.past),
                                  p(self.granted), p(self.starts), p(self.table), stride, **work),
                mm.MatmulLaunch([M(layer.o)], p(self.mixed), [p(self.product)]),
                sv.ResidualNorm(c.hidden, branch=p(self.product), residual_out=p(self.hidden), weight=p(layer.after), **norm),
                mm.MatmulLaunch([M(layer.gate), M(layer.up)], p(self.normed), [p(self.gated)], epilogue=mm.Epilogue.GatedActivation),
                mm.MatmulLaunch([M(layer.down)], p(self.gated), [p(self.product)]),
                sv.ResidualNorm(c.hidden, branch=p(self.product), residual_out=p(self.hidden), weight=p(following), **norm)))
        self.head = mm.MatmulLaunch([M(model.table)], p(self.last), [p(self.logits)])
        s = {n: p(t) for n, t in self.settings.items()}
        self.draw = sv.Sample(p(self.logits), p(self.tokens), together, c.vocabulary, chances=p(self.chances), **s, **work)

    def add(self, request):
        if len(request.prompt) + request.tokens > self.longest:
            raise ValueError(f"a request of {len(request.prompt)} + {request.tokens} tokens, past the longest of {self.longest}")
        if -(-(len(request.prompt) + request.tokens) // self.page_tokens) > self.pages:
            raise ValueError("a request that the pool does not hold by itself")
        if not request.prompt:
            raise ValueError("a request without a prompt")
        if len(request.taken) >= request.tokens:
            raise ValueError(f"a request of {request.tokens} tokens, of which it has {len(request.taken)}")
        if min(request.prompt) < 0 or max(request.prompt) >= self.model.config.vocabulary:
            raise ValueError(f"a prompt with a token past the vocabulary of {self.model.config.vocabulary}")
        self.waiting.append(request)

    def _layers(self, rows, most, stream):
        ctx = self.ctx
        mm.gather(ctx, self.model.table, self.ids.data_ptr(), rows, self.hidden.data_ptr(), stream=stream)
        sv.residual_norm(ctx, self.first, rows, stream=stream)
        for qkv, turn, pool, attend, out, middle, gated, down, end in self.calls:
            if attend.most != most:
                attend.most = most
            mm.launch(ctx, qkv, rows, stream=stream)
            sv.head_norm_rope(ctx, turn, rows, stream=stream)
            pool.append(self.k.data_ptr(), self.v.data_ptr(), self.slots.data_ptr(), rows, stream=stream)
            sv.paged_attention(ctx, attend, stream=stream)
            mm.launch(ctx, out, rows, stream=stream)
            sv.residual_norm(ctx, middle, rows, stream=stream)
            mm.launch(ctx, gated, rows, stream=stream)
            mm.launch(ctx, down, rows, stream=stream)
            sv.residual_norm(ctx, end, rows, stream=stream)

    def step(self):
        """A step of whatever is there; whether something was."""
        for r, request in enumerate(self.active):
            if request is None and self.waiting and not self.crowded:
                self.active[r], self.read[r], self.came[r] = self.waiting.popleft(), 0, self.arrivals
                self.arrivals += 1
        here = [r for r, request in enumerate(self.active) if request is not None]
        # a token of each, then the prompts' blocks in the order in which they came
        counts, left = np.zeros(self.together, np.int64), self.rows - len(here)
        counts[here] = 1
        for r in sorted(here, key=lambda r: self.came[r]):
            more = min(left, len(self.active[r].line()) - self.read[r] - 1)
            counts[r] += more
            left -= more
        rows = int(counts.sum())
        if rows == 0 and not self.held.any():
            return False
        ids = [t for r in here for t in self.active[r].line()[self.read[r]:self.read[r] + counts[r]]]
        self.ids[:rows] = torch.tensor(ids, dtype=torch.int32)
        self.past.copy_(torch.tensor(self.read, dtype=torch.int32))
        self.counts.copy_(torch.tensor(counts, dtype=torch.int32))
        stream = torch.cuda.current_stream().cuda_stream
        sv.page_plan(self.ctx, self.plan, stream=stream)
        if rows == 0:  # the last ended: their pages have gone back
            return False
        self._layers(rows, int(counts.max()), stream)
        # the requests whose line is read draw their next token
        drawing = [r for r in here if self.read[r] + counts[r] == len(self.active[r].line())]
        if drawing:
            n, active = len(drawing), [self.active[r] for r in drawing]
            rows_of = torch.tensor(np.cumsum(counts)[drawing] - 1, device=self.device)
            torch.index_select(self.normed, 0, rows_of, out=self.last[:n])
            given = {"temperatures": [x.temperature for x in active], "top_ks": [x.top_k for x in active],
                     "top_ps": [x.top_p for x in active], "min_ps": [x.min_p for x in active],
                     "uniforms": [x.random.random(dtype=np.float32) for x in active]}
            for name, values in given.items():
                self.settings[name][:n] = torch.tensor(np.array(values), dtype=self.settings[name].dtype)
            mm.launch(self.ctx, self.head, n, stream=stream)
            self.draw.rows = n
            sv.sample(self.ctx, self.draw, stream=stream)
        granted, tokens, chances = (t.cpu().numpy() for t in (self.granted, self.tokens, self.chances))
        for at, r in enumerate(drawing):
            if granted[r] and tokens[at] < 0:  # a row of NaNs and -inf
                self.active[r].failed = True
            elif granted[r]:
                self.active[r].taken.append(int(tokens[at]))
                self.active[r].chances.append(float(chances[at]))
            else:
                self.active[r].random = _before(self.active[r])
        self.read += granted
        self.steps += 1
        done = [r for r in here if self.active[r].failed or len(self.active[r].taken) >= self.active[r].tokens]
        for r in done:
            self.finished.append(self.active[r])
            self.active[r], self.read[r], self.crowded = None, 0, False
        if not done and any(counts[r] and not granted[r] for r in here):
            # no pages: the last that came gives its own back, and waits until another ends
            r = max(here, key=lambda r: self.came[r])
            self.waiting.appendleft(self.active[r])
            self.active[r], self.read[r], self.crowded = None, 0, True
        return True

    def run(self, requests):
        """Each request's tokens, in `taken`, with their chances; in the order in which they end."""
        self.finished, self.crowded = [], False
        for request in requests:
            self.add(request)
        while self.step():
            pass
        return self.finished

    def free(self):
        for pool in self.pools:
            pool.free()


def _before(request):
    """A request's random numbers as they were before the last, which it did not use."""
    again = np.random.default_rng(request.seed)
    for _ in request.taken:
        again.random(dtype=np.float32)
    return again


def main():
    parser = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    parser.add_argument("--requests", type=int, default=40)
    parser.add_argument("--together", type=int, default=16)
    parser.add_argument("--prompt", type=int, default=300, help="the longest prompt")
    parser.add_argument("--tokens", type=int, default=64)
    parser.add_argument("--pages", type=int, default=400)
    parser.add_argument("--page-tokens", type=int, default=32)
    parser.add_argument("--rows", type=int, default=256)
    parser.add_argument("--temperature", type=float, default=0.8)
    parser.add_argument("--top-k", type=int, default=50)
    parser.add_argument("--top-p", type=float, default=0.95)
    parser.add_argument("--min-p", type=float, default=0.0)
    parser.add_argument("--cache", choices=["q8_0", "q4_0", "f16"], default="q8_0")
    a = parser.parse_args()
    with mm.Context(0) as ctx:
        model = sp.Model(ctx)
        rng = np.random.default_rng(0)
        batch = Batch(model, a.together, a.pages, a.page_tokens, a.rows, cache_type=mm.TensorType[a.cache.upper()])

        def requests(n):
            return [Request(rng.integers(0, model.config.vocabulary, rng.integers(1, a.prompt + 1)).tolist(), a.tokens, a.temperature,
                            a.top_k, a.top_p, a.min_p, seed=i) for i in range(n)]

        batch.run(requests(2))  # the kernels loaded
        torch.cuda.synchronize()
        before, start = batch.steps, time.perf_counter()
        done = batch.run(requests(a.requests))
        torch.cuda.synchronize()
        took = time.perf_counter() - start
        print(f"{len(done)} requests, {sum(len(x.prompt) for x in done)} tokens read and {sum(len(x.taken) for x in done)} generated "
              f"in {batch.steps - before} steps: {sum(len(x.taken) for x in done) / took:.0f} tokens/s")
        batch.free()


if __name__ == "__main__":
    main()
