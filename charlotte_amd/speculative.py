"""Speculative decoding of a small synthetic model: the products of
charlotte_amd.matmul and the steps between them (charlotte_amd.serving) as a
program would run them.

    python -m charlotte_amd.speculative [--depth 4] [--width 2] [--temperature 0.8] [--cache q8_0] ...

A step of `tokens` nodes a sequence is, for each layer: queries, keys and values
in one product, their norms and rotation, the keys and values appended to the
quantized cache, attention over it, and the products after it; then the head,
its probabilities, and their verification. Drafts come of the model's own first
layers, as a chain (drawn from their probabilities) or, with a width, as a tree
(the likeliest first tokens, each continued with the likeliest); the accepted
path's slots are moved together in both caches. Past lengths stay on the device.

torch holds the memory, does the layers' norms and the sums of the residual
stream (charlotte_amd/batching.py has them of the library) and finds the drafts'
largest logits. It brings a HIP runtime of its own, so a process imports torch
(or this module) before the rest.
"""

import argparse
import time
from dataclasses import dataclass

import numpy as np
import torch

from charlotte_amd import matmul as mm
from charlotte_amd import serving as sv
from charlotte_amd import synthetic


@dataclass(frozen=True)
class Config:
    vocabulary: int = 2048
    hidden: int = 512
    layers: int = 8
    draft_layers: int = 2
    heads: int = 8
    kv_heads: int = 4
    head_dim: int = 64
    feed_forward: int = 1024
    weights: mm.TensorType = mm.TensorType.Q4_0
    epsilon: float = 1e-6


class Layer:
    def __init__(self, ctx, c, rng, device):
        def weight(rows, columns):
            return mm.Weight(ctx, c.weights, rows, columns, synthetic.weight(rng, int(c.weights), rows, columns))

        def norm(n):
            return torch.tensor(1 + 0.1 * rng.standard_normal(n), dtype=torch.float32, device=device)

        self.q, self.k, self.v = (weight(n * c.head_dim, c.hidden) for n in (c.heads, c.kv_heads, c.kv_heads))
        self.o = weight(c.hidden, c.heads * c.head_dim)
        self.gate, self.up = weight(c.feed_forward, c.hidden), weight(c.feed_forward, c.hidden)
        self.down = weight(c.hidden, c.feed_forward)
        self.before, self.after = norm(c.hidden), norm(c.hidden)
        self.q_norm, self.k_norm = norm(c.head_dim), norm(c.head_dim)


class Model:
    """Random weights from a seed, on device 0."""

    def __init__(self, ctx, config=Config(), seed=0, positions=4096):
        rng = np.random.default_rng(seed)
        self.ctx, self.config, self.device = ctx, config, torch.device("cuda:0")
        self.table = mm.Weight(ctx, config.weights, config.vocabulary, config.hidden,
                               synthetic.weight(rng, int(config.weights), config.vocabulary, config.hidden))
        self.layers = [Layer(ctx, config, rng, self.device) for _ in range(config.layers)]
        self.final = torch.ones(config.hidden, device=self.device)
        cosines, sines = sv.rope_table(positions, config.head_dim)
        self.cosines, self.sines = (torch.tensor(t, device=self.device) for t in (cosines, sines))


class Decoder:
    """The model's first `layers` layers with caches of their own, for steps of up to `most` tokens a sequence."""

    def __init__(self, model, layers, sequences, capacity, most, cache_type):
        c, ctx, device = model.config, model.ctx, model.device
        if capacity > model.cosines.shape[0]:
            raise ValueError(f"a capacity of {capacity}, past the rotation's tables of {model.cosines.shape[0]} positions")
        most = min(most, capacity)
        self.model, self.ctx, self.sequences, self.most, self.capacity = model, ctx, sequences, most, capacity
        rows = sequences * most

        def room(*shape, dtype=torch.float32):
            return torch.zeros(shape, dtype=dtype, device=device)

        self.past = room(sequences, dtype=torch.int32)
        self.ids, self.positions = room(rows, dtype=torch.int32), room(rows, dtype=torch.int32)
        self.parents = room(rows, dtype=torch.int32)
        self.hidden, self.normed, self.product = (room(rows, c.hidden) for _ in range(3))
        self.q, self.k, self.v = (room(rows, n * c.head_dim) for n in (c.heads, c.kv_heads, c.kv_heads))
        self.mixed, self.gated = room(rows, c.heads * c.head_dim), room(rows, c.feed_forward)
        self.logits, self.probabilities = room(rows, c.vocabulary), room(rows, c.vocabulary)
        self.caches = [sv.Cache(ctx, cache_type, sequences, c.kv_heads, c.head_dim, capacity) for _ in range(layers)]
        need = max(sv.attention_workspace_bytes(ctx, self.caches[0], c.heads, most),
                   sv.probabilities_workspace_bytes(rows, c.vocabulary),
                   sv.verify_workspace_bytes(sequences, most, c.vocabulary))
        self.workspace = room(max(16, need), dtype=torch.uint8)
        self.room = {"workspace": self.workspace.data_ptr(), "workspace_bytes": need}

        M, p = mm.Member, torch.Tensor.data_ptr
        self.calls = []
        for layer, cache in zip(model.layers, self.caches):
            qkv = mm.MatmulLaunch([M(layer.q), M(layer.k), M(layer.v)], p(self.normed), [p(self.q), p(self.k), p(self.v)],
                                  epilogue=mm.Epilogue.QKV)
            turn = sv.HeadNormRope([sv.Heads(p(self.q), p(self.q), c.heads, p(layer.q_norm)),
                                    sv.Heads(p(self.k), p(self.k), c.kv_heads, p(layer.k_norm))],
                                   c.head_dim, c.epsilon, sv.Rope.Halves, cosines=p(model.cosines), sines=p(model.sines),
                                   table_rows=model.cosines.shape[0], positions=p(self.positions))
            attend = {tree: sv.Attention(cache, p(self.q), p(self.mixed), c.heads, c.head_dim ** -0.5, past=p(self.past),
                                         parents=p(self.parents) if tree else 0, **self.room) for tree in (False, True)}
            out = mm.MatmulLaunch([M(layer.o)], p(self.mixed), [p(self.product)])
            gated = mm.MatmulLaunch([M(layer.gate), M(layer.up)], p(self.normed), [p(self.gated)],
                                    epilogue=mm.Epilogue.GatedActivation)
            down = mm.MatmulLaunch([M(layer.down)], p(self.gated), [p(self.product)])
            self.calls.append((layer, cache, qkv, turn, attend, out, gated, down))
        self.head = mm.MatmulLaunch([M(model.table)], p(self.normed), [p(self.logits)])

    def _norm(self, rows, weight):
        x = self.hidden[:rows]
        torch.mul(x * torch.rsqrt(x.square().mean(-1, keepdim=True) + self.model.config.epsilon), weight,
                  out=self.normed[:rows])

    def step(self, nodes, parents=None, depths=None, head=True):
        """nodes [sequences, tokens] appended behind `past` (which stays) and, with `head`, their logits.

        parents [tokens] with depths, their distances from node 0: one tree's, the same in every sequence."""
        stream = torch.cuda.current_stream().cuda_stream
        tokens = nodes.shape[1]
        rows = self.sequences * tokens
        self.ids[:rows] = nodes.reshape(-1)
        depths = torch.arange(tokens, dtype=torch.int32, device=nodes.device) if depths is None else depths
        self.positions[:rows] = (self.past[:, None] + depths).reshape(-1)
        if parents is not None:
            self.parents[:rows] = parents.repeat(self.sequences)
        mm.gather(self.ctx, self.model.table, self.ids.data_ptr(), rows, self.hidden.data_ptr(), stream=stream)
        for layer, cache, qkv, turn, attend, out, gated, down in self.calls:
            self._norm(rows, layer.before)
            mm.launch(self.ctx, qkv, rows, stream=stream)
            sv.head_norm_rope(self.ctx, turn, rows, stream=stream)
            cache.append(self.k.data_ptr(), self.v.data_ptr(), self.past.data_ptr(), tokens, stream=stream)
            sv.attention(self.ctx, attend[parents is not None], tokens, stream=stream)
            mm.launch(self.ctx, out, rows, stream=stream)
            self.hidden[:rows] += self.product[:rows]
            self._norm(rows, layer.after)
            mm.launch(self.ctx, gated, rows, stream=stream)
            mm.launch(self.ctx, down, rows, stream=stream)
            self.hidden[:rows] += self.product[:rows]
        if head:
            self._norm(rows, self.model.final)
            mm.launch(self.ctx, self.head, rows, stream=stream)
            return self.logits[:rows].view(self.sequences, tokens, -1)

    def soften(self, tokens, temperature):
        """The last step's probabilities, [sequences * tokens, vocabulary]."""
        rows = self.sequences * tokens
        call = sv.Probabilities(self.logits.data_ptr(), self.probabilities.data_ptr(), rows, self.model.config.vocabulary,
                                temperature, **self.room)
        sv.probabilities(self.ctx, call, stream=torch.cuda.current_stream().cuda_stream)
        return self.probabilities[:rows]

    def verify(self, nodes, uniforms, draft=None, accepts=None, parents=None):
        """The step's nodes against the probabilities of `soften`: path, emitted [sequences, tokens] and count."""
        tokens = nodes.shape[1]
        ids, uniforms = nodes.to(torch.int32).contiguous(), uniforms.contiguous()
        path, emitted = torch.empty_like(ids), torch.empty_like(ids)
        count = torch.empty(self.sequences, dtype=torch.int32, device=ids.device)
        kept = [x.contiguous() for x in (draft, accepts) if x is not None]
        if parents is not None:
            parents = parents.repeat(self.sequences)
        call = sv.Verify(ids.data_ptr(), self.probabilities.data_ptr(), uniforms.data_ptr(), self.model.config.vocabulary,
                         path.data_ptr(), emitted.data_ptr(), count.data_ptr(), *(x.data_ptr() for x in kept),
                         parents=0 if parents is None else parents.data_ptr(), **self.room)
        sv.verify(self.ctx, call, self.sequences, tokens, stream=torch.cuda.current_stream().cuda_stream)
        return path, emitted, count

    def keep(self, path, count, moved):
        """`past` moved behind the accepted nodes, and with `moved` (a tree) their slots together first."""
        if moved:
            for cache in self.caches:
                cache.keep(self.past.data_ptr(), path.data_ptr(), count.data_ptr(), path.shape[1],
                           stream=torch.cuda.current_stream().cuda_stream)
        self.past += count

    def read(self, prompt):
        """A prompt [sequences, tokens] into the caches, in blocks."""
        if int(self.past.max()) + prompt.shape[1] > self.capacity:
            raise ValueError(f"a prompt of {prompt.shape[1]} tokens passes the capacity of {self.capacity}")
        for at in range(0, prompt.shape[1], self.most):
            block = prompt[:, at:at + self.most]
            self.step(block, head=False)
            self.past += block.shape[1]

    def free(self):
        for cache in self.caches:
            cache.free()


class Speculative:
    """A target and its draft, a chain of `depth` tokens or a tree of `width` such chains."""

    def __init__(self, model, sequences, capacity, depth, width=0, temperature=0.0, cache_type=mm.TensorType.Q8_0,
                 seed=0, block=64):
        self.nodes = 1 + depth * max(1, width)  # a round's
        most = max(block, self.nodes)
        c = model.config
        self.target = Decoder(model, c.layers, sequences, capacity, most, cache_type)
        self.draft = Decoder(model, c.draft_layers, sequences, capacity, most, cache_type)
        self.depth, self.width, self.temperature, self.sequences = depth, width, temperature, sequences
        self.generator = torch.Generator(device=model.device)
        self.generator.manual_seed(seed)
        levels = [(1 + level * width + b, level) for level in range(depth) for b in range(width)]
        parents = [-1] + [0 if level == 0 else node - width for node, level in levels]
        depths = [0] + [1 + level for _, level in levels]
        self.parents, self.depths = (torch.tensor(x, dtype=torch.int32, device=model.device) for x in (parents, depths))

    def _uniforms(self, *shape):
        return torch.rand(shape, generator=self.generator, device=self.target.past.device)

    def _chain(self, root):
        """The draft's tokens one after the other, each drawn from its probabilities, which verification needs."""
        nodes, rows, past = [root], [], self.draft.past.clone()
        for _ in range(self.depth):
            self.draft.step(nodes[-1])
            rows.append(self.draft.soften(1, self.temperature).clone())
            nodes.append(self.draft.verify(nodes[-1], self._uniforms(self.sequences, 1))[1])
            self.draft.past += 1
        self.draft.step(nodes[-1], head=False)  # its keys, should every token be accepted
        self.draft.past.copy_(past)
        return torch.cat(nodes, 1), torch.stack(rows, 1)

    def _tree(self, root):
        nodes = root
        for level in range(self.depth):
            n = nodes.shape[1]
            logits = self.draft.step(nodes, self.parents[:n], self.depths[:n])
            if level == 0:
                tokens = logits[:, 0].topk(self.width).indices
            else:
                tokens = logits[:, n - self.width:].argmax(-1)
            nodes = torch.cat([nodes, tokens.to(torch.int32)], 1)
        self.draft.step(nodes, self.parents, self.depths, head=False)
        return nodes

    def round(self, root):
        """From the last token taken [sequences, 1]: the tokens after it, [sequences, count], -1 past each count."""
        tree = self.width > 0
        if tree:
            nodes, draft = self._tree(root), None
            self.target.step(nodes, self.parents, self.depths)
        else:
            nodes, draft = self._chain(root)
            self.target.step(nodes)
        tokens = nodes.shape[1]
        self.target.soften(tokens, self.temperature)
        path, emitted, count = self.target.verify(
            nodes, self._uniforms(self.sequences, tokens), draft, None if tree else self._uniforms(self.sequences, tokens),
            self.parents if tree else None)
        self.target.keep(path, count, tree)
        self.draft.keep(path, count, tree)
        return emitted, count

    def generate(self, prompt, tokens):
        """At least `tokens` tokens after each prompt [sequences, length]; lists, and the number of rounds."""
        if prompt.shape[1] - 1 + self.nodes > self.target.capacity:
            raise ValueError(f"a prompt of {prompt.shape[1]} tokens and a round pass the capacity of {self.target.capacity}")
        for decoder in (self.target, self.draft):
            decoder.past.zero_()
            decoder.read(prompt[:, :-1])
        root = prompt[:, -1:].to(torch.int32)
        out, rounds = [[] for _ in range(self.sequences)], 0
        while min(map(len, out)) < tokens:
            if int(self.target.past.max()) + self.nodes > self.target.capacity:
                raise ValueError("the caches are full")
            emitted, count = self.round(root)
            root = emitted.gather(1, count[:, None].long() - 1)
            rounds += 1
            for line, taken, n in zip(out, emitted.tolist(), count.tolist()):
                line.extend(taken[:n])
        return out, rounds

    def free(self):
        self.target.free()
        self.draft.free()


def decode(model, prompt, tokens, temperature=0.0, cache_type=mm.TensorType.Q8_0, capacity=4096, seed=0, block=64):
    """The same without drafts: a token a step."""
    if prompt.shape[1] - 1 + tokens > capacity:
        raise ValueError(f"a prompt of {prompt.shape[1]} tokens and {tokens} after it pass the capacity of {capacity}")
    decoder = Decoder(model, model.config.layers, prompt.shape[0], capacity, block, cache_type)
    generator = torch.Generator(device=model.device)
    generator.manual_seed(seed)
    decoder.read(prompt[:, :-1])
    root, taken = prompt[:, -1:].to(torch.int32), []
    for _ in range(tokens):
        decoder.step(root)
        decoder.soften(1, temperature)
        uniforms = torch.rand(root.shape, generator=generator, device=model.device)
        path, root, count = decoder.verify(root, uniforms)
        decoder.keep(path, count, False)
        taken.append(root)
    out = torch.cat(taken, 1).tolist()
    decoder.free()
    return out


def main():
    parser = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    parser.add_argument("--prompt", type=int, default=300)
    parser.add_argument("--tokens", type=int, default=128)
    parser.add_argument("--sequences", type=int, default=1)
    parser.add_argument("--depth", type=int, default=4)
    parser.add_argument("--width", type=int, default=0, help="chains of a tree; 0: one chain, drawn")
    parser.add_argument("--temperature", type=float, default=0.0)
    parser.add_argument("--cache", choices=["q8_0", "q4_0", "f16"], default="q8_0")
    parser.add_argument("--capacity", type=int, default=4096)
    a = parser.parse_args()
    kind = mm.TensorType[a.cache.upper()]
    with mm.Context(0) as ctx:
        model = Model(ctx, positions=a.capacity)
        prompt = torch.randint(model.config.vocabulary, (a.sequences, a.prompt), device=model.device, dtype=torch.int32)
        pair = Speculative(model, a.sequences, a.capacity, a.depth, a.width, a.temperature, kind)
        pair.generate(prompt, 2 * (a.depth + 1))  # the kernels loaded
        torch.cuda.synchronize()
        start = time.perf_counter()
        out, rounds = pair.generate(prompt, a.tokens)
        torch.cuda.synchronize()
        took = time.perf_counter() - start
        start = time.perf_counter()
        plain = decode(model, prompt, a.tokens, a.temperature, kind, a.capacity)
        torch.cuda.synchronize()
        alone = time.perf_counter() - start
        made = sum(map(len, out))
        print(f"{made} tokens of {a.sequences} sequences in {rounds} rounds, {made / rounds / a.sequences:.2f} a round: "
              f"{made / took:.0f} tokens/s; a token a step {a.sequences * a.tokens / alone:.0f} tokens/s")
        if a.temperature == 0:
            same = all(x[:a.tokens] == y for x, y in zip(out, plain))
            print("the same tokens" if same else "tokens that differ")
        pair.free()


if __name__ == "__main__":
    main()
