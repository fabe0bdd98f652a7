"""The operators between a step's products whose speed is measured: what a
decoding step with drafted tokens runs beside charlotte_amd.matmul, through
charlotte_amd.serving, and each in its plain form of elementary torch
operations.

A case's fields:
  kind      "heads": norms of queries and keys for each head and the position
            rotation, in one pass.
            "cache": keys and values written into a quantized cache, and the
            slots written read back as the values they stand for.
            "attention": a step's rows over the cache: one token, a chain of
            tokens (a prompt's block) or a tree of drafted ones.
            "probabilities": softmax of the head's logits at a temperature.
            "verify": drafted tokens against the target's probabilities from
            given uniform numbers: a chain with its draft's probabilities, or
            a tree by the target's own draws.
  sequences, tokens   a step's rows: tokens (nodes) of each sequence
  heads, kv_heads, dim   query heads, key heads, a head's values
  type      the cache's format;  past: cached tokens before the step
  tree      whether the step's tokens are a tree (else a chain)
Activations, probabilities and outputs are f32, as the products' are.
"""

import math

import torch

own = False

# Heads of models this repository names: query heads, key heads, values a head.
QWEN3_0_6B = {"heads": 16, "kv_heads": 8, "dim": 128}
LLAMA_3_2_1B = {"heads": 32, "kv_heads": 8, "dim": 64}
LLAMA_3_8B = {"heads": 32, "kv_heads": 8, "dim": 128}
GEMMA_3_1B = {"heads": 4, "kv_heads": 1, "dim": 256}

STORED = {"f16": 2.0, "q8_0": 34 / 32, "q4_0": 18 / 32}
UNITS = 1 << 44  # a draw's weights: probabilities in whole units of 2^-44
EPSILON = 1e-6


def listed():
    return [
        # One token of a small model, layer after layer: a launch's latency.
        {"name": "heads_1_token", "kind": "heads", "tokens": 1, "norm": True, "pairing": "halves", "rotated": 128,
         "strided": False, "positions": 4096, **QWEN3_0_6B},
        # A long prompt of a model without head norms, neighbours rotated, Q and
        # K read out of one fused buffer: bound by bytes.
        {"name": "heads_2048_tokens", "kind": "heads", "tokens": 2048, "norm": False, "pairing": "neighbours",
         "rotated": 128, "strided": True, "positions": 8192, **LLAMA_3_8B},
        # A few drafted tokens appended and read back.
        {"name": "cache_5_tokens_q8_0", "kind": "cache", "type": "q8_0", "sequences": 1, "tokens": 5, "past": 1019,
         **QWEN3_0_6B},
        # Two prompts' blocks written at an odd length, 4 bits a value.
        {"name": "cache_2048_tokens_q4_0", "kind": "cache", "type": "q4_0", "sequences": 2, "tokens": 2048, "past": 77,
         **LLAMA_3_8B},
        # One token over a short chat: a launch's latency again.
        {"name": "attention_1_over_911", "kind": "attention", "type": "q8_0", "sequences": 1, "tokens": 1, "past": 911,
         "tree": False, "window": 0, **QWEN3_0_6B},
        # One token over a long context: bound by the cache's bytes.
        {"name": "attention_1_over_65536", "kind": "attention", "type": "q8_0", "sequences": 1, "tokens": 1,
         "past": 65536, "tree": False, "window": 0, **LLAMA_3_8B},
        # A tree of drafted tokens over some thousand tokens, 4 bits a value.
        {"name": "attention_tree_21_over_8191", "kind": "attention", "type": "q4_0", "sequences": 1, "tokens": 21,
         "past": 8191, "tree": True, "window": 0, **LLAMA_3_2_1B},
        # The engine's prefill block, 512 tokens, late in a long prompt: compute-bound, the largest work.
        {"name": "attention_512_over_15873", "kind": "attention", "type": "q8_0", "sequences": 1, "tokens": 512,
         "past": 15873, "tree": False, "window": 0, **LLAMA_3_8B},
        # The head's logits of a chain of five drafted tokens and its root.
        {"name": "probabilities_6_rows", "kind": "probabilities", "rows": 6, "vocab": 151936, "temperature": 0.7},
        # The same for eight sequences' trees, the widest vocabulary here.
        {"name": "probabilities_168_rows", "kind": "probabilities", "rows": 168, "vocab": 262144, "temperature": 1.0},
        # Eight sequences' chains of up to five drafted tokens.
        {"name": "verify_chain_8x6", "kind": "verify", "tree": False, "sequences": 8, "tokens": 6, "vocab": 128256},
        # A tree of drafted tokens.
        {"name": "verify_tree_21", "kind": "verify", "tree": True, "sequences": 1, "tokens": 21, "vocab": 151936},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _shape(rng):
    """Heads: mostly those of models, some of other widths and group sizes."""
    if rng.random() < 0.6:
        return dict(rng.choice([QWEN3_0_6B, LLAMA_3_2_1B, LLAMA_3_8B, GEMMA_3_1B]))
    kv = rng.choice([1, 2, 3, 4, 5, 8])
    return {"heads": kv * rng.choice([1, 2, 3, 4, 5, 7, 8]), "kv_heads": kv, "dim": rng.choice([32, 64, 96, 128, 160, 192, 256])}


def draw(rng):
    """Another case of the ranges the listed ones stand for: 1 to 2,048 tokens
    a pass, caches of 0 to 65,536 tokens in each format, trees of 2 to 64
    nodes, 1 to 8 sequences, vocabularies of 16,384 to 262,144."""
    kind = rng.choices(["heads", "cache", "attention", "probabilities", "verify"], weights=[3, 3, 7, 2, 4])[0]
    if kind == "heads":
        shape = _shape(rng)
        rotated = shape["dim"] if rng.random() < 0.7 else rng.randrange(8, shape["dim"] + 1, 8)
        tokens = 1 if rng.random() < 0.3 else _log(rng, 2, 2048)
        return {"kind": kind, "tokens": tokens, "norm": rng.random() < 0.6, "pairing": rng.choice(["halves", "neighbours"]),
                "rotated": rotated, "strided": rng.random() < 0.4, "positions": _log(rng, tokens, 32768), **shape}
    if kind == "cache":
        shape = _shape(rng)
        sequences = rng.choice([1, 1, 2, 4, 8])
        tokens = 1 if rng.random() < 0.3 else _log(rng, 2, 4096 // sequences)
        return {"kind": kind, "type": rng.choice(["q8_0", "q4_0", "f16"]), "sequences": sequences, "tokens": tokens,
                "past": rng.choice([0, _log(rng, 1, 8192)]), **shape}
    if kind == "attention":
        shape = _shape(rng)
        tree, sequences, tokens = False, rng.choice([1, 1, 1, 2, 4, 8]), 1
        pick = rng.random()
        if pick < 0.35:
            tree, tokens = True, _log(rng, 2, 64)
        elif pick < 0.65:
            sequences, tokens = 1, _log(rng, 2, 512)
        most = min(65536 // sequences, int(512 * 15873 * 32 / (sequences * tokens * shape["heads"])))
        return {"kind": kind, "type": rng.choice(["q8_0", "q8_0", "q4_0", "f16"]), "sequences": sequences,
                "tokens": tokens, "past": rng.choice([0, *[_log(rng, 1, most)] * 9]), "tree": tree,
                "window": rng.choice([0, 0, 0, 512, _log(rng, 2, 4096)]), **shape}
    vocab = _log(rng, 16384, 262144)
    if kind == "probabilities":
        return {"kind": kind, "rows": _log(rng, 1, min(168, 44e6 / vocab)), "vocab": vocab,
                "temperature": rng.choice([0.0, 0.6, 0.7, 1.0, 1.3])}
    tree = rng.random() < 0.5
    sequences = rng.choice([1, 1, 2, 4, 8])
    return {"kind": kind, "tree": tree, "sequences": sequences, "vocab": vocab,
            "tokens": _log(rng, 2, max(2, min(64, int(12e6 / (vocab * sequences))))) if tree else rng.randint(1, 8)}


# ---- inputs ------------------------------------------------------------------


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def _uniform(g, *shape):
    return torch.rand(*shape, generator=g, device="cuda", dtype=torch.float32)


def _tree(g, sequences, tokens):
    """Random trees, node 0 the root: a node's parent is one of the up to eight nodes before it."""
    i = torch.arange(tokens, device="cuda")
    back = (_uniform(g, sequences, tokens) * i.clamp(max=8)).floor().long().clamp(min=0) + 1
    return (i - back).clamp(min=-1).to(torch.int32).contiguous()


def _keys_and_values(g, sequences, tokens, kv_heads, dim):
    """Keys with a few large channels and values, as layers make them: [sequences][tokens][kv_heads * dim]."""
    spread = 0.3 + 1.7 * _uniform(g, kv_heads * dim) ** 4
    return _normal(g, sequences, tokens, kv_heads * dim) * spread, _normal(g, sequences, tokens, kv_heads * dim) * 0.7


def _blocks(x):
    return x.reshape(*x.shape[:-1], x.shape[-1] // 32, 32)


def _quantize(x, format_):
    """A cache's codes and scales for values x [..., dim]: blocks of 32, as the cache's formats are defined."""
    b = _blocks(x)
    if format_ == "f16":
        codes = b.half()
        scales = torch.ones(b.shape[:-1], device=b.device, dtype=torch.float16)
        bad = ~torch.isfinite(codes).all(-1)
        return codes.masked_fill(bad[..., None], 0), scales.masked_fill(bad, float("nan"))
    largest, at = b.abs().max(-1, keepdim=True)
    d = (largest / 127).half() if format_ == "q8_0" else (b.gather(-1, at) / -8).half()
    low, high = (-127, 127) if format_ == "q8_0" else (-8, 7)
    step = d.float()
    codes = torch.where(step == 0, torch.zeros_like(b), torch.round(b / step)).clamp(low, high)
    bad = ~torch.isfinite(step) | ~torch.isfinite(b).all(-1, keepdim=True)
    return (codes.masked_fill(bad, 0).to(torch.int8), d.masked_fill(bad, float("nan")).squeeze(-1))


def _values(codes, scales):
    """The f32 values that codes and scales stand for, [..., dim]."""
    return (codes.float() * scales.float()[..., None]).flatten(-2)


def _inputs(case, seed):
    """A case's data: from the seed alone, the same for the plain form, the kernels and the 64-bit results."""
    g, c, s = _generator(seed), case, {}
    kind = c["kind"]
    if kind == "heads":
        q_width, k_width = c["heads"] * c["dim"], c["kv_heads"] * c["dim"]
        if c["strided"]:  # the QKV product's rows in one buffer
            fused = _normal(g, c["tokens"], q_width + 2 * k_width) * 3
            s["q"], s["k"] = fused[:, :q_width], fused[:, q_width:q_width + k_width]
        else:
            s["q"], s["k"] = _normal(g, c["tokens"], q_width) * 3, _normal(g, c["tokens"], k_width) * 3
        if c["norm"]:
            s["q_weight"], s["k_weight"] = 1 + 0.3 * _normal(g, c["dim"]), 1 + 0.3 * _normal(g, c["dim"])
        pairs = c["rotated"] // 2
        angle = torch.arange(c["positions"], device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (
            -torch.arange(pairs, device="cuda", dtype=torch.float64) / pairs)
        s["cosines"], s["sines"] = angle.cos().float(), angle.sin().float()
        first = int(torch.randint(0, c["positions"] - c["tokens"] + 1, (1,), generator=g, device="cuda"))
        s["positions"] = torch.arange(first, first + c["tokens"], device="cuda", dtype=torch.int32)
    elif kind == "cache":
        s["k"], s["v"] = _keys_and_values(g, c["sequences"], c["tokens"], c["kv_heads"], c["dim"])
    elif kind == "attention":
        n = c["past"] + c["tokens"]
        k, v = _keys_and_values(g, c["sequences"], n, c["kv_heads"], c["dim"])
        split = (c["sequences"], n, c["kv_heads"], c["dim"])
        s["k_codes"], s["k_scales"] = _quantize(k.view(split), c["type"])
        s["v_codes"], s["v_scales"] = _quantize(v.view(split), c["type"])
        s["q"] = _normal(g, c["sequences"], c["tokens"], c["heads"] * c["dim"])
        # sequences of one batch are of different lengths
        shorter = (_uniform(g, c["sequences"]) * (c["past"] // 2 + 1)).floor().to(torch.int32)
        shorter[0] = 0
        s["past"] = c["past"] - shorter
        if c["tree"]:
            s["parents"] = _tree(g, c["sequences"], c["tokens"])
        s["scale"] = 1 / math.sqrt(c["dim"])
    elif kind == "probabilities":
        s["logits"] = _normal(g, c["rows"], c["vocab"]) * 2.5
        s["logits"][torch.arange(c["rows"]), torch.randint(0, c["vocab"], (c["rows"],), generator=g, device="cuda")] += 12
    else:
        n, shape = c["tokens"], (c["sequences"], c["tokens"], c["vocab"])
        logits = _normal(g, *shape) * 2.5
        logits[..., :64] += 9 * _uniform(g, c["sequences"], n, 64)
        s["target"] = torch.softmax(logits, -1)
        s["uniforms"] = _uniform(g, c["sequences"], n)
        # Drafted tokens: what a draft model near the target draws.
        near = torch.softmax(logits + 0.7 * _normal(g, *shape), -1)
        race = near / (-torch.log(_uniform(g, *shape).clamp(min=1e-30)))  # argmax: a draw from `near`
        drawn = race.argmax(-1).to(torch.int32)
        del race, logits
        s["node_tokens"] = torch.randint(0, c["vocab"], (c["sequences"], n), generator=g, device="cuda", dtype=torch.int32)
        if c["tree"]:
            s["parents"] = _tree(g, c["sequences"], n)
            up = s["parents"].long().clamp(min=0)
            likely = s["target"].gather(1, up[..., None].expand(shape)).topk(4, -1).indices
            rank = (_uniform(g, c["sequences"], n, 1) * 4).long().clamp(max=3)
            s["node_tokens"] = torch.where(s["parents"] < 0, s["node_tokens"], likely.gather(-1, rank)[..., 0].to(torch.int32))
        else:
            s["node_tokens"][:, 1:] = drawn[:, :-1]
            s["draft"] = near[:, :-1].contiguous()
            s["accepts"] = _uniform(g, c["sequences"], n)
            # chains of one batch are of different lengths
            s["lengths"] = (n - (_uniform(g, c["sequences"]) * ((n + 1) // 2)).floor()).to(torch.int32)
    return s


def prepare(case, seed):
    """The inputs and, for the kernels, the context, cache, buffers and descriptor that a serving loop keeps."""
    s = _inputs(case, seed)
    s["case"] = case
    if own:
        _prepare_own(case, s)
    return s


_CONTEXT = []


def _prepare_own(c, s):
    from charlotte_amd import matmul as mm
    from charlotte_amd import serving as sv

    if not _CONTEXT:
        _CONTEXT.append(mm.Context(0))
    ctx = s["ctx"] = _CONTEXT[0]
    kind = c["kind"]
    like = lambda *shape, dtype=torch.float32: torch.empty(*shape, device="cuda", dtype=dtype)  # noqa: E731

    def workspace(nbytes):
        s["workspace"] = like(max(nbytes, 16), dtype=torch.uint8)
        return {"workspace": s["workspace"].data_ptr(), "workspace_bytes": nbytes}

    def cache(capacity):
        types = {"q8_0": mm.TensorType.Q8_0, "q4_0": mm.TensorType.Q4_0, "f16": mm.TensorType.F16}
        s["cache"] = sv.Cache(ctx, types[c["type"]], c["sequences"], c["kv_heads"], c["dim"], capacity)
        return s["cache"]

    if kind == "heads":
        s["out"] = [like(c["tokens"], c[h] * c["dim"]) for h in ("heads", "kv_heads")]
        parts = [sv.Heads(s[n].data_ptr(), o.data_ptr(), c[h], weight=s[n + "_weight"].data_ptr() if c["norm"] else 0,
                          input_stride=s[n].stride(0))
                 for n, o, h in zip(("q", "k"), s["out"], ("heads", "kv_heads"))]
        s["call"] = sv.HeadNormRope(parts, c["dim"], epsilon=EPSILON, rope=sv.Rope[c["pairing"].capitalize()],
                                    rope_dims=c["rotated"], cosines=s["cosines"].data_ptr(), sines=s["sines"].data_ptr(),
                                    table_rows=c["positions"], positions=s["positions"].data_ptr())
    elif kind == "cache":
        cache(c["past"] + c["tokens"])
        s["past"] = torch.full((c["sequences"],), c["past"], device="cuda", dtype=torch.int32)
        s["out"] = [torch.empty_like(s["k"]), torch.empty_like(s["v"])]
    elif kind == "attention":
        n = c["past"] + c["tokens"]
        k, v = (_values(s[x + "_codes"], s[x + "_scales"]).flatten(2) for x in "kv")
        zero = torch.zeros(c["sequences"], device="cuda", dtype=torch.int32)
        stream = torch.cuda.current_stream().cuda_stream
        cache(n).append(k.data_ptr(), v.data_ptr(), zero.data_ptr(), n, stream=stream)
        torch.cuda.synchronize()
        for name in ("k_codes", "k_scales", "v_codes", "v_scales"):
            del s[name]
        s["out"] = torch.empty_like(s["q"])
        s["call"] = sv.Attention(s["cache"], s["q"].data_ptr(), s["out"].data_ptr(), c["heads"], s["scale"],
                                 past=s["past"].data_ptr(), longest=n, window=c["window"],
                                 parents=s["parents"].data_ptr() if c["tree"] else 0,
                                 **workspace(sv.attention_workspace_bytes(ctx, s["cache"], c["heads"], c["tokens"])))
    elif kind == "probabilities":
        s["out"] = torch.empty_like(s["logits"])
        s["call"] = sv.Probabilities(s["logits"].data_ptr(), s["out"].data_ptr(), c["rows"], c["vocab"], c["temperature"],
                                     **workspace(sv.probabilities_workspace_bytes(c["rows"], c["vocab"])))
    else:
        shape = (c["sequences"], c["tokens"])
        s["out"] = [like(*shape, dtype=torch.int32), like(*shape, dtype=torch.int32), like(c["sequences"], dtype=torch.int32)]
        more = {"parents": s["parents"].data_ptr()} if c["tree"] else {
            "draft": s["draft"].data_ptr(), "accepts": s["accepts"].data_ptr(), "lengths": s["lengths"].data_ptr()}
        s["call"] = sv.Verify(s["node_tokens"].data_ptr(), s["target"].data_ptr(), s["uniforms"].data_ptr(), c["vocab"],
                              path=s["out"][0].data_ptr(), emitted=s["out"][1].data_ptr(), count=s["out"][2].data_ptr(),
                              **more, **workspace(sv.verify_workspace_bytes(c["sequences"], c["tokens"], c["vocab"])))


# ---- one pass ------------------------------------------------------------------


def run(state):
    return _run_own(state) if own else _PLAIN[state["case"]["kind"]](state["case"], state)


def _run_own(s):
    from charlotte_amd import serving as sv

    c, ctx = s["case"], s["ctx"]
    kind, stream = c["kind"], torch.cuda.current_stream().cuda_stream
    if kind == "heads":
        sv.head_norm_rope(ctx, s["call"], c["tokens"], stream=stream)
    elif kind == "cache":
        s["cache"].append(s["k"].data_ptr(), s["v"].data_ptr(), s["past"].data_ptr(), c["tokens"], stream=stream)
        s["cache"].read(s["out"][0].data_ptr(), s["out"][1].data_ptr(), s["past"].data_ptr(), c["tokens"], stream=stream)
    elif kind == "attention":
        sv.attention(ctx, s["call"], c["tokens"], stream=stream)
    elif kind == "probabilities":
        sv.probabilities(ctx, s["call"], stream=stream)
    else:
        sv.verify(ctx, s["call"], c["sequences"], c["tokens"], stream=stream)
    return s["out"]


def _heads(c, s):
    def one(x, heads, weight):
        x = x.reshape(c["tokens"], heads, c["dim"])
        if weight is not None:
            x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPSILON) * weight
        at = s["positions"].long()
        cosines, sines = s["cosines"][at][:, None], s["sines"][at][:, None]
        turned, rest = x[..., :c["rotated"]], x[..., c["rotated"]:]
        if c["pairing"] == "halves":
            a, b = turned.chunk(2, -1)
            turned = torch.cat([a * cosines - b * sines, b * cosines + a * sines], -1)
        else:
            a, b = turned[..., 0::2], turned[..., 1::2]
            turned = torch.stack([a * cosines - b * sines, b * cosines + a * sines], -1).flatten(-2)
        return torch.cat([turned, rest], -1).flatten(1)

    return [one(s["q"], c["heads"], s.get("q_weight")), one(s["k"], c["kv_heads"], s.get("k_weight"))]


def _cache(c, s):
    return [_values(*_quantize(s[x].view(c["sequences"], c["tokens"], c["kv_heads"], c["dim"]), c["type"])).flatten(2)
            for x in "kv"]


def _ancestors(parents):
    """[sequences][row][node]: whether a row's node is the row itself or above it; and each row's depth."""
    n = parents.shape[1]
    up = (parents[..., None] == torch.arange(n, device=parents.device)).float()
    reach = up + torch.eye(n, device=parents.device)
    for _ in range(max(1, (n - 1).bit_length())):
        reach = ((reach @ reach) > 0).float()
    return reach > 0, reach.sum(-1).long() - 1


def _visible(c, s, keys):
    """[sequences][row][key]"""
    n, past = c["tokens"], s["past"].long()[:, None, None]
    key, row = torch.arange(keys, device="cuda")[None, None], torch.arange(n, device="cuda")[None, :, None]
    if c["tree"]:
        above, depth = _ancestors(s["parents"])
        node = (key - past).clamp(0, n - 1).expand(c["sequences"], n, keys)
        seen = (key < past) | ((key < past + n) & above.gather(2, node))
        depth_of_key = torch.where(key < past, key - past, depth[:, None].expand(-1, n, -1).gather(2, node))
        depth = depth[..., None]
    else:
        seen, depth, depth_of_key = key <= past + row, row, key - past
    return seen & (depth - depth_of_key < c["window"]) if c["window"] else seen


def _attention(c, s):
    keys, group = c["past"] + c["tokens"], c["heads"] // c["kv_heads"]
    k, v = (_values(s[x + "_codes"], s[x + "_scales"]).transpose(1, 2) for x in "kv")  # [sequences][kv head][key][dim]
    q = s["q"].view(c["sequences"], c["tokens"], c["kv_heads"], group, c["dim"]).permute(0, 2, 1, 3, 4)
    q = q.reshape(c["sequences"], c["kv_heads"], c["tokens"] * group, c["dim"])
    scores = torch.matmul(q, k.transpose(2, 3).contiguous()) * s["scale"]
    seen = _visible(c, s, keys)[:, None].repeat_interleave(group, 2)
    scores = torch.where(seen, scores, torch.full_like(scores[:1, :1, :1, :1], -math.inf))
    e = torch.exp(scores - scores.amax(-1, keepdim=True))
    out = torch.matmul(e, v.contiguous()) / e.sum(-1, keepdim=True)
    return out.view(c["sequences"], c["kv_heads"], c["tokens"], group, c["dim"]).permute(0, 2, 1, 3, 4).reshape(s["q"].shape)


def _probabilities(c, s):
    if c["temperature"] == 0:
        out = torch.zeros_like(s["logits"])
        return out.scatter_(1, s["logits"].argmax(1, keepdim=True), 1.0)
    e = torch.exp((s["logits"] - s["logits"].amax(1, keepdim=True)) / c["temperature"])
    return e / e.sum(1, keepdim=True)


def _drawn(weights, uniforms):
    """The index each row of weights [..., vocab] gives for its uniform number: in whole numbers, exact."""
    units = (weights.clamp(0, 1) * UNITS).long()
    running = units.cumsum(-1)
    total, r = running[..., -1], (uniforms * (1 << 31)).long()
    at = (total >> 31) * r + (((total & ((1 << 31) - 1)) * r) >> 31)
    return (running <= at[..., None]).sum(-1) * (total > 0)


def _verify(c, s):
    n, tokens = c["tokens"], s["node_tokens"]
    index = torch.arange(n, device="cuda")
    if c["tree"]:
        drawn = _drawn(s["target"], s["uniforms"])
        up = s["parents"].long()
        right = (up >= 0) & (tokens == drawn.gather(1, up.clamp(min=0)))
        # of siblings with one token, the first
        twin = (up[:, :, None] == up[:, None]) & (tokens[:, :, None] == tokens[:, None]) & (index[:, None] > index)
        right = (right & ~twin.any(-1)) | (index == 0)
        above, depth = _ancestors(s["parents"])
        taken = ~(above & ~right[:, None]).any(-1) & above[..., 0]
        count = taken.sum(1)
        path = torch.where(taken, depth, n).argsort(dim=1, stable=True)
        path = torch.where(index < count[:, None], path, -1)
        emitted = torch.where(path >= 0, drawn.gather(1, path.clamp(min=0)), -1)
        return [path.int(), emitted.int(), count.int()]
    length = s["lengths"].long()[:, None]
    at = tokens[:, 1:, None].long()
    p, q = s["target"][:, :-1].gather(2, at)[..., 0], s["draft"].gather(2, at)[..., 0]
    accepted = (s["accepts"][:, 1:] * q < p) & (index[1:] < length)
    count = accepted.int().cumprod(1).sum(1, keepdim=True) + 1
    wide = (count - 1)[..., None].expand(-1, 1, c["vocab"])
    row = s["target"].gather(1, wide)[:, 0]
    if n > 1:
        refused = s["draft"].gather(1, wide.clamp(max=n - 2))[:, 0]
        row = torch.where(count < length, row - refused, row)
    last = _drawn(row, s["uniforms"].gather(1, count - 1)[:, 0])[:, None]
    path = torch.where(index < count, index, -1)
    after = torch.cat([tokens[:, 1:].long(), last], 1)
    emitted = torch.where(index < count - 1, after, torch.where(index == count - 1, last, -1))
    return [path.int(), emitted.int(), count[:, 0].int()]


_PLAIN = {"heads": _heads, "cache": _cache, "attention": _attention, "probabilities": _probabilities, "verify": _verify}


# ---- what a pass cannot do without --------------------------------------------


def work(case):
    c, kind = case, case["kind"]
    if kind == "heads":
        values = c["tokens"] * (c["heads"] + c["kv_heads"]) * c["dim"]
        return {"bytes": 8 * values + 4 * c["tokens"] * c["rotated"], "flops": (7 if c["norm"] else 3) * values}
    if kind == "cache":  # f32 in, codes and scales out, and back
        values = 2 * c["sequences"] * c["tokens"] * c["kv_heads"] * c["dim"]
        return {"bytes": (8 + 2 * STORED[c["type"]]) * values, "flops": 4 * values}
    if kind == "attention":
        keys = min(c["past"], c["window"] or c["past"]) + c["tokens"]
        seen = min(c["past"] + (1 if c["tokens"] == 1 else c["tokens"] / 2), c["window"] or math.inf)
        values = c["sequences"] * c["tokens"] * c["heads"] * c["dim"]
        stored = 2 * c["sequences"] * keys * c["kv_heads"] * c["dim"] * STORED[c["type"]]
        return {"bytes": stored + 8 * values, "flops": 4 * values * seen}
    if kind == "probabilities":
        values = c["rows"] * c["vocab"]
        return {"bytes": 8 * values, "flops": 4 * values}
    rows = c["sequences"] * (c["tokens"] if c["tree"] else 2 if c["tokens"] > 1 else 1)
    return {"bytes": 4 * rows * c["vocab"], "flops": 2 * rows * c["vocab"]}


# ---- the definitions in 64 bits --------------------------------------------------


def exact(case, seed):
    s, c = _inputs(case, seed), case
    if c["kind"] == "heads":
        out = []
        for name, heads in (("q", c["heads"]), ("k", c["kv_heads"])):
            x = s[name].double().reshape(-1, heads, c["dim"])
            if c["norm"]:
                x = x * (x.pow(2).sum(-1, keepdim=True) / c["dim"] + EPSILON).rsqrt() * s[name + "_weight"].double()
            half, at = c["rotated"] // 2, s["positions"].long()
            turn = torch.complex(s["cosines"].double()[at], s["sines"].double()[at])[:, None]
            first = torch.arange(half, device="cuda") * (1 if c["pairing"] == "halves" else 2)
            second = first + (half if c["pairing"] == "halves" else 1)
            z = torch.complex(x[..., first], x[..., second]) * turn
            y = x.clone()
            y[..., first], y[..., second] = z.real, z.imag
            out.append(y.flatten(1))
        return out
    if c["kind"] == "cache":
        out = []
        for x in (s["k"], s["v"]):
            b = x.double().unflatten(-1, (-1, 32))
            if c["type"] == "f16":
                out.append(x.half().double())
                continue
            extreme = b.gather(-1, b.abs().argmax(-1, keepdim=True))
            d = (extreme.abs() / 127 if c["type"] == "q8_0" else extreme / -8).half().double()
            code = torch.where(d == 0, 0.0, b / d).round()
            code = code.clamp(-127, 127) if c["type"] == "q8_0" else code.clamp(-8, 7)
            out.append((code * d).flatten(-2))
        return out
    if c["kind"] == "attention":
        if c["sequences"] * c["tokens"] * c["heads"] * (c["past"] + c["tokens"]) > 512 * 17000 * 32:
            return None
        out = torch.zeros(s["q"].shape, device="cuda", dtype=torch.float64)
        group = c["heads"] // c["kv_heads"]
        for i in range(c["sequences"]):
            past = int(s["past"][i])
            n = past + c["tokens"]
            seen = torch.zeros(c["tokens"], n, dtype=torch.bool)
            parents = s["parents"][i].tolist() if c["tree"] else list(range(-1, c["tokens"] - 1))
            for row in range(c["tokens"]):
                line, node = [], row
                while node >= 0:
                    line.append(node)
                    node = parents[node]
                reach = c["window"] or n + 1
                seen[row, [past + node for node in line[:reach]]] = True
                seen[row, max(0, past - max(0, reach - len(line))):past] = True
            seen = seen.cuda()
            for h in range(c["kv_heads"]):
                k, v = ((s[x + "_codes"][i, :n, h].double() * s[x + "_scales"][i, :n, h].double()[..., None]).flatten(1)
                        for x in "kv")
                for j in range(h * group, h * group + group):
                    at = slice(j * c["dim"], (j + 1) * c["dim"])
                    score = (s["q"][i, :, at].double() @ k.T * s["scale"]).masked_fill(~seen, -math.inf)
                    out[i, :, at] = torch.softmax(score, 1) @ v
        return out
    if c["kind"] == "probabilities" and c["temperature"] > 0:
        return torch.softmax(s["logits"].double() / c["temperature"], 1)
    return None
