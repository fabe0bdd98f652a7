"""The operators of a step that serves several requests at once, whose speed is
measured: what runs beside charlotte_amd.matmul when requests of any lengths
share a pool of cache pages, through charlotte_amd.serving, and each in its
plain form of elementary torch operations.

A case's fields:
  kind      "pages": block tables and slot maps built from the requests' lengths
            (pages given back and taken), the step's keys and values written
            through them, and read back as the values they stand for.
            "attention": each request's new tokens over its pages.
            "norm": a block's output normalised, gated, scaled and added to the
            residual stream, and the stream normalised for the next block.
            "sample": a token drawn from each row of logits, by temperature,
            top-k, top-p, min-p and a given uniform number.
  requests, shortest, longest   requests, and the range of their cached tokens
  prompts, chunk   so many of them bring `chunk` tokens, the others one
  type, page   the pool's format and tokens a page
  heads, kv_heads, dim   query heads, key heads, a head's values
Activations and outputs are f32, as the products' are.
"""

import math
import random

import torch

own = False

# Heads of models this repository names: query heads, key heads, values a head.
QWEN3_0_6B = {"heads": 16, "kv_heads": 8, "dim": 128}
LLAMA_3_2_1B = {"heads": 32, "kv_heads": 8, "dim": 64}
LLAMA_3_8B = {"heads": 32, "kv_heads": 8, "dim": 128}
GEMMA_3_1B = {"heads": 4, "kv_heads": 1, "dim": 256}

STORED = {"f16": 2.0, "q8_0": 34 / 32, "q4_0": 18 / 32}
EPSILON = 1e-6
WHOLE = 1 << 40  # a largest token's weight in a draw


def listed():
    return [
        # A decoding step of 24 chats, one token each; one of them has ended: launches' latency.
        {"name": "pages_24_requests", "kind": "pages", "type": "q8_0", "page": 32, "requests": 24, "shortest": 20,
         "longest": 4000, "prompts": 0, "chunk": 1, "ending": 1, "spare": 40, **QWEN3_0_6B},
        # The same step with two prompts' blocks among 64 requests, 4 bits a value, at the ends of the free pages.
        {"name": "pages_2_prompts", "kind": "pages", "type": "q4_0", "page": 64, "requests": 64, "shortest": 1,
         "longest": 16000, "prompts": 2, "chunk": 2048, "ending": 3, "spare": 0, **LLAMA_3_8B},
        # Three short chats in a layer with a window: latency.
        {"name": "attention_3_short", "kind": "attention", "type": "f16", "page": 32, "requests": 3, "shortest": 90,
         "longest": 911, "prompts": 0, "chunk": 1, "window": 512, **GEMMA_3_1B},
        # One long context by itself, 4 bits a value: few rows, everything along the cache's length.
        {"name": "attention_1_over_65536", "kind": "attention", "type": "q4_0", "page": 64, "requests": 1,
         "shortest": 65536, "longest": 65536, "prompts": 0, "chunk": 1, "window": 0, **LLAMA_3_2_1B},
        # 64 requests of very different lengths: bound by the cache's bytes, if the work is shared evenly.
        {"name": "attention_64_ragged", "kind": "attention", "type": "q8_0", "page": 32, "requests": 64, "shortest": 50,
         "longest": 32768, "prompts": 0, "chunk": 1, "window": 0, **LLAMA_3_8B},
        # Two prompts' blocks read beside 14 requests that decode: bound by products.
        {"name": "attention_2_prompts", "kind": "attention", "type": "q8_0", "page": 128, "requests": 16,
         "shortest": 100, "longest": 8000, "prompts": 2, "chunk": 512, "window": 0, **LLAMA_3_2_1B},
        # One token's residual stream between two blocks.
        {"name": "norm_1_token", "kind": "norm", "rows": 1, "width": 1024, "after": False, "gate": "none",
         "scaled": False, "strided": False},
        # A prompt's block in a model with norms before and after each block.
        {"name": "norm_2048_tokens", "kind": "norm", "rows": 2048, "width": 4096, "after": True, "gate": "none",
         "scaled": False, "strided": False},
        # A batch of tokens with a gate a channel and scales, at an odd width.
        {"name": "norm_333_tokens_gated", "kind": "norm", "rows": 333, "width": 1155, "after": True, "gate": "shared",
         "scaled": True, "strided": True},
        # One chat's next token.
        {"name": "sample_1_row", "kind": "sample", "rows": 1, "vocab": 151936, "plain": False},
        # 64 requests' next tokens, each with settings of its own.
        {"name": "sample_64_rows", "kind": "sample", "rows": 64, "vocab": 128256, "plain": False},
        # The widest vocabulary here, by temperature alone.
        {"name": "sample_24_rows_untruncated", "kind": "sample", "rows": 24, "vocab": 262144, "plain": True},
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
    """Another case of the ranges the listed ones stand for: 1 to 96 requests of
    0 to 65,536 cached tokens, up to two prompts' blocks of 2 to 512 (attention)
    or 2,048 tokens, pages of 32 to 256 tokens in each format; 1 to 2,048 rows
    of 64 to 8,192 values; 1 to 64 rows of 4,096 to 262,144 logits."""
    kind = rng.choices(["pages", "attention", "norm", "sample"], weights=[3, 6, 3, 3])[0]
    if kind == "pages":
        shape, requests = _shape(rng), _log(rng, 1, 96)
        prompts = min(rng.choice([0, 0, 1, 2]), requests)
        chunk = _log(rng, 2, min(2048, 2048 * 1024 // (shape["kv_heads"] * shape["dim"]))) if prompts else 1
        return {"kind": kind, "type": rng.choice(["q8_0", "q4_0", "f16"]), "page": rng.choice([32, 64, 96, 128, 256]),
                "requests": requests, "shortest": _log(rng, 1, 500), "longest": _log(rng, 500, 16000), "prompts": prompts,
                "chunk": chunk, "ending": rng.choice([0, 0, 1, 2]) if requests > 4 else 0,
                "spare": rng.choice([0, 7, 100, -1]), **shape}
    if kind == "attention":
        shape, requests = _shape(rng), _log(rng, 1, 96)
        prompts = min(rng.choice([0, 0, 0, 1, 2]), requests)
        chunk = _log(rng, 2, 512) if prompts else 1
        # no more bytes than the longest listed, no more products
        most = min(65536, int(1.6e8 / (requests * shape["kv_heads"] * shape["dim"])))
        if prompts:
            most = min(most, int(1.4e10 / (prompts * chunk * shape["heads"] * shape["dim"])))
        longest = _log(rng, 1, max(2, most))
        return {"kind": kind, "type": rng.choice(["q8_0", "q8_0", "q4_0", "f16"]), "page": rng.choice([32, 64, 96, 128, 256]),
                "requests": requests, "shortest": rng.choice([0, _log(rng, 1, longest), _log(rng, 1, longest)]),
                "longest": longest, "prompts": prompts, "chunk": chunk,
                "window": rng.choice([0, 0, 0, 512, _log(rng, 2, 4096)]), **shape}
    if kind == "norm":
        rows = 1 if rng.random() < 0.3 else _log(rng, 2, 2048)
        width = rng.choice([1024, 1152, 2048, 4096, _log(rng, 64, 8192)])
        gate = rng.choice(["none", "none", "shared", "rows"])
        most = 2048 * 4096 * 3 // 4 if gate == "rows" else 2048 * 4096
        return {"kind": kind, "rows": rows, "width": min(width, most // rows), "after": rng.random() < 0.5, "gate": gate,
                "scaled": rng.random() < 0.5, "strided": rng.random() < 0.3}
    vocab = rng.choice([128256, 151936, 262144, _log(rng, 4096, 262144)])
    return {"kind": kind, "rows": _log(rng, 1, min(64, 8.2e6 / vocab)), "vocab": vocab, "plain": rng.random() < 0.3}


# ---- inputs ------------------------------------------------------------------


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def _uniform(g, *shape):
    return torch.rand(*shape, generator=g, device="cuda", dtype=torch.float32)


def _ints(values):
    return torch.tensor(values, device="cuda", dtype=torch.int32)


def _lengths(c):
    """Cached tokens of each request, spread evenly over their logarithm (a shortest of 0: the first's alone)."""
    n, low, high = c["requests"], max(1, min(c["shortest"], c["longest"])), c["longest"]
    lengths = [int(round(low * (high / low) ** ((i + 1) / n if n == 1 else i / (n - 1)))) for i in range(n)]
    return lengths if c["shortest"] else [0, *lengths[1:]]


def _counts(c):
    """New tokens of each request, before they are shuffled: the longest are the prompts."""
    return [1] * (c["requests"] - c["prompts"]) + [c["chunk"]] * c["prompts"]


def _requests(c, seed):
    """[(past, count)] in the order of a seed's batch."""
    pairs = list(zip(_lengths(c), _counts(c)))
    random.Random(int(seed)).shuffle(pairs)
    return pairs


def _keys_and_values(g, tokens, kv_heads, dim):
    """Keys with a few large channels and values, as layers make them: [tokens][kv_heads * dim]."""
    spread = 0.3 + 1.7 * _uniform(g, kv_heads * dim) ** 4
    return _normal(g, tokens, kv_heads * dim) * spread, _normal(g, tokens, kv_heads * dim) * 0.7


def _quantize(x, format_):
    """The pool's codes and scales for values x [..., dim]: blocks of 32, as the cache's formats are defined."""
    b = x.reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    if format_ == "f16":
        return b.half(), torch.ones(b.shape[:-1], device=b.device, dtype=torch.float16)
    largest, at = b.abs().max(-1, keepdim=True)
    d = (largest / 127).half() if format_ == "q8_0" else (b.gather(-1, at) / -8).half()
    low, high = (-127, 127) if format_ == "q8_0" else (-8, 7)
    step = d.float()
    codes = torch.where(step == 0, torch.zeros_like(b), torch.round(b / step)).clamp(low, high)
    return codes.to(torch.int8), d.squeeze(-1)


def _values(codes, scales):
    """The f32 values that codes and scales stand for, [..., dim]."""
    return (codes.float() * scales.float()[..., None]).flatten(-2)


def _pages_inputs(c, seed, g, s):
    pairs, p = _requests(c, seed), c["page"]
    one = [r for r, (_, count) in enumerate(pairs) if count == 1]
    s["ended"] = random.Random(int(seed) + 1).sample(one, c["ending"])
    held = [-(-past // p) for past, _ in pairs]
    past = [0 if r in s["ended"] else n for r, (n, _) in enumerate(pairs)]
    counts = [0 if r in s["ended"] else n for r, (_, n) in enumerate(pairs)]
    need = [-(-(n + m) // p) for n, m in zip(past, counts)]
    takes = sum(max(0, n - h) for n, h in zip(need, held))
    gives = sum(max(0, h - n) for n, h in zip(need, held))
    free = max(0, takes - gives + c["spare"])
    largest = [-(-(n + m) // p) for n, m in pairs]
    s["rows"], s["stride"] = sum(counts) + 3, max(largest) + 1
    s["pages"] = sum(largest) + max(0, c["spare"]) + 8
    order = torch.randperm(s["pages"], generator=g, device="cuda").to(torch.int32)
    s["table"] = torch.full((c["requests"], s["stride"]), -1, device="cuda", dtype=torch.int32)
    at = 0
    for r, n in enumerate(held):
        s["table"][r, :n] = order[at:at + n]
        at += n
    s["free"] = torch.full((s["pages"],), -1, device="cuda", dtype=torch.int32)
    s["free"][:free] = order[at:at + free]
    s["free_count"] = _ints([free])
    s["past"], s["counts"], s["held"] = _ints(past), _ints(counts), _ints(held)
    s["k"], s["v"] = _keys_and_values(g, s["rows"], c["kv_heads"], c["dim"])


def _attention_inputs(c, seed, g, s):
    pairs, p = _requests(c, seed), c["page"]
    s["lines"] = pairs
    held = [-(-(n + m) // p) for n, m in pairs]
    s["pages"], s["stride"] = sum(held) + 5, max(held)
    order = torch.randperm(s["pages"], generator=g, device="cuda").to(torch.int32)
    s["table"] = torch.full((c["requests"], s["stride"]), -1, device="cuda", dtype=torch.int32)
    shape = (s["pages"], p, c["kv_heads"], c["dim"] // 32)
    kind = torch.float16 if c["type"] == "f16" else torch.int8
    for x in "kv":
        s[x + "_codes"] = torch.zeros(*shape, 32, device="cuda", dtype=kind)
        s[x + "_scales"] = torch.zeros(shape, device="cuda", dtype=torch.float16)
    at = 0
    for r, n in enumerate(held):
        s["table"][r, :n] = mine = order[at:at + n]
        at += n
        made = _keys_and_values(g, n * p, c["kv_heads"], c["dim"])
        for x, values in zip("kv", made):
            codes, scales = _quantize(values.view(n, p, c["kv_heads"], c["dim"]), c["type"])
            s[x + "_codes"][mine.long()] = codes
            s[x + "_scales"][mine.long()] = scales
    counts = [m for _, m in pairs]
    s["rows"] = sum(counts)
    s["past"], s["counts"] = _ints([n for n, _ in pairs]), _ints(counts)
    s["starts"] = _ints([sum(counts[:i]) for i in range(len(counts) + 1)])
    s["q"] = _normal(g, s["rows"], c["heads"] * c["dim"])
    s["scale"] = 1 / math.sqrt(c["dim"])


def _norm_inputs(c, g, s):
    rows, width = c["rows"], c["width"]
    wide = width + 8 if c["strided"] else width
    s["x"], s["y"] = (_normal(g, rows, wide)[:, :width] * f for f in (4.0, 1.0))
    s["x"][:, 7 % width] += 60  # a channel that stands out, as in models
    s["weight"] = 1 + 0.3 * _normal(g, width)
    if c["after"]:
        s["after"] = 0.5 + 0.3 * _normal(g, width)
    if c["gate"] != "none":
        s["gate"] = _normal(g, rows if c["gate"] == "rows" else 1, width)
    s["scales"] = (0.875, 0.22) if c["scaled"] else (1.0, 1.0)


def _sample_inputs(c, seed, g, s):
    rows, vocab = c["rows"], c["vocab"]
    s["logits"] = _normal(g, rows, vocab) * 2.5
    at = torch.arange(48, device="cuda") * (vocab // 48) + torch.randint(0, vocab // 48, (rows, 48), generator=g, device="cuda")
    s["logits"].scatter_add_(1, at, 9 * _uniform(g, rows, 48))  # likely tokens, apart from each other
    s["uniforms"] = _uniform(g, rows)
    rng = random.Random(int(seed))
    each = {"temperatures": [0.6, 0.7, 0.8, 1.0, 1.3, 0.0], "top_ks": [0, 0, 20, 50, 1000],
            "top_ps": [1.0, 0.8, 0.9, 0.95], "min_ps": [0.0, 0.0, 0.05, 0.1]}
    for name, choices in each.items():
        picked = [rng.choice(choices[:3]), *(rng.choice(choices) for _ in range(rows - 1))]
        if c["plain"]:
            picked = [{"temperatures": 0.9, "top_ks": 0, "top_ps": 1.0, "min_ps": 0.0}[name]] * rows
        s[name] = torch.tensor(picked, device="cuda", dtype=torch.int32 if name == "top_ks" else torch.float32)


def _inputs(case, seed):
    """A case's data: from the seed alone, the same for the plain form, the kernels and the 64-bit results."""
    g, s = _generator(seed), {}
    if case["kind"] == "pages":
        _pages_inputs(case, seed, g, s)
    elif case["kind"] == "attention":
        _attention_inputs(case, seed, g, s)
    elif case["kind"] == "norm":
        _norm_inputs(case, g, s)
    else:
        _sample_inputs(case, seed, g, s)
    return s


def prepare(case, seed):
    """The inputs and, for the kernels, the context, pool, buffers and descriptors that a serving loop keeps."""
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
    kind, p = c["kind"], torch.Tensor.data_ptr
    types = {"q8_0": mm.TensorType.Q8_0, "q4_0": mm.TensorType.Q4_0, "f16": mm.TensorType.F16}

    def workspace(nbytes):
        s["workspace"] = torch.empty(max(nbytes, 16), device="cuda", dtype=torch.uint8)
        return {"workspace": p(s["workspace"]), "workspace_bytes": nbytes}

    if kind == "pages":
        s["pool"] = sv.PagePool(ctx, types[c["type"]], s["pages"], c["page"], c["kv_heads"], c["dim"])
        like = lambda n: torch.zeros(n, device="cuda", dtype=torch.int32)  # noqa: E731
        after, left, starts = like(c["requests"]), like(1), like(c["requests"] + 1)
        granted, slots, positions = like(c["requests"]), like(s["rows"]), like(s["rows"])
        back = [torch.zeros_like(s["k"]), torch.zeros_like(s["v"])]
        s["out"] = [s["table"], after, s["free"], left, starts, granted, slots, positions, *back]
        s["call"] = sv.PagePlan(
            requests=c["requests"], rows=s["rows"], pages=s["pages"], page_tokens=c["page"], past=p(s["past"]),
            counts=p(s["counts"]), table=p(s["table"]), table_stride=s["stride"], held=p(s["held"]), held_after=p(after),
            free_pages=p(s["free"]), free_count=p(s["free_count"]), free_count_after=p(left), starts=p(starts),
            granted=p(granted), slots=p(slots), positions=p(positions))
        s["slots"] = slots
    elif kind == "attention":
        s["pool"] = sv.PagePool(ctx, types[c["type"]], s["pages"], c["page"], c["kv_heads"], c["dim"])
        stream, tokens = torch.cuda.current_stream().cuda_stream, s["pages"] * c["page"]
        step = max(1, (1 << 28) // (c["kv_heads"] * c["dim"]))
        for at in range(0, tokens, step):
            n = min(step, tokens - at)
            k, v = (_values(s[x + "_codes"].flatten(0, 1)[at:at + n], s[x + "_scales"].flatten(0, 1)[at:at + n]).flatten(1)
                    for x in "kv")
            slots = torch.arange(at, at + n, device="cuda", dtype=torch.int32)
            s["pool"].append(p(k), p(v), p(slots), n, stream=stream)
            torch.cuda.synchronize()
        for name in ("k_codes", "k_scales", "v_codes", "v_scales"):
            del s[name]
        s["out"] = torch.zeros_like(s["q"])
        most = max(m for _, m in s["lines"])
        s["call"] = sv.PagedAttention(
            s["pool"], queries=p(s["q"]), output=p(s["out"]), query_heads=c["heads"], scale=s["scale"],
            requests=c["requests"], rows=s["rows"], past=p(s["past"]), counts=p(s["counts"]), starts=p(s["starts"]),
            table=p(s["table"]), table_stride=s["stride"], window=c["window"], most=most,
            **workspace(sv.paged_attention_workspace_bytes(ctx, s["pool"], c["heads"], most)))
    elif kind == "norm":
        s["out"] = [torch.empty(c["rows"], c["width"], device="cuda") for _ in range(2)]
        gate = {"gate": p(s["gate"]), "gate_stride": c["width"] if c["gate"] == "rows" else 0} if "gate" in s else {}
        s["call"] = sv.ResidualNorm(
            c["width"], residual=p(s["x"]), branch=p(s["y"]), residual_out=p(s["out"][0]), normed=p(s["out"][1]),
            weight=p(s["weight"]), branch_weight=p(s["after"]) if c["after"] else 0, residual_scale=s["scales"][0],
            branch_scale=s["scales"][1], epsilon=EPSILON, residual_stride=s["x"].stride(0),
            branch_stride=s["y"].stride(0), **gate)
    else:
        s["out"] = [torch.empty(c["rows"], device="cuda", dtype=torch.int32), torch.empty(c["rows"], device="cuda")]
        s["call"] = sv.Sample(
            p(s["logits"]), tokens=p(s["out"][0]), chances=p(s["out"][1]), rows=c["rows"], vocabulary=c["vocab"],
            uniforms=p(s["uniforms"]), temperatures=p(s["temperatures"]), top_ks=p(s["top_ks"]), top_ps=p(s["top_ps"]),
            min_ps=p(s["min_ps"]), **workspace(sv.sample_workspace_bytes(c["rows"], c["vocab"])))


# ---- one pass ------------------------------------------------------------------


def run(state):
    return _run_own(state) if own else _PLAIN[state["case"]["kind"]](state["case"], state)


def _run_own(s):
    from charlotte_amd import serving as sv

    c, ctx = s["case"], s["ctx"]
    kind, stream = c["kind"], torch.cuda.current_stream().cuda_stream
    if kind == "pages":
        sv.page_plan(ctx, s["call"], stream=stream)
        s["pool"].append(s["k"].data_ptr(), s["v"].data_ptr(), s["slots"].data_ptr(), s["rows"], stream=stream)
        s["pool"].read(s["out"][8].data_ptr(), s["out"][9].data_ptr(), s["slots"].data_ptr(), s["rows"], stream=stream)
    elif kind == "attention":
        sv.paged_attention(ctx, s["call"], stream=stream)
    elif kind == "norm":
        sv.residual_norm(ctx, s["call"], c["rows"], stream=stream)
    else:
        sv.sample(ctx, s["call"], stream=stream)
    return s["out"]


def _pages(c, s):
    page, pages, stride, rows = c["page"], s["pages"], s["stride"], s["rows"]
    past, counts, held, left = s["past"].long(), s["counts"].long(), s["held"].long(), s["free_count"].long()
    ends = counts.cumsum(0)
    starts = ends - counts
    need = (past + counts + page - 1) // page
    fits = ((counts == 0) | (ends <= rows)) & (need <= stride)
    # pages given back, onto the stack's top
    entry = torch.arange(stride, device="cuda")
    given = fits[:, None] & (entry >= need[:, None]) & (entry < held[:, None])
    rank = given.flatten().cumsum(0).view_as(given)
    free = torch.cat([s["free"], s["free"].new_zeros(1)])
    free.scatter_(0, torch.where(given, left + rank - 1, pages).flatten(), s["table"].flatten())
    left = left + rank[-1, -1]
    # and taken from it, in the requests' order while they last
    takes = torch.where(fits, (need - held).clamp(min=0), 0)
    served = fits & ((takes == 0) | (takes.cumsum(0) <= left))
    takes = torch.where(served, takes, 0)
    before = takes.cumsum(0) - takes
    taken = (entry >= held[:, None]) & (entry < (held + takes)[:, None])
    source = (left - 1 - before[:, None] - (entry - held[:, None])).clamp(0, pages - 1)
    table = torch.where(taken, free[source], s["table"])
    left = left - takes.sum()
    after = torch.where(served, need, held)
    granted = torch.where(served, counts, 0)
    # each row's request, place and slot
    row = torch.arange(rows, device="cuda")
    request = (ends <= row[:, None]).sum(1)
    live = request < c["requests"]
    request = request.clamp(max=c["requests"] - 1)
    position = torch.where(live, past[request] + row - starts[request], 0)
    at = table[request, (position // page).clamp(max=stride - 1)].long()
    live = live & served[request] & (at >= 0) & (at < pages)
    slots = torch.where(live, at * page + position % page, -1)
    back = [torch.where(live[:, None], _values(*_quantize(s[x].view(rows, c["kv_heads"], c["dim"]), c["type"])).flatten(1), 0.0)
            for x in "kv"]
    return [table, after.int(), free[:pages], left.int(), torch.cat([starts, ends[-1:]]).int(), granted.int(), slots.int(),
            position.int(), *back]


def _attention(c, s):
    group, out, at = c["heads"] // c["kv_heads"], [], 0
    for r, (past, count) in enumerate(s["lines"]):
        n = past + count
        first = max(0, past + 1 - c["window"]) // c["page"] if c["window"] else 0
        mine = s["table"][r, first:-(-n // c["page"])].long()
        first *= c["page"]
        k, v = (_values(s[x + "_codes"][mine].flatten(0, 1)[:n - first], s[x + "_scales"][mine].flatten(0, 1)[:n - first])
                .transpose(0, 1) for x in "kv")  # [kv head][key][dim]
        q = s["q"][at:at + count].view(count, c["kv_heads"], group, c["dim"]).transpose(0, 1).flatten(1, 2)
        scores = torch.matmul(q, k.transpose(1, 2).contiguous()) * s["scale"]
        row, key = past + torch.arange(count, device="cuda")[:, None], first + torch.arange(n - first, device="cuda")
        seen = (key <= row) & (row - key < c["window"]) if c["window"] else key <= row
        if count > 1 or c["window"]:
            scores = scores.masked_fill(~seen.repeat_interleave(group, 0), -math.inf)
        e = torch.exp(scores - scores.amax(-1, keepdim=True))
        o = torch.matmul(e, v.contiguous()) / e.sum(-1, keepdim=True)
        out.append(o.view(c["kv_heads"], count, group, c["dim"]).transpose(0, 1).reshape(count, -1))
        at += count
    return torch.cat(out)


def _norm(c, s):
    y = s["y"]
    if c["after"]:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + EPSILON) * s["after"]
    if c["gate"] != "none":
        y = y * s["gate"]
    r = s["x"] * s["scales"][0] + y * s["scales"][1] if c["scaled"] else s["x"] + y
    return [r, r / torch.sqrt((r * r).mean(-1, keepdim=True) + EPSILON) * s["weight"]]


def _sample(c, s):
    """In whole numbers from weights on: exact, so that a token at a border is the same in every form."""
    logits, order = torch.sort(s["logits"], dim=-1, descending=True, stable=True)
    temperature = s["temperatures"].double()[:, None]
    greedy = temperature < 1e-6
    x = (logits.double() - logits[:, :1].double()) / temperature.masked_fill(greedy, 1.0)
    weights = torch.floor(torch.exp(x) * WHOLE).long()
    index = torch.arange(c["vocab"], device="cuda")
    top_k = torch.where(s["top_ks"] > 0, s["top_ks"], c["vocab"]).long()[:, None]
    kept = (index < top_k) & ((index == 0) | ~greedy)
    running = (weights * kept).cumsum(-1)
    least = torch.ceil(s["top_ps"].double()[:, None] * running[:, -1:].double())
    kept = kept & ((index == 0) | (s["top_ps"][:, None] >= 1) | ((running - weights).double() < least))
    kept = kept & ((index == 0) | (weights >= torch.ceil(s["min_ps"].double()[:, None] * WHOLE)))
    running = (weights * kept).cumsum(-1)
    total, r = running[:, -1], (s["uniforms"] * (1 << 31)).long()
    at = (total >> 31) * r + (((total & ((1 << 31) - 1)) * r) >> 31)
    place = (running <= at[:, None]).sum(-1, keepdim=True)
    chance = weights.gather(1, place)[:, 0].double() / total.double()
    return [order.gather(1, place)[:, 0].int(), chance.float()]


_PLAIN = {"pages": _pages, "attention": _attention, "norm": _norm, "sample": _sample}


# ---- what a pass cannot do without --------------------------------------------


def work(case):
    c, kind = case, case["kind"]
    if kind == "pages":  # lengths and tables, a slot and a position a row; f32 in, codes and scales out, and back
        rows = sum(_counts(c)) - c["ending"]
        values = 2 * rows * c["kv_heads"] * c["dim"]
        return {"bytes": (8 + 2 * STORED[c["type"]]) * values + 8 * rows + 24 * c["requests"], "flops": 4 * values}
    if kind == "attention":
        stored = products = rows = 0
        for past, count in zip(_lengths(c), _counts(c)):
            window = c["window"] or math.inf
            stored += min(past, window - 1) + count
            products += count * min(past + (count + 1) / 2, window)
            rows += count
        return {"bytes": 2 * stored * c["kv_heads"] * c["dim"] * STORED[c["type"]] + 8 * rows * c["heads"] * c["dim"],
                "flops": 4 * c["heads"] * c["dim"] * products}
    if kind == "norm":
        values = c["rows"] * c["width"]
        gates = {"none": 0, "shared": c["width"], "rows": values}[c["gate"]]
        return {"bytes": 16 * values + 4 * gates + (8 if c["after"] else 4) * c["width"], "flops": (11 if c["after"] else 7) * values}
    return {"bytes": 4 * c["rows"] * c["vocab"], "flops": 4 * c["rows"] * c["vocab"]}


# ---- the definitions in 64 bits --------------------------------------------------


def _pages_exact(c, s):
    page, pages = c["page"], s["pages"]
    past, counts, held, table = (s[n].tolist() for n in ("past", "counts", "held", "table"))
    stack, top, rows = s["free"].tolist(), int(s["free_count"]), s["rows"]
    ends = [sum(counts[:r + 1]) for r in range(len(counts))]
    need = [-(-(n + m) // page) for n, m in zip(past, counts)]
    fits = [(m == 0 or e <= rows) and n <= s["stride"] for m, e, n in zip(counts, ends, need)]
    after, granted, short = list(held), [0] * len(counts), False
    for r, n in enumerate(need):
        for j in range(n, held[r]) if fits[r] else ():
            stack[top] = table[r][j]
            top += 1
    wanted, there = 0, top
    for r, n in enumerate(need):
        if not fits[r]:
            continue
        wanted += max(0, n - held[r])
        if n > held[r] and wanted > there:
            continue
        for j in range(held[r], n):
            top -= 1
            table[r][j] = stack[top]
        after[r], granted[r] = n, counts[r]
    slots, positions = [-1] * rows, [0] * rows
    for r, m in enumerate(counts):
        for t in range(m):
            i, at = ends[r] - m + t, past[r] + t
            if i < rows:
                positions[i] = at
                entry = table[r][at // page] if at // page < s["stride"] else -1
                if granted[r] and 0 <= entry < pages:
                    slots[i] = entry * page + at % page
    back = []
    for x in (s["k"], s["v"]):
        b = x.double().unflatten(-1, (-1, 32))
        if c["type"] == "f16":
            y = x.half().double()
        else:
            extreme = b.gather(-1, b.abs().argmax(-1, keepdim=True))
            d = (extreme.abs() / 127 if c["type"] == "q8_0" else extreme / -8).half().double()
            code = torch.where(d == 0, 0.0, b / d).round()
            y = ((code.clamp(-127, 127) if c["type"] == "q8_0" else code.clamp(-8, 7)) * d).flatten(-2)
        y[[i for i, at in enumerate(slots) if at < 0]] = 0
        back.append(y)
    return [_ints(table), _ints(after), _ints(stack), _ints([top]), _ints([e - m for e, m in zip(ends, counts)] + ends[-1:]),
            _ints(granted), _ints(slots), _ints(positions), *back]


def _attention_exact(c, s):
    out = torch.zeros(s["q"].shape, device="cuda", dtype=torch.float64)
    group, at = c["heads"] // c["kv_heads"], 0
    for r, (past, count) in enumerate(s["lines"]):
        n = past + count
        place = torch.arange(n, device="cuda")
        page, slot = s["table"][r].long()[place // c["page"]], place % c["page"]
        row = past + torch.arange(count, device="cuda")[:, None]
        hidden = (place > row) | (row - place >= (c["window"] or n + 1))
        for h in range(c["kv_heads"]):
            k, v = ((s[x + "_codes"][page, slot, h].double() * s[x + "_scales"][page, slot, h].double()[..., None]).flatten(1)
                    for x in "kv")
            for j in range(h * group, h * group + group):
                part = slice(j * c["dim"], (j + 1) * c["dim"])
                score = (s["q"][at:at + count, part].double() @ k.T * s["scale"]).masked_fill(hidden, -math.inf)
                out[at:at + count, part] = torch.softmax(score, 1) @ v
        at += count
    return out


def _norm_exact(c, s):
    x, y = s["x"].double(), s["y"].double()

    def normal(z, w):
        return z * (z.pow(2).sum(-1, keepdim=True) / c["width"] + EPSILON).rsqrt() * w.double()

    y = normal(y, s["after"]) if c["after"] else y
    y = y * s["gate"].double() if "gate" in s else y
    r = s["scales"][0] * x + s["scales"][1] * y
    return [r, normal(r, s["weight"])]


def _sample_exact(c, s):
    import numpy as np

    tokens, chances = [], []
    settings = list(zip(*(s[n].tolist() for n in ("temperatures", "top_ks", "top_ps", "min_ps", "uniforms"))))
    for logits, (temperature, top_k, top_p, min_p, u) in zip(s["logits"].cpu().numpy(), settings):
        order = np.lexsort((np.arange(c["vocab"]), -logits.astype(np.float64)))
        z = logits.astype(np.float64)[order]
        n = 1 if temperature < 1e-6 else min(top_k, c["vocab"]) if top_k > 0 else c["vocab"]
        # no token below 2^-40 of the largest weighs anything
        x = np.maximum((z[:n] - z[0]) / (temperature or 1.0), -60.0)
        weights = [int(w) for w in np.floor(np.exp(x) * float(WHOLE)) if w > 0]
        if top_p < 1:
            least, total = math.ceil(top_p * float(sum(weights))), 0
            for n, w in enumerate(weights, 1):
                total += w
                if total >= least:
                    break
            weights = weights[:n]
        weights = weights[:1] + [w for w in weights[1:] if w >= math.ceil(min_p * WHOLE)]
        total = sum(weights)
        at, place = total * int(u * (1 << 31)) >> 31, 0
        while at >= weights[place]:
            at -= weights[place]
            place += 1
        tokens.append(int(order[place]))
        chances.append(weights[place] / total)
    return [_ints(tokens), torch.tensor(chances, device="cuda", dtype=torch.float64)]


def exact(case, seed):
    s = _inputs(case, seed)
    return {"pages": _pages_exact, "attention": _attention_exact, "norm": _norm_exact, "sample": _sample_exact}[case["kind"]](case, s)
