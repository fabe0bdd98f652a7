"""Plain restatements of charlotte_amd.serving's operators, in 64 bits (the
cache's blocks in the arithmetic that defines them, f32 and binary16), and
helpers that run them on the device (test infrastructure)."""

import numpy as np

from charlotte_amd import harness as hx
from charlotte_amd import matmul as mm
from charlotte_amd import serving as sv

FORMATS = {"q8_0": mm.TensorType.Q8_0, "q4_0": mm.TensorType.Q4_0, "f16": mm.TensorType.F16}


def stored(x, format_):
    """The values a cache of `format_` stands for after x [..., dim] is written (f32)."""
    b = np.asarray(x, np.float32).reshape(-1, 32)
    with np.errstate(all="ignore"):
        if format_ == "f16":
            out = b.astype(np.float16).astype(np.float32)
            bad = ~np.isfinite(out).all(1)
        else:
            magnitude = np.where(np.isnan(b), np.inf, np.abs(b))
            extreme = np.take_along_axis(b, magnitude.argmax(1)[:, None], 1)
            d = (np.abs(extreme) / np.float32(127) if format_ == "q8_0" else extreme / np.float32(-8)).astype(np.float16)
            step = d.astype(np.float32)
            low, high = (-127, 127) if format_ == "q8_0" else (-8, 7)
            codes = np.where(step == 0, np.float32(0), np.rint(b / step))
            codes = np.clip(codes, low, high)
            out = codes * step
            bad = ~(np.isfinite(step[:, 0]) & np.isfinite(b).all(1))
        out[bad] = np.nan
    return out.reshape(np.shape(x))


def ancestors(parents, tokens):
    """Each token's line, itself first, or None where it or one above it is unused."""
    lines = []
    for t in range(tokens):
        line, node = [], t
        while node is not None and node >= 0:
            line.append(node)
            up = int(parents[node])
            node = up if -1 <= up < node else None
        lines.append(line if node is not None else None)
    return lines


def sees(past, tokens, parents=None, window=0):
    """[token][slot] over past + tokens slots."""
    seen = np.zeros((tokens, past + tokens), bool)
    for t, line in enumerate(ancestors(parents if parents is not None else range(-1, tokens - 1), tokens)):
        if line is None:
            continue
        reach = window or past + tokens + 1
        seen[t, [past + n for n in line[:reach]]] = True
        if reach > len(line):
            seen[t, max(0, past - (reach - len(line))):past] = True
    return seen


def attention(q, k, v, past, scale, parents=None, window=0):
    """One sequence: q [tokens, heads, dim], k and v [slots, kv_heads, dim]; also sum p |v| and the scores' size."""
    tokens, heads, dim = q.shape
    group = heads // k.shape[1]
    n = past + tokens
    seen = sees(past, tokens, parents, window)
    out, weight, size = (np.zeros(q.shape) for _ in range(3))
    for h in range(heads):
        kh, vh = k[:n, h // group].astype(np.float64), v[:n, h // group].astype(np.float64)
        for t in range(tokens):
            at = seen[t]
            if not at.any():
                continue
            s = kh[at] @ q[t, h].astype(np.float64) * scale
            p = np.exp(s - s.max())
            p /= p.sum()
            out[t, h], weight[t, h] = p @ vh[at], p @ np.abs(vh[at])
            size[t, h] = (np.abs(kh[at]) @ np.abs(q[t, h].astype(np.float64))).max() * abs(scale)
    return out, weight, size


def attention_bound(weight, size, slots, dim):
    """How far the kernel may be. A score: its query's parts leave 2^-21, its f32 sums round at most dim times at 2^-24
    of sum |q k|, and again exp2's argument, of that size at the most, at 2^-23. Those move p by a factor, so o by twice as
    much of sum p |v|; the probabilities' own parts leave 2^-20; the outputs' f32 sums round once for each of a wave's
    tiles, 32 times in one and 8 in the joins."""
    u = 2.0 ** -24
    return weight * (2 * size * (8 * u + dim * u + 4 * u) + 16 * u + (slots / 32 + 40) * u) + 1e-30


def units(x):
    x = np.asarray(x, np.float32)
    x = np.where(np.isnan(x), np.float32(0), np.clip(x, 0, 1)).astype(np.float64)
    return [int(v) for v in np.floor(x * 2.0 ** 44)]


def drawn(row, uniform):
    w = units(row)
    total = sum(w)
    if total == 0:
        return 0
    r = int(np.floor(np.float64(min(max(np.float32(uniform), np.float32(0)), np.float32(0.99999994))) * 2.0 ** 31))
    at, so_far = total * r >> 31, 0
    for i, x in enumerate(w):
        so_far += x
        if so_far > at:
            return i
    raise AssertionError


def verify(node_tokens, target, uniforms, draft=None, accepts=None, parents=None, length=None):
    """One sequence: (path, emitted)."""
    n = len(node_tokens) if length is None else length
    vocabulary = target.shape[1]
    if n == 0:
        return [], []
    path, emitted = [0], []
    if draft is not None:
        while True:
            i = path[-1]
            if i + 1 == n:
                return path, emitted + [drawn(target[i], uniforms[i])]
            t = int(node_tokens[i + 1])
            if 0 <= t < vocabulary and np.float32(accepts[i + 1]) * draft[i][t] < target[i][t]:
                path.append(i + 1)
                emitted.append(t)
            else:
                return path, emitted + [drawn(target[i] - draft[i], uniforms[i])]
    while True:
        i = path[-1]
        t = drawn(target[i], uniforms[i])
        emitted.append(t)
        children = [j for j in range(i + 1, n) if (parents[j] == i if parents is not None else j == i + 1) and node_tokens[j] == t]
        if not children:
            return path, emitted
        path.append(children[0])


class Device:
    """Arrays on the device, freed together."""

    def __init__(self, ctx):
        self.ctx, self.owned = ctx, []

    def put(self, array, offset=0):
        """`offset` bytes into an allocation of its own: for alignments other than an allocation's."""
        a = np.ascontiguousarray(array)
        b = hx.Buffer(a.nbytes + offset + 16)
        b.write(a, offset)
        self.owned.append(b)
        return b.ptr + offset

    def room(self, count, dtype=np.float32, offset=0, byte=0xFF):
        b = hx.Buffer(count * np.dtype(dtype).itemsize + offset)
        b.fill(byte)
        self.owned.append(b)
        return b.ptr + offset, lambda: b.read(dtype, count, offset)

    def free(self):
        hx.sync()
        for b in self.owned:
            b.free()
        self.owned = []

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.free()

    def cache(self, format_, k, v, capacity, past=None, device=None, nbytes=0):
        """A cache holding k, v [sequences, tokens, kv_heads, dim] from slot past (0) on."""
        s, n, heads, dim = k.shape
        c = sv.Cache(self.ctx, FORMATS[format_], s, heads, dim, capacity, device=device, nbytes=nbytes)
        if n:
            first = self.put(np.full(s, 0 if past is None else past, np.uint32))
            c.append(self.put(k.astype(np.float32)), self.put(v.astype(np.float32)), first, n)
            hx.sync()
        return c

    def attend(self, cache, q, past, scale, parents=None, window=0, longest=0, query_stride=0, output_stride=0):
        """q [sequences, tokens, heads, dim] -> the same shape."""
        s, tokens, heads, dim = q.shape
        width = heads * dim
        rows = np.zeros((s * tokens, query_stride or width), np.float32)
        rows[:, :width] = q.reshape(s * tokens, width)
        need = sv.attention_workspace_bytes(self.ctx, cache, heads, tokens)
        work, _ = self.room(max(need, 16), np.uint8)
        out, read = self.room(s * tokens * (output_stride or width))
        call = sv.Attention(cache, self.put(rows), out, heads, scale, past=self.put(np.asarray(past, np.uint32)),
                            parents=0 if parents is None else self.put(np.asarray(parents, np.int32)), window=window,
                            longest=longest, query_stride=query_stride, output_stride=output_stride, workspace=work,
                            workspace_bytes=need)
        sv.attention(self.ctx, call, tokens)
        hx.sync()
        return read().reshape(s * tokens, output_stride or width)[:, :width].reshape(q.shape)
