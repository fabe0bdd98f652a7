"""What a decoder step runs between its products and after its head, over the
C ABI (include/charlotte_hip_matmul.h): norms of queries and keys with the
position rotation, the quantized cache, attention over it for one token, a
chain or a tree of drafted ones, softmax of the head's logits, and the
verification of drafted tokens.

As in charlotte_amd.matmul, calls take device pointers (ints), run on a HIP
stream, allocate nothing (a Cache aside) and raise ``MatmulError``. Lengths and
positions are device memory, so a captured step can be replayed as they grow.
Activations are f32. charlotte_amd/speculative.py runs them together.
"""

import ctypes
import enum
import itertools
from dataclasses import dataclass, field
from typing import Optional, Sequence

from charlotte_amd.matmul import (
    Context, TensorType, _AttentionDesc, _Heads, _HeadNormRopeDesc, _ProbabilitiesDesc, _VerifyDesc, lib)

# The most tokens of a sequence a step with parents may hold.
TREE_TOKENS = 256


class Rope(enum.IntEnum):
    """How a head's values pair for the rotation: i with i + rope_dims / 2, or 2i with 2i + 1."""

    NoRope = 0
    Halves = 1
    Neighbours = 2


def rope_table(positions, rope_dims, base=10000.0, factors=None):
    """The tables head_norm_rope reads, cosines and sines [positions][rope_dims / 2] in f32, from angles in f64:
    position p's pair i turns by p * base^(-2i / rope_dims), divided by factors[i] where given."""
    import numpy as np

    frequencies = float(base) ** (-np.arange(0, rope_dims, 2, dtype=np.float64) / rope_dims)
    if factors is not None:
        frequencies = frequencies / np.asarray(factors, np.float64)
    angles = np.arange(positions, dtype=np.float64)[:, None] * frequencies
    return np.cos(angles).astype(np.float32), np.sin(angles).astype(np.float32)


class _Call:
    """A call's fields, whose C descriptor is built for the first call and after a field is set."""

    def __setattr__(self, name, value):
        object.__setattr__(self, name, value)
        if name != "_desc":
            object.__setattr__(self, "_desc", None)


_STAMPS = itertools.count()


@dataclass
class Heads:
    """The queries or the keys of a step: charlotte_hip_matmul_heads."""

    input: int
    output: int
    heads: int
    weight: int = 0
    input_stride: int = 0
    output_stride: int = 0

    def __setattr__(self, name, value):
        object.__setattr__(self, name, value)
        object.__setattr__(self, "_stamp", next(_STAMPS))  # no other state of any Heads has it


@dataclass
class HeadNormRope(_Call):
    """charlotte_hip_matmul_head_norm_rope_desc."""

    parts: Sequence[Heads]
    head_dim: int
    epsilon: float = 1e-6
    rope: Rope = Rope.Halves
    rope_dims: int = 0
    cosines: int = 0
    sines: int = 0
    table_rows: int = 0
    positions: int = 0
    _desc: Optional[_HeadNormRopeDesc] = field(default=None, repr=False)

    def desc(self):
        d = _HeadNormRopeDesc()
        for i, p in enumerate(self.parts[:2]):
            d.parts[i] = _Heads(p.input, p.output, p.input_stride, p.output_stride, p.weight, p.heads, 0)
        d.part_count, d.head_dim = len(self.parts), self.head_dim
        d.rope, d.rope_dims = int(self.rope), self.rope_dims
        d.cosines, d.sines, d.positions, d.table_rows = self.cosines, self.sines, self.positions, self.table_rows
        d.epsilon = self.epsilon
        d.stamps = [p._stamp for p in self.parts]
        return d


def head_norm_rope(ctx: Context, call: HeadNormRope, tokens: int, stream=None):
    """Each head normalised and rotated, queries and keys in one launch."""
    if call._desc is None or call._desc.stamps != [p._stamp for p in call.parts]:
        call._desc = call.desc()
    ctx.check(lib.charlotte_hip_matmul_head_norm_rope(ctx.handle, ctypes.byref(call._desc), tokens, stream))


def cache_bytes(gguf_type, sequences, kv_heads, head_dim, capacity):
    return lib.charlotte_hip_matmul_cache_bytes(int(gguf_type), sequences, kv_heads, head_dim, capacity)


class Cache:
    """Keys and values of `sequences` sequences of up to `capacity` tokens, in Q8_0, Q4_0 or F16
    (charlotte_hip_matmul_cache); in memory of its own, or in `device` (nbytes of it), borrowed."""

    def __init__(self, ctx: Context, gguf_type, sequences, kv_heads, head_dim, capacity, device=None, nbytes=0):
        self.handle = None
        h = ctypes.c_void_p()
        shape = (int(gguf_type), sequences, kv_heads, head_dim, capacity)
        if device is None:
            ctx.check(lib.charlotte_hip_matmul_cache_create(ctx.handle, *shape, ctypes.byref(h)))
        else:
            ctx.check(lib.charlotte_hip_matmul_cache_wrap(ctx.handle, *shape, device, nbytes, ctypes.byref(h)))
        self.ctx, self.handle, self.type = ctx, h, TensorType(gguf_type)
        self.sequences, self.kv_heads, self.head_dim, self.capacity = sequences, kv_heads, head_dim, capacity

    def append(self, keys, values, past, tokens, key_stride=0, value_stride=0, stream=None):
        """The step's keys and values, quantized, into slots past[s] .. past[s] + tokens - 1."""
        self.ctx.check(lib.charlotte_hip_matmul_cache_append(self.ctx.handle, self.handle, keys, values, key_stride,
                                                             value_stride, past, tokens, stream))

    def read(self, keys, values, first, tokens, key_stride=0, value_stride=0, stream=None):
        """Slots first[s] .. first[s] + tokens - 1 as the f32 values they stand for."""
        self.ctx.check(lib.charlotte_hip_matmul_cache_read(self.ctx.handle, self.handle, keys, values, key_stride,
                                                           value_stride, first, tokens, stream))

    def keep(self, past, path, count, tokens, stream=None):
        """The accepted path's slots moved together behind past[s] (verify's path and count)."""
        self.ctx.check(lib.charlotte_hip_matmul_cache_keep(self.ctx.handle, self.handle, past, path, count, tokens,
                                                           stream))

    def free(self):
        if self.handle and lib:
            lib.charlotte_hip_matmul_cache_free(self.handle)
            self.handle = None

    def __del__(self):
        self.free()


@dataclass
class Attention(_Call):
    """charlotte_hip_matmul_attention_desc."""

    cache: Cache
    queries: int
    output: int
    query_heads: int
    scale: float
    past: int = 0
    parents: int = 0
    window: int = 0
    longest: int = 0
    query_stride: int = 0
    output_stride: int = 0
    workspace: int = 0
    workspace_bytes: int = 0
    _desc: Optional[_AttentionDesc] = field(default=None, repr=False)

    def desc(self):
        return _AttentionDesc(self.cache.handle, self.queries, self.output, self.query_stride, self.output_stride,
                              self.query_heads, self.window, self.scale, self.longest, self.past, self.parents,
                              self.workspace, self.workspace_bytes)


def attention_workspace_bytes(ctx: Context, cache: Cache, query_heads: int, tokens: int):
    return lib.charlotte_hip_matmul_attention_workspace_bytes(ctx.handle, cache.handle, query_heads, tokens)


def attention(ctx: Context, call: Attention, tokens: int, stream=None):
    """The step's tokens, already appended, over their sequences' caches."""
    if call._desc is None or not call.cache.handle:  # (a cache that was freed is refused)
        call._desc = call.desc()
    ctx.check(lib.charlotte_hip_matmul_attention(ctx.handle, ctypes.byref(call._desc), tokens, stream))


@dataclass
class Probabilities(_Call):
    """charlotte_hip_matmul_probabilities_desc."""

    logits: int
    output: int
    rows: int
    vocabulary: int
    temperature: float = 1.0
    logit_stride: int = 0
    output_stride: int = 0
    workspace: int = 0
    workspace_bytes: int = 0
    _desc: Optional[_ProbabilitiesDesc] = field(default=None, repr=False)

    def desc(self):
        return _ProbabilitiesDesc(self.logits, self.output, self.logit_stride, self.output_stride, self.rows,
                                  self.vocabulary, self.temperature, 0, self.workspace, self.workspace_bytes)


def probabilities_workspace_bytes(rows: int, vocabulary: int):
    return lib.charlotte_hip_matmul_probabilities_workspace_bytes(rows, vocabulary)


def probabilities(ctx: Context, call: Probabilities, stream=None):
    """softmax(logits / temperature), row by row; at temperature 0 the largest's one."""
    if call._desc is None:
        call._desc = call.desc()
    ctx.check(lib.charlotte_hip_matmul_probabilities(ctx.handle, ctypes.byref(call._desc), stream))


@dataclass
class Verify(_Call):
    """charlotte_hip_matmul_verify_desc."""

    node_tokens: int
    target: int
    uniforms: int
    vocabulary: int
    path: int
    emitted: int
    count: int
    draft: int = 0
    accepts: int = 0
    parents: int = 0
    lengths: int = 0
    target_stride: int = 0
    draft_stride: int = 0
    workspace: int = 0
    workspace_bytes: int = 0
    _desc: Optional[_VerifyDesc] = field(default=None, repr=False)

    def desc(self):
        return _VerifyDesc(self.node_tokens, self.target, self.draft, self.uniforms, self.accepts, self.parents,
                           self.lengths, self.path, self.emitted, self.count, self.target_stride, self.draft_stride,
                           self.vocabulary, 0, self.workspace, self.workspace_bytes)


def verify_workspace_bytes(sequences: int, tokens: int, vocabulary: int):
    return lib.charlotte_hip_matmul_verify_workspace_bytes(sequences, tokens, vocabulary)


def verify(ctx: Context, call: Verify, sequences: int, tokens: int, stream=None):
    """The drafted tokens accepted, and the one drawn after them, of every sequence."""
    if call._desc is None:
        call._desc = call.desc()
    ctx.check(lib.charlotte_hip_matmul_verify(ctx.handle, ctypes.byref(call._desc), sequences, tokens, stream))
