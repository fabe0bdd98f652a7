"""The steps between a decoder step's products and after its head
(charlotte_amd.serving) on the device, against plain restatements in 64 bits:
every head width, format, mask and length at which they can go wrong. The
cache's blocks and the verification's tokens are compared exactly."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.fixture(scope="module")
def ctx():
    from charlotte_amd import matmul as mm

    c = mm.Context(0)
    yield c
    c.close()


@pytest.fixture
def dev(ctx):
    from tests.support.serving_ref import Device

    with Device(ctx) as d:
        yield d


# ---- head_norm_rope ---------------------------------------------------------


def _heads_exact(x, weight, epsilon, pairing, rope_dims, cosines, sines):
    """x [tokens, heads, dim]; also |a c| + |b s| of every value (the error's scale)."""
    y = x.astype(np.float64)
    if weight is not None:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + np.float32(epsilon)) * weight.astype(np.float64)
    size = np.abs(y)
    if pairing != "NoRope":
        half = rope_dims // 2
        first = np.arange(half) * (1 if pairing == "Halves" else 2)
        second = first + (half if pairing == "Halves" else 1)
        a, b = y[..., first], y[..., second]
        c, s = cosines.astype(np.float64)[:, None], sines.astype(np.float64)[:, None]
        y, size = y.copy(), size.copy()
        y[..., first], y[..., second] = a * c - b * s, b * c + a * s
        size[..., first], size[..., second] = np.abs(a * c) + np.abs(b * s), np.abs(b * c) + np.abs(a * s)
    return y, size


@pytest.mark.parametrize("dim,rope_dims,pairing,norm,tokens,heads", [
    (128, 128, "Halves", True, 1, (16, 8)), (128, 64, "Halves", True, 7, (4, 2)), (64, 64, "Neighbours", False, 5, (32, 8)),
    (256, 256, "Halves", True, 3, (4, 1)), (96, 96, "Halves", True, 9, (3, 1)), (96, 40, "Neighbours", True, 2, (5, 5)),
    (32, 8, "Halves", True, 33, (1, 1)), (160, 160, "Halves", False, 2, (7, 7)), (8, 8, "Neighbours", True, 11, (3, 2)),
    (24, 16, "Halves", True, 5, (2, 1)), (200, 104, "Halves", True, 3, (2, 3)), (128, 128, "NoRope", True, 4, (2, 2)),
    (224, 224, "Neighbours", True, 300, (9, 3))])
@pytest.mark.parametrize("fused", [False, True])
def test_head_norm_rope(ctx, dev, dim, rope_dims, pairing, norm, tokens, heads, fused):
    from charlotte_amd import harness as hx
    from charlotte_amd import serving as sv

    rng = np.random.default_rng(dim * tokens + fused)
    positions = rng.integers(0, 500, tokens).astype(np.uint32)
    cosines, sines = sv.rope_table(500, rope_dims)
    # queries and keys read out of one buffer, written in place; or apart
    width = sum(heads) * dim + (12 if fused else 0)
    rows = (rng.standard_normal((tokens, width)) * 3).astype(np.float32)
    rows[0, :dim] = 0.0  # a head of zeros: epsilon alone
    base = dev.put(rows)
    parts, want, reads, at = [], [], [], 0
    for h in heads:
        x = rows[:, at:at + h * dim].reshape(tokens, h, dim)
        w = (1 + 0.3 * rng.standard_normal(dim)).astype(np.float32) if norm else None
        want.append(_heads_exact(x, w, 1e-6, pairing, rope_dims, cosines[positions], sines[positions]))
        if fused:
            to, stride = base + 4 * at, width
        else:
            to, read = dev.room(tokens * h * dim)
            stride = 0
            reads.append(read)
        parts.append(sv.Heads(base + 4 * at, to, h, weight=dev.put(w) if norm else 0, input_stride=width,
                              output_stride=stride))
        at += h * dim
    call = sv.HeadNormRope(parts, dim, rope=sv.Rope[pairing], rope_dims=rope_dims, cosines=dev.put(cosines),
                           sines=dev.put(sines), table_rows=500, positions=dev.put(positions))
    print("head_norm_rope", dim, rope_dims, pairing, tokens, heads, fused, flush=True)
    sv.head_norm_rope(ctx, call, tokens)
    hx.sync()
    if fused:
        whole = dev.owned[0].read(np.float32, rows.size).reshape(rows.shape)
        assert (whole[:, at:] == rows[:, at:]).all()  # what lies beside the heads
        got = [whole[:, :heads[0] * dim], whole[:, heads[0] * dim:at]]
    else:
        got = [r().reshape(tokens, -1) for r in reads]
    for (y, size), g in zip(want, got):
        # 9 roundings of the squares' sum, 2 of the mean, halved by the root, and 6 more
        assert (np.abs(g.reshape(y.shape) - y) <= 12 * U * size + 1e-30).all()


def test_head_norm_rope_takes_a_position_past_the_tables_as_nan(ctx, dev):
    from charlotte_amd import harness as hx
    from charlotte_amd import serving as sv

    x = np.ones((3, 2 * 64), np.float32)
    cosines, sines = sv.rope_table(10, 32)
    to, read = dev.room(x.size)
    call = sv.HeadNormRope([sv.Heads(dev.put(x), to, 2)], 64, rope_dims=32, cosines=dev.put(cosines), sines=dev.put(sines),
                           table_rows=10, positions=dev.put(np.array([9, 10, 0xFFFFFFFF], np.uint32)))
    sv.head_norm_rope(ctx, call, 3)
    hx.sync()
    got = read().reshape(3, 2, 64)
    assert np.isfinite(got[0]).all()
    assert np.isnan(got[1:, :, :32]).all() and (got[1:, :, 32:] == 1).all()


# ---- the cache ------------------------------------------------------------------


def _edge_values(rng, shape):
    """Blocks with everything a format has to decide about among ordinary ones."""
    x = (rng.standard_normal(shape) * 2).astype(np.float32)
    b = x.reshape(-1, 32)
    special = [0.0, 1e-7, 3e-8, 1e-12, 65504.0, 65519.9, 65520.0, 1e5, 8e6, 8.4e6, 1e30, np.inf, -np.inf, np.nan, -0.0, 1e-39]
    for i, value in enumerate(special):
        if 2 * i + 1 < len(b):
            b[2 * i + 1, (5 * i) % 32] = value
            if i in (1, 2, 3, 15):  # nothing larger beside it
                b[2 * i + 1] = np.where(np.arange(32) == (5 * i) % 32, np.float32(value), np.float32(value) / 3)
    if len(b) > 40:
        b[40] = 0
        b[38, 3], b[38, 9] = 7.0, -7.0  # the first of two equal magnitudes
        b[36, 9], b[36, 30] = -9.0, 9.0
    return x


@pytest.mark.parametrize("format_", ["q8_0", "q4_0", "f16"])
@pytest.mark.parametrize("sequences,heads,dim,tokens,past,capacity", [
    (1, 8, 128, 1, 0, 1), (1, 2, 64, 5, 30, 64), (2, 3, 96, 33, 7, 41), (3, 1, 256, 31, 1, 32), (1, 4, 32, 100, 29, 129),
    (2, 1, 160, 64, 32, 100)])
def test_a_cache_reads_back_what_its_format_holds(ctx, dev, format_, sequences, heads, dim, tokens, past, capacity):
    from charlotte_amd import harness as hx
    from tests.support import serving_ref as ref

    rng = np.random.default_rng(dim + tokens)
    # sequences at different lengths, rows with space between them
    first = np.array([min(past + 3 * s, capacity - tokens) for s in range(sequences)], np.uint32)
    k, v = (_edge_values(rng, (sequences * tokens, heads * dim)) for _ in range(2))
    pad = np.full((sequences * tokens, 8), 5.0, np.float32)
    print("cache", format_, sequences, heads, dim, tokens, past, capacity, flush=True)
    c = dev.cache(format_, np.zeros((sequences, 0, heads, dim)), np.zeros(0), capacity)
    slots = dev.put(first)
    c.append(dev.put(np.concatenate([k, pad], 1)), dev.put(v), slots, tokens, key_stride=heads * dim + 8)
    (ko, kr), (vo, vr) = dev.room(k.size), dev.room(sequences * tokens * (heads * dim + 4))
    c.read(ko, vo, slots, tokens, value_stride=heads * dim + 4)
    hx.sync()
    got_k = kr().reshape(k.shape)
    got_v = vr().reshape(sequences * tokens, -1)[:, :heads * dim]
    assert np.array_equal(got_k, ref.stored(k, format_), equal_nan=True)
    assert np.array_equal(got_v, ref.stored(v, format_), equal_nan=True)
    c.free()


@pytest.mark.parametrize("format_,most", [("q8_0", 127), ("q4_0", 8)])
@pytest.mark.parametrize("tokens", [16, 64])
def test_codes_at_every_scale(ctx, dev, format_, most, tokens):
    """Every finite scale of binary16 above zero, and around each tie between two codes
    the values next to it: the code is that of the quotient, rounded once."""
    from charlotte_amd import harness as hx
    from tests.support import serving_ref as ref

    rng = np.random.default_rng(51)
    d = np.arange(1, 0x7C00, dtype=np.uint16).view(np.float16).astype(np.float32)
    blocks = -(-len(d) // (tokens * 8)) * tokens * 8
    d = np.concatenate([d, np.ones(blocks - len(d), np.float32)])
    half = rng.integers(-most, most, (blocks, 32)) + np.float32(0.5)
    x = (half * d[:, None]).astype(np.float32)
    beside = [x, np.nextafter(x, np.float32(np.inf)), np.nextafter(x, np.float32(-np.inf))]
    x = np.choose(rng.integers(0, 3, x.shape), beside)
    x[:, 5] = -most * d  # the scale is d
    assert (np.abs(x) <= most * d[:, None]).all()
    sequences = blocks // (tokens * 8)
    x = x.reshape(sequences * tokens, 8 * 32)
    c = dev.cache(format_, np.zeros((sequences, 0, 2, 128)), None, tokens)
    zero = dev.put(np.zeros(sequences, np.uint32))
    c.append(dev.put(x), dev.put(x), zero, tokens)
    (ko, kr), (vo, vr) = dev.room(x.size), dev.room(x.size)
    c.read(ko, vo, zero, tokens)
    hx.sync()
    want = ref.stored(x, format_)
    assert np.array_equal(kr().reshape(x.shape), want) and np.array_equal(vr().reshape(x.shape), want)
    c.free()


@pytest.mark.parametrize("format_", ["q8_0", "q4_0", "f16"])
def test_appending_leaves_the_other_slots(ctx, dev, format_):
    from charlotte_amd import harness as hx
    from tests.support import serving_ref as ref

    rng = np.random.default_rng(5)
    k, v = (rng.standard_normal((1, 70, 2, 64)).astype(np.float32) for _ in range(2))
    c = dev.cache(format_, k, v, 70)
    one = rng.standard_normal((1, 1, 2, 64)).astype(np.float32)
    for slot in (0, 17, 33, 69):
        c.append(dev.put(one), dev.put(one), dev.put(np.array([slot], np.uint32)), 1)
        k[0, slot] = v[0, slot] = one[0, 0]
    # past the capacity: the first of these two tokens has a slot, the second none
    c.append(dev.put(np.repeat(one, 2, 1) * 2), dev.put(np.repeat(one, 2, 1) * 2), dev.put(np.array([69], np.uint32)), 2)
    c.append(dev.put(one), dev.put(one), dev.put(np.array([0xFFFFFFFF], np.uint32)), 1)
    k[0, 69] = v[0, 69] = one[0, 0] * 2
    (ko, kr), (vo, vr) = dev.room(k.size), dev.room(v.size)
    c.read(ko, vo, dev.put(np.zeros(1, np.uint32)), 70)
    hx.sync()
    assert np.array_equal(kr().reshape(k.shape), ref.stored(k, format_))
    assert np.array_equal(vr().reshape(v.shape), ref.stored(v, format_))
    c.free()


@pytest.mark.parametrize("format_", ["q8_0", "q4_0", "f16"])
def test_keep_moves_an_accepted_path_together(ctx, dev, format_):
    from charlotte_amd import harness as hx
    from tests.support import serving_ref as ref

    rng = np.random.default_rng(6)
    tokens, capacity = 40, 100
    k, v = (rng.standard_normal((3, capacity, 2, 96)).astype(np.float32) for _ in range(2))
    c = dev.cache(format_, k, v, capacity)
    past = np.array([20, 31, 90], np.uint32)
    paths = [[0, 3, 4, 9, *range(15, 39)], [5, 2, 7], [0, 4, 9, 10, 11]]  # the second does not rise, the third leaves the cache
    moved = [len(paths[0]), 1, 3]
    path = np.full((3, tokens), -1, np.int32)
    for i, p in enumerate(paths):
        path[i, :len(p)] = p
    c.keep(dev.put(past), dev.put(path), dev.put(np.array([len(p) for p in paths], np.uint32)), tokens)
    (ko, kr), (vo, vr) = dev.room(k.size), dev.room(v.size)
    c.read(ko, vo, dev.put(np.zeros(3, np.uint32)), capacity)
    hx.sync()
    for x in (k, v):
        for i in range(3):
            before = x[i].copy()
            for j in range(moved[i]):
                x[i, past[i] + j] = before[past[i] + paths[i][j]]
    assert np.array_equal(kr().reshape(k.shape), ref.stored(k, format_))
    assert np.array_equal(vr().reshape(v.shape), ref.stored(v, format_))
    c.free()


# ---- attention ----------------------------------------------------------------------


def _check_attention(dev, format_, sequences, heads, kv_heads, dim, tokens, past, parents=None, window=0, scale=None,
                     seed=0, spread=1.0, capacity=None, **kw):
    from tests.support import serving_ref as ref

    rng = np.random.default_rng(seed)
    past = np.asarray(past)
    slots = int(past.max()) + tokens
    k = rng.standard_normal((sequences, slots, kv_heads, dim)).astype(np.float32)
    v = (rng.standard_normal((sequences, slots, kv_heads, dim)) * spread).astype(np.float32)
    q = rng.standard_normal((sequences, tokens, heads, dim)).astype(np.float32)
    scale = dim ** -0.5 if scale is None else scale
    print("attention", format_, sequences, heads, kv_heads, dim, tokens, past.tolist(), window, flush=True)
    c = dev.cache(format_, k, v, capacity or slots)
    got = dev.attend(c, q, past, scale, parents=parents, window=window, **kw)
    for s in range(sequences):
        line = None if parents is None else parents[s]
        want, weight, size = ref.attention(q[s], ref.stored(k[s], format_), ref.stored(v[s], format_), int(past[s]), scale,
                                           line, window)
        assert (np.abs(got[s] - want) <= ref.attention_bound(weight, size, past[s] + tokens, dim)).all()
        assert np.abs(got[s] - want).max() <= 1e-5 * np.abs(want).max()  # the tolerance of the library's other paths
    c.free()
    return got


@pytest.mark.parametrize("format_", ["q8_0", "q4_0", "f16"])
@pytest.mark.parametrize("dim", [32, 64, 96, 128, 160, 192, 224, 256])
def test_attention_at_every_head_width(ctx, dev, format_, dim):
    _check_attention(dev, format_, 1, 4, 2, dim, 1, [70], seed=dim)       # a token: two rows
    _check_attention(dev, format_, 1, 6, 2, dim, 13, [45], seed=dim + 1)  # 39 rows


@pytest.mark.parametrize("format_", ["q8_0", "q4_0", "f16"])
@pytest.mark.parametrize("dim", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("tokens", [19, 41, 91])
def test_attention_of_many_rows_at_every_head_width(ctx, dev, format_, dim, tokens):
    """57, 123 and 273 rows of a key head: workgroups of four waves and of eight, the last with few rows."""
    _check_attention(dev, format_, 1, 3, 1, dim, tokens, [150], seed=dim + tokens)


@pytest.mark.parametrize("format_", ["q8_0", "f16"])
@pytest.mark.parametrize("tokens,past,heads,kv_heads", [
    (1, 0, 4, 4), (1, 1, 8, 1), (1, 31, 2, 2), (1, 32, 2, 1), (1, 2000, 16, 8), (2, 0, 7, 1), (5, 27, 3, 3), (32, 0, 2, 1),
    (33, 95, 5, 1), (64, 64, 4, 4), (200, 0, 3, 1), (130, 333, 6, 2), (1, 5000, 24, 3), (17, 1, 33, 1)])
def test_attention_of_a_token_and_of_chains(ctx, dev, format_, tokens, past, heads, kv_heads):
    _check_attention(dev, format_, 1, heads, kv_heads, 64, tokens, [past], seed=tokens + past)


def _random_tree(rng, tokens, unused=()):
    parents = np.array([rng.integers(max(-1, t - 6), t) for t in range(tokens)], np.int32)
    parents[0] = -1
    for t in unused:
        parents[t] = -2
    return parents


@pytest.mark.parametrize("format_", ["q8_0", "q4_0", "f16"])
@pytest.mark.parametrize("tokens,past,sequences", [(2, 0, 1), (21, 500, 2), (64, 31, 1), (256, 40, 1), (40, 1999, 3), (1, 9, 2)])
@pytest.mark.parametrize("window", [0, 3, 37])
def test_attention_of_a_tree(ctx, dev, format_, tokens, past, sequences, window):
    rng = np.random.default_rng(tokens + window)
    parents = np.stack([_random_tree(rng, tokens) for _ in range(sequences)])
    lengths = [max(0, past - 5 * s) for s in range(sequences)]
    _check_attention(dev, format_, sequences, 4, 2, 64, tokens, lengths, parents=parents, window=window, seed=tokens)


@pytest.mark.parametrize("window", [1, 2, 31, 64, 100, 1000])
@pytest.mark.parametrize("tokens,past", [(1, 200), (1, 63), (20, 150), (70, 10)])
def test_attention_in_a_window(ctx, dev, tokens, past, window):
    _check_attention(dev, "q8_0", 1, 4, 1, 128, tokens, [past], window=window, seed=window)


def test_a_tree_of_a_line_is_a_chain(ctx, dev):
    a = _check_attention(dev, "q8_0", 1, 8, 2, 128, 24, [77], seed=3)
    b = _check_attention(dev, "q8_0", 1, 8, 2, 128, 24, [77], parents=np.arange(-1, 23)[None], seed=3)
    assert (a == b).all()


def test_unused_tokens_see_nothing_and_are_seen_by_none(ctx, dev):
    rng = np.random.default_rng(8)
    parents = _random_tree(rng, 30, unused=(4, 11))
    parents[20], parents[25], parents[29] = 25, 25, 1000  # not below their token
    parents[7], parents[8] = 4, 7  # under an unused one
    got = _check_attention(dev, "f16", 1, 4, 2, 64, 30, [50], parents=parents[None], seed=9)
    for t in (4, 11, 20, 25, 29, 7, 8):
        assert (got[0, t] == 0).all() and not np.signbit(got[0, t]).any()
    # a step of nothing but unused tokens, over an empty cache and over a full one
    for past in (0, 100):
        got = _check_attention_empty(dev, past)
        assert (got == 0).all()


def _check_attention_empty(dev, past):
    rng = np.random.default_rng(1)
    k = rng.standard_normal((1, past + 3, 1, 64)).astype(np.float32)
    c = dev.cache("q8_0", k, k, past + 3)
    got = dev.attend(c, rng.standard_normal((1, 3, 2, 64)).astype(np.float32), [past], 0.1, parents=[[-2, -2, -2]])
    c.free()
    return got


@pytest.mark.parametrize("longest", [1, 40, 1 << 30])
def test_the_bound_on_lengths_changes_no_answer(ctx, dev, longest):
    _check_attention(dev, "q4_0", 2, 8, 4, 64, 3, [700, 40], longest=longest, capacity=5000)


def test_strides_and_rows_beside_them(ctx, dev):
    _check_attention(dev, "q8_0", 2, 4, 2, 96, 3, [40, 77], query_stride=4 * 96 + 64, output_stride=4 * 96 + 20)


@pytest.mark.parametrize("format_", ["q8_0", "q4_0", "f16"])
@pytest.mark.parametrize("spread", [1e-4, 0.01, 300.0, 30000.0])
def test_values_of_any_size_keep_their_precision(ctx, dev, format_, spread):
    if format_ == "f16":
        spread = min(spread, 10000.0)
    if format_ == "q4_0":
        spread = max(spread, 0.01)
    _check_attention(dev, format_, 1, 4, 2, 64, 5, [300], spread=spread, seed=4)


def test_values_that_grow_along_the_cache(ctx, dev):
    """Every few tiles a larger scale than all before it, and a larger score."""
    from tests.support import serving_ref as ref

    rng = np.random.default_rng(12)
    n = 900
    grow = 2.0 ** (np.arange(n) / 40)
    k = (rng.standard_normal((1, n, 1, 64)) * 0.3).astype(np.float32)
    v = (rng.standard_normal((1, n, 1, 64)) * grow[None, :, None, None] * 1e-3).astype(np.float32)
    q = (rng.standard_normal((1, 2, 3, 64)) * 2).astype(np.float32)
    for turned in (False, True):
        kk, vv = (x[:, ::-1].copy() if turned else x for x in (k, v))
        c = dev.cache("q8_0", kk, vv, n)
        got = dev.attend(c, q, [n - 2], 1.0)
        want, weight, size = ref.attention(q[0], ref.stored(kk[0], "q8_0"), ref.stored(vv[0], "q8_0"), n - 2, 1.0)
        assert (np.abs(got[0] - want) <= ref.attention_bound(weight, size, n, 64)).all()
        c.free()


@pytest.mark.parametrize("format_", ["q8_0", "q4_0", "f16"])
def test_what_a_row_does_not_see_does_not_reach_it(ctx, dev, format_):
    """NaNs and infinities in a sibling's keys and values, in what lies past the
    last token, and in tokens before a window."""
    from tests.support import serving_ref as ref

    rng = np.random.default_rng(13)
    past, tokens = 61, 6
    parents = np.array([[-1, 0, 0, 1, 2, 3]], np.int32)  # 0-1-3-5 and 0-2-4
    shape = (1, past + tokens + 40, 2, 64)
    k, v = (rng.standard_normal(shape).astype(np.float32) for _ in range(2))
    clean_k, clean_v = k.copy(), v.copy()
    k[0, past + 2, 0, 5], v[0, past + 2, :, 40] = np.nan, np.inf   # the second line alone sees token 2
    v[0, past + 2, 1, 3] = np.nan
    k[0, past + tokens:], v[0, past + tokens:] = np.nan, np.nan    # stale slots
    q = rng.standard_normal((1, tokens, 4, 64)).astype(np.float32)
    c = dev.cache(format_, k, v, shape[1])
    got = dev.attend(c, q, [past], 0.125, parents=parents)
    want, weight, size = ref.attention(q[0], ref.stored(clean_k[0], format_), ref.stored(clean_v[0], format_), past, 0.125,
                                       parents[0])
    for t in (0, 1, 3, 5):
        assert (np.abs(got[0, t] - want[t]) <= ref.attention_bound(weight, size, past + tokens, 64)[t]).all()
    for t in (2, 4):
        assert np.isnan(got[0, t, :2]).all()                 # a NaN score
        assert np.isnan(got[0, t, 2:]).all(0)[:].sum() == 64  # both blocks of its values
    # before a window
    k[0, :20], v[0, :20] = np.inf, np.nan
    k[0, 20:past + tokens], v[0, 20:past + tokens] = clean_k[0, 20:past + tokens], clean_v[0, 20:past + tokens]
    c2 = dev.cache(format_, k, v, shape[1])
    got = dev.attend(c2, q, [past], 0.125, window=41)  # token 0 sees from slot 21
    want, weight, size = ref.attention(q[0], ref.stored(clean_k[0], format_), ref.stored(clean_v[0], format_), past, 0.125,
                                       window=41)
    assert (np.abs(got[0] - want) <= ref.attention_bound(weight, size, past + tokens, 64)).all()
    c.free()
    c2.free()


@pytest.mark.parametrize("format_", ["q8_0", "q4_0", "f16"])
@pytest.mark.parametrize("byte", [0xFF, 0x7E])
def test_a_cache_in_memory_of_any_contents(ctx, dev, format_, byte):
    """Every slot not appended is bytes that read as NaN scales and codes."""
    from charlotte_amd import serving as sv
    from tests.support import serving_ref as ref

    rng = np.random.default_rng(14)
    need = sv.cache_bytes(ref.FORMATS[format_], 1, 2, 96, 300)
    memory, _ = dev.room(need, np.uint8, byte=byte)
    k, v = (rng.standard_normal((1, 41, 2, 96)).astype(np.float32) for _ in range(2))
    c = dev.cache(format_, k, v, 300, device=memory, nbytes=need)
    q = rng.standard_normal((1, 3, 4, 96)).astype(np.float32)
    got = dev.attend(c, q, [38], 0.1)
    want, weight, size = ref.attention(q[0], ref.stored(k[0], format_), ref.stored(v[0], format_), 38, 0.1)
    assert (np.abs(got[0] - want) <= ref.attention_bound(weight, size, 41, 96)).all()
    c.free()


def test_queries_that_are_not_finite_spoil_their_own_row(ctx, dev):
    rng = np.random.default_rng(15)
    k = rng.standard_normal((1, 50, 2, 64)).astype(np.float32)
    q = rng.standard_normal((1, 4, 4, 64)).astype(np.float32)
    c = dev.cache("q8_0", k, k, 50)
    clean = dev.attend(c, q, [46], 0.1)
    q[0, 1, 2, 7], q[0, 2, 0, 63], q[0, 3, 3, 0] = np.nan, np.inf, -np.inf
    got = dev.attend(c, q, [46], 0.1)
    spoilt = np.zeros((4, 4), bool)
    spoilt[1, 2] = spoilt[2, 0] = spoilt[3, 3] = True
    assert np.isnan(got[0][spoilt]).all()
    assert (got[0][~spoilt] == clean[0][~spoilt]).all()
    c.free()


@pytest.mark.parametrize("size", [1e-38, 1e-12, 1e12, 1e34])
def test_queries_of_any_size(ctx, dev, size):
    from tests.support import serving_ref as ref

    rng = np.random.default_rng(16)
    k = rng.standard_normal((1, 90, 1, 64)).astype(np.float32)
    q = rng.standard_normal((1, 1, 2, 64)) * size
    c = dev.cache("q8_0", k, k, 90)
    got = dev.attend(c, q.astype(np.float32), [89], float(np.float32(0.125 / size)) if size < 1e30 else 1e-34)
    want, weight, span = ref.attention(q[0].astype(np.float32), ref.stored(k[0], "q8_0"), ref.stored(k[0], "q8_0"), 89,
                                       float(np.float32(0.125 / size)) if size < 1e30 else float(np.float32(1e-34)))
    if size > 1e-30:
        assert (np.abs(got[0] - want) <= ref.attention_bound(weight, span, 90, 64)).all()
    else:  # the queries are subnormal: they have few bits, and scale / ln 2 may pass f32
        assert np.isfinite(got).all() or np.isnan(got).all()
    c.free()


def test_offsets_past_32_bits(ctx, dev):
    """The last sequence's head lies over 4 GiB into its cache."""
    from charlotte_amd import harness as hx
    from charlotte_amd import serving as sv
    from tests.support import serving_ref as ref

    rng = np.random.default_rng(17)
    heads, dim, capacity = 4, 256, 700_000
    c = sv.Cache(ctx, ref.FORMATS["f16"], 2, heads, dim, capacity)
    assert sv.cache_bytes(ref.FORMATS["f16"], 2, heads, dim, capacity) > 5 << 30
    k, v = (rng.standard_normal((2, 40, heads, dim)).astype(np.float32) for _ in range(2))
    c.append(dev.put(k), dev.put(v), dev.put(np.array([0, 0], np.uint32)), 40)
    q = rng.standard_normal((2, 1, heads, dim)).astype(np.float32)
    got = dev.attend(c, q, [39, 39], 0.0625)
    for s in range(2):
        want, weight, size = ref.attention(q[s], ref.stored(k[s], "f16"), ref.stored(v[s], "f16"), 39, 0.0625)
        assert (np.abs(got[s] - want) <= ref.attention_bound(weight, size, 40, dim)).all()
    # and the last slots of the last sequence
    c.append(dev.put(k), dev.put(v), dev.put(np.array([capacity - 40] * 2, np.uint32)), 40)
    (ko, kr), (vo, vr) = dev.room(k.size), dev.room(v.size)
    c.read(ko, vo, dev.put(np.array([capacity - 40] * 2, np.uint32)), 40)
    got = dev.attend(c, q, [capacity - 1] * 2, 0.0625, window=40)
    hx.sync()
    assert np.array_equal(kr().reshape(k.shape), ref.stored(k, "f16"))
    assert np.array_equal(vr().reshape(v.shape), ref.stored(v, "f16"))
    for s in range(2):
        want, weight, size = ref.attention(q[s], ref.stored(k[s], "f16"), ref.stored(v[s], "f16"), 39, 0.0625)
        assert (np.abs(got[s] - want) <= ref.attention_bound(weight, size, 40, dim)).all()
    c.free()


def test_attention_is_the_same_bits_twice(ctx, dev):
    a = _check_attention(dev, "q8_0", 1, 16, 8, 128, 1, [3000], seed=21)
    b = _check_attention(dev, "q8_0", 1, 16, 8, 128, 1, [3000], seed=21)
    assert (a == b).all()


def test_a_captured_step_replays_as_its_cache_grows(ctx, dev):
    from charlotte_amd import harness as hx
    from charlotte_amd import serving as sv
    from tests.support import serving_ref as ref

    rng = np.random.default_rng(22)
    n, heads, dim = 200, 2, 64
    k, v = (rng.standard_normal((1, n, heads, dim)).astype(np.float32) for _ in range(2))
    q = rng.standard_normal((1, n, 4, dim)).astype(np.float32)
    c = dev.cache("q8_0", k[:, :150], v[:, :150], n)
    step_k, step_v, step_q = (hx.Buffer(4 * w) for w in (heads * dim, heads * dim, 4 * dim))
    past = hx.Buffer(16)
    out, read = dev.room(4 * dim)
    need = sv.attention_workspace_bytes(ctx, c, 4, 1)
    work, _ = dev.room(max(16, need), np.uint8)
    call = sv.Attention(c, step_q.ptr, out, 4, 0.125, past=past.ptr, workspace=work, workspace_bytes=need)
    stream = hx.Stream()

    def step():
        c.append(step_k.ptr, step_v.ptr, past.ptr, 1, stream=stream.handle)
        sv.attention(ctx, call, 1, stream=stream.handle)

    graph = hx.Graph(stream, step, global_mode=True)
    for at in range(150, 156):
        step_k.write(k[0, at])
        step_v.write(v[0, at])
        step_q.write(q[0, at])
        past.write(np.array([at], np.uint32))
        graph.launch()
        stream.sync()
        want, weight, size = ref.attention(q[0, at:at + 1], ref.stored(k[0], "q8_0"), ref.stored(v[0], "q8_0"), at, 0.125)
        assert (np.abs(read().reshape(want.shape) - want) <= ref.attention_bound(weight, size, at + 1, dim)).all()
    graph.destroy()
    stream.destroy()
    for b in (step_k, step_v, step_q, past):
        b.free()
    c.free()


# ---- probabilities -----------------------------------------------------------------


def _probabilities(ctx, dev, rows, temperature, stride=0, offset=0, output_offset=0, in_place=False):
    from charlotte_amd import harness as hx
    from charlotte_amd import serving as sv

    n, vocabulary = rows.shape
    wide = np.full((n, stride or vocabulary), 3.0, np.float32)
    wide[:, :vocabulary] = rows
    at = dev.put(wide, offset)
    held = dev.owned[-1]
    need = sv.probabilities_workspace_bytes(n, vocabulary)
    work, _ = dev.room(need, np.uint8)
    if in_place:
        to, read = at, lambda: held.read(np.float32, wide.size, offset)
    else:
        to, read = dev.room(n * vocabulary, offset=output_offset)
    call = sv.Probabilities(at, to, n, vocabulary, temperature, logit_stride=stride,
                            output_stride=stride if in_place else 0, workspace=work, workspace_bytes=need)
    sv.probabilities(ctx, call)
    hx.sync()
    got = read().reshape(n, -1)
    if in_place and stride:
        assert (got[:, vocabulary:] == 3.0).all()
    return got[:, :vocabulary]


@pytest.mark.parametrize("rows,vocabulary,temperature,layout", [
    (1, 1, 1.0, {}), (2, 3, 0.5, {}), (3, 2047, 1.0, {"offset": 4}), (1, 151936, 0.7, {}), (5, 32001, 1.3, {"offset": 8}),
    (7, 4099, 1.0, {"in_place": True}), (4, 5000, 0.8, {"stride": 5003, "in_place": True}),
    (3, 30001, 1.0, {"output_offset": 4}), (300, 6001, 1.0, {"stride": 6007}), (2, 262144, 1e-3, {}),
    # past what the caches hold: rows read once
    (130, 131072, 0.9, {}), (513, 32769, 1.0, {"stride": 32773, "offset": 4, "output_offset": 8}), (300, 60001, 1.0, {"offset": 12}),
    (140, 120003, 1.1, {"in_place": True}), (3000, 5700, 1.0, {"output_offset": 12})])
def test_probabilities(ctx, dev, rows, vocabulary, temperature, layout):
    rng = np.random.default_rng(vocabulary)
    x = (rng.standard_normal((rows, vocabulary)) * 3).astype(np.float32)
    x[:, rng.integers(0, vocabulary)] += 9
    if vocabulary > 10:
        x[0, 3:8] = -np.inf
        x[-1, -1] = -np.inf
    print("probabilities", rows, vocabulary, temperature, layout, flush=True)
    got = _probabilities(ctx, dev, x, temperature, **layout).astype(np.float64)
    away = (x.astype(np.float64) - x.max(1, keepdims=True).astype(np.float64)) / np.float32(temperature)
    want = np.exp(away)
    want /= want.sum(1, keepdims=True)
    # exp2's argument rounds three times, of its size; its result, the sum's chunks and the quotient at the rest
    with np.errstate(invalid="ignore"):
        bound = want * (np.where(np.isfinite(away), np.abs(away), 0) * 1.45 * 3 * U + 100 * U) + 1e-37
    assert (np.abs(got - want) <= bound).all()


@pytest.mark.parametrize("rows,vocabulary", [(6, 9001), (200, 90001)])  # two passes, and rows read once
def test_probabilities_at_temperature_zero_take_the_first_largest(ctx, dev, rows, vocabulary):
    rng = np.random.default_rng(31)
    x = rng.integers(-5, 6, (rows, vocabulary)).astype(np.float32)
    x[1] = -np.inf
    x[2, :] = np.nan
    x[2, 77] = -4.0
    x[3, 8000] = np.inf
    x[4] = 2.0
    got = _probabilities(ctx, dev, x, 0.0)
    want = np.zeros_like(x)
    for i in (0, 3, 4, *range(5, rows)):
        want[i, x[i].argmax()] = 1
    want[2, 77] = 1
    assert (got == want).all()


@pytest.mark.parametrize("rows,vocabulary", [(5, 5001), (250, 70001)])
def test_probabilities_of_rows_with_nothing_or_not_finite(ctx, dev, rows, vocabulary):
    x = np.zeros((rows, vocabulary), np.float32)
    x[0] = -np.inf
    x[1] = -np.inf
    x[1, 4000] = -3e38
    x[2, 17] = np.nan
    x[3, 4999] = np.inf
    got = _probabilities(ctx, dev, x, 1.0)
    assert (got[0] == 0).all()
    assert got[1, 4000] == 1 and got[1].sum() == 1
    assert np.isnan(got[2]).all() and np.isnan(got[3]).all()
    assert np.abs(got[4:] * np.float64(vocabulary) - 1).max() < 100 * U


# ---- verify ----------------------------------------------------------------------


def _verify(ctx, dev, node_tokens, target, uniforms, draft=None, accepts=None, parents=None, lengths=None, stride=0,
            offset=0, draft_offset=0):
    from charlotte_amd import harness as hx
    from charlotte_amd import serving as sv

    sequences, tokens, vocabulary = target.shape

    def rows(x, at):
        wide = np.zeros((*x.shape[:2], stride or vocabulary), np.float32)
        wide[..., :vocabulary] = x
        return dev.put(wide, at)

    need = sv.verify_workspace_bytes(sequences, tokens, vocabulary)
    work, _ = dev.room(need, np.uint8)
    outs = [dev.room(sequences * tokens, np.int32) for _ in range(2)] + [dev.room(sequences, np.uint32)]
    call = sv.Verify(dev.put(np.asarray(node_tokens, np.int32)), rows(target, offset), dev.put(np.asarray(uniforms, np.float32)),
                     vocabulary, path=outs[0][0], emitted=outs[1][0], count=outs[2][0],
                     draft=0 if draft is None else rows(draft, draft_offset),
                     accepts=0 if accepts is None else dev.put(np.asarray(accepts, np.float32)),
                     parents=0 if parents is None else dev.put(np.asarray(parents, np.int32)),
                     lengths=0 if lengths is None else dev.put(np.asarray(lengths, np.uint32)),
                     target_stride=stride, draft_stride=stride, workspace=work, workspace_bytes=need)
    sv.verify(ctx, call, sequences, tokens)
    hx.sync()
    return outs[0][1]().reshape(sequences, tokens), outs[1][1]().reshape(sequences, tokens), outs[2][1]()


def _expect(got, want, tokens):
    path, emitted, count = got
    for s, (p, e) in enumerate(want):
        assert count[s] == len(p) == len(e)
        assert path[s].tolist() == p + [-1] * (tokens - len(p))
        assert emitted[s].tolist() == e + [-1] * (tokens - len(e))


def _distributions(rng, *shape, peak=6.0):
    x = rng.standard_normal(shape) * 1.5
    x[..., : min(8, shape[-1])] += peak * rng.random((*shape[:-1], min(8, shape[-1])))
    p = np.exp(x - x.max(-1, keepdims=True))
    return (p / p.sum(-1, keepdims=True)).astype(np.float32)


@pytest.mark.parametrize("sequences,tokens,vocabulary,layout", [
    (1, 1, 11, {}), (3, 2, 1000, {"offset": 4}), (8, 6, 5003, {"offset": 8, "draft_offset": 4}), (2, 70, 64, {}),
    (5, 9, 20001, {"stride": 20004}), (40, 4, 777, {}), (2, 5, 262144, {})])
def test_verify_a_chain(ctx, dev, sequences, tokens, vocabulary, layout):
    from tests.support import serving_ref as ref

    rng = np.random.default_rng(tokens * vocabulary)
    target = _distributions(rng, sequences, tokens, vocabulary)
    draft = _distributions(rng, sequences, max(tokens - 1, 1), vocabulary) if tokens > 1 else np.zeros((sequences, 1, vocabulary), np.float32)
    if tokens > 2:  # most are near the target, so that chains end everywhere
        draft = (0.8 * target[:, :-1] + 0.2 * draft).astype(np.float32)
    node_tokens = rng.integers(0, vocabulary, (sequences, tokens))
    for s in range(sequences):
        for i in range(tokens - 1):
            node_tokens[s, i + 1] = draft[s, i].argmax() if rng.random() < 0.7 else rng.integers(0, vocabulary)
    uniforms, accepts = rng.random((2, sequences, tokens)).astype(np.float32)
    uniforms.ravel()[0] = 0.0
    if sequences > 1:
        uniforms[1] = np.float32(1) - np.float32(2.0 ** -24)
        node_tokens[1, 1] = vocabulary + 5 if sequences > 2 else -1
    lengths = rng.integers(0, tokens + 1, sequences) if sequences > 3 else np.full(sequences, tokens)
    if sequences > 3:
        lengths[2] = 0
    print("verify chain", sequences, tokens, vocabulary, layout, flush=True)
    got = _verify(ctx, dev, node_tokens, target, uniforms, draft=draft, accepts=accepts, lengths=lengths, **layout)
    want = [ref.verify(node_tokens[s], target[s], uniforms[s], draft[s], accepts[s], length=int(lengths[s]))
            for s in range(sequences)]
    _expect(got, want, tokens)


@pytest.mark.parametrize("sequences,tokens,vocabulary,layout", [
    (1, 1, 5, {}), (2, 21, 4001, {"offset": 4}), (1, 64, 500, {}), (3, 130, 90, {"stride": 95, "offset": 12}), (1, 12, 151936, {})])
def test_verify_a_tree(ctx, dev, sequences, tokens, vocabulary, layout):
    from tests.support import serving_ref as ref

    rng = np.random.default_rng(tokens + vocabulary)
    target = _distributions(rng, sequences, tokens, vocabulary, peak=12.0)
    parents = np.stack([_random_tree(rng, tokens) for _ in range(sequences)])
    if tokens > 20:
        parents[0, 9] = -2
    uniforms = rng.random((sequences, tokens)).astype(np.float32)
    # children mostly of likely tokens; twins among them, of which the first counts
    node_tokens = rng.integers(0, min(8, vocabulary), (sequences, tokens))
    lengths = np.array([tokens - 3 * s for s in range(sequences)])
    print("verify tree", sequences, tokens, vocabulary, layout, flush=True)
    got = _verify(ctx, dev, node_tokens, target, uniforms, parents=parents, lengths=lengths, **layout)
    want = [ref.verify(node_tokens[s], target[s], uniforms[s], parents=parents[s], length=int(lengths[s])) for s in range(sequences)]
    _expect(got, want, tokens)
    # no parents: a chain by the target's own draws
    got = _verify(ctx, dev, node_tokens, target, uniforms, **layout)
    _expect(got, [ref.verify(node_tokens[s], target[s], uniforms[s]) for s in range(sequences)], tokens)


def test_draws_at_their_edges(ctx, dev):
    """One entry, all of them alike, none, NaNs, more than one, less than a unit."""
    from tests.support import serving_ref as ref

    vocabulary = 3000
    rows = np.zeros((8, 1, vocabulary), np.float32)
    rows[0, 0, 2999] = 1e-9
    rows[1, 0] = 1.0 / vocabulary
    rows[3, 0, 5:9] = np.nan
    rows[3, 0, 1234] = 0.25
    rows[4, 0] = 7.0                 # each counts as one
    rows[5, 0] = 1e-14               # below 2^-44
    rows[5, 0, 17] = 6e-14
    rows[6, 0] = -1.0
    rows[6, 0, [100, 200]] = 0.5
    rows[7, 0, [100, 200]] = np.inf
    tokens = np.zeros((8, 1))
    for u in (0.0, 0.25, 0.5, 0.75, 0.99999994, 1.0, -1.0, np.nan):
        got = _verify(ctx, dev, tokens, rows, np.full((8, 1), u, np.float32))
        plain = 0.0 if np.isnan(u) else u
        assert got[1][:, 0].tolist() == [ref.drawn(rows[i, 0], plain) for i in range(8)]
        assert (got[2] == 1).all()


def test_draws_follow_the_probabilities(ctx, dev):
    """Uniform numbers on a fine grid draw each token as often as its probability says, to one step."""
    rng = np.random.default_rng(41)
    p = _distributions(rng, 200)
    n = 4000
    uniforms = ((np.arange(n) + 0.5) / n).astype(np.float32)
    got = _verify(ctx, dev, np.zeros((n, 1)), np.broadcast_to(p, (n, 1, 200)), uniforms[:, None])
    counts = np.bincount(got[1][:, 0], minlength=200)
    assert np.abs(counts - p * n).max() <= 1.01


# ---- refusals ---------------------------------------------------------------------


def _refused(call, status):
    from charlotte_amd import matmul as mm

    with pytest.raises(mm.MatmulError) as e:
        call()
    assert e.value.status == status, e.value
    assert str(e.value).split(": ", 1)[1]


def test_head_norm_rope_refuses(ctx, dev):
    from charlotte_amd import matmul as mm
    from charlotte_amd import serving as sv

    bad = mm.Status.INVALID_ARGUMENT
    x, y, t = dev.put(np.zeros((4, 256), np.float32)), dev.room(1024)[0], dev.put(np.zeros(1024, np.uint32))

    def call(tokens=1, heads=2, dim=128, part=None, **kw):
        parts = [sv.Heads(**{"input": x, "output": y, "heads": heads, **(part or {})})]
        kw = {"cosines": x, "sines": x, "positions": t, "table_rows": 4, **kw}
        return lambda: sv.head_norm_rope(ctx, sv.HeadNormRope(parts, dim, **kw), tokens)

    call()()
    for c in (call(tokens=0), call(heads=0), call(dim=0), call(dim=12), call(dim=264), call(rope_dims=12), call(rope_dims=136),
              call(part={"input": 0}), call(part={"output": 0}), call(part={"input": x + 4}), call(part={"weight": x + 8}),
              call(part={"input_stride": 252}), call(part={"input_stride": 258}), call(part={"output_stride": 8}),
              call(part={"output": x, "input_stride": 512}), call(cosines=0), call(sines=x + 4), call(positions=0), call(positions=t + 1),
              call(epsilon=-1.0), call(epsilon=float("nan")), call(rope=3)):
        _refused(c, bad)
    with pytest.raises(mm.MatmulError):
        sv.head_norm_rope(ctx, sv.HeadNormRope([], 128), 1)


def test_caches_refuse(ctx, dev):
    from charlotte_amd import matmul as mm
    from charlotte_amd import serving as sv

    bad, T = mm.Status.INVALID_ARGUMENT, mm.TensorType
    for shape in ((0, 2, 64, 8), (1, 0, 64, 8), (1, 2, 0, 8), (1, 2, 48, 8), (1, 2, 288, 8), (1, 2, 64, 0), (1, 2, 64, 1 << 31)):
        _refused(lambda: sv.Cache(ctx, T.Q8_0, *shape), bad)
    for t in (T.F32, T.Q4_1, T.Q6_K, T.BF16):
        _refused(lambda: sv.Cache(ctx, t, 1, 2, 64, 8), mm.Status.UNSUPPORTED_TYPE)
    need = sv.cache_bytes(T.Q8_0, 1, 2, 64, 8)
    memory, _ = dev.room(need + 16, np.uint8)
    _refused(lambda: sv.Cache(ctx, T.Q8_0, 1, 2, 64, 8, device=memory, nbytes=need - 1), bad)
    _refused(lambda: sv.Cache(ctx, T.Q8_0, 1, 2, 64, 8, device=memory + 8, nbytes=need), bad)
    c = sv.Cache(ctx, T.Q8_0, 1, 2, 64, 8)
    x, n = dev.put(np.zeros((16, 128), np.float32)), dev.put(np.zeros(16, np.uint32))
    for call in (lambda: c.append(0, x, n, 1), lambda: c.append(x, 0, n, 1), lambda: c.append(x, x, 0, 1),
                 lambda: c.append(x, x, n, 0), lambda: c.append(x, x, n, 9), lambda: c.append(x + 4, x, n, 1),
                 lambda: c.append(x, x, n + 2, 1), lambda: c.append(x, x, n, 1, key_stride=124),
                 lambda: c.append(x, x, n, 1, value_stride=130), lambda: c.read(x, x + 8, n, 1), lambda: c.read(x, x, n, 9),
                 lambda: c.keep(n, n, n, 0), lambda: c.keep(n, 0, n, 1), lambda: c.keep(0, n, n, 1), lambda: c.keep(n, n, 0, 1)):
        _refused(call, bad)
    other = mm.Context(0)
    d = sv.Cache(other, T.Q8_0, 1, 2, 64, 8)
    d.ctx = ctx
    _refused(lambda: d.append(x, x, n, 1), bad)
    other.close()
    d.free()  # outlives its context
    c.free()


def test_attention_refuses(ctx, dev):
    from charlotte_amd import matmul as mm
    from charlotte_amd import serving as sv

    bad = mm.Status.INVALID_ARGUMENT
    c = sv.Cache(ctx, mm.TensorType.Q8_0, 1, 2, 64, 4096)
    q, o, n = dev.put(np.zeros((300, 256), np.float32)), dev.room(300 * 256)[0], dev.put(np.zeros(300, np.uint32))
    need = sv.attention_workspace_bytes(ctx, c, 4, 1)
    assert need > 0
    work, _ = dev.room(need, np.uint8)

    def call(tokens=1, **kw):
        kw = {"cache": c, "queries": q, "output": o, "query_heads": 4, "scale": 0.1, "past": n, "workspace": work,
              "workspace_bytes": need, **kw}
        return lambda: sv.attention(ctx, sv.Attention(**kw), tokens)

    call()()
    for b in (call(tokens=0), call(tokens=4097), call(query_heads=0), call(query_heads=3), call(scale=float("inf")), call(queries=0),
              call(queries=q + 4), call(output=0), call(output=o + 8), call(past=0), call(parents=n + 1), call(query_stride=252),
              call(output_stride=257), call(workspace=0), call(workspace_bytes=need // 8), call(workspace=work + 4)):
        _refused(b, bad)
    _refused(call(tokens=257, parents=n), mm.Status.UNSUPPORTED)
    assert sv.attention_workspace_bytes(ctx, c, 3, 1) == 0
    c.free()


def test_probabilities_and_verify_refuse(ctx, dev):
    from charlotte_amd import matmul as mm
    from charlotte_amd import serving as sv

    bad = mm.Status.INVALID_ARGUMENT
    x, w = dev.put(np.zeros((6, 100), np.float32)), dev.room(4096, np.uint8)[0]

    def soft(**kw):
        kw = {"logits": x, "output": x, "rows": 2, "vocabulary": 100, "temperature": 1.0, "workspace": w, "workspace_bytes": 4096, **kw}
        return lambda: sv.probabilities(ctx, sv.Probabilities(**kw))

    soft()()
    for b in (soft(logits=0), soft(output=x + 2), soft(rows=0), soft(vocabulary=0), soft(temperature=-1.0), soft(temperature=1e-9),
              soft(temperature=float("nan")), soft(logit_stride=99), soft(logit_stride=101), soft(workspace=0),
              soft(workspace_bytes=8)):
        _refused(b, bad)

    def check(sequences=1, tokens=2, **kw):
        kw = {"node_tokens": x, "target": x, "uniforms": x, "vocabulary": 100, "path": w, "emitted": w + 64, "count": w + 128,
              "draft": x, "accepts": x, "workspace": w + 512, "workspace_bytes": 2048, **kw}
        return lambda: sv.verify(ctx, sv.Verify(**kw), sequences, tokens)

    check()()
    for b in (check(sequences=0), check(tokens=0), check(vocabulary=0), check(vocabulary=(1 << 18) + 1), check(node_tokens=0),
              check(target=0), check(uniforms=0), check(path=0), check(emitted=0), check(count=0), check(accepts=0),
              check(draft=x + 2), check(lengths=x + 1), check(target_stride=64), check(workspace=0), check(workspace_bytes=4),
              check(sequences=1 << 14, tokens=1 << 12)):
        _refused(b, bad)
    _refused(check(parents=x), mm.Status.UNSUPPORTED)


@pytest.mark.parametrize("format_", ["q8_0", "q4_0", "f16"])
@pytest.mark.parametrize("tokens", [5, 32, 71])
def test_blocks_whose_largest_magnitude_has_both_signs(ctx, dev, format_, tokens):
    """Q4_0's scale takes the sign of the first value of the largest magnitude, by a few tokens and by whole units;
    zeros of both signs, and blocks that are not held beside them."""
    from charlotte_amd import harness as hx
    from tests.support import serving_ref as ref

    rng = np.random.default_rng(tokens)
    k, v = (rng.integers(-3, 4, (2, tokens, 2, 96)).astype(np.float32) for _ in range(2))
    for x in (k, v):
        x *= np.float32(0.37)
        x[0, 0, 0, :32] = np.where(np.arange(32) % 2, np.float32(0.0), np.float32(-0.0))
        x[0, 1, 1, 32:64] = 5.0
        x[0, 1, 1, 40] = x[1, 2, 0, 95] = -5.0
        x[1, 2, 0, 64:95] = 5.0
        x[1, 3, 0, 0], x[1, 3, 0, 1], x[1, 3, 0, 33], x[1, 3, 1, 70] = np.nan, -np.nan, -np.inf, 1e30
    c = dev.cache(format_, k, v, tokens + 9, past=7)
    (ko, kr), (vo, vr) = dev.room(k.size), dev.room(v.size)
    c.read(ko, vo, dev.put(np.full(2, 7, np.uint32)), tokens)
    hx.sync()
    assert np.array_equal(kr().reshape(k.shape), ref.stored(k, format_), equal_nan=True)
    assert np.array_equal(vr().reshape(v.shape), ref.stored(v, format_), equal_nan=True)
    c.free()


@pytest.mark.parametrize("rows,vocabulary,temperature,layout", [
    # a workgroup a row up to a chunk of 16,384 (at any alignment), from 48 rows up to two; else two passes
    (3, 16381, 1.0, {"offset": 4}), (2, 16382, 1.0, {}), (5, 16384, 0.5, {"in_place": True}), (47, 20001, 1.0, {"offset": 8}),
    (48, 16382, 1.0, {"offset": 12}), (50, 32765, 0.9, {"in_place": True}), (64, 32765, 1.0, {"stride": 32771, "offset": 4}),
    (70, 20001, 1.0, {"output_offset": 4}), (60, 32766, 1.0, {}), (6, 70001, 0.7, {"stride": 70003, "in_place": True})])
def test_probabilities_by_one_workgroup_and_by_several(ctx, dev, rows, vocabulary, temperature, layout):
    test_probabilities(ctx, dev, rows, vocabulary, temperature, layout)


@pytest.mark.parametrize("rows,vocabulary", [(6, 40001), (60, 20001), (6, 12001)])
def test_probabilities_at_temperature_zero_by_each_form(ctx, dev, rows, vocabulary):
    test_probabilities_at_temperature_zero_take_the_first_largest(ctx, dev, rows, vocabulary)


@pytest.mark.parametrize("rows,vocabulary", [(6, 40001), (60, 20001), (6, 12001)])
def test_probabilities_of_rows_not_finite_by_each_form(ctx, dev, rows, vocabulary):
    test_probabilities_of_rows_with_nothing_or_not_finite(ctx, dev, rows, vocabulary)


@pytest.mark.parametrize("sequences,tokens,vocabulary", [(2, 7, 5003), (2, 7, 40001), (3, 26, 140001)])
def test_a_captured_verification_replays_on_new_logits(ctx, dev, sequences, tokens, vocabulary):
    """Probabilities (a workgroup a row, two passes, rows read once), a tree's verification and the slots kept, in one
    graph, each replay against the same calls made eagerly."""
    from charlotte_amd import harness as hx
    from charlotte_amd import serving as sv

    rng = np.random.default_rng(vocabulary)
    rows, past, dim = sequences * tokens, 40, 64
    parents = np.stack([_random_tree(rng, tokens) for _ in range(sequences)])
    k = rng.standard_normal((sequences, past + tokens, 1, dim)).astype(np.float32)
    logits, uniforms, nodes = hx.Buffer(4 * rows * vocabulary), hx.Buffer(4 * rows), hx.Buffer(4 * rows)
    need = max(sv.probabilities_workspace_bytes(rows, vocabulary), sv.verify_workspace_bytes(sequences, tokens, vocabulary))
    work, _ = dev.room(need, np.uint8)
    at, tree = dev.put(np.full(sequences, past, np.uint32)), dev.put(parents)

    class Side:
        def __init__(self):
            self.out, self.read = dev.room(rows * vocabulary)
            self.cache = dev.cache("q8_0", k, k, past + tokens)
            self.results = [dev.room(rows, np.int32), dev.room(rows, np.int32), dev.room(sequences, np.uint32)]
            self.soft = sv.Probabilities(logits.ptr, self.out, rows, vocabulary, 0.9, workspace=work, workspace_bytes=need)
            self.check = sv.Verify(nodes.ptr, self.out, uniforms.ptr, vocabulary, *(r[0] for r in self.results), parents=tree,
                                   workspace=work, workspace_bytes=need)
            self.slots = dev.room(k.size), dev.room(k.size)

        def run(self, stream):
            sv.probabilities(ctx, self.soft, stream=stream)
            sv.verify(ctx, self.check, sequences, tokens, stream=stream)
            self.cache.keep(at, self.results[0][0], self.results[2][0], tokens, stream=stream)

        def all(self):
            (ko, kr), (vo, vr) = self.slots
            self.cache.read(ko, vo, dev.put(np.zeros(sequences, np.uint32)), past + tokens)
            hx.sync()
            return [self.read(), *(r[1]() for r in self.results), kr(), vr()]

    eager, captured = Side(), Side()
    stream = hx.Stream()
    graph = hx.Graph(stream, lambda: captured.run(stream.handle), global_mode=True)
    for replay in range(4):
        x = rng.standard_normal((rows, vocabulary)).astype(np.float32)
        x[:, :3] += 8 + replay
        logits.write(x)
        uniforms.write(rng.random(rows, np.float32))
        nodes.write(rng.integers(0, 3, rows).astype(np.int32))
        graph.launch()
        stream.sync()
        eager.run(None)
        hx.sync()
        for a, b in zip(captured.all(), eager.all()):
            assert np.array_equal(a, b)
    graph.destroy()
    stream.destroy()
    for b in (logits, uniforms, nodes):
        b.free()
    for side in (eager, captured):
        side.cache.free()


@pytest.mark.parametrize("format_", ["q8_0", "q4_0", "f16"])
@pytest.mark.parametrize("tokens", [16, 40])
def test_blocks_behind_the_capacity_reach_nothing(ctx, dev, format_, tokens):
    """Steps written and read by whole units whose first slot lies past the capacity, at any place
    of a tile: no slot of the cache, of any sequence or head, and no row read back changes."""
    from charlotte_amd import harness as hx
    from tests.support import serving_ref as ref

    rng = np.random.default_rng(7)
    k, v = (rng.standard_normal((2, 70, 2, 64)).astype(np.float32) for _ in range(2))
    c = dev.cache(format_, k, v, 70)
    step = dev.put(rng.standard_normal((2 * tokens, 2 * 64)).astype(np.float32))
    rows = np.full((2 * tokens, 2 * 64), 5.0, np.float32)
    for past in ([70, 71], [95, 96], [101, 1000], [0x7FFFFFF1, 0xFFFFFFFF]):
        slots = dev.put(np.array(past, np.uint32))
        c.append(step, step, slots, tokens)
        (ko, kr), (vo, vr) = dev.room(rows.size), dev.room(rows.size)
        c.read(ko, vo, dev.put(np.zeros(2, np.uint32)), tokens)
        hx.sync()
        before = kr().copy(), vr().copy()
        c.read(ko, vo, slots, tokens)
        hx.sync()
        assert np.array_equal(kr(), before[0]) and np.array_equal(vr(), before[1])
    (ko, kr), (vo, vr) = dev.room(k.size), dev.room(v.size)
    c.read(ko, vo, dev.put(np.zeros(2, np.uint32)), 70)
    hx.sync()
    assert np.array_equal(kr().reshape(k.shape), ref.stored(k, format_))
    assert np.array_equal(vr().reshape(v.shape), ref.stored(v, format_))
    c.free()
