"""Attention's three forms - workgroups of 16 rows, of 32, and waves of 32 rows
over shared operands - at the same questions.

Which form a step takes follows from its rows and the cache's capacity (with no
bound on the lengths given), so a roomy cache brings few rows to the forms for
many. `FORMS` names (tokens, capacity) for three query heads a key head.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

ROOMY = 150_000
FORMS = [(19, None), (41, None), (19, ROOMY), (41, ROOMY), (91, ROOMY), (200, ROOMY)]


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


def _random(rng, *shape):
    return rng.standard_normal(shape).astype(np.float32)


def _close(got, q, k, v, format_, past, scale, parents=None, window=0, rows=slice(None)):
    from tests.support import serving_ref as ref

    n, dim = past + q.shape[0], q.shape[-1]
    want, weight, size = ref.attention(q, ref.stored(k, format_), ref.stored(v, format_), past, scale, parents, window)
    error = np.abs(got - want)[rows]
    assert (error <= ref.attention_bound(weight, size, n, dim)[rows]).all()
    return want


@pytest.mark.parametrize("format_", ["q8_0", "q4_0", "f16"])
@pytest.mark.parametrize("dim", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("tokens,capacity", FORMS[2:])
def test_every_head_width(ctx, dev, format_, dim, tokens, capacity):
    rng = np.random.default_rng(dim + tokens)
    past, heads = 70, 1
    k, v = _random(rng, 1, past + tokens, heads, dim), _random(rng, 1, past + tokens, heads, dim)
    q = _random(rng, 1, tokens, 3, dim)
    print("forms", format_, dim, tokens, capacity, flush=True)
    c = dev.cache(format_, k, v, capacity)
    _close(dev.attend(c, q, [past], dim ** -0.5)[0], q[0], k[0], v[0], format_, past, dim ** -0.5)
    c.free()


@pytest.mark.parametrize("format_", ["q8_0", "f16"])
@pytest.mark.parametrize("tokens,capacity", FORMS)
@pytest.mark.parametrize("window", [0, 5, 90])
@pytest.mark.parametrize("past", [0, 45, 1500])
def test_trees_and_windows(ctx, dev, format_, tokens, capacity, window, past):
    rng = np.random.default_rng(tokens + window)
    parents = np.array([rng.integers(max(-1, t - 6), t) for t in range(tokens)], np.int32)
    parents[0] = -1
    lengths = [past, max(0, past - 3)]
    k, v = _random(rng, 2, past + tokens, 2, 64), _random(rng, 2, past + tokens, 2, 64)
    q = _random(rng, 2, tokens, 6, 64)
    print("tree", format_, tokens, capacity, window, past, flush=True)
    c = dev.cache(format_, k, v, capacity or past + tokens)
    for line in (parents, None):
        got = dev.attend(c, q, lengths, 0.125, parents=None if line is None else np.stack([line, line]), window=window)
        for s in range(2):
            _close(got[s], q[s], k[s], v[s], format_, lengths[s], 0.125, line, window)
    c.free()


@pytest.mark.parametrize("format_", ["q8_0", "q4_0", "f16"])
@pytest.mark.parametrize("tokens,capacity", FORMS)
def test_unseen_values_that_are_not_finite(ctx, dev, format_, tokens, capacity):
    """Two lines leave the root; one runs through a token of NaNs and infinities."""
    rng = np.random.default_rng(tokens)
    past = 77
    parents = np.array([-1, 0, 0, *range(1, tokens - 2)], np.int32)  # 0-1-3-5-..., 0-2-4-...
    bad = np.zeros(tokens, bool)
    bad[2::2] = True
    k, v = _random(rng, 1, past + tokens, 1, 64), _random(rng, 1, past + tokens, 1, 64)
    clean_k, clean_v = k.copy(), v.copy()
    k[0, past + 2, 0, 5], v[0, past + 2, 0, 40] = np.nan, np.inf
    q = _random(rng, 1, tokens, 3, 64)
    c = dev.cache(format_, k, v, capacity or past + tokens)
    got = dev.attend(c, q, [past], 0.125, parents=parents[None])[0]
    _close(got, q[0], clean_k[0], clean_v[0], format_, past, 0.125, parents, rows=~bad)
    assert np.isnan(got[bad]).all()
    c.free()
    # slots before a window, and those past the last token (in a cache with room)
    window = tokens + 8
    first = past + 1 - window  # the first slot that any row sees
    k, v = clean_k.copy(), clean_v.copy()
    if first > 0:
        k[0, :first], v[0, :first] = np.inf, np.nan
    if capacity:
        k = np.concatenate([k, np.full((1, 50, 1, 64), np.nan, np.float32)], 1)
        v = np.concatenate([v, np.full((1, 50, 1, 64), -np.inf, np.float32)], 1)
    c = dev.cache(format_, k, v, capacity or k.shape[1])
    got = dev.attend(c, q, [past], 0.125, window=window)[0]
    _close(got, q[0], clean_k[0], clean_v[0], format_, past, 0.125, window=window)
    c.free()


@pytest.mark.parametrize("tokens,capacity", FORMS)
def test_queries_and_tokens_that_leave_nothing(ctx, dev, tokens, capacity):
    rng = np.random.default_rng(tokens + 1)
    past = 50
    k = _random(rng, 1, past + tokens, 1, 64)
    q = _random(rng, 1, tokens, 3, 64)
    c = dev.cache("q8_0", k, k, capacity or past + tokens)
    clean = dev.attend(c, q, [past], 0.1)[0]
    spoilt = np.zeros((tokens, 3), bool)
    for t, h, x in ((0, 1, np.nan), (7, 0, np.inf), (tokens - 1, 2, -np.inf)):
        q[0, t, h, 3 * h], spoilt[t, h] = x, True
    got = dev.attend(c, q, [past], 0.1)[0]
    assert np.isnan(got[spoilt]).all() and (got[~spoilt] == clean[~spoilt]).all()
    assert (dev.attend(c, q, [past], 0.1, parents=np.full((1, tokens), -2, np.int32)) == 0).all()
    c.free()


@pytest.mark.parametrize("format_", ["q8_0", "q4_0", "f16"])
@pytest.mark.parametrize("tokens,capacity", FORMS)
def test_values_and_scores_that_grow(ctx, dev, format_, tokens, capacity):
    rng = np.random.default_rng(tokens + 2)
    n = 600 + tokens
    grow = (2.0 ** (np.arange(n) / 60) * (0.05 if format_ == "q4_0" else 1e-2)).astype(np.float32)
    k, q = _random(rng, 1, n, 1, 64) * np.float32(0.3), _random(rng, 1, tokens, 3, 64) * np.float32(2)
    v = _random(rng, 1, n, 1, 64) * grow[None, :, None, None]
    for turned in (False, True):
        kk, vv = (np.ascontiguousarray(x[:, ::-1]) if turned else x for x in (k, v))
        c = dev.cache(format_, kk, vv, capacity or n)
        _close(dev.attend(c, q, [600], 1.0)[0], q[0], kk[0], vv[0], format_, 600, 1.0)
        c.free()


@pytest.mark.parametrize("format_,dim", [("f16", 256), ("f16", 64), ("q8_0", 128), ("q4_0", 160)])
def test_one_workspace_serves_every_bound_on_the_lengths(ctx, dev, format_, dim):
    rng = np.random.default_rng(dim)
    past, capacity = 20, 5000
    for tokens in (1, 6, 90):
        k, v = _random(rng, 1, past + tokens, 1, dim), _random(rng, 1, past + tokens, 1, dim)
        q = _random(rng, 1, tokens, 4, dim)
        c = dev.cache(format_, k, v, capacity)
        for longest in (past + tokens, 256, 300, 500, 1000, 2000, 2048, 2049, 3000, 4096, 5000, 0):
            print("bound", format_, dim, tokens, longest, flush=True)
            _close(dev.attend(c, q, [past], dim ** -0.5, longest=longest)[0], q[0], k[0], v[0], format_, past, dim ** -0.5)
        c.free()


def test_a_long_prompt_in_one_step(ctx, dev):
    """33,000 tokens of 64 query heads: past 2^21 rows, their memory past 2^28 bytes."""
    rng = np.random.default_rng(33)
    tokens, heads, dim = 33_000, 64, 32
    k, v = _random(rng, 1, tokens, 1, dim), _random(rng, 1, tokens, 1, dim)
    q = rng.random((1, tokens, heads, dim), np.float32) - np.float32(0.5)
    c = dev.cache("q8_0", k, v, tokens)
    got = dev.attend(c, q, [0], 0.5)[0]
    for t in (0, 1, 31, 32, 8191, 16_384, 29_999, 32_999):
        _close(got[t:t + 1], q[0, t:t + 1], k[0, :t + 1], v[0, :t + 1], "q8_0", t, 0.5)
    c.free()
