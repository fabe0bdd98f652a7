"""Attention over values whose blocks or tokens are of unlike sizes: a block far
below its head's largest, a token far above the others that a row does not see
or gives next to nothing, in each form (test_gpu_attention_forms.py's FORMS and
single tokens). What a row gets is right beside what it sees itself."""
import numpy as np
import pytest

from tests.test_gpu_attention_forms import FORMS, _random

pytestmark = pytest.mark.gpu

FORMS = [(1, None), (5, None), *FORMS]
PAST = 150


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


def _sizes(format_, octaves):
    """The ordinary values' size and the others', 2^octaves times that, both in reach of the format's scales."""
    low = {"q8_0": 2.0 ** -4, "q4_0": 2.0 ** -8, "f16": 2.0 ** -14}[format_]
    return np.float32(low), np.float32(low * 2.0 ** octaves)


def _check(dev, format_, q, k, v, capacity, parents=None, window=0, octaves=0):
    """Against 64 bits, of what each row sees: a probability's two binary16 parts leave 2^-20 of it
    (attention_bound), or 2^-36 of the row's largest, which is 1 at the most, times a value: of values
    in binary16 the largest that the row sees, of others one of a tile or a split whose scales lie
    within 2^16, which leaves 2^-20 of its smallest block's."""
    from tests.support import serving_ref as ref

    tokens, dim = q.shape[1], q.shape[-1]
    past = k.shape[1] - tokens
    print("spread", format_, tokens, capacity, window, octaves, parents is not None, flush=True)
    c = dev.cache(format_, k, v, capacity or past + tokens)
    got = dev.attend(c, q, [past], 1.0, parents=None if parents is None else parents[None], window=window)[0]
    c.free()
    sk, sv = ref.stored(k[0], format_), ref.stored(v[0], format_)
    want, weight, size = ref.attention(q[0], sk, sv, past, 1.0, parents, window)
    bound = ref.attention_bound(weight, size, past + tokens, dim)
    if format_ == "f16":
        seen = ref.sees(past, tokens, parents, window)
        largest = [np.abs(sv[line]).max() if line.any() else 0.0 for line in seen]
        bound = bound + 2.0 ** -36 * np.array(largest)[:, None, None]
    assert (np.abs(got - want) <= bound).all()


def _inputs(rng, tokens, dim=64, heads=1):
    n = PAST + tokens
    return (_random(rng, 1, tokens, 3 * heads, dim) * np.float32(0.2), _random(rng, 1, n, heads, dim),
            _random(rng, 1, n, heads, dim))


@pytest.mark.parametrize("format_", ["q8_0", "q4_0", "f16"])
@pytest.mark.parametrize("tokens,capacity", FORMS)
@pytest.mark.parametrize("octaves", [9, 14, 18, 24])
def test_a_block_far_below_its_heads_largest(ctx, dev, format_, tokens, capacity, octaves):
    rng = np.random.default_rng(tokens + octaves)
    q, k, v = _inputs(rng, tokens, 128)
    low, high = _sizes(format_, octaves)
    v[..., :32] *= high
    v[..., 32:] *= low
    v[..., 64:96] = 0.0
    _check(dev, format_, q, k, v, capacity, octaves=octaves)


@pytest.mark.parametrize("format_", ["q8_0", "q4_0", "f16"])
@pytest.mark.parametrize("tokens,capacity", FORMS[1:])
@pytest.mark.parametrize("octaves", [10, 18, 24])
def test_a_larger_token_that_a_row_does_not_see(ctx, dev, format_, tokens, capacity, octaves):
    """The chain's last token, a tree's sibling and a slot before the window."""
    rng = np.random.default_rng(tokens + octaves)
    q, k, v = _inputs(rng, tokens)
    low, high = _sizes(format_, octaves)
    for at, parents, window in (
            (PAST + tokens - 1, None, 0),
            (PAST + 2, np.array([-1, 0, 0, *range(1, tokens - 2)], np.int32), 0),
            (PAST - 40, None, 40)):
        x = v * low
        x[0, at] = v[0, at] * high
        _check(dev, format_, q, k, x, capacity, parents, window, octaves)


@pytest.mark.parametrize("format_", ["q8_0", "q4_0", "f16"])
@pytest.mark.parametrize("tokens,capacity", FORMS)
@pytest.mark.parametrize("octaves", [10, 15, 20, 24])
@pytest.mark.parametrize("below", [12.0, 24.0, 60.0])
def test_a_larger_token_of_next_to_no_probability(ctx, dev, format_, tokens, capacity, octaves, below):
    """e^-below of the others', in the first tile, within one and alone in the last of the past's."""
    rng = np.random.default_rng(tokens + octaves)
    q, k, v = _inputs(rng, tokens)
    low, high = _sizes(format_, octaves)
    q[..., 0], k[..., 0] = 4.0, 0.0
    for at in (0, 77, PAST - 1):
        kk, x = k.copy(), v * low
        kk[0, at, 0, 0] = -below / 4
        x[0, at] = v[0, at] * high
        _check(dev, format_, q, kk, x, capacity, octaves=octaves)


@pytest.mark.parametrize("format_", ["q8_0", "q4_0", "f16"])
@pytest.mark.parametrize("tokens,capacity", FORMS)
@pytest.mark.parametrize("octaves", [12, 24])
def test_values_that_shrink_and_grow_again(ctx, dev, format_, tokens, capacity, octaves):
    """Tiles far larger than those before and after, seen with next to no probability, NaNs among the unseen."""
    rng = np.random.default_rng(tokens + octaves)
    q, k, v = _inputs(rng, tokens)
    low, high = _sizes(format_, octaves)
    q[..., 0], k[..., 0] = 4.0, 0.0
    large = np.arange(PAST + tokens) // 32 % 2 == 0
    k[0, large, 0, 0] = -0.25 * octaves
    x = np.where(large[None, :, None, None], v * high, v * low)
    k[0, :4], x[0, :4] = np.nan, np.nan
    k[0, 40:44], x[0, 40:44] = 0.0, 0.0
    _check(dev, format_, q, k, x, capacity, window=PAST - 8, octaves=octaves)


@pytest.mark.parametrize("format_", ["q8_0", "q4_0", "f16"])
@pytest.mark.parametrize("tokens,capacity", FORMS)
@pytest.mark.parametrize("octaves", [12, 16])
def test_queries_far_below_their_rows_largest(ctx, dev, format_, tokens, capacity, octaves):
    """A query's largest value where every key is zero: the scores come of the rest, whose parts leave 2^-21 of them
    down to 2^-17 of the row's largest."""
    rng = np.random.default_rng(tokens + octaves)
    q, k, v = _inputs(rng, tokens)
    q[..., 5] = 2.0 ** octaves
    k[..., 5] = 0.0
    _check(dev, format_, q, k, v, capacity, octaves=octaves)


@pytest.mark.parametrize("format_", ["q8_0", "q4_0", "f16"])
def test_subnormal_queries_keep_their_bits(ctx, dev, format_):
    rng = np.random.default_rng(16)
    k, q = _random(rng, 1, 90, 1, 64), (rng.standard_normal((1, 1, 2, 64)) * 1e-38).astype(np.float32)
    scale = float(np.float32(0.125 / 1e-38))  # times log2(e) 1.8e37: inside f32
    from tests.support import serving_ref as ref

    c = dev.cache(format_, k, k, 90)
    got = dev.attend(c, q, [89], scale)[0]
    c.free()
    stored = ref.stored(k[0], format_)
    want, weight, size = ref.attention(q[0], stored, stored, 89, scale)
    assert (np.abs(got - want) <= ref.attention_bound(weight, size, 90, 64)).all()
