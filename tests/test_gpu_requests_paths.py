"""Forms of a step's operators over several requests (charlotte_amd.serving) that
their sizes choose: a pool's whole tiles through strides, many rows of a workgroup
each sampled, norms of many odd rows, tables of a few thousand rows."""

import numpy as np
import pytest

from tests.test_gpu_requests import (NOWHERE, _check_plan, _check_sample, _Pool, _settings, _state, _words)

pytestmark = pytest.mark.gpu


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


@pytest.mark.parametrize("format_", ["q8_0", "q4_0", "f16"])
def test_whole_tiles_through_strides(ctx, dev, format_):
    """Rows of keys and of values each as far apart as they like; what lies between them is left."""
    from charlotte_amd import harness as hx
    from tests.support import serving_ref as ref

    rng = np.random.default_rng(4)
    heads, dim, page_tokens, rows = 4, 160, 96, 1000
    width, pages = heads * dim, 13
    order = rng.permutation(pages)
    place = np.arange(17, 17 + rows)
    slots = order[place // page_tokens] * page_tokens + place % page_tokens
    slots[500:540] = slots[500:540][::-1]  # a run that is no tile's
    given = np.where(rng.random(rows) < 0.01, NOWHERE, slots)
    held = given != NOWHERE
    strides = (width + 12, width + 64)
    k, v = (rng.standard_normal((rows, s)).astype(np.float32) for s in strides)
    pool = _Pool(dev, format_, pages, page_tokens, heads, dim, byte=0)
    pool.write(k, v, given, *strides)
    to = [dev.put(np.full((rows, s), 5, np.float32)) for s in strides]
    buffers = dev.owned[-2:]
    pool.pool.read(*to, dev.put(_words(given)), rows, *strides)
    hx.sync()
    for b, s, x in zip(buffers, strides, (k, v)):
        got = b.read(np.float32, rows * s).reshape(rows, s)
        assert (got[:, width:] == 5).all()
        want = ref.stored(x[:, :width].reshape(rows, heads, dim), format_).reshape(rows, width)
        assert np.array_equal(got[:, :width], np.where(held[:, None], want, np.float32(5)))
    pool.pool.free()


@pytest.mark.parametrize("rows,vocabulary", [(700, 9001), (513, 2049)])
def test_many_rows_sampled(ctx, dev, rows, vocabulary):
    rng = np.random.default_rng(rows)
    logits = (rng.standard_normal((rows, vocabulary)) * 3).astype(np.float32)
    _check_sample(ctx, dev, logits, _settings(rng, rows), {"stride": vocabulary + 2, "offset": 8})


@pytest.mark.parametrize("rows,width,offset", [(600, 1301, 4), (600, 2048, 0), (1100, 4096, 0), (520, 4097, 0)])
def test_norms_of_many_rows(ctx, dev, rows, width, offset):
    from charlotte_amd import harness as hx
    from charlotte_amd import serving as sv
    from tests.support import requests_ref as ref

    rng = np.random.default_rng(width)
    x, y, g = (rng.standard_normal((rows, width)).astype(np.float32) for _ in range(3))
    w, v = (rng.standard_normal(width).astype(np.float32) for _ in range(2))
    (r_at, read_r), (n_at, read_n) = (dev.room(rows * width, offset=offset) for _ in range(2))
    sv.residual_norm(ctx, sv.ResidualNorm(width, dev.put(x, offset), dev.put(y, offset), r_at, n_at, dev.put(v, offset), dev.put(w, offset),
                                          dev.put(g, offset), 0.5, 0.3, gate_stride=width), rows)
    hx.sync()
    r, n, off_r, off_n = ref.residual_norm(x, y, w, g, v, 0.5, 0.3, 1e-6)
    assert (np.abs(read_r().reshape(rows, width) - r) <= off_r).all()
    assert (np.abs(read_n().reshape(rows, width) - n) <= off_n).all()


@pytest.mark.parametrize("requests,longest,most,rows", [(40, 900, 60, 1500), (256, 100, 8, 2048), (256, 100, 8, 2049), (257, 60, 3, 900)])
def test_tables_of_about_as_many_rows_as_a_launch_takes(ctx, dev, requests, longest, most, rows):
    rng = np.random.default_rng(rows)
    past, held, table, free, pages = _state(rng, requests, 32, longest, 300)
    counts = rng.integers(0, most + 1, requests)
    assert counts.sum() <= rows
    _check_plan(ctx, dev, past, counts, held, table, free, 300, rows, 32, pages)
