"""Paged attention's form of many rows (charlotte_amd.serving), in steps that are load
enough for it: each test looks up, in what the form leaves in the workspace, that it is
the one that ran. Against a restatement in 64 bits."""

import numpy as np
import pytest

from tests.test_gpu_requests import NOWHERE, _Pool, _words

pytestmark = pytest.mark.gpu

# every format and width that has the form
FORMS = [("q8_0", d) for d in (32, 64, 96, 128)] + [("q4_0", d) for d in (32, 64, 96, 128)] + \
    [("f16", d) for d in (32, 64, 96, 128, 160, 192, 224, 256)]


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


def _attention(q, k, v, past, scale, window):
    """tests/support/serving_ref.py's attention of a chain, all rows of a key head at once."""
    tokens, heads, dim = q.shape
    n, kv_heads, _ = k.shape
    group = heads // kv_heads
    place = past + np.arange(tokens)[:, None]
    seen = np.arange(n) <= place
    if window:
        seen &= np.arange(n) > place - window
    seen = np.repeat(seen, group, 0)
    out, weight, size = (np.zeros((tokens, heads, dim)) for _ in range(3))
    for h in range(kv_heads):
        at = slice(h * group, (h + 1) * group)
        rows, kh, vh = q[:, at].reshape(-1, dim).astype(np.float64), k[:, h].astype(np.float64), v[:, h].astype(np.float64)
        bad = np.isnan(vh)
        vh = np.where(bad, 0, vh)
        p = np.where(seen, rows @ kh.T * scale, -np.inf)
        p = np.exp(p - p.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
        o = p @ vh
        if bad.any():
            o[seen.astype(np.float32) @ bad.astype(np.float32) > 0] = np.nan
        top = np.where(seen, np.abs(rows) @ np.abs(kh).T, 0).max(1, keepdims=True) * abs(scale)
        for to, x in ((out, o), (weight, p @ np.abs(vh)), (size, np.broadcast_to(top, o.shape))):
            to[:, at] = x.reshape(tokens, group, dim)
    return out, weight, size


class _Step:
    """requests: (past, count) each; `gone`: (request, page of its row) that the pool does not have; `short`: pages a row of
    the table has, where that is fewer than a request needs; `held`: the most past and count, where a step is run again."""

    def __init__(self, ctx, dev, format_, requests, heads, kv_heads, dim, page_tokens=64, window=0, seed=0, spread=1.0, grow=0,
                 gone=(), short=0, stride=0, query_stride=0, output_stride=0, spoil=(), most=None, longest=0, rows=0):
        from charlotte_amd import serving as sv
        from tests.support import serving_ref as ref

        rng = np.random.default_rng(seed)
        self.ctx, self.requests, self.page_tokens, self.window = ctx, requests, page_tokens, window
        self.heads, self.dim, self.scale = heads, dim, dim ** -0.5
        counts = [c for _, c in requests]
        self.starts = [sum(counts[:i]) for i in range(len(counts) + 1)]
        self.rows = rows or self.starts[-1]
        need = [-(-(p + c) // page_tokens) for p, c in requests]
        pages = sum(need) + 2
        order = rng.permutation(pages).tolist()
        self.stride = stride or short or max(need)
        self.table = np.full((len(requests), self.stride), NOWHERE, np.uint64)
        self.pool = _Pool(dev, format_, pages, page_tokens, kv_heads, dim)
        self.keys, self.values, keys, values, slots = [], [], [], [], []
        for r, (past, count) in enumerate(requests):
            n = past + count
            held = [order.pop() for _ in range(need[r])]
            self.table[r, :min(need[r], self.stride)] = held[:self.stride]
            k = rng.standard_normal((n, kv_heads, dim)).astype(np.float32)
            v = (rng.standard_normal((n, kv_heads, dim)) * spread).astype(np.float32)
            if grow:
                v *= (2.0 ** -rng.integers(0, grow, (n, 1, 1))).astype(np.float32) * np.float32(2.0 ** (grow // 2))
            for of, token, head, at, x in spoil:
                if of[0] == r:
                    (k if of[1] == "k" else v)[token, head, at] = x
            keys.append(k)
            values.append(v)
            slots.append(np.array(held)[np.arange(n) // page_tokens] * page_tokens + np.arange(n) % page_tokens)
            self.keys.append(ref.stored(k, format_))
            self.values.append(ref.stored(v, format_))
        self.pool.write(np.concatenate(keys).reshape(-1, kv_heads * dim), np.concatenate(values).reshape(-1, kv_heads * dim),
                        np.concatenate(slots))
        for r, page in gone:
            self.table[r, page] = (pages, NOWHERE, pages + 5)[page % 3]
            self.keys[r] = self.keys[r].copy()
            self.keys[r][page * page_tokens:(page + 1) * page_tokens] = np.nan
        width = heads * dim
        self.q = rng.standard_normal((self.rows, heads, dim)).astype(np.float32)
        given = np.zeros((self.rows, query_stride or width), np.float32)
        given[:, :width] = self.q.reshape(self.rows, -1)
        most = max(counts) if most is None else most
        self.need = sv.paged_attention_workspace_bytes(ctx, self.pool.pool, heads, most)
        self.work, self.read_work = dev.room(self.need, np.uint8)
        self.out_width = output_stride or width
        out, self.read_out = dev.room(self.rows * self.out_width)
        self.at = {n: dev.put(_words(x)) for n, x in (("past", [p for p, _ in requests]), ("counts", counts), ("starts", self.starts))}
        self.buffers = dict(zip(self.at, dev.owned[-3:]))
        self.call = sv.PagedAttention(self.pool.pool, dev.put(given), out, heads, self.scale, len(requests), self.rows,
                                      self.at["past"], self.at["counts"], self.at["starts"], dev.put(_words(self.table)), self.stride,
                                      window, most, query_stride, output_stride, self.work, self.need, longest)
        # a part's join, behind the pieces of two units of its workgroup's rows and their offsets and sums
        per_row = 4 * dim + 8
        parts = sv.paged_attention_workspace_bytes(ctx, self.pool.pool, kv_heads, 1) // (2 * 16 * per_row)
        self.joins = slice(2 * parts * (256 if dim <= 128 else 128) * per_row // 4, None)
        self.parts = parts

    def run(self, stream=None):
        from charlotte_amd import serving as sv

        sv.paged_attention(self.ctx, self.call, stream=stream)

    def form(self):
        """Of how many parts a unit goes on past it: None where the form of many rows was not launched."""
        words = self.read_work().view(np.uint32)[self.joins].reshape(-1, 6)
        if len(words) == 0 or (words[:, 4] == NOWHERE).all():
            return None
        assert len(words) == self.parts and (words[:, 4] <= self.parts).all()
        return int((words[:, 4] > 1).sum())

    def got(self):
        return self.read_out().reshape(self.rows, self.out_width)

    def check(self, got, requests=None):
        """Every row against the restatement; what is behind a row, and rows of no request, as they were."""
        from tests.support import serving_ref as ref

        width = self.heads * self.dim
        assert (got[:, width:].view(np.uint32) == NOWHERE).all()
        got = got[:, :width].reshape(self.rows, self.heads, self.dim)
        touched = np.zeros(self.rows, bool)
        start = 0
        for r, (past, count) in enumerate(requests or self.requests):
            at = slice(start, start + count)
            start += count
            touched[at] = True
            n = past + count
            if count == 0:
                continue
            if n > self.stride * self.page_tokens:
                assert np.isnan(got[at]).all(), r
                continue
            want, weight, size = _attention(self.q[at], self.keys[r][:n], self.values[r][:n], past, self.scale, self.window)
            none = np.isnan(want)
            assert np.array_equal(np.isnan(got[at]), none), r
            bound = ref.attention_bound(weight, size, n + 32 * 256, self.dim)
            assert (np.abs(got[at] - want) <= bound)[~none].all(), r
        assert (got[~touched].view(np.uint32) == NOWHERE).all()


def _check(ctx, dev, *args, form=True, **kw):
    """A step run twice, at the same bits, and against the restatement; whether its units of many rows ran, in pieces."""
    from charlotte_amd import harness as hx

    print("many rows", args, kw, flush=True)
    step = _Step(ctx, dev, *args, **kw)
    step.run()
    hx.sync()
    assert step.form() if form else not step.form(), step.form()
    got = step.got()
    step.check(got)
    step.run()
    hx.sync()
    assert np.array_equal(step.got().view(np.uint32), got.view(np.uint32))
    step.pool.pool.free()


def _long(dim):
    """Tokens of a prompt of 900 rows on four key heads that are load enough."""
    return 8400 if dim <= 64 else 3300 if dim <= 128 else 1000


@pytest.mark.parametrize("format_,dim", FORMS)
def test_every_format_and_width(ctx, dev, format_, dim):
    """Rows of three heads a token, of which units of 256 and 128 begin and end inside tokens; short ones, a single token and
    one without tokens beside them."""
    _check(ctx, dev, format_, [(_long(dim), 300), (40, 1), (700, 131), (5, 0), (0, 86), (333, 9)], 12, 4, dim, seed=dim)


@pytest.mark.parametrize("format_,dim,heads,kv_heads,count", [
    ("q8_0", 128, 16, 8, 1200), ("q4_0", 64, 16, 8, 1500), ("f16", 256, 8, 4, 700), ("f16", 32, 16, 8, 1500)])
@pytest.mark.parametrize("window", [1, 31, 32, 500, 5000])
def test_in_a_window(ctx, dev, format_, dim, heads, kv_heads, count, window):
    """A unit's tiles begin where its own first row's window does."""
    _check(ctx, dev, format_, [(901, count), (2000, 1), (90, 129)], heads, kv_heads, dim, window=window, seed=window)


@pytest.mark.parametrize("format_,dim,window", [("q8_0", 128, 0), ("q4_0", 96, 0), ("f16", 160, 0), ("q8_0", 128, 1300),
                                                ("q4_0", 96, 1300), ("f16", 160, 200)])
def test_pages_that_the_pool_does_not_have(ctx, dev, format_, dim, window):
    """NaNs for the rows that see one: the later ones, or with a window the earlier ones; a request that passes the table's
    row, of many rows and of few, NaNs alone."""
    long = _long(dim) - (500 if window else 0)
    gone = [(0, (long - window + 50) // 64)] if window else [(0, long // 64 + 1), (0, long // 64 + 3)]
    requests = [(long, 300), (long, 300), (long + 400, 300), (130, 200), (77, 1), (long + 600, 2), (long + 100, 90)]
    _check(ctx, dev, format_, requests, 12, 4, dim, window=window, seed=5, gone=gone + [(3, 2), (4, 0)], short=-(-(long + 320) // 64))


@pytest.mark.parametrize("format_,dim,grow,spread", [
    ("q8_0", 64, 40, 1.0), ("q8_0", 128, 24, 1.0), ("q4_0", 64, 28, 1.0), ("q4_0", 128, 40, 1.0), ("q4_0", 32, 18, 1.0),
    ("q8_0", 96, 0, 1e-4), ("q8_0", 96, 0, 3e4), ("f16", 128, 0, 1.3e4), ("f16", 256, 40, 1.0)])
def test_values_of_any_size(ctx, dev, format_, dim, grow, spread):
    """Scales too far apart to be laid out, and values past what the format holds: NaNs in blocks."""
    _check(ctx, dev, format_, [(_long(dim), 300), (64, 1), (500, 90)], 12, 4, dim, seed=3, grow=grow, spread=spread)


@pytest.mark.parametrize("format_,dim", [("q8_0", 32), ("q8_0", 128), ("q4_0", 64), ("f16", 64), ("f16", 224)])
def test_tokens_that_are_not_numbers(ctx, dev, format_, dim):
    """Keys and values that no block holds: seen by all rows, by the last ones, and by none."""
    past = _long(dim)
    spoil = [((0, "k"), past + 200, 1, 3, np.nan), ((0, "v"), 70, 2, dim - 1, np.inf), ((0, "v"), past + 299, 3, 0, np.nan),
             ((0, "k"), past + 298, 0, 0, -np.inf)]
    _check(ctx, dev, format_, [(past, 300), (64, 1)], 12, 4, dim, seed=6, spoil=spoil)


@pytest.mark.parametrize("format_,dim,heads,kv_heads,past,count,page_tokens", [
    ("q8_0", 64, 64, 1, 8000, 65, 32), ("q4_0", 128, 8, 8, 9000, 150, 2048), ("f16", 192, 5, 1, 4901, 128, 96),
    ("f16", 96, 1, 1, 700, 4100, 32), ("q8_0", 32, 257, 1, 30000, 16, 64)])
def test_groups_and_pages_of_any_size(ctx, dev, format_, dim, heads, kv_heads, past, count, page_tokens):
    _check(ctx, dev, format_, [(past, count), (31, 1)], heads, kv_heads, dim, page_tokens=page_tokens, seed=heads)


def test_strides_and_rows_of_no_request(ctx, dev):
    _check(ctx, dev, "q8_0", [(3300, 300), (40, 1), (0, 100)], 12, 4, 128, query_stride=12 * 128 + 64, output_stride=12 * 128 + 20,
           stride=77, rows=409, seed=2)
    _check(ctx, dev, "f16", [(1000, 300), (40, 1)], 12, 4, 224, query_stride=12 * 224 + 4, output_stride=13 * 224, stride=40,
           rows=333, seed=2)


def test_the_step_that_is_not_load_enough(ctx, dev):
    """Tables and rows that may be load enough, requests that are not: the form is launched and leaves them to the other."""
    from charlotte_amd import harness as hx

    step = _Step(ctx, dev, "q8_0", [(300, 200), (90, 1), (0, 150)], 12, 4, 64, stride=400, rows=360, seed=9)
    step.run()
    hx.sync()
    assert step.form() == 0
    step.check(step.got())
    # and where the longest is named, it is not launched
    named = _Step(ctx, dev, "q8_0", [(300, 200), (90, 1), (0, 150)], 12, 4, 64, stride=400, rows=360, seed=9, longest=500)
    named.run()
    hx.sync()
    assert named.form() is None
    assert np.array_equal(named.got().view(np.uint32), step.got().view(np.uint32))
    step.pool.pool.free()
    named.pool.pool.free()


@pytest.mark.parametrize("format_,dim", [("q8_0", 128), ("f16", 256)])
def test_captured_steps_replay_as_requests_grow(ctx, dev, format_, dim):
    """One graph whose requests' lengths change between its replays, so that the form takes them in some and not in others;
    each replay against the eager call."""
    from charlotte_amd import harness as hx

    long = _long(dim)
    most = [(long, 300), (500, 1), (700, 200)]
    eager, captured = (_Step(ctx, dev, format_, most, 12, 4, dim, seed=4) for _ in range(2))
    stream = hx.Stream()
    graph = hx.Graph(stream, lambda: captured.run(stream.handle), global_mode=True)
    seen = []
    for replay, requests in enumerate([most, [(3, 1), (0, 1), (77, 2)], [(long // 2, 300), (500, 1), (700, 200)], [(0, 5), (0, 0), (0, 300)],
                                       [(long, 300), (500, 1), (0, 0)], most, [(long, 1), (500, 1), (700, 1)], most]):
        counts = [c for _, c in requests]
        starts = [sum(counts[:i]) for i in range(4)]
        for step in (eager, captured):
            for name, x in (("past", [p for p, _ in requests]), ("counts", counts), ("starts", starts)):
                step.buffers[name].write(_words(x))
            next(b for b in dev.owned if b.ptr == step.call.output).write(np.full(step.rows * step.out_width, NOWHERE, np.uint32))
        graph.launch()
        stream.sync()
        eager.run()
        hx.sync()
        assert captured.form() == eager.form()
        seen.append(captured.form() > 0)
        got = captured.got()
        assert np.array_equal(got.view(np.uint32), eager.got().view(np.uint32)), replay
        captured.check(got, requests)
    assert seen[0] and seen[5] and seen[7] and not seen[1] and not seen[6]
    graph.destroy()
    stream.destroy()
    for step in (eager, captured):
        step.pool.pool.free()


def test_two_streams_at_once(ctx, dev):
    """Two pools, each with a workspace and a stream of its own."""
    from charlotte_amd import harness as hx

    steps = [_Step(ctx, dev, "q8_0", [(3300, 300), (40, 1), (0, 90)], 12, 4, 128, seed=1),
             _Step(ctx, dev, "f16", [(1000, 300), (40, 1), (200, 170)], 12, 4, 160, seed=2)]
    streams, want = [hx.Stream(), hx.Stream()], []
    for step in steps:
        step.run()
        hx.sync()
        assert step.form()
        want.append(step.got().view(np.uint32))
        step.check(step.got())
    for _ in range(5):
        for step, stream in zip(steps, streams):
            step.run(stream.handle)
        for stream in streams:
            stream.sync()
        for step, w in zip(steps, want):
            assert np.array_equal(step.got().view(np.uint32), w)
    for stream in streams:
        stream.destroy()
    for step in steps:
        step.pool.pool.free()


def test_units_that_are_not_in_pieces(ctx, dev):
    """A unit a workgroup, each of one length, and as many of two lengths."""
    from charlotte_amd import harness as hx

    for requests in ([(416, 64)] * 64, [(416, 64), (380, 60)] * 40):
        step = _Step(ctx, dev, "q8_0", requests, 16, 4, 128, seed=11)
        step.run()
        hx.sync()
        assert step.form() is not None
        step.check(step.got())
        step.pool.pool.free()
