"""A step over several requests (charlotte_amd.serving) on the device, against
plain restatements in 64 bits and whole numbers: the tables and slots, what the
pool holds and the tokens drawn are compared exactly."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

FORMATS = ["q8_0", "q4_0", "f16"]


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


def _words(x):
    return np.asarray(x, np.uint64).astype(np.uint32)


# ---- page_plan ----------------------------------------------------------------


class _Plan:
    """The call over device copies of past, counts, held, table, free pages and their count."""

    def __init__(self, ctx, dev, past, counts, held, table, free, free_count, rows, page_tokens, pages, in_place=False):
        from charlotte_amd import serving as sv

        self.ctx, self.dev, self.n, self.rows = ctx, dev, len(past), rows
        self.shape = np.shape(table)
        rooms = {"table": np.size(table), "free": len(free), "free_count": 1, "held": self.n, "granted": self.n,
                 "starts": self.n + 1, "slots": rows, "positions": rows}
        self.out = {k: dev.room(v, np.uint32) for k, v in rooms.items()}
        put = {k: dev.put(_words(v)) for k, v in (("past", past), ("counts", counts), ("held", held), ("count", [free_count]))}
        self._write("table", table)
        self._write("free", free)
        if in_place:
            self._write("held", held)
            self._write("free_count", [free_count])
            put["held"], put["count"] = self.out["held"][0], self.out["free_count"][0]
        p = {k: v[0] for k, v in self.out.items()}
        self.call = sv.PagePlan(self.n, rows, pages, page_tokens, put["past"], put["counts"], p["table"], self.shape[1],
                                put["held"], p["held"], p["free"], put["count"], p["free_count"], p["starts"], p["granted"],
                                p["slots"], p["positions"])

    def _write(self, name, values):
        from charlotte_amd import harness as hx

        hx.sync()
        next(b for b in self.dev.owned if b.ptr == self.out[name][0]).write(_words(values).ravel())

    def run(self, stream=None):
        from charlotte_amd import serving as sv

        sv.page_plan(self.ctx, self.call, stream=stream)

    def results(self):
        from charlotte_amd import harness as hx

        hx.sync()
        got = {k: read() for k, (_, read) in self.out.items()}
        got["table"] = got["table"].reshape(self.shape)
        return got


def _check_plan(ctx, dev, past, counts, held, table, free, free_count, rows, page_tokens, pages, **kw):
    from tests.support import requests_ref as ref

    print("page_plan", len(past), rows, page_tokens, pages, flush=True)
    plan = _Plan(ctx, dev, past, counts, held, table, free, free_count, rows, page_tokens, pages, **kw)
    plan.run()
    got = plan.results()
    want = ref.page_plan([int(x) for x in past], [int(x) for x in counts], [int(x) for x in held],
                         [[int(x) for x in r] for r in table], [int(x) for x in free], free_count, rows, page_tokens, pages)
    for name, value in want.items():
        assert np.array_equal(got[name], _words(np.atleast_1d(value)).reshape(got[name].shape)), name
    return plan, got


def _state(rng, requests, page_tokens, longest, spare):
    """Requests of random lengths with their pages, and `spare` free ones."""
    past = rng.integers(0, longest + 1, requests)
    held = -(-past // page_tokens)
    stride = int(held.max()) + 40
    pages = int(held.sum()) + spare
    order, at = rng.permutation(pages), 0
    table = np.full((requests, stride), 0xFFFFFFFF, np.uint64)
    for r, n in enumerate(held):
        table[r, :n] = order[at:at + n]
        at += n
    free = np.full(pages, 0xFFFFFFFE, np.uint64)
    free[:spare] = order[at:]
    return past, held, table, free, pages


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("requests,page_tokens,longest,spare,most,extra", [
    (1, 32, 0, 3, 1, 0), (1, 32, 64, 3, 1, 5), (1, 64, 5000, 40, 2000, 0), (5, 32, 200, 6, 3, 2), (24, 96, 900, 9, 40, 1),
    (64, 32, 4000, 5, 90, 0), (300, 32, 100, 150, 2, 7), (1024, 32, 60, 500, 1, 0), (1025, 64, 90, 700, 2, 3),
    (2500, 32, 40, 1000, 3, 0), (40, 128, 3000, 200, 600, 100), (3, 32, 100, 400, 9000, 11)])
def test_page_plan(ctx, dev, requests, page_tokens, longest, spare, most, extra, in_place):
    rng = np.random.default_rng(requests + most)
    past, held, table, free, pages = _state(rng, requests, page_tokens, longest, spare)
    counts = rng.integers(0, most + 1, requests) if most > 1 else np.ones(requests, np.int64)
    ended = rng.random(requests) < 0.1
    past, counts = np.where(ended, 0, past), np.where(ended, 0, counts)
    cut = rng.random(requests) < 0.1  # tokens taken back
    past = np.where(cut, past // 3, past)
    rows = max(1, int(counts.sum()) + extra)
    _check_plan(ctx, dev, past, counts, held, table, free, spare, rows, page_tokens, pages, in_place=in_place)


def test_page_plan_without_enough_pages(ctx, dev):
    """From the first request that is not served on, those that need pages get none."""
    table = [[7, 99, 99], [8, 99, 99], [9, 5, 99], [1, 99, 99]]
    for spare in range(5):
        free = [2, 3, 4, 6, 0, 0, 0, 0, 0, 0]
        _, got = _check_plan(ctx, dev, [32, 32, 40, 31], [1, 33, 1, 1], [1, 1, 2, 1], table, free, spare, 40, 32, 10)
        assert got["granted"].tolist() == [[0, 0, 1, 1], [1, 0, 1, 1], [1, 0, 1, 1], [1, 33, 1, 1], [1, 33, 1, 1]][spare]
    # a page given back in the step serves a request before it
    _, got = _check_plan(ctx, dev, [32, 0], [1, 0], [1, 2], [[7, 99], [5, 6]], [0, 0, 0, 0, 0, 0, 0, 0], 0, 1, 32, 8)
    assert got["granted"].tolist() == [1, 0] and got["table"][0].tolist() == [7, 6] and got["free_count"][0] == 1


def test_page_plan_of_requests_that_do_not_fit(ctx, dev):
    table = [[1, 2], [3, 4], [5, 6], [0, 9]]
    free = [7, 8, 0, 0, 0, 0, 0, 0, 0, 0]
    # more pages than a table's row; more rows than the step's; lengths past 32 bits
    _check_plan(ctx, dev, [64, 10, 20, 3], [1, 1, 1, 0], [2, 1, 1, 1], table, free, 2, 3, 32, 10)
    _check_plan(ctx, dev, [10, 30, 20, 0], [3, 4, 5, 0], [1, 1, 1, 2], table, free, 2, 9, 32, 10)
    _check_plan(ctx, dev, [0xFFFFFFFF, 10, 20, 0], [0xFFFFFFFF, 1, 0xFFFFFFFF, 0], [2, 1, 1, 0], table, free, 2, 5, 32, 10)


def test_page_plan_over_tables_that_are_wrong(ctx, dev):
    """Entries that are no page, more held than a row has, a stack's count past its end: nothing out of bounds."""
    table = [[1, 0xFFFFFFFF], [3, 10], [0x80000000, 6]]
    _check_plan(ctx, dev, [40, 33, 5], [1, 1, 1], [2, 2, 1], table, [7, 0xFFFFFFFF] + [0] * 8, 2, 4, 32, 10)
    _check_plan(ctx, dev, [0, 33, 5], [0, 1, 40], [0xFFFFFFFF, 2, 1], table, [7, 20] + [0] * 8, 2, 50, 32, 10)
    _check_plan(ctx, dev, [0, 0, 0], [0, 0, 0], [2, 2, 2], table, list(range(10)), 9, 1, 32, 10)    # more than the stack holds
    _check_plan(ctx, dev, [0, 0, 0], [40, 40, 40], [0, 0, 0], table, list(range(10)), 1 << 31, 200, 32, 10)


@pytest.mark.parametrize("requests,rows", [(30, 60), (900, 1000), (6, 9000)])
def test_page_plan_step_after_step(ctx, dev, requests, rows):
    """Requests that come, grow, are cut and end, the state in place; no page is ever in two hands."""
    from tests.support import requests_ref as ref

    rng = np.random.default_rng(rows)
    page_tokens, pages, stride = 32, 40 + 4 * requests, 320
    past, held = np.zeros(requests, np.int64), [0] * requests
    table, free, left = [[NOWHERE] * stride for _ in range(requests)], rng.permutation(pages).tolist(), pages
    plan = _Plan(ctx, dev, past, past, held, table, free, left, rows, page_tokens, pages, in_place=True)
    inputs = {n: next(b for b in dev.owned if b.ptr == p) for n, p in (("past", plan.call.past), ("counts", plan.call.counts))}
    for step in range(12):
        wish = rng.choice([0, 1, 1, 1, 5, rows // 3], requests)
        counts = np.where(np.cumsum(wish) <= rows + 3, wish, 0)
        gone = rng.random(requests) < 0.15
        past, counts = np.where(gone, 0, past), np.where(gone, 0, counts)
        inputs["past"].write(_words(past))
        inputs["counts"].write(_words(counts))
        plan.run()
        got = plan.results()
        want = ref.page_plan(past.tolist(), counts.tolist(), held, table, free, left, rows, page_tokens, pages)
        for name, value in want.items():
            assert np.array_equal(got[name], _words(np.atleast_1d(value)).reshape(got[name].shape)), (step, name)
        table, free, left, held = want["table"], want["free"], want["free_count"], want["held"]
        hands = free[:left] + [p for r, n in enumerate(held) for p in table[r][:n]]
        assert sorted(hands) == list(range(pages))
        past = past + np.array(want["granted"])


NOWHERE = 0xFFFFFFFF


# ---- the pool -------------------------------------------------------------------


class _Pool:
    """A pool whose unwritten bytes are `byte`, and its memory."""

    def __init__(self, dev, format_, pages, page_tokens, kv_heads, dim, byte=0xFF):
        from charlotte_amd import serving as sv
        from tests.support import serving_ref as ref

        nbytes = sv.page_pool_bytes(ref.FORMATS[format_], pages, page_tokens, kv_heads, dim)
        memory, _ = dev.room(nbytes, np.uint8, byte=byte)
        self.pool = sv.PagePool(dev.ctx, ref.FORMATS[format_], pages, page_tokens, kv_heads, dim, device=memory, nbytes=nbytes)
        self.dev = dev

    def write(self, k, v, slots, key_stride=0, value_stride=0):
        from charlotte_amd import harness as hx

        self.pool.append(self.dev.put(k), self.dev.put(v), self.dev.put(_words(slots)), len(slots), key_stride, value_stride)
        hx.sync()

    def read(self, slots, width, fill=5.0):
        from charlotte_amd import harness as hx

        to = [self.dev.put(np.full((len(slots), width), fill, np.float32)) for _ in range(2)]
        held = self.dev.owned[-2:]
        self.pool.read(*to, self.dev.put(_words(slots)), len(slots))
        hx.sync()
        return [b.read(np.float32, len(slots) * width).reshape(len(slots), width) for b in held]


@pytest.mark.parametrize("format_", FORMATS)
@pytest.mark.parametrize("heads,dim,page_tokens,pages,rows", [
    (2, 64, 32, 9, 1), (1, 32, 32, 3, 40), (3, 96, 64, 6, 77), (8, 128, 96, 5, 130), (1, 256, 128, 4, 300), (2, 224, 32, 40, 900)])
def test_a_pool_reads_back_what_its_format_holds(ctx, dev, format_, heads, dim, page_tokens, pages, rows):
    """Slots in any order, runs of whole tiles among them, and rows without a slot."""
    from tests.support import serving_ref as ref

    rng = np.random.default_rng(rows + dim)
    print("page_append", format_, heads, dim, page_tokens, pages, rows, flush=True)
    width, all_ = heads * dim, pages * page_tokens
    slots = rng.permutation(all_)[:rows]
    if rows >= 77:  # a prompt's run over two pages, from the middle of a tile on
        run = [p * page_tokens + t for p in (2, 0) for t in range(page_tokens)][11:11 + 50]
        others = [s for s in slots.tolist() if s not in run]
        slots = np.array((others[:13] + run + others[13:])[:rows])
    bad = rng.random(len(slots)) < 0.1
    given = np.where(bad, rng.choice([NOWHERE, all_, all_ + 7, 0x80000000], len(slots)), slots)
    k, v = (rng.standard_normal((len(slots), width)).astype(np.float32) * 3 for _ in range(2))
    k[0, 3], v[-1, 7] = np.nan, np.inf  # blocks that no format holds
    pool = _Pool(dev, format_, pages, page_tokens, heads, dim, byte=0)
    before = pool.read(np.arange(all_), width)
    wide = [np.concatenate([x, np.full((len(slots), 12), np.nan, np.float32)], 1) for x in (k, v)]
    pool.write(*wide, given, width + 12, width + 12)
    for got, x, old in zip(pool.read(given, width), (k, v), before):
        want = ref.stored(x.reshape(-1, heads, dim), format_).reshape(x.shape)
        assert np.array_equal(got, np.where(bad[:, None], np.float32(5), want), equal_nan=True)
    rest = np.setdiff1d(np.arange(all_), given[~bad])
    for got, old in zip(pool.read(rest, width), before):
        assert np.array_equal(got, old[rest], equal_nan=True)
    pool.pool.free()


@pytest.mark.parametrize("format_,heads,dim,page_tokens,lengths", [
    ("q8_0", 8, 128, 64, (530, 1, 1, 97, 1)), ("q4_0", 4, 256, 32, (1, 31, 32, 33, 300, 250)), ("f16", 8, 128, 2048, (700,)),
    ("q8_0", 1, 32, 128, (9000, 1, 7400, 1, 5)), ("f16", 2, 224, 96, (640, 640))])
def test_a_pool_of_many_rows(ctx, dev, format_, heads, dim, page_tokens, lengths):
    """Prompts of any lengths, each from the middle of a page on, over pages in any order."""
    from tests.support import serving_ref as ref

    rng = np.random.default_rng(dim + len(lengths))
    print("page_append", format_, heads, dim, page_tokens, lengths, flush=True)
    width, slots = heads * dim, []
    pages = sum(n // page_tokens + 2 for n in lengths)
    order = rng.permutation(pages).tolist()
    for n in lengths:
        past = int(rng.integers(page_tokens))
        held = [order.pop() for _ in range(-(-(past + n) // page_tokens))]
        slots += [held[t // page_tokens] * page_tokens + t % page_tokens for t in range(past, past + n)]
    slots = np.array(slots)
    k, v = (rng.standard_normal((len(slots), width)).astype(np.float32) for _ in range(2))
    pool = _Pool(dev, format_, pages, page_tokens, heads, dim, byte=0)
    bad = rng.random(len(slots)) < 0.01
    given = np.where(bad, NOWHERE, slots)
    rest = np.setdiff1d(np.arange(pages * page_tokens), given[~bad])
    before = pool.read(rest, width)
    pool.write(k, v, given)
    for got, x in zip(pool.read(given, width), (k, v)):
        want = ref.stored(x.reshape(-1, heads, dim), format_).reshape(x.shape)
        assert np.array_equal(got, np.where(bad[:, None], np.float32(5), want))
    for got, old in zip(pool.read(rest, width), before):
        assert np.array_equal(got, old)
    pool.pool.free()


# ---- paged attention --------------------------------------------------------------


def _check_paged(dev, format_, requests, heads, kv_heads, dim, page_tokens=32, window=0, seed=0, most=None, rows=None,
                 granted=None, scale=None, spread=1.0, query_stride=0, output_stride=0, stride=None, twice=False, grow=0, longest=0):
    """requests: (past, count) each. Every row of theirs against the restatement, others left as they were."""
    from charlotte_amd import harness as hx
    from charlotte_amd import serving as sv
    from tests.support import serving_ref as ref

    rng = np.random.default_rng(seed)
    counts = [c for _, c in requests]
    starts = [sum(counts[:i]) for i in range(len(counts) + 1)]
    rows = rows or max(1, starts[-1])
    granted = counts if granted is None else granted
    held = [-(-(p + c) // page_tokens) for p, c in requests]
    pages = sum(held) + 3
    order = rng.permutation(pages).tolist()
    width = max(max(held), 1) if stride is None else stride
    table = np.full((len(requests), width), NOWHERE, np.uint64)
    print("paged_attention", format_, len(requests), requests[:4], heads, kv_heads, dim, page_tokens, window, flush=True)
    pool = _Pool(dev, format_, pages, page_tokens, kv_heads, dim)
    keys, values = [], []
    for r, (p, c) in enumerate(requests):
        table[r, :held[r]] = [order.pop() for _ in range(held[r])]
        n = p + c
        k = rng.standard_normal((n, kv_heads, dim)).astype(np.float32)
        v = (rng.standard_normal((n, kv_heads, dim)) * spread).astype(np.float32)
        if grow:  # in octaves, a token's values less or more than another's
            v *= (2.0 ** -rng.integers(0, grow, (n, 1, 1))).astype(np.float32) * np.float32(2.0 ** (grow // 2))
        keys.append(k)
        values.append(v)
    slots = [int(table[r, t // page_tokens]) * page_tokens + t % page_tokens
             for r, (p, c) in enumerate(requests) for t in range(p + c)]
    if slots:
        pool.write(np.concatenate(keys).reshape(len(slots), -1), np.concatenate(values).reshape(len(slots), -1), slots)
    q = rng.standard_normal((rows, heads, dim)).astype(np.float32)
    scale = dim ** -0.5 if scale is None else scale
    in_width, out_width = query_stride or heads * dim, output_stride or heads * dim
    given = np.zeros((rows, in_width), np.float32)
    given[:, :heads * dim] = q.reshape(rows, -1)
    most = max(counts) if most is None else most
    need = sv.paged_attention_workspace_bytes(dev.ctx, pool.pool, heads, most)
    work, _ = dev.room(need, np.uint8)
    out, read = dev.room(rows * out_width)
    call = sv.PagedAttention(pool.pool, dev.put(given), out, heads, scale, len(requests), rows,
                             dev.put(_words([p for p, _ in requests])), dev.put(_words(granted)), dev.put(_words(starts)),
                             dev.put(_words(table)), width, window, most, query_stride, output_stride, work, need, longest)
    sv.paged_attention(dev.ctx, call)
    hx.sync()
    got = read().reshape(rows, out_width)
    for _ in range(2 if twice else 0):
        sv.paged_attention(dev.ctx, call)
        hx.sync()
        assert np.array_equal(read().view(np.uint32), got.ravel().view(np.uint32))
    assert (got[:, heads * dim:].view(np.uint32) == NOWHERE).all()
    got = got[:, :heads * dim].reshape(rows, heads, dim)
    touched = np.zeros(rows, bool)
    for r, (past, count) in enumerate(requests):
        if granted[r] == 0 or starts[r] + granted[r] > rows:
            continue
        at = slice(starts[r], starts[r] + count)
        touched[at] = True
        want, weight, size = ref.attention(q[at], ref.stored(keys[r], format_), ref.stored(values[r], format_), past, scale,
                                           window=window)
        # as attention's, and once more for each piece that is joined; NaNs where a block is not held
        none = np.isnan(want)
        assert np.array_equal(np.isnan(got[at]), none), r
        assert (np.abs(got[at] - want) <= ref.attention_bound(weight, size, past + count + 32 * 256, dim))[~none].all(), r
    assert (got[~touched].view(np.uint32) == NOWHERE).all()
    pool.pool.free()
    return got


@pytest.mark.parametrize("format_", FORMATS)
@pytest.mark.parametrize("dim", [32, 64, 96, 128, 160, 192, 224, 256])
def test_paged_attention_at_every_head_width(ctx, dev, format_, dim):
    _check_paged(dev, format_, [(70, 1), (0, 1), (31, 1), (400, 1)], 4, 2, dim, seed=dim)
    _check_paged(dev, format_, [(45, 13), (0, 3), (90, 1)], 6, 2, dim, page_tokens=64, seed=dim + 1)  # 39 rows


@pytest.mark.parametrize("format_", FORMATS)
@pytest.mark.parametrize("requests,heads,kv_heads,page_tokens", [
    ([(0, 1)], 4, 4, 32), ([(31, 1), (32, 1), (33, 1)], 8, 1, 32), ([(5000, 1)], 16, 8, 96), ([(12, 0), (700, 1), (3, 0)], 7, 7, 64),
    ([(0, 200)], 3, 1, 32), ([(333, 130), (0, 1), (64, 64)], 6, 2, 128), ([(9, 1), (2000, 2), (100, 40)], 33, 1, 32),
    ([(100, 17), (5, 300), (6000, 1), (0, 2)], 4, 4, 2048)])
def test_paged_attention_of_requests_of_any_lengths(ctx, dev, format_, requests, heads, kv_heads, page_tokens):
    _check_paged(dev, format_, requests, heads, kv_heads, 64, page_tokens=page_tokens, seed=heads, twice=True)


@pytest.mark.parametrize("dim,heads,kv_heads,lengths", [
    (32, 1, 1, [40000]), (32, 2, 2, [30000, 10, 5, 0, 900, 12000]), (64, 4, 4, [100] * 70 + [9000] + [30] * 40),
    (32, 1, 1, [33] * 600), (32, 2, 1, list(range(0, 1300))), (128, 8, 8, [3000, 1, 2000, 17, 500, 4000])])
def test_paged_attention_shares_its_work_evenly(ctx, dev, dim, heads, kv_heads, lengths):
    """Lines of several parts: units in many pieces, many units in one part, more requests than threads."""
    _check_paged(dev, "q8_0", [(n, 1) for n in lengths], heads, kv_heads, dim, seed=len(lengths), twice=True)


@pytest.mark.parametrize("format_", FORMATS)
@pytest.mark.parametrize("dim", [32, 64, 96, 128, 160, 256])
def test_paged_attention_of_many_rows(ctx, dev, format_, dim):
    """Requests that bring 256 rows of a key head and more, beside others: workgroups of many rows, in pieces and whole."""
    _check_paged(dev, format_, [(150, 91), (40, 1), (700, 86), (0, 85)], 3, 1, dim, page_tokens=64, seed=dim, twice=True)


@pytest.mark.parametrize("requests,heads,kv_heads,page_tokens,window", [
    ([(0, 700)], 2, 2, 32, 0), ([(3000, 300)], 2, 1, 96, 0), ([(33000, 130)], 2, 1, 32, 0),   # more pages than LDS keeps
    ([(500, 256), (10, 255), (20, 257), (0, 1)], 1, 1, 32, 0), ([(500, 300), (0, 260)], 4, 2, 32, 70),
    ([(900, 280), (77, 1)], 1, 1, 32, 1), ([(100, 300), (4000, 300)], 8, 8, 128, 1000)])
def test_paged_attention_of_many_rows_in_pieces(ctx, dev, requests, heads, kv_heads, page_tokens, window):
    _check_paged(dev, "q8_0", requests, heads, kv_heads, 64, page_tokens=page_tokens, window=window, seed=heads, twice=True)
    _check_paged(dev, "f16", requests, heads, kv_heads, 32, page_tokens=page_tokens, window=window, seed=heads, spread=100.0)


def test_many_rows_of_scales_far_apart(ctx, dev):
    """Values whose scales a layout is not made for; the largest are past what Q4_0's scales hold."""
    _check_paged(dev, "q8_0", [(300, 130), (64, 1)], 2, 1, 64, seed=3, grow=40)
    _check_paged(dev, "q4_0", [(300, 130), (64, 1)], 2, 1, 64, seed=3, grow=28)
    _check_paged(dev, "q4_0", [(300, 130), (64, 1)], 2, 1, 64, seed=3, grow=40)


def test_pages_that_the_pool_does_not_have_of_many_rows(ctx, dev):
    from charlotte_amd import harness as hx
    from charlotte_amd import serving as sv
    from tests.support import serving_ref as ref

    rng = np.random.default_rng(15)
    pool = _Pool(dev, "q8_0", 12, 32, 1, 32)
    k, v = (rng.standard_normal((12 * 32, 32)).astype(np.float32) for _ in range(2))
    pool.write(k, v, np.arange(384))
    table = _words([[3, 4, 5, 6, 12, 8, 9, 10, 11], [0, 1, 2, 3, 4, 5, 6, 7, 8], [0, 1, 2, 3, 4, 5, 6, 7, 8]])
    past, counts, starts = [20, 20, 40], [260, 260, 260], [0, 260, 520, 780]  # the last passes nine pages
    q = rng.standard_normal((780, 1, 32)).astype(np.float32)
    need = sv.paged_attention_workspace_bytes(ctx, pool.pool, 1, 260)
    work, _ = dev.room(need, np.uint8)
    for window in (0, 40):
        out, read = dev.room(780 * 32)
        sv.paged_attention(ctx, sv.PagedAttention(pool.pool, dev.put(q), out, 1, 0.2, 3, 780, dev.put(_words(past)),
                                                  dev.put(_words(counts)), dev.put(_words(starts)), dev.put(table), 9, window, 260,
                                                  workspace=work, workspace_bytes=need))
        hx.sync()
        got = read().reshape(780, 1, 32)
        # page 4 has places 128 .. 159; token t stands at 20 + t
        t = np.arange(260) + 20
        sees = (t >= 128) & ((window == 0) | (t - window + 1 <= 159))
        assert np.isnan(got[:260][sees]).all() and np.isfinite(got[:260][~sees]).all()
        assert np.isnan(got[520:]).all()
        of = [int(table[1][i // 32]) * 32 + i % 32 for i in range(280)]
        want, weight, size = ref.attention(q[260:520], ref.stored(k, "q8_0")[of][:, None], ref.stored(v, "q8_0")[of][:, None], 20, 0.2,
                                           window=window)
        assert (np.abs(got[260:520] - want) <= ref.attention_bound(weight, size, 400, 32)).all()
    pool.pool.free()


@pytest.mark.parametrize("window", [1, 2, 31, 64, 100, 1000])
def test_paged_attention_in_a_window(ctx, dev, window):
    _check_paged(dev, "q8_0", [(200, 1), (63, 1), (150, 20), (10, 70), (0, 1), (3000, 2)], 4, 1, 128, window=window, seed=window)


@pytest.mark.parametrize("most", [0, 1, 7, 1000])
def test_the_most_tokens_named_change_no_answer(ctx, dev, most):
    _check_paged(dev, "q4_0", [(200, 9), (63, 1), (150, 20)], 8, 4, 64, most=most, seed=1)


@pytest.mark.parametrize("longest", [1, 300, 1 << 30])
def test_the_longest_named_changes_no_answer(ctx, dev, longest):
    _check_paged(dev, "q8_0", [(4000, 90), (17, 1), (0, 260), (3000, 3)], 8, 1, 64, page_tokens=64, longest=longest, seed=3)


def test_requests_that_share_pages(ctx, dev):
    """Two continuations of one prompt, whose pages stand in both rows."""
    from charlotte_amd import harness as hx
    from charlotte_amd import serving as sv
    from tests.support import serving_ref as ref

    rng = np.random.default_rng(8)
    heads, kv_heads, dim, shared = 8, 2, 64, 5 * 32
    pool = _Pool(dev, "q8_0", 9, 32, kv_heads, dim)
    past, counts = [shared + 3, shared + 7], [2, 1]
    table = np.array([[8, 0, 7, 2, 5, 1], [8, 0, 7, 2, 5, 6]])
    slots = [table[0, t // 32] * 32 + t % 32 for t in range(shared + 5)] + [6 * 32 + t for t in range(8)]
    k, v = (rng.standard_normal((len(slots), kv_heads, dim)).astype(np.float32) for _ in range(2))
    pool.write(k.reshape(len(slots), -1), v.reshape(len(slots), -1), slots)
    q = rng.standard_normal((3, heads, dim)).astype(np.float32)
    need = sv.paged_attention_workspace_bytes(ctx, pool.pool, heads, 2)
    work, _ = dev.room(need, np.uint8)
    out, read = dev.room(3 * heads * dim)
    sv.paged_attention(ctx, sv.PagedAttention(pool.pool, dev.put(q), out, heads, 0.1, 2, 3, dev.put(_words(past)),
                                              dev.put(_words(counts)), dev.put(_words([0, 2, 3])), dev.put(_words(table)), 6, most=2,
                                              workspace=work, workspace_bytes=need))
    hx.sync()
    got = read().reshape(3, heads, dim)
    own = [slice(shared, shared + 5), slice(shared + 5, shared + 13)]
    for at, p, mine in zip((slice(0, 2), slice(2, 3)), past, own):
        kv = [ref.stored(np.concatenate([x[:shared], x[mine]]), "q8_0") for x in (k, v)]
        want, weight, size = ref.attention(q[at], *kv, p, 0.1)
        assert (np.abs(got[at] - want) <= ref.attention_bound(weight, size, shared + 8 + 32 * 256, dim)).all()
    pool.pool.free()


@pytest.mark.parametrize("format_,dim,rows", [("q8_0", 128, 128), ("q4_0", 64, 256), ("f16", 160, 128)])
def test_requests_of_about_many_rows(ctx, dev, format_, dim, rows):
    """A row less than takes the form of many rows, as many, one more, and few, in one step."""
    _check_paged(dev, format_, [(3300, rows - 1), (3300, rows), (7, 1), (3301, rows + 1)], 16, 16, dim, page_tokens=64, seed=dim,
                 twice=True)


def test_many_rows_over_long_pieces(ctx, dev):
    """Pieces of more tiles than a workgroup keeps the places of, beside a short request; rows here and there against 64 bits."""
    from charlotte_amd import harness as hx
    from charlotte_amd import serving as sv
    from tests.support import serving_ref as ref

    rng = np.random.default_rng(67)
    heads, kv_heads, dim, page_tokens = 64, 2, 32, 64
    past, counts = [67003, 40], [512, 2]
    held = [-(-(p + c) // page_tokens) for p, c in zip(past, counts)]
    pages, stride = sum(held), max(held)
    order = rng.permutation(pages)
    table = np.full((2, stride), NOWHERE, np.uint64)
    table[0, :held[0]], table[1, :held[1]] = order[:held[0]], order[held[0]:]
    slots = [np.arange(p + c) % page_tokens + table[r, np.arange(p + c) // page_tokens] * page_tokens
             for r, (p, c) in enumerate(zip(past, counts))]
    k, v = ([rng.standard_normal((len(x), kv_heads, dim)).astype(np.float32) for x in slots] for _ in range(2))
    pool = _Pool(dev, "q8_0", pages, page_tokens, kv_heads, dim)
    pool.write(*(np.concatenate(x).reshape(-1, kv_heads * dim) for x in (k, v)), np.concatenate(slots))
    rows = sum(counts)
    q = rng.standard_normal((rows, heads, dim)).astype(np.float32)
    need = sv.paged_attention_workspace_bytes(ctx, pool.pool, heads, 512)
    work, _ = dev.room(need, np.uint8)
    out, read = dev.room(rows * heads * dim)
    sv.paged_attention(ctx, sv.PagedAttention(pool.pool, dev.put(q), out, heads, dim ** -0.5, 2, rows, dev.put(_words(past)),
                                              dev.put(_words(counts)), dev.put(_words([0, 512, 514])), dev.put(_words(table)), stride,
                                              most=512, workspace=work, workspace_bytes=need))
    hx.sync()
    got = read().reshape(rows, heads, dim)
    assert np.isfinite(got).all()
    held_kv = [[ref.stored(x, "q8_0") for x in kv] for kv in zip(k, v)]
    for row in (0, 1, 255, 301, 511, 512, 513):
        r, t = (0, row) if row < 512 else (1, row - 512)
        n = past[r] + t + 1
        want, weight, size = ref.attention(q[row:row + 1], *(x[:n] for x in held_kv[r]), past[r] + t, dim ** -0.5)
        assert (np.abs(got[row:row + 1] - want) <= ref.attention_bound(weight, size, n + 32 * 256, dim)).all(), row
    pool.pool.free()


def test_rows_of_no_request_are_left_as_they_were(ctx, dev):
    _check_paged(dev, "q8_0", [(20, 3), (50, 1), (90, 2)], 4, 2, 64, rows=9, seed=2)
    _check_paged(dev, "q8_0", [(20, 3), (50, 1), (90, 2)], 4, 2, 64, granted=[3, 0, 2], seed=2)
    _check_paged(dev, "q8_0", [(20, 3), (50, 1), (90, 2)], 4, 2, 64, rows=5, seed=2)  # the last does not fit
    _check_paged(dev, "q8_0", [(20, 0), (50, 0)], 4, 2, 64, rows=2, seed=2)


def test_paged_strides(ctx, dev):
    _check_paged(dev, "f16", [(40, 3), (77, 1)], 4, 2, 96, query_stride=4 * 96 + 64, output_stride=4 * 96 + 20, stride=9)


@pytest.mark.parametrize("format_", FORMATS)
@pytest.mark.parametrize("spread", [1e-2, 300.0])
def test_paged_values_of_any_size(ctx, dev, format_, spread):
    _check_paged(dev, format_, [(300, 5), (2000, 1)], 4, 2, 64, spread=spread, seed=4)


def test_pages_that_the_pool_does_not_have(ctx, dev):
    """NaNs for the rows that see such a page, or a token past the table's row; the others as they should be."""
    from charlotte_amd import harness as hx
    from charlotte_amd import serving as sv
    from tests.support import serving_ref as ref

    rng = np.random.default_rng(5)
    pool = _Pool(dev, "q8_0", 8, 32, 1, 64)
    k, v = (rng.standard_normal((8 * 32, 64)).astype(np.float32) for _ in range(2))
    pool.write(k, v, np.arange(256))
    table = [[0, 8, 2], [3, 4, 5], [NOWHERE, 6, 7], [1, 1, 1], [0, 1, 2]]
    past, counts = [70, 70, 70, 40, 97], [2, 2, 1, 1, 1]
    starts = [0, 2, 4, 5, 6, 7]
    q = rng.standard_normal((7, 2, 64)).astype(np.float32)
    need = sv.paged_attention_workspace_bytes(ctx, pool.pool, 2, 2)
    work, _ = dev.room(need, np.uint8)
    for window in (0, 20, 40):
        out, read = dev.room(7 * 128)
        sv.paged_attention(ctx, sv.PagedAttention(pool.pool, dev.put(q), out, 2, 0.125, 5, 7, dev.put(_words(past)),
                                                  dev.put(_words(counts)), dev.put(_words(starts)), dev.put(_words(table)), 3,
                                                  window, 2, workspace=work, workspace_bytes=need))
        hx.sync()
        got = read().reshape(7, 2, 64)
        # request 0's page 1 holds places 32 .. 63: 70's window of 20 begins at 51, of 40 at 31
        assert np.isnan(got[0:2]).all()
        assert (np.isfinite(got[4]) if window == 20 else np.isnan(got[4])).all()  # page 0's places are 0 .. 31
        assert np.isnan(got[6]).all()  # place 97 is past three pages
        for r, at in ((1, slice(2, 4)), (3, slice(5, 6))):
            of = [table[r][t // 32] * 32 + t % 32 for t in range(past[r] + counts[r])]
            want, weight, size = ref.attention(q[at], ref.stored(k, "q8_0")[of][:, None], ref.stored(v, "q8_0")[of][:, None],
                                               past[r], 0.125, window=window)
            assert (np.abs(got[at] - want) <= ref.attention_bound(weight, size, 300, 64)).all()
    pool.pool.free()


def test_starts_and_counts_that_are_no_steps(ctx, dev):
    """Requests whose counts together pass every bound: nothing past the output is written, and the call ends."""
    from charlotte_amd import harness as hx
    from charlotte_amd import serving as sv

    rows, requests = 4096, 65536
    pool = _Pool(dev, "q4_0", 4, 2048, 1, 32).pool
    need = sv.paged_attention_workspace_bytes(ctx, pool, 16)
    work, _ = dev.room(need, np.uint8)
    q = dev.put(np.ones((rows, 16 * 32), np.float32))
    out, read = dev.room(rows * 16 * 32 + 4096)
    full = {n: dev.put(np.full(requests, v, np.uint32)) for n, v in (("past", 3000), ("counts", rows), ("starts", 0), ("none", 0xFFFFFFFF))}
    table = dev.put(np.zeros((requests, 60), np.uint32))
    for past, counts, starts in (("past", "counts", "starts"), ("none", "none", "none"), ("past", "none", "starts")):
        sv.paged_attention(ctx, sv.PagedAttention(pool, q, out, 16, 0.1, requests, rows, full[past], full[counts], full[starts],
                                                  table, 60, workspace=work, workspace_bytes=need))
        hx.sync()
        assert (read()[rows * 16 * 32:].view(np.uint32) == NOWHERE).all()
    pool.free()


def test_pool_offsets_past_32_bits(ctx, dev):
    """A pool of more than 4 GiB, its last pages."""
    from charlotte_amd import harness as hx
    from charlotte_amd import serving as sv
    from tests.support import serving_ref as ref

    rng = np.random.default_rng(3)
    pages, page_tokens, kv_heads, dim = 2200, 256, 8, 256
    assert sv.page_pool_bytes(ref.FORMATS["f16"], pages, page_tokens, kv_heads, dim) > 1 << 32
    pool = sv.PagePool(ctx, ref.FORMATS["f16"], pages, page_tokens, kv_heads, dim)
    table, past = np.array([[pages - 1, 3, pages - 2]]), 600
    slots = _words([table[0, t // page_tokens] * page_tokens + t % page_tokens for t in range(past + 1)])
    k, v = (rng.standard_normal((past + 1, kv_heads, dim)).astype(np.float32) for _ in range(2))
    pool.append(dev.put(k), dev.put(v), dev.put(slots), past + 1)
    q = rng.standard_normal((1, kv_heads, dim)).astype(np.float32)
    need = sv.paged_attention_workspace_bytes(ctx, pool, kv_heads, 1)
    work, _ = dev.room(need, np.uint8)
    out, read = dev.room(q.size)
    sv.paged_attention(ctx, sv.PagedAttention(pool, dev.put(q), out, kv_heads, 0.0625, 1, 1, dev.put(_words([past])),
                                              dev.put(_words([1])), dev.put(_words([0, 1])), dev.put(_words(table)), 3,
                                              workspace=work, workspace_bytes=need))
    hx.sync()
    want, weight, size = ref.attention(q, ref.stored(k, "f16"), ref.stored(v, "f16"), past, 0.0625)
    assert (np.abs(read().reshape(q.shape) - want) <= ref.attention_bound(weight, size, past + 32 * 256, dim)).all()
    pool.free()


# ---- residual_norm ------------------------------------------------------------------


@pytest.mark.parametrize("rows,width,branch,after,gate,scales,layout", [
    (1, 1024, True, False, None, (1.0, 1.0), {}), (3, 1, True, True, "shared", (0.5, 2.0), {}), (7, 3, True, False, "rows", (1, 1), {}),
    (5, 64, True, True, None, (1.0, 1.0), {"stride": 68}), (2, 255, True, True, "rows", (1.0, -0.25), {"offset": 4}),
    (9, 1152, False, False, None, (1.0, 1.0), {}), (4, 1155, True, True, "shared", (0.875, 0.22), {"stride": 1163}),
    (300, 2048, True, True, None, (1.0, 1.0), {"in_place": True}), (2, 4096, True, False, "shared", (1.0, 0.1), {"in_place": True}),
    (33, 4100, True, True, "rows", (1.0, 1.0), {"offset": 8}), (1, 8192, True, True, None, (2.0, 1.0), {}),
    (3, 16384, True, True, "rows", (1.0, 1.0), {}), (2, 16385, True, True, "shared", (1.0, 1.0), {"offset": 4}),
    (2, 32768, True, True, "rows", (1.0, 1.0), {}), (2, 32767, True, True, "rows", (1.0, 1.0), {}),
    (2000, 96, True, True, None, (0.0, 1.0), {}), (5, 640, False, False, None, (0.5, 7.0), {"offset": 12})])
@pytest.mark.parametrize("results", ["both", "residual", "normed"])
def test_residual_norm(ctx, dev, rows, width, branch, after, gate, scales, layout, results):
    from charlotte_amd import harness as hx
    from charlotte_amd import serving as sv
    from tests.support import requests_ref as ref

    rng = np.random.default_rng(rows + width)
    stride, offset = layout.get("stride", width), layout.get("offset", 0)
    x, y = (rng.standard_normal((rows, stride)).astype(np.float32) * s for s in (4, 0.5))
    x[0, :width], y[0, :width] = 0.0, 0.0  # rows of zeros: epsilon alone
    x[-1, 0] += 300
    w, v = (rng.standard_normal(width).astype(np.float32) for _ in range(2))
    g = rng.standard_normal((rows if gate == "rows" else 1, width)).astype(np.float32)
    print("residual_norm", rows, width, branch, after, gate, scales, layout, results, flush=True)
    xp = dev.put(x, offset)
    x_at = dev.owned[-1]
    to, read = dev.room(rows * stride, offset=offset)
    if layout.get("in_place"):
        to, read = xp, lambda: x_at.read(np.float32, rows * stride, offset)
    normed, read_normed = dev.room(rows * stride, offset=offset)
    call = sv.ResidualNorm(width, xp, dev.put(y, offset) if branch else 0, to if results != "normed" else 0,
                           normed if results != "residual" else 0, dev.put(v, offset) if results != "residual" else 0,
                           dev.put(w, offset) if after else 0, dev.put(g) if gate else 0, *scales, 1e-6, stride, stride,
                           width if gate == "rows" else 0, stride, stride)
    sv.residual_norm(ctx, call, rows)
    hx.sync()
    r, n, off_r, off_n = ref.residual_norm(x[:, :width], y[:, :width] if branch else None, w if after else None,
                                           g if gate else None, v, *scales, 1e-6)
    untouched = np.uint32(NOWHERE)
    for wanted, got, want, off in ((results != "normed", read, r, off_r), (results != "residual", read_normed, n, off_n)):
        if not wanted:
            continue
        got = got().reshape(rows, stride)
        assert (np.abs(got[:, :width] - want) <= off + 1e-30).all()
        if not layout.get("in_place"):
            assert (got[:, width:].view(np.uint32) == untouched).all()


def test_residual_norm_over_its_inputs(ctx, dev):
    """The stream's norm where the branch was, the stream where it was; values that are not finite keep to their row."""
    from charlotte_amd import harness as hx
    from charlotte_amd import serving as sv
    from tests.support import requests_ref as ref

    rng = np.random.default_rng(6)
    x, y = (rng.standard_normal((6, 512)).astype(np.float32) for _ in range(2))
    x[1, 5], y[2, 9] = np.inf, np.nan
    w, v = (rng.standard_normal(512).astype(np.float32) for _ in range(2))
    xp, yp = dev.put(x), dev.put(y)
    at = dev.owned[-2:]
    sv.residual_norm(ctx, sv.ResidualNorm(512, xp, yp, xp, yp, dev.put(v), dev.put(w)), 6)
    hx.sync()
    with np.errstate(all="ignore"):
        r, n, off_r, off_n = ref.residual_norm(x, y, w, None, v, 1, 1, 1e-6)
    got_r, got_n = (b.read(np.float32, 6 * 512).reshape(6, 512) for b in at)
    fine = [0, 3, 4, 5]
    assert (np.abs(got_r - r)[fine] <= off_r[fine]).all() and (np.abs(got_n - n)[fine] <= off_n[fine]).all()
    assert got_r[1, 5] == np.inf and np.isnan(got_n[1, 5]) and np.isnan(got_r[2]).all() and np.isnan(got_n[2]).all()


# ---- sample -----------------------------------------------------------------------


def _check_sample(ctx, dev, logits, settings, layout=None):
    """settings: (temperature, top_k, top_p, min_p, uniform) of each row."""
    from charlotte_amd import harness as hx
    from charlotte_amd import serving as sv
    from tests.support import requests_ref as ref

    layout = layout or {}
    rows, vocabulary = logits.shape
    stride, offset = layout.get("stride", vocabulary), layout.get("offset", 0)
    wide = np.full((rows, stride), 1e30, np.float32)
    wide[:, :vocabulary] = logits
    print("sample", rows, vocabulary, layout, flush=True)
    arrays = [np.array(a, np.int32 if i == 1 else np.float32) for i, a in enumerate(zip(*settings))]
    need = sv.sample_workspace_bytes(rows, vocabulary)
    work, _ = dev.room(need, np.uint8)
    (out, read), (chances, read_chances) = dev.room(rows, np.int32), dev.room(rows)
    pointers = [dev.put(a) for a in arrays]
    at = dev.put(wide, offset)
    calls = [sv.Sample(at, out, rows, vocabulary, pointers[4], 9.0, 3, 0.1, 0.9, *pointers[:4], chances=chances,
                       logit_stride=stride, workspace=work, workspace_bytes=need)]
    if len(set(map(tuple, (np.nan_to_num(np.array(s[:4], np.float64), nan=-7.0) for s in settings)))) == 1:
        t, k, p, m, _ = settings[0]
        calls.append(sv.Sample(at, out, rows, vocabulary, pointers[4], t, k, p, m, chances=chances, logit_stride=stride,
                               workspace=work, workspace_bytes=need))
    want = [ref.sample(l, *s) for l, s in zip(logits, settings)]
    for call in calls:
        sv.sample(ctx, call)
        hx.sync()
        assert read().tolist() == [t for t, _, _ in want]
        for got, (token, weight, total) in zip(read_chances(), want):
            # f32's rounding, and a unit of a weight either way
            assert abs(float(got) - weight / total) <= 2.0 ** -24 * weight / total + 2 / total
    return read()


CHOICES = dict(t=[0.6, 0.7, 1.0, 1.3, 0.0, 3.0], k=[0, 0, 20, 50, 1000, 1, -5], p=[1.0, 0.8, 0.95, 0.999, 0.1],
               m=[0.0, 0.0, 0.05, 0.3])


def _settings(rng, rows):
    return [(rng.choice(CHOICES["t"]), int(rng.choice(CHOICES["k"])), rng.choice(CHOICES["p"]), rng.choice(CHOICES["m"]),
             rng.random(dtype=np.float32)) for _ in range(rows)]


@pytest.mark.parametrize("rows,vocabulary,layout", [
    (3, 1, {}), (9, 2, {}), (20, 5, {"stride": 7}), (40, 300, {"offset": 4}), (64, 1024, {}), (33, 4097, {"offset": 12}),
    (24, 5000, {"stride": 5003}), (17, 32000, {}), (6, 50257, {"offset": 8}), (12, 128256, {}), (1, 151936, {}), (70, 20001, {}),
    (5, 262144, {"stride": 262147, "offset": 4})])
@pytest.mark.parametrize("spread", [0.5, 2.5, 12.0])
def test_sample(ctx, dev, rows, vocabulary, layout, spread):
    rng = np.random.default_rng(rows + vocabulary)
    logits = (rng.standard_normal((rows, vocabulary)) * spread).astype(np.float32)
    logits[:, rng.integers(0, vocabulary, 30)] += 6 * rng.random((rows, 30), np.float32)
    _check_sample(ctx, dev, logits, _settings(rng, rows), layout)


@pytest.mark.parametrize("vocabulary", [300, 40001, 262144])
def test_sample_among_equals(ctx, dev, vocabulary):
    """Logits of a few values, of one, and of one but for the last: of equals the lowest index is first."""
    rng = np.random.default_rng(vocabulary)
    logits = rng.integers(-3, 4, (12, vocabulary)).astype(np.float32)
    logits[3:6] = 1.5
    logits[5, -1] = 1.75
    logits[6] = np.where(np.arange(vocabulary) % 2, np.float32(0.0), np.float32(-0.0))
    logits[7] = -np.inf
    logits[7, ::7] = 2.0
    logits[8] = np.round(rng.standard_normal(vocabulary) * 8) / 8
    settings = _settings(rng, 12)
    settings[3] = (1.0, 0, 0.5, 0.0, np.float32(0.7))
    settings[4] = (1.0, vocabulary // 2, 1.0, 0.0, np.float32(0.99999994))
    settings[5] = (0.5, 0, 1.0, 0.0, np.float32(0.5))
    settings[6] = (1.0, 100, 0.9, 0.5, np.float32(0.33))
    settings[7] = (2.0, 0, 0.9, 0.0, np.float32(0.6))
    _check_sample(ctx, dev, logits, settings)


@pytest.mark.parametrize("vocabulary", [5, 5000, 151936])
def test_sample_rows_with_nothing_or_not_finite(ctx, dev, vocabulary):
    rng = np.random.default_rng(1)
    logits = rng.standard_normal((9, vocabulary)).astype(np.float32)
    logits[0] = -np.inf
    logits[1] = np.nan
    logits[2, 1:] = -np.inf
    logits[3, 2], logits[3, 4] = np.inf, np.inf
    logits[4, 0], logits[4, 3] = np.nan, 9.0
    logits[5] = np.where(np.arange(vocabulary) % 3 == 1, logits[5], -np.inf)
    logits[6] *= np.float32(1e37)
    logits[7] = np.float32(3.4e38) * np.sign(logits[7])
    logits[8] *= np.float32(1e-42)
    for settings in ((1.0, 0, 1.0, 0.0), (0.7, 3, 0.9, 0.01), (0.0, 0, 1.0, 0.0)):
        got = _check_sample(ctx, dev, logits, [(*settings, u) for u in rng.random(9, np.float32)])
        assert got[:3].tolist() == [-1, -1, 0]


@pytest.mark.parametrize("vocabulary", [1, 2, 7, 5000, 151936])
@pytest.mark.parametrize("settings", [(1.0, 0, 1.0, 0.0), (0.7, 3, 1.0, 0.0), (2.0, 0, 0.6, 0.0), (1.0, 0, 1.0, 0.3), (1e-3, 2, 0.9, 1.0)])
def test_sample_rows_of_infinities_alone(ctx, dev, vocabulary, settings):
    """A token forced by +inf among -inf, several of them, and nothing else: those of +inf weigh 2^40, the rest nothing."""
    rng = np.random.default_rng(vocabulary)
    logits = np.full((6, vocabulary), -np.inf, np.float32)
    logits[0] = np.inf
    logits[1, -1] = np.inf
    logits[2, vocabulary // 2] = np.inf
    logits[3, ::3] = np.inf
    logits[4] = np.where(np.arange(vocabulary) % 2, np.float32(np.nan), np.float32(np.inf))
    logits[5, vocabulary // 3:] = np.inf
    for u in (0.0, 0.5, 0.99999994):
        got = _check_sample(ctx, dev, logits, [(*settings, u)] * 6, {"stride": vocabulary + 3, "offset": 4})
        assert got[1] == vocabulary - 1 and got[2] == vocabulary // 2
    # each row's own setting, and rows with finite logits beside them
    logits = np.concatenate([logits, rng.standard_normal((3, vocabulary)).astype(np.float32)])
    _check_sample(ctx, dev, logits, _settings(rng, 9))


@pytest.mark.parametrize("vocabulary", [40, 50001])
def test_sample_settings_at_their_ends(ctx, dev, vocabulary):
    rng = np.random.default_rng(2)
    nan = float("nan")
    ends = [(1.0, 0, 0.0, 0.0), (1.0, 0, -3.0, 0.0), (1.0, 0, nan, 0.0), (1.0, 0, 2.0, nan), (1.0, 0, 1.0, 1.0), (1.0, 0, 1.0, 7.0),
            (1.0, 0, 1.0, -1.0), (nan, 0, 1.0, 0.0), (9e-7, 0, 1.0, 0.0), (1e-6, 0, 1.0, 0.0), (1e30, 0, 1.0, 0.0),
            (1.0, vocabulary, 1.0, 0.0), (1.0, vocabulary - 1, 1.0, 0.0), (1.0, vocabulary + 1, 1.0, 0.0), (1.0, 2, 0.9999999, 0.0),
            (1.0, -(1 << 31), 1.0, 0.0), (1.0, (1 << 31) - 1, 1e-9, 0.0), (float("inf"), 0, 0.25, 0.0), (1.0, 2, 1.0, 0.0),
            (-2.0, 0, 1.0, 0.0)]
    for u in (0.0, 0.5, 0.99999994, 1.0, 1.5, -1.0, nan):
        _check_sample(ctx, dev, rng.standard_normal((len(ends), vocabulary)).astype(np.float32), [(*e, u) for e in ends])


@pytest.mark.parametrize("temperature", [0.3, 1.0, 5.0, 1e4, float("inf")])
def test_sample_where_many_tokens_are_alike(ctx, dev, temperature):
    """Draws from where a row's tokens lie closest, one of them past what is kept."""
    rng = np.random.default_rng(23)
    logits = (rng.standard_normal((9, 262144)) * np.array([1, 1, 1, 0.01, 1e-6, 1e-30, 3, 1, 1])[:, None]).astype(np.float32)
    logits[7] = np.round(logits[7])  # many equal ones
    logits[8, 1000:] = -np.inf
    settings = [(temperature, 0, 1.0, 0.0, u) for u in (0.02, 0.5, 0.98, 0.5, 0.3, 0.7, 0.9)]
    settings += [(temperature, 100000, 0.9, 1e-7, 0.6), (temperature, 900, 0.5, 0.5, 0.9)]
    _check_sample(ctx, dev, logits, settings)


@pytest.mark.parametrize("temperature", [1e12, 1e15, 3e16, 1e18, 3e38, float("inf")])
@pytest.mark.parametrize("vocabulary", [40, 1000, 50001])
def test_sample_among_weights_that_f64_does_not_tell_apart(ctx, dev, temperature, vocabulary, monkeypatch):
    """Temperatures so far above the logits that the exponential of many, or of all, is one: min_p keeps them all. Here the
    last bit decides what is kept, so the exponential is the correctly rounded one, 1 + expm1 where it is within 2^-26 of 1
    (numpy's own is 1 - 2^-53 at -5e-17, and 1 - 2^-52 at -1.6e-16, where the nearest are 1 and 1 - 2^-53)."""
    from tests.support import requests_ref as ref

    class Rounded:
        def __getattr__(self, name):
            return getattr(np, name)

        @staticmethod
        def exp(x):
            return 1 + np.expm1(x)

    monkeypatch.setattr(ref, "np", Rounded())
    rng = np.random.default_rng(vocabulary)
    logits = (rng.standard_normal((10, vocabulary)) * 2).astype(np.float32)
    logits[2] *= np.float32(1e-20)
    settings = [(temperature, 0, 1.0, 1.0), (temperature, vocabulary // 2, 1.0, 1.0), (temperature, 0, 1.0, 1.0),
                (temperature, 0, 0.7, 1.0), (temperature, 0, 1.0, 0.9999999)]
    _check_sample(ctx, dev, logits, [(*s, u) for u in (0.3, 0.99999994) for s in settings])


def test_sample_logits_as_far_apart_as_f32_has_them(ctx, dev):
    logits = np.array([[-3e38, 3e38, 0.0, 1e38, -1e38] * 40, [3.4e38, -3.4e38, 1.0, 2.0, -np.inf] * 40], np.float32)
    _check_sample(ctx, dev, logits, [(1e38, 0, 1.0, 0.0, 0.97), (2e38, 90, 1.0, 0.01, 0.999)])


def _whole_weight(logit, temperature):
    """2^40 exp(logit / temperature) of f32s, to 60 digits."""
    import decimal

    with decimal.localcontext() as c:
        c.prec = 60
        return (decimal.Decimal(float(logit)) / decimal.Decimal(float(temperature))).exp() * (1 << 40)


def _about_a_whole_number(rng, temperature, above):
    """A logit whose weight is 2 - 12 units of f64's last place above a whole number, or below one, and below 2^40 by less than half."""
    while True:
        logits = (-rng.random(4096) * 0.69 * temperature).astype(np.float32)
        weights = np.exp(logits.astype(np.longdouble) / np.longdouble(temperature)) * (1 << 40)
        parts = (weights % 1 if above else 1 - weights % 1) * 8192
        for logit in logits[(parts > 2) & (parts < 12)]:
            part = float(_whole_weight(logit, temperature) % 1) * 8192
            if 2 < (part if above else 8192 - part) < 12:
                return logit


@pytest.mark.parametrize("temperature", [1.0, 0.7, 3.3])
@pytest.mark.parametrize("vocabulary", [37, 30001])
def test_sample_weights_are_whole_numbers_of_the_exponential(ctx, dev, temperature, vocabulary):
    """Rows whose weights are 2^40 and others that together are 2^40 + 1, or 2^40: with top_p of a half the first token is
    not all that is kept, or is. Among them is one whose exponential lies 2 to 12 units of f64's last place from a whole
    number, so that one that is off by as much makes it the other; those of the rest lie far from one."""
    from charlotte_amd import harness as hx
    from charlotte_amd import serving as sv

    rng = np.random.default_rng(vocabulary)
    t = np.float32(temperature)
    rows, lines, want = 24, [], []
    for row in range(rows):
        above = row % 2 == 0  # what is too small by a unit falls below the whole number
        logits = [np.float32(0), _about_a_whole_number(rng, t, above)]
        left = (1 << 40) + (1 if above else 0) - int(_whole_weight(logits[1], t))
        while left:
            logit = np.float32(float(t) * np.log((left + 0.5) * 2.0 ** -40))
            while not (int(_whole_weight(logit, t)) <= left and 0.1 < _whole_weight(logit, t) % 1 < 0.9):
                logit = np.nextafter(logit, np.float32(-np.inf))
            logits.append(logit)
            left -= int(_whole_weight(logit, t))
        weights = [int(_whole_weight(x, t)) for x in logits]
        assert sum(weights) == (2 << 40) + (1 if above else 0)
        line = np.full(vocabulary, -np.inf if row % 3 else -1e4, np.float32)
        places = rng.permutation(vocabulary)[:len(logits)]
        line[places] = logits
        lines.append(line)
        order = sorted(range(len(logits)), key=lambda i: (-logits[i], places[i]))
        kept = order[:2] if above else order[:1]
        total, u = sum(weights[i] for i in kept), 0.99999994
        token = next(i for n, i in enumerate(kept) if sum(weights[j] for j in kept[:n + 1]) > total * int(u * 2.0 ** 31) >> 31)
        want.append((places[token], weights[token] / total))
    need = sv.sample_workspace_bytes(rows, vocabulary)
    work, _ = dev.room(need, np.uint8)
    (out, read), (chances, read_chances) = dev.room(rows, np.int32), dev.room(rows)
    sv.sample(ctx, sv.Sample(dev.put(np.array(lines)), out, rows, vocabulary, dev.put(np.full(rows, 0.99999994, np.float32)),
                             temperature, 0, 0.5, chances=chances, workspace=work, workspace_bytes=need))
    hx.sync()
    assert read().tolist() == [x for x, _ in want]
    assert np.abs(read_chances() - [c for _, c in want]).max() <= 2.0 ** -24


def test_samples_follow_the_weights(ctx, dev):
    """Every token's share of many draws over a grid of uniform numbers, to one draw."""
    from tests.support import requests_ref as ref

    logits = np.log(np.array([0.1, 0.4, 0.05, 0.3, 0.15], np.float32))
    n = 4000
    got = _check_sample(ctx, dev, np.tile(logits, (n, 1)), [(1.0, 0, 1.0, 0.0, np.float32((i + 0.5) / n)) for i in range(n)])
    assert np.abs(np.bincount(got, minlength=5) - n * np.exp(logits)).max() <= 1
    assert ref.sample(logits, 1.0, 2, 1.0, 0.0, 0.6)[0] == 3


# ---- a step as a whole ---------------------------------------------------------------


@pytest.mark.parametrize("format_,heads,kv_heads,dim", [("q8_0", 8, 2, 64), ("f16", 4, 1, 128)])
def test_a_captured_step_replays_as_requests_grow(ctx, dev, format_, heads, kv_heads, dim):
    """page_plan, the stream's norm, page_append, paged_attention and sample in one graph: each replay, with requests that
    grow, end and come, against the same calls made eagerly."""
    from charlotte_amd import harness as hx
    from charlotte_amd import serving as sv
    from tests.support import serving_ref as ref

    rng = np.random.default_rng(dim)
    requests, page_tokens, pages, stride, vocabulary = 6, 32, 60, 20, 3001
    rows, width = requests, heads * dim
    past_at, counts_at = hx.Buffer(4 * requests), hx.Buffer(4 * requests)
    queries, branch, logits, uniforms = (hx.Buffer(4 * n) for n in (rows * width, rows * width, rows * vocabulary, rows))
    keys, values = (hx.Buffer(4 * rows * kv_heads * dim) for _ in range(2))
    weight = dev.put(rng.standard_normal(width).astype(np.float32))

    class Side:
        def __init__(self):
            zero = np.zeros(requests, np.int64)
            table = np.full((requests, stride), NOWHERE, np.uint64)
            self.plan = _Plan(ctx, dev, zero, zero, zero, table, np.arange(pages), pages, rows, page_tokens, pages, in_place=True)
            c = self.plan.call
            c.past, c.counts = past_at.ptr, counts_at.ptr
            self.pool = _Pool(dev, format_, pages, page_tokens, kv_heads, dim).pool
            need = sv.paged_attention_workspace_bytes(ctx, self.pool, heads)
            work, _ = dev.room(max(need, sv.sample_workspace_bytes(rows, vocabulary)), np.uint8)
            stream, self.read_stream = dev.room(rows * width, byte=0)
            normed, self.read_normed = dev.room(rows * width, byte=0)
            self.mixed, self.read_mixed = dev.room(rows * width, byte=0)
            tokens, self.read_tokens = dev.room(rows, np.int32)
            self.norm = sv.ResidualNorm(width, stream, branch.ptr, stream, normed, weight)
            self.attend = sv.PagedAttention(self.pool, queries.ptr, self.mixed, heads, 0.1, requests, rows, past_at.ptr, c.granted,
                                            c.starts, c.table, stride, workspace=work, workspace_bytes=need)
            self.draw = sv.Sample(logits.ptr, tokens, rows, vocabulary, uniforms.ptr, 0.8, 40, 0.95, 0.01, workspace=work,
                                  workspace_bytes=sv.sample_workspace_bytes(rows, vocabulary))

        def run(self, stream):
            self.plan.run(stream)
            sv.residual_norm(ctx, self.norm, rows, stream=stream)
            self.pool.append(keys.ptr, values.ptr, self.plan.call.slots, rows, stream=stream)
            sv.paged_attention(ctx, self.attend, stream=stream)
            sv.sample(ctx, self.draw, stream=stream)

        def all(self):
            got = self.plan.results()
            return [*got.values(), self.read_stream(), self.read_normed(), self.read_mixed(), self.read_tokens()]

    eager, captured = Side(), Side()
    stream = hx.Stream()
    graph = hx.Graph(stream, lambda: captured.run(stream.handle), global_mode=True)
    past = np.zeros(requests, np.int64)
    held_k = [np.zeros((0, kv_heads, dim), np.float32)] * requests
    held_v = list(held_k)
    for replay in range(70):
        counts = np.array([1, replay % 2, 1, int(replay > 20), 1, int(replay % 5 != 4)])
        if replay in (33, 50):
            past[2], held_k[2], held_v[2] = 0, held_k[2][:0], held_v[2][:0]
        past_at.write(_words(past))
        counts_at.write(_words(counts))
        data = {b: rng.standard_normal(b.nbytes // 4).astype(np.float32) for b in (queries, branch, logits, keys, values)}
        for b, x in data.items():
            b.write(x)
        uniforms.write(rng.random(rows, np.float32))
        graph.launch()
        stream.sync()
        eager.run(None)
        hx.sync()
        for a, b in zip(captured.all(), eager.all()):
            assert np.array_equal(a.view(np.uint32), b.view(np.uint32)), replay
        k, v = (data[b].reshape(rows, kv_heads, dim) for b in (keys, values))
        starts = np.concatenate([[0], np.cumsum(counts)])
        for r in range(requests):
            n = starts[r]
            held_k[r] = np.concatenate([held_k[r], k[n:n + counts[r]]])
            held_v[r] = np.concatenate([held_v[r], v[n:n + counts[r]]])
            if counts[r] and replay % 9 == 0:
                got = eager.read_mixed().reshape(rows, heads, dim)[n]
                want, w, size = ref.attention(data[queries].reshape(rows, heads, dim)[n:n + 1], ref.stored(held_k[r], format_),
                                              ref.stored(held_v[r], format_), int(past[r]), 0.1)
                assert (np.abs(got - want) <= ref.attention_bound(w, size, 100 + 32 * 256, dim)).all()
        past = past + counts
    graph.destroy()
    stream.destroy()
    for b in (past_at, counts_at, queries, branch, logits, uniforms, keys, values):
        b.free()
    for side in (eager, captured):
        side.pool.free()


def test_steps_on_two_streams_at_once(ctx, dev):
    """Two pools, each with a workspace and a stream of its own, and the same calls one after the other; then two graphs that
    share a workspace on one stream."""
    from charlotte_amd import harness as hx
    from charlotte_amd import serving as sv

    rng = np.random.default_rng(12)
    heads, kv_heads, dim, vocabulary = 8, 2, 64, 20001
    past, counts = [700, 0, 31, 4000], [1, 120, 1, 2]
    starts, rows = np.concatenate([[0], np.cumsum(counts)]), sum(counts)
    held = [-(-(p + c) // 64) for p, c in zip(past, counts)]
    stride = max(held)
    uniforms = dev.put(rng.random(rows, np.float32))

    class Side:
        def __init__(self):
            pages = sum(held) + 1
            order = rng.permutation(pages).tolist()
            table = np.full((4, stride), NOWHERE, np.uint64)
            for r, n in enumerate(held):
                table[r, :n] = [order.pop() for _ in range(n)]
            self.pool = _Pool(dev, "q8_0", pages, 64, kv_heads, dim)
            slots = [int(table[r, t // 64]) * 64 + t % 64 for r in range(4) for t in range(past[r] + counts[r])]
            k, v = (rng.standard_normal((len(slots), kv_heads * dim)).astype(np.float32) for _ in range(2))
            self.pool.write(k, v, slots)
            q, logits = (dev.put(rng.standard_normal((rows, n)).astype(np.float32)) for n in (heads * dim, vocabulary))
            self.need = max(sv.paged_attention_workspace_bytes(ctx, self.pool.pool, heads, 120),
                            sv.sample_workspace_bytes(rows, vocabulary))
            work, _ = dev.room(self.need, np.uint8)
            (out, self.read_out), (tokens, self.read_tokens) = dev.room(rows * heads * dim), dev.room(rows, np.int32)
            self.attend = sv.PagedAttention(self.pool.pool, q, out, heads, 0.1, 4, rows, dev.put(_words(past)),
                                            dev.put(_words(counts)), dev.put(_words(starts)), dev.put(_words(table)), stride, most=120,
                                            workspace=work, workspace_bytes=self.need)
            self.draw = sv.Sample(logits, tokens, rows, vocabulary, uniforms, 0.9, 0, 0.9, workspace=work, workspace_bytes=self.need)

        def run(self, stream):
            sv.paged_attention(ctx, self.attend, stream=stream)
            sv.sample(ctx, self.draw, stream=stream)

        def all(self):
            return [self.read_out().view(np.uint32), self.read_tokens()]

    sides, streams, want = [Side(), Side()], [hx.Stream(), hx.Stream()], []
    for side in sides:
        side.run(None)
        hx.sync()
        want.append(side.all())
    for _ in range(10):
        for side, stream in zip(sides, streams):
            side.run(stream.handle)
        for stream in streams:
            stream.sync()
        for side, w in zip(sides, want):
            assert all(np.array_equal(a, b) for a, b in zip(side.all(), w))
    for call in (sides[1].attend, sides[1].draw):
        call.workspace = sides[0].attend.workspace
    graphs = [hx.Graph(streams[0], lambda: side.run(streams[0].handle), global_mode=True) for side in sides]
    for turn in range(6):
        for graph in graphs[::1 if turn % 2 else -1]:
            graph.launch()
        streams[0].sync()
        for side, w in zip(sides, want):
            assert all(np.array_equal(a, b) for a, b in zip(side.all(), w)), turn
    for x in (*graphs, *streams):
        x.destroy()
    for side in sides:
        side.pool.pool.free()


# ---- refusals -------------------------------------------------------------------------


def _refused(call, status):
    from charlotte_amd import matmul as mm

    with pytest.raises(mm.MatmulError) as e:
        call()
    assert e.value.status == status


def test_pools_refuse(ctx, dev):
    from charlotte_amd import matmul as mm
    from charlotte_amd import serving as sv

    bad = mm.Status.INVALID_ARGUMENT
    x, _ = dev.room(1 << 16, np.uint8)
    good = (mm.TensorType.Q8_0, 4, 32, 1, 64)
    _refused(lambda: sv.PagePool(ctx, mm.TensorType.F32, *good[1:]), mm.Status.UNSUPPORTED_TYPE)
    for i, v in ((1, 0), (2, 0), (2, 33), (2, 16), (2, 4096), (1, 1 << 26), (3, 0), (3, 65536), (4, 0), (4, 80), (4, 288)):
        shape = [*good[:i], v, *good[i + 1:]]
        _refused(lambda: sv.PagePool(ctx, *shape), bad)
    _refused(lambda: sv.PagePool(ctx, *good, device=x + 8, nbytes=1 << 16), bad)
    _refused(lambda: sv.PagePool(ctx, *good, device=x, nbytes=100), bad)
    pool = sv.PagePool(ctx, *good)
    for args, kw in (((0, x, x, 1), {}), ((x, 0, x, 1), {}), ((x, x, 0, 1), {}), ((x, x, x, 0), {}), ((x + 4, x, x, 1), {}),
                     ((x, x + 8, x, 1), {}), ((x, x, x + 2, 1), {}), ((x, x, x, 1), {"key_stride": 60}),
                     ((x, x, x, 1), {"value_stride": 66}), ((x, x, x, 1 << 31), {})):
        _refused(lambda: pool.append(*args, **kw), bad)
        _refused(lambda: pool.read(*args, **kw), bad)
    other = mm.Context(0)
    pool.ctx = other
    _refused(lambda: pool.append(x, x, x, 1), bad)
    pool.ctx = ctx
    other.close()
    pool.free()
    _refused(lambda: pool.append(x, x, x, 1), bad)


def test_page_plan_refuses(ctx, dev):
    from charlotte_amd import matmul as mm
    from charlotte_amd import serving as sv

    x, _ = dev.room(1 << 12, np.uint8, byte=0)
    good = {"requests": 1, "rows": 1, "pages": 4, "page_tokens": 32, "table_stride": 2,
            **{n: x + 64 * i for i, n in enumerate(("past", "counts", "table", "held", "held_after", "free_pages", "free_count",
                                                    "free_count_after", "starts", "granted", "slots"))}}
    sv.page_plan(ctx, sv.PagePlan(**good))
    for name, value in (("requests", 0), ("requests", 65537), ("rows", 0), ("rows", 1 << 31), ("pages", 0), ("page_tokens", 0),
                        ("page_tokens", 48), ("page_tokens", 4096), ("pages", 1 << 27), ("table_stride", 0), ("table_stride", 1 << 26),
                        ("positions", 2), *((n, 0) for n in good if n not in ("requests", "rows", "pages", "page_tokens", "table_stride")),
                        ("past", x + 2), ("slots", x + 1)):
        _refused(lambda: sv.page_plan(ctx, sv.PagePlan(**{**good, name: value})), mm.Status.INVALID_ARGUMENT)


def test_paged_attention_refuses(ctx, dev):
    from charlotte_amd import matmul as mm
    from charlotte_amd import serving as sv

    bad = mm.Status.INVALID_ARGUMENT
    pool = sv.PagePool(ctx, mm.TensorType.Q8_0, 4, 32, 2, 64)
    need = sv.paged_attention_workspace_bytes(ctx, pool, 4, 1)
    assert need and not sv.paged_attention_workspace_bytes(ctx, pool, 3, 1) and not sv.paged_attention_workspace_bytes(ctx, pool, 0, 1)
    assert sv.paged_attention_workspace_bytes(ctx, pool, 4, 9) == 2 * need  # 18 rows a request
    x, _ = dev.room(1 << 13, np.uint8, byte=0)
    w, _ = dev.room(need, np.uint8)
    good = {"pool": pool, "queries": x, "output": x + 2048, "query_heads": 4, "scale": 0.1, "requests": 1, "rows": 1, "past": x + 4096,
            "counts": x + 4160, "starts": x + 4224, "table": x + 4288, "table_stride": 4, "workspace": w, "workspace_bytes": need}
    sv.paged_attention(ctx, sv.PagedAttention(**good))
    for name, value in (("queries", 0), ("queries", x + 4), ("output", 0), ("output", x + 8), ("query_heads", 0), ("query_heads", 3),
                        ("scale", float("nan")), ("requests", 0), ("requests", 65537), ("rows", 0), ("rows", (1 << 20) + 1),
                        ("past", 0), ("counts", 0), ("starts", 0), ("table", 0), ("table", x + 2), ("table_stride", 0),
                        ("table_stride", 1 << 26), ("query_stride", 128), ("query_stride", 258), ("output_stride", 100),
                        ("workspace", 0), ("workspace", w + 4), ("workspace_bytes", need - 1), ("most", 9)):
        _refused(lambda: sv.paged_attention(ctx, sv.PagedAttention(**{**good, name: value})), bad)
    call = sv.PagedAttention(**good)
    pool.free()
    _refused(lambda: sv.paged_attention(ctx, call), bad)


def test_residual_norm_and_sample_refuse(ctx, dev):
    from charlotte_amd import matmul as mm
    from charlotte_amd import serving as sv

    bad = mm.Status.INVALID_ARGUMENT
    x, _ = dev.room(1 << 14, np.uint8, byte=0)
    good = {"width": 64, "residual": x, "branch": x + 256, "residual_out": x + 512, "normed": x + 768, "weight": x + 1024}
    sv.residual_norm(ctx, sv.ResidualNorm(**good), 1)
    for change in ({"width": 0}, {"width": 32769}, {"residual": 0}, {"residual": x + 2}, {"weight": 0}, {"weight": x + 1},
                   {"branch": x + 1}, {"branch": 0, "gate": x}, {"branch": 0, "branch_weight": x}, {"residual_out": 0, "normed": 0},
                   {"epsilon": -1.0}, {"epsilon": float("inf")}, {"residual_scale": float("nan")}, {"branch_scale": float("inf")},
                   {"residual_stride": 63}, {"branch_stride": 1}, {"gate": x, "gate_stride": 7}, {"residual_out_stride": 5},
                   {"normed_stride": 5}, {"residual_out": x, "residual_out_stride": 80}, {"normed": x + 512},
                   {"normed": x + 256, "normed_stride": 72}, {"gate": x + 2048, "normed": x + 2048}, {"normed": x + 1024},
                   {"branch_weight": x + 512}):
        _refused(lambda: sv.residual_norm(ctx, sv.ResidualNorm(**{**good, **change}), 1), bad)
    for rows in (0, 0xFFFFFFFF):
        _refused(lambda: sv.residual_norm(ctx, sv.ResidualNorm(**good), rows), bad)

    need = sv.sample_workspace_bytes(2, 100)
    good = {"logits": x, "tokens": x + 4096, "rows": 2, "vocabulary": 100, "uniforms": x + 8192, "workspace": x + 8448,
            "workspace_bytes": need}
    w, _ = dev.room(need, np.uint8)
    good["workspace"] = w
    sv.sample(ctx, sv.Sample(**good))
    for change in ({"rows": 0}, {"rows": 1 << 23}, {"vocabulary": 0}, {"vocabulary": (1 << 18) + 1}, {"logits": 0}, {"logits": x + 2},
                   {"tokens": 0}, {"uniforms": 0}, {"temperature": -1.0}, {"temperature": float("nan")}, {"temperatures": x + 1},
                   {"top_ks": x + 2}, {"top_ps": x + 3}, {"min_ps": x + 1}, {"chances": x + 2}, {"logit_stride": 99},
                   {"workspace": 0}, {"workspace": w + 4}, {"workspace_bytes": need - 1}):
        _refused(lambda: sv.sample(ctx, sv.Sample(**{**good, **change})), bad)
