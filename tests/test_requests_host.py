"""The operators of a step over several requests on the CPU: what they compute
without a device, and the restatements their device tests compare with, against
small known answers."""

import numpy as np

from charlotte_amd import matmul as mm
from charlotte_amd import serving as sv
from tests.support import requests_ref as ref


def test_pool_bytes():
    # a page is whole 32-token tiles of every head, as a cache's
    assert sv.page_pool_bytes(mm.TensorType.Q8_0, 7, 64, 8, 128) == sv.cache_bytes(mm.TensorType.Q8_0, 7, 8, 128, 64)
    assert sv.page_pool_bytes(mm.TensorType.Q4_0, 3, 32, 1, 32) == 3 * (2 * 512 + 128)
    for bad in ((mm.TensorType.F32, 1, 32, 1, 64), (mm.TensorType.Q8_0, 0, 32, 1, 64), (mm.TensorType.Q8_0, 1, 16, 1, 64),
                (mm.TensorType.Q8_0, 1, 40, 1, 64), (mm.TensorType.Q8_0, 1, 4096, 1, 64), (mm.TensorType.Q8_0, 1, 32, 0, 64),
                (mm.TensorType.Q8_0, 1, 32, 1, 80), (mm.TensorType.Q8_0, 1 << 26, 32, 1, 64)):
        assert sv.page_pool_bytes(*bad) == 0


def test_sample_workspace():
    assert sv.sample_workspace_bytes(1, 1) > 0
    for rows, vocabulary in ((0, 5), (5, 0), (1, (1 << 18) + 1), (1 << 31, 5)):
        assert sv.sample_workspace_bytes(rows, vocabulary) == 0


def test_calls_without_a_context_are_refused():
    for name, args in (("page_plan", (None, None, None)), ("paged_attention", (None, None, None)),
                       ("residual_norm", (None, None, 1, None)), ("sample", (None, None, None))):
        assert getattr(mm.lib, "charlotte_hip_matmul_" + name)(*args) == mm.Status.INVALID_ARGUMENT
    assert mm.lib.charlotte_hip_matmul_page_pool_free(None) == mm.Status.OK
    assert mm.lib.charlotte_hip_matmul_paged_attention_workspace_bytes(None, None, 4, 1) == 0


def test_page_plan_reference():
    # request 0 grows into a second page, 1 has ended, 2 is new and takes what 1 gave back
    got = ref.page_plan([32, 0, 0], [1, 0, 2], [1, 2, 0], [[4, 9], [5, 6], [9, 9]], [7, 0, 0, 0], 1, 4, 32, 8)
    assert got["table"] == [[4, 6], [5, 6], [5, 9]] and got["free"][:3] == [7, 5, 6] and got["free_count"] == 1
    assert got["held"] == [2, 0, 1] and got["granted"] == [1, 0, 2] and got["starts"] == [0, 1, 1, 3]
    assert got["slots"] == [6 * 32, 5 * 32, 5 * 32 + 1, ref.NONE] and got["positions"] == [32, 0, 1, 0]


def test_residual_norm_reference():
    r, n, _, _ = ref.residual_norm([[3.0, 4.0]], [[1.0, -1.0]], None, [2.0, 1.0], np.array([1.0, 2.0]), 2.0, 1.0, 0.0)
    assert r.tolist() == [[8.0, 7.0]]
    assert np.allclose(n, np.array([[8.0, 14.0]]) / np.sqrt(113 / 2))


def test_sample_reference():
    logits = np.log(np.array([0.1, 0.4, 0.1, 0.3, 0.1], np.float32))  # in order: 1, 3, then 0, 2, 4
    assert [ref.sample(logits, 1.0, 0, 1.0, 0.0, u)[0] for u in (0.0, 0.39, 0.41, 0.69, 0.75, 0.85, 0.99)] == [1, 1, 3, 3, 0, 2, 4]
    assert [ref.sample(logits, 1.0, 3, 1.0, 0.0, u)[0] for u in (0.45, 0.55, 0.9)] == [1, 3, 0]
    assert ref.sample(logits, 1.0, 0, 0.3, 0.0, 0.99)[0] == 1
    assert ref.sample(logits, 1.0, 0, 0.5, 0.0, 0.99)[0] == 3
    assert ref.sample(logits, 1.0, 0, 1.0, 0.5, 0.99)[0] == 3
    assert ref.sample(logits, 0.0, 0, 1.0, 0.0, 0.99)[0] == 1
    assert ref.sample(np.full(4, -np.inf), 1.0, 0, 1.0, 0.0, 0.5)[0] == -1


class _Recorded:
    """A library that keeps copies of the descriptors it is called with, and a context of it."""

    handle = None

    def __init__(self):
        self.descs = []

    def __getattr__(self, name):
        def call(handle, desc, *rest):
            self.descs.append(type(desc._obj).from_buffer_copy(desc._obj))
            return 0
        return call

    def check(self, status):
        assert status == 0


def test_a_field_set_between_calls_reaches_the_next(monkeypatch):
    seen = _Recorded()
    monkeypatch.setattr(sv, "lib", seen)
    norm = sv.ResidualNorm(64, 16, normed=32, weight=48)
    sv.residual_norm(seen, norm, 1)
    norm.branch_scale = 0.5
    sv.residual_norm(seen, norm, 1)
    draw = sv.Sample(16, 32, 2, 100, 48)
    sv.sample(seen, draw)
    draw.top_k = 7
    sv.sample(seen, draw)
    plan = sv.PagePlan(1, 2, 3, 32, *(16 * i for i in range(12)))
    sv.page_plan(seen, plan)
    plan.rows = 9
    sv.page_plan(seen, plan)
    assert [d.branch_scale for d in seen.descs[:2]] == [1.0, 0.5]
    assert [d.top_k for d in seen.descs[2:4]] == [0, 7]
    assert [d.rows for d in seen.descs[4:]] == [2, 9]
