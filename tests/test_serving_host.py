"""charlotte_amd.serving on the CPU: what it computes without a device, and the
plain restatements its device tests compare with, against small known answers."""

import numpy as np
import pytest

from charlotte_amd import matmul as mm
from charlotte_amd import serving as sv
from tests.support import serving_ref as ref


def test_cache_bytes():
    # 32-token tiles; per block of 32 values and tile: codes of keys and of values, and their scales
    assert sv.cache_bytes(mm.TensorType.Q8_0, 1, 8, 128, 1024) == 32 * 8 * 4 * (2 * 1024 + 128)
    assert sv.cache_bytes(mm.TensorType.Q4_0, 2, 1, 32, 33) == 2 * 2 * (2 * 512 + 128)
    assert sv.cache_bytes(mm.TensorType.F16, 1, 1, 256, 1) == 8 * (2 * 2048 + 64)
    for bad in ((mm.TensorType.F32, 1, 1, 64, 8), (mm.TensorType.Q8_0, 0, 1, 64, 8), (mm.TensorType.Q8_0, 1, 1, 80, 8),
                (mm.TensorType.Q8_0, 1, 1, 288, 8), (mm.TensorType.Q8_0, 1, 1, 64, 0),
                (mm.TensorType.F16, 65535, 65535, 256, 0x7FFFFFFF)):  # past what 64 bits hold
        assert sv.cache_bytes(*bad) == 0


def test_workspaces():
    assert sv.probabilities_workspace_bytes(0, 5) == 0
    assert sv.verify_workspace_bytes(1, 1, (1 << 18) + 1) == 0
    assert sv.verify_workspace_bytes(2, 3, 2048) == 6 * 9 * 8 + 2 * 4  # segments of 256, at any alignment
    assert sv.verify_workspace_bytes(1, 1025, 2048) == 0


def test_rope_table():
    c, s = sv.rope_table(5, 8, base=100.0, factors=[1, 1, 2, 4])
    angle = 3 * 100.0 ** (-2 * 2 / 8) / 2
    assert c.shape == s.shape == (5, 4)
    assert c[3, 2] == np.float32(np.cos(angle)) and s[3, 2] == np.float32(np.sin(angle))


def test_calls_without_a_context_are_refused():
    for name, args in (("head_norm_rope", (None, None, 1, None)), ("attention", (None, None, 1, None)),
                       ("probabilities", (None, None, None)), ("verify", (None, None, 1, 1, None))):
        assert getattr(mm.lib, "charlotte_hip_matmul_" + name)(*args) == mm.Status.INVALID_ARGUMENT
    assert mm.lib.charlotte_hip_matmul_cache_free(None) == mm.Status.OK


def test_stored_blocks():
    x = np.zeros((1, 32), np.float32)
    x[0, 0], x[0, 1] = 127.0, -63.4
    assert ref.stored(x, "q8_0")[0, :2].tolist() == [127.0, -63.0]
    x[0, 0], x[0, 1] = -8.0, 7.6
    assert ref.stored(x, "q4_0")[0, :2].tolist() == [-8.0, 7.0]
    x[0, 0] = 65520.0
    assert np.isnan(ref.stored(x, "f16")).all()


def test_sees():
    assert ref.sees(2, 3).astype(int).tolist() == [[1, 1, 1, 0, 0], [1, 1, 1, 1, 0], [1, 1, 1, 1, 1]]
    assert ref.sees(2, 3, [-1, 0, 0]).astype(int).tolist() == [[1, 1, 1, 0, 0], [1, 1, 1, 1, 0], [1, 1, 1, 0, 1]]
    assert ref.sees(2, 3, [-1, -2, 1]).astype(int).tolist() == [[1, 1, 1, 0, 0], [0] * 5, [0] * 5]
    assert ref.sees(2, 3, [-1, 0, 0], window=2).astype(int).tolist() == [[0, 1, 1, 0, 0], [0, 0, 1, 1, 0], [0, 0, 1, 0, 1]]


@pytest.mark.parametrize("uniform,token", [(0.0, 1), (0.249, 1), (0.25, 3), (0.99999994, 3), (1.0, 3), (-1.0, 1)])
def test_drawn(uniform, token):
    assert ref.drawn(np.array([0, 0.25, 0, 0.75], np.float32), uniform) == token


def test_verify_reference():
    target = np.array([[0.5, 0.5, 0], [0, 0, 1], [1, 0, 0]], np.float32)
    draft = np.array([[0.5, 0.5, 0], [0.9, 0.1, 0]], np.float32)
    # token 1 is accepted (1 x 0.5 < 0.5 is not: 0.9 is), token 0 refused, and 2 all that is left
    assert ref.verify([7, 1, 0], target, [0, 0, 0], draft, [0, 0.9, 0.0]) == ([0, 1], [1, 2])
    assert ref.verify([7, 1, 0], target, [0, 0, 0], draft, [0, 1.0, 0.0]) == ([0], [0])
    assert ref.verify([7, 1, 1], target, [0.6, 0.1, 0], parents=[-1, 0, 0]) == ([0, 1], [1, 2])


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


class _CacheOf:
    def __init__(self, handle):
        self.handle = handle


def test_a_field_set_between_calls_reaches_the_next(monkeypatch):
    seen = _Recorded()
    monkeypatch.setattr(sv, "lib", seen)

    soft = sv.Probabilities(16, 32, 2, 100, temperature=1.0, workspace=48, workspace_bytes=64)
    sv.probabilities(seen, soft)
    kept = soft._desc
    sv.probabilities(seen, soft)
    assert soft._desc is kept  # built once while nothing changes
    soft.temperature, soft.workspace = 0.5, 4096
    sv.probabilities(seen, soft)
    assert [(d.temperature, d.workspace) for d in seen.descs] == [(1.0, 48), (1.0, 48), (0.5, 4096)]

    seen.descs.clear()
    cache = _CacheOf(16)
    attend = sv.Attention(cache, 16, 32, 4, 0.125, past=64)
    sv.attention(seen, attend, 1)
    attend.longest, attend.workspace_bytes = 300, 128
    sv.attention(seen, attend, 1)
    cache.handle = None  # freed
    sv.attention(seen, attend, 1)
    assert [(d.longest, d.workspace_bytes, d.cache) for d in seen.descs] == [(0, 0, 16), (300, 128, 16), (300, 128, None)]

    seen.descs.clear()
    check = sv.Verify(16, 32, 48, 100, 64, 80, 96)
    sv.verify(seen, check, 1, 2)
    check.draft, check.accepts = 112, 128
    sv.verify(seen, check, 1, 2)
    assert [(d.draft, d.accepts) for d in seen.descs] == [(None, None), (112, 128)]

    seen.descs.clear()
    q, k = sv.Heads(16, 32, 4), sv.Heads(48, 64, 2)
    turn = sv.HeadNormRope([q], 64)
    sv.head_norm_rope(seen, turn, 1)
    turn.epsilon = 0.5
    sv.head_norm_rope(seen, turn, 1)
    q.input = 80
    sv.head_norm_rope(seen, turn, 1)
    turn.parts.append(k)
    sv.head_norm_rope(seen, turn, 1)
    turn.parts[0] = k
    sv.head_norm_rope(seen, turn, 1)
    sv.head_norm_rope(seen, turn, 1)
    assert [(d.part_count, d.parts[0].input, d.epsilon) for d in seen.descs] == [
        (1, 16, np.float32(1e-6)), (1, 16, 0.5), (1, 80, 0.5), (2, 80, 0.5), (2, 48, 0.5), (2, 48, 0.5)]
