"""Rows read once by several workgroups (charlotte_amd.serving.probabilities): the
bits are the same whether a workgroup meets the others' sums or finds them itself."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    from charlotte_amd import matmul as mm

    c = mm.Context(0)
    yield c
    c.close()


@pytest.mark.parametrize("rows,vocabulary,layout", [
    (513, 32769, {"stride": 32773, "offset": 4, "output_offset": 8}), (300, 60001, {"offset": 12}), (150, 131072, {}),
    (60, 262147, {"offset": 4}), (6, 1048573, {"output_offset": 4})])
@pytest.mark.parametrize("temperature", [1.0, 0.3, 0.0])
def test_a_workgroup_that_does_not_wait(ctx, rows, vocabulary, layout, temperature):
    from charlotte_amd import harness as hx
    from charlotte_amd import matmul as mm
    from charlotte_amd import serving as sv
    from tests.support.serving_ref import Device

    rng = np.random.default_rng(vocabulary)
    x = rng.standard_normal((rows, vocabulary), np.float32) * np.float32(3)
    x[0, 5:-7], x[1] = -np.inf, -np.inf
    x[2, vocabulary - 3], x[3, 17], x[4, 30000] = np.nan, np.inf, -np.nan
    x[5] = rng.integers(-5, 6, vocabulary)
    stride, offset, output_offset = (layout.get(n, 0) for n in ("stride", "offset", "output_offset"))
    wide = np.zeros((rows, stride or vocabulary), np.float32)
    wide[:, :vocabulary] = x
    need = sv.probabilities_workspace_bytes(rows, vocabulary)
    print("patience", rows, vocabulary, temperature, layout, flush=True)
    with Device(ctx) as dev:
        got = []
        try:
            logits, work = dev.put(wide, offset), dev.room(need, np.uint8)[0]
            for looks in (mm.PATIENCE, 0, 1):
                ctx.set_patience(looks)
                to, read = dev.room(rows * vocabulary, offset=output_offset)
                sv.probabilities(ctx, sv.Probabilities(logits, to, rows, vocabulary, temperature, logit_stride=stride,
                                                       workspace=work, workspace_bytes=need))
                hx.sync()
                got.append(read().view(np.uint32))
        finally:
            ctx.set_patience(mm.PATIENCE)
    assert np.array_equal(got[0], got[1]) and np.array_equal(got[0], got[2])


def test_patience_refuses(ctx):
    from charlotte_amd import matmul as mm

    with pytest.raises(mm.MatmulError) as e:
        ctx.set_patience(mm.PATIENCE + 1)
    assert e.value.status == mm.Status.INVALID_ARGUMENT
