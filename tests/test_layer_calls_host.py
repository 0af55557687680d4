"""Calls of the layer's raw entry points that must be refused on the host,
before anything reaches a GPU (so they run on CPU tensors)."""

import numpy as np
import pytest
import torch

from tlora_b200 import ops

BF = torch.bfloat16


def state(rows=40, d_in=64, d_out=48, dt=BF, ranks=(8, 16), scaling=(0.5, 0.75)):
    table = ops.AdapterTable.build(list(range(len(ranks))), list(ranks))
    ids = torch.arange(len(ranks)).repeat_interleave(-(-rows // len(ranks)))[:rows]
    plan = ops.route(ids, table, torch.device("cpu"))
    return ops.LayerState(table, np.array(scaling, np.float32), plan, torch.zeros(table.r_pack, d_in, dtype=dt),
                          torch.zeros(d_out, table.r_pack, dtype=dt))


def backward(st, dy, xs="as it is", z=None, rows8=None, rows=40, d_in=64, dt=BF):
    if isinstance(xs, str):
        xs = torch.zeros(rows, d_in, dtype=dt)
    z = torch.zeros(1 << 20, dtype=torch.uint8) if z is None else z
    return ops.backward_raw(dy, xs, torch.zeros(48, 64, dtype=dt), z, st, True, True, True, rows8)


@pytest.mark.parametrize("shape", [(40, 47), (40, 49), (39, 48), (41, 48), (40 * 48,), (1, 40, 48)])
def test_upstream_gradient_of_another_shape(shape):
    with pytest.raises(ValueError, match="dy"):
        backward(state(), torch.zeros(shape, dtype=BF))


@pytest.mark.parametrize("dt", [torch.float32, torch.float16, torch.float64])
def test_upstream_gradient_of_another_type(dt):
    with pytest.raises(RuntimeError, match="dy"):
        backward(state(), torch.zeros(40, 48, dtype=dt))


def test_saved_tensors_of_another_call():
    dy = torch.zeros(40, 48, dtype=BF)
    with pytest.raises(ValueError, match="saved input"):
        backward(state(), dy, torch.zeros(39, 64, dtype=BF))
    with pytest.raises(ValueError, match="saved input"):
        backward(state(), dy, torch.zeros(40, 64))
    with pytest.raises(ValueError, match="saved input"):
        backward(state(), dy, None, rows8=ops.Int8Rows(torch.zeros(39, 64, dtype=torch.int8), torch.ones(39), 64))
    with pytest.raises(ValueError, match="saved input"):
        backward(state(), dy, None, rows8=ops.Int8Rows(torch.zeros(40, 64, dtype=torch.int8), torch.ones(40), 63))
    with pytest.raises(ValueError, match="saved intermediate"):
        backward(state(), dy, z=torch.zeros(16, dtype=torch.uint8))
