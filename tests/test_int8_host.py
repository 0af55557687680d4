"""8-bit operators, host side: argument checks, layout, module switches."""

import ctypes

import numpy as np
import pytest
import torch

import tlora_b200
from tlora_b200 import MultiLoRALinear, _lib, ops
from tlora_b200.multi_lora_linear import Int8Base, IndependentLoRALinear


def rows8(rows, cols):
    return ops.Int8Rows(torch.zeros(rows, ops.q8_ld(cols), dtype=torch.int8), torch.ones(rows), cols)


@pytest.mark.parametrize("cols", [1, 15, 16, 17, 1000, 4096])
def test_leading_dimension_matches_the_library(cols):
    assert ops.q8_ld(cols) == _lib.lib().mlora_q8_ld(cols)
    assert rows8(3, cols).shape == (3, cols)


def test_int8_rows_layout_is_checked():
    with pytest.raises(ValueError):
        ops.Int8Rows(torch.zeros(2, 17, dtype=torch.int8), torch.ones(2), 17)
    with pytest.raises(ValueError):
        ops.Int8Rows(torch.zeros(2, 32, dtype=torch.uint8), torch.ones(2), 17)
    with pytest.raises(ValueError):
        ops.Int8Rows(torch.zeros(2, 32, dtype=torch.int8), torch.ones(3), 17)
    with pytest.raises(ValueError):
        ops.Int8Rows(torch.zeros(2, 32, dtype=torch.int8), torch.ones(2, dtype=torch.float64), 17)
    with pytest.raises(ValueError):
        ops.Int8Rows(torch.zeros(2, 64, dtype=torch.int8)[:, ::2], torch.ones(2), 17)


def test_no_cpu_path():
    for call in (lambda: ops.quantize_rows(torch.ones(2, 16)), lambda: ops.dequantize_rows(rows8(2, 16)),
                 lambda: ops.int8_linear(torch.ones(2, 16), rows8(4, 16))):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
    with pytest.raises(RuntimeError, match="CUDA"):
        MultiLoRALinear(16, 16, {0: 4}).quantize_base()


def test_weight_must_be_int8_rows():
    with pytest.raises(TypeError):
        ops.int8_linear(torch.ones(2, 16), torch.ones(4, 16))


def test_save_input_is_checked():
    m = MultiLoRALinear(16, 16, {0: 4})
    assert m.save_input == "full"
    m.save_input = "int4"
    with pytest.raises(ValueError, match="save_input"):
        m(torch.ones(2, 16), torch.zeros(2, dtype=torch.int64))
    one = IndependentLoRALinear(16, 16, 4)
    one.save_input = "half"
    with pytest.raises(ValueError, match="save_input"):
        one(torch.ones(2, 16))


@pytest.mark.parametrize("cast", [torch.bfloat16, torch.float16, torch.float64])
def test_scales_stay_float32_under_casts(cast):
    b = Int8Base(ops.Int8Rows(torch.ones(4, 16, dtype=torch.int8), torch.tensor([0.1, 0.2, 0.3, 1e-30]), 16),
                 torch.zeros(4))
    b = b.to(cast)
    assert b.weight_scale.dtype == torch.float32 and b.bias.dtype == cast
    assert torch.equal(b.weight_scale, torch.tensor([0.1, 0.2, 0.3, 1e-30]))
    assert b.weight_q8.dtype == torch.int8 and not any(p.requires_grad for p in b.parameters())
    assert b.rows8.shape == (4, 16)


def test_state_dict_of_an_8bit_base_round_trips():
    a, b = MultiLoRALinear(17, 4, {0: 4}), MultiLoRALinear(17, 4, {0: 4})
    for m, fill in ((a, 3), (b, 0)):
        m.base = Int8Base(ops.Int8Rows(torch.full((4, 32), fill, dtype=torch.int8), torch.full((4,), 0.5 + fill), 17),
                          m.base.bias)
    keys = set(a.state_dict())
    assert {"base.weight_q8", "base.weight_scale", "base.bias", "adapters.0.A", "adapters.0.B"} == keys
    b.load_state_dict(a.state_dict())
    assert torch.equal(b.base.weight_q8, a.base.weight_q8) and torch.equal(b.base.weight_scale, a.base.weight_scale)
    # switching twice changes nothing
    assert b.quantize_base() is b and isinstance(b.base, Int8Base)


def test_an_8bit_base_is_not_sharded():
    from tlora_b200.overlap import ShardedLayer

    m = MultiLoRALinear(256, 64, {0: 4})
    m.base = Int8Base(rows8(64, 256), None)
    with pytest.raises(NotImplementedError, match="8 bits"):
        ShardedLayer(m, 0, 1)


# ---- the C entry points refuse before they launch: nothing here reaches a GPU

P = ctypes.c_void_p(4096)   # stands for a device address; never read on the host
ODD = ctypes.c_void_p(4100)


def problem(rows=4, d_in=64, d_out=32, dtype=_lib.BF16, max_ctas=0):
    return _lib.Problem(rows, d_in, d_out, dtype, _lib.IMPL_AUTO, max_ctas)


@pytest.mark.parametrize("args, status", [
    ((P, -1, 16, 16, _lib.BF16, None, P, P), _lib.ERR_INVALID_ARG),
    ((P, 4, 0, 16, _lib.BF16, None, P, P), _lib.ERR_INVALID_ARG),
    ((P, 4, 16, 15, _lib.BF16, None, P, P), _lib.ERR_INVALID_ARG),   # rows overlap
    ((P, 4, 16, 16, 7, None, P, P), _lib.ERR_UNSUPPORTED),
    ((P, 4, (1 << 30) + 1, 1 << 31, _lib.BF16, None, P, P), _lib.ERR_UNSUPPORTED),
    ((None, 4, 16, 16, _lib.BF16, None, P, P), _lib.ERR_INVALID_ARG),
    ((P, 4, 16, 16, _lib.BF16, None, None, P), _lib.ERR_INVALID_ARG),
    ((P, 4, 16, 16, _lib.BF16, None, ODD, P), _lib.ERR_UNSUPPORTED),  # 8-bit rows start on 16 bytes
    ((ctypes.c_void_p(4097), 4, 16, 16, _lib.BF16, None, P, P), _lib.ERR_UNSUPPORTED),
    ((None, 0, 16, 16, _lib.BF16, None, None, None), _lib.OK),        # no rows: nothing to do
])
def test_quantize_refusals(args, status):
    assert _lib.lib().mlora_q8_quantize(*args, None) == status


@pytest.mark.parametrize("args, status", [
    ((P, P, 4, 16, 9, P), _lib.ERR_UNSUPPORTED),
    ((None, P, 4, 16, _lib.F32, P), _lib.ERR_INVALID_ARG),
    ((ODD, P, 4, 16, _lib.F32, P), _lib.ERR_UNSUPPORTED),
    ((P, P, 4, 16, _lib.F32, ctypes.c_void_p(4098)), _lib.ERR_UNSUPPORTED),
    ((None, None, 0, 16, _lib.F32, None), _lib.OK),
])
def test_dequantize_refusals(args, status):
    assert _lib.lib().mlora_q8_dequantize(*args, None) == status


@pytest.mark.parametrize("prob, ops_, status", [
    (problem(d_in=_lib.Q8_MAX_K + 1), (P, 1 << 20, P, P, P, P, None, P), _lib.ERR_UNSUPPORTED),
    (problem(d_in=0), (P, 64, P, P, P, P, None, P), _lib.ERR_INVALID_ARG),
    (problem(dtype=5), (P, 64, P, P, P, P, None, P), _lib.ERR_UNSUPPORTED),
    (problem(max_ctas=-1), (P, 64, P, P, P, P, None, P), _lib.ERR_INVALID_ARG),
    (problem(), (P, 63, P, P, P, P, None, P), _lib.ERR_INVALID_ARG),
    (problem(), (P, 64, None, P, P, P, None, P), _lib.ERR_INVALID_ARG),
    (problem(), (P, 64, P, P, None, P, None, P), _lib.ERR_INVALID_ARG),
    (problem(), (P, 64, P, P, P, P, None, None), _lib.ERR_INVALID_ARG),
    (problem(), (P, 64, P, P, ODD, P, None, P), _lib.ERR_UNSUPPORTED),
    (problem(), (P, 64, P, ctypes.c_void_p(4098), P, P, None, P), _lib.ERR_UNSUPPORTED),
    (problem(rows=0), (None, 0, None, None, None, None, None, None), _lib.OK),
])
def test_linear_refusals(prob, ops_, status):
    assert _lib.lib().mlora_q8_linear(ctypes.byref(prob), *ops_, None) == status


@pytest.mark.parametrize("prob, ops_, status", [
    (problem(d_out=_lib.Q8_MAX_K + 1), (P, P, P, P, P, P), _lib.ERR_UNSUPPORTED),
    (problem(), (P, None, P, P, P, P), _lib.ERR_INVALID_ARG),
    (problem(), (P, P, P, P, None, P), _lib.ERR_INVALID_ARG),
    (problem(), (P, ODD, P, P, P, P), _lib.ERR_UNSUPPORTED),
    (problem(rows=0), (None,) * 6, _lib.OK),
])
def test_linear_dx_refusals(prob, ops_, status):
    assert _lib.lib().mlora_q8_linear_dx(ctypes.byref(prob), *ops_, None) == status


def test_layer_call_refusals():
    one = np.array([0, 4], np.int32)
    route = _lib.Routing(0, None, None, 0, None, None, None, 0, None)
    lib = _lib.lib()
    big = 1 << 30

    def fwd(q8, W=None, prob=None):
        return lib.mlora_forward_q8(ctypes.byref(prob or problem()), ctypes.byref(route), ctypes.byref(q8), P, W, None,
                                    None, None, P, None, P, big, None)

    a = 4096
    assert one.size == 2
    assert fwd(_lib.Q8(a, a, None, None, None, None)) == _lib.ERR_INVALID_ARG       # nowhere to put the rows of X
    assert fwd(_lib.Q8(a, None, a, a, None, None)) == _lib.ERR_INVALID_ARG          # no scales
    assert fwd(_lib.Q8(a, a, a, a, None, None), W=P) == _lib.ERR_INVALID_ARG        # two backbones
    assert fwd(_lib.Q8(None, None, a, None, None, None)) == _lib.ERR_INVALID_ARG
    assert fwd(_lib.Q8(a + 4, a, a, a, None, None)) == _lib.ERR_UNSUPPORTED
    assert fwd(_lib.Q8(a, a, a, a, None, None), prob=problem(d_in=_lib.Q8_MAX_K + 8)) == _lib.ERR_UNSUPPORTED
    assert lib.mlora_forward_q8(ctypes.byref(problem()), ctypes.byref(route), None, P, None, None, None, None, P, None,
                                P, big, None) == _lib.ERR_INVALID_ARG

    def bwd(q8, dX=P, dA=None, X=None, W=None):
        return lib.mlora_backward_q8(ctypes.byref(problem()), ctypes.byref(route), ctypes.byref(q8), P, X, W, None,
                                     None, None, dX, dA, None, P, big, None)

    assert bwd(_lib.Q8(a, a, None, None, None, None)) == _lib.ERR_INVALID_ARG       # no room for the rows of dY
    assert bwd(_lib.Q8(a, a, None, None, a, a), W=P) == _lib.ERR_INVALID_ARG
    assert bwd(_lib.Q8(a, a, a, None, a, a)) == _lib.ERR_INVALID_ARG
    assert bwd(_lib.Q8(a, a, None, None, a + 8, a)) == _lib.ERR_UNSUPPORTED


def test_public_names():
    for name in ("Int8Rows", "quantize_rows", "dequantize_rows", "int8_linear"):
        assert hasattr(tlora_b200.ops, name)
