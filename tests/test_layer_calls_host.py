"""Calls of the layer's raw entry points that must be refused on the host,
before anything reaches a GPU (so they run on CPU tensors)."""

import ctypes

import numpy as np
import pytest
import torch

from tlora_b200 import MultiLoRALinear, _lib, ops
from tlora_b200.multi_lora_linear import Int8Base

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


# ------------------------------------------------------------------ plans that change between calls

def call_of(st, rows=40):
    return ops._Call(rows, 64, 48, ops.mlora_dtype(BF), st)


def segments(call):
    r = call.route
    return [r.seg_start[i] for i in range(r.n_seg + 1)], [r.seg_adapter[i] for i in range(r.n_seg)]


def test_calls_follow_a_plan_whose_arrays_are_replaced():
    st = state()
    assert segments(call_of(st)) == ([0, 20, 40], [0, 1])
    st.plan.seg_start = np.array([0, 5, 40], np.int32)
    assert segments(call_of(st)) == ([0, 5, 40], [0, 1])
    st.plan.seg_adapter = np.array([1, -1], np.int32)
    assert segments(call_of(st)) == ([0, 5, 40], [1, -1])
    st.plan.perm = torch.arange(40, dtype=torch.int32)
    assert call_of(st).route.out_rows == st.plan.perm.data_ptr()
    st.plan.perm = None
    assert call_of(st).route.out_rows is None


def test_calls_follow_a_plan_edited_in_place():
    st = state(rows=600)
    st.plan.seg_start[:] = [0, 100, 600]   # the tiles of adapter 1: 0 to 2 instead of 1 to 2
    assert segments(call_of(st, 600)) == ([0, 100, 600], [0, 1])
    before = call_of(st, 600).zbytes
    st.plan.seg_start[:] = [0, 600, 600]   # one adapter, one chunk a tile
    after = call_of(st, 600)
    assert segments(after) == ([0, 600, 600], [0, 1])
    assert after.zbytes == 3 * 256 * 64 * 2 and before == 4 * 256 * 64 * 2
    st.plan.seg_start[:] = [0, 300, 600]
    assert call_of(st, 600).zbytes == 4 * 256 * 64 * 2


def test_calls_follow_a_replaced_plan():
    import dataclasses

    st = state()
    call_of(st)
    st.plan = dataclasses.replace(st.plan, seg_start=np.array([0, 7, 40], np.int32))
    assert segments(call_of(st)) == ([0, 7, 40], [0, 1])


def test_kept_descriptions_are_copies():
    st = state()
    kept = st.plan.seg_start
    call_of(st)
    kept[:] = [0, 9, 40]
    call_of(st)
    st.plan.seg_start = np.array([0, 20, 40], np.int32)  # as it was, in another array
    assert segments(call_of(st)) == ([0, 20, 40], [0, 1])
    st.scaling[1] = 3.0
    assert call_of(st).route.scaling[1] == 3.0
    st.scaling = np.array([0.5, 0.75], np.float32)
    assert call_of(st).route.scaling[1] == 0.75


def test_tables_follow_their_ranks():
    import dataclasses

    table = ops.AdapterTable.build([0, 1], [8, 16])
    first = table.layout()
    assert table.spans() == [(0, 8), (64, 16)] and table.pieces() == ([0, 8, 56, 16, 48], [1, 3])
    other = dataclasses.replace(table, rank=np.array([4, 20], np.int32))
    assert other.spans() == [(0, 4), (64, 20)] and other.pieces() == ([0, 4, 60, 20, 44], [1, 3])
    table.rank[0] = 2
    assert table.spans() == [(0, 2), (64, 16)] and table.pieces() == ([0, 2, 62, 16, 48], [1, 3])
    assert len({first, other.layout(), table.layout()}) == 3
    # packed in another order, with a gap before the first
    third = ops.AdapterTable([5, 7], np.array([8, 64], np.int32), np.array([128, 64], np.int32), 192)
    assert third.pieces() == ([64, 64, 0, 8, 56], [3, 1])


# ------------------------------------------------------------------ resident plans

def resident(st, rows=40, d_in=64, d_out=48):
    """The workspace that a call with this state finds, or None."""
    call = ops._Call(rows, d_in, d_out, ops.mlora_dtype(BF), st)
    ws, flags = ops._workspace(st, call, call.wbytes, torch.device("cpu"))
    return ws if flags & _lib.PLAN_RESIDENT else None


@pytest.fixture
def uploads(monkeypatch):
    """mlora_plan_upload without a GPU: what it was called for."""
    seen, call = [], _lib.call

    def fake(name, *args):
        if name != "mlora_plan_upload":
            return call(name, *args)
        seen.append(args)
    monkeypatch.setattr(_lib, "call", fake)
    monkeypatch.setattr(ops, "_stream", lambda device: 0)
    return seen


def make(st):
    return ops.make_resident(st, 40, 64, 48, BF, torch.device("cpu"))


def test_layers_of_one_shape_share_a_resident_plan(uploads):
    # scalings and ranks are part of the uploaded tables
    one = state(ranks=(64, 128))
    assert make(one) is make(one) and len(uploads) == 1
    for other in (state(ranks=(64, 128), scaling=(0.5, 1.0)), state(ranks=(128, 64)), state(ranks=(60, 128))):
        other.plan = one.plan
        assert other.table.r_pack == one.table.r_pack
        assert resident(other) is None
        ws = make(other)
        assert ws is not make(one) and resident(other) is ws
    assert len(uploads) == 4 and resident(one) is make(one)


def test_staged_calls_find_the_resident_plan(uploads):
    st = state()
    ws = make(st)
    fw = ops.StagedForward(torch.zeros(40, 64, dtype=BF), None, None, st)
    bw = ops.StagedBackward(torch.zeros(40, 48, dtype=BF), None, None, fw.z, st)
    assert fw.ws is ws and bw.ws is ws
    assert fw.args.prob.flags & _lib.PLAN_RESIDENT and bw.args.prob.flags & _lib.PLAN_RESIDENT


def test_a_changed_plan_is_not_resident(uploads):
    st = state()
    make(st)
    assert resident(st) is not None
    st.plan.seg_start[:] = [0, 3, 40]
    assert resident(st) is None
    make(st)
    assert resident(st) is not None and len(uploads) == 2


# ------------------------------------------------------------------ forward-mode derivatives

def test_tensors_with_tangents_are_refused():
    import torch.autograd.forward_ad as fw

    m = MultiLoRALinear(64, 48, {0: 4})
    ids, x = torch.zeros(3, dtype=torch.int64), torch.ones(3, 64)
    w8 = ops.Int8Rows(torch.zeros(48, 64, dtype=torch.int8), torch.ones(48), 64)
    with fw.dual_level():
        dual = fw.make_dual(x, torch.ones_like(x))
        for grad in (False, True):
            with torch.set_grad_enabled(grad):
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    m(dual, ids)
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    ops.int8_linear(dual, w8)
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    ops.int8_linear(x, w8, fw.make_dual(torch.zeros(48), torch.ones(48)))
        with pytest.raises(RuntimeError, match="CUDA"):  # without a tangent: the usual check
            m(x, ids)
    m = MultiLoRALinear(64, 48, {0: 4})
    for p in (m.adapters["0"].A, m.adapters["0"].B, m.base.weight, m.base.bias):
        p.requires_grad_(False)
    with fw.dual_level():
        for name in ("adapters.0.A", "adapters.0.B", "base.weight", "base.bias"):
            p = dict(m.named_parameters())[name]
            with pytest.raises(NotImplementedError, match="forward-mode"):
                torch.func.functional_call(m, {name: fw.make_dual(p.detach(), torch.ones_like(p))}, (x, ids))


# ------------------------------------------------------------------ limits of a native call

def test_contraction_limits():
    """Each call is limited by the length of its own sums: d_in of the forward,
    d_out of dX.  No rows: nothing is launched."""
    lib, none, over = _lib.lib(), ctypes.c_void_p(None), _lib.Q8_MAX_K + 8

    def linear(d_in, d_out):
        p = _lib.Problem(0, d_in, d_out, _lib.BF16, _lib.IMPL_AUTO)
        return (lib.mlora_q8_linear(ctypes.byref(p), none, 0, *[none] * 7),
                lib.mlora_q8_linear_dx(ctypes.byref(p), *[none] * 7))
    assert linear(64, over) == (_lib.OK, _lib.ERR_UNSUPPORTED)
    assert linear(over, 64) == (_lib.ERR_UNSUPPORTED, _lib.OK)
    assert linear(64, (1 << 30) + 1)[0] == _lib.ERR_UNSUPPORTED

    def layer(d_in, d_out, dx):
        p = _lib.Problem(0, d_in, d_out, _lib.BF16, _lib.IMPL_AUTO)
        r, a = _lib.Routing(0, None, None, 0, None, None, None, 0, None), ctypes.c_void_p(4096)
        q8 = _lib.Q8(4096, 4096, 4096, 4096, 4096, 4096)
        return (lib.mlora_forward_q8(ctypes.byref(p), ctypes.byref(r), ctypes.byref(q8), a, *[none] * 7, 0, none),
                lib.mlora_backward_q8(ctypes.byref(p), ctypes.byref(r), ctypes.byref(q8), a, none, none, none, none,
                                      none, a if dx else none, none, none, none, 0, none))
    assert layer(64, over, False) == (_lib.OK, _lib.OK)
    assert layer(64, over, True) == (_lib.OK, _lib.ERR_UNSUPPORTED)
    assert layer(over, 64, True) == (_lib.ERR_UNSUPPORTED, _lib.OK)


# ------------------------------------------------------------------ settings that a path does not have

def test_staged_calls_refuse_8_bits():
    base8 = ops.Int8Rows(torch.zeros(48, 64, dtype=torch.int8), torch.ones(48), 64)
    x, dy = torch.zeros(40, 64, dtype=BF), torch.zeros(40, 48, dtype=BF)
    for changed in ({"base8": base8}, {"save8": True}):
        st = state()
        for k, v in changed.items():
            setattr(st, k, v)
        with pytest.raises(NotImplementedError, match="8 bits"):
            ops.StagedForward(x, None, None, st)
        with pytest.raises(NotImplementedError, match="8 bits"):
            ops.StagedBackward(dy, x, None, torch.zeros(1), st)


def test_sharded_layers_refuse_inputs_saved_in_8_bits():
    from tlora_b200.overlap import ShardedLayer

    m = MultiLoRALinear(256, 64, {0: 4})
    m.save_input = "int8"
    with pytest.raises(NotImplementedError, match="save_input"):
        ShardedLayer(m, 0, 1)
    m.save_input = "eight"
    with pytest.raises(ValueError, match="save_input"):
        ShardedLayer(m, 0, 1)


# ------------------------------------------------------------------ modules that were changed by hand

def test_bias_of_another_length():
    base8 = ops.Int8Rows(torch.zeros(48, 64, dtype=torch.int8), torch.ones(48), 64)
    for bad in (torch.zeros(47), torch.zeros(49), torch.zeros(1, 48)):
        with pytest.raises(ValueError, match="bias"):
            Int8Base(base8, bad)
    m = MultiLoRALinear(64, 48, {0: 4})
    pk = m._pack()
    pk.sync()
    x, A, B = torch.zeros(3, 64), pk.A_pack, pk.B_pack
    ops.check_base(x, A, B, m.base.weight, m.base.bias, None)
    ops.check_base(x, A, B, None, None, base8)
    for W, bias, b8 in ((m.base.weight[:, 1:], None, None), (m.base.weight[1:], None, None),
                        (m.base.weight, torch.zeros(47), None), (None, torch.zeros(47), base8),
                        (None, None, ops.Int8Rows(torch.zeros(47, 64, dtype=torch.int8), torch.ones(47), 64))):
        with pytest.raises(ValueError):
            ops.check_base(x, A, B, W, bias, b8)
    with pytest.raises(RuntimeError, match="bias"):
        ops.check_base(x, A, B, None, torch.zeros(48, dtype=BF), base8)


def test_adapter_weights_that_are_plain_tensors():
    # as functional training loops set them: no longer parameters, still the weights
    m = MultiLoRALinear(64, 48, {0: 4, 1: 8})
    ad, pk = m.adapters["0"], m._pack()
    pk.sync()
    new = torch.randn(4, 64, requires_grad=True)
    del ad.A
    ad.A = new
    assert pk.params()[0] is new and pk.params()[1] is ad.B
    pk.sync()
    assert torch.equal(pk.A_pack[:4], new.detach())


# ------------------------------------------------------------------ the oracle itself

@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [8, 64, 200])
def test_bound_of_saved_dA_sees_a_lost_low_part(dt, n):
    import _saved_ref as saved

    g = torch.Generator().manual_seed(n)
    x = torch.randn(n, 256, generator=g).to(dt)
    dy, B = (torch.randn(n, 192, generator=g) * 0.1).to(dt), (torch.randn(192, 16, generator=g) * 0.05).to(dt)
    v, bound = saved.dA_saved(x, B, 0.75, dy)
    assert bool(((saved.dA_both(x, B, 0.75, dy).double() - v).abs() <= bound).all())
    lost = (saved.dA_high_only(x, B, 0.75, dy).double() - v).abs() > bound
    assert int(lost.sum()) >= 16  # of 4096: elements whose terms nearly cancel


# ------------------------------------------------------------------ devices and plain containers

def test_streams_of_devices(monkeypatch):
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda i: 100 + i, raising=False)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 3)
    assert ops._stream(torch.device("cuda", 1)) == 101
    assert ops._stream(torch.device("cuda")) == 103 and ops._stream("cuda") == 103 and ops._stream("cuda:2") == 102
    for bad in (torch.device("cpu"), torch.device("cpu", 0), "cpu"):  # host pointers must not reach a kernel
        with pytest.raises(ValueError, match="CUDA"):
            ops._stream(bad)
    x, perm = torch.zeros(2, 16, device="cpu:0"), torch.zeros(2, dtype=torch.int32)
    for call in (ops.gather_rows, ops.scatter_rows):
        with pytest.raises(ValueError, match="CUDA"):
            call(x, perm)


def test_plans_and_scalings_given_as_lists():
    a = state()
    b = state()
    b.plan = ops.RoutePlan(40, [0, 20, 40], [0, 1])
    b.scaling = [0.5, 0.75]
    assert segments(call_of(a)) == segments(call_of(b))
    assert [call_of(b).route.scaling[i] for i in range(2)] == [0.5, 0.75]
    b.plan.seg_start[1] = 7
    assert segments(call_of(b)) == ([0, 7, 40], [0, 1])


def test_active_adapters_of_a_call():
    st = state()
    assert call_of(st).active == [True, True]
    st.plan.seg_start, st.plan.seg_adapter = np.array([0, 40, 40], np.int32), np.array([1, 0], np.int32)
    assert call_of(st).active == [False, True]
    st.plan.seg_start, st.plan.seg_adapter = np.array([0, 40], np.int32), np.array([-1], np.int32)
    assert call_of(st).active == [False, False]
