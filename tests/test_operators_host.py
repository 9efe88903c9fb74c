"""Grouped routing, 8-bit float products and block norms: what their entry points refuse, without a GPU."""
import ctypes as C

import numpy as np
import pytest
import torch

from oco_b200 import _lib, build


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.lib()


def router(lib, **kw):
    d = dict(hidden=512, experts=64, top_k=6, score=0, groups=8, top_groups=3, group_best=2, normalize=1, scale=1.0)
    d.update(kw)
    h = C.c_void_p()
    rc = lib.oco_moe_router_create(C.byref(_lib.RouterDesc(**d)), C.byref(h))
    return rc, h


def test_router_descriptions(lib):
    rc, h = router(lib)
    assert rc == _lib.OK
    assert lib.oco_moe_router_workspace_bytes(h, 100) >= 100 * 64 * 4 and lib.oco_moe_router_workspace_bytes(h, 0) == 0
    assert lib.oco_moe_router_forward(h, None, 1, None, None, None, None) == _lib.INVALID_ARGUMENT and b"bind" in lib.oco_moe_router_last_error(h)
    assert lib.oco_moe_router_select(h, None, 1, None, None, None) == _lib.INVALID_ARGUMENT
    assert lib.oco_moe_router_bind_workspace(h, None, 0, 1) == _lib.INVALID_ARGUMENT
    assert lib.oco_moe_router_bind_workspace(h, C.c_void_p(4096), 16, 1) == _lib.INVALID_ARGUMENT and b"small" in lib.oco_moe_router_last_error(h)
    assert lib.oco_moe_router_bind_workspace(h, C.c_void_p(4100), 1 << 30, 1) == _lib.INVALID_ARGUMENT and b"aligned" in lib.oco_moe_router_last_error(h)
    assert lib.oco_moe_router_bind_weights(h, None, None) == _lib.INVALID_ARGUMENT
    assert lib.oco_moe_router_bind_weights(h, C.c_void_p(4100), None) == _lib.INVALID_ARGUMENT
    lib.oco_moe_router_destroy(h)
    for kw, code in ((dict(hidden=100), _lib.UNSUPPORTED_SHAPE), (dict(hidden=-32), _lib.UNSUPPORTED_SHAPE), (dict(hidden=16416), _lib.UNSUPPORTED_SHAPE),
                     (dict(experts=0), _lib.UNSUPPORTED_SHAPE), (dict(experts=520), _lib.UNSUPPORTED_SHAPE), (dict(groups=7), _lib.UNSUPPORTED_SHAPE),
                     (dict(groups=0), _lib.UNSUPPORTED_SHAPE), (dict(groups=64), _lib.UNSUPPORTED_SHAPE), (dict(top_groups=0), _lib.INVALID_ARGUMENT),
                     (dict(top_groups=9), _lib.INVALID_ARGUMENT), (dict(top_k=0), _lib.UNSUPPORTED_SHAPE), (dict(top_k=17), _lib.UNSUPPORTED_SHAPE),
                     (dict(top_groups=1, top_k=9), _lib.INVALID_ARGUMENT), (dict(group_best=3), _lib.INVALID_ARGUMENT), (dict(score=2), _lib.INVALID_ARGUMENT)):
        rc, h = router(lib, **kw)
        assert rc == code and lib.oco_moe_router_last_error(h), kw
        lib.oco_moe_router_destroy(h)
    assert lib.oco_moe_router_create(None, None) == _lib.INVALID_ARGUMENT
    lib.oco_moe_router_destroy(None)
    for f in (lib.oco_moe_router_poll,):
        assert f(None, None) == _lib.INVALID_ARGUMENT
    assert lib.oco_moe_router_forward(None, None, 1, None, None, None, None) == _lib.INVALID_ARGUMENT
    assert lib.oco_moe_router_last_error(None) == b"null plan"
    # a plan without rows selects only
    rc, h = router(lib, hidden=0)
    assert rc == _lib.OK and lib.oco_moe_router_forward(h, None, 1, None, None, None, None) == _lib.INVALID_ARGUMENT
    assert lib.oco_moe_router_bind_weights(h, C.c_void_p(4096), None) == _lib.INVALID_ARGUMENT
    assert lib.oco_moe_router_bind_weights(h, None, None) == _lib.OK
    assert lib.oco_moe_router_select(h, None, 0, None, None, None) == _lib.OK
    assert lib.oco_moe_router_select(h, None, -1, None, None, None) == _lib.INVALID_ARGUMENT
    assert lib.oco_moe_router_select(h, C.c_void_p(4098), 1, C.c_void_p(4096), C.c_void_p(4096), None) == _lib.INVALID_ARGUMENT
    lib.oco_moe_router_destroy(h)


def test_f8_descriptions(lib):
    h = C.c_void_p()
    good = dict(hidden=256, ffn=160, experts=8, top_k=2)
    assert lib.oco_moe_f8_plan_create(C.byref(_lib.F8Desc(**good)), C.byref(h)) == _lib.OK
    one, many = lib.oco_moe_f8_workspace_bytes(h, 1), lib.oco_moe_f8_workspace_bytes(h, 4096)
    assert 0 < one < many and many > 4096 * 2 * (256 + 160 + 2 * 256) and lib.oco_moe_f8_workspace_bytes(h, 0) == 0
    assert lib.oco_moe_f8_forward(h, None, None, None, None, None, 1, None) == _lib.INVALID_ARGUMENT and b"bind" in lib.oco_moe_f8_last_error(h)
    assert lib.oco_moe_f8_bind_weights(h, None) == _lib.INVALID_ARGUMENT
    w = _lib.F8Weights(gate_w=4096, up_w=4096, down_w=4104, gate_s=4096, up_s=4096, down_s=4096)
    assert lib.oco_moe_f8_bind_weights(h, C.byref(w)) == _lib.INVALID_ARGUMENT and b"aligned" in lib.oco_moe_f8_last_error(h)
    w = _lib.F8Weights(gate_w=4096, up_w=4096, down_w=4096, gate_s=4096, up_s=4096)
    assert lib.oco_moe_f8_bind_weights(h, C.byref(w)) == _lib.INVALID_ARGUMENT and b"down_s" in lib.oco_moe_f8_last_error(h)
    assert lib.oco_moe_f8_bind_workspace(h, C.c_void_p(4096), 100, 1) == _lib.INVALID_ARGUMENT
    assert lib.oco_moe_f8_bind_workspace(h, C.c_void_p(4096), 1 << 62, (1 << 30)) == _lib.UNSUPPORTED_SHAPE
    lib.oco_moe_f8_plan_destroy(h)
    for kw in (dict(hidden=48), dict(hidden=0), dict(ffn=33), dict(ffn=131072), dict(experts=0), dict(experts=513), dict(top_k=0), dict(top_k=17)):
        assert lib.oco_moe_f8_plan_create(C.byref(_lib.F8Desc(**{**good, **kw})), C.byref(h)) == _lib.UNSUPPORTED_SHAPE, kw
        assert lib.oco_moe_f8_last_error(h)
        lib.oco_moe_f8_plan_destroy(h)
    assert lib.oco_moe_f8_plan_create(None, None) == _lib.INVALID_ARGUMENT
    assert lib.oco_moe_f8_poll(None, None) == _lib.INVALID_ARGUMENT and lib.oco_moe_f8_last_error(None) == b"null plan"
    lib.oco_moe_f8_plan_destroy(None)


def test_f8_dense_plans(lib):
    h = C.c_void_p()
    for kind, hidden, ffn, code in ((0, 256, 96, _lib.OK), (2, 256, 160, _lib.OK), (1, 256, 256, _lib.UNSUPPORTED_SHAPE), (0, 40, 64, _lib.UNSUPPORTED_SHAPE),
                                    (2, 256, 40, _lib.UNSUPPORTED_SHAPE), (7, 256, 256, _lib.INVALID_ARGUMENT)):
        d = _lib.DenseDesc(kind=kind, weight_format=128, hidden=hidden, ffn=ffn)
        assert lib.oco_dense_plan_create(C.byref(d), C.byref(h)) == code, (kind, hidden, ffn)
        if code == _lib.OK:
            assert lib.oco_dense_workspace_bytes(h, 10) > 10 * hidden
            assert lib.oco_dense_bind_scales(h, C.byref(_lib.DenseScales(up_s=4096))) == _lib.INVALID_ARGUMENT        # codes come first
            assert lib.oco_dense_bind_weights(h, C.byref(_lib.DenseWeights())) == _lib.INVALID_ARGUMENT
            assert lib.oco_dense_bind_weights(h, None) == _lib.INVALID_ARGUMENT
            assert lib.oco_dense_forward(h, None, None, 1, None) == _lib.INVALID_ARGUMENT
        assert lib.oco_dense_last_error(h) or code == _lib.OK
        lib.oco_dense_plan_destroy(h)
    # the block formats carry their scales
    d = _lib.DenseDesc(kind=0, weight_format=39, hidden=256, ffn=256)
    assert lib.oco_dense_plan_create(C.byref(d), C.byref(h)) == _lib.OK
    assert lib.oco_dense_bind_scales(h, C.byref(_lib.DenseScales(up_s=4096))) == _lib.INVALID_ARGUMENT
    lib.oco_dense_plan_destroy(h)
    assert lib.oco_dense_bind_scales(None, None) == _lib.INVALID_ARGUMENT


def test_block_norm_arguments(lib):
    err = C.create_string_buffer(160)
    good = dict(width=256, hidden=4096, block=4096, norm_out=4096, pre_w=4096, epsilon=1e-6)
    assert lib.oco_moe_block_norm(C.byref(_lib.BlockNormArgs(**good)), 0, None, err, 160) == _lib.OK
    for kw, code in ((dict(width=0), _lib.UNSUPPORTED_SHAPE), (dict(width=252), _lib.UNSUPPORTED_SHAPE), (dict(width=40000), _lib.UNSUPPORTED_SHAPE),
                     (dict(hidden=None), 1), (dict(norm_out=None), 1), (dict(kind=2), 1), (dict(gate_type=1), 1), (dict(gate=4096), 1),
                     (dict(gate=4096, gate_type=3), 1), (dict(gate_act=3), 1), (dict(gate_rows=-1), 1), (dict(block=None, post_w=4096), 1),
                     (dict(pre_b=4096), 1), (dict(kind=1, post_b=4096), 1), (dict(epsilon=-1.0), 1), (dict(epsilon=float("nan")), 1), (dict(hidden=4100), 1),
                     (dict(pre_w=4104), 1), (dict(hidden_stride=248), 1), (dict(block_stride=260), 1), (dict(norm_out_stride=-256), 1)):
        rc = lib.oco_moe_block_norm(C.byref(_lib.BlockNormArgs(**{**good, **kw})), 0, None, err, 160)
        assert rc == code and err.value, kw
    assert lib.oco_moe_block_norm(C.byref(_lib.BlockNormArgs(**good)), -1, None, None, 0) == _lib.INVALID_ARGUMENT
    assert lib.oco_moe_block_norm(None, 1, None, None, 0) == _lib.INVALID_ARGUMENT


def test_python_refusals_without_a_gpu(lib):
    from oco_b200 import dense, moe, synth
    with pytest.raises(_lib.OcoError, match="score"):
        moe.RouterPlan.new(256, 8, 2, score="tanh")
    with pytest.raises(_lib.OcoError, match="groups"):
        moe.RouterPlan.new(256, 9, 2, groups=2)
    with pytest.raises(_lib.OcoError, match="hidden"):
        moe.F8ExpertPlan.new(40, 32, 4, 2)
    plan = dense.DensePlan(dense.PROJECTION, synth.FMT_F8_E4M3, 128, 64)
    with pytest.raises(_lib.OcoError, match="scales"):
        plan.bind(np.zeros((64, 128), np.uint8))
    x = torch.zeros((2, 256), dtype=torch.bfloat16)
    with pytest.raises(_lib.OcoError, match="CUDA"):
        moe.block_norm(x, norm_out=x)
    r = moe.RouterPlan.new(256, 8, 2)
    with pytest.raises(_lib.OcoError, match="CUDA"):
        r.forward(x, torch.zeros(4, dtype=torch.int32), torch.zeros(4), 2)


def test_the_plain_forms_of_the_tests():
    """The tests' references on cases small enough to see: group choice, ties, a short last block."""
    from tests import opref
    l = np.array([[0.0, 3.0, 1.0, 2.5, 2.6, 0.1]])
    ids, p = opref.route(l, None, 6, 2, "sigmoid", 3, 1, 2, False, 1.0)       # groups (0,3) (1,2.5) (2.6,.1)
    assert ids.tolist() == [[3, 2]]
    ids, _ = opref.route(np.zeros((1, 6)), None, 6, 3, "softmax", 3, 2, 1, True, 1.0)
    assert ids.tolist() == [[0, 1, 2]]
    x = torch.zeros((1, 130), dtype=torch.float64)
    x[0, 0], x[0, 1], x[0, 129] = 448.0, 17.0, -3.0
    codes, scales = opref.quantize(x)
    assert codes[0, 1] == 16.0 and codes[0, 129] == -448.0 and scales.tolist() == [[1.0, 3.0 / 448.0]]


def test_f8_matrices_of_other_types(lib):
    """Codes are e4m3 or bytes and scales f32: other types of the same size would be read as something else."""
    from oco_b200 import moe
    codes, scales = torch.zeros((64, 128), dtype=torch.uint8), torch.ones((1, 1))
    for c, s in ((codes.view(torch.float8_e5m2), scales), (codes.view(torch.bool), scales), (codes, scales.view(torch.int32))):
        with pytest.raises(_lib.OcoError, match="contiguous elements"):
            moe.f8_matrix(c, s, (), 64, 128, "cpu", "up")
    with pytest.raises(_lib.OcoError, match="current device"):
        moe.f8_matrix(codes, scales, (), 64, 128, "cpu", "up")


def test_block_norm_overlaps(lib):
    """Rows that an output shares with an input of other rows; interleaved rows are no overlap. Refused before any CUDA call."""
    B = 1 << 20
    base = dict(width=64, kind=0, gate_type=1, gate_rows=1, gate_act=0, epsilon=1e-6, residual_scale=1.0, block_scale=1.0, hidden=B, block=2 * B, gate=3 * B,
                hidden_out=4 * B, norm_out=5 * B)
    err = C.create_string_buffer(160)
    refused = lambda **kw: (lib.oco_moe_block_norm(C.byref(_lib.BlockNormArgs(**{**base, **kw})), 8, None, err, len(err)) == _lib.INVALID_ARGUMENT  # noqa: E731
                            and b"overlap" in err.value)
    assert refused(hidden_out=B + 128) and refused(hidden_out=B, hidden_stride=128) and refused(norm_out=B) and refused(norm_out=2 * B + 16)
    assert refused(hidden_out=2 * B) and refused(hidden_out=3 * B + 7 * 128) and refused(norm_out=4 * B + 64) and refused(hidden_out=2 * B - 16)
    assert refused(hidden_out=B + 64, hidden_stride=128, hidden_out_stride=128) and refused(hidden_out=B - 64, hidden_stride=128, hidden_out_stride=128)
    halves = dict(hidden_stride=128, hidden_out_stride=128)
    if not torch.cuda.is_available():      # these go on to the launch, which has no device
        assert not refused() and not refused(hidden_out=B) and not refused(norm_out=2 * B) and not refused(hidden_out=3 * B + 8 * 128)
        assert not refused(hidden_out=B + 128, **halves) and not refused(hidden_out=B - 128, **halves)


def test_a_workspace_on_another_device_than_the_weights(lib):
    from oco_b200 import dense, moe, synth

    class OnSecondDevice:
        def get_device(self):
            return 1
    there = OnSecondDevice()
    plans = moe.RouterPlan.new(256, 8, 2), moe.F8ExpertPlan.new(128, 128, 4, 2), dense.DensePlan(dense.PROJECTION, synth.FMT_F8_E4M3, 128, 64)
    for plan, held in zip(plans, ((there, None), {"gate_w": there}, {"up": (there, there)})):
        plan._weights = held
        with pytest.raises(_lib.OcoError, match="another device"):
            plan.reserve(8, device="cpu")
        assert plan.workspace is None


def test_weights_on_another_device_than_the_workspace(lib, monkeypatch):
    """The other order: reserved on one device, bound while another one is current; and a bias that the current device has not."""
    from oco_b200 import dense, moe, synth

    class On:
        def __init__(self, number):
            self.number, self.device = number, f"cuda:{number}"

        def get_device(self):
            return self.number
    for module in (moe, dense):
        monkeypatch.setattr(module, "f8_matrix", lambda *a: (On(1), On(1)))
    experts, projection = moe.F8ExpertPlan.new(128, 128, 4, 2), dense.DensePlan(dense.PROJECTION, synth.FMT_F8_E4M3, 128, 64)
    for plan, args in ((experts, (moe.F8Experts(*[None] * 6),)), (projection, (None,))):
        plan.workspace = On(0)
        with pytest.raises(_lib.OcoError, match="another device"):
            plan.bind(*args)
        assert not plan._weights
    router = moe.RouterPlan.new(0, 8, 2)
    router._weights, router._bias = (None, On(1)), On(1)
    monkeypatch.setattr(moe, "_current_device", lambda: 0)
    with pytest.raises(_lib.OcoError, match="bias is on cuda:1"):
        router.select(None, None, None, 1)


def test_other_types_of_the_same_size(lib):
    """A tensor whose elements are as large as the right ones is refused all the same."""
    from oco_b200 import moe
    for types, good, bad in ((moe.BF16, (torch.bfloat16,), (torch.float16, torch.int16, torch.uint16)), (moe.F32, (torch.float32,), (torch.int32, torch.uint32)),
                             (moe.IDS, (torch.int32, torch.uint32), (torch.float32,))):
        for t in good:
            moe.need(torch.zeros(4, dtype=t), "x", types, 4, -1)
        for t in bad:
            with pytest.raises(_lib.OcoError, match="is needed"):
                moe.need(torch.zeros(4, dtype=t), "x", types, 4, -1)


def test_streams_without_torch_s_shortcut(monkeypatch):
    """The handle of the current stream by the public call, where torch has no other."""
    from oco_b200 import moe

    class Stream:
        cuda_stream = 0x7100
    monkeypatch.setattr(moe, "_raw_stream", None)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda: Stream)
    assert moe._stream_ptr().value == 0x7100
    monkeypatch.setattr(moe, "_raw_stream", lambda device: 0x7200 + device)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 3)
    assert moe._stream_ptr().value == 0x7203
