"""
Argument checks of the operators on device tensors, on a machine without a GPU: every refusal comes before the first call
that needs a device, with a status and a message, and never ends the process.
"""
import ctypes

import pytest

from ios.contrib import ios_runtime as rt

ARGUMENT, LIMIT = 3, 6
F32, F16, BF16, S8 = 0, 1, 2, 3
SOME = 4096        # stands for a device address; no refused call may look at it


@pytest.fixture(scope='module')
def lib():
    return rt.load_ios_library()


def route(lib, **change):
    a = dict(logits=SOME, type=F32, tokens=4, experts=8, stride=8, k=2, renormalize=1, chosen=SOME, gates=SOME, offsets=SOME,
             rows=SOME, slots=SOME, workspace=None, bytes=0)
    assert not set(change) - set(a)
    a.update(change)
    return lib.ios_route_experts(*a.values(), None)


@pytest.mark.parametrize('change,status', [
    (dict(type=S8), ARGUMENT), (dict(type=9), ARGUMENT), (dict(tokens=-1), ARGUMENT), (dict(experts=0), ARGUMENT),
    (dict(k=0), ARGUMENT), (dict(k=9), ARGUMENT), (dict(stride=-8), ARGUMENT), (dict(experts=1025), LIMIT),
    (dict(experts=64, k=33), LIMIT), (dict(tokens=2 ** 29, k=4), LIMIT), (dict(logits=None), ARGUMENT), (dict(slots=None), ARGUMENT),
    (dict(offsets=None), ARGUMENT), (dict(tokens=5000), ARGUMENT), (dict(tokens=5000, workspace=SOME, bytes=64), ARGUMENT)])
def test_route_refuses(lib, change, status):
    assert route(lib, **change) == status
    assert b'route_experts' in lib.ios_last_error()


def test_route_workspace(lib):
    size = ctypes.c_size_t(7)
    assert lib.ios_route_experts_workspace(1, 64, 8, ctypes.byref(size)) == 0 and size.value == 0
    assert lib.ios_route_experts_workspace(100000, 1024, 8, ctypes.byref(size)) == 0
    assert 0 < size.value <= 128 * 1024 * 4
    assert lib.ios_route_experts_workspace(1, 0, 8, ctypes.byref(size)) == ARGUMENT
    assert lib.ios_route_experts_workspace(1, 8, 2, None) == ARGUMENT


def grouped(lib, **change):
    a = dict(x=SOME, type=BF16, x_rows=10, x_stride=64, w=SOME, groups=2, channels=32, inner=64, w_stride=64, w_group_stride=2048,
             offsets=SOME, rows=None, total=10, row_scale=None, channel_scale=None, bias=None, act=0, gated=0, y=SOME, y_type=BF16,
             y_stride=32)
    assert not set(change) - set(a)
    a.update(change)
    return lib.ios_grouped_matmul(*a.values(), None)


@pytest.mark.parametrize('change,status', [
    (dict(type=4), ARGUMENT), (dict(y_type=S8), ARGUMENT), (dict(offsets=None), ARGUMENT), (dict(act=5), ARGUMENT),
    (dict(act=-1), ARGUMENT), (dict(channels=0), ARGUMENT), (dict(inner=0), ARGUMENT), (dict(total=-1), ARGUMENT),
    (dict(groups=0), LIMIT), (dict(groups=1025), LIMIT), (dict(x_stride=-1), ARGUMENT), (dict(y_stride=31), ARGUMENT),
    (dict(type=S8, inner=131072, x_stride=131072), LIMIT), (dict(x_rows=9), ARGUMENT), (dict(x=None), ARGUMENT),
    (dict(w=None), ARGUMENT), (dict(y=None), ARGUMENT), (dict(channels=2 ** 30, y_stride=2 ** 30), LIMIT), (dict(total=2 ** 30 + 1, x_rows=2 ** 31), LIMIT),
    (dict(total=2 ** 29, x_rows=2 ** 29, channels=2 ** 20, y_stride=2 ** 20), LIMIT)])
def test_grouped_refuses(lib, change, status):
    assert grouped(lib, **change) == status
    assert b'grouped_matmul' in lib.ios_last_error()


def test_no_rows_are_no_error(lib):
    assert grouped(lib, total=0, x_rows=0, x=None, y=None, offsets=None) == 0
    assert lib.ios_last_error() == b''
    assert lib.ios_matmul_int8(None, 8, None, 8, 0, 4, 8, None, None, None, 0, None, F32, 4, None) == 0
    assert lib.ios_quantize_rows(None, F32, 0, 8, 8, None, 0, None, 8, None, None) == 0
    assert lib.ios_combine_experts(None, F32, 0, 8, None, None, 0, 2, 8, None, F32, 8, None) == 0


def test_int8_refuses(lib):
    def call(a=SOME, b=SOME, rows=4, channels=8, inner=16, act=0, y=SOME, y_type=F32, y_stride=8):
        return lib.ios_matmul_int8(a, 16, b, 16, rows, channels, inner, None, None, None, act, y, y_type, y_stride, None)
    for status, change in ((ARGUMENT, dict(a=None)), (ARGUMENT, dict(b=None)), (ARGUMENT, dict(y=None)), (ARGUMENT, dict(act=7)),
                           (ARGUMENT, dict(y_type=S8)), (ARGUMENT, dict(rows=-1)), (ARGUMENT, dict(y_stride=7)),
                           (LIMIT, dict(inner=1 << 17))):
        assert call(**change) == status, change
        assert b'matmul_int8' in lib.ios_last_error()


def test_quantize_and_combine_refuse(lib):
    def quantize(x=SOME, type=F32, x_rows=4, inner=8, total=4, q=SOME, q_stride=8, scale=SOME):
        return lib.ios_quantize_rows(x, type, x_rows, 8, inner, None, total, q, q_stride, scale, None)
    for change in (dict(x=None), dict(type=S8), dict(inner=0), dict(x_rows=3), dict(total=-1), dict(q=None), dict(q_stride=7),
                   dict(scale=None)):
        assert quantize(**change) == ARGUMENT, change
        assert b'quantize_rows' in lib.ios_last_error()

    def combine(y=SOME, type=F32, y_rows=4, gates=SOME, slots=SOME, tokens=2, k=2, channels=8, out=SOME, out_type=F32, stride=8):
        return lib.ios_combine_experts(y, type, y_rows, 8, gates, slots, tokens, k, channels, out, out_type, stride, None)
    assert quantize(total=2 ** 30 + 1, x_rows=2 ** 31) == LIMIT and combine(tokens=2 ** 30 + 1) == LIMIT
    assert combine(channels=2 ** 24, stride=2 ** 24) == LIMIT
    for change in (dict(y=None), dict(type=S8), dict(out_type=S8), dict(gates=None), dict(slots=None), dict(tokens=-1), dict(k=0),
                   dict(channels=0), dict(out=None), dict(stride=7), dict(y_rows=-1)):
        assert combine(**change) == ARGUMENT, change
        assert b'combine_experts' in lib.ios_last_error()


def test_python_refuses_what_is_no_gpu_tensor():
    torch = pytest.importorskip('torch')
    x, w, offsets = torch.zeros(4, 8), torch.zeros(2, 4, 8), torch.zeros(3, dtype=torch.int32)
    for call in (lambda: rt.route_experts(x, 2), lambda: rt.grouped_matmul(x, w, offsets), lambda: rt.quantize_rows(x),
                 lambda: rt.combine_experts(x, x, x)):
        with pytest.raises(ValueError, match='GPU'):
            call()
    with pytest.raises(ValueError, match='type'):
        rt.matmul_int8(x, x)
    with pytest.raises(ValueError, match='axes'):
        rt.route_experts(x[0], 2)
    with pytest.raises(ValueError, match='torch.Tensor'):
        rt.quantize_rows([[1.0]])
    with pytest.raises(ValueError, match='type'):
        rt.quantize_rows(x.double())
