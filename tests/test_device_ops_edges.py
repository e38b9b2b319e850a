"""
Arguments of the operators on device tensors at the edges of what they take, on a machine without a GPU.
"""
import ctypes

import pytest

from ios.contrib import ios_runtime as rt


def test_what_a_wait_may_take_is_checked():
    for bad in (-1, 2000001):
        with pytest.raises(RuntimeError, match='product_wait_us'):
            rt.set_option('product_wait_us', bad)
    rt.set_option('product_wait_us', 0)


def test_status_of_no_device_is_refused():
    for device in (-1, 64):
        assert rt.load_ios_library().ios_device_ops_status(device, None) == 3
        assert b'device_ops_status' in rt.load_ios_library().ios_last_error()


def test_route_workspace_of_long_calls():
    """A row of counts per block of 8192 pairs, and beyond 128 blocks one more; linear in the tokens."""
    lib, size = rt.load_ios_library(), ctypes.c_size_t(0)
    for tokens, rows in ((131072, 128), (131073, 130), (1 << 27, (1 << 17) + 1)):
        assert lib.ios_route_experts_workspace(tokens, 64, 8, ctypes.byref(size)) == 0
        assert size.value == rows * 64 * 4


def test_status_asks_about_the_device_that_is_meant(monkeypatch):
    """'cuda' without a number is the current device, as everywhere in torch."""
    torch = pytest.importorskip('torch')
    from ios.contrib import device_ops
    asked = []

    class Library:
        def ios_device_ops_status(self, index, stream):
            asked.append((index, stream))
            return 0

    monkeypatch.setattr(device_ops, 'torch', torch)
    monkeypatch.setattr(device_ops, '_lib', Library())
    monkeypatch.setattr(device_ops, '_raw_stream', lambda index: 100 + index)
    monkeypatch.setattr(torch.cuda, 'current_device', lambda: 3)
    for device in (None, 'cuda', torch.device('cuda'), 'cuda:2', torch.device('cuda', 0), 1):
        rt.device_ops_status(device)
    assert asked == [(index, 100 + index) for index in (3, 3, 3, 2, 0, 1)]
    with pytest.raises(ValueError, match='not a GPU'):
        rt.device_ops_status('cpu')


def test_route_workspace_refuses_what_route_refuses():
    """(2^31 - 1 tokens passed 32 bits on the way and came out as a size of some sort.)"""
    lib, size = rt.load_ios_library(), ctypes.c_size_t(7)
    for status, args in ((6, (2 ** 31 - 1, 1024, 1)), (6, (2 ** 30, 8, 2)), (6, (1, 1025, 1)), (6, (1, 64, 33)), (3, (10, 4, 8)), (3, (-1, 4, 2))):
        assert lib.ios_route_experts_workspace(*args, ctypes.byref(size)) == status, args
        assert b'route_experts' in lib.ios_last_error() and size.value == 7


def test_16_bit_products_of_too_long_rows_are_refused():
    lib = rt.load_ios_library()
    for kind in (1, 2):
        assert lib.ios_grouped_matmul(4096, kind, 1, 0, 4096, 1, 8, 2 ** 25 + 1, 0, 0, 4096, None, 1, None, None, None, 0, 0, 4096, 0, 8, None) == 6
        assert b'2^25' in lib.ios_last_error()
