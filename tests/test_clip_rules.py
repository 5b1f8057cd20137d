"""Lists that clipping must refuse because two of its workgroups would meet in one tensor's memory: the
C ABI's check reads addresses alone, so it is tested without a GPU (no kernel runs)."""

import ctypes

import pytest

from ksdraft_amd import _lib

F32, BF16 = 0, 1


def scale(grads, outs, sizes, types):
    n = len(sizes)
    return _lib.load().ksd_grad_scale((ctypes.c_void_p * n)(*grads), (ctypes.c_void_p * n)(*outs), (ctypes.c_int64 * n)(*sizes),
                                      (ctypes.c_int32 * n)(*types), n, ctypes.c_void_p(0x10), None)


def message():
    buf = ctypes.create_string_buffer(256)
    _lib.load().ksd_last_error(buf, 256)
    return buf.value


@pytest.mark.parametrize("grads,outs,sizes,types", [
    ([0x1000, 0x1000], [0x1000, 0x1000], [8, 8], [F32, F32]),                    # one tensor twice, in place
    ([0x1000, 0x9000, 0x1000], [0x1000, 0x9000, 0x1000], [8, 8, 8], [F32] * 3),  # with another between
    ([0x1000, 0x101c], [0x1000, 0x101c], [8, 8], [F32, F32]),                    # the last element of one
    ([0x1000, 0x2000], [0x5000, 0x5000], [8, 8], [F32, F32]),                    # one output for two
    ([0x2000, 0x1000], [0x500e, 0x5000], [8, 8], [BF16, BF16]),
    ([0x1000, 0x2000], [0x2000, 0x3000], [8, 8], [F32, F32]),                    # a later one's gradient as output
    ([0x1000, 0x2000], [0x3000, 0x1000], [8, 8], [F32, F32]),                    # an earlier one's
    ([0x1000], [0x1004], [8], [F32]),                                            # its own, shifted
    ([0x1004], [0x1000], [8], [F32]),
    ([0x1000, 0x3000], [0x1000, 0x101c], [8, 8], [F32, F32]),                    # in place beside another's output
])
def test_shared_memory_is_refused(grads, outs, sizes, types):
    assert scale(grads, outs, sizes, types) == 1
    assert b"memory" in message()
