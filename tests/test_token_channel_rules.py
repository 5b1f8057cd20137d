"""The token/channel product's choice of tile and parts at shapes where the forms were timed on MI355X
and one is clearly the fastest, and its C ABI's refusals (CPU only: no kernel runs)."""

import ctypes

import pytest

from ksdraft_amd import _lib


def form(M, N, K):
    v = [ctypes.c_int() for _ in range(4)]
    _lib.call("ksd_tc_gemm_form", M, N, K, *[ctypes.byref(x) for x in v])
    return tuple(x.value for x in v)  # tile rows, tile columns, workgroups per CU, parts


# (rows, columns, K, times in us by (tile rows, tile columns, workgroups per CU))
TIMES = [(8192, 8192, 8192, {(256, 256, 1): 480, (256, 192, 1): 547, (128, 128, 2): 614, (128, 128, 1): 688, (64, 64, 2): 921}),
         (8192, 1536, 1536, {(256, 192, 1): 24.7, (256, 256, 1): 26.0, (128, 128, 2): 30.3, (128, 128, 1): 35.9, (64, 128, 2): 33.7}),
         (1021, 1792, 597, {(64, 64, 2): 8.5, (128, 128, 2): 11.1, (256, 192, 1): 17.2, (128, 128, 1): 12.2}),
         (300, 500, 333, {(64, 64, 2): 6.2, (64, 128, 2): 7.1, (128, 128, 2): 9.5, (256, 192, 1): 13.0}),
         (2047, 1792, 1792, {(64, 128, 2): 15.9, (128, 128, 1): 18.1, (64, 64, 2): 19.6, (128, 128, 2): 27.9}),
         (2047, 1792, 6869, {(128, 128, 1): 38.5, (64, 128, 2): 40.5, (128, 128, 2): 45.8, (256, 192, 1): 50.3}),
         (1536, 1536, 8192, {(128, 128, 1): 39.5, (128, 128, 2): 40.3, (256, 192, 1): 42.7, (64, 128, 2): 48.9, (64, 64, 2): 65.4})]


@pytest.mark.parametrize("M,N,K,times", TIMES)
def test_form(M, N, K, times):
    got = form(M, N, K)[:3]
    assert times[got] <= 1.05 * min(times.values())


def test_long_reductions_are_split():
    """No part's int32 sum can pass 31 bits: at most 131072 products of 127^2."""
    for K in (1, 128, 131072, 131073, 150144, 1 << 20):
        for M, N in ((1, 1), (5000, 5000)):
            parts = form(M, N, K)[3]
            steps = -(-K // 128)
            assert -(-steps // parts) <= 1024


def test_every_form_is_reached():
    assert {form(*s)[:3] for s in [(8192, 8192, 512), (8192, 1536, 1536), (4685, 801, 129), (1536, 1536, 8192), (2047, 1792, 1792),
                                   (300, 500, 333)]} == {(256, 256, 1), (256, 192, 1), (128, 128, 2), (128, 128, 1), (64, 128, 2), (64, 64, 2)}


def test_refusals_without_gpu():
    lib = _lib.load()
    n = ctypes.c_int64()
    assert lib.ksd_tc_quantize_rows(None, 0, 4, 20, 20, None, 20, None, None) == 1   # pitch not rounded up
    assert lib.ksd_tc_quantize_rows(None, 7, 4, 20, 20, None, 32, None, None) == 2   # type
    assert lib.ksd_tc_quantize_rows(None, 0, 0, 20, 20, None, 32, None, None) == 0   # no rows
    assert lib.ksd_tc_gemm(None, 16, 0, None, None, 16, 0, None, 4, 4, 20, None, None, None, 0, None, 0, None) == 1  # pitch
    assert lib.ksd_tc_gemm(None, 32, 1, None, None, 32, 0, None, 4, 4, 20, None, None, None, 0, None, 0, None) == 1  # a_t alone
    assert lib.ksd_tc_gemm(None, 32, 0, None, None, 32, 0, None, 4, 4, 20, None, None, None, 9, None, 0, None) == 2
    assert lib.ksd_tc_gemm(None, 32, 0, None, None, 32, 0, None, 4, 4, 20, None, None, None, 0, None, 0, None) == 1  # null
    assert lib.ksd_tc_linear(None, 0, 4, 0, 0, None, 16, None, 4, None, None, None, 0, None, 0, None) == 1
    assert lib.ksd_tc_linear_backward_workspace(0, 4, 4, 1, 1, ctypes.byref(n)) == 1
    assert lib.ksd_embedding_lookup(None, 0, 10, 4, 3, None, 1, 2, 1.0, None, 0, None) == 1   # stride
    assert lib.ksd_embedding_lookup(None, 0, 0, 4, 4, None, 1, 2, 1.0, None, 0, None) == 1    # empty table
    assert lib.ksd_embedding_gradient(None, 0, 2, 4, 4, None, 1, 10, -1, 1.0, 0, None, 9, None, 0, None) == 2
    assert lib.ksd_embedding_gradient(None, 0, 1 << 31, 4, 4, None, 1, 10, -1, 1.0, 0, None, 0, None, 0, None) == 1
    sizes, types, ptrs = (ctypes.c_int64 * 1)(5), (ctypes.c_int32 * 1)(9), (ctypes.c_void_p * 1)(None)
    assert lib.ksd_grad_norm(ptrs, sizes, types, 1, 0, 1.0, 1.0, None, None, None, 0, None) == 2  # type
    types[0] = 0
    assert lib.ksd_grad_norm(ptrs, sizes, types, 1, 0, 1.0, 1.0, None, None, None, 0, None) == 1  # null gradient
    assert lib.ksd_grad_scale(ptrs, None, sizes, types, 1, None, None) == 1
    assert lib.ksd_grad_norm_workspace(sizes, 1, ctypes.byref(n)) == 0 and n.value == 8
