"""CPU tests of what the C entries of the class losses refuse before any device
work, beyond sizes and options: pointers that the kernels' accesses would fault
on."""
import ctypes

import pytest

from gs_voxelizer_b200._lib import CeOptions, lib

P = 4096


def options():
    return CeOptions(-100, 0.0, 0.0, 0.0, 2)


def refused(status):
    return status == 1 and b"aligned" in lib.gsv_last_error()


def call(fn, head, pointers, dtype, tail):
    """fn with `pointers` = {name: address} in the entry's order, options where
    the name is `opt`."""
    args = [options() if k == "opt" else ctypes.c_void_p(v) for k, v in pointers.items()]
    return fn(*head, dtype, *args, *tail)


@pytest.mark.parametrize("dtype,size", [(0, 4), (1, 2), (2, 2)])
@pytest.mark.parametrize("classes", [5, 5000])
def test_softmax_entries_refuse_misaligned_pointers(dtype, size, classes):
    names = dict(scores=size, labels=8, opt=0, loss=4, lse=8, count=4, ws=8)
    for name, size_of in names.items():
        if name == "opt":
            continue
        ptr = {k: P for k in names}
        ptr[name] += size_of // 2
        assert refused(call(lib.gsv_softmax_ce_forward, (7, classes), ptr, dtype,
                            (1 << 20, None))), name
    names = dict(scores=size, labels=8, opt=0, lse=8, count=4, grad_loss=4, grad_scores=size)
    for name, size_of in names.items():
        if name == "opt":
            continue
        ptr = {k: P for k in names}
        ptr[name] += size_of // 2
        assert refused(call(lib.gsv_softmax_ce_backward, (7, classes), ptr, dtype,
                            (None,))), name


@pytest.mark.parametrize("dtype,size", [(0, 4), (1, 2), (2, 2)])
@pytest.mark.parametrize("sizes", [(7, 20, 4), (20000, 9, 64), (3, 500, 64), (700, 500, 64)])
def test_linear_entries_refuse_misaligned_pointers(dtype, size, sizes):
    names = dict(features=size, weight=size, labels=8, opt=0, loss=4, state=16, ws=256)
    for name, size_of in names.items():
        if name == "opt":
            continue
        ptr = {k: P for k in names}
        ptr[name] += size_of // 2
        assert refused(call(lib.gsv_linear_ce_forward, sizes, ptr, dtype,
                            (1 << 40, None))), name
    names = dict(features=size, weight=size, labels=8, opt=0, state=16, grad_loss=4,
                 grad_features=size, grad_weight=size, ws=256)
    for name, size_of in names.items():
        if name == "opt":
            continue
        ptr = {k: P for k in names}
        ptr[name] += size_of // 2
        assert refused(call(lib.gsv_linear_ce_backward, sizes, ptr, dtype,
                            (1 << 40, None))), name


@pytest.mark.parametrize("cap", [1e-31, 1e-40, 1e31, float("nan")])
def test_caps_that_float32_cannot_divide_by(cap):
    """1 / cap would be infinite, and a score of 0 NaN."""
    p = ctypes.c_void_p(P)
    opt = CeOptions(-100, 0.0, cap, 0.0, 2)
    assert lib.gsv_softmax_ce_forward(7, 5, 0, p, p, opt, p, p, p, p, 1 << 20, None) == 1
    assert b"softcap" in lib.gsv_last_error()
    assert lib.gsv_linear_ce_forward(7, 5, 4, 0, p, p, p, opt, p, p, p, 1 << 40, None) == 1
    assert lib.gsv_linear_ce_workspace_bytes(7, 5, 4, 0, opt, 0) == 0


BACKWARD, STATE, ALIGNED, NO_STATE = 1, 2, 4, 8


def test_memory_of_the_linear_loss():
    """Nothing is asked for that the call does not use."""
    def ws(rows, V, D, dtype, call):
        return lib.gsv_linear_ce_workspace_bytes(rows, V, D, dtype, options(), call)

    # 256^3 voxels of few channels: 8 bytes a row of logsumexp, once
    n = 256 ** 3
    assert 8 * n <= lib.gsv_linear_ce_state_bytes(n, 20, 4, 0) < 8 * n + 4096
    assert ws(n, 20, 4, 0, STATE) < n
    assert 8 * n <= ws(n, 20, 4, 0, NO_STATE) < 9 * n
    # scores of few classes are the state's alone
    n = 1 << 23
    assert lib.gsv_linear_ce_state_bytes(n, 16, 64, 0) < (8 + 4 * 16) * n + 4096
    assert ws(n, 16, 64, 0, NO_STATE) < 9 * n and ws(n, 16, 64, 0, STATE) < n
    # a table of 1 GB that is read in place, rows too large to be kept
    n, V, D = 8192, 131072, 4096
    assert ws(n, V, D, 1, STATE | ALIGNED) < 2 * n * D + (32 << 20)
    assert ws(n, V, D, 1, BACKWARD | ALIGNED) < 2 * n * D + 4 * n * D + (600 << 20)
    # rows that are read in place
    assert ws(256 ** 3, 20, 64, 1, ALIGNED | NO_STATE) < 64 * 256 ** 3
    # a few rows, loss alone: no packed operands
    assert ws(4, 32768, 2048, 1, ALIGNED | NO_STATE) < 1 << 17
    # without the bits it is enough for either
    for sizes in ((700, 500, 64, 1), (3, 500, 64, 1), (20000, 9, 64, 0), (70000, 20, 4, 0),
                  (100000, 2000, 72, 2), (300, 2000, 264, 2), (300, 2000, 33, 0)):
        for call in (STATE, NO_STATE, ALIGNED, STATE | ALIGNED, NO_STATE | ALIGNED):
            assert 0 < ws(*sizes, call) <= ws(*sizes, 0)
        assert 0 < ws(*sizes, BACKWARD | ALIGNED) <= ws(*sizes, BACKWARD)


def test_memory_of_the_scores_loss():
    assert lib.gsv_softmax_ce_lse_bytes(0, 5) == 0 and lib.gsv_softmax_ce_lse_bytes(7, 0) == 0
    assert lib.gsv_softmax_ce_lse_bytes(10 ** 6, 1024) == 0
    assert lib.gsv_softmax_ce_lse_bytes(10 ** 6, 1025) == 8 * 10 ** 6
    p = ctypes.c_void_p(P)
    # needed where it is not empty
    assert lib.gsv_softmax_ce_forward(7, 1025, 0, p, p, options(), p, None, p, p, 1 << 20,
                                      None) == 1
    assert lib.gsv_softmax_ce_backward(7, 1025, 0, p, p, options(), None, p, p, p, None) == 1
