"""CPU tests of the class losses: refusals of the entry points before any
device work, workspace queries, and the float64 reference of the GPU tests
against torch and against differences."""
import ctypes

import pytest
import torch

from tests._class_ref import reference


def options(ignore=-100, smoothing=0.0, cap=0.0, z=0.0, reduction=2):
    from gs_voxelizer_b200._lib import CeOptions
    return CeOptions(ignore, smoothing, cap, z, reduction)


def test_python_refuses_host_tensors():
    from gs_voxelizer_b200.losses import linear_cross_entropy, softmax_cross_entropy
    y = torch.zeros(3, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="scores must be a CUDA tensor"):
        softmax_cross_entropy(torch.zeros(3, 4), y)
    with pytest.raises(RuntimeError, match="features must be a CUDA tensor"):
        linear_cross_entropy(torch.zeros(3, 4), torch.zeros(5, 4), y)


def test_c_entries_refuse_bad_arguments():
    from gs_voxelizer_b200._lib import lib
    p = ctypes.c_void_p(256)

    def soft(rows=4, V=5, dtype=0, opt=options(), scores=p, ws=p, ws_bytes=1 << 20):
        return lib.gsv_softmax_ce_forward(rows, V, dtype, scores, p, opt, p, p, p, ws,
                                          ws_bytes, None)

    def lin(rows=4, V=5, D=6, dtype=1, opt=options(), weight=p, ws=p, ws_bytes=1 << 40,
            state=p):
        return lib.gsv_linear_ce_forward(rows, V, D, dtype, p, weight, p, opt, p, state, ws,
                                         ws_bytes, None)

    def back(ws_bytes=1 << 40, grad=p, ws=p):
        return lib.gsv_linear_ce_backward(4, 5, 6, 1, p, p, p, options(), p, grad, p, p, ws,
                                          ws_bytes, None)

    for fn in (soft, lin):
        assert fn(rows=0) == 1 and b"positive" in lib.gsv_last_error()
        assert fn(V=0) == 1
        assert fn(rows=2 ** 31) == 4
        assert fn(V=2 ** 24 + 1) == 4
        assert fn(dtype=3) == 1 and fn(dtype=-1) == 1
        assert fn(opt=None) == 1
        for bad in (options(smoothing=1.0), options(smoothing=-0.5), options(cap=-1.0),
                    options(cap=float("nan")), options(z=float("inf")), options(reduction=3)):
            assert fn(opt=bad) == 1
        assert fn(ws=None) == 3
    assert soft(scores=None) == 1
    assert soft(ws_bytes=7) == 3 and b"workspace" in lib.gsv_last_error()
    assert lin(weight=None) == 1
    assert lin(D=0) == 1 and lin(D=2 ** 20 + 1) == 4
    assert lin(ws_bytes=255) == 3
    assert lin(ws=ctypes.c_void_p(264)) == 1 and b"aligned" in lib.gsv_last_error()
    assert lin(state=ctypes.c_void_p(260)) == 1
    assert back(ws_bytes=255) == 3 and back(grad=None) == 1
    assert back(ws=ctypes.c_void_p(264)) == 1


def test_workspace_queries():
    from gs_voxelizer_b200._lib import lib
    assert lib.gsv_softmax_ce_workspace_bytes(0, 5) == 0
    assert lib.gsv_softmax_ce_workspace_bytes(1000, 4) >= 8 * 4
    assert lib.gsv_softmax_ce_workspace_bytes(1000, 5000) >= 8 * 1000
    assert lib.gsv_linear_ce_state_bytes(0, 10, 10, 0) == 0
    assert lib.gsv_linear_ce_state_bytes(1000, 10, 10, 3) == 0
    assert lib.gsv_linear_ce_state_bytes(1000, 10, 4, 0) >= 8 * 1000
    # the packed operands are kept up to 16 MB each
    small = lib.gsv_linear_ce_state_bytes(8192, 1024, 64, 1)
    assert small >= 2 * 64 * (8192 + 1024)
    assert lib.gsv_linear_ce_state_bytes(8192, 131072, 4096, 1) < 32 * 8192
    assert lib.gsv_linear_ce_workspace_bytes(10, 0, 4, 1, options(), 0) == 0
    # far below the scores: a long batch over a large vocabulary
    n, V, D = 65536, 131072, 1024
    for backward in (0, 1):
        b = lib.gsv_linear_ce_workspace_bytes(n, V, D, 1, options(), backward)
        assert 0 < b < n * V * 2 // 4


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_reference_against_torch(reduction):
    g = torch.Generator().manual_seed(1)
    s = torch.randn(40, 9, generator=g, dtype=torch.float64, requires_grad=True)
    y = torch.randint(0, 9, (40,), generator=g)
    y[::7] = -100
    want = torch.nn.functional.cross_entropy(s, y, reduction=reduction, label_smoothing=0.2)
    up = torch.rand(want.shape, generator=g, dtype=torch.float64)
    (gw,) = torch.autograd.grad(want, s, up)
    ref = reference(s.detach(), y, smoothing=0.2, reduction=reduction, upstream=up)
    assert torch.allclose(ref["loss"], want.detach(), rtol=1e-12)
    assert torch.allclose(ref["ds"], gw, rtol=1e-10, atol=1e-14)


def test_reference_gradient_against_differences():
    g = torch.Generator().manual_seed(2)
    s = 3 * torch.randn(6, 7, generator=g, dtype=torch.float64)
    y = torch.tensor([0, 3, -100, 6, 2, 2])
    opt = dict(smoothing=0.1, softcap=4.0, z_loss=0.05, reduction="sum")
    ds = reference(s, y, upstream=torch.ones(()), **opt)["ds"]
    h = 1e-6
    for i in range(6):
        for j in range(7):
            e = torch.zeros_like(s)
            e[i, j] = h
            d = (reference(s + e, y, **opt)["loss"] - reference(s - e, y, **opt)["loss"]) / (2 * h)
            assert float(ds[i, j]) == pytest.approx(float(d), rel=1e-6, abs=1e-8)
