"""CPU: calls of nirrt_star_amd.nnops that are refused, or that are decided before anything is launched."""
import ctypes as C

import pytest
import torch


def test_cross_entropy_refuses_rows_of_more_than_4_mb():
    from nirrt_star_amd import nnops
    L = nnops._lib()
    p = C.c_void_p(4096)            # (never read: every call is refused)
    for dt, most in ((0, 1 << 20), (1, 1 << 21), (2, 1 << 21)):
        assert L.nirrt_nn_cross_entropy_workspace(dt, 9, 20, most) > 0 and L.nirrt_nn_cross_entropy_backward_workspace(dt, 9, 20, most) > 0
        k = most + 1
        assert L.nirrt_nn_cross_entropy_workspace(dt, 9, 20, k) == -1 and L.nirrt_nn_cross_entropy_backward_workspace(dt, 9, 20, k) == -1
        assert L.nirrt_nn_cross_entropy(dt, p, k, p, k, None, p, None, -100, p, p, p, 9, 20, k, p, None) == -1
        assert L.nirrt_nn_cross_entropy_backward(dt, p, k, p, k, None, p, None, -100, p, p, 0, None, p, p, None, 9, 20, k, p, None) == -1


def test_traces_are_refused():
    """(whatever the device: a trace would hold the allocation of the result and not what fills it)"""
    from torch.fx.experimental.proxy_tensor import make_fx
    from nirrt_star_amd import nnops
    x, w, t = torch.zeros(3, 4), torch.zeros(5, 4), torch.zeros(3, dtype=torch.int64)
    for call in (lambda x: nnops.linear_act(x, w), lambda x: nnops.linear_cross_entropy(x, w, t), lambda x: nnops.grad_norm([x]),
                 lambda x: nnops.clip_grad_norm_([x], 1.0)):
        with pytest.raises(RuntimeError, match="traced"):
            torch.jit.trace(call, (x,), check_trace=False)
        with pytest.raises(RuntimeError, match="traced"):
            make_fx(call)(x)


def test_dimensions_are_bounded():
    """kernels look a little past an index in 32 bits"""
    from nirrt_star_amd import nnops
    L = nnops._lib()
    p = C.c_void_p(4096)            # (never read)
    most = (1 << 31) - 4096
    assert nnops._DIM_MAX == most
    for dims in ((most, 1, 1), (1, most, 1), (1, 1, most)):
        m, n, k = dims
        assert L.nirrt_nn_linear_workspace(1, p, k, p, k, m, n, k) >= 0 and L.nirrt_nn_linear_backward_workspace(1, 1, p, k, p, k, p, n, m, n, k) >= 0
        m, n, k = (d + (d == most) for d in dims)
        assert L.nirrt_nn_linear_workspace(1, p, k, p, k, m, n, k) == -1 and L.nirrt_nn_linear_backward_workspace(1, 1, p, k, p, k, p, n, m, n, k) == -1
        assert L.nirrt_nn_linear(1, 0, p, k, p, k, None, None, n, p, n, None, m, n, k, p, None) == -1
        assert L.nirrt_nn_linear_backward(1, 0, p, k, p, k, None, p, n, p, p, p, m, n, k, p, None) == -1
    assert L.nirrt_nn_cross_entropy_workspace(1, 1 << 29, 8, 8) > 0 and L.nirrt_nn_cross_entropy_workspace(1, 1 << 29, 9, 8) == -1
    assert L.nirrt_nn_cross_entropy_workspace(1, most + 1, 2, 8) == -1 and L.nirrt_nn_cross_entropy_workspace(1, 8, most + 1, 8) == -1
