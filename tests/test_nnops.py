"""CPU: what nirrt_star_amd.nnops refuses before anything is launched, and its C entry points' checks (include/nirrt_nnops.h)."""
import ctypes as C
import os
import re

import pytest
import torch

from conftest import ROOT


def test_library_exports_the_header():
    from nirrt_star_amd import _hip, build
    build.build()
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "nirrt_nnops.h")).read(), flags=re.S)
    names = sorted(set(re.findall(r"\b(nirrt_nn_[a-z0-9_]+)\s*\(", text)))
    assert len(names) == 11
    for n in names:
        assert hasattr(_hip.load(), n), n


def test_tensor_record_matches_the_header(tmp_path):
    import subprocess
    from nirrt_star_amd import nnops
    src = tmp_path / "t.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "nirrt_nnops.h"\nint main(void) { printf("%zu %zu %zu %zu %zu\\n", sizeof(nirrt_nn_tensor), '
                   'offsetof(nirrt_nn_tensor, out), offsetof(nirrt_nn_tensor, n), offsetof(nirrt_nn_tensor, dtype), offsetof(nirrt_nn_tensor, out_dtype)); return 0; }\n')
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "t")])
    size, out, n, dt, odt = (int(v) for v in subprocess.check_output([str(tmp_path / "t")], text=True).split())
    f = nnops._TENSOR.fields
    assert nnops._TENSOR.itemsize == size and (f["out"][1], f["n"][1], f["dtype"][1], f["out_dtype"][1]) == (out, n, dt, odt)


def test_cpu_tensors_are_refused():
    from nirrt_star_amd import nnops
    x, w, t = torch.zeros(3, 4), torch.zeros(2, 4), torch.zeros(3, dtype=torch.int64)
    for call in (lambda: nnops.linear_act(x, w), lambda: nnops.linear_cross_entropy(x, w, t), lambda: nnops.grad_norm([x]),
                 lambda: nnops.clip_grad_norm_([x], 1.0)):
        with pytest.raises(RuntimeError, match="CPU tensor"):
            call()


def test_arguments_without_a_device():
    from nirrt_star_amd import nnops
    x, w = torch.zeros(3, 4), torch.zeros(2, 4)
    with pytest.raises(ValueError, match="activation"):
        nnops.linear_act(x, w, activation="tanh")
    with pytest.raises(ValueError, match="reduction"):
        nnops.linear_cross_entropy(x, w, torch.zeros(3, dtype=torch.int64), reduction="avg")
    for bad in (-1.0, float("nan")):
        with pytest.raises(ValueError, match="max_norm"):
            nnops.clip_grad_norm_([x], bad)
    with pytest.raises(ValueError, match="no tensors"):
        nnops.grad_norm([None])
    with pytest.raises(ValueError, match="outputs"):
        nnops.clip_grad_norm_([x, None], 1.0, out=[x, x])


def test_c_entry_points_refuse_bad_arguments():
    """none of these reaches a launch: they need no GPU"""
    from nirrt_star_amd import nnops
    L = nnops._lib()
    p = C.c_void_p(4096)            # (never read: every call is refused by its other arguments)
    assert L.nirrt_nn_linear_workspace(3, p, 1, p, 1, 1, 1, 1) == -1 and L.nirrt_nn_linear_workspace(0, p, 1, p, 1, -1, 1, 1) == -1
    assert L.nirrt_nn_linear_workspace(0, p, 1, p, 1, 1 << 31, 1, 1) == -1
    assert L.nirrt_nn_linear(7, 0, p, 4, p, 4, None, None, 4, p, 4, None, 4, 4, 4, p, None) == -1       # element type
    assert L.nirrt_nn_linear(0, 4, p, 4, p, 4, None, None, 4, p, 4, None, 4, 4, 4, p, None) == -1       # activation
    assert L.nirrt_nn_linear(0, 0, p, 3, p, 4, None, None, 4, p, 4, None, 4, 4, 4, p, None) == -1       # row stride below the row
    assert L.nirrt_nn_linear(0, 0, None, 4, p, 4, None, None, 4, p, 4, None, 4, 4, 4, p, None) == -1
    assert L.nirrt_nn_linear(0, 0, p, 4, p, 4, None, p, 3, p, 4, None, 4, 4, 4, p, None) == -1          # residual stride
    assert L.nirrt_nn_linear(0, 0, p, 4, p, 4, None, None, 4, p, 4, None, 0, 4, 4, None, None) == 0     # nothing to do
    big = 1 << 16
    assert L.nirrt_nn_linear_workspace(0, p, big, p, big, 64, 64, big) > 0
    assert L.nirrt_nn_linear(0, 0, p, big, p, big, None, None, 64, p, 64, None, 64, 64, big, None, None) == -1   # workspace missing
    for m, n, k in ((0, 4, 4), (4, 0, 4), (4, 4, 0), (0, 0, 0)):                                         # empty sizes have a size too
        assert L.nirrt_nn_linear_workspace(0, p, 4, p, 4, m, n, k) == 0 and L.nirrt_nn_linear_backward_workspace(0, 1, p, 4, p, 4, p, 4, m, n, k) >= 0
        assert L.nirrt_nn_cross_entropy_workspace(0, m, 4, k) >= 0 and L.nirrt_nn_cross_entropy_backward_workspace(0, m, 4, k) >= 0
    assert L.nirrt_nn_linear_backward(0, 2, p, 4, p, 4, None, p, 4, p, p, p, 4, 4, 4, p, None) == -1    # z missing
    assert L.nirrt_nn_cross_entropy_workspace(0, 4, 0, 4) == -1                                          # no classes
    assert L.nirrt_nn_cross_entropy(0, p, 4, p, 4, None, None, None, -100, p, p, p, 4, 4, 4, p, None) == -1     # targets missing
    assert L.nirrt_nn_cross_entropy_backward(0, p, 4, p, 4, None, p, None, -100, p, p, 2, None, p, p, None, 4, 4, 4, p, None) == -1
    assert L.nirrt_nn_norm(None, 1, p, p, None) == -1 and L.nirrt_nn_norm_workspace(None, -1) == -1
    import numpy as np
    tab = np.zeros(1, dtype=nnops._TENSOR)
    tab["n"] = 5
    assert L.nirrt_nn_norm(tab.ctypes.data, 1, p, p, None) == -1                                         # no data
    tab["data"], tab["dtype"] = 4096, 9
    assert L.nirrt_nn_norm(tab.ctypes.data, 1, p, p, None) == -1
    tab["dtype"] = 0
    assert L.nirrt_nn_scale_by_norm(tab.ctypes.data, 1, p, 1.0, None) == -1                              # no output
    tab["out"] = 4096
    assert L.nirrt_nn_scale_by_norm(tab.ctypes.data, 1, p, float("nan"), None) == -1
