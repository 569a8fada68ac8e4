"""Refusals of the enqueue-only operators that need no GPU: nothing is launched
and no array is looked at before the dimensions, types and settings are in
order."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def lib():
    from sunnynet_b200 import _lib, build
    if not _lib.LIB_PATH.exists():
        build.build()
    return _lib.load()


X = np.zeros(64, np.float64)
A = X.ctypes.data


def test_capability_bits(lib):
    caps = lib.sn_abi_caps()
    assert caps & (1 << 10) and caps & (1 << 11)


@pytest.mark.parametrize("change", [{"dtype": 3}, {"wdtype": 1}, {"rows": -1}, {"D": 0}, {"ldx": 7},
                                    {"eps": -1.0}, {"eps": float("nan")}, {"x": None}, {"y": None},
                                    {"rows": 1 << 31}])
def test_layer_norm(lib, change):
    a = dict(x=A, ldx=8, w=None, b=None, y=A, mean=None, rstd=None, dtype=0, wdtype=0, rows=4, D=8,
             eps=1e-5, stream=None)
    assert lib.sn_abi_layer_norm(*{**a, "rows": 0}.values()) == 0
    assert lib.sn_abi_layer_norm(*{**a, **change}.values()) == -1


@pytest.mark.parametrize("change", [{"dtype": -1}, {"wdtype": 2}, {"rows": -1}, {"D": -5}, {"lddy": 7},
                                    {"ldx": 0}, {"dy": None}, {"x": None}, {"mean": None}, {"rstd": None}])
def test_layer_norm_bwd(lib, change):
    a = dict(dy=A, lddy=8, x=A, ldx=8, w=None, mean=A, rstd=A, dx=A, dw=None, db=None, ws=None, n=0,
             dtype=0, wdtype=0, rows=4, D=8, stream=None)
    assert lib.sn_abi_layer_norm_bwd(*{**a, "dx": None}.values()) == 0  # nothing is wanted
    assert lib.sn_abi_layer_norm_bwd(*{**a, **change}.values()) == -1
    assert lib.sn_abi_layer_norm_bwd_ws(-1, 8, 0) == lib.sn_abi_layer_norm_bwd_ws(4, 8, 9) == 0
    assert lib.sn_abi_layer_norm_bwd_ws(4, 8, 0) > 0


@pytest.mark.parametrize("change", [{"dtype": 7}, {"grad": -2}, {"bits": 16}, {"step": 0}, {"count": -1},
                                    {"b1": 1.0}, {"b2": -0.1}, {"b2": float("nan")}, {"eps": -1e-8},
                                    {"eps": float("inf")}, {"lr": float("nan")}, {"wd": float("inf")},
                                    {"params": None}, {"sizes": None}, {"bits": 8},
                                    {"sizes": (ctypes.c_int64 * 1)(-4)},
                                    {"params": (ctypes.c_void_p * 1)(None)}])
def test_adamw_step(lib, change):
    one = (ctypes.c_void_p * 1)(A)
    a = dict(count=1, params=one, grads=one, avg=one, sq=one, ms=None, vs=None,
             sizes=(ctypes.c_int64 * 1)(4), dtype=0, grad=0, bits=32, step=1, step_dev=None, lr=1e-3,
             lr_dev=None, b1=0.9, b2=0.99, eps=1e-8, wd=0.1, stream=None)
    assert lib.sn_abi_adamw_step(*{**a, "count": 0}.values()) == 0
    assert lib.sn_abi_adamw_step(*{**a, "sizes": (ctypes.c_int64 * 1)(0)}.values()) == 0
    assert lib.sn_abi_adamw_step(*{**a, **change}.values()) == -1


@pytest.mark.parametrize("change", [{"dtype": 5}, {"B": -1}, {"V": 0}, {"ld": 7}, {"t0": float("inf")},
                                    {"t0": float("nan")}, {"q0": 1.5}, {"q0": float("nan")},
                                    {"p0": float("nan")}, {"logits": None}, {"u": None}, {"out": None},
                                    {"B": 1 << 30}])
def test_sample(lib, change):
    a = dict(logits=A, ld=8, dtype=0, u=A, wide=0, t=None, t0=1.0, k=None, k0=0, p=None, p0=1.0, q=None,
             q0=0.0, B=2, V=8, out=A, stream=None)
    assert lib.sn_abi_sample(*{**a, "B": 0}.values()) == 0
    assert lib.sn_abi_sample(*{**a, **change}.values()) == -1


def test_python_refusals_before_the_library():
    from sunnynet_b200 import kernels
    from sunnynet_b200.sampling import sample
    x = torch.zeros(2, 8)
    with pytest.raises(ValueError, match="GPU"):
        sample(x, torch.zeros(2))
    with pytest.raises(ValueError, match="GPU"):
        kernels.adamw_step([x], [x], [x], [x], 1)
    with pytest.raises(ValueError, match="length"):
        kernels.adamw_step([x], [], [x], [x], 1)
    with pytest.raises(ValueError):
        kernels.layer_norm(torch.zeros(3, 0))


def test_lists_of_tensors_are_refused_before_a_gpu_is_asked(lib):
    from sunnynet_b200 import kernels
    read = kernels._torch_calls().read
    a, f = [torch.zeros(3), torch.zeros(0)], torch.float32
    for bad, error, text in (
            (lambda: read((a, a), (f, f), 256), ValueError, "one GPU"),
            (lambda: read((a, a[:1]), (f, f), 256), ValueError, "one GPU|length"),
            (lambda: read((a,), (torch.float64,), 256), TypeError, "float64"),
            (lambda: read(([1.0],), (f,), 256), TypeError, "tensors"),
            (lambda: read((iter(a),), (f,), 256), TypeError, "lists"),
            (lambda: read((a,), (f, f), 256), ValueError, "dtype"),
            (lambda: read((a,), (3,), 256), TypeError, "dtype"),
            (lambda: kernels._torch_calls().layer_norm(1, None, None, 0.1), TypeError, "tensors")):
        with pytest.raises(error, match=text):
            bad()
