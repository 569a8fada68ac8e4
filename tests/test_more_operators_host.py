"""Refusals of the embedding, the gradients' norm and linear attention that need no
GPU: nothing is launched, and no array is looked at, before sizes, types and
settings are in order."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from test_operators_host import lib  # noqa: F401

torch = pytest.importorskip("torch")

X = np.zeros(64, np.float64)
A = X.ctypes.data
I64, V = ctypes.c_int64, ctypes.c_void_p


def test_capability_bit(lib):  # noqa: F811
    assert lib.sn_abi_caps() & (1 << 12)


@pytest.mark.parametrize("change", [{"bits": 16}, {"n": -1}, {"n": 1 << 31}, {"n": (1 << 31) - 1}, {"V": -1}, {"V": (1 << 31) - 1}, {"D": -1},
                                    {"D": (1 << 30) + 1}, {"D": (1 << 22) + 1}, {"ld": -1}, {"dtype": 3}, {"scale": float("nan")},
                                    {"scale": float("inf")}, {"tokens": None}, {"W": None}, {"out": None}])
def test_embedding(lib, change):  # noqa: F811
    a = dict(tokens=A, bits=64, n=4, W=A, ld=8, V=8, D=8, dtype=0, scale=1.0, out=A, stream=None)
    assert lib.sn_abi_embedding(*{**a, "n": 0}.values()) == 0
    assert lib.sn_abi_embedding(*{**a, "D": 0}.values()) == 0
    assert lib.sn_abi_embedding(*{**a, **change}.values()) == -1


@pytest.mark.parametrize("change", [{"bits": 8}, {"n": -1}, {"V": -2}, {"D": -1}, {"ld": -1}, {"dtype": -1},
                                    {"scale": float("nan")}, {"tokens": None}, {"dout": None}, {"dW": None}])
def test_embedding_bwd(lib, change):  # noqa: F811
    a = dict(tokens=A, bits=32, n=4, dout=A, ld=8, V=8, D=8, dtype=0, scale=1.0, dW=A, ws=None, bytes=0, stream=None)
    assert lib.sn_abi_embedding_bwd(*{**a, "V": 0}.values()) == 0
    assert lib.sn_abi_embedding_bwd(*{**a, **change}.values()) == -1
    assert lib.sn_abi_embedding_bwd_ws(-1, 8, 8) == lib.sn_abi_embedding_bwd_ws(4, 8, -8) == -1
    assert lib.sn_abi_embedding_bwd_ws(0, 8, 8) == 0 < lib.sn_abi_embedding_bwd_ws(4, 8, 8)


@pytest.mark.parametrize("change", [{"count": -1}, {"grads": None}, {"sizes": None}, {"dtypes": None}, {"max": -1.0},
                                    {"max": float("nan")}, {"sizes": (I64 * 1)(-4)}, {"sizes": (I64 * 1)(1 << 47)},
                                    {"dtypes": (ctypes.c_int32 * 1)(7)}, {"grads": (V * 1)(None)}, {"ws": None},
                                    {"bytes": 7}])
def test_gradient_norm(lib, change):  # noqa: F811
    a = dict(count=1, grads=(V * 1)(A), sizes=(I64 * 1)(4), dtypes=(ctypes.c_int32 * 1)(0), max=1.0, norm=A, factor=A, ws=A,
             bytes=8, stream=None)
    for f in (lib.sn_abi_grad_norm, lib.sn_abi_clip_grads):
        assert f(*{**a, **change}.values()) == -1
    assert lib.sn_abi_grad_norm_ws(1, a["sizes"]) == 8 and lib.sn_abi_grad_norm_ws(0, None) == 0
    assert lib.sn_abi_grad_norm_ws(-1, None) == lib.sn_abi_grad_norm_ws(1, None) == -1


class Call(ctypes.Structure):
    _fields_ = [(n, V) for n in ("q", "k", "v", "log_decay", "state", "lengths")] + \
        [(n + "_stride", I64 * 3) for n in ("q", "k", "v", "log_decay")] + \
        [(n, ctypes.c_int32) for n in ("dtype", "B", "T", "H", "Hk", "dk", "dv")] + [("scale", ctypes.c_float)]


def call(**change):
    c = Call(q=A, k=A, v=A, log_decay=A, dtype=0, B=1, T=2, H=4, Hk=2, dk=8, dv=8, scale=1.0)
    for n, v in change.items():
        setattr(c, n, v)
    return c


SIZES = [{"dtype": 5}, {"B": -1}, {"T": -1}, {"H": 0}, {"Hk": 0}, {"Hk": 3}, {"dk": 0}, {"dk": 129}, {"dv": 0}, {"dv": 129},
         {"T": (1 << 31) - 1}, {"B": 1 << 30}, {"scale": float("nan")}, {"scale": float("inf")}]


@pytest.mark.parametrize("change", SIZES + [{"q": None}, {"k": None}, {"v": None}, {"log_decay": None}])
def test_linear_attention(lib, change):  # noqa: F811
    stride = (I64 * 3)(1, 1, 1)
    forward = lambda c: lib.sn_abi_linear_attention(ctypes.byref(c), A, A, None, 0, None)  # noqa: E731
    back = lambda c: lib.sn_abi_linear_attention_bwd(ctypes.byref(c), A, stride, None, A, A, A, None, 0, None, None, 0, None)  # noqa: E731
    step = lambda c: lib.sn_abi_linear_attention_step(ctypes.byref(c), A, 256, A, None)  # noqa: E731
    assert forward(call(B=0)) == back(call(B=0)) == step(call(B=0, T=1)) == 0
    assert forward(call(**change)) == back(call(**change)) == -1
    assert step(call(**{"T": 1, **change})) == -1 and step(call()) == -1  # one token at a time
    ws = lambda c, *a: lib.sn_abi_linear_attention_ws(ctypes.byref(c), *a)  # noqa: E731
    if change in SIZES:
        assert ws(call(**change), 0, 0) == ws(call(**change), 1, 1) == -1
    assert ws(call(B=0), 1, 1) == 0 < ws(call(), 0, 0) < ws(call(), 1, 0) < ws(call(), 1, 1)


def test_linear_attention_pointers(lib):  # noqa: F811
    c, stride = ctypes.byref(call()), (I64 * 3)(1, 1, 1)
    assert lib.sn_abi_linear_attention(None, A, A, None, 0, None) == -1
    assert lib.sn_abi_linear_attention(c, None, A, None, 0, None) == -1
    assert lib.sn_abi_linear_attention(c, A, None, None, 0, None) == -1
    for i in (1, 2, 4, 5, 6):
        a = [c, A, stride, None, A, A, A, None, 0, None, None, 0, None]
        a[i] = None
        assert lib.sn_abi_linear_attention_bwd(*a) == -1
    one = ctypes.byref(call(T=1, B=2))
    assert lib.sn_abi_linear_attention_step(one, None, 256, A, None) == -1
    assert lib.sn_abi_linear_attention_step(one, A, 256, None, None) == -1
    assert lib.sn_abi_linear_attention_step(one, A, 255, A, None) == -1  # states overlap


def test_python_refusals_without_a_gpu(lib):  # noqa: F811
    from sunnynet_b200 import kernels
    x = torch.zeros(2, 5, 2, 8)
    v, g = torch.zeros(2, 5, 4, 16), torch.zeros(2, 5, 4)
    for bad, error, text in (
            (lambda: kernels.linear_attention(x, x, v, g), ValueError, "one GPU"),
            (lambda: kernels.linear_attention(x, x[:, :4], v, g), ValueError, "dk"),
            (lambda: kernels.linear_attention(x, x, v[:, :, :3], g), ValueError, "multiple"),
            (lambda: kernels.linear_attention(x.double(), x.double(), v.double(), g), TypeError, "float32"),
            (lambda: kernels.linear_attention(x, x, None, g), TypeError, "tensors"),
            (lambda: kernels.linear_attention(x, x, v, g, scale="a"), TypeError, None),
            (lambda: kernels.linear_attention_step(x, x, v, g, v), ValueError, "Hk"),
            (lambda: kernels.linear_attention(x[:, 0], x[:, 0], v[:, 0], g[:, 0]), ValueError, "T, Hk"),
            (lambda: kernels.linear_attention_step(x[:, 0], x[:, 0], v[:, 0], g[:, 0], v), ValueError, "one GPU"),
            (lambda: kernels.embedding(torch.zeros(3).long(), v[0, 0]), ValueError, "GPU"),
            (lambda: kernels.embedding(3, v[0, 0]), TypeError, "tensors"),
            (lambda: kernels.grad_norm([]), ValueError, "no gradients"),
            (lambda: kernels.grad_norm([x]), ValueError, "one GPU"),
            (lambda: kernels.grad_norm([x.long()]), TypeError, "float32"),
            (lambda: kernels.grad_norm([1.0]), TypeError, "tensors"),
            (lambda: kernels.clip_grads([x], -1.0), ValueError, "negative"),
            (lambda: kernels.clip_grads([x], float("nan")), ValueError, "negative")):
        with pytest.raises(error, match=text):
            bad()


def test_tensors_with_a_tangent(lib):  # noqa: F811
    import torch.autograd.forward_ad as fwd

    from sunnynet_b200 import kernels
    x, v, g = torch.randn(1, 2, 1, 8), torch.randn(1, 2, 1, 8), torch.zeros(1)
    with fwd.dual_level():
        d = fwd.make_dual(x, torch.ones_like(x))
        with pytest.raises(RuntimeError, match="forward-mode"):
            kernels.linear_attention(d, x, v, g)
        with pytest.raises(RuntimeError, match="forward-mode"):
            kernels.linear_attention_step(x[:, 0], d[:, 0], v[:, 0], g, torch.zeros(1, 1, 8, 8))


def test_optimiser_refuses_a_negative_norm():
    from sunnynet_b200.optim import AdamW
    with pytest.raises(ValueError, match="max_norm"):
        AdamW([torch.nn.Parameter(torch.zeros(3))], max_norm=-1.0)


def test_a_copy_of_the_optimiser_keeps_its_bound():
    import copy

    from sunnynet_b200.optim import AdamW
    p = torch.nn.Parameter(torch.zeros(3))
    assert copy.deepcopy(AdamW([p], max_norm=2.0)).max_norm == 2.0
    assert copy.deepcopy(AdamW([p])).max_norm is None
    old = AdamW.__new__(AdamW)  # as one of before the argument unpickles
    old.__setstate__({k: v for k, v in AdamW([p]).__getstate__().items() if k != "max_norm"})
    assert old.max_norm is None and old.grad_norm is None


def text(lib):  # noqa: F811
    buf = ctypes.create_string_buffer(512)
    lib.sn_abi_last_error(buf, 512)
    return buf.value


def empty_and_refused(lib):  # noqa: F811
    """Calls that return before they look at an array, with what each returns."""
    null, stride = ctypes.c_void_p(), (I64 * 3)(1, 1, 1)
    adamw = lambda count, step: (count, null, null, null, null, null, null, null, 0, 0, 32, step, None, 1e-3, None,  # noqa: E731
                                 0.9, 0.999, 1e-8, 0.0)
    norm = lambda dtype, rows: (A, 8, None, None, A, None, None, dtype, 0, rows, 8, 1e-5, None)  # noqa: E731
    norm_bwd = lambda dtype: (A, 8, A, 8, None, A, A, None, None, None, None, 0, dtype, 0, 4, 8, None)  # noqa: E731
    draw = lambda B, V_: (A, V_, 0, A, 0, None, 1.0, None, 0, None, 1.0, None, 0.0, B, V_, A, None)  # noqa: E731
    back = lambda c: lib.sn_abi_linear_attention_bwd(c, A, stride, None, A, A, A, None, 0, None, None, 0, None)  # noqa: E731
    of = lambda **c: ctypes.byref(call(**c))  # noqa: E731
    return {
        "embedding, empty": lambda: lib.sn_abi_embedding(A, 64, 0, A, 8, 8, 8, 0, 1.0, A, None),
        "embedding, refused": lambda: lib.sn_abi_embedding(A, 64, 4, A, 8, 8, 8, 9, 1.0, A, None),
        "embedding_bwd, empty": lambda: lib.sn_abi_embedding_bwd(A, 64, 4, A, 8, 0, 8, 0, 1.0, A, None, 0, None),
        "embedding_bwd, refused": lambda: lib.sn_abi_embedding_bwd(A, 64, 4, A, 8, 8, 8, 9, 1.0, A, None, 0, None),
        "linear_attention, empty": lambda: lib.sn_abi_linear_attention(of(B=0), A, A, None, 0, None),
        "linear_attention, refused": lambda: lib.sn_abi_linear_attention(of(dtype=9), A, A, None, 0, None),
        "linear_attention_bwd, empty": lambda: back(of(B=0)),
        "linear_attention_bwd, refused": lambda: back(of(dtype=9)),
        "linear_attention_step, empty": lambda: lib.sn_abi_linear_attention_step(of(B=0, T=1), A, 256, A, None),
        "linear_attention_step, refused": lambda: lib.sn_abi_linear_attention_step(of(), A, 256, A, None),
        "grad_norm, refused": lambda: lib.sn_abi_grad_norm(1, None, None, None, 1.0, A, A, A, 8, None),
        "clip_grads, refused": lambda: lib.sn_abi_clip_grads(1, None, None, None, 1.0, A, A, A, 8, None),
        "adamw_step, refused": lambda: lib.sn_abi_adamw_step(*adamw(1, 1), None),
        "adamw_step_scaled, refused": lambda: lib.sn_abi_adamw_step_scaled(*adamw(0, 0), None, None),
        "layer_norm, empty": lambda: lib.sn_abi_layer_norm(*norm(0, 0)),
        "layer_norm, refused": lambda: lib.sn_abi_layer_norm(*norm(9, 1)),
        "layer_norm_bwd, empty": lambda: lib.sn_abi_layer_norm_bwd(*norm_bwd(0)),
        "layer_norm_bwd, refused": lambda: lib.sn_abi_layer_norm_bwd(*norm_bwd(9)),
        "sample, empty": lambda: lib.sn_abi_sample(*draw(0, 8)),
        "sample, refused": lambda: lib.sn_abi_sample(*draw(1, 0)),
    }


def test_what_a_caller_vouches_for_ends_with_its_next_call(lib):  # noqa: F811
    """sn_abi_arrays_on counts for one call, one that does nothing or is refused too: the call after it asks for
    its arrays, and refuses these, which lie in host memory."""
    asks = lambda: lib.sn_abi_embedding(A, 64, 4, A, 8, 8, 8, 0, 1.0, A, None)  # noqa: E731
    rc, said = asks(), text(lib)
    assert rc != 0
    for name, f in empty_and_refused(lib).items():
        lib.sn_abi_arrays_on(0)
        assert (f() == 0) == name.endswith("empty"), name
        assert (asks(), text(lib)) == (rc, said), name


def test_an_error_names_its_operator(lib):  # noqa: F811
    from sunnynet_b200 import kernels
    calls, x = kernels._torch_calls(), torch.zeros(2, 5, 2, 8)
    for bad, name in ((lambda: calls.layer_norm(3, None, None, 1e-5), "layer_norm"),
                      (lambda: calls.layer_norm(x, 3, None, 1e-5), "layer_norm"),
                      (lambda: kernels.embedding(x, 3), "embedding"),
                      (lambda: kernels.linear_attention(x, 3, x, x), "linear_attention"),
                      (lambda: kernels.linear_attention(x, None, x, x), "linear_attention"),
                      (lambda: kernels.linear_attention_step(x, x, x, x, 3), "linear_attention_step"),
                      (lambda: kernels.linear_attention_step(x, x, None, x, x), "linear_attention_step"),
                      (lambda: kernels.grad_norm([3]), "grad_norm"), (lambda: kernels.clip_grads([3], 1.0), "clip_grads")):
        with pytest.raises(TypeError, match="^" + name + ": tensors are wanted"):
            bad()
