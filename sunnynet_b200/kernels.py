"""The reference's hand-written kernels module on a B200: the loader and the
torch autograd operators of ``sunnynet/kernels`` (``__init__.py``,
``core_auto.py``, ``scan_auto.py``), backed by libsunnynet_cuda.so.

Same names and argument meaning, so training code switches by import:
``load_kernel`` / ``load_scan_kernel`` return the library with the argtypes
set; ``CoreCUDA`` (the reference's ``CoreAVX2``) takes q (B,T,2D) = [u_raw |
gate], delta (D,), s0 (B,D) and returns (u, states); ``ScanCUDA`` (the
reference's ``ScanAVX2``) takes u, p (B,T,N), s0 (B,N) and returns the states;
``step_core`` and ``dw_step`` are the decode-time single steps. Tensors may be
on the GPU (then the kernels read them in place, on torch's current stream)
or on the host (staged through device memory). There is no CPU fallback.

Beside them stand the two other operators of a training step, which the
reference leaves to torch: ``layer_norm`` (its CenteredScaleNorm with
eps = s_min^2 + 1e-5) with its gradients, and ``adamw_step``, one AdamW update
of all of a model's tensors with states in 32 or 8 bits
(``sunnynet_b200.optim.AdamW`` keeps the states). These only enqueue on
torch's current stream of their tensors' device, so a training step of them
can be captured into a CUDA graph.
"""
from __future__ import annotations

import ctypes

from . import _lib
from ._lib import check, current_stream, dtype_code, ptr
from .runtime import bind_stream, load_runtime

__all__ = ["load_kernel", "load_scan_kernel", "kernel_available", "set_kernel_threads",
           "CoreCUDA", "core_forward", "step_core", "dw_step", "ScanCUDA", "scan_auto",
           "layer_norm", "adamw_step", "STATE_BLOCK"]

_MAX_WIDTH = (1 << 31) - (1 << 14)  # of layer_norm's rows
STATE_BLOCK = 256  # values of an 8-bit optimiser state that share one scale


def load_kernel(force_rebuild: bool = False):
    """The library, with the argtypes of the kernels module set."""
    return load_runtime(force_rebuild)


def load_scan_kernel(force_rebuild: bool = False):
    return load_kernel(force_rebuild)


def kernel_available() -> bool:
    return _lib.LIB_PATH.exists()


def set_kernel_threads(n: int) -> None:
    """Kept for the reference's interface; the GPU ignores host thread counts."""
    load_kernel().sn_set_threads(int(n))


def _call(name: str, *args) -> None:
    """Call a void entry point; its failure is the message it leaves."""
    lib = load_kernel()
    lib.sn_abi_clear_error()
    getattr(lib, name)(*args)
    msg = _lib.last_error()
    if msg:
        raise _lib.SnError(-1, f"{name}: {msg}")


def _f32(t):
    return t.contiguous().float()


class CoreCUDA:
    """Fused competition gate + decay gate + scan as an autograd operator:
    (q, delta, s0) -> (u, states) (reference core_auto.CoreAVX2)."""

    @staticmethod
    def apply(q, delta, s0):
        return _core_fn().apply(q, delta, s0)


_CORE = None


def _core_fn():
    global _CORE
    if _CORE is not None:
        return _CORE
    import torch

    class _Core(torch.autograd.Function):
        @staticmethod
        def forward(ctx, q, delta, s0):
            B, T, D2 = q.shape
            D = D2 // 2
            q_c, delta_c, s0_c = _f32(q), _f32(delta), _f32(s0)
            states = torch.empty(B, T, D, dtype=torch.float32, device=q.device)
            u = torch.empty_like(states)
            p = torch.empty_like(states)
            bind_stream(q_c)
            _call("core_fwd_f32", ptr(q_c), ptr(delta_c), ptr(s0_c), ptr(states), ptr(u),
                  ptr(p), B, T, D)
            ctx.save_for_backward(q_c, delta_c, s0_c, states, u, p)
            return u, states

        @staticmethod
        def backward(ctx, du, dstate):
            q_c, delta_c, s0_c, states, u, p = ctx.saved_tensors
            B, T, D2 = q_c.shape
            D = D2 // 2
            du = torch.zeros_like(u) if du is None else _f32(du)
            dstate = torch.zeros_like(states) if dstate is None else _f32(dstate)
            dq = torch.empty_like(q_c)
            ddelta = torch.zeros(D, dtype=torch.float32, device=q_c.device)
            ds0 = torch.empty_like(s0_c)
            bind_stream(q_c)
            _call("core_bwd_f32", ptr(q_c), ptr(delta_c), ptr(s0_c), ptr(states), ptr(u),
                  ptr(p), ptr(dstate), ptr(du), ptr(dq), ptr(ddelta), ptr(ds0), B, T, D)
            return dq, ddelta, ds0

    _CORE = _Core
    return _CORE


def core_forward(q, delta, s0):
    """(u, states) of the fused core (reference core_auto.core_forward)."""
    return CoreCUDA.apply(q, delta, s0)


def step_core(q, delta, s):
    """One decode step: q (B,2D), delta (D,), s (B,D) -> (u, s_new)
    (reference core_auto.step_core)."""
    import torch
    B, D2 = q.shape
    D = D2 // 2
    q, delta, s = _f32(q), _f32(delta), _f32(s)
    s_new = torch.empty_like(s)
    u = torch.empty(B, D, dtype=torch.float32, device=q.device)
    bind_stream(q)
    _call("step_core_f32", ptr(q), ptr(delta), ptr(s), ptr(s_new), ptr(u), B, D)
    return u, s_new


def dw_step(x, hist, w_t, taps: int):
    """Depthwise causal taps, one step: x (B,D), hist (B,taps-1,D), w (taps,D)
    -> acc (B,D) (reference core_auto.dw_step)."""
    import torch
    B, D = x.shape
    x, hist, w_t = _f32(x), _f32(hist), _f32(w_t)
    acc = torch.empty(B, D, dtype=torch.float32, device=x.device)
    bind_stream(x)
    _call("dw_step_f32", ptr(x), ptr(hist), ptr(w_t), ptr(acc), B, D, int(taps))
    return acc


_SCAN = None


def _scan_fn():
    global _SCAN
    if _SCAN is not None:
        return _SCAN
    import torch

    class _Scan(torch.autograd.Function):
        @staticmethod
        def forward(ctx, u, p, s0):
            B, T, N = u.shape
            u_c, p_c, s0_c = _f32(u), _f32(p), _f32(s0)
            out = torch.empty_like(u_c)
            send = torch.empty_like(s0_c)
            bind_stream(u_c)
            _call("scan_f32", ptr(p_c), ptr(u_c), ptr(s0_c), ptr(out), ptr(send), B, T, N)
            ctx.save_for_backward(u_c, p_c, s0_c, out)
            return out

        @staticmethod
        def backward(ctx, dout):
            u_c, p_c, s0_c, out = ctx.saved_tensors
            B, T, N = u_c.shape
            dout_c = _f32(dout)
            dp = torch.empty_like(p_c)
            du = torch.empty_like(u_c)
            ds0 = torch.empty_like(s0_c)
            bind_stream(u_c)
            _call("scan_bwd_f32", ptr(p_c), ptr(u_c), ptr(s0_c), ptr(out), ptr(dout_c),
                  ptr(dp), ptr(du), ptr(ds0), B, T, N)
            return du, dp, ds0

    _SCAN = _Scan
    return _SCAN


class ScanCUDA:
    """s_t = p_t*s_{t-1} + (1-p_t)*u_t forward and backward as an autograd
    operator: (u, p, s0) -> states (reference scan_auto.ScanAVX2)."""

    @staticmethod
    def apply(u, p, s0):
        return _scan_fn().apply(u, p, s0)


def scan_auto(u, p, s0, chunk: int = 64, p_min_hint=None):
    """(states, last state) of the gated scan (reference scan_auto.scan_auto;
    chunk and p_min_hint only steer the reference's torch fallback, which this
    module does not have)."""
    states = ScanCUDA.apply(u, p, s0)
    return states, states[:, -1]


def _lib_loaded():
    """The library, without a look at the file where it is loaded already."""
    return _lib._lib or load_kernel()


_TORCH_CALLS = None


def _torch_calls():
    """The extension module for torch's tensors, given the library's entry points."""
    global _TORCH_CALLS
    if _TORCH_CALLS is None:
        import torch  # noqa: F401  (its libraries first)

        from . import build
        lib = load_kernel()
        if not build.TORCH_CALLS.exists():  # as load_runtime does with the library
            build.build()
        try:
            from . import _torch_calls as m
        except ImportError as e:
            raise RuntimeError(f"{build.TORCH_CALLS} was built for another torch; run "
                               "`python -m sunnynet_b200.build --force`") from e
        m.use(*(ctypes.cast(f, ctypes.c_void_p).value for f in (
            lib.sn_abi_layer_norm, lib.sn_abi_layer_norm_bwd, lib.sn_abi_layer_norm_bwd_ws,
            lib.sn_abi_last_error)))
        _TORCH_CALLS = m
    return _TORCH_CALLS


def _address(data: bytes) -> int:
    return ctypes.cast(data, ctypes.c_void_p).value


def layer_norm(x, weight=None, bias=None, eps: float = 1e-5):
    """(x - mean) / sqrt(var + eps) * weight + bias over the last axis of x
    (float32, bfloat16 or float16; the variance biased; sums in fp32).
    weight, bias: None or (D,) of float32 or x's type. Differentiable in x,
    weight and bias, once and in reverse mode (a tensor with a forward-mode
    tangent is refused); rows may lie at a stride. The same call gives the same
    bits every time; a row's bits depend on its place among the rows only
    where the width is no multiple of 16 bytes."""
    import torch
    if x.dim() == 0 or not 0 < x.shape[-1] <= _MAX_WIDTH:
        raise ValueError("layer_norm: x needs a last axis of 1 to 2^31 - 2^14 values")
    if not x.is_cuda:  # host tensors are staged, as by the other kernels
        to = lambda t: None if t is None else t.cuda()  # noqa: E731
        return layer_norm(x.cuda(), to(weight), to(bias), eps).to(x.device)
    D, kind = x.shape[-1], None
    dtype_code(x.dtype)
    for t in (weight, bias):
        if t is not None:
            if t.dim() != 1 or t.shape[0] != D or t.get_device() != x.get_device() or \
                    (t.dtype != torch.float32 and t.dtype != x.dtype) or \
                    (kind is not None and t.dtype != kind):
                raise ValueError(f"layer_norm: weight and bias have {D} values of float32 or "
                                 f"{x.dtype} on {x.device}, both the same")
            kind = t.dtype
    if not eps >= 0:
        raise ValueError("layer_norm: eps must not be negative")
    return _torch_calls().layer_norm(x, weight, bias, eps)


def adamw_step(params, grads, exp_avg, exp_avg_sq, step, lr=1e-3, beta1=0.9, beta2=0.999,
               eps=1e-8, weight_decay=0.01, avg_scale=None, sq_scale=None) -> None:
    """One AdamW step (decoupled weight decay) of all `params` in place, in one
    launch for each few hundred tensors.

    Lists of equal length: params of one float type, grads of one float type,
    and for each the states, updated in place: exp_avg and exp_avg_sq in
    float32, or, with avg_scale and sq_scale (float32, one for each
    ``STATE_BLOCK`` values), float8_e4m3fn codes of the first moment and of
    the square root of the second. All contiguous, on one GPU; no parameter or
    state twice, or overlapping another. `step` counts from 1. step (an int64
    tensor of one value) and lr (a float64 one) may be on the GPU: then a
    captured step reads them anew at each replay."""
    import torch
    Tensor = torch.Tensor
    lists = [params, grads, exp_avg, exp_avg_sq]
    if (avg_scale is None) != (sq_scale is None):
        raise ValueError("adamw_step: 8-bit states have avg_scale and sq_scale")
    bits = 32 if avg_scale is None else 8
    if bits == 8:
        lists += [avg_scale, sq_scale]
    lists = [x if isinstance(x, (list, tuple)) else list(x) for x in lists]
    n = len(lists[0])
    if any(len(x) != n for x in lists):
        raise ValueError("adamw_step: the lists differ in length")
    if n == 0:
        return
    first, grad = lists[0][0], lists[1][0]
    state = torch.float32 if bits == 32 else torch.float8_e4m3fn
    at, sizes = _torch_calls().read(
        tuple(lists), (first.dtype, grad.dtype, state, state, torch.float32, torch.float32)[:len(lists)],
        STATE_BLOCK)
    on_gpu = {}
    for name, v, dt in (("step", step, torch.int64), ("lr", lr, torch.float64)):
        if isinstance(v, Tensor):
            if v.dtype != dt or v.numel() != 1 or v.device != first.device:
                raise TypeError(f"adamw_step: {name} as a tensor is one {dt} value on "
                                f"{first.device}")
            on_gpu[name] = v.data_ptr()
    to = [_address(at) + 8 * n * i for i in range(len(lists))]
    rc = _lib_loaded().sn_abi_adamw_step(
        n, *to[:4], *(to[4:] or (None, None)), _address(sizes), dtype_code(first.dtype),
        dtype_code(grad.dtype), bits,
        0 if "step" in on_gpu else int(step), on_gpu.get("step"),
        0.0 if "lr" in on_gpu else float(lr), on_gpu.get("lr"), float(beta1), float(beta2),
        float(eps), float(weight_decay), current_stream(first))
    if rc:
        check(rc, "adamw_step")
    torch.autograd.graph.increment_version(lists[0])  # a graph that saved one must not use it
