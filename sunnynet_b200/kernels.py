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
from operator import attrgetter

from . import _lib
from ._lib import check, dtype_code, ptr
from .runtime import bind_stream, load_runtime

__all__ = ["load_kernel", "load_scan_kernel", "kernel_available", "set_kernel_threads",
           "CoreCUDA", "core_forward", "step_core", "dw_step", "ScanCUDA", "scan_auto",
           "layer_norm", "adamw_step", "STATE_BLOCK"]

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


def _stream(device) -> int:
    import torch
    return torch.cuda.current_stream(device).cuda_stream


_NORM = None


def _norm_fn():
    global _NORM
    if _NORM is not None:
        return _NORM
    import torch

    class _Norm(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, weight, bias, eps):
            D = x.shape[-1]
            rows = x.numel() // D
            x2 = x.reshape(rows, D)  # a view wherever the rows lie at one stride
            if x2.stride(1) != 1 or (rows > 1 and x2.stride(0) < D):
                x2 = x2.contiguous()
            w, b = (None if t is None else t.contiguous() for t in (weight, bias))
            y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
            keep = any(ctx.needs_input_grad)
            stats = torch.empty(2, rows, dtype=torch.float32, device=x.device) if keep else None
            wdtype = dtype_code(next((t.dtype for t in (w, b) if t is not None), x.dtype))
            check(load_kernel().sn_abi_layer_norm(
                x2.data_ptr(), max(x2.stride(0), D), _addr(w), _addr(b), y.data_ptr(),
                _addr(stats), _addr(stats) and stats[1:].data_ptr(), dtype_code(x.dtype), wdtype,
                rows, D, eps, _stream(x.device)), "layer_norm")
            if keep:
                ctx.save_for_backward(x2, w, stats)
                ctx.wdtype = wdtype
            return y

        @staticmethod
        @torch.autograd.function.once_differentiable
        def backward(ctx, dy):
            x, w, stats = ctx.saved_tensors
            rows, D = x.shape
            want_x, want_w, want_b = ctx.needs_input_grad[:3]
            g = dy.reshape(rows, D)
            if g.stride(1) != 1 or (rows > 1 and g.stride(0) < D):
                g = g.contiguous()  # among them what a sum's gradient broadcasts
            lib = load_kernel()
            dx = torch.empty(dy.shape, dtype=x.dtype, device=x.device) if want_x else None
            wt = (torch.float32, torch.bfloat16, torch.float16)[ctx.wdtype]
            dw, db = (torch.empty(D, dtype=wt, device=x.device) if want else None
                      for want in (want_w, want_b))
            ws, need = None, 0
            if want_w or want_b:
                with torch.cuda.device(x.device):
                    need = lib.sn_abi_layer_norm_bwd_ws(rows, D, dtype_code(x.dtype))
                ws = torch.empty(need, dtype=torch.uint8, device=x.device)
            check(lib.sn_abi_layer_norm_bwd(
                g.data_ptr(), max(g.stride(0), D), x.data_ptr(), max(x.stride(0), D), _addr(w),
                stats.data_ptr(), stats[1:].data_ptr(), _addr(dx), _addr(dw), _addr(db),
                _addr(ws), need, dtype_code(x.dtype), ctx.wdtype, rows, D, _stream(x.device)),
                "layer_norm_bwd")
            return dx, dw, db, None

    _NORM = _Norm
    return _NORM


def _addr(t):
    return None if t is None else t.data_ptr()


def layer_norm(x, weight=None, bias=None, eps: float = 1e-5):
    """(x - mean) / sqrt(var + eps) * weight + bias over the last axis of x
    (float32, bfloat16 or float16; the variance biased; sums in fp32).
    weight, bias: None or (D,) of float32 or x's type. Differentiable in x,
    weight and bias; rows may lie at a stride; the gradients do not depend on
    scheduling."""
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError("layer_norm: x needs a last axis of at least one value")
    if not x.is_cuda:  # host tensors are staged, as by the other kernels
        to = lambda t: None if t is None else t.cuda()  # noqa: E731
        return layer_norm(x.cuda(), to(weight), to(bias), eps).to(x.device)
    dtype_code(x.dtype)
    params = [t for t in (weight, bias) if t is not None]
    for t in params:
        if tuple(t.shape) != (x.shape[-1],) or t.device != x.device or \
                t.dtype != params[0].dtype or str(t.dtype) not in ("torch.float32", str(x.dtype)):
            raise ValueError(f"layer_norm: weight and bias have {x.shape[-1]} values of float32 "
                             f"or {x.dtype} on {x.device}, both the same")
    if not eps >= 0:
        raise ValueError("layer_norm: eps must not be negative")
    return _norm_fn().apply(x, weight, bias, float(eps))


def _addresses(tensors):
    import torch
    return (ctypes.c_void_p * len(tensors))(*map(torch.Tensor.data_ptr, tensors))


def adamw_step(params, grads, exp_avg, exp_avg_sq, step, lr=1e-3, beta1=0.9, beta2=0.999,
               eps=1e-8, weight_decay=0.01, avg_scale=None, sq_scale=None) -> None:
    """One AdamW step (decoupled weight decay) of all `params` in place, in one
    launch for each few hundred tensors.

    Lists of equal length: params of one float type, grads of one float type,
    and for each the states, updated in place: exp_avg and exp_avg_sq in
    float32, or, with avg_scale and sq_scale (float32, one for each
    ``STATE_BLOCK`` values), float8_e4m3fn codes of the first moment and of
    the square root of the second. All contiguous, on one GPU; no parameter
    twice. `step` counts from 1. step (an int64 tensor of one value) and lr (a
    float64 one) may be on the GPU: then a captured step reads them anew at
    each replay."""
    import torch
    params, grads, exp_avg, exp_avg_sq = map(list, (params, grads, exp_avg, exp_avg_sq))
    lists = [params, grads, exp_avg, exp_avg_sq]
    if (avg_scale is None) != (sq_scale is None):
        raise ValueError("adamw_step: 8-bit states have avg_scale and sq_scale")
    bits = 32 if avg_scale is None else 8
    scales = [] if bits == 32 else [list(avg_scale), list(sq_scale)]
    n = len(params)
    if any(len(x) != n for x in lists + scales):
        raise ValueError("adamw_step: the lists differ in length")
    if n == 0:
        return
    sizes = list(map(torch.Tensor.numel, params))
    if any(list(map(torch.Tensor.numel, x)) != sizes for x in lists[1:]):
        raise ValueError("adamw_step: a gradient or state differs in size from its parameter")
    if any(list(map(torch.Tensor.numel, x)) != [-(-k // STATE_BLOCK) for k in sizes]
           for x in scales):
        raise ValueError(f"adamw_step: one scale for each {STATE_BLOCK} values is wanted")
    kinds = [set(map(attrgetter("dtype"), x)) for x in lists + scales]
    state = torch.float32 if bits == 32 else torch.float8_e4m3fn
    if any(len(k) != 1 for k in kinds) or kinds[2] != {state} or kinds[3] != {state} or \
            any(k != {torch.float32} for k in kinds[4:]):
        raise TypeError(f"adamw_step: params of one type, grads of one type, states of {state} "
                        "and scales of float32 are wanted")
    for x in lists + scales:
        if not all(map(torch.Tensor.is_contiguous, x)):
            raise ValueError("adamw_step: every tensor must be contiguous")
    device = params[0].device
    if device.type != "cuda" or len(set().union(*(map(torch.Tensor.get_device, x)
                                                  for x in lists + scales))) != 1:
        raise ValueError("adamw_step: every tensor must be on one GPU")
    on_gpu = {}
    for name, v, dt in (("step", step, torch.int64), ("lr", lr, torch.float64)):
        if isinstance(v, torch.Tensor):
            if v.dtype != dt or v.numel() != 1 or v.device != device:
                raise TypeError(f"adamw_step: {name} as a tensor is one {dt} value on {device}")
            on_gpu[name] = v.data_ptr()
    at = [_addresses(x) for x in lists + scales]
    where = [a for a, k in zip(at[0], sizes) if k]
    if len(set(where)) != len(where):
        raise ValueError("adamw_step: a parameter appears twice")
    check(load_kernel().sn_abi_adamw_step(
        n, *at[:4], *(at[4:] or (None, None)), (ctypes.c_int64 * n)(*sizes),
        dtype_code(params[0].dtype), dtype_code(grads[0].dtype), bits,
        0 if "step" in on_gpu else int(step), on_gpu.get("step"),
        0.0 if "lr" in on_gpu else float(lr), on_gpu.get("lr"), float(beta1), float(beta2),
        float(eps), float(weight_decay), _stream(device)), "adamw_step")
