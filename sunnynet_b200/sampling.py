"""The draw of the next token on the GPU: the reference's sample_logits
(serve.py:30-57) and min-p for a batch of rows, from given uniform numbers.

``serve.BatchEngine`` draws with it; a decode loop of its own calls ``sample``
on the logits that ``SunnyBatch.step`` or ``Rwkv7Batch.step`` left on the GPU.
"""
from __future__ import annotations

import math

import numpy as np

from . import _lib
from ._lib import check, current_stream, dtype_code
from .runtime import load_runtime

__all__ = ["sample", "settings_to"]


def _setting(name, v, B, device, dtype):
    """(address or None, one value, what keeps the address alive)."""
    import torch
    if not isinstance(v, torch.Tensor):
        return None, v, None
    if v.dim() != 1 or v.shape[0] != B or v.get_device() != device:
        raise ValueError(f"sample: {name} is one number or {B} of them on cuda:{device}")
    if dtype == torch.int32 and v.dtype != dtype:  # beyond 31 bits: every id, as a number would
        v = v.to(torch.int64).clamp(0, 0x7fffffff)
    v = v.to(dtype).contiguous()
    return v.data_ptr(), 0, v


def settings_to(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """u and the settings of ``sample``, from host arrays (or single numbers) to
    the logits' GPU in one copy."""
    import torch
    B = logits.shape[0]
    pack = np.zeros((5, B), np.float64)  # top_k is a whole number below 2^31: exact
    k = np.clip(np.asarray(top_k), 0, 0x7fffffff)
    for to, v in zip(pack, (u, temperature, top_p, min_p, k)):
        to[:] = v
    if not np.isfinite(pack).all():
        raise ValueError("sample: the settings are finite numbers")
    u, t, p, q, k = torch.from_numpy(pack).to(logits.device)
    return u, t, k.to(torch.int32), p, q


def sample(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, out=None):
    """Tokens (B,) int32 drawn from logits (B, V) (float32, bfloat16 or
    float16, on a GPU; rows may lie at a stride) with uniform numbers u (B,) in
    [0, 1) (float32 or float64).

    temperature, top_k, top_p, min_p: a number for all rows, or a tensor (B,)
    on the logits' GPU (float64, top_k int32; others are converted there).
    temperature <= 0 takes the lowest id of the largest logit. top_k of 0 (or
    >= V), top_p of 1 and min_p of 0 keep every id; ids as likely as the k-th
    stay. A row without a logit above -inf gives -1. Only enqueues, on torch's
    current stream of that GPU."""
    import torch
    if logits.dim() != 2 or not logits.is_cuda:
        raise ValueError("sample: logits (B, V) on a GPU are wanted")
    B, V = logits.shape
    if not 0 < V < 1 << 31 or B >= 1 << 31:
        raise ValueError("sample: rows of 1 to 2^31 - 1 logits are wanted, and fewer rows than 2^31")
    ld, along = logits.stride()
    if V > 1 and along != 1 or B > 1 and ld < V:
        raise ValueError("sample: the logits of a row must lie side by side")
    dev = logits.get_device()
    if u.dim() != 1 or u.shape[0] != B or u.get_device() != dev or \
            u.dtype not in (torch.float32, torch.float64):
        raise ValueError(f"sample: u has {B} numbers of float32 or float64 on cuda:{dev}")
    if out is None:
        out = logits.new_empty(B, dtype=torch.int32)
    elif out.dim() != 1 or out.shape[0] != B or out.dtype != torch.int32 or \
            out.get_device() != dev or not out.is_contiguous():
        raise ValueError(f"sample: out has {B} contiguous int32 values on cuda:{dev}")
    u = u.contiguous()
    t, t0, keep_t = _setting("temperature", temperature, B, dev, torch.float64)
    k, k0, keep_k = _setting("top_k", top_k, B, dev, torch.int32)
    p, p0, keep_p = _setting("top_p", top_p, B, dev, torch.float64)
    q, q0, keep_q = _setting("min_p", min_p, B, dev, torch.float64)
    if not math.isfinite(t0) or not math.isfinite(p0) or not q0 <= 1:
        raise ValueError("sample: temperature and top_p are finite, min_p is at most 1")
    rc = (_lib._lib or load_runtime()).sn_abi_sample(
        logits.data_ptr(), max(ld, V), dtype_code(logits.dtype), u.data_ptr(),
        int(u.dtype == torch.float64), t, float(t0), k, max(0, min(int(k0), 0x7fffffff)), p,
        float(p0), q, float(q0), B, V, out.data_ptr(), current_stream(logits))
    if rc:
        check(rc, "sample")
    return out
