"""Calls of the enqueue-only operators at the edge of what they take; no GPU is asked."""
from __future__ import annotations

import numpy as np
import pytest

from test_operators_host import lib  # noqa: F401

torch = pytest.importorskip("torch")

X = np.zeros(64, np.float64)
A = X.ctypes.data


@pytest.mark.parametrize("D", [(1 << 31) - 1, (1 << 31) - (1 << 14) + 1])
def test_widths_that_32_bit_columns_cannot_count(lib, D):  # noqa: F811
    from sunnynet_b200 import kernels
    for dtype in (0, 1, 2):
        assert lib.sn_abi_layer_norm(A, D, None, None, A, None, None, dtype, 0, 1, D, 1e-5, None) == -1
        assert lib.sn_abi_layer_norm_bwd(A, D, A, D, None, A, A, A, None, None, None, 0, dtype, 0, 1, D,
                                         None) == -1
        assert lib.sn_abi_layer_norm_bwd_ws(1, D, dtype) == 0
    with pytest.raises(ValueError, match="last axis"):
        kernels.layer_norm(torch.zeros(1).expand(1, D))
    assert lib.sn_abi_layer_norm(A, D, None, None, A, None, None, 0, 0, 0, (1 << 31) - (1 << 14), 1e-5, None) == 0


def test_layer_norm_of_tensors_with_a_tangent(lib):  # noqa: F811
    """Refused, not computed without their tangent."""
    import torch.autograd.forward_ad as fwd

    from sunnynet_b200 import kernels
    norm = kernels._torch_calls().layer_norm
    x, w = torch.randn(4, 8), torch.randn(8)
    for grad in (True, False):
        with torch.set_grad_enabled(grad), fwd.dual_level():
            dx, dw = fwd.make_dual(x, torch.ones_like(x)), fwd.make_dual(w, torch.ones_like(w))
            for args in ((dx, None, None), (x, dw, None), (x, w, dw)):
                with pytest.raises(RuntimeError, match="forward-mode"):
                    norm(*args, 1e-5)
