"""Lists of parameters and states that share memory."""
from __future__ import annotations

import pytest

from test_gpu_adamw import adamw_step  # noqa: F401

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def test_tensors_that_overlap_are_refused(adamw_step):  # noqa: F811
    """Each pair shares values without beginning at the same address."""
    flat = torch.randn(2000, device="cuda")
    g, m, v = (torch.rand(1000, device="cuda") for _ in range(3))
    before = flat.clone()
    one = [g[:300]], [m[:300]], [v[:300]]
    two = [g[:300], g[300:600]], [m[:300], m[300:600]], [v[:300], v[300:600]]
    codes = torch.zeros(2048, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    scales = torch.zeros(8, device="cuda")
    for bad in (lambda: adamw_step([flat[:300], flat[299:599]], *two, 1),
                lambda: adamw_step([flat[4:304], flat[:300]], *two, 1),
                lambda: adamw_step([flat[:300]], one[0], [flat[200:500]], one[2], 1),
                lambda: adamw_step([flat[:300]], one[0], [m[:300]], [m[100:400]], 1),
                lambda: adamw_step([flat[:600]], [g[:600]], [codes[:600]], [codes[512:1112]], 1,
                                   avg_scale=[scales[:3]], sq_scale=[scales[4:7]]),
                lambda: adamw_step([flat[:600]], [g[:600]], [codes[:600]], [codes[1024:1624]], 1,
                                   avg_scale=[scales[:3]], sq_scale=[scales[2:5]])):
        with pytest.raises(ValueError, match="overlaps"):
            bad()
    assert torch.equal(flat, before)


def test_neighbours_in_one_buffer(adamw_step):  # noqa: F811
    """Views that lie side by side are separate tensors."""
    g, start = torch.randn(2000, device="cuda"), torch.randn(2000, device="cuda")
    cuts = [0, 7, 8, 300, 301, 1555, 2000]
    flat, m, v = start.clone(), torch.zeros(2000, device="cuda"), torch.zeros(2000, device="cuda")
    of = lambda t: [t[a:b] for a, b in zip(cuts, cuts[1:])]  # noqa: E731
    whole = start.clone()
    adamw_step(of(flat), of(g), of(m), of(v), 1)
    adamw_step([whole], [g], [torch.zeros_like(g)], [torch.zeros_like(g)], 1)
    assert torch.equal(flat, whole)
