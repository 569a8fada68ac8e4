"""BatchEngine asks for torch only where a request is drawn on the GPU, and serves
without it where it is not installed."""
from __future__ import annotations

import sys

import numpy as np
import pytest

from sunnynet_b200.serve import BatchEngine
from test_serve import V, FakeHandle, _alone


class Handle(FakeHandle):
    """One that could draw on the GPU, and must not be asked to."""

    def prefill(self, toks, chunk=256):
        assert isinstance(toks, np.ndarray)
        return super().prefill(toks, chunk)

    def step_sample(self, *a):
        raise AssertionError("no GPU here")


def test_greedy_requests_stay_with_numpy():
    rng = np.random.default_rng(0)
    prompts = [list(rng.integers(0, V, n)) for n in (5, 9, 9, 17, 3)]
    eng = BatchEngine(slots=3, handle_factory=Handle)
    reqs = [eng.submit(p, 7, temperature=t) for p, t in zip(prompts, (0.0, -1.0, None, 0.0, float("nan")))]
    eng.run()
    assert [r.tokens for r in reqs] == [_alone(p, 7) for p in prompts]


@pytest.mark.parametrize("samp", [{}, {"temperature": 0.8, "top_p": 0.9, "top_k": 20, "seed": 3}])
def test_served_without_torch(monkeypatch, samp):
    monkeypatch.setitem(sys.modules, "torch", None)  # as where it is not installed
    with pytest.raises(ImportError):
        import torch  # noqa: F401
    rng = np.random.default_rng(1)
    prompts = [list(rng.integers(0, V, n)) for n in (4, 8, 8)]
    eng = BatchEngine(slots=2, handle_factory=Handle)
    reqs = [eng.submit(p, 9, **samp) for p in prompts]
    eng.run()
    assert [r.tokens for r in reqs] == [_alone(p, 9, **samp) for p in prompts]
