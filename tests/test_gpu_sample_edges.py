"""The draw's rows at their edges. Tokens are compared exactly with the rule in 64
bits, as in test_gpu_sample."""
from __future__ import annotations

import numpy as np
import pytest

from test_gpu_sample import names, rows_of, sample, token  # noqa: F401

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("n,V", [(1, 32000), (9, 5003), (70, 9001)])
def test_clusters_that_start_beside_other_work(sample, n, V):  # noqa: F811
    """A row's CTAs come to run while another stream keeps the SMs busy."""
    rng = np.random.default_rng(V)
    t, x = rows_of(rng.standard_normal((n, V)) * 2, torch.float32)
    u = rng.random(n)
    rule = {"T": 0.9, "k": 40, "p": 0.95}
    want = [token(r, v, **rule) for r, v in zip(x, u)]
    greedy = x.argmax(1).tolist()
    c = torch.from_numpy(u).cuda()
    a = torch.randn(2048, 2048, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(40):
        with torch.cuda.stream(side):
            a = (a @ a).clamp_(-1, 1)
        got += [sample(t, c, **names(rule)), sample(t, c, 0.0)]
    torch.cuda.synchronize()
    assert all(g.tolist() == want for g in got[::2]) and all(g.tolist() == greedy for g in got[1::2])
