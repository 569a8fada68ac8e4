"""The draw where few ids can stay or the border lies far below the largest logit:
low temperatures and rows with fewer allowed ids than top-k; clusters that start
beside other work.

The bins that narrow a row down reach 32 temperatures below the largest of its
first 1024 logits, 56 / 1020 of a temperature each; the last two have no far edge
that counts. Tokens are compared exactly with the rule in 64 bits, as in
test_gpu_sample.
"""
from __future__ import annotations

import numpy as np
import pytest

from test_gpu_sample import names, rows_of, sample, token  # noqa: F401

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


BIN = 56 / 1020  # of a temperature


def far_rows(rng, n, V, T, k, below):
    """Rows whose k-th logit lies `below` temperatures under the largest, which is
    among the first 1024; the others lie farther down."""
    x = -T * (below + 0.3 + 20 * rng.random((n, V)))
    for r in x:
        at = rng.choice(V, k, replace=False)
        r[at] = -T * 3 * rng.random(k)
        if k > 1:
            r[at[-1]] = -T * below
        at = at[0]
        if at >= 1024:
            r[rng.integers(min(V, 1024))], r[at] = 0.0, -T * (below + 0.3)
        else:
            r[at] = 0.0
    return x


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


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,V", [(1, 1000), (1, 32000), (3, 8192), (40, 9001), (160, 5003), (160, 16384)])
def test_the_kth_logit_in_the_last_bins(sample, n, V, dtype):  # noqa: F811
    """Bins 1021, 1022 and 1023 (the largest lies in bin 437), and far behind them."""
    rng = np.random.default_rng(V)
    for T, k, b in ((1.0, 2, 1022), (1.0, 40, 1021), (1.0, 40, 1022), (1.0, 40, 1023), (0.1, 100, 1022),
                    (0.15, 40, 1021.52), (0.5, 256, 1022), (0.25, 300, 1022), (1.0, 40, 1100)):
        t, x = rows_of(far_rows(rng, n, V, T, k, (b - 437.14) * BIN), dtype)
        u = rng.random(n)
        got = sample(t, torch.from_numpy(u).cuda(), T, top_k=k).cpu().numpy()
        assert np.array_equal(got, [token(r, v, T=T, k=k) for r, v in zip(x, u)]), (T, k, b)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,V,gap,off", [(200, 20011, 0, 0), (300, 10003, 0, 1), (200, 9973, 13, 3), (150, 20001, 5, 0),
                                         (160, 5003, 0, 1), (40, 9001, 3, 0), (2, 32001, 0, 5)])
def test_fewer_allowed_ids_than_top_k(sample, n, V, gap, off, dtype):  # noqa: F811
    """Ten allowed ids, the first of each row among them and the largest of all; what
    lies between the rows and behind the last is larger still."""
    rng = np.random.default_rng(V)
    flat = np.full(off + n * (V + gap) + 64, 3e4)
    x = np.full((n, V), -np.inf)
    for r in x:
        r[rng.choice(V, 8, replace=False)] = rng.standard_normal(8)
        r[:2] = 20.0 + rng.random(2)
    np.lib.stride_tricks.as_strided(flat[off:], (n, V), ((V + gap) * 8, 8))[:] = x
    f, _ = rows_of(flat, dtype)
    t = f[0].as_strided((n, V), (V + gap, 1), off)
    x = t.double().cpu().numpy()
    u = rng.random(n)
    for rule in ({"k": 40}, {"T": 12.0, "k": 40}, {"T": 0.1, "k": 40, "p": 0.9}, {"T": 9.0, "k": 300, "q": 0.1},
                 {"T": 5.0, "p": 0.97}, {"T": 1e300, "q": 0.5}):
        got = sample(t, torch.from_numpy(u).cuda(), **names(rule)).cpu().numpy()
        assert np.array_equal(got, [token(r, v, **rule) for r, v in zip(x, u)]), rule


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,V", [(60, 1000), (2, 32000), (160, 5003), (160, 20011), (300, 10003)])
def test_low_temperatures(sample, n, V, dtype):  # noqa: F811
    rng = np.random.default_rng(V + n)
    t, x = rows_of(rng.standard_normal((n, V)) * 2.5, dtype)
    u = rng.random(n)
    for T in (0.05, 0.1, 0.2):
        for k in (5, 40, 300):
            got = sample(t, torch.from_numpy(u).cuda(), T, top_k=k).cpu().numpy()
            assert np.array_equal(got, [token(r, v, T=T, k=k) for r, v in zip(x, u)]), (T, k)


@pytest.mark.parametrize("n,V", [(5, 1001), (1, 32001), (160, 5003), (160, 20011)])
def test_every_id_can_stay(sample, n, V):  # noqa: F811
    """Borders in the open bin of wide rows, and a min-p edge below every number."""
    rng = np.random.default_rng(V)
    t, x = rows_of(rng.standard_normal((n, V)) * 30, torch.float32)
    u = rng.random(n)
    for rule in ({"T": 60.0, "p": 0.9}, {"T": 60.0, "k": V - 3}, {"T": 60.0, "k": V // 2, "p": 0.9},
                 {"T": 1e300, "q": 0.5}, {"T": 1e39, "q": 1e-3}):
        got = sample(t, torch.from_numpy(u).cuda(), **names(rule)).cpu().numpy()
        assert np.array_equal(got, [token(r, v, **rule) for r, v in zip(x, u)]), rule


def test_top_k_beyond_31_bits(sample):  # noqa: F811
    """In a wider type: as many ids as a number of that size would keep."""
    rng = np.random.default_rng(6)
    t, x = rows_of(rng.standard_normal((4, 500)), torch.float32)
    u = np.array([0.9, 0.97, 0.5, 0.99])
    k = torch.tensor([(1 << 32) + 1, 3, -(1 << 33) + 2, (1 << 31) + 2], device="cuda")
    want = [token(r, v, k=j) for r, v, j in zip(x, u, (0, 3, 0, 0))]
    assert sample(t, torch.from_numpy(u).cuda(), top_k=k).tolist() == want
    assert sample(t, torch.from_numpy(u).cuda(), top_k=k.double()).tolist() == want


def test_step_sample_of_torch_tensors_on_the_host():
    import tempfile
    from pathlib import Path

    from sunnynet_b200 import formats
    from sunnynet_b200.model import SunnyBatch
    shape = formats.SunnyShape(700, 64, 96, 32, 4, 2)
    with tempfile.TemporaryDirectory() as td:
        p = Path(td) / "m.usnn"
        formats.write_usnn(p, formats.random_sunny(shape, seed=3, perturb=True))
        a, b = SunnyBatch(p, 3), SunnyBatch(p, 3)
        toks, u, k = np.array([5, 600, 31], np.int32), np.array([0.1, 0.5, 0.9]), np.array([0, 7, 40])
        for _ in range(3):
            want = b.step_sample(toks, u, 0.8, k)
            got = a.step_sample(torch.from_numpy(toks), torch.from_numpy(u), 0.8, torch.from_numpy(k))
            assert isinstance(want, np.ndarray) and got.dtype == torch.int32 and not got.is_cuda
            assert got.tolist() == want.tolist()
            toks = want
