"""The draw of the next token on the GPU against the rule in 64 bits (numpy).

Tokens are compared exactly: u is placed in the middle of an id's share of the
kept weight, where the kernel's weights (cut at 2^-44 of the largest) cannot
move the answer, or drawn at random, where the chance that a border lies
within 2^-40 of u is below 1e-9 for all cases together.
"""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def sample():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from sunnynet_b200.sampling import sample
    return sample


def kept(x, T=1.0, k=0, p=1.0, q=0.0):
    """Weights of a row's ids in fp64, 0 where they are not kept; None: nothing to draw."""
    x = np.where(np.isnan(x), -np.inf, np.asarray(x, np.float64))
    best = x.max()
    if best == -np.inf:
        return None
    if not T > 0 or best == np.inf:
        w = np.zeros(x.size)
        w[np.argmax(x)] = 1.0
        return w
    w = np.exp((x - best) / T)
    if 0 < k < x.size:
        w = np.where(x >= np.sort(x)[x.size - k], w, 0.0)
    if 0 < p < 1:
        by = np.argsort(-np.where(w > 0, x, -np.inf), kind="stable")
        ahead = np.concatenate(([0.0], np.cumsum(w[by])[:-1]))
        w[by[~(ahead < p * w.sum())]] = 0.0
    return np.where(w >= q, w, 0.0)


def token(x, u, **rule):
    w = kept(x, **rule)
    if w is None:
        return -1
    upto = np.cumsum(w)
    return int(np.argmax(upto > u * upto[-1]))


def rows_of(x, dtype):
    """x (fp64) in the tested type, and as the numbers it then holds."""
    t = torch.from_numpy(np.atleast_2d(x)).to(dtype).cuda()
    return t, t.double().cpu().numpy()


DTYPES = [torch.float32, torch.bfloat16, torch.float16]
RULES = [{}, {"T": 0.7}, {"k": 5}, {"p": 0.8}, {"q": 0.05}, {"T": 0.8, "k": 40, "p": 0.95},
         {"T": 1.7, "k": 300, "p": 0.6, "q": 0.01}, {"p": 1e-9}, {"k": 1}, {"T": 30.0, "p": 0.999}]


def names(rule):
    return {{"T": "temperature", "k": "top_k", "p": "top_p", "q": "min_p"}[n]: v
            for n, v in rule.items()}


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [1, 2, 7, 37, 513, 3001, 8193, 32000, 65521])
@pytest.mark.parametrize("rule", RULES)
def test_every_kept_id_has_its_share(sample, V, dtype, rule):
    rng = np.random.default_rng(V)
    t, x = rows_of(rng.standard_normal(V) * 2.5, dtype)
    w = kept(x[0], **rule)
    ids = np.flatnonzero(w)
    # half a share above what V weights cut at 2^-44 can add up to: 65521 * 2^-44 = 3.8e-9
    ids = ids[w[ids] > 1e-7 * w.max()]
    if ids.size > 64:
        ids = np.concatenate((ids[:8], rng.choice(ids, 48, replace=False), ids[-8:]))
    upto = np.cumsum(w)
    u = torch.from_numpy((upto[ids] - w[ids] / 2) / upto[-1]).cuda()
    got = sample(t.expand(len(ids), V).contiguous(), u, **names(rule)).cpu().numpy()
    assert np.array_equal(got, ids)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [64, 1000, 20011])
def test_ties(sample, V, dtype):
    """Few distinct values: equal logits stay together in top-k and go by id in top-p."""
    rng = np.random.default_rng(3)
    t, x = rows_of(rng.integers(-2, 3, (40, V)).astype(np.float64), dtype)
    u = rng.random(40)
    for rule in ({"k": 3}, {"k": V // 2}, {"p": 0.1}, {"p": 0.5}, {"p": 0.97}, {"k": V // 3, "p": 0.5},
                 {"q": 0.3}, {"T": 5.0, "p": 0.31}):
        got = sample(t, torch.from_numpy(u).cuda(), **names(rule)).cpu().numpy()
        assert np.array_equal(got, [token(r, v, **rule) for r, v in zip(x, u)]), rule


@pytest.mark.parametrize("V", [5, 3000, 40000])
def test_equal_logits(sample, V):
    """A row of one value: id floor(u V) of those that stay."""
    u = np.array([0.0, 0.123, 0.5, 0.75, 0.999999])
    for value in (0.0, -3.5, 1e30, float(np.finfo(np.float32).min)):
        t = torch.full((5, V), value, device="cuda")
        got = sample(t, torch.from_numpy(u).cuda()).cpu().numpy()
        assert np.array_equal(got, np.floor(u * V))
        got = sample(t, torch.from_numpy(u).cuda(), top_p=0.4, top_k=2).cpu().numpy()
        stay = int(np.ceil(0.4 * V))
        assert np.array_equal(got, np.floor(u * stay))


def test_masked_and_infinite(sample):
    inf, nan, low = np.inf, np.nan, float(np.finfo(np.float32).min)
    rows = [[-inf] * 6, [nan] * 6, [-inf, nan, -inf, nan, nan, -inf],   # nothing to draw
            [-inf, 1, -inf, -inf, -inf, -inf], [nan, nan, nan, 0.0, nan, nan],
            [0, inf, 3, inf, -inf, nan], [low] * 6, [low, low, 5, low, 5, -inf],
            [-0.0, 0.0, -0.0, -1, nan, -inf], [low, -inf, -inf, -inf, -inf, nan]]
    t = torch.tensor(rows, dtype=torch.float32).cuda()
    for T in (1.0, 0.0, 1e-12, 1e12):
        for rule in ({}, {"k": 2}, {"p": 0.5}, {"k": 3, "p": 0.9, "q": 0.1}):
            for u in (0.0, 0.4, 0.99):
                got = sample(t, torch.full((len(rows),), u, device="cuda", dtype=torch.float64),
                             T, **names(rule)).tolist()
                assert got == [token(np.array(r), u, T=T, **rule) for r in rows], (T, rule, u)


def test_settings_of_each_row(sample):
    rng = np.random.default_rng(11)
    n, V = 301, 5003
    t, x = rows_of(rng.standard_normal((n, V)) * 3, torch.float32)
    T = np.where(rng.random(n) < 0.2, 0.0, rng.uniform(0.2, 2.0, n))
    k = np.where(rng.random(n) < 0.4, 0, rng.integers(1, 2 * V, n)).astype(np.int32)
    p = np.where(rng.random(n) < 0.4, 1.0, rng.random(n))
    q = np.where(rng.random(n) < 0.4, 0.0, rng.random(n) * 0.2)
    u = rng.random(n)
    c = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    got = sample(t, c(u), c(T), c(k), c(p), c(q)).cpu().numpy()
    want = [token(r, v, T=a, k=int(b), p=d, q=e) for r, v, a, b, d, e in zip(x, u, T, k, p, q)]
    assert np.array_equal(got, want)
    u32 = u.astype(np.float32)
    got = sample(t, c(u32), c(T).float().double(), c(k)).cpu().numpy()
    T32 = T.astype(np.float32).astype(np.float64)
    assert np.array_equal(got, [token(r, v, T=a, k=int(b)) for r, v, a, b in
                                zip(x, u32.astype(np.float64), T32, k)])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V,ld,off", [(1000, 1000, 1), (1001, 1001, 0), (1003, 1027, 5),
                                      (30011, 30016, 3)])
def test_strides_and_odd_addresses(sample, V, ld, off, dtype):
    rng = np.random.default_rng(V)
    n = 9
    flat, _ = rows_of(rng.standard_normal(off + n * ld) * 2, dtype)
    t = flat[0].as_strided((n, V), (ld, 1), off)
    u = rng.random(n)
    rule = {"T": 0.9, "k": 50, "p": 0.9}
    got = sample(t, torch.from_numpy(u).cuda(), **names(rule)).cpu().numpy()
    assert np.array_equal(got, [token(r, v, **rule) for r, v in zip(t.double().cpu().numpy(), u)])


@pytest.mark.parametrize("V", [200003, 450001, 1200007])
def test_long_rows(sample, V):
    """Slices of more keys than a 32 KB slice, and (the last two) than shared memory."""
    rng = np.random.default_rng(V)
    t, x = rows_of(rng.standard_normal((2, V)) * 2, torch.bfloat16)
    u = np.array([0.3, 0.95])
    for rule in ({}, {"k": 1000}, {"p": 0.9}, {"T": 2.0, "k": 60, "p": 0.9, "q": 0.05}):
        got = sample(t, torch.from_numpy(u).cuda(), **names(rule)).cpu().numpy()
        assert np.array_equal(got, [token(r, v, **rule) for r, v in zip(x, u)]), rule


@pytest.mark.parametrize("V", [70001, 930001, 1040001])
@pytest.mark.parametrize("copies", [55, 110, 220])
def test_long_rows_of_many_requests(sample, V, copies):
    """A CTA to each of 165, 330 and 660 rows, their lists of three lengths."""
    rng = np.random.default_rng(V)
    t, x = rows_of(rng.standard_normal((3, V)) * 2, torch.bfloat16)
    u = np.array([0.3, 0.8, 0.95])
    many, us = t.repeat(copies, 1), torch.from_numpy(u).cuda().repeat(copies)
    for rule in ({"k": 9000}, {"k": 20000, "p": 0.8}, {"p": 0.6}):
        got = sample(many, us, **names(rule)).cpu().numpy().reshape(copies, 3)
        assert (got == [token(r, v, **rule) for r, v in zip(x, u)]).all(), rule


def test_borders_among_crowded_logits(sample):
    """Thousands of distinct logits within one bin of the first histogram: the later rounds."""
    rng = np.random.default_rng(8)
    V = 24000
    x = np.empty((4, V), np.float32)
    x[0] = 1 + rng.permutation(V) * 2.0 ** -22
    x[1] = x[0]
    x[1, 77] = 60.0
    x[2] = -1e-3 + rng.permutation(V) * 2.0 ** -36
    x[2, 5] = np.finfo(np.float32).min
    x[3] = np.where(rng.random(V) < 0.5, 1e-30, 1e-38) * rng.random(V)
    t = torch.from_numpy(x).cuda()
    for rule in ({"k": 777}, {"k": 20000}, {"T": 100.0, "p": 0.37}, {"T": 100.0, "k": 9999, "p": 0.5}):
        for u in (0.01, 0.49, 0.98):
            got = sample(t, torch.full((4,), u, dtype=torch.float64, device="cuda"),
                         **names(rule)).tolist()
            assert got == [token(r, u, **rule) for r in x.astype(np.float64)], (rule, u)


def test_extreme_settings(sample):
    rng = np.random.default_rng(2)
    t, x = rows_of(rng.standard_normal((6, 4001)) * 4, torch.float32)
    u = np.array([0.0, 2.0 ** -53, 0.25, 0.5, 1 - 2.0 ** -20, 1 - 2.0 ** -53])
    for rule in ({"T": 1e-300}, {"T": 1e-5}, {"T": 1e8}, {"T": 1e300}, {"p": 1e-300}, {"k": 4000},
                 {"k": 4001}, {"k": 2 ** 31 - 1}, {"q": 1.0}, {"T": 1e8, "p": 0.999}):
        got = sample(t, torch.from_numpy(u).cuda(), **names(rule)).cpu().numpy()
        want = [token(r, v, **rule) for r, v in zip(x, u)]
        # the last u lies within 2^-53 of the end: any kept id of vanishing weight may be last
        assert np.array_equal(got[:5], want[:5]), rule
        assert kept(x[5], **rule)[got[5]] > 0 or got[5] == want[5]
    # outside [0, 1): the first and the last kept id
    got = sample(t[:3].contiguous(), torch.tensor([-1.0, 1.0, 7.0], device="cuda"), top_k=3).tolist()
    top3 = [sorted(np.argsort(-r)[:3]) for r in x[:3]]
    assert got == [top3[0][0], top3[1][2], top3[2][2]]


def test_no_rows_and_out(sample):
    t = torch.randn(4, 100, device="cuda")
    assert sample(t[:0], torch.empty(0, device="cuda")).shape == (0,)
    out = torch.full((6,), 99, dtype=torch.int32, device="cuda")
    r = sample(t, torch.rand(4, device="cuda"), 0.0, out=out[1:5])
    assert r.data_ptr() == out[1:].data_ptr()
    assert out.tolist() == [99, *t.argmax(1).tolist(), 99]


def test_captured_and_replayed_beside_another_stream(sample):
    """One captured draw replayed on new logits while another stream draws others."""
    g = torch.Generator(device="cuda").manual_seed(4)
    t = torch.randn(33, 7001, device="cuda", generator=g)
    u = torch.rand(33, device="cuda", dtype=torch.float64, generator=g)
    other = torch.randn(50, 9001, device="cuda", generator=g)
    uo = torch.rand(50, device="cuda", dtype=torch.float64, generator=g)
    want_other = sample(other, uo, 0.7, 20, 0.9)
    sample(t, u, 0.8, 30, 0.9)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = sample(t, u, 0.8, 30, 0.9)
    side = torch.cuda.Stream()
    for step in range(5):
        t.copy_(torch.randn(t.shape, device="cuda", generator=g))
        u.copy_(torch.rand(33, device="cuda", dtype=torch.float64, generator=g))
        with torch.cuda.stream(side):
            beside = sample(other, uo, 0.7, 20, 0.9)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, sample(t, u, 0.8, 30, 0.9)), step
        assert torch.equal(beside, want_other)


def test_refusals(sample):
    t, u = torch.randn(3, 10, device="cuda"), torch.rand(3, device="cuda")
    for bad in (lambda: sample(t.cpu(), u), lambda: sample(t, u.cpu()), lambda: sample(t[0], u),
                lambda: sample(t, u[:2]), lambda: sample(t.t(), torch.rand(10, device="cuda")),
                lambda: sample(t[:, :0], u), lambda: sample(t.double(), u),
                lambda: sample(t, u, float("nan")), lambda: sample(t, u, min_p=1.5),
                lambda: sample(t, u, torch.ones(2, device="cuda")),
                lambda: sample(t, u.half()), lambda: sample(t[:1].expand(3, 10), u),
                lambda: sample(t, u, out=torch.empty(3, device="cuda"))):
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            bad()
    from sunnynet_b200 import _lib
    L = _lib.load()
    host = np.zeros((3, 10), np.float32)
    out = torch.empty(3, dtype=torch.int32, device="cuda")
    rc = L.sn_abi_sample(host.ctypes.data, 10, 0, u.data_ptr(), 0, None, 1.0, None, 0, None, 1.0,
                         None, 0.0, 3, 10, out.data_ptr(), None)
    assert rc == -1 and "device memory" in _lib.last_error()


def test_engine_draws_on_the_gpu_what_the_host_draws():
    """Requests of every kind of settings, served among others: the same tokens
    from the GPU's draw as from numpy's on the same logits and generators."""
    import tempfile
    from pathlib import Path

    from sunnynet_b200 import formats
    from sunnynet_b200.model import SunnyBatch
    from sunnynet_b200.serve import BatchEngine
    shape = formats.SunnyShape(1500, 128, 224, 80, 4, 3)
    rng = np.random.default_rng(5)
    specs = [dict(temperature=0.8, top_k=40, top_p=0.95, seed=1), dict(),
             dict(temperature=1.2, seed=2), dict(temperature=0.7, top_p=0.5, seed=3),
             dict(temperature=1.5, min_p=0.05, seed=4), dict(temperature=1.0, top_k=3, seed=5),
             dict(temperature=0.9, top_k=0, top_p=0.0, seed=6)]
    prompts = [list(rng.integers(0, shape.vocab, n)) for n in (4, 9, 9, 3, 17, 4, 8)]
    with tempfile.TemporaryDirectory() as td:
        p = Path(td) / "m.usnn"
        formats.write_usnn(p, formats.random_sunny(shape, seed=2, perturb=True))

        class HostDraws(SunnyBatch):
            step_sample = property()  # not offered

        tokens = []
        for factory in (SunnyBatch, HostDraws):
            eng = BatchEngine(slots=3, prefill_chunk=8, handle_factory=lambda n: factory(p, n))
            assert hasattr(eng.main, "step_sample") == (factory is SunnyBatch)
            reqs = [eng.submit(q, 12, **s) for q, s in zip(prompts, specs)]
            eng.run()
            tokens.append([r.tokens for r in reqs])
        assert tokens[0] == tokens[1] and all(len(t) == 12 for t in tokens[0])


def test_step_sample_of_a_handle():
    import tempfile
    from pathlib import Path

    from sunnynet_b200 import formats
    from sunnynet_b200.model import SunnyBatch
    shape = formats.SunnyShape(700, 64, 96, 32, 4, 2)
    with tempfile.TemporaryDirectory() as td:
        p = Path(td) / "m.usnn"
        formats.write_usnn(p, formats.random_sunny(shape, seed=3, perturb=True))
        a, b = SunnyBatch(p, 5), SunnyBatch(p, 5)
        rng = np.random.default_rng(0)
        toks = rng.integers(0, shape.vocab, 5).astype(np.int32)
        T, k = np.array([0.0, 0.5, 1.0, 2.0, 0.8]), np.array([0, 5, 0, 50, 10])
        for _ in range(4):
            u = rng.random(5)
            logits = np.asarray(b.step(toks))
            want = [token(r, v, T=t, k=int(j)) for r, v, t, j in zip(logits.astype(np.float64), u, T, k)]
            got = a.step_sample(toks, u, T, k)
            assert got.dtype == np.int32 and got.tolist() == want
            toks = got
        c = lambda x: torch.from_numpy(x).cuda()  # noqa: E731
        got = a.step_sample(c(toks), c(u), c(T), c(k.astype(np.int32)))
        assert got.is_cuda and got.tolist() == [
            token(r, v, T=t, k=int(j)) for r, v, t, j in
            zip(np.asarray(b.step(toks)).astype(np.float64), u, T, k)]
