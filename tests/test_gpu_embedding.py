"""The rows of an embedding and its gradient. Forward: the rows times the scale,
rounded once to fp32 and once to the stored type: equal bits. Gradient: against
sums in 64 bits; a row's sum of m values has at most m + 2 roundings of fp32 (the
pieces of a long row, and the scale), 2^-24 of the sum of magnitudes each, and
the store's half step."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def kernels():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from sunnynet_b200 import kernels
    return kernels


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def words(n, V, how, seed=0):
    u = torch.rand(n, device="cuda", generator=gen(seed), dtype=torch.float64)
    if how == "even":
        return (u * V).long().clamp_max(V - 1)
    if how == "one":
        return torch.full((n,), V // 2, device="cuda")
    if how == "two":
        return torch.where(u < 0.5, 0, V - 1)
    return torch.exp(u * torch.tensor(float(V), dtype=torch.float64).log().item()).long().clamp_max(V) - 1


def check(dw, tokens, dout, scale, V):
    D = dout.shape[-1]
    rows = dout.double().reshape(-1, D)
    ok = (tokens.reshape(-1) >= 0) & (tokens.reshape(-1) < V)
    at = tokens.reshape(-1)[ok].long()
    want = torch.zeros(V, D, dtype=torch.float64, device="cuda").index_add_(0, at, rows[ok]) * scale
    most = torch.zeros(V, D, dtype=torch.float64, device="cuda").index_add_(0, at, rows[ok].abs()) * abs(scale)
    m = torch.bincount(at, minlength=V)[:, None]
    e = torch.finfo(dw.dtype).eps / 2
    bound = (m + 2) * 2.0 ** -24 * most
    tiny = torch.finfo(dw.dtype).smallest_normal * e
    assert ((dw.double() - want).abs() <= bound + e * (want.abs() + bound) + tiny).all()
    assert (dw[(m == 0)[:, 0]] == 0).all()


def grad(kernels, tokens, w, dout, scale):
    w = w.detach().requires_grad_()
    out = kernels.embedding(tokens, w, scale)
    return out.detach(), torch.autograd.grad(out, w, dout)[0]


SIZES = [(1, 1, 1), (1, 300, 64), (2, 5, 7), (63, 255, 128), (64, 256, 512), (300, 257, 33), (1000, 70000, 8),
         (4097, 32000, 768), (5003, 4999, 1001), (40000, 16384, 48), (17, 20, 5000), (150000, 100, 16)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,V,D", SIZES)
@pytest.mark.parametrize("how", ["rank", "even", "one", "two"])
def test_rows_and_gradient(kernels, n, V, D, dtype, how):
    tokens = words(n, V, how, n)
    w = torch.randn(V, D, device="cuda", generator=gen(1)).to(dtype)
    dout = torch.randn(n, D, device="cuda", generator=gen(2)).to(dtype)
    out, dw = grad(kernels, tokens, w, dout, 1.7)
    assert torch.equal(out, (w[tokens].float() * torch.tensor(1.7, device="cuda")).to(dtype))
    assert dw.dtype == dtype and dw.shape == w.shape
    check(dw, tokens, dout, float(torch.tensor(1.7)), V)


def test_rows_as_long_as_a_chunk(kernels):
    """Runs of every length around the chunks' borders, in every order."""
    g = gen(5)
    for n in (15, 16, 17, 33, 64, 200, 1000):
        for longest in (1, 2, 15, 16, 17, 18, 31, 32, 33, 48, 49, 100):
            lengths = torch.randint(1, longest + 1, (n,), device="cuda", generator=g)
            tokens = torch.repeat_interleave(torch.arange(n, device="cuda"), lengths)[:n]
            tokens = tokens[torch.randperm(n, device="cuda", generator=g)]
            dout = torch.randn(n, 8, device="cuda", generator=g)
            check(grad(kernels, tokens, torch.zeros(n, 8, device="cuda"), dout, 1.0)[1], tokens, dout, 1.0, n)
        tokens = torch.arange(n, device="cuda").flip(0) // 16
        check(grad(kernels, tokens, torch.zeros(n, 8, device="cuda"), dout, 1.0)[1], tokens, dout, 1.0, n)


def test_strangers(kernels):
    """Tokens outside the vocabulary: rows of NaN, no gradient."""
    for kind in (torch.int32, torch.int64):
        for V in (1, 100, 255, 256, 65535, 65536):
            tokens = words(600, V, "even").to(kind)
            tokens[::7] = V
            tokens[1::50] = -1
            tokens[2::90] = torch.iinfo(kind).min
            tokens[3::90] = torch.iinfo(kind).max
            if kind == torch.int64:
                tokens[4::100] += 1 << 32
            bad = (tokens < 0) | (tokens >= V)
            w = torch.randn(V, 24, device="cuda")
            dout = torch.randn(600, 24, device="cuda")
            dout[bad] = float("nan")
            out, dw = grad(kernels, tokens, w, dout, 1.0)
            assert torch.equal(out.isnan().all(1), bad) and torch.equal(out[~bad], w[tokens[~bad].long()])
            check(dw, tokens, torch.where(bad[:, None], 0.0, dout), 1.0, V)
    out, dw = grad(kernels, torch.full((40,), 9, device="cuda"), torch.randn(9, 4, device="cuda"), torch.ones(40, 4, device="cuda"), 1.0)
    assert out.isnan().all() and (dw == 0).all()


def test_shapes_strides_and_nothing(kernels):
    w = torch.randn(50, 80, device="cuda")
    tokens = torch.randint(0, 50, (4, 6, 3), device="cuda", generator=gen(1))
    part = w[:, 3:67]  # rows at a stride, at an odd address
    assert torch.equal(kernels.embedding(tokens, part), part[tokens])
    assert torch.equal(kernels.embedding(tokens.permute(2, 0, 1), part), part[tokens.permute(2, 0, 1)])
    turned = w.t()  # values of a row apart
    assert torch.equal(kernels.embedding(tokens, turned[:, :50]), turned[:, :50][tokens])
    assert torch.equal(kernels.embedding(tokens[0, 0, 0], w), w[tokens[0, 0, 0]])
    assert kernels.embedding(tokens[:0], w).shape == (0, 6, 3, 80)
    leaf = w.clone().requires_grad_()
    for dout in (torch.ones(4, 6, 3, 64, device="cuda"), torch.ones((), device="cuda").expand(4, 6, 3, 64),
                 torch.randn(4, 6, 3, 70, device="cuda")[..., 5:69], torch.randn(64, 3, 6, 4, device="cuda").permute(3, 2, 1, 0)):
        (dw,) = torch.autograd.grad(kernels.embedding(tokens, leaf[:, 3:67]), leaf, dout)
        assert (dw[:, :3] == 0).all() and (dw[:, 67:] == 0).all()
        check(dw[:, 3:67], tokens, dout, 1.0, 50)
    for empty in (torch.zeros(0, dtype=torch.int64, device="cuda"), torch.zeros(3, 0, dtype=torch.int32, device="cuda")):
        out = kernels.embedding(empty, leaf)
        (dw,) = torch.autograd.grad(out, leaf, torch.zeros_like(out))
        assert (dw == 0).all()
    assert kernels.embedding(tokens, torch.zeros(0, 7, device="cuda")).isnan().all()
    assert kernels.embedding(tokens, torch.zeros(5, 0, device="cuda")).shape == (4, 6, 3, 0)


def test_same_bits_and_captured(kernels):
    tokens = words(20000, 5000, "rank")
    dout = torch.randn(20000, 96, device="cuda", generator=gen(3)).bfloat16()
    w = torch.randn(5000, 96, device="cuda").bfloat16()
    out, dw = grad(kernels, tokens, w, dout, 2.0)
    for _ in range(3):
        assert torch.equal(grad(kernels, tokens, w, dout, 2.0)[1], dw)
    static = tokens.clone()
    leaf = w.clone().requires_grad_()
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        y = kernels.embedding(static, leaf, 2.0)
        (got,) = torch.autograd.grad(y, leaf, dout)
    other = words(20000, 5000, "even", 9)
    for t in (tokens, other, tokens):
        static.copy_(t)
        g.replay()
        want = grad(kernels, t, w, dout, 2.0)
        assert torch.equal(y.detach(), want[0]) and torch.equal(got, want[1])


def test_rows_beyond_31_bits(kernels):
    """A table of more than 2^31 values, and rows of it on both sides of that."""
    V, D = 70000, 40000
    w = torch.empty(V, D, dtype=torch.bfloat16, device="cuda")
    at = torch.tensor([0, 53686, 53687, 53688, V - 1], device="cuda")
    w[at] = torch.arange(5 * 64, device="cuda", dtype=torch.bfloat16).repeat_interleave(D // 64).view(5, D)
    out = kernels.embedding(at, w)
    assert torch.equal(out, w[at])
    leaf = w.requires_grad_()
    (dw,) = torch.autograd.grad(kernels.embedding(at, leaf), leaf, out)
    assert torch.equal(dw[at], w[at])
    assert not dw[53680:53686].any() and not dw[53689:53700].any() and not dw[1:5].any() and not dw[V - 5:V - 1].any()


def test_refusals(kernels):
    w = torch.zeros(5, 4, device="cuda")
    t = torch.zeros(3, dtype=torch.int64, device="cuda")
    for tokens, weight in ((t, w[0]), (t.float(), w), (t.cpu(), w), (t, w.cpu()), (t, w.double()), (t, w.long())):
        with pytest.raises((ValueError, TypeError)):
            kernels.embedding(tokens, weight)
    with pytest.raises(ValueError, match="scale"):
        kernels.embedding(t, w, float("nan"))
    x = w.requires_grad_()
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(kernels.embedding(t, x).sum(), x, create_graph=True)


def test_views_with_a_sign(kernels):
    """The imaginary part of a conjugate is a view whose sign is not in memory: it counts in rows and gradients."""
    view = lambda t: torch.complex(torch.zeros_like(t), -t).conj().imag  # noqa: E731
    w, tokens, dout = torch.randn(9, 1, device="cuda"), words(40, 9, "even"), torch.randn(40, 1, device="cuda")
    assert view(w).is_neg()
    out, dw = grad(kernels, tokens, w, dout, 1.5)
    assert torch.equal(kernels.embedding(tokens, view(w), 1.5), out)
    assert torch.equal(grad(kernels, tokens, w, view(dout), 1.5)[1], dw)
