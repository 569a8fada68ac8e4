"""Layer norm and its gradients on the GPU against the formulas in 64 bits.

Tolerances are worst-case rounding bounds, formed element by element from the
64-bit values (h = 2^-24, a rounding of fp32; e = eps of the stored type / 2):
with A = max|x| / sd of a row, and sums whose longest chain has d roundings,
  |centred - true| <= h (d + 2) max|x|
  |xhat - true|    <= h ((d + 2) A (1 + |xhat|) + |xhat| (d + 8) / 2)
and so on below, each times the factor it meets on its way to the output, plus
e |output| for the store. d: 32 values of a thread (or D / 512 of the widest
form), 5 shuffles, up to 16 warps, and a few operations.
"""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

H = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def norm():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from sunnynet_b200.kernels import layer_norm
    return layer_norm


def truth(x, w, b, eps, dy=None):
    """(y, dx, dw, db) in fp64 and the bound of each one's error before it is stored."""
    x = x.double()
    D = x.shape[1]
    w = torch.ones(D, dtype=torch.float64, device=x.device) if w is None else w.double()
    b = torch.zeros_like(w) if b is None else b.double()
    d = 60 + D / 512
    mean = x.mean(1, keepdim=True)
    sd = ((x - mean).square().mean(1, keepdim=True) + eps).sqrt()
    xh = (x - mean) / sd
    A = x.abs().amax(1, keepdim=True) / sd
    exh = H * ((d + 2) * A * (1 + xh.abs()) + xh.abs() * (d + 8) / 2)
    y = xh * w + b
    ey = exh * w.abs() + 3 * H * ((xh * w).abs() + b.abs())
    if dy is None:
        return y, ey
    dy = dy.double()
    du = dy * w
    s1, s2 = du.mean(1, keepdim=True), (du * xh).mean(1, keepdim=True)
    dx = (du - s1 - xh * s2) / sd
    es1 = H * (d + 2) * du.abs().mean(1, keepdim=True)
    es2 = H * (d + 3) * (du * xh).abs().mean(1, keepdim=True) + (du.abs() * exh).mean(1, keepdim=True)
    rstd = H * (2 * (d + 2) * A + (d + 8) / 2)  # relative
    edx = (4 * H * (du.abs() + s1.abs() + (xh * s2).abs()) + es1 + xh.abs() * es2 + s2.abs() * exh
           + rstd * (du - s1 - xh * s2).abs()) / sd
    n = x.shape[0] + 40  # roundings of a sum down the rows, in whatever order
    dw, db = (dy * xh).sum(0), dy.sum(0)
    edw = (dy.abs() * exh).sum(0) + H * n * (dy * xh).abs().sum(0)
    edb = H * n * dy.abs().sum(0)
    return (y, dx, dw, db), (ey, edx, edw, edb)


def near(got, want, err, dtype):
    e = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps  # below normal numbers
    assert got.dtype == dtype
    bad = (got.double() - want).abs() > err + e * (want.abs() + err) + tiny
    assert not bad.any(), (int(bad.sum()), float((got.double() - want).abs().max()))


def inputs(rows, D, dtype, wdtype, seed, shift=0.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    return ((r(rows, D) * 2 + shift).to(dtype), (1 + 0.2 * r(D)).to(wdtype),
            (0.3 * r(D)).to(wdtype), r(rows, D).to(dtype))


# each form of the kernels: lanes of a warp, a warp, a CTA, the widest; packed and single elements
SHAPES = [(1, 1), (3, 2), (5, 7), (301, 8), (77, 16), (130, 24), (9, 33), (65, 64), (40, 100),
          (257, 128), (33, 250), (19, 384), (600, 512), (31, 768), (7, 1000), (12, 1001),
          (300, 1024), (11, 1536), (5, 2047), (64, 2048), (4, 4096), (3, 5001), (3, 8192),
          (2, 9000), (3, 8201), (2, 16384), (2, 16390), (2, 33000)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,D", SHAPES)
def test_forward_and_gradients(norm, rows, D, dtype):
    x, w, b, dy = inputs(rows, D, dtype, torch.float32, D)
    x.requires_grad_(), w.requires_grad_(), b.requires_grad_()
    y = norm(x, w, b, 1e-3)
    got = (y, *torch.autograd.grad(y, (x, w, b), dy))
    want, err = truth(x.detach(), w.detach(), b.detach(), 1e-3, dy)
    for g, t, e, kind in zip(got, want, err, (dtype, dtype, torch.float32, torch.float32)):
        near(g.detach(), t, e, kind)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,D", [(100, 96), (41, 1001), (16, 2048), (4, 9000)])
def test_weights_of_the_rows_type(norm, rows, D, dtype):
    x, w, b, dy = inputs(rows, D, dtype, dtype, D)
    x.requires_grad_(), w.requires_grad_(), b.requires_grad_()
    y = norm(x, w, b)
    got = (y, *torch.autograd.grad(y, (x, w, b), dy))
    want, err = truth(x.detach(), w.detach(), b.detach(), 1e-5, dy)
    for g, t, e in zip(got, want, err):
        near(g.detach(), t, e, dtype)


@pytest.mark.parametrize("rows,D", [(37, 512), (8, 1001), (3, 10000)])
def test_without_weight_or_bias_and_single_gradients(norm, rows, D):
    x, w, b, dy = inputs(rows, D, torch.float32, torch.float32, 1)
    for ww, bb in ((None, None), (w, None), (None, b)):
        want, err = truth(x, ww, bb, 1e-5, dy)
        near(norm(x, ww, bb), want[0], err[0], torch.float32)
        for leaf in range(3):
            args = [t.detach().clone() if t is not None else None for t in (x, ww, bb)]
            if args[leaf] is None:
                continue
            args[leaf].requires_grad_()
            g, = torch.autograd.grad(norm(*args), args[leaf], dy)
            near(g, want[1 + leaf], err[1 + leaf], torch.float32)


@pytest.mark.parametrize("D", [3, 40, 1001])
def test_gradients_against_differences(norm, D):
    """Central differences of the definition in 64 bits (step 1e-5: their own
    error is about 1e-9 of the loss's curvature, below the fp32 bounds)."""
    x, w, b, dy = inputs(6, D, torch.float32, torch.float32, 5)
    x.requires_grad_(), w.requires_grad_(), b.requires_grad_()
    grads = torch.autograd.grad(norm(x, w, b, 1e-2), (x, w, b), dy)
    at = [t.detach().double() for t in (x, w, b)]

    def loss(x, w, b):
        c = x - x.mean(1, keepdim=True)
        return ((c / (c.square().mean(1, keepdim=True) + 1e-2).sqrt() * w + b) * dy.double()).sum()

    _, err = truth(*at, 1e-2, dy)
    rng = np.random.default_rng(0)
    for which, g in enumerate(grads):
        for i in rng.choice(g.numel(), min(12, g.numel()), replace=False):
            up, down = [t.clone() for t in at], [t.clone() for t in at]
            up[which].view(-1)[i] += 1e-5
            down[which].view(-1)[i] -= 1e-5
            diff = (loss(*up) - loss(*down)) / 2e-5
            bound = err[1 + which].reshape(-1)[i] + H * g.reshape(-1)[i].abs() + 1e-7 * dy.abs().sum()
            assert abs(diff - g.reshape(-1)[i]) <= bound, (which, i)


@pytest.mark.parametrize("dtype", DTYPES)
def test_strided_rows_and_shapes(norm, dtype):
    x, w, b, dy = inputs(60, 200, dtype, torch.float32, 9)
    for view, grad in ((x[:, 3:190], dy[:, 5:192]), (x[::2, :187], dy[1::2, 1:188]),
                       (x.view(3, 20, 200)[:, 4:9, 8:128], dy.view(3, 20, 200)[:, 1:6, 8:128]),
                       (x.view(5, 12, 200).transpose(0, 1), dy.view(5, 12, 200).transpose(0, 1))):
        D = view.shape[-1]
        leaf = view.detach().requires_grad_()
        ww = w[:D].clone().requires_grad_()
        y = norm(leaf, ww, b[:D])
        assert y.shape == view.shape and y.is_contiguous()
        gx, gw = torch.autograd.grad(y, (leaf, ww), grad)
        want, err = truth(view.reshape(-1, D), w[:D], b[:D], 1e-5, grad.reshape(-1, D))
        near(y.detach().reshape(-1, D), want[0], err[0], dtype)
        near(gx.reshape(-1, D), want[1], err[1], dtype)
        near(gw, want[2], err[2], torch.float32)
    # a sum's gradient is one value at strides of zero
    leaf = x.detach().requires_grad_()
    g, = torch.autograd.grad(norm(leaf, w, b).sum(), leaf)
    want, err = truth(x, w, b, 1e-5, torch.ones_like(x))
    near(g, want[1], err[1], dtype)
    # one row given to many
    leaf = x[:1].detach().requires_grad_()
    y = norm(leaf.expand(60, 200), w, b)
    g, = torch.autograd.grad(y, leaf, dy.float().to(dtype))
    want, err = truth(x[:1].expand(60, 200), w, b, 1e-5, dy)
    e = torch.finfo(dtype).eps / 2
    bound = err[1].sum(0) + 61 * e * want[1].abs().sum(0)  # torch adds the 60 rows in dtype
    assert ((g[0].double() - want[1].sum(0)).abs() <= bound + 60 * torch.finfo(dtype).smallest_normal).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,D", [(30001, 7), (20000, 33), (9477, 250), (5003, 1001), (2500, 2047),
                                    (1190, 5003)])
def test_many_rows_of_an_odd_width(norm, rows, D, dtype):
    """Rows that a group of threads walks, the last of them not all alike; the
    rows and the weights of a view, of both types, and with one of the two only."""
    x, w, b, _ = inputs(rows, D + 5, dtype, torch.float32, 2)
    for off, ww, bb in ((0, w, b), (3, w.to(dtype), b.to(dtype)), (5, None, b), (1, w, None)):
        view = x[:, off:off + D]
        ww, bb = (t if t is None else t[off:off + D] for t in (ww, bb))
        want, err = truth(view, ww, bb, 1e-5)
        near(norm(view, ww, bb), want, err, dtype)


def test_no_rows_constant_rows_and_large_means(norm):
    w, b = torch.rand(48, device="cuda").requires_grad_(), torch.rand(48, device="cuda").requires_grad_()
    x = torch.empty(0, 48, device="cuda", requires_grad=True)
    y = norm(x, w, b)
    gx, gw, gb = torch.autograd.grad(y, (x, w, b), torch.empty(0, 48, device="cuda"))
    assert y.shape == gx.shape == (0, 48) and not gw.any() and not gb.any()
    # powers of two: the mean is exact, the rows' variance 0
    x = torch.full((4, 64), 8.0, device="cuda")
    assert torch.equal(norm(x, None, b[:1].detach().expand(64).contiguous()),
                       b[:1].detach().expand(4, 64))
    x = 1000 + torch.randn(32, 768, device="cuda")
    want, err = truth(x, None, None, 1e-5)
    near(norm(x), want, err, torch.float32)


def test_nan_and_infinity_stay_in_their_rows(norm):
    x = torch.randn(9, 1000, device="cuda")
    clean = norm(x)
    x[2, 5], x[6, 999] = float("nan"), float("inf")
    y = norm(x)
    for r in range(9):
        assert torch.isnan(y[r]).any() if r in (2, 6) else torch.equal(y[r], clean[r])


@pytest.mark.parametrize("rows,D,dtype", [(4000, 768, torch.bfloat16), (3000, 1001, torch.float32)])
def test_same_bits_every_time_and_replayed(norm, rows, D, dtype):
    x, w, b, dy = inputs(rows, D, dtype, torch.float32, 3)
    for t in (x, w, b):
        t.requires_grad_()

    def step():
        y = norm(x, w, b)
        return (y, *torch.autograd.grad(y, (x, w, b), dy))

    first = [t.detach().clone() for t in step()]
    assert all(torch.equal(a, c) for a, c in zip(first, step()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(first, held))
    with torch.no_grad():
        x.copy_(x.flip(0))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(step(), held))


def test_host_tensors_are_staged(norm):
    x, w, b, dy = (t.cpu() for t in inputs(10, 96, torch.float32, torch.float32, 2))
    x.requires_grad_(), w.requires_grad_()
    y = norm(x, w, b)
    gx, gw = torch.autograd.grad(y, (x, w), dy)
    assert not y.is_cuda and not gx.is_cuda and not gw.is_cuda
    want, err = truth(x.detach(), w.detach(), b, 1e-5, dy)
    near(y.detach(), want[0], err[0], torch.float32)
    near(gx, want[1], err[1], torch.float32)
    near(gw, want[2], err[2], torch.float32)


def test_differentiated_once_and_inputs_unchanged(norm):
    x, w, b, dy = inputs(8, 40, torch.float32, torch.float32, 11)
    x.requires_grad_(), w.requires_grad_()
    y = norm(x, w, b)
    with pytest.raises(RuntimeError, match="differentiated once"):
        torch.autograd.grad(y, x, dy, create_graph=True)
    y = norm(x, w, b)
    with torch.no_grad():
        x.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        torch.autograd.grad(y, x, dy)
    with torch.no_grad():
        assert not norm(x, w, b).requires_grad
    assert not norm(x.detach(), w.detach(), b).requires_grad


def test_two_threads_on_streams_of_their_own(norm):
    import threading

    from sunnynet_b200.kernels import adamw_step
    from sunnynet_b200.sampling import sample

    def run(seed, out):
        with torch.cuda.stream(torch.cuda.Stream()):
            x, w, b, dy = inputs(700, 515, torch.bfloat16, torch.float32, seed)
            x.requires_grad_(), w.requires_grad_(), b.requires_grad_()
            m, v = torch.zeros_like(w), torch.zeros_like(w)
            u = torch.linspace(0, 0.99, 700, device="cuda")
            for t in range(1, 30):
                y = norm(x, w, b)
                gx, gw, gb = torch.autograd.grad(y, (x, w, b), dy)
                adamw_step([w.detach()], [gw], [m], [v], t)
                tokens = sample(y.detach(), u, top_k=9, top_p=0.9)
            torch.cuda.current_stream().synchronize()
            out.append([a.detach().clone() for a in (y, gx, gb, w, tokens)])
            torch.cuda.current_stream().synchronize()

    alone, beside = [[], []], [[], []]
    for s in range(2):
        run(s, alone[s])
    threads = [threading.Thread(target=run, args=(s, beside[s])) for s in range(2)]
    [t.start() for t in threads], [t.join() for t in threads]
    for a, c in zip(alone, beside):
        assert all(torch.equal(p, q) for p, q in zip(a[0], c[0]))


def test_refusals(norm):
    x, w = torch.randn(4, 8, device="cuda"), torch.ones(8, device="cuda")
    for bad in (lambda: norm(x.double()), lambda: norm(x, w[:7]), lambda: norm(x, w.half()),
                lambda: norm(x, w.cpu()), lambda: norm(x, w, w.bfloat16()), lambda: norm(x[:, :0]),
                lambda: norm(x.sum()), lambda: norm(x, w, None, -1.0),
                lambda: norm(x[:1, :1].expand(1, 1 << 32))):
        with pytest.raises((ValueError, TypeError)):
            bad()
    from sunnynet_b200 import _lib
    L = _lib.load()
    y, s = torch.empty_like(x), torch.empty(2, 4, device="cuda")
    host = np.zeros((4, 8), np.float32)
    assert L.sn_abi_layer_norm(host.ctypes.data, 8, None, None, y.data_ptr(), None, None, 0, 0, 4, 8,
                               1e-5, None) == -1
    assert "device memory" in _lib.last_error()
    assert L.sn_abi_layer_norm(x.data_ptr() + 2, 8, None, None, y.data_ptr(), None, None, 0, 0, 3, 8,
                               1e-5, None) == -1
    assert "aligned" in _lib.last_error()
    assert L.sn_abi_layer_norm_bwd(x.data_ptr(), 8, x.data_ptr(), 8, None, s.data_ptr(),
                                   s.data_ptr(), None, w.data_ptr(), None, None, 0, 0, 0, 4, 8,
                                   None) == -1
    assert "workspace" in _lib.last_error()
