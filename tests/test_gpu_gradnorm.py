"""The norm of many gradients, clipping, and the AdamW step that takes the factor.

The norm: squares of up to eight values are added in fp32 (8 roundings of 2^-24 of
their sum), the rest in fp64; the root halves a relative error; one rounding to
fp32: 5 * 2^-24. Scaled values: the factor has the norm's error and its own
rounding, 7 * 2^-24, the product one more, the store half a step."""
from __future__ import annotations

import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

H = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def kernels():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from sunnynet_b200 import kernels
    return kernels


def true_norm(grads):
    return math.sqrt(sum(float(g.double().square().sum()) for g in grads))


def near(norm, grads):
    want = true_norm(grads)
    assert norm.dtype == torch.float32 and norm.dim() == 0
    assert abs(float(norm) - want) <= 5 * H * want, (float(norm), want)


LISTS = [[1], [5, 0, 3], [4096], [4097], [8, 1, 4095, 100000], [3] * 33, [17] * 1281, [1000] * 2600, [5000001], [0, 0]]


@pytest.mark.parametrize("sizes", LISTS)
@pytest.mark.parametrize("mixed", [False, True])
def test_norm_and_clipping(kernels, sizes, mixed):
    g = torch.Generator(device="cuda").manual_seed(len(sizes))
    r = lambda n: torch.randn(n, device="cuda", generator=g)  # noqa: E731
    for dtype in DTYPES:
        grads = [r(n).to(DTYPES[i % 3] if mixed else dtype) for i, n in enumerate(sizes)]
        want = true_norm(grads)
        norm, factor = kernels.grad_norm(grads)
        near(norm, grads)
        assert float(factor) == 1.0
        norm, factor = kernels.grad_norm(iter(grads), want / 3)
        near(norm, grads)
        f = min(1.0, want / 3 / (want + 1e-6))
        assert abs(float(factor) - f) <= 7 * H * f
        before = [x.clone() for x in grads]
        kernels.clip_grads(grads, want * 1.01 + 1)
        assert all(torch.equal(a, b) for a, b in zip(grads, before))
        near(kernels.clip_grads(grads, want / 3), before)
        for a, b in zip(grads, before):
            e = torch.finfo(a.dtype).eps / 2
            to = b.double() * f
            err = 8 * H * to.abs()
            tiny = torch.finfo(a.dtype).smallest_normal * e
            assert ((a.double() - to).abs() <= err + e * (to.abs() + err) + tiny).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_odd_addresses_and_dense_orders(kernels, dtype):
    """Views into one buffer at every offset; transposed tensors; what lies between stays."""
    flat = torch.randn(200000, device="cuda").to(dtype)
    cuts = [(1, 2), (3, 20), (25, 4200), (5001, 9000), (9003, 9003), (10007, 80021), (80022, 199999)]
    kept = flat.clone()
    grads = [flat[a:b] for a, b in cuts]
    grads[-2] = grads[-2][:70000].view(7, 100, 100).permute(2, 0, 1)
    near(kernels.grad_norm(grads, 1.0)[0], grads)
    kernels.clip_grads(grads, 0.0)
    inside = torch.zeros(200000, dtype=torch.bool, device="cuda")
    for a, b in cuts[:-2] + [(10007, 80007)] + cuts[-1:]:
        inside[a:b] = True
    assert (flat[inside] == 0).all() and torch.equal(flat[~inside], kept[~inside])


def test_magnitudes(kernels):
    """Squares beyond fp32's range count, zeros among them or not."""
    for size in (1e-45, 1e-30, 1e-20, 1.0, 1e18, 1e30, 3e38):
        x = torch.full((10001,), size, device="cuda")
        x[::3] = 0.0
        norm = kernels.grad_norm([x])[0]
        want = true_norm([x])
        assert abs(float(norm) - want) <= 5 * H * want + 2.0 ** -150 or want > 3.4e38 and float(norm) == math.inf
    x = torch.zeros(5000, device="cuda")
    x[7], x[8] = 1e-25, 1.0
    near(kernels.grad_norm([x])[0], [x])


def test_values_that_are_not_numbers(kernels):
    x = torch.ones(100, device="cuda")
    x[50] = float("nan")
    norm, factor = kernels.grad_norm([torch.ones(5, device="cuda"), x], 1.0)
    assert norm.isnan() and factor.isnan()
    x[50] = float("inf")
    norm, factor = kernels.grad_norm([x], 1.0)
    assert norm.isinf() and factor == 0
    assert kernels.grad_norm([x])[1] == 1
    kernels.clip_grads([x], 1.0)
    assert x[50].isnan() and (x[:50] == 0).all()
    z = torch.zeros(9, device="cuda")
    norm, factor = kernels.grad_norm([z], 0.0)
    assert norm == 0 and factor == 0
    assert kernels.grad_norm([z], 1.0)[1] == 1


def test_refusals(kernels):
    x = torch.ones(8, device="cuda")
    for bad in ([x.cpu()], [x.double()], [x, x.cpu()], [torch.ones(4, 4, device="cuda")[:, :2]], [x.expand(3, 8)], [1.0],
                [torch.ones(3, device="cuda").to_sparse()], []):
        with pytest.raises((ValueError, TypeError)):
            kernels.grad_norm(bad)
    for bad in ([x, x], [x, x[4:]]):
        with pytest.raises(ValueError, match="twice"):
            kernels.clip_grads(bad, 1.0)
    assert abs(float(kernels.grad_norm([x, x])[0]) - 4.0) < 1e-5  # reading twice is fine
    for m in (-1.0, float("nan")):
        with pytest.raises(ValueError):
            kernels.grad_norm([x], m)
    w = torch.ones(8, device="cuda", requires_grad=True)
    y = (w * x).sum()
    kernels.clip_grads([x], 0.5)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.backward()


def test_same_bits_captured_and_side_by_side(kernels):
    grads = [torch.randn(n, device="cuda").bfloat16() for n in (1000003, 77, 5000)] + [torch.randn(100000, device="cuda")]
    first = [x.clone() for x in grads]
    want = kernels.grad_norm(grads, 1.0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = kernels.clip_grads(grads, 1.0)
    for _ in range(3):
        for x, y in zip(grads, first):
            x.copy_(y)
        graph.replay()
        assert torch.equal(norm, want[0])
        a = [x.clone() for x in grads]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for x, y in zip(grads, first):
            x.copy_(y)
        kernels.clip_grads(grads, 1.0)
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(a, grads))


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", DTYPES)
def test_the_optimiser_takes_the_factor(kernels, bits, dtype):
    """A step with the factor is a step of gradients multiplied by it (in fp32)."""
    from sunnynet_b200.optim import AdamW
    gen = torch.Generator(device="cuda").manual_seed(3)
    shapes = [(257, 130), (5,), (64, 64), (3, 1001)]
    start = [torch.randn(*s, device="cuda", generator=gen) for s in shapes]
    grads = [torch.randn(*s, device="cuda", generator=gen).to(dtype) for s in shapes]
    sides = []
    for fused in (True, False):
        params = [torch.nn.Parameter(x.clone()) for x in start]
        m, v = ([torch.zeros_like(x) for x in start] for _ in range(2))
        scales = {}
        if bits == 8:
            m, v = ([torch.zeros(x.shape, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for x in start] for _ in range(2))
            scales = {k: [torch.zeros(-(-x.numel() // 256), device="cuda") for x in start] for k in ("avg_scale", "sq_scale")}
        _, factor = kernels.grad_norm(grads, 0.7)
        with torch.no_grad():
            for step in (1, 2):
                if fused:
                    kernels.adamw_step(params, grads, m, v, step, grad_scale=factor, **scales)
                else:
                    kernels.adamw_step(params, [g.float() * factor for g in grads], m, v, step, **scales)
        sides.append(params + m + v + [x for s in scales.values() for x in s])
    for a, b in zip(*sides):
        assert torch.equal(a.detach().view(torch.uint8) if a.element_size() == 1 else a.detach(),
                           b.detach().view(torch.uint8) if b.element_size() == 1 else b.detach())
    if dtype == torch.float32:
        params = [torch.nn.Parameter(x.clone()) for x in start]
        opt = AdamW([{"params": params[:2]}, {"params": params[2:], "weight_decay": 0.01}], state_bits=bits, max_norm=0.7)
        for p, g in zip(params, grads):
            p.grad = g.clone()
        opt.step()
        near(opt.grad_norm, grads)
        assert all(torch.equal(p.grad, g) for p, g in zip(params, grads))
        opt.step()
        assert all(torch.equal(a.detach(), b.detach()) for a, b in zip(params, sides[0]))
    for bad in (factor.double(), factor.cpu(), torch.ones(2, device="cuda"), grads[0]):
        with pytest.raises(TypeError, match="grad_scale"):
            kernels.adamw_step([start[0]], [grads[0]], [torch.zeros_like(start[0])], [torch.zeros_like(start[0])], 1, grad_scale=bad)
    with pytest.raises(ValueError):
        AdamW([torch.nn.Parameter(start[0])], max_norm=-1.0)


def test_a_factor_that_is_no_tensor(kernels):
    x = [torch.ones(4, device="cuda") for _ in range(4)]
    for bad in (0.5, [1.0], "1"):
        with pytest.raises(TypeError, match="grad_scale"):
            kernels.adamw_step(*([t] for t in x), 1, grad_scale=bad)
    assert all(torch.equal(t, torch.ones_like(t)) for t in x)
