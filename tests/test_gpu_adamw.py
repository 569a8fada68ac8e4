"""adamw_step and optim.AdamW on the GPU.

Every operation of the update is one correctly rounded fp32 operation, so the
same operations in torch give the same bits: the kernels are held to that, and
those torch operations to the formulas in 64 bits (see the bounds there).
"""
from __future__ import annotations

import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

BLOCK = 256
F8 = torch.float8_e4m3fn
RULE = {"lr": 3e-3, "beta1": 0.9, "beta2": 0.95, "eps": 1e-8, "weight_decay": 0.1}
KINDS = [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16),
         (torch.float16, torch.float16), (torch.bfloat16, torch.float32),
         (torch.float32, torch.bfloat16)]
SIZES = [1, 3, 4, 255, 256, 257, 0, 1000, 1024, 4096, 4097, 70001, 300000]


@pytest.fixture(scope="module")
def adamw_step():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from sunnynet_b200.kernels import adamw_step
    return adamw_step


def encode(x, floor):
    b = torch.nn.functional.pad(x, (0, -x.numel() % BLOCK)).view(-1, BLOCK)
    scale = b.abs().amax(1) * torch.tensor(1 / 448, dtype=torch.float32, device=x.device)
    q = torch.where(scale[:, None] > 0, b / scale[:, None], 0.0)
    if floor:
        q = torch.where(b > 0, q.clamp_min(2.0 ** -9), q)
    return q.view(-1)[:x.numel()].to(F8), scale


def decode(codes, scale):
    return codes.float() * scale.repeat_interleave(BLOCK)[:codes.numel()]


def update(p, g, m, v, t, lr, beta1, beta2, eps, weight_decay):
    """(p, m, v, sqrt v) of one step, each operation rounded in fp32."""
    m = m * beta1 + g * (1 - beta1)
    v = v * beta2 + g.square() * (1 - beta2)
    r = v.sqrt()
    p = p * (1 - lr * weight_decay) - m / (r * (1 / math.sqrt(1 - beta2 ** t)) + eps) * (
        lr / (1 - beta1 ** t))
    return p, m, v, r


def make(sizes, kind, bits, seed=0, offset=0):
    """Lists params, grads, avg, sq (, avg_scale, sq_scale); offset: elements the tensors lie off 16 bytes."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def place(x):
        room = torch.zeros(x.numel() + 16, dtype=x.dtype, device="cuda")
        out = room[offset:offset + x.numel()]
        out.copy_(x)
        return out

    lists = [[] for _ in range(6 if bits == 8 else 4)]
    for n in sizes:
        r = lambda: torch.randn(n, device="cuda", generator=g)  # noqa: B023,E731
        used = torch.rand(n, device="cuda", generator=g) > 0.2
        p, grad, m, v = r() * 0.05, r() * 1e-2 * used, r() * 1e-3 * used, (r() * 1e-2).square() * used
        row = [p.to(kind[0]), grad.to(kind[1]), m, v]
        if bits == 8:
            (m, ms), (r_, rs) = encode(m, False), encode(v.sqrt(), True)
            row = [*row[:2], m, r_, ms, rs]
        for to, x in zip(lists, row):
            to.append(place(x) if x.dtype != F8 else place(x.view(torch.uint8)).view(F8))
    return lists


def expected(lists, t, rule):
    out = []
    for row in zip(*lists):
        p, g, m, v = row[0].float(), row[1].float(), row[2], row[3]
        if len(row) == 6:
            m, v = decode(row[2], row[4]), decode(row[3], row[5]).square()
        p, m, v, r = update(p, g, m, v, t, **rule)
        p = p.to(row[0].dtype)
        if len(row) == 6:
            (m, ms), (r, rs) = encode(m, False), encode(r, True)
            out.append((p, None, m, r, ms, rs))
        else:
            out.append((p, None, m, v))
    return out


def call(adamw_step, lists, t, **rule):
    scales = {"avg_scale": lists[4], "sq_scale": lists[5]} if len(lists) == 6 else {}
    adamw_step(*lists[:4], t, **scales, **rule)


def same(a, b):
    if a.dtype == F8:
        a, b = a.view(torch.uint8), b.view(torch.uint8)
    return torch.equal(a, b)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("offset", [0, 3])
def test_bits_of_the_update(adamw_step, kind, bits, offset):
    lists = make(SIZES, kind, bits, 1, offset)
    grads = [g.clone() for g in lists[1]]
    for t in (1, 2, 1000):
        want = expected(lists, t, RULE)
        call(adamw_step, lists, t, **RULE)
        for row, w in zip(zip(*lists), want):
            for a, b in zip(row, w):
                assert b is None or same(a, b), (row[0].numel(), t)
    assert all(torch.equal(a, b) for a, b in zip(lists[1], grads))


def test_roots_and_quotients_of_every_size(adamw_step):
    """p = -(m / 2) / (2 sqrt(3 v / 4) + eps), each operation rounded once (the
    rates are powers of two), for magnitudes inside and outside 2^-80 .. 2^80,
    against torch's division and root, which round correctly."""
    n = 1 << 21
    g = torch.Generator(device="cuda").manual_seed(3)
    r = lambda: torch.rand(n, device="cuda", generator=g, dtype=torch.float64)  # noqa: E731
    for lo, hi in ((-75, 75), (-20, 4), (-130, 120)):
        m = ((r() - 0.5).sign() * (1 + r()) * 2.0 ** (lo + (hi - lo) * r()).floor()).float()
        v = ((1 + r()) * 2.0 ** (lo + (hi - lo) * r()).floor()).float()
        for eps in (1e-8, 0.0):
            p, state = torch.zeros(n, device="cuda"), [m.clone(), v.clone()]
            adamw_step([p], [torch.zeros(n, device="cuda")], state[:1], state[1:], 1, lr=0.5,
                       beta1=0.5, beta2=0.75, eps=eps, weight_decay=0.0)
            want = 0 - (m * 0.5) / ((v * 0.75).sqrt() * 2.0 + torch.tensor(eps, device="cuda"))
            assert torch.equal(p, want), (lo, hi, eps)
            assert torch.equal(state[0], m * 0.5) and torch.equal(state[1], v * 0.75)


def test_a_step_is_seen_by_autograd(adamw_step):
    """A graph that saved a parameter refuses its backward pass after the step."""
    p, g, m, v = make([64], KINDS[0], 32)
    p[0].requires_grad_()
    loss = (p[0] * p[0]).sum()
    adamw_step([p[0].detach()], g, m, v, 1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        loss.backward()


@pytest.mark.parametrize("bits", [32, 8])
def test_a_large_launch_and_many_tensors(adamw_step, bits):
    """The wide chunks, and more tensors than one launch takes."""
    for sizes in ([5_000_001, 1_000_000], [1 + 37 * i % 600 for i in range(1100)]):
        lists = make(sizes, KINDS[0], bits, 2)
        want = expected(lists, 7, RULE)
        call(adamw_step, lists, 7, **RULE)
        assert all(b is None or same(a, b) for row, w in zip(zip(*lists), want) for a, b in zip(row, w))


def test_formula_in_64_bits(adamw_step):
    """h = 2^-24. m: two products and a sum, 2h(|m b1| + |g c|); v alike, one
    rounding more; m / (...) * size is then off by at most 12 h of itself (m 2,
    root 1.5, product, sum, quotient, product, the rates' own roundings) where
    the sum that makes m does not cancel, so m's own error is carried apart; p:
    the decayed p, the difference."""
    h = 2.0 ** -24
    lists = make([100003], KINDS[0], 32, 3)
    p, g, m, v = (x[0].double() for x in lists)
    call(adamw_step, lists, 11, **RULE)
    em = 3 * h * (m.abs() * RULE["beta1"] + g.abs() * (1 - RULE["beta1"]))
    m = m * RULE["beta1"] + g * (1 - RULE["beta1"])
    v = v * RULE["beta2"] + g ** 2 * (1 - RULE["beta2"])
    size = RULE["lr"] / (1 - RULE["beta1"] ** 11)
    under = (v / (1 - RULE["beta2"] ** 11)).sqrt() + RULE["eps"]
    to = m / under * size
    new = p * (1 - RULE["lr"] * RULE["weight_decay"]) - to
    assert ((lists[2][0].double() - m).abs() <= em).all()
    assert ((lists[3][0].double() - v).abs() <= 4 * h * v).all()
    assert ((lists[0][0].double() - new).abs() <=
            h * (2 * p.abs() + new.abs() + 12 * to.abs()) + em / under * size).all()


def test_codes_are_within_their_step(adamw_step):
    """An e4m3 code is off by at most 2^-4 of the value (2^-10 of the scale near
    zero); a root above zero keeps at least 2^-9 of the scale."""
    lists = make([70001], KINDS[0], 8, 4)
    p, g = lists[0][0].float(), lists[1][0].float()
    m, v = decode(lists[2][0], lists[4][0]), decode(lists[3][0], lists[5][0]).square()
    _, m, v, r = update(p, g, m, v, 5, **RULE)
    call(adamw_step, lists, 5, **RULE)
    for codes, scale, x, least in ((lists[2][0], lists[4][0], m, 0), (lists[3][0], lists[5][0], r, 1)):
        wide = scale.repeat_interleave(BLOCK)[:x.numel()]
        off = (codes.float() * wide - x).abs()
        bound = torch.maximum(x.abs() * 2.0 ** -4, wide * 2.0 ** (-9 if least else -10)) * (1 + 2.0 ** -20)
        assert (off <= bound).all()
    assert ((lists[3][0].float() > 0) == (r > 0)).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_zero_and_not_finite_gradients(adamw_step, bits):
    lists = make([1024, 600], KINDS[0], bits, 5)
    for x in lists[2:]:  # a block, and a whole tensor, that has seen nothing
        (x[0].view(torch.uint8) if x[0].dtype == F8 else x[0])[:256 if x[0].numel() > 4 else 1] = 0
        (x[1].view(torch.uint8) if x[1].dtype == F8 else x[1]).zero_()
    lists[1][0][:256] = 0
    lists[1][1].zero_()
    lists[1][0][300], lists[1][0][900] = float("nan"), float("inf")
    want = expected(lists, 3, RULE)
    call(adamw_step, lists, 3, **RULE)
    for row, w in zip(zip(*lists), want):
        for a, b in zip(row, w):
            if b is None:
                continue
            a, b = a.float(), b.float()
            assert torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(a.nan_to_num(7), b.nan_to_num(7))
    assert torch.isfinite(lists[0][1]).all() and torch.isfinite(lists[0][0][:256]).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_step_and_rate_on_the_gpu_in_a_graph(adamw_step, bits):
    """A captured step reads the step number and rate anew at each replay. The
    rates come from the GPU's pow in 64 bits: a last bit of one fp32 rate may
    differ, so p may by 3 roundings of the update and one of p, and codes by
    what that changes: only p and 32-bit states are compared."""
    a, b = make([4097, 300], KINDS[0], bits, 6), make([4097, 300], KINDS[0], bits, 6)
    step = torch.tensor([1], dtype=torch.int64, device="cuda")
    lr = torch.tensor([1e-3], dtype=torch.float64, device="cuda")
    rule = {k: v for k, v in RULE.items() if k != "lr"}
    warm = make([4097, 300], KINDS[0], bits, 6)
    call(adamw_step, warm, step, lr=lr, **rule)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(adamw_step, a, step, lr=lr, **rule)
        step.add_(1)
    for t in range(1, 4):
        lr.fill_(1e-3 * t)
        before = [p.clone() for p in b[0]]
        graph.replay()
        call(adamw_step, b, t, lr=1e-3 * t, **rule)
        torch.cuda.synchronize()
        for p, q, o in zip(a[0], b[0], before):
            bound = 2.0 ** -22 * t * ((q - o).abs() + q.abs() * 0.5)
            assert ((p - q).abs() <= bound).all()
        if bits == 32:
            for k in (2, 3):
                assert all(torch.equal(x, y) for x, y in zip(a[k], b[k]))
    assert step.item() == 4


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_optimizer_follows_torch(dtype):
    """Ten steps beside torch's AdamW. Per step the two formulas, equal in real
    numbers, differ by at most 16 roundings of the update (at most 4 lr here:
    |m'| / sqrt(v') with ten alike-sized gradients) and 3 of p, and p is
    rounded to its type in each: twice half a step of it."""
    from sunnynet_b200.optim import AdamW
    g = torch.Generator(device="cuda").manual_seed(1)
    start = [torch.randn(s, device="cuda", generator=g).to(dtype) * 0.1 for s in ((64, 33), (7,), (300, 5))]
    mine, his = ([x.clone().requires_grad_() for x in start] for _ in range(2))
    a = AdamW([{"params": mine[:2]}, {"params": mine[2:], "weight_decay": 0.0}], lr=1e-2, weight_decay=0.05)
    wide = [x.detach().float().requires_grad_() for x in his]  # torch's own states would be half precision
    b = torch.optim.AdamW([{"params": wide[:2]}, {"params": wide[2:], "weight_decay": 0.0}], lr=1e-2,
                          weight_decay=0.05)
    sched = torch.optim.lr_scheduler.StepLR(a, 4, 0.5), torch.optim.lr_scheduler.StepLR(b, 4, 0.5)
    e = torch.finfo(dtype).eps / 2
    for t in range(10):
        for i, (x, y) in enumerate(zip(mine, wide)):
            grad = torch.randn(x.shape, device="cuda", generator=g).to(dtype)
            x.grad = grad if (t, i) != (0, 1) else None  # a parameter that joins a step later
            y.grad = grad.float() if (t, i) != (0, 1) else None
        a.step(), b.step(), [s.step() for s in sched]
        h = 2.0 ** -24
        for x, y in zip(mine, wide):
            bound = (t + 1) * (16 * h * 4e-2 + 3 * h * (y.abs() + 1) + (2 * e * (y.abs() + 0.1) if dtype != torch.float32 else 0))
            assert ((x.double() - y.double()).abs() <= bound).all(), t


@pytest.mark.parametrize("bits", [32, 8])
def test_optimizer_state_saved_and_loaded(bits, tmp_path):
    from sunnynet_b200.optim import AdamW
    g = torch.Generator(device="cuda").manual_seed(2)
    start = [torch.randn(s, device="cuda", generator=g).bfloat16() for s in ((50, 40), (3,))]
    a = [x.clone().requires_grad_() for x in start]
    oa = AdamW(a, state_bits=bits)

    def step(params, opt, seed):
        r = torch.Generator(device="cuda").manual_seed(seed)
        for p in params:
            p.grad = torch.randn(p.shape, device="cuda", generator=r).bfloat16()
        opt.step()

    step(a, oa, 5)
    torch.save(oa.state_dict(), tmp_path / "opt.pt")
    b = [x.detach().clone().requires_grad_() for x in a]
    ob = AdamW(b, state_bits=bits)
    ob.load_state_dict(torch.load(tmp_path / "opt.pt"))
    for s in range(6, 9):
        step(a, oa, s), step(b, ob, s)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    want = torch.float32 if bits == 32 else F8
    assert all(ob.state[p]["exp_avg"].dtype == want and ob.state[p]["step"] == 4 for p in b)


def test_state_of_torchs_optimizer_is_loaded():
    """One more step of either from there; bounds as in test_optimizer_follows_torch."""
    from sunnynet_b200.optim import AdamW
    g = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn(500, device="cuda", generator=g).requires_grad_()
    b = torch.optim.AdamW([x], lr=1e-2)
    for _ in range(3):
        x.grad = torch.randn(500, device="cuda", generator=g)
        b.step()
    y = x.detach().clone().requires_grad_()
    a = AdamW([y])
    a.load_state_dict(b.state_dict())
    x.grad = torch.randn(500, device="cuda", generator=g)
    y.grad = x.grad.clone()
    a.step(), b.step()
    assert a.state[y]["step"] == 4
    h = 2.0 ** -24
    assert ((x.double() - y.double()).abs() <= 16 * h * 4e-2 + 3 * h * (x.abs() + 1)).all()


def test_refusals(adamw_step):
    from sunnynet_b200.optim import AdamW
    def lists():
        return make([300, 20], KINDS[0], 32, 7)
    l8 = make([300, 20], KINDS[0], 8, 7)
    p, g, m, v = lists()
    before = [x.clone() for x in p]
    bad = [
        lambda: adamw_step(p, g[:1], m, v, 1), lambda: adamw_step(p, g, m, v, 0),
        lambda: adamw_step([p[0], p[0]], [g[0], g[0]], [m[0], m[0]], [v[0], v[0]], 1),
        lambda: adamw_step(p, g, [m[0], m[1]], [v[0], m[1]], 1),
        lambda: adamw_step(p, g, [p[0], m[1]], v, 1),
        lambda: adamw_step([p[0].cpu(), p[1]], g, m, v, 1),
        lambda: adamw_step([p[0].half(), p[1]], g, m, v, 1),
        lambda: adamw_step([x.double() for x in p], g, m, v, 1),
        lambda: adamw_step(p, g, [x.half() for x in m], v, 1),
        lambda: adamw_step([p[0][::2], p[1]], [g[0][:150], g[1]], [m[0][:150], m[1]], [v[0][:150], v[1]], 1),
        lambda: adamw_step(p, [g[0][:299], g[1]], m, v, 1),
        lambda: adamw_step(p, g, m, v, 1, beta1=1.0), lambda: adamw_step(p, g, m, v, 1, lr=float("nan")),
        lambda: adamw_step(p, g, m, v, 1, eps=-1.0),
        lambda: adamw_step(*l8[:4], 1), lambda: adamw_step(*l8[:4], 1, avg_scale=l8[4]),
        lambda: adamw_step(*l8[:4], 1, avg_scale=[l8[4][0][:1], l8[4][1]], sq_scale=l8[5]),
        lambda: adamw_step(p, g, m, v, torch.tensor([1], device="cuda", dtype=torch.int32)),
        lambda: adamw_step(p, g, m, v, torch.tensor([1])),
        lambda: AdamW([p[0]], state_bits=16), lambda: AdamW([p[0]], betas=(0.9, 1.0)),
    ]
    for i, f in enumerate(bad):
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            f()
            pytest.fail(f"call {i} was taken")
    assert all(torch.equal(a, b) for a, b in zip(p, before))
    adamw_step([], [], [], [], 1)
    q = p[0].clone().requires_grad_()
    opt = AdamW([q])
    q.grad = g[0].clone()
    opt.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="capture"):
        with torch.cuda.graph(graph):
            opt.step()
