"""Linear attention with a decay for each head, its gradients and its form for
single tokens, against the recurrence in 64 bits (its gradients by autograd).

Tolerances. Every output is a sum of products of the inputs, so the same
recurrence of their absolute values bounds the sum of the magnitudes of its
terms (M below, one number for each output). A term of an fp32 result meets at most
 - three matrix products of factors in three bf16 parts: products of parts that
   are left out, below 2 * 2^-24 + 2^-32 of a factor's product each, 2^-22 in all;
 - fp32 sums in matrix instructions, which cut a step's sum off (2^-23): of 128 + 128
   values by 16, in up to six products each, 96 steps, 2^-16.4;
 - one sum a chunk of 32 tokens or more, 2^-24 each, 2^-16 for T up to 8192;
 - three decays: ex2.approx 2^-22, and the argument's rounding, 2^-24 of at most
   2^5 (what is smaller than 2^-32 is lost beside its neighbours): 3 * 2^-19;
together below 2^-14.9. The gradient of a token's decay is the difference, within
its chunk, of two sums that hold the same terms of pairs on one side of the token:
at most 128 + 7 roundings of 2^-24 of the chunk's terms, whatever is left of them
(SPREAD: 2^-16 of the sum of |q . dq| over the 128 tokens around). What goes to a 16-bit output is rounded to one bf16 part
between two products (2^-8, for a score or a state), or, for float16, to two, whose low
parts' product is left out (2^-16 in each of three products, 2^-14 with the
parts' own). The store adds a half step of the stored type.
"""
from __future__ import annotations

import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
FINE = 2.0 ** -14.9
PARTS = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -14}


@pytest.fixture(scope="module")
def kernels():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from sunnynet_b200 import kernels
    return kernels


def recurrence(q, k, v, log_decay, state, lengths, scale):
    """The definition, token by token, in the inputs' type."""
    B, T, H, dv = v.shape
    Hk, dk = q.shape[2:]
    q, k = (x.repeat_interleave(H // Hk, 2) for x in (q, k))
    f = log_decay.exp().expand(B, T, H)
    S = torch.zeros(B, H, dk, dv, dtype=v.dtype, device=v.device) if state is None else state
    out = []
    for t in range(T):
        new = S * f[:, t, :, None, None] + k[:, t, :, :, None] * v[:, t, :, None, :]
        o = (q[:, t, :, :, None] * new).sum(2) * scale
        if lengths is not None:
            on = (t < lengths)[:, None, None]
            new, o = torch.where(on[..., None], new, S), torch.where(on, o, 0.0)
        S = new
        out.append(o)
    return torch.stack(out, 1) if T else torch.zeros_like(v), S


def make(B, T, H, Hk, dk, dv, dtype, decay="token", state=True, lengths=None, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed + 1000 * T + dk)
    r = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
    x = {"q": r(B, T, Hk, dk).to(dtype), "k": r(B, T, Hk, dk).to(dtype), "v": r(B, T, H, dv).to(dtype)}
    if decay == "head":
        x["log_decay"] = -torch.exp2(-1.0 - 7.0 * torch.rand(H, device="cuda", generator=gen))
    else:
        x["log_decay"] = -torch.nn.functional.softplus(r(B, T, H) * 2 - 2)
    x["state"] = r(B, H, dk, dv) if state else None
    x["lengths"] = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    return x


def truth(x, scale, ends=None):
    """(out, state[, gradients of what requires them]) in 64 bits, and the same of absolute values."""
    got = []
    for take in (lambda t: t, torch.abs):
        leaves = {n: (take(t.detach().double()) if n not in ("lengths", "log_decay") else
                      t.detach().double() if n == "log_decay" else t) if t is not None else None
                  for n, t in x.items()}
        if ends is not None:
            for n, t in leaves.items():
                if t is not None and n != "lengths":
                    t.requires_grad_()
        out, state = recurrence(**leaves, scale=scale)
        res = [out, state]
        if ends is not None:
            into = [t for n, t in leaves.items() if t is not None and n != "lengths"]
            outs = [(o, take(e.double())) for o, e in zip((out, state), ends) if e is not None]
            res += torch.autograd.grad([o for o, _ in outs], into, [e for _, e in outs], allow_unused=True,
                                       materialize_grads=True)
        got.append([t.detach() for t in res])
    return got


def spread(x, most):
    """What the gradient of log_decay may be off beside FINE, from the gradients of absolute values."""
    B, T, H = x["v"].shape[:3]
    w = (x["q"].double().abs() * most[2]).sum(-1).repeat_interleave(H // x["q"].shape[2], 2)
    if x["lengths"] is not None:
        w = torch.where(torch.arange(T, device="cuda")[:, None] < x["lengths"][:, None, None], w, 0.0)
    w = torch.cat([w, w.new_zeros(B, -T % 128, H)], 1).unflatten(1, (-1, 128)).sum(2, keepdim=True)
    w = w.expand(-1, -1, 128, -1).flatten(1, 2)[:, :T] * 2.0 ** -16
    return w.sum((0, 1)) if x["log_decay"].dim() == 1 else w


def near(got, want, most, dtype, more=0.0):
    assert got.dtype == dtype and got.shape == want.shape
    e = torch.finfo(dtype).eps / 2
    bound = (PARTS[dtype] + FINE) * most + more
    tiny = torch.finfo(dtype).smallest_normal * e  # half a step below the normal numbers
    bad = ~((got.double() - want).abs() <= bound + e * (want.abs() + bound) + tiny).flatten()
    if bad.any():
        at = bad.nonzero()[:4, 0]
        pytest.fail(f"{int(bad.sum())} of {got.numel()}: at {at.tolist()} {got.flatten()[at].tolist()} for "
                    f"{want.flatten()[at].tolist()}, bound {bound.flatten()[at].tolist()}")
    if want.numel() >= 4096 and want.norm() > 0:
        # as independent roundings (at most 2^-8 / sqrt 3 for each value and each of two stages) add up
        far = float((got.double() - want).norm() / want.norm())
        assert far <= {torch.float32: 2.0 ** -18, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[dtype], far


SIZES = [(1, 1, 1, 1, 1, 1), (2, 3, 2, 1, 5, 7), (1, 64, 2, 2, 64, 64), (2, 65, 3, 3, 64, 48), (1, 63, 1, 1, 33, 17),
         (2, 130, 4, 2, 64, 64), (1, 31, 2, 1, 128, 128), (2, 97, 3, 1, 72, 127), (1, 200, 2, 1, 16, 100),
         (1, 700, 3, 3, 64, 32), (2, 1100, 2, 1, 40, 72), (1, 1000, 2, 2, 128, 128), (1, 515, 1, 1, 9, 3),
         (5, 70, 100, 50, 8, 8), (2, 150, 2, 1, 100, 30), (1, 300, 160, 160, 128, 64), (1, 300, 2, 2, 64, 128)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,T,H,Hk,dk,dv", SIZES)
def test_outputs_and_states(kernels, B, T, H, Hk, dk, dv, dtype):
    for n, (decay, state) in enumerate((("token", True), ("head", False))):
        x = make(B, T, H, Hk, dk, dv, dtype, decay, state, seed=n)
        got = kernels.linear_attention(**x, scale=0.3)
        (out, S), (mo, ms) = truth(x, 0.3)
        near(got[0], out, mo, dtype)
        near(got[1], S, ms, torch.float32)


def gradients(kernels, x, scale, ends):
    leaves = {n: t.detach().clone().requires_grad_() if t is not None and n != "lengths" else t for n, t in x.items()}
    out = kernels.linear_attention(**leaves, scale=scale)
    into = [t for n, t in leaves.items() if t is not None and n != "lengths"]
    outs = [(o, e) for o, e in zip(out, ends) if e is not None]
    return [t.detach() for t in out] + list(torch.autograd.grad([o for o, _ in outs], into, [e for _, e in outs]))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,T,H,Hk,dk,dv", SIZES)
def test_gradients(kernels, B, T, H, Hk, dk, dv, dtype):
    for n, (decay, state) in enumerate((("token", True), ("head", False))):
        x = make(B, T, H, Hk, dk, dv, dtype, decay, state, seed=n)
        gen = torch.Generator(device="cuda").manual_seed(7)
        ends = (torch.randn(B, T, H, dv, device="cuda", generator=gen).to(dtype),
                torch.randn(B, H, dk, dv, device="cuda", generator=gen) if state else None)
        got = gradients(kernels, x, 0.3, ends)
        want, most = truth(x, 0.3, ends)
        kinds = [dtype, torch.float32] + [dtype] * 3 + [torch.float32] * 2
        for n, (g, w, m, kind) in enumerate(zip(got, want, most, kinds)):
            near(g, w, m, kind, spread(x, most) if n == 5 else 0.0)


def test_gradients_against_differences(kernels):
    """Central differences of the 64-bit recurrence along random directions; the
    sum's error is that of near(), the differences' own below 1e-8 of it."""
    x = make(1, 150, 2, 1, 24, 40, torch.float32)
    gen = torch.Generator(device="cuda").manual_seed(1)
    ends = (torch.randn(1, 150, 2, 40, device="cuda", generator=gen), torch.randn(1, 2, 24, 40, device="cuda", generator=gen))
    got = gradients(kernels, x, 0.3, ends)[2:]
    _, most = truth(x, 0.3, ends)
    wide = {n: t.double() if t is not None else None for n, t in x.items()}
    loss = lambda y: sum(float((o * e.double()).sum()) for o, e in zip(recurrence(**y, scale=0.3), ends))  # noqa: E731
    for (n, g), m in zip(zip(("q", "k", "v", "log_decay", "state"), got), most[2:]):
        way = torch.randn(g.shape, device="cuda", generator=gen, dtype=torch.float64)
        h = 1e-5
        diff = (loss({**wide, n: wide[n] + h * way}) - loss({**wide, n: wide[n] - h * way})) / (2 * h)
        assert abs(diff - float((g.double() * way).sum())) <= 2 * FINE * float((m * way.abs()).sum()), n


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,lengths", [(100, [100, 64, 1, 0, 65]), (1300, [1300, 600, 0, 513, 1024])])
def test_padded_batches(kernels, T, lengths, dtype):
    """What lies behind a sequence's end is not read: NaN there leaves no trace."""
    x = make(5, T, 2, 1, 64, 32, dtype, lengths=lengths)
    ends = (torch.randn(5, T, 2, 32, device="cuda").to(dtype), torch.randn(5, 2, 64, 32, device="cuda"))
    want, most = truth(x, 0.2, ends)
    more = spread(x, most)
    behind = torch.arange(T, device="cuda") >= x["lengths"][:, None]
    for n in ("q", "k", "v", "log_decay"):
        x[n][behind] = float("nan")
    ends[0][behind] = float("nan")
    got = gradients(kernels, x, 0.2, ends)
    for n, (g, w, m, kind) in enumerate(zip(got, want, most, [dtype, torch.float32] + [dtype] * 3 + [torch.float32] * 2)):
        near(g, w, m, kind, more if n == 5 else 0.0)
    for g in (got[0], *got[2:6]):
        assert (g[behind] == 0).all()


@pytest.mark.parametrize("T", [40, 900])
def test_decays_that_forget(kernels, T):
    """Minus infinity begins anew: several sequences in one row give what each alone gives."""
    x = make(1, T, 3, 3, 64, 64, torch.float32, state=False)
    cuts = [0, 1, 7, T // 2, T // 2 + 1, T - 3]
    for c in cuts:
        x["log_decay"][:, c] = -float("inf")
    x["log_decay"][:, 3] = -1e30
    x["log_decay"][:, 5] = 0.0
    x["state"] = torch.randn(1, 3, 64, 64, device="cuda")  # forgotten at once
    out, S = kernels.linear_attention(**x, scale=1.0)
    cuts.insert(2, 3)
    for a, b in zip(cuts, cuts[1:] + [T]):
        part = {n: x[n][:, a:b] for n in ("q", "k", "v", "log_decay")}
        part["log_decay"] = part["log_decay"].clamp_min(-1e4)
        (o, s), (mo, ms) = truth({**part, "state": None, "lengths": None}, 1.0)
        near(out[:, a:b], o, mo, torch.float32)
    near(S, s, ms, torch.float32)
    # near tokens keep their weight exactly however far the sum of decays is from zero
    x["log_decay"][:] = -40.0
    x["log_decay"][:, 20] = 0.0
    out, _ = kernels.linear_attention(**x, scale=1.0)
    (o, _), (mo, _) = truth(x, 1.0)
    near(out, o, mo, torch.float32)


def test_values_without_finite_numbers_stay_in_their_place(kernels):
    """A NaN in v reaches its own column of what comes after it, and nothing before."""
    x = make(1, 200, 2, 2, 64, 64, torch.float32, state=False)
    clean, _ = kernels.linear_attention(**x)
    x["v"][0, 130, 1, 5] = float("nan")
    out, S = kernels.linear_attention(**x)
    assert out[0, 130:, 1, 5].isnan().all() and S[0, 1, :, 5].isnan().all()
    hit = torch.zeros_like(out, dtype=torch.bool)
    hit[0, 128:, 1] = True  # (the chunk of the token shares its products' rows)
    assert torch.equal(out[~hit], clean[~hit])
    assert not out[0, :130].isnan().any() and not out[0, :, 0].isnan().any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name", ["q", "k", "v"])
def test_what_is_not_finite_reaches_nothing_before(kernels, name, dtype):
    """The outputs of the tokens before are the definition's, what it reaches is not finite."""
    for value in (float("nan"), float("inf")):
        x = make(1, 150, 2, 2, 64, 64, dtype, state=False)
        (want, _), (most, _) = truth(x, 0.3)
        x[name][0, 73, 1, 5] = value
        out, S = kernels.linear_attention(**x, scale=0.3)
        near(out[:, :73], want[:, :73], most[:, :73], dtype)
        near(out[:, :, 0], want[:, :, 0], most[:, :, 0], dtype)
        if name == "q":
            assert not out[0, 73, 1].isfinite().any()
            near(out[:, 74:], want[:, 74:], most[:, 74:], dtype)
        else:
            at = (1, 5) if name == "v" else (1,)
            assert not (out[0, 73:, *at].isfinite().any() or S[0, 1, 5].isfinite().all())


def test_layouts(kernels):
    """Views of one projection, of transposed tensors, at odd addresses, broadcast ones."""
    for dtype in DTYPES:
        for dk, dv, off in ((64, 64, 0), (64, 64, 1), (24, 40, 3), (33, 65, 0)):
            wide = torch.randn(2, 300, off + 2 * 2 * dk + 4 * dv, device="cuda").to(dtype)
            q, k, v = wide[..., off:].split([2 * dk, 2 * dk, 4 * dv], 2)
            x = {"q": q.unflatten(2, (2, dk)), "k": k.unflatten(2, (2, dk)), "v": v.unflatten(2, (4, dv)),
                 "log_decay": -torch.rand(300, 4, 2, device="cuda").permute(2, 0, 1), "state": None, "lengths": None}
            x["state"] = torch.randn(2, dk, dv, 4, device="cuda").permute(0, 3, 1, 2)
            whole = {n: t.contiguous() if t is not None else None for n, t in x.items()}
            for a, b in zip(kernels.linear_attention(**x), kernels.linear_attention(**whole)):
                assert torch.equal(a, b)
            x["q"] = whole["q"].transpose(1, 3).contiguous().transpose(1, 3)
            x["k"] = whole["k"][:1, :1].expand(2, 300, 2, dk)
            whole["k"] = x["k"].contiguous()
            for a, b in zip(kernels.linear_attention(**x), kernels.linear_attention(**whole)):
                assert torch.equal(a, b)
    x = make(2, 200, 2, 2, 64, 64, torch.bfloat16)
    base = gradients(kernels, x, 0.1, (torch.ones(2, 200, 2, 64, device="cuda", dtype=torch.bfloat16), None))
    same = gradients(kernels, x, 0.1, (torch.ones((), device="cuda", dtype=torch.bfloat16).expand(2, 200, 2, 64), None))
    assert all(torch.equal(a, b) for a, b in zip(base, same))


def test_nothing_to_do(kernels):
    x = make(2, 0, 3, 1, 8, 16, torch.float32)
    out, S = kernels.linear_attention(**x)
    assert out.shape == (2, 0, 3, 16) and torch.equal(S, x["state"])
    got = gradients(kernels, x, 1.0, (out, torch.ones_like(S)))
    assert torch.equal(got[-1], torch.ones_like(S)) and got[2].shape == (2, 0, 1, 8)
    x = make(0, 5, 3, 1, 8, 16, torch.float32, decay="head")
    out, S = kernels.linear_attention(**x)
    assert out.shape == (0, 5, 3, 16) and S.shape == (0, 3, 8, 16)
    got = gradients(kernels, x, 1.0, (out, None))
    assert torch.equal(got[-2], torch.zeros(3, device="cuda"))
    assert kernels.linear_attention_step(x["q"][:, 0], x["k"][:, 0], x["v"][:, 0], x["log_decay"], S).shape == (0, 3, 16)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,H,Hk,dk,dv", [(1, 12, 12, 64, 64), (3, 4, 2, 128, 128), (5, 3, 1, 7, 33), (2, 2, 2, 1, 1),
                                          (300, 2, 1, 40, 72), (2, 3, 3, 100, 4), (4, 1, 1, 128, 2)])
def test_single_tokens(kernels, B, H, Hk, dk, dv, dtype):
    """fp32 throughout: a state takes three roundings and the decay's 2^-21 a token,
    an output a sum of dk more."""
    x = make(B, 6, H, Hk, dk, dv, dtype)
    wide = torch.randn(B, 2, H, dk, dv, device="cuda")
    wide[:, 0] = x["state"]
    S, other = wide[:, 0], wide[:, 1].clone()
    want, most = truth(x, 0.3)
    for t in range(6):
        at = lambda n: x[n][:, t]  # noqa: B023,E731
        out = kernels.linear_attention_step(at("q"), at("k"), at("v"), at("log_decay"), S, 0.3)
        err = (dk + 40) * 2.0 ** -24 + 6 * 2.0 ** -21
        e = torch.finfo(dtype).eps / 2
        assert out.dtype == dtype
        far = (out.double() - want[0][:, t]).abs()
        assert (far <= err * most[0][:, t] + e * (want[0][:, t].abs() + err * most[0][:, t])).all()
    assert ((S.double() - want[1]).abs() <= 6 * (2.0 ** -22 + 2.0 ** -21) * most[1]).all()
    assert torch.equal(wide[:, 1], other)
    # one decay for each head, and one that forgets
    head = torch.full((H,), -0.5, device="cuda")
    head[0] = -float("inf")
    before = S.double().clone()
    kernels.linear_attention_step(x["q"][:, 0], x["k"][:, 0], x["v"][:, 0], head, S, 0.3)
    k, v = x["k"][:, 0].double().repeat_interleave(H // Hk, 1), x["v"][:, 0].double()
    to = before * head.double().exp()[:, None, None] + k[..., None] * v[:, :, None]
    assert ((S.double() - to).abs() <= 2.0 ** -20 * (before.abs() + (k[..., None] * v[:, :, None]).abs())).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_prompt_in_parts_and_its_next_tokens(kernels, dtype):
    """A whole prompt; in three parts, the state handed on; by single tokens."""
    x = make(2, 700, 4, 2, 64, 64, dtype)
    x["lengths"] = None
    want, most = truth(x, 0.2)
    S, outs = x["state"], []
    for a, b in ((0, 1), (1, 333), (333, 690)):
        part = {n: x[n][:, a:b] for n in ("q", "k", "v", "log_decay")}
        out, S = kernels.linear_attention(**part, state=S, scale=0.2)
        outs.append(out)
    for t in range(690, 700):
        outs.append(kernels.linear_attention_step(*(x[n][:, t] for n in ("q", "k", "v", "log_decay")), S, 0.2)[:, None])
    near(torch.cat(outs, 1), want[0], most[0], dtype)
    near(S, want[1], most[1], torch.float32)


def test_same_bits_captured_and_on_other_streams(kernels):
    xs = [make(1, 1500, 3, 3, 64, 64, torch.bfloat16, seed=n) for n in range(2)]
    want = [kernels.linear_attention(**x) for x in xs]
    again = kernels.linear_attention(**xs[0])
    assert all(torch.equal(a, b) for a, b in zip(want[0], again))
    torch.cuda.synchronize()
    graphs, got = [], []
    for x in xs:  # two graphs, run at the same time: each has its own workspace
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got.append(kernels.linear_attention(**x))
        graphs.append(g)
    for _ in range(3):
        for pair in got:
            for t in pair:
                t.zero_()
        torch.cuda.synchronize()
        sides = [torch.cuda.Stream() for _ in graphs]
        for g, s in zip(graphs, sides):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for a, b in zip(want, got):
            assert all(torch.equal(x, y) for x, y in zip(a, b))
    ends = (torch.ones_like(want[0][0]), None)
    first = gradients(kernels, xs[0], 1.0, ends)
    for a, b in zip(first, gradients(kernels, xs[0], 1.0, ends)):
        assert torch.equal(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = gradients(kernels, xs[0], 1.0, ends)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, other))


def test_only_once_differentiable_and_versions(kernels):
    x = make(1, 10, 2, 2, 8, 8, torch.float32)
    x["q"].requires_grad_()
    out, S = kernels.linear_attention(**x)
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(out.sum(), x["q"], create_graph=True)
    state = torch.zeros(1, 2, 8, 8, device="cuda")
    w = torch.ones(1, 2, 8, 8, device="cuda", requires_grad=True)
    y = (w * state).sum()
    kernels.linear_attention_step(x["q"].detach()[:, 0], x["k"][:, 0], x["v"][:, 0], x["log_decay"][:, 0], state)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.backward()


def test_inference_mode(kernels):
    """States of inference mode are updated in it, and outside are refused untouched."""
    with torch.inference_mode():
        x = make(2, 1, 2, 2, 8, 8, torch.float32, "head")
        one = {n: t[:, 0] if n in "qkv" else t for n, t in x.items() if n != "lengths"}
        (out, end), (mo, me) = truth(x, 8 ** -0.5)
        near(kernels.linear_attention_step(**one), out[:, 0], mo[:, 0], torch.float32)
        near(one["state"], end, me, torch.float32)
    before = one["state"].clone()
    with torch.no_grad(), pytest.raises(RuntimeError, match="inference"):
        kernels.linear_attention_step(**one)
    assert torch.equal(one["state"], before)


def test_growing_states(kernels):
    """Positive log decays, up to e^20 over the sequence."""
    x = make(1, 200, 2, 1, 24, 40, torch.float32)
    x["log_decay"] = x["log_decay"].abs().clamp(max=0.1)
    got = kernels.linear_attention(**x, scale=0.2)
    (out, S), (mo, ms) = truth(x, 0.2)
    near(got[0], out, mo, torch.float32)
    near(got[1], S, ms, torch.float32)


def test_refusals_on_the_gpu(kernels):
    x = make(2, 5, 4, 2, 8, 16, torch.float32)
    for change in ({"q": x["q"][:, :4]}, {"k": x["k"][..., :7]}, {"v": x["v"][:, :, :3]}, {"q": x["q"].bfloat16()},
                   {"v": x["v"].cpu()}, {"log_decay": x["log_decay"].double()}, {"log_decay": x["log_decay"][:, :1]},
                   {"log_decay": x["log_decay"].cpu()}, {"state": x["state"][:1]}, {"state": x["state"].bfloat16()},
                   {"lengths": torch.ones(2, device="cuda")}, {"lengths": torch.ones(3, dtype=torch.int32, device="cuda")},
                   {"q": torch.zeros(2, 5, 2, 129, device="cuda"), "k": torch.zeros(2, 5, 2, 129, device="cuda"), "state": None}):
        with pytest.raises((ValueError, TypeError)):
            kernels.linear_attention(**{**x, **change})
    s = {n: x[n][:, 0] for n in ("q", "k", "v", "log_decay")}
    for state in (x["state"].bfloat16(), x["state"][:1], x["state"].cpu(), x["state"].transpose(2, 3).contiguous().transpose(2, 3),
                  x["state"].clone().requires_grad_()):
        with pytest.raises((ValueError, RuntimeError)):
            kernels.linear_attention_step(**s, state=state)
    with pytest.raises(ValueError, match="overlap"):
        kernels.linear_attention_step(**s, state=x["state"][:1].expand(2, 4, 8, 16))


def test_lengths_beyond_the_batch(kernels):
    """Lengths below zero are none, lengths above T all tokens."""
    x = make(3, 70, 2, 2, 16, 16, torch.float32, lengths=[-5, 70 + 9, 2 ** 31 - 1])
    want, most = truth({**x, "lengths": torch.tensor([0, 70, 70], device="cuda")}, 0.3)
    for g, w, m in zip(kernels.linear_attention(**x, scale=0.3), want, most):
        near(g, w, m, torch.float32)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_offsets_beyond_32_bits(kernels, dtype):
    """Tokens, heads and sequences that lie further apart than 2^32 bytes."""
    x = make(2, 9, 2, 2, 16, 16, dtype, state=False)
    far = torch.empty((1 << 33) // x["q"].element_size() + (1 << 29), dtype=dtype, device="cuda")
    T = 1 << 28  # values from one token to the next: nine of them are beyond 2^31
    wide = far.as_strided((2, 9, 2, 16), ((1 << 31) // 4 + 64, T - (1 << 24), 64, 1))
    base = [t for t in kernels.linear_attention(**x)]
    for n in ("q", "k", "v"):
        wide.copy_(x[n])
        got = kernels.linear_attention(**{**x, n: wide})
        assert all(torch.equal(a, b) for a, b in zip(got, base)), n


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,H,dk,dv", [(64, 16, 128, 128), (2, 3, 64, 64)])
def test_batches_without_a_token(kernels, B, H, dk, dv, dtype):
    """Every length zero: outputs and gradients are zeros, the states pass through, and what is enqueued
    directly behind a call finds them, and may take its workspace."""
    x = make(B, 130, H, H, dk, dv, dtype, "head", lengths=[0] * B)
    ends = (torch.ones(B, 130, H, dv, device="cuda", dtype=dtype), torch.randn(B, H, dk, dv, device="cuda"))
    for _ in range(3):
        out, S = kernels.linear_attention(**x)
        after = S.clone()
        torch.full((1 << 26,), 7.0, device="cuda")
        assert torch.equal(after, x["state"]) and torch.equal(S, x["state"]) and not out.any()
        got = gradients(kernels, x, 1.0, ends)
        after = got[-1].clone()
        torch.full((1 << 26,), 7.0, device="cuda")
        assert torch.equal(after, ends[1]) and torch.equal(got[-1], ends[1])
        assert not any(g.any() for g in got[2:6])


def test_thousands_of_single_tokens(kernels):
    """Slow decays, one token after the other: an error of the factor, the same each time, would add up. One ulp of
    exp(g) - 1 (2^-33 for these g) makes 2^-21 of 4096 tokens. Roundings of a state, at most 2^-24 of it each and
    two a token, fall either way: 2^-24 sqrt(2 / 3) sqrt(4096) as a standard deviation, 2^-15.2 for eight of them."""
    gen = torch.Generator(device="cuda").manual_seed(5)
    r = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
    H, d, n, bound = 64, 16, 4096, 2.0 ** -15.2 + 2.0 ** -21
    g = -(2.0 ** -11) * (1 + torch.rand(H, device="cuda", generator=gen))
    f = g.double().exp()[:, None, None]
    start = r(1, H, d, d)
    q, k, v = r(n, 1, H, d), r(n, 1, H, d), r(n, 1, H, d)
    alone, S, want, most = start.clone(), start.clone(), start.double(), start.double().abs()
    for t in range(n):
        kernels.linear_attention_step(q[t], torch.zeros_like(k[t]), v[t], g, alone)
        kernels.linear_attention_step(q[t], k[t], v[t], g, S)
        want = want * f + k[t].double()[..., None] * v[t].double()[:, :, None]
        most = torch.maximum(most, want.abs())
    gone = start.double() * (n * g.double()).exp()[:, None, None]
    assert float(((alone.double() - gone) / gone).abs().max()) <= bound
    assert float(((S.double() - want).abs() / most).max()) <= bound
    # a prompt of the same tokens ends in the same state
    _, end = kernels.linear_attention(*(x.transpose(0, 1) for x in (q, k, v)), g, start)
    assert float(((end.double() - want).abs() / most).max()) <= bound


@pytest.mark.parametrize("g", [-0.0, -2.0 ** -30, -0.1, -0.49, -0.5, -0.51, -3.0, -20.0, -87.0, 2.0 ** -20, 0.3, 0.5, 0.7, 20.0])
def test_the_factor_of_a_single_token(kernels, g):
    """A token that writes nothing leaves exp(g) S: the state's rounding (2^-150 below the normal numbers), and the
    factor's, by CUDA's bounds of its functions: an ulp of exp(g) - 1 (2^-23 of that at most) near zero, two of
    exp(g) elsewhere."""
    gen = torch.Generator(device="cuda").manual_seed(6)
    S = torch.randn(1, 2, 64, 64, device="cuda", generator=gen)
    x = torch.ones(1, 2, 64, device="cuda")
    decay = torch.full((2,), g, device="cuda")
    want = S.double() * decay.double().exp()[:, None, None]
    kernels.linear_attention_step(x, x * 0, x, decay, S)
    far = 2.0 ** -23 * abs(math.expm1(g)) / math.exp(g) if abs(g) < 0.5 else 2.0 ** -22
    assert ((S.double() - want).abs() <= (2.0 ** -24 + 2.0 ** -40 + far) * want.abs() + 2.0 ** -150).all()


def test_views_with_a_sign(kernels):
    """The imaginary part of a conjugate is a view whose sign is not in memory: inputs and gradients count with
    it, and a state that would be written through it is refused."""
    view = lambda t: torch.complex(torch.zeros_like(t), -t).conj().imag  # noqa: E731
    x = make(2, 70, 2, 2, 1, 1, torch.float32)
    assert view(x["log_decay"]).is_neg() and torch.equal(view(x["log_decay"]), x["log_decay"])
    ends = (torch.randn(2, 70, 2, 1, device="cuda"), torch.randn(2, 2, 1, 1, device="cuda"))
    want = gradients(kernels, x, 0.3, ends)
    for n in ("q", "k", "v", "log_decay", "state"):
        leaf = x[n].detach().clone().requires_grad_()
        got = kernels.linear_attention(**{**x, n: view(leaf)}, scale=0.3)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), n
        got = torch.autograd.grad(got, leaf, [view(e) for e in ends])[0]
        assert torch.equal(got, want[2 + ["q", "k", "v", "log_decay", "state"].index(n)]), n
    one = {n: x[n][:, 0] for n in ("q", "k", "v", "log_decay")}
    S = x["state"].clone()
    want = kernels.linear_attention_step(**one, state=S)
    for n in one:
        T = x["state"].clone()
        assert torch.equal(kernels.linear_attention_step(**{**one, n: view(one[n])}, state=T), want) and torch.equal(S, T), n
    with pytest.raises(ValueError, match="state"):
        kernels.linear_attention_step(**{n: t[:1, :1] if t.dim() > 1 else t for n, t in one.items()}, state=view(x["state"][:1, :1]))


# sequences times heads of 148 or more (74 with gradients): a CTA walks the chunks of a head in turn
WALKS = [(4, 330, 40, 20, 64, 64), (2, 290, 75, 75, 64, 128), (3, 290, 50, 25, 128, 64), (2, 290, 75, 75, 128, 128)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,T,H,Hk,dk,dv", WALKS)
@pytest.mark.parametrize("padded", [False, True])
def test_many_heads_over_many_chunks(kernels, B, T, H, Hk, dk, dv, dtype, padded):
    x = make(B, T, H, Hk, dk, dv, dtype, lengths=[T - 1, 129, 0, 257][:B] if padded else None)
    got = kernels.linear_attention(**x, scale=0.3)
    (out, S), (mo, ms) = truth(x, 0.3)
    near(got[0], out, mo, dtype)
    near(got[1], S, ms, torch.float32)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,T,H,Hk,dk,dv", [(4, 330, 40, 20, 64, 64), (2, 290, 38, 38, 64, 128), (2, 290, 38, 19, 128, 64),
                                            (2, 290, 38, 38, 128, 128)])
@pytest.mark.parametrize("padded", [False, True])
def test_gradients_of_many_heads_over_many_chunks(kernels, B, T, H, Hk, dk, dv, dtype, padded):
    x = make(B, T, H, Hk, dk, dv, dtype, "token" if padded else "head", lengths=[T - 1, 129, 0, 257][:B] if padded else None)
    gen = torch.Generator(device="cuda").manual_seed(8)
    ends = (torch.randn(B, T, H, dv, device="cuda", generator=gen).to(dtype),
            torch.randn(B, H, dk, dv, device="cuda", generator=gen))
    got = gradients(kernels, x, 0.3, ends)
    want, most = truth(x, 0.3, ends)
    for n, (g, w, m, kind) in enumerate(zip(got, want, most, [dtype, torch.float32] + [dtype] * 3 + [torch.float32] * 2)):
        near(g, w, m, kind, spread(x, most) if n == 5 else 0.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,T,H", [(1, 40, 3), (2, 300, 3), (2, 300, 40)])
def test_gradients_of_packed_sequences(kernels, B, T, H, dtype):
    """Minus infinity begins a sequence anew: no gradient crosses it, and its own is zero but for the sums' roundings."""
    x = make(B, T, H, H, 64, 32, dtype)
    for c in (0, 1, 7, T // 2, T // 2 + 1, T - 3):
        x["log_decay"][:, c] = -float("inf")
    gen = torch.Generator(device="cuda").manual_seed(9)
    ends = (torch.randn(B, T, H, 32, device="cuda", generator=gen).to(dtype), torch.randn(B, H, 64, 32, device="cuda", generator=gen))
    got = gradients(kernels, x, 0.3, ends)
    want, most = truth(x, 0.3, ends)
    for n, (g, w, m, kind) in enumerate(zip(got, want, most, [dtype, torch.float32] + [dtype] * 3 + [torch.float32] * 2)):
        near(g, w, m, kind, spread(x, most) if n == 5 else 0.0)
    assert not got[6].any()  # the first state is forgotten at once


def test_gradients_of_growing_states(kernels):
    """Positive log decays, up to e^20 over the sequence."""
    x = make(1, 200, 2, 1, 24, 40, torch.float32)
    x["log_decay"] = x["log_decay"].abs().clamp(max=0.1)
    gen = torch.Generator(device="cuda").manual_seed(9)
    ends = (torch.randn(1, 200, 2, 40, device="cuda", generator=gen), torch.randn(1, 2, 24, 40, device="cuda", generator=gen))
    got = gradients(kernels, x, 0.2, ends)
    want, most = truth(x, 0.2, ends)
    for n, (g, w, m) in enumerate(zip(got, want, most)):
        near(g, w, m, torch.float32, spread(x, most) if n == 5 else 0.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("wanted", [("q",), ("k",), ("v",), ("q", "k", "v"), ("log_decay",), ("state",)])
def test_a_part_of_the_gradients(kernels, dtype, wanted):
    """What is asked for has the bits that it has beside the others, fixed decays among them; of either result alone."""
    x = make(2, 150, 4, 2, 64, 64, dtype)
    ends = (torch.randn(2, 150, 4, 64, device="cuda").to(dtype), torch.randn(2, 4, 64, 64, device="cuda"))
    for end in (ends, (ends[0], None), (None, ends[1])):
        if wanted == ("q",) and end[0] is None:
            continue  # (the last state does not depend on q)
        all_ = dict(zip(("q", "k", "v", "log_decay", "state"), gradients(kernels, x, 0.3, end)[2:]))
        leaves = {n: t.detach().clone().requires_grad_(n in wanted) if t is not None and n != "lengths" else t
                  for n, t in x.items()}
        outs = [(o, e) for o, e in zip(kernels.linear_attention(**leaves, scale=0.3), end) if e is not None]
        got = torch.autograd.grad([o for o, _ in outs], [leaves[n] for n in wanted], [e for _, e in outs])
        assert all(torch.equal(g, all_[n]) for g, n in zip(got, wanted)), end


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_gradient_of_outputs_beyond_32_bits(kernels, dtype):
    """Its tokens and sequences lie further apart than 2^32 bytes."""
    x = make(2, 9, 2, 2, 16, 16, dtype, state=False)
    dout = torch.randn(2, 9, 2, 16, device="cuda").to(dtype)
    want = gradients(kernels, x, 0.3, (dout, None))
    far = torch.empty((1 << 33) // dout.element_size() + (1 << 29), dtype=dtype, device="cuda")
    wide = far.as_strided((2, 9, 2, 16), ((1 << 31) // 4 + 64, (1 << 28) - (1 << 24), 64, 1))
    wide.copy_(dout)
    assert all(torch.equal(a, b) for a, b in zip(gradients(kernels, x, 0.3, (wide, None)), want))


def test_function_transforms_are_refused(kernels):
    """torch.func's wrappers have no memory to read: an error, and nothing is launched."""
    x = make(2, 5, 2, 2, 8, 8, torch.float32)
    w, tokens = torch.randn(9, 8, device="cuda"), torch.arange(4, device="cuda")
    rest = {n: x[n] for n in ("k", "v", "log_decay")}
    one = {n: x[n][:, 0] for n in ("q", "k", "v", "log_decay")}
    for call in (lambda: torch.func.grad(lambda t: kernels.embedding(tokens, t).sum())(w),
                 lambda: torch.func.vmap(lambda t: kernels.embedding(t, w))(tokens),
                 lambda: torch.func.grad(lambda t: kernels.linear_attention(t, **rest)[0].sum())(x["q"]),
                 lambda: torch.func.jvp(lambda t: kernels.linear_attention(t, **rest)[0], (x["q"],), (x["q"],)),
                 lambda: torch.func.vmap(lambda t: kernels.linear_attention(t, **rest)[0])(x["q"][None]),
                 lambda: torch.func.vmap(lambda t: kernels.linear_attention_step(**one, state=t))(x["state"][None]),
                 lambda: torch.func.vmap(lambda t: kernels.grad_norm([t])[0])(w),
                 lambda: torch.func.vmap(lambda t: kernels.clip_grads([t], 0.1))(w)):
        with pytest.raises((RuntimeError, NotImplementedError)):
            call()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,T,H,dk,dv", [(2, 4, 2, 11, 1), (2, 5, 90, 118, 3), (2, 128, 3, 64, 64), (1, 349, 21, 4, 3), (2, 70, 80, 128, 128)])
def test_gradients_of_fast_decays_from_the_last_state(kernels, B, T, H, dk, dv, dtype):
    """Nothing is subtracted on the way from the last state to a decay's gradient: it is as good as its own terms,
    however much larger those of later tokens are."""
    x = make(B, T, H, H, dk, dv, dtype)
    x["log_decay"] *= 8
    gen = torch.Generator(device="cuda").manual_seed(4)
    ends = (None, torch.randn(B, H, dk, dv, device="cuda", generator=gen))
    got = gradients(kernels, x, 0.3, ends)[5]
    want, most = truth(x, 0.3, ends)
    near(got, want[5], most[5], torch.float32, 2.0 ** -116)  # (what an exp2 flushes to zero, times 2^10)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fast", [1.0, 8.0, 40.0])
@pytest.mark.parametrize("B,T,H,Hk,dk,dv", [(2, 4, 2, 2, 11, 1), (2, 17, 6, 3, 118, 3), (2, 128, 3, 3, 64, 64), (1, 349, 21, 7, 4, 3),
                                            (3, 64, 40, 40, 64, 64), (2, 70, 80, 80, 128, 128), (2, 200, 4, 4, 64, 128)])
def test_gradients_of_decays_are_as_good_as_their_terms(kernels, B, T, H, Hk, dk, dv, dtype, fast):
    """The same with gradients of the outputs: a decay's own pairs of tokens, however large its neighbours' are.
    (What goes into them is rounded as in fp32 for every type.)"""
    x = make(B, T, H, Hk, dk, dv, dtype, lengths=[T, T - 1, T // 3][:B])
    x["log_decay"] *= fast
    gen = torch.Generator(device="cuda").manual_seed(4)
    ends = (torch.randn(B, T, H, dv, device="cuda", generator=gen).to(dtype),
            torch.randn(B, H, dk, dv, device="cuda", generator=gen))
    got = gradients(kernels, x, 0.3, ends)[5]
    want, most = truth(x, 0.3, ends)
    near(got, want[5], most[5], torch.float32, 2.0 ** -116)
