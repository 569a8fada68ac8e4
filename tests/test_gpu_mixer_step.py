"""A block with linear attention trained and decoded as it would be used: embedding
-> norm -> projections -> linear attention -> norm -> tied head, its gradients,
their norm and an AdamW step that takes the factor; then a prompt, its state, and
single tokens with the draw. Against the same in torch in fp64.

Gradients: torch's own matrix products in fp32 lie between the kernels, so the
bound is an end-to-end one: relative to the largest value of each gradient, 2^-24
times the length of the longest sum on its path (B T V = 4096 terms at most, each
rounded once) with a factor of 4 for the layers it passes: 1e-3.
"""
from __future__ import annotations

import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

B, T, V, D, H, DK = 2, 24, 80, 64, 4, 16
EPS = 1e-5


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def make():
    g = torch.Generator(device="cuda").manual_seed(5)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    params = {"embed": r(V, D) / 8, "g1": 1 + 0.1 * r(D), "b1": 0.1 * r(D), "qkv": r(3 * H * DK, D) / 8, "decay": r(H),
              "out": r(D, H * DK) / 8, "g2": 1 + 0.1 * r(D), "b2": 0.1 * r(D)}
    return params, torch.randint(0, V, (B, T + 1), device="cuda", generator=g)


def ours():
    from sunnynet_b200 import kernels
    return (lambda t, w: kernels.embedding(t, w, math.sqrt(D)), lambda x, w, b: kernels.layer_norm(x, w, b, EPS),
            lambda q, k, v, g: kernels.linear_attention(q, k, v, g))


def plain_norm(x, w, b):
    c = x - x.mean(-1, keepdim=True)
    return c / (c.square().mean(-1, keepdim=True) + EPS).sqrt() * w + b


def plain_attention(q, k, v, g):
    S, out = torch.zeros(B, H, DK, DK, dtype=v.dtype, device=v.device), []
    for t in range(q.shape[1]):
        S = S * g.exp()[:, None, None] + k[:, t, :, :, None] * v[:, t, :, None, :]
        out.append((q[:, t, :, :, None] * S).sum(2) * DK ** -0.5)
    return torch.stack(out, 1), S


def plain():
    return (lambda t, w: w[t] * math.sqrt(D)), plain_norm, plain_attention


def forward(p, tokens, ops):
    embed, norm, attention = ops
    x = embed(tokens, p["embed"])
    q, k, v = (norm(x, p["g1"], p["b1"]) @ p["qkv"].T).unflatten(-1, (3, H, DK)).unbind(2)
    y, S = attention(q, k, v, -torch.nn.functional.softplus(p["decay"]))
    return norm(x + y.flatten(2) @ p["out"].T, p["g2"], p["b2"]) @ p["embed"].T, S


def loss_of(logits, targets):
    return torch.nn.functional.cross_entropy(logits.flatten(0, 1), targets.flatten())


def test_gradients_of_a_block():
    params, tokens = make()
    got = {k: v.clone().requires_grad_() for k, v in params.items()}
    loss = loss_of(forward(got, tokens[:, :-1], ours())[0], tokens[:, 1:])
    loss.backward()
    want = {k: v.double().requires_grad_() for k, v in params.items()}
    ref = loss_of(forward(want, tokens[:, :-1], plain())[0], tokens[:, 1:])
    ref.backward()
    assert abs(loss.item() - ref.item()) <= 1e-3 * ref.item()
    for k in params:
        w = want[k].grad
        assert ((got[k].grad.double() - w).abs() <= 1e-3 * w.abs().max()).all(), k


@pytest.mark.parametrize("bits", [32, 8])
def test_steps_with_the_norm_bounded(bits):
    """The first step's update is lr * g / (|g| + eps) whatever the factor, but for eps,
    which it weighs against f * g; .grad stays, and the norm is that of all of them."""
    from sunnynet_b200.optim import AdamW
    params, tokens = make()
    leaves = {k: torch.nn.Parameter(v.clone()) for k, v in params.items()}
    opt = AdamW(leaves.values(), lr=1e-3, weight_decay=0.0, state_bits=bits, max_norm=0.01)
    loss_of(forward(leaves, tokens[:, :-1], ours())[0], tokens[:, 1:]).backward()
    opt.step()
    norm = math.sqrt(sum(float(v.grad.double().square().sum()) for v in leaves.values()))
    assert abs(float(opt.grad_norm) - norm) <= 5 * 2.0 ** -24 * norm
    f = min(1.0, 0.01 / (norm + 1e-6))
    assert f < 1
    for k, v in leaves.items():
        g = f * v.grad.double()
        moved = v.detach().double() - params[k].double()
        want = -1e-3 * g / (g.abs() + 1e-8)
        # f and f * g are rounded (8 * 2^-24 of g, which the quotient passes on where g is near eps), p by half a step
        assert ((moved - want).abs() <= 2.0 ** -24 * params[k].abs() + 1e-3 * 2.0 ** -19).all(), k
    for _ in range(2):
        opt.zero_grad()
        loss_of(forward(leaves, tokens[:, :-1], ours())[0], tokens[:, 1:]).backward()
        opt.step()
    assert all(torch.isfinite(v).all() for v in leaves.values())


def test_a_captured_step():
    """Forward, backward, the norm and the update in one graph: replays leave the
    parameters of the same steps run one by one (all kernels here are the same bits
    every time; torch's products may choose others in a capture: 1e-5 of the largest value)."""
    from sunnynet_b200 import kernels
    params, tokens = make()
    runs = []
    for captured in (False, True):
        leaves = [v.clone().requires_grad_() for v in params.values()]
        m, s = ([torch.zeros_like(v) for v in leaves] for _ in range(2))
        step = torch.zeros(1, dtype=torch.int64, device="cuda")

        def one():
            step.add_(1)
            logits, _ = forward(dict(zip(params, leaves)), tokens[:, :-1], ours())
            grads = torch.autograd.grad(loss_of(logits, tokens[:, 1:]), leaves)
            with torch.no_grad():
                _, factor = kernels.grad_norm(grads, 0.5)
                kernels.adamw_step(leaves, [g.contiguous() for g in grads], m, s, step, lr=1e-3, grad_scale=factor)

        if captured:
            before = [v.detach().clone() for v in leaves]
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                one()
            torch.cuda.current_stream().wait_stream(side)
            with torch.no_grad():
                for v, a in zip(leaves, before):
                    v.copy_(a)
                for x in m + s + [step]:
                    x.zero_()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                one()
            for _ in range(3):
                graph.replay()
        else:
            for _ in range(3):
                one()
        torch.cuda.synchronize()
        runs.append([v.detach().clone() for v in leaves])
    for a, b in zip(*runs):
        assert ((a - b).abs() <= 1e-5 * a.abs().max()).all()


def test_a_prompt_and_its_next_tokens():
    """Logits of single tokens from a prompt's state are those of the whole sequence
    at once (bound as above), and the draw from them takes the same tokens."""
    from sunnynet_b200 import kernels
    from sunnynet_b200.sampling import sample
    params, tokens = make()
    whole, end = forward(params, tokens, ours())
    ref, _ = forward({k: v.double() for k, v in params.items()}, tokens, plain())
    _, S = forward(params, tokens[:, :10], ours())
    embed, norm, _ = ours()
    g = -torch.nn.functional.softplus(params["decay"])
    for t in range(10, T + 1):
        x = embed(tokens[:, t], params["embed"])
        q, k, v = (norm(x, params["g1"], params["b1"]) @ params["qkv"].T).unflatten(-1, (3, H, DK)).unbind(1)
        y = kernels.linear_attention_step(q, k, v, g, S)
        logits = norm(x + y.flatten(1) @ params["out"].T, params["g2"], params["b2"]) @ params["embed"].T
        for other in (whole[:, t], ref[:, t]):
            assert ((logits.double() - other).abs() <= 1e-3 * ref.abs().max()).all()
        top = ref[:, t].topk(2).values
        clear = top[:, 0] - top[:, 1] > 2e-3 * ref.abs().max()
        got = sample(logits, torch.zeros(B, device="cuda"), temperature=0.0)
        assert torch.equal(got[clear].long(), ref[:, t].argmax(-1)[clear])
    assert ((S - end).abs() <= 1e-3 * end.abs().max()).all()
