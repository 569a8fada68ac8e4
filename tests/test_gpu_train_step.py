"""The operators of a training step and of the draw, together as they are used: a
block of norm -> projection -> core -> norm -> tied head, its gradients, one
AdamW step of all of it in 32- and 8-bit states, and tokens drawn from the
trained model's logits; against the same in torch in fp64.

Gradients: torch's own matrix products in fp32 lie between the kernels, so the
bound is an end-to-end one: relative to the largest value of each gradient,
2^-24 times the length of the longest sum on its path (B T V = 4096 terms at
most, each rounded once) with a factor of 4 for the four layers it passes,
4 * 4096 * 2^-24 = 1e-3.
"""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

B, T, D, V = 2, 16, 64, 128
EPS = 0.02 * 0.02 + 1e-5


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def make():
    g = torch.Generator(device="cuda").manual_seed(3)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    params = {"embed": r(V, D), "g1": 1 + 0.1 * r(D), "b1": 0.1 * r(D), "proj": r(2 * D, D) / 8,
              "delta": torch.rand(D, device="cuda", generator=g) * 0.4 + 0.05, "g2": 1 + 0.1 * r(D),
              "b2": 0.1 * r(D)}
    tokens = torch.randint(0, V, (B, T + 1), device="cuda", generator=g)
    return params, tokens


def plain_norm(x, w, b):
    c = x - x.mean(-1, keepdim=True)
    return c / (c.square().mean(-1, keepdim=True) + EPS).sqrt() * w + b


def plain_core(q, delta, s0):
    """u, states of the competition gate, decay gate and scan (groups of 8)."""
    u, gate = q[..., :D], q[..., D:]
    grouped = gate.unflatten(-1, (-1, 8))
    win = torch.sigmoid(grouped - grouped.roll(-1, -1)) * torch.sigmoid(grouped - grouped.roll(-2, -1))
    u = u * win.flatten(-2)
    p = 1 - delta + delta * torch.sigmoid(gate)
    s, states = s0, []
    for t in range(q.shape[1]):
        s = p[:, t] * s + (1 - p[:, t]) * u[:, t]
        states.append(s)
    return u, torch.stack(states, 1)


def forward(params, tokens, norm, core):
    x = params["embed"][tokens]
    h = norm(x, params["g1"], params["b1"])
    _, states = core(h @ params["proj"].T, params["delta"], torch.zeros_like(x[:, 0]))
    return norm(x + states, params["g2"], params["b2"]) @ params["embed"].T / 8


def loss_of(logits, targets):
    return torch.nn.functional.cross_entropy(logits.flatten(0, 1), targets.flatten())


def ours():
    from sunnynet_b200 import kernels
    return (lambda x, w, b: kernels.layer_norm(x, w, b, EPS)), kernels.core_forward


def test_gradients_of_a_block():
    params, tokens = make()
    got = {k: v.clone().requires_grad_() for k, v in params.items()}
    loss = loss_of(forward(got, tokens[:, :-1], *ours()), tokens[:, 1:])
    loss.backward()
    want = {k: v.double().requires_grad_() for k, v in params.items()}
    ref = loss_of(forward(want, tokens[:, :-1], plain_norm, plain_core), tokens[:, 1:])
    ref.backward()
    assert abs(loss.item() - ref.item()) <= 1e-3 * ref.item()
    for k in params:
        w = want[k].grad
        assert ((got[k].grad.double() - w).abs() <= 1e-3 * w.abs().max()).all(), k


@pytest.mark.parametrize("bits", [32, 8])
def test_steps_and_draws(bits):
    """Three optimiser steps: the parameters move by what the formula makes of the
    gradients in hand (the first step's update is lr * sign(g) in either kind of
    state), everything stays finite; then decoding with the model's logits draws
    what the rule in numpy draws."""
    from sunnynet_b200.optim import AdamW
    from sunnynet_b200.sampling import sample
    params, tokens = make()
    leaves = {k: v.clone().requires_grad_() for k, v in params.items()}
    opt = AdamW(leaves.values(), lr=1e-3, weight_decay=0.0, state_bits=bits)
    for step in range(3):
        opt.zero_grad()
        loss_of(forward(leaves, tokens[:, :-1], *ours()), tokens[:, 1:]).backward()
        before = {k: v.detach().clone() for k, v in leaves.items()}
        opt.step()
        for k, v in leaves.items():
            assert torch.isfinite(v).all()
            moved = (v.detach() - before[k]).double()
            g = v.grad.double()
            if step == 0:
                # m' / (sqrt(v') + eps) = g / (|g| + eps); p rounds by half a step of itself
                want = -1e-3 * g / (g.abs() + 1e-8)
                assert ((moved - want).abs() <= 2.0 ** -24 * before[k].abs() + 1e-3 * 2.0 ** -20).all(), k
    logits = forward({k: v.detach() for k, v in leaves.items()}, tokens[:, :-1], *ours())[:, -1]
    rng = np.random.default_rng(1)
    for _ in range(8):
        u = rng.random(B)
        got = sample(logits, torch.from_numpy(u).cuda(), 0.8, 20, 0.9).tolist()
        for row, v, t in zip(logits.double().cpu().numpy(), u, got):
            w = np.exp((row - row.max()) / 0.8)
            w[row < np.sort(row)[-20]] = 0
            by = np.argsort(-w, kind="stable")
            w[by[np.cumsum(w[by]) - w[by] >= 0.9 * w.sum()]] = 0
            assert t == int(np.argmax(np.cumsum(w) > v * w.sum()))


def test_a_captured_step_of_the_whole_block():
    """Forward, backward and the update in one graph, the step number on the GPU:
    replays leave the parameters of the same steps run one by one. (Atomics in
    torch's embedding gradient and in the core's delta gradient may add in
    another order: 1e-5 of the largest value, three steps of lr 1e-3.)"""
    from sunnynet_b200 import kernels
    params, tokens = make()
    runs = []
    for captured in (False, True):
        leaves = [v.clone().requires_grad_() for v in params.values()]
        m, s = ([torch.zeros_like(v) for v in leaves] for _ in range(2))
        step = torch.zeros(1, dtype=torch.int64, device="cuda")

        def one():
            step.add_(1)
            named = dict(zip(params, leaves))
            x = forward_without_core(named, tokens[:, :-1])
            grads = torch.autograd.grad(loss_of(x, tokens[:, 1:]), leaves, allow_unused=True)
            grads = [torch.zeros_like(v) if g is None else g.contiguous() for g, v in zip(grads, leaves)]
            with torch.no_grad():
                kernels.adamw_step(leaves, grads, m, s, step, lr=1e-3)

        if captured:
            state = [v.detach().clone() for v in leaves]
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                one()
            torch.cuda.current_stream().wait_stream(side)
            with torch.no_grad():
                for v, a in zip(leaves, state):
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
        assert step.item() == 3
        runs.append([v.detach().clone() for v in leaves])
    for a, b in zip(*runs):
        assert ((a - b).abs() <= 1e-5 * a.abs().max()).all()


def forward_without_core(params, tokens):
    """(The core's calls wait for the GPU, as the reference's return when done:
    they cannot be captured.)"""
    from sunnynet_b200.kernels import layer_norm
    x = params["embed"][tokens]
    q = layer_norm(x, params["g1"], params["b1"], EPS) @ params["proj"].T
    s = q[..., :D] * torch.sigmoid(q[..., D:]) * params["delta"]
    return layer_norm(x + s, params["g2"], params["b2"], EPS) @ params["embed"].T / 8
