"""Cases for the operators at the ends and in the middle of a training step:
the embedding of tokens with its gradient, the norm and the clipping of all
gradients, and linear attention with a decay for each head, for prompts and
training and, as a recurrence, for single tokens.

``run`` computes a case either by the framework's calls (``own``) or in plain
torch: elementary operations in 32 bits (the sums of decays in 64, as their
differences are what counts), rounded once at the end. ``exact`` gives the same
outputs from the definitions in 64 bits.

Widths and vocabularies are those of the model shapes the benchmark runs
(d512 i896 r320 V16384 L4; d768 i1344 r480 V32000 L12; d1536; heads of 64) and
generic odd sizes around them.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
SIZE = {"float32": 4, "bfloat16": 2, "float16": 2}
CHUNK = 64  # tokens of one chunk of the plain form


def listed():
    return [
        # the rows of one decode step of 64 conversations
        {"name": "embed 64 of 16384x512", "op": "embed", "tokens": 64, "vocab": 16384, "width": 512, "dtype": "float32", "grad": False},
        # a training batch of 16 x 2048 tokens, few of the words making most of it
        {"name": "embed grad 32768 of 32000x768", "op": "embed", "tokens": 32768, "vocab": 32000, "width": 768, "dtype": "bfloat16", "grad": True},
        # odd numbers throughout
        {"name": "embed grad 5003 of 4999x1001", "op": "embed", "tokens": 5003, "vocab": 4999, "width": 1001, "dtype": "float32", "grad": True},
        # one small layer fine-tuned: nine tensors of a few hundred to some ten thousand values
        {"name": "clip 1 layer d64", "op": "clip", "layers": 1, "width": 64, "inner": 96, "rank": 32, "vocab": 512, "dtype": "float32", "scale": True},
        # the norm alone, as a step that hands its factor to the optimiser or only logs it
        {"name": "norm 11 layers d509 bf16", "op": "clip", "layers": 11, "width": 509, "inner": 893, "rank": 319, "vocab": 5003, "dtype": "bfloat16", "scale": False},
        # the 100M-class model, scaled in place
        {"name": "clip 12 layers d768", "op": "clip", "layers": 12, "width": 768, "inner": 1344, "rank": 480, "vocab": 32000, "dtype": "float32", "scale": True},
        # one conversation's next token
        {"name": "step 1 x 12 of 64", "op": "step", "batch": 1, "heads": 12, "shared": 1, "dk": 64, "dv": 64, "dtype": "bfloat16", "decay": "head"},
        # a decode batch's, its decays computed from the tokens
        {"name": "step 256 x 12 of 64", "op": "step", "batch": 256, "heads": 12, "shared": 1, "dk": 64, "dv": 64, "dtype": "bfloat16", "decay": "token"},
        # one long prompt, queries, keys and values as one projection left them
        {"name": "prompt 8192 x 12 of 128", "op": "mix", "batch": 1, "time": 8192, "heads": 12, "shared": 1, "dk": 128, "dv": 128, "dtype": "bfloat16", "decay": "head", "ragged": False, "state": False, "grad": False},
        # a padded batch of prompts of different lengths that go on from earlier states
        {"name": "prompts 64 x 257 ragged", "op": "mix", "batch": 64, "time": 257, "heads": 12, "shared": 1, "dk": 64, "dv": 64, "dtype": "float32", "decay": "token", "ragged": True, "state": True, "grad": False},
        # a training batch of 16 x 2048 tokens
        {"name": "mix grad 16 x 2048", "op": "mix", "batch": 16, "time": 2048, "heads": 12, "shared": 1, "dk": 64, "dv": 64, "dtype": "bfloat16", "decay": "token", "ragged": False, "state": False, "grad": True},
        # odd sizes, three heads to each head of queries and keys, gradients through the state
        {"name": "mix grad 3 x 1001 shared", "op": "mix", "batch": 3, "time": 1001, "heads": 6, "shared": 3, "dk": 40, "dv": 72, "dtype": "float32", "decay": "head", "ragged": False, "state": True, "grad": True},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["embed", "embed grad", "clip", "step", "mix", "mix", "mix grad"])
    dtype = rng.choice(["float32", "bfloat16", "float16"])
    if op in ("embed", "embed grad"):
        width = _log(rng, 8, 2048)
        return {"op": "embed", "tokens": _log(rng, 1, min(65536, 25000000 // width)), "vocab": _log(rng, 16, min(100000, 25000000 // width)), "width": width,
                "dtype": dtype, "grad": op == "embed grad"}
    if op == "clip":
        width = _log(rng, 16, 768)
        return {"op": "clip", "layers": rng.randint(1, 12), "width": width, "inner": width * 7 // 4 + rng.randint(0, 1), "rank": width * 5 // 8 + rng.randint(0, 1),
                "vocab": _log(rng, 64, 32000), "dtype": dtype, "scale": rng.random() < 0.5}
    shared = rng.choice([1, 1, 2, 4])
    heads = shared * rng.randint(1, 16 // shared)
    size = lambda: rng.choice([64, 128, 8 * rng.randint(1, 16), rng.randint(3, 128)])  # noqa: E731
    case = {"op": "step", "heads": heads, "shared": shared, "dk": size(), "dv": size(), "dtype": dtype, "decay": rng.choice(["head", "token"])}
    if op == "step":
        return {**case, "batch": _log(rng, 1, min(1024, 12000000 // (heads * case["dk"] * case["dv"])))}
    most = 6000000 // (heads * max(case["dk"], case["dv"]))  # tokens
    time = _log(rng, 1, min(8192, most))
    return {**case, "op": "mix", "time": time, "batch": _log(rng, 1, min(64, most // time)), "ragged": rng.random() < 0.3, "state": rng.random() < 0.5, "grad": op == "mix grad"}


def _shapes(case):
    """The tensors of one model: embedding, final norm, and for each layer its norm, taps, memory vector and five matrices."""
    d, i, r = case["width"], case["inner"], case["rank"]
    layer = [(d,), (d,), (4, d), (d,), (r, d), (2 * d, r), (i, d), (d, i), (d,), (d, d)]
    return [(case["vocab"], d), (d,), (d,)] + layer * case["layers"]


def _lengths(case):
    """Tokens of each sequence of a padded batch: the whole, and less and less."""
    B, T = case["batch"], case["time"]
    return [T - (37 * b) % (T // 2 + 1) for b in range(B)] if case["ragged"] else [T] * B


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype = DTYPES[case["dtype"]]
    randn = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    rand = lambda *shape: torch.rand(*shape, generator=g, device="cuda")  # noqa: E731
    if case["op"] == "embed":
        n, v, d = case["tokens"], case["vocab"], case["width"]
        # words come about as often as one over their rank
        s = {"op": "embed", "grad": case["grad"], "scale": math.sqrt(d), "tokens": torch.exp(rand(n).double() * math.log(v)).long().clamp_max(v) - 1}
        s["weight"] = (randn(v, d) / math.sqrt(d)).to(dtype)
        if case["grad"]:
            s["dout"] = randn(n, d).to(dtype)
            s["weight"].requires_grad_(True)
        return s
    if case["op"] == "clip":
        shapes = _shapes(case)
        at = [0]
        for t in shapes:
            at.append(at[-1] + -(-math.prod(t) // 64) * 64)  # one buffer, each tensor behind the other
        flat = randn(at[-1])
        flat *= rand(at[-1]) > 0.1  # rows of words that did not occur, among others
        flat = flat.to(dtype)
        grads = [flat[a:a + math.prod(t)].view(t) for a, t in zip(at, shapes)]
        return {"op": "clip", "flat": flat, "grads": grads, "scale": case["scale"], "max_norm": 0.5 * math.sqrt(sum(math.prod(t) for t in shapes))}
    B, H, dk, dv = case["batch"], case["heads"], case["dk"], case["dv"]
    Hk, T = H // case["shared"], case.get("time", 1)
    wide = randn(B, T, Hk * dk * 2 + H * dv).to(dtype)  # one projection
    q, k, v = wide.split([Hk * dk, Hk * dk, H * dv], dim=2)
    s = {"op": case["op"], "grad": case.get("grad", False), "q": q.unflatten(2, (Hk, dk)), "k": k.unflatten(2, (Hk, dk)), "v": v.unflatten(2, (H, dv)),
         "scale": 1 / dk, "lengths": None}
    if case["decay"] == "head":  # half-lives from some tokens to thousands
        s["log_decay"] = torch.log1p(-torch.exp2(-3.0 - 8.0 * torch.arange(H, device="cuda") / H))
    else:
        s["log_decay"] = -torch.nn.functional.softplus(randn(B, T, H) - 2.0)
    if case["op"] == "step":
        s = {**s, **{n: s[n][:, 0] for n in ("q", "k", "v")}, "state": randn(B, H, dk, dv)}
        if case["decay"] == "token":
            s["log_decay"] = s["log_decay"][:, 0]
        return s
    s["state"] = randn(B, H, dk, dv) if case["state"] else None
    if case["ragged"]:
        s["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")
    if s["grad"]:
        for n in ("q", "k", "v", "log_decay", "state"):
            if s[n] is not None:
                s[n] = s[n].contiguous().requires_grad_(True)
        s["dout"] = randn(B, T, H, dv).to(dtype)
        s["dstate"] = randn(B, H, dk, dv) if case["state"] else None
    return s


def _leaves(s):
    return [s[n] for n in ("q", "k", "v", "log_decay", "state") if s[n] is not None]


def _plain_embed(s):
    w, tokens, d = s["weight"].detach(), s["tokens"], s["weight"].shape[1]
    out = (w[tokens].float() * s["scale"]).to(w.dtype)
    if not s["grad"]:
        return out
    dw = torch.zeros(w.shape, device=w.device).index_add_(0, tokens, s["dout"].float().view(-1, d)) * s["scale"]
    return out, dw.to(w.dtype)


def _plain_clip(s):
    total = torch.stack([x.float().square().sum() for x in s["grads"]]).sum().sqrt()
    factor = (s["max_norm"] / (total + 1e-6)).clamp_max(1.0)
    if s["scale"]:
        for x in s["grads"]:
            x.copy_(x.float() * factor)
        return total, s["flat"]
    return total, factor


def _wide(x, heads):
    return x.float().repeat_interleave(heads // x.shape[-2], dim=-2)


def _plain_step(s):
    H = s["v"].shape[1]
    q, k, v = _wide(s["q"], H), _wide(s["k"], H), s["v"].float()
    new = s["state"] * torch.exp(s["log_decay"])[..., None, None] + k[..., :, None] * v[..., None, :]
    s["state"].copy_(new)
    out = (q[..., :, None] * new).sum(-2) * s["scale"]
    return out.to(s["v"].dtype), s["state"]


def _plain_mix(q, k, v, log_decay, state, lengths, scale):
    """Chunks of the sequence: within each by products of its tokens, from one to the next by the state."""
    B, T, H, dv = v.shape
    q, k, v = _wide(q, H), _wide(k, H), v.float()
    dk, N = q.shape[-1], -(-T // CHUNK)
    decay = log_decay.double().expand(B, T, H)
    inside = None
    if lengths is not None:
        inside = torch.arange(T, device=v.device)[None, :, None] < lengths[:, None, None]
        k, v, decay = (torch.where(inside[..., None], k, 0.0), torch.where(inside[..., None], v, 0.0), torch.where(inside, decay, 0.0))
    pad = lambda x, *more: torch.cat([x, x.new_zeros(B, N * CHUNK - T, H, *more)], 1).unflatten(1, (N, CHUNK)).movedim(3, 1)  # noqa: E731
    q, k, v, c = pad(q, dk), pad(k, dk), pad(v, dv), pad(decay).cumsum(-1)
    upto = torch.ones(CHUNK, CHUNK, dtype=torch.bool, device=v.device).tril()
    near = torch.where(upto, c[..., :, None] - c[..., None, :], -math.inf).float().exp()
    out = ((q @ k.transpose(-1, -2)) * near) @ v
    q = q * c.float().exp()[..., None]
    last = k * (c[..., -1:] - c).float().exp()[..., None]
    whole = c[..., -1].float().exp()[..., None, None]
    S = state if state is not None else v.new_zeros(B, H, dk, dv)
    before = []
    for n in range(N):
        before.append(S)
        S = S * whole[:, :, n] + last[:, :, n].transpose(-1, -2) @ v[:, :, n]
    out = (out + q @ torch.stack(before, 2)).movedim(1, 3).flatten(1, 2)[:, :T] * scale
    return out if inside is None else torch.where(inside[..., None], out, 0.0), S


def _run_mix(s):
    leaves = _leaves(s)
    if not own:
        out, state = _plain_mix(s["q"], s["k"], s["v"], s["log_decay"], s["state"], s["lengths"], s["scale"])
        out = out.to(s["v"].dtype)
    else:
        from sunnynet_b200.kernels import linear_attention

        out, state = linear_attention(s["q"], s["k"], s["v"], s["log_decay"], s["state"], s["lengths"], s["scale"])
    if not s["grad"]:
        return out, state
    ends, grads = ([out], [s["dout"]]) if s["dstate"] is None else ([out, state], [s["dout"], s["dstate"]])
    return (out.detach(), state.detach(), *torch.autograd.grad(ends, leaves, grads))


def run(state):
    s = state
    if s["op"] == "clip":
        s["max_norm"] *= 0.999  # a little below what the last pass left: each pass has to scale
    if s["op"] == "mix":
        return _run_mix(s)
    if not own:
        return {"embed": _plain_embed, "clip": _plain_clip, "step": _plain_step}[s["op"]](s)
    from sunnynet_b200 import kernels

    if s["op"] == "embed":
        out = kernels.embedding(s["tokens"], s["weight"], s["scale"])
        return (out.detach(), *torch.autograd.grad(out, s["weight"], s["dout"])) if s["grad"] else out
    if s["op"] == "step":
        return kernels.linear_attention_step(s["q"], s["k"], s["v"], s["log_decay"], s["state"], s["scale"]), s["state"]
    if s["scale"]:
        return kernels.clip_grads(s["grads"], s["max_norm"]), s["flat"]
    return kernels.grad_norm(s["grads"], s["max_norm"])


def work(case):
    e = SIZE[case["dtype"]]
    if case["op"] == "embed":
        n, v, d = case["tokens"], case["vocab"], case["width"]
        rows = v * (1 - math.exp(-n / (v * math.log(v)) * 2)) if v > 1 else 1  # about as many of them are read
        bytes_, flops = n * 8 + (n + min(n, v, rows)) * d * e, n * d
        return {"bytes": bytes_ + (n + v) * d * e, "flops": 2 * flops} if case["grad"] else {"bytes": bytes_, "flops": flops}
    if case["op"] == "clip":
        n = sum(math.prod(t) for t in _shapes(case))
        return {"bytes": n * e * (2 if case["scale"] else 1), "flops": n * (3 if case["scale"] else 2)}
    B, H, dk, dv = case["batch"], case["heads"], case["dk"], case["dv"]
    Hk = H // case["shared"]
    gates = 4 * H if case["decay"] == "token" else 0
    token = (2 * Hk * dk + H * dv) * e + gates
    if case["op"] == "step":
        return {"bytes": B * (token + H * dv * e + 8 * H * dk * dv), "flops": 5 * B * H * dk * dv}
    n, states = sum(_lengths(case)), 4 * B * H * dk * dv
    bytes_ = n * token + B * case["time"] * H * dv * e + states * (2 if case["state"] else 1)
    if not case["grad"]:
        return {"bytes": bytes_, "flops": 4 * n * H * dk * dv}
    bytes_ += n * (token + H * dv * e) + B * case["time"] * token + states * (2 if case["state"] else 0)
    return {"bytes": bytes_, "flops": 14 * n * H * dk * dv}


def _exact_embed(s):
    w, tokens = s["weight"].detach().double(), s["tokens"]
    out = w.index_select(0, tokens) * s["scale"]
    if not s["grad"]:
        return out
    # the rows in the order of their words, and differences of their running sums where a word ends
    order = torch.argsort(tokens, stable=True)
    upto = s["dout"].double()[order].cumsum(0)
    ends = torch.bincount(tokens, minlength=w.shape[0]).cumsum(0)
    at = torch.cat([torch.zeros_like(upto[:1]), upto])[ends]
    return out, torch.diff(at, dim=0, prepend=torch.zeros_like(at[:1])) * s["scale"]


def _exact_clip(s):
    total = math.sqrt(sum(float((x.double() ** 2).sum()) for x in s["grads"]))
    factor = min(1.0, s["max_norm"] * 0.999 / (total + 1e-6))
    norm = torch.tensor(total, dtype=torch.float64, device=s["flat"].device)
    if not s["scale"]:
        return norm, torch.full_like(norm, factor)
    new, at = s["flat"].double(), 0
    for x in s["grads"]:
        new[at:at + x.numel()] *= factor
        at += -(-x.numel() // 64) * 64
    return norm, new


def _exact_mix(s, step):
    """Token by token: the state and, for the gradients, its gradient backwards."""
    D = {n: s[n].detach().double() for n in ("q", "k", "v", "log_decay")}
    if step:
        D = {n: x[:, None] if n != "log_decay" or x.dim() == 2 else x for n, x in D.items()}
    q, k, v = D["q"], D["k"], D["v"]
    B, T, H, dv = v.shape
    Hk, dk = q.shape[2:]
    each = torch.arange(H, device=v.device) // (H // Hk)  # its head of queries and keys
    f = D["log_decay"].exp().expand(B, T, H)
    live = torch.ones(B, T, 1, dtype=torch.float64, device=v.device)
    if s["lengths"] is not None:
        live = (torch.arange(T, device=v.device)[None] < s["lengths"][:, None]).double()[..., None]
    f = f * live + (1 - live)  # behind a sequence's end the state stays
    S = torch.zeros(B, H, dk, dv, dtype=torch.float64, device=v.device)
    if s["state"] is not None:
        S = s["state"].detach().double().clone()
    out, dq = torch.zeros_like(v), torch.zeros(B, T, H, dk, dtype=torch.float64, device=v.device)
    do = s["dout"].double() * live[..., None] if s["grad"] else None
    for t in range(T):
        S = S * f[:, t, :, None, None] + (k[:, t, each] * live[:, t, :, None])[..., None] * v[:, t, :, None, :]
        out[:, t] = torch.einsum("bhk,bhkv->bhv", q[:, t, each], S) * live[:, t, :, None]
        if s["grad"]:
            dq[:, t] = torch.einsum("bhkv,bhv->bhk", S, do[:, t]) * s["scale"]
    out = out * s["scale"]
    if not s["grad"]:
        return out[:, 0] if step else out, S
    dk_, dv_ = torch.zeros_like(dq), torch.zeros_like(v)
    dS = torch.zeros_like(S) if s["dstate"] is None else s["dstate"].double()
    dg = torch.zeros(B, T, H, dtype=torch.float64, device=v.device)
    right = (dS * S).sum((-1, -2))  # what the next token's decay is worth
    for t in reversed(range(T)):
        on = live[:, t, :, None]
        dS = dS + (q[:, t, each] * s["scale"])[..., None] * do[:, t, :, None, :]
        dk_[:, t] = torch.einsum("bhkv,bhv->bhk", dS, v[:, t]) * on
        dv_[:, t] = torch.einsum("bhkv,bhk->bhv", dS, k[:, t, each]) * on
        right = right + ((q[:, t, each] * dq[:, t]).sum(-1) - (k[:, t, each] * dk_[:, t]).sum(-1))
        dg[:, t] = right * live[:, t]
        dS = dS * f[:, t, :, None, None]
    fold = lambda x: x.unflatten(2, (Hk, H // Hk)).sum(3)  # noqa: E731
    dg = dg.sum((0, 1)) if s["log_decay"].dim() == 1 else dg
    return (out, S, fold(dq), fold(dk_), dv_, dg) + ((dS,) if s["state"] is not None else ())


def exact(case, seed):
    with torch.no_grad():
        s = prepare(case, seed)
        if s["op"] == "embed":
            return _exact_embed(s)
        if s["op"] == "clip":
            return _exact_clip(s)
        return _exact_mix(s, s["op"] == "step")
