"""Cases for the operators a training step and a serving step leave to the
caller: the draw of the next token, layer norm with its gradients, and the
AdamW update of a model's tensors.

``run`` computes a case either by the framework's calls (``own``) or in plain
torch: elementary operations in 32 bits (the draw in 64, where cumulative
sums decide between neighbouring tokens), rounded once at the end. ``exact``
gives the same outputs from the definitions in 64 bits.

Widths and vocabularies are those of the model shapes the benchmark runs
(d512 i896 r320 V16384 L4; d768 i1344 r480 V32000 L12; d1536; V65536) and
generic odd sizes around them.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
SIZE = {"float32": 4, "bfloat16": 2, "float16": 2}
BLOCK = 256  # values that share one scale in the 8-bit states
F8 = torch.float8_e4m3fn
F8_MAX, F8_MIN = 448.0, 2.0 ** -9  # largest value, smallest above zero
HYPER = {"lr": 3e-4, "beta1": 0.9, "beta2": 0.95, "eps": 1e-8, "weight_decay": 0.1}


def listed():
    return [
        # one conversation: latency of the usual nucleus draw
        {"name": "sample 1x32000 k40 p0.95", "op": "sample", "rows": 1, "vocab": 32000, "dtype": "float32", "mix": "topkp"},
        # a serving batch whose requests each bring their own settings, greedy ones and masked vocabularies among them
        {"name": "sample 256x16384 mixed", "op": "sample", "rows": 256, "vocab": 16384, "dtype": "float32", "mix": "mixed"},
        # half-precision logits in a padded buffer, an odd vocabulary, min-p
        {"name": "sample 64x65521 bf16 min-p", "op": "sample", "rows": 64, "vocab": 65521, "dtype": "bfloat16", "mix": "minp"},
        # a full decode batch, nucleus over the whole vocabulary
        {"name": "sample 1024x32000 p0.9", "op": "sample", "rows": 1024, "vocab": 32000, "dtype": "float32", "mix": "topp"},
        # the norm of one decode step
        {"name": "norm 64x512", "op": "norm", "rows": 64, "width": 512, "dtype": "float32", "grad": False},
        # the norm of one prefill chunk: 64 sequences of 256 tokens
        {"name": "norm 16384x1536", "op": "norm", "rows": 16384, "width": 1536, "dtype": "float32", "grad": False},
        # forward and backward of a training batch in half precision
        {"name": "norm grad 32768x768 bf16", "op": "norm", "rows": 32768, "width": 768, "dtype": "bfloat16", "grad": True},
        # an odd width and a ragged number of rows
        {"name": "norm grad 5003x1001", "op": "norm", "rows": 5003, "width": 1001, "dtype": "float32", "grad": True},
        # fine-tuning the vectors and one small layer
        {"name": "adamw 1 layer d64", "op": "adamw", "layers": 1, "width": 64, "inner": 96, "rank": 32, "vocab": 512, "bits": 32, "dtype": "float32"},
        # the small model, full states
        {"name": "adamw 4 layers d512", "op": "adamw", "layers": 4, "width": 512, "inner": 896, "rank": 320, "vocab": 16384, "bits": 32, "dtype": "float32"},
        # odd sizes throughout, half-precision weights and gradients, full states
        {"name": "adamw 11 layers d509 bf16", "op": "adamw", "layers": 11, "width": 509, "inner": 893, "rank": 319, "vocab": 5003, "bits": 32, "dtype": "bfloat16"},
        # the 100M-class model with states in 8 bits
        {"name": "adamw 12 layers d768 8-bit", "op": "adamw", "layers": 12, "width": 768, "inner": 1344, "rank": 480, "vocab": 32000, "bits": 8, "dtype": "float32"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["sample", "sample", "norm", "norm grad", "adamw"])
    dtype = rng.choice(["float32", "bfloat16", "float16"])
    if op == "sample":
        rows = _log(rng, 1, 1024)
        vocab = _log(rng, 2, min(200000, 32768000 // rows))
        return {"op": "sample", "rows": rows, "vocab": vocab, "dtype": dtype, "mix": rng.choice(["topkp", "mixed", "minp", "topp"])}
    if op in ("norm", "norm grad"):
        width = _log(rng, 16, 20000)
        return {"op": "norm", "rows": _log(rng, 1, min(100000, 25000000 // width)), "width": width, "dtype": dtype, "grad": op == "norm grad"}
    width = _log(rng, 16, 768)
    return {"op": "adamw", "layers": rng.randint(1, 12), "width": width, "inner": width * 7 // 4 + rng.randint(0, 1), "rank": width * 5 // 8 + rng.randint(0, 1),
            "vocab": _log(rng, 64, 32000), "bits": rng.choice([8, 32]), "dtype": dtype}


def _shapes(case):
    """The tensors of one model: embedding, final norm, and for each layer its norm, taps, memory vector and five matrices."""
    d, i, r = case["width"], case["inner"], case["rank"]
    layer = [(d,), (d,), (4, d), (d,), (r, d), (2 * d, r), (i, d), (d, i), (d,), (d, d)]
    return [(case["vocab"], d), (d,), (d,)] + layer * case["layers"]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def _rand(g, *shape, dtype=torch.float32):
    return torch.rand(*shape, generator=g, device="cuda", dtype=dtype)


def _encode(x, floor):
    """8-bit codes and block scales of x: scale = max|x| / 448; where `floor`, what is above zero stays above zero."""
    blocks = torch.nn.functional.pad(x.reshape(-1), (0, -x.numel() % BLOCK)).view(-1, BLOCK)
    scale = blocks.abs().amax(1) * torch.tensor(1.0 / F8_MAX, dtype=x.dtype, device=x.device)
    q = torch.where(scale[:, None] > 0, blocks / scale[:, None], 0.0)
    if floor:
        q = torch.where(blocks > 0, q.clamp_min(F8_MIN), q)
    return q.reshape(-1)[: x.numel()].float().to(F8), scale


def _decode(codes, scale, kind):
    return codes.to(kind) * scale.to(kind).repeat_interleave(BLOCK)[: codes.numel()]


def prepare(case, seed):
    g = _gen(seed)
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "sample":
        n, v = case["rows"], case["vocab"]
        wide = -(-v // 64) * 64 if case["mix"] == "minp" else v  # min-p rows lie in a padded buffer, as a padded head leaves them
        x = (_randn(g, n, wide) * 2.5).to(dtype)
        s = {"op": "sample", "logits": x[:, :v]}
        if case["mix"] == "mixed":
            masked = _rand(g, n, 1) < 0.25  # a quarter of the requests may use a tenth of the vocabulary only
            s["logits"].masked_fill_(masked & (_rand(g, n, v) > 0.1), -math.inf)
            pick = torch.arange(n, device="cuda") % 4
            s["temperature"] = torch.where(pick == 0, 0.0, 0.5 + _rand(g, n, dtype=torch.float64))
            s["top_k"] = torch.where(pick == 1, 0, 1 + (_rand(g, n) * 100).int()).int()
            s["top_p"] = torch.where(pick == 2, 1.0, 0.5 + 0.5 * _rand(g, n, dtype=torch.float64))
            s["min_p"] = torch.where(pick == 3, 0.1 * _rand(g, n, dtype=torch.float64), 0.0)
        else:
            s.update({"topkp": {"temperature": 0.8, "top_k": 40, "top_p": 0.95, "min_p": 0.0},
                      "topp": {"temperature": 1.0, "top_k": 0, "top_p": 0.9, "min_p": 0.0},
                      "minp": {"temperature": 1.3, "top_k": 0, "top_p": 1.0, "min_p": 0.02}}[case["mix"]])
        s["u"] = _rand(g, n, dtype=torch.float64)
        return s
    if case["op"] == "norm":
        n, d = case["rows"], case["width"]
        s = {"op": "norm", "grad": case["grad"], "eps": 1e-5}
        s["x"] = (_randn(g, n, d) * 1.5 + 0.25).to(dtype)
        s["weight"], s["bias"] = 1 + 0.1 * _randn(g, d), 0.1 * _randn(g, d)
        if case["grad"]:
            s["dy"] = _randn(g, n, d).to(dtype)
            for k in ("x", "weight", "bias"):
                s[k].requires_grad_(True)
        return s
    # one buffer for each kind of value, the model's tensors lying in it one behind the other at multiples of a block
    shapes = _shapes(case)
    sizes = [math.prod(t) for t in shapes]
    at = [0]
    for n in sizes:
        at.append(at[-1] + -(-n // BLOCK) * BLOCK)
    views = lambda flat: [flat[a:a + n].view(t) for a, n, t in zip(at, sizes, shapes)]  # noqa: E731
    total = at[-1]
    s = {"op": "adamw", "bits": case["bits"], "step": 100}
    param = (0.02 * _randn(g, total)).to(dtype)
    used = _rand(g, total) > 0.1  # embedding rows of tokens that have not occurred, among others
    grad = (1e-3 * _randn(g, total) * used).to(dtype)
    avg = 3e-4 * _randn(g, total) * used
    sq = (1e-3 * _randn(g, total)).square() * used
    s["flat"] = {"param": param}
    if case["bits"] == 8:
        for name, x in (("exp_avg", avg), ("exp_avg_sq", sq.sqrt())):
            s["flat"][name], s["flat"][name + "_scale"] = _encode(x, name == "exp_avg_sq")
            s[name] = views(s["flat"][name])
            s[name + "_scale"] = [s["flat"][name + "_scale"][a // BLOCK:b // BLOCK] for a, b in zip(at, at[1:])]
    else:
        s["flat"]["exp_avg"], s["flat"]["exp_avg_sq"] = avg, sq
        s["exp_avg"], s["exp_avg_sq"] = views(avg), views(sq)
    s["params"], s["grads"] = views(param), views(grad)
    return s


def _column(v, like):
    return v[:, None] if isinstance(v, torch.Tensor) else torch.full((like.shape[0], 1), v, device=like.device)


def _plain_sample(s):
    x = s["logits"].float()
    n, v = x.shape
    top = x.amax(1, keepdim=True)
    ids = torch.arange(v, device=x.device)
    greedy = torch.where(x == top, ids, v).amin(1)
    temp, k = _column(s["temperature"], x).double(), _column(s["top_k"], x).long()
    top_p, min_p = _column(s["top_p"], x).double(), _column(s["min_p"], x).double()
    xs, order = torch.sort(x, dim=1, descending=True, stable=True)
    w = torch.exp((xs.double() - top.double()) / torch.where(temp > 0, temp, 1.0)).nan_to_num(0.0)
    kth = xs.gather(1, torch.where((k > 0) & (k < v), k, v) - 1)
    w = w * (xs >= kth)
    upto = w.cumsum(1)
    w = w * (((upto - w) < top_p * upto[:, -1:]) | (top_p >= 1))
    w = w * (w >= min_p)
    upto = torch.zeros_like(w).scatter_(1, order, w).cumsum(1)
    drawn = (upto <= s["u"].double()[:, None] * upto[:, -1:]).sum(1).clamp_max(v - 1)
    token = torch.where(temp[:, 0] > 0, drawn, greedy)
    return torch.where(top[:, 0] > -math.inf, token, -1).int()


def _plain_norm(s):
    x, w = s["x"].detach().float(), s["weight"].detach()
    centred = x - x.mean(1, keepdim=True)
    rstd = torch.rsqrt(centred.square().mean(1, keepdim=True) + s["eps"])
    unit = centred * rstd
    y = (unit * w + s["bias"].detach()).to(s["x"].dtype)
    if not s["grad"]:
        return y
    dy = s["dy"].float()
    du = dy * w
    dx = rstd * (du - du.mean(1, keepdim=True) - unit * (du * unit).mean(1, keepdim=True))
    return y, dx.to(s["x"].dtype), (dy * unit).sum(0), dy.sum(0)


def _factors(step):
    """What a step's number makes of the rates: the step size with the first moment's correction, and the factor of the second moment's root."""
    return HYPER["lr"] / (1 - HYPER["beta1"] ** step), 1 / math.sqrt(1 - HYPER["beta2"] ** step)


def _plain_adamw(s):
    size, root = _factors(s["step"])
    b1, b2 = HYPER["beta1"], HYPER["beta2"]
    for i, (param, grad, avg, sq) in enumerate(zip(s["params"], s["grads"], s["exp_avg"], s["exp_avg_sq"])):
        p, g = param.reshape(-1).float(), grad.reshape(-1).float()
        if s["bits"] == 8:
            m = _decode(avg.reshape(-1), s["exp_avg_scale"][i], torch.float32)
            v = _decode(sq.reshape(-1), s["exp_avg_sq_scale"][i], torch.float32).square()
        else:
            m, v = avg.reshape(-1), sq.reshape(-1)
        m = m * b1 + g * (1 - b1)
        v = v * b2 + g.square() * (1 - b2)
        r = v.sqrt()
        p = p * (1 - HYPER["lr"] * HYPER["weight_decay"]) - m / (r * root + HYPER["eps"]) * size
        param.view(-1).copy_(p)
        if s["bits"] == 8:
            for to, scale, x in ((avg, s["exp_avg_scale"][i], m), (sq, s["exp_avg_sq_scale"][i], r)):
                codes, blocks = _encode(x, x is r)
                to.view(-1).copy_(codes)
                scale.copy_(blocks)
        else:
            avg.view(-1).copy_(m)
            sq.view(-1).copy_(v)


def _own(s):
    if s["op"] == "sample":
        from sunnynet_b200.sampling import sample

        return sample(s["logits"], s["u"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])
    from sunnynet_b200 import kernels

    if s["op"] == "norm":
        y = kernels.layer_norm(s["x"], s["weight"], s["bias"], s["eps"])
        return (y.detach(), *torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), s["dy"])) if s["grad"] else y
    kernels.adamw_step(s["params"], s["grads"], s["exp_avg"], s["exp_avg_sq"], s["step"], avg_scale=s.get("exp_avg_scale"),
                       sq_scale=s.get("exp_avg_sq_scale"), **HYPER)


def run(state):
    if state["op"] == "adamw":
        state["step"] += 1
    if own:
        out = _own(state)
    else:
        out = {"sample": _plain_sample, "norm": _plain_norm, "adamw": _plain_adamw}[state["op"]](state)
    return state["flat"] if state["op"] == "adamw" else out


def work(case):
    e = SIZE[case["dtype"]]
    if case["op"] == "sample":
        n, v = case["rows"], case["vocab"]
        return {"bytes": n * v * e + 8 * n + 4 * n, "flops": 3 * n * v}
    if case["op"] == "norm":
        n, d = case["rows"], case["width"]
        bytes_ = n * d * e * 2 + 8 * d
        return {"bytes": bytes_ + (n * d * e * 2 + 12 * d if case["grad"] else 0), "flops": n * d * (20 if case["grad"] else 8)}
    n = sum(math.prod(t) for t in _shapes(case))
    return {"bytes": n * (3 * e + (4 + 16 / BLOCK if case["bits"] == 8 else 16)), "flops": 15 * n}


def _exact_sample(s):
    """Each row by itself: the kept set by values, then the first id whose weight and those before it exceed u of the whole."""
    x, u = s["logits"].double().cpu(), s["u"].double().cpu()
    setting = {k: _column(s[k], x).double().cpu()[:, 0].tolist() for k in ("temperature", "top_k", "top_p", "min_p")}
    tokens = []
    for row, (r, t, k, p, least) in enumerate(zip(x, *setting.values())):
        best = float(r.max())
        if best == -math.inf:
            tokens.append(-1)
        elif t <= 0:
            tokens.append(int((r == best).nonzero()[0]))
        else:
            ids = (r > -math.inf).nonzero()[:, 0]
            if 0 < k < len(r) and k < len(ids):
                ids = ids[r[ids] >= r[ids].topk(int(k)).values[-1]]
            w = torch.exp((r[ids] - best) / t)
            if 0 < p < 1:
                by = torch.argsort(-r[ids], stable=True)
                ahead = torch.cat([torch.zeros(1, dtype=torch.float64), w[by].cumsum(0)[:-1]])
                few = by[ahead < p * w.sum()].sort().values
                ids, w = ids[few], w[few]
            ids, w = ids[w >= least], w[w >= least]
            upto = w.cumsum(0)
            tokens.append(int(ids[min(int(torch.searchsorted(upto, u[row] * upto[-1], right=True)), len(ids) - 1)]))
    return torch.tensor(tokens, dtype=torch.int32)


def _exact_norm(s):
    x, w, b = (s[k].detach().double() for k in ("x", "weight", "bias"))
    var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
    sd = (var + s["eps"]).sqrt()
    y = (x - mean) / sd * w + b
    if not s["grad"]:
        return y
    dy = s["dy"].double()
    # y_i depends on x_j by w_i/sd (delta_ij - 1/d - (x_i - mean)(x_j - mean)/(d sd^2))
    t = dy * w
    dx = (t - t.mean(1, keepdim=True) - (x - mean) * (t * (x - mean)).mean(1, keepdim=True) / sd ** 2) / sd
    return y, dx, (dy * (x - mean) / sd).sum(0), dy.sum(0)


def _exact_adamw(s):
    t = s["step"] + 1
    out = {k: v.double() for k, v in s["flat"].items()}
    g = torch.zeros_like(out["param"])
    start = 0
    for x in s["grads"]:
        g[start:start + x.numel()] = x.reshape(-1).double()
        start += -(-x.numel() // BLOCK) * BLOCK
    inside = torch.zeros_like(g, dtype=torch.bool)
    start = 0
    for x in s["grads"]:
        inside[start:start + x.numel()] = True
        start += -(-x.numel() // BLOCK) * BLOCK
    wide = {k: v.repeat_interleave(BLOCK) for k, v in out.items() if k.endswith("_scale")}
    eight = s["bits"] == 8
    m = out["exp_avg"] * wide["exp_avg_scale"] if eight else out["exp_avg"]
    v = (out["exp_avg_sq"] * wide["exp_avg_sq_scale"]) ** 2 if eight else out["exp_avg_sq"]
    m = HYPER["beta1"] * m + (1 - HYPER["beta1"]) * g
    v = HYPER["beta2"] * v + (1 - HYPER["beta2"]) * g ** 2
    to = m / (1 - HYPER["beta1"] ** t) / ((v / (1 - HYPER["beta2"] ** t)).sqrt() + HYPER["eps"])
    new = {"param": out["param"] * (1 - HYPER["lr"] * HYPER["weight_decay"]) - HYPER["lr"] * to}
    if eight:
        for k, x in (("exp_avg", m), ("exp_avg_sq", v.sqrt())):
            blocks = torch.where(inside, x, 0.0).view(-1, BLOCK)
            scale = blocks.abs().amax(1) / F8_MAX
            q = blocks / scale.clamp_min(1e-300)[:, None]
            if k == "exp_avg_sq":
                q = torch.where(blocks > 0, q.clamp_min(F8_MIN), q)
            new[k], new[k + "_scale"] = q.reshape(-1).float().to(F8).double(), scale
    else:
        new["exp_avg"], new["exp_avg_sq"] = m, v
    return {k: torch.where(inside, x, out[k]) if x.shape == inside.shape else x for k, x in new.items()}


def exact(case, seed):
    with torch.no_grad():
        return {"sample": _exact_sample, "norm": _exact_norm, "adamw": _exact_adamw}[case["op"]](prepare(case, seed))
