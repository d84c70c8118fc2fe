"""What the dense (unquantised) projection and expert operators are measured on.

Three operators of the package, each with its plain form in elementary torch operations:

* ``linear``        out = act(x W^T + b) + r, rounded once
* ``gated_linear``  out = act(x Wg^T) * (x Wu^T), rounded once
* ``moe``           a whole mixture-of-experts layer from hidden states for a few tokens: router
                    projection, routing, gated experts, weighted sum, shared expert, residual

Layer sizes are those of the package's own configurations (hidden 2048 / 4096, expert sizes 768, 1408,
5632 and 14336, 128 / 60 / 8 experts), or generic odd ones.
"""
import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # attention's output projection in a decode step: one token, the residual stream added
        dict(name="linear 1x2048x2048", op="linear", m=1, n=2048, k=2048, type="bf16", act="none", bias=False, residual=True),
        # a small decode batch through an MLP's first projection with bias
        dict(name="linear 7x14336x4096", op="linear", m=7, n=14336, k=4096, type="fp16", act="gelu", bias=True, residual=False),
        # a short prompt, down projection of one expert-sized MLP, bias and residual
        dict(name="linear 200x2048x1408", op="linear", m=200, n=2048, k=1408, type="bf16", act="none", bias=True, residual=True),
        # sizes that no tile divides, as of a classifier head or an adapter
        dict(name="linear 333x1001x1000", op="linear", m=333, n=1001, k=1000, type="fp16", act="gelu_tanh", bias=True, residual=False),
        # down projection of a prompt of 2048 tokens, residual added
        dict(name="linear 2048x4096x14336", op="linear", m=2048, n=4096, k=14336, type="bf16", act="none", bias=False, residual=True),
        # gate and up projections of one token: a shared expert's sizes
        dict(name="gated 1x5632x2048", op="gated", m=1, n=5632, k=2048, type="bf16", act="silu"),
        # a decode batch of 37 requests, or a short prompt
        dict(name="gated 37x14336x4096", op="gated", m=37, n=14336, k=4096, type="fp16", act="silu"),
        # a long prompt
        dict(name="gated 4096x14336x4096", op="gated", m=4096, n=14336, k=4096, type="bf16", act="silu"),
        # one decode step of one request: 128 experts, 8 for the token
        dict(name="moe 1 token 128x768", op="moe", t=1, e=128, topk=8, h=2048, i=768, shared=0, type="bf16", softmax=True,
             renorm=True, residual=True),
        # six requests: 60 experts, 4 for each token, and a shared expert
        dict(name="moe 6 tokens 60x1408", op="moe", t=6, e=60, topk=4, h=2048, i=1408, shared=5632, type="bf16", softmax=True,
             renorm=False, residual=True),
        # sixteen drafted or batched tokens over many small experts
        dict(name="moe 16 tokens 128x768", op="moe", t=16, e=128, topk=8, h=2048, i=768, shared=0, type="bf16", softmax=True,
             renorm=True, residual=False),
        # few large experts, softmax over the chosen ones only, half precision
        dict(name="moe 5 tokens 8x14336", op="moe", t=5, e=8, topk=2, h=4096, i=14336, shared=0, type="fp16", softmax=False,
             renorm=True, residual=False),
    ]


def _log_between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["linear", "gated", "moe"])
    dt = rng.choice(["bf16", "fp16"])
    if kind == "moe":
        while True:
            e = _log_between(rng, 4, 128)
            c = dict(op="moe", t=rng.randint(1, 16), e=e, topk=rng.randint(1, min(8, e)), h=16 * _log_between(rng, 16, 256),
                     i=16 * _log_between(rng, 8, 896), shared=rng.choice([0, 0, 16 * _log_between(rng, 8, 352)]), type=dt,
                     softmax=rng.random() < 0.7, renorm=rng.random() < 0.5, residual=rng.random() < 0.5)
            # no more weights than the largest listed layer, nor more gathered pairs
            if c["e"] * c["h"] * c["i"] <= 8 * 4096 * 14336 and c["t"] * c["topk"] * c["h"] * c["i"] <= 10 * 4096 * 14336:
                return c
    while True:
        m, n, k = _log_between(rng, 1, 4096), _log_between(rng, 64, 14336), 8 * _log_between(rng, 8, 1792)
        if m * n * k * (2 if kind == "gated" else 1) <= 2048 * 4096 * 14336:
            break
    if kind == "gated":
        return dict(op="gated", m=m, n=n, k=k, type=dt, act=rng.choice(["silu", "silu", "gelu_tanh"]))
    return dict(op="linear", m=m, n=n, k=k, type=dt, act=rng.choice(["none", "none", "silu", "gelu", "gelu_tanh", "relu"]),
                bias=rng.random() < 0.5, residual=rng.random() < 0.5)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _TYPES[case["type"]]

    def rand(*shape, scale=1.0):
        return torch.empty(*shape, dtype=dt, device="cuda").normal_(0.0, scale, generator=g)

    s = dict(case)
    if case["op"] == "moe":
        t, e, h, i, sh = case["t"], case["e"], case["h"], case["i"], case["shared"]
        s["x"] = rand(t, h)
        # routers favour some experts: rows of unequal length
        length = torch.empty(e, 1, device="cuda").uniform_(0.5, 2.0, generator=g)
        s["router"] = (rand(e, h, scale=1.0 / math.sqrt(h)).float() * length).to(dt)
        s["gate"], s["up"] = rand(e, i, h, scale=1.0 / math.sqrt(h)), rand(e, i, h, scale=1.0 / math.sqrt(h))
        s["down"] = rand(e, h, i, scale=1.0 / math.sqrt(i))
        s["shared_w"] = None
        if sh:
            s["shared_w"] = dict(gate=rand(sh, h, scale=1.0 / math.sqrt(h)), up=rand(sh, h, scale=1.0 / math.sqrt(h)),
                                 down=rand(h, sh, scale=1.0 / math.sqrt(sh)), gate_vec=rand(h, scale=1.0 / math.sqrt(h)))
        s["r"] = rand(t, h) if case["residual"] else None
        # the caller's buffers for the routing, as a model that reports it keeps them
        s["ids"] = torch.empty(t, case["topk"], dtype=torch.int64, device="cuda")
        s["w"] = torch.empty(t, case["topk"], dtype=dt, device="cuda")
        s["out"] = torch.empty(t, h, dtype=dt, device="cuda")
        if own:  # the layer that a program keeps beside its weights: it borrows them and copies nothing
            from nano_ktrans_b200 import DenseMoeLayer

            s["layer"] = DenseMoeLayer(s["gate"], s["up"], s["down"], top_k=case["topk"], router_use_softmax=case["softmax"],
                                       normalize_topk_prob=case["renorm"], shared=s["shared_w"])
        return s
    m, n, k = case["m"], case["n"], case["k"]
    s["x"] = rand(m, k)
    if case["op"] == "gated":
        s["gate"], s["up"] = rand(n, k, scale=1.0 / math.sqrt(k)), rand(n, k, scale=1.0 / math.sqrt(k))
    else:
        s["weight"] = rand(n, k, scale=1.0 / math.sqrt(k))
        s["bias"] = rand(n) if case["bias"] else None
        s["r"] = rand(m, n) if case["residual"] else None
    s["out"] = torch.empty(m, n, dtype=dt, device="cuda")
    return s


def _act(v, name):
    if name == "silu":
        return v / (1.0 + torch.exp(-v))
    if name == "gelu":
        return 0.5 * v * (1.0 + torch.erf(v * math.sqrt(0.5)))
    if name == "gelu_tanh":
        return 0.5 * v * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (v + 0.044715 * v * v * v)))
    if name == "relu":
        return v.clamp_min(0.0)
    return v


def _routing(s):
    """Expert ids and weights of each token.  Logits, probabilities and their sum are rounded to the layer's type,
    as the model's own modules round them; they are computed in 64 bits first, because a value beside a rounding
    border would otherwise pick another expert.  Equal values go to the lowest expert."""
    dt, k = s["x"].dtype, s["topk"]
    logits = (s["x"].double() @ s["router"].double().T).to(dt).double()
    if s["softmax"]:
        p = torch.exp(logits - logits.amax(1, keepdim=True))
        p = (p / p.sum(1, keepdim=True)).to(dt)
        w, ids = torch.sort(p, dim=1, descending=True, stable=True)
        w, ids = w[:, :k], ids[:, :k]
        if s["renorm"]:
            w = (w.double() / w.double().sum(1, keepdim=True).to(dt).double()).to(dt)
    else:
        v, ids = torch.sort(logits, dim=1, descending=True, stable=True)
        v, ids = v[:, :k], ids[:, :k]
        w = torch.exp(v - v[:, :1])
        w = (w / w.sum(1, keepdim=True)).to(dt)
    return ids, w


def _plain_moe(s):
    ids, w = _routing(s)
    x = s["x"].float()
    g = torch.einsum("tkih,th->tki", s["gate"][ids].float(), x)
    u = torch.einsum("tkih,th->tki", s["up"][ids].float(), x)
    a = _act(g, "silu") * u * w.float().unsqueeze(2)
    out = torch.einsum("tkhi,tki->th", s["down"][ids].float(), a)
    if s["shared_w"] is not None:
        sw = s["shared_w"]
        a = _act(x @ sw["gate"].float().T, "silu") * (x @ sw["up"].float().T)
        open_ = 1.0 / (1.0 + torch.exp(-(x @ sw["gate_vec"].float())))
        out = out + open_.unsqueeze(1) * (a @ sw["down"].float().T)
    if s["r"] is not None:
        out = out + s["r"].float()
    return [out.to(s["x"].dtype), ids, w.contiguous()]


def run(state):
    s = state
    if own:
        import nano_ktrans_b200 as nk

        if s["op"] == "moe":
            s["layer"].forward_x(s["x"], s["router"], residual=s["r"], out=s["out"], out_ids=s["ids"], out_weights=s["w"])
            return [s["out"], s["ids"], s["w"]]
        if s["op"] == "gated":
            return nk.gated_linear(s["x"], s["gate"], s["up"], activation=s["act"], out=s["out"])
        return nk.linear(s["x"], s["weight"], s["bias"], activation=s["act"], residual=s["r"], out=s["out"])
    if s["op"] == "moe":
        return _plain_moe(s)
    x = s["x"].float()
    if s["op"] == "gated":
        return (_act(x @ s["gate"].float().T, s["act"]) * (x @ s["up"].float().T)).to(s["x"].dtype)
    v = x @ s["weight"].float().T
    if s["bias"] is not None:
        v = v + s["bias"].float()
    v = _act(v, s["act"])
    if s["r"] is not None:
        v = v + s["r"].float()
    return v.to(s["x"].dtype)


def work(case):
    if case["op"] == "moe":
        t, e, k, h, i, sh = (case[n] for n in ("t", "e", "topk", "h", "i", "shared"))
        used = e * (1.0 - (1.0 - k / e) ** t)  # experts that at least one token picks, routed evenly
        weights = e * h + used * 3 * h * i + 3 * h * sh + (h if sh else 0)
        rows = t * h * (3 if case["residual"] else 2)
        return {"bytes": 2 * (weights + rows) + t * k * 10, "flops": 2 * t * (e * h + 3 * k * h * i + 3 * h * sh)}
    m, n, k = case["m"], case["n"], case["k"]
    if case["op"] == "gated":
        return {"bytes": 2 * (m * k + 2 * n * k + m * n), "flops": 4 * m * n * k}
    extra = (m * n if case["residual"] else 0) + (n if case["bias"] else 0)
    return {"bytes": 2 * (m * k + n * k + m * n + extra), "flops": 2 * m * n * k}


def exact(case, seed):
    s = prepare(case, seed)
    f64 = torch.float64

    def act(v):
        name = case["act"]
        if name == "silu":
            return v * torch.sigmoid(v)
        if name == "gelu":
            return v * torch.special.ndtr(v)
        if name == "gelu_tanh":
            return v * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (v + 0.044715 * v.pow(3)))
        if name == "relu":
            return torch.where(v > 0, v, torch.zeros_like(v))
        return v

    x = s["x"].to(f64)
    if case["op"] == "linear":
        v = torch.matmul(x, s["weight"].to(f64).t())
        v = act(v if s["bias"] is None else v + s["bias"].to(f64))
        return v if s["r"] is None else v + s["r"].to(f64)
    if case["op"] == "gated":
        return act(torch.matmul(x, s["gate"].to(f64).t())) * torch.matmul(x, s["up"].to(f64).t())
    # the layer, token by token and expert by expert; the routing is rounded by its definition
    ids, w = _routing(s)
    total = torch.zeros_like(x) if s["r"] is None else s["r"].to(f64).clone()
    for t, row in enumerate(ids.tolist()):
        for j, e in enumerate(row):
            g, u = s["gate"][e].to(f64) @ x[t], s["up"][e].to(f64) @ x[t]
            total[t] += w[t, j].to(f64) * (s["down"][e].to(f64) @ (g * torch.sigmoid(g) * u))
    if s["shared_w"] is not None:
        sw = {name: v.to(f64) for name, v in s["shared_w"].items()}
        g, u = x @ sw["gate"].t(), x @ sw["up"].t()
        total += torch.sigmoid(x @ sw["gate_vec"]).unsqueeze(1) * ((g * torch.sigmoid(g) * u) @ sw["down"].t())
    return [total, None, None]
