"""The dense gated feed-forward block and the low-rank adapters, as a program uses them, with inputs, work and exact values.

A case names what is called (`op`) and its sizes:

  ffn       gated_ffn: y = (silu(x Wg^T) * (x Wu^T)) Wd^T on bf16 activations, decode and prefill sizes
  train     gated_ffn that saves for the backward pass, then gated_ffn_backward: output and all gradients
  linear    adapter_linear: y = x W^T + scale (x A^T) B^T, every token with the adapter of its request
  adapted   gated_ffn with adapters on its three projections

Requests are runs of tokens; request j uses adapter order[j % n], every eighth request none (id -1).
"""
import math

import torch

own = False
DEVICE = "cuda"


def listed():
    return [
        # one user decoding through a small dense block: nothing but latency
        {"name": "ffn_t1", "op": "ffn", "tokens": 1, "d": 2048, "ff": 2816},
        # an odd decode batch on a large model: the weights are read once
        {"name": "ffn_t37", "op": "ffn", "tokens": 37, "d": 4096, "ff": 14336},
        # a short prompt of odd length
        {"name": "ffn_t333", "op": "ffn", "tokens": 333, "d": 2048, "ff": 5632},
        # prefill of a long prompt
        {"name": "ffn_t5000", "op": "ffn", "tokens": 5000, "d": 2048, "ff": 5632},
        # a training step of a test model
        {"name": "train_t64", "op": "train", "tokens": 64, "d": 512, "ff": 1408},
        # fine-tuning on one ragged sequence
        {"name": "train_t1021", "op": "train", "tokens": 1021, "d": 2048, "ff": 5632},
        # fine-tuning of a large block on a packed batch
        {"name": "train_t4096", "op": "train", "tokens": 4096, "d": 4096, "ff": 14336},
        # one user with an adapter on a small projection
        {"name": "linear_t1", "op": "linear", "tokens": 1, "d": 2048, "out": 2048, "rank": 8, "adapters": 4, "requests": 1},
        # a decode batch in which nearly every request has its own adapter
        {"name": "linear_t64", "op": "linear", "tokens": 64, "d": 4096, "out": 4096, "rank": 16, "adapters": 80, "requests": 64},
        # prompts of several requests in one batch, high rank, wide projection
        {"name": "linear_t2501", "op": "linear", "tokens": 2501, "d": 4096, "out": 14336, "rank": 64, "adapters": 12, "requests": 7},
        # decode through a large block, adapters on all three projections
        {"name": "adapted_t48", "op": "adapted", "tokens": 48, "d": 4096, "ff": 14336, "rank": 16, "adapters": 32, "requests": 48},
        # prompts and decoding requests mixed
        {"name": "adapted_t1100", "op": "adapted", "tokens": 1100, "d": 2048, "ff": 5632, "rank": 32, "adapters": 16, "requests": 40},
    ]


def _log_int(rng, lo, hi, step=1):
    return max(lo, step * int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)))


def draw(rng):
    op = rng.choice(["ffn", "train", "linear", "adapted"])
    case = {"op": op, "tokens": _log_int(rng, 1, 4096 if op == "train" else 8192), "d": _log_int(rng, 256, 4096, 16)}
    case["out" if op == "linear" else "ff"] = _log_int(rng, 256, 14336, 16)
    if op in ("linear", "adapted"):
        case["rank"] = rng.choice([8, 16, 24, 32, 64, 128])
        case["adapters"] = _log_int(rng, 1, 96)
        case["requests"] = min(case["tokens"], _log_int(rng, 1, 96))
    largest = 4096 * 4096 * 14336
    width = case.get("ff", case.get("out"))
    while case["tokens"] * case["d"] * width * (1 if op == "train" else 0.5) > largest:
        case["tokens"] //= 2
    return case


def _used(case):
    return len({j % case["adapters"] for j in range(case["requests"]) if j % 8 != 7})


def work(case):
    T, d, op = case["tokens"], case["d"], case["op"]
    if op == "linear":
        r, out = case["rank"], case["out"]
        return {"bytes": 2 * (T * d + d * out + T * out + _used(case) * r * (d + out)) + 4 * T,
                "flops": 2 * T * d * out + 2 * T * r * (d + out)}
    F = case["ff"]
    if op == "train":
        return {"bytes": 2 * (4 * T * d + 6 * d * F), "flops": 18 * T * d * F}
    w = {"bytes": 2 * (2 * T * d + 3 * d * F), "flops": 6 * T * d * F}
    if op == "adapted":
        w["bytes"] += 2 * _used(case) * 3 * case["rank"] * (d + F) + 4 * T
        w["flops"] += 6 * T * case["rank"] * (d + F)
    return w


def _adapter_ids(case, gen):
    T, n, R = case["tokens"], case["adapters"], case["requests"]
    cuts = torch.randperm(T - 1, generator=gen, device=DEVICE)[: R - 1] + 1 if R > 1 else torch.empty(0, device=DEVICE, dtype=torch.int64)
    starts = torch.zeros(T, device=DEVICE, dtype=torch.int64)
    starts[cuts] = 1
    request = torch.cumsum(starts, 0)
    order = torch.randperm(n, generator=gen, device=DEVICE)
    return torch.where(request % 8 == 7, -1, order[request % n]).to(torch.int32)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(int(seed))

    def rand(std, *shape):
        return (torch.randn(shape, generator=gen, device=DEVICE) * std).to(torch.bfloat16)

    T, d, op = case["tokens"], case["d"], case["op"]
    s = {"op": op, "x": rand(1.0, T, d)}
    shapes = {"weight": (case["out"], d)} if op == "linear" else {"gate": (case["ff"], d), "up": (case["ff"], d), "down": (d, case["ff"])}
    for name, shape in shapes.items():
        s[name] = rand(0.02, *shape)
    if op == "train":
        s["dy"] = rand(1.0, T, d)
    if op in ("linear", "adapted"):
        s["ids"] = _adapter_ids(case, gen)
        n, r = case["adapters"], case["rank"]
        s["adapters"] = {}
        for name, (rows, cols) in shapes.items():
            a, b = rand(cols ** -0.5, n, r, cols), rand(0.02, n, rows, r)
            s["adapters"][name] = (a, b, torch.rand(n, generator=gen, device=DEVICE) + 1.0)
    return s


def _delta(x, ids, adapter):
    a, b, scale = (t.float() for t in adapter)
    n, r, _ = a.shape
    mine = (ids[:, None] == torch.arange(n, device=x.device)).float() * scale
    v = (x @ a.flatten(0, 1).T).view(-1, n, r) * mine[:, :, None]
    return v.flatten(1) @ b.transpose(1, 2).reshape(n * r, -1)


def _project(s, name, x):
    y = x @ s[name].float().T
    return y + _delta(x, s["ids"], s["adapters"][name]) if "adapters" in s else y


def run(s):
    if own:
        from ateniaengine_b200 import LowRankAdapters, adapter_linear, gated_ffn, gated_ffn_backward

        if s["op"] == "linear":
            return adapter_linear(s["x"], s["weight"], LowRankAdapters(*s["adapters"]["weight"]), s["ids"])
        w = s["gate"], s["up"], s["down"]
        if s["op"] == "ffn":
            return gated_ffn(s["x"], *w)
        if s["op"] == "adapted":
            adapters = {name: LowRankAdapters(*abs_) for name, abs_ in s["adapters"].items()}
            return gated_ffn(s["x"], *w, adapters=adapters, adapter_ids=s["ids"])
        y, saved = gated_ffn(s["x"], *w, save=True)
        return (y, *gated_ffn_backward(s["dy"], s["x"], *w, saved))
    low = torch.bfloat16
    x = s["x"].float()
    if s["op"] == "linear":
        return _project(s, "weight", x).to(low)
    g, u = _project(s, "gate", x), _project(s, "up", x)
    sig = 1 / (1 + torch.exp(-g))
    h = g * sig * u
    y = _project(s, "down", h).to(low)
    if s["op"] != "train":
        return y
    dy = s["dy"].float()
    dh = dy @ s["down"].float()
    dg, du = dh * u * sig * (1 + g * (1 - sig)), dh * g * sig
    dx = dg @ s["gate"].float() + du @ s["up"].float()
    return y, dx.to(low), (dg.T @ x).to(low), (du.T @ x).to(low), (dy.T @ h).to(low)


def exact(case, seed):
    s = prepare(case, seed)
    x = s["x"].double()

    def project(name, z):
        y = z @ s[name].double().T
        if "adapters" in s:
            a, b, scale = s["adapters"][name]
            for i in torch.unique(s["ids"]).tolist():
                if i >= 0:
                    rows = torch.nonzero(s["ids"] == i)[:, 0]
                    y[rows] += scale[i].double() * (z[rows] @ a[i].double().T @ b[i].double().T)
        return y

    if s["op"] == "linear":
        return project("weight", x)
    g, u = project("gate", x), project("up", x)
    sig = torch.sigmoid(g)
    h = g * sig * u
    y = project("down", h)
    if s["op"] != "train":
        return y
    dy = s["dy"].double()
    dh = dy @ s["down"].double()
    dg = dh * u * (sig + g * sig * (1 - sig))
    du = dh * g * sig
    return y, dg @ s["gate"].double() + du @ s["up"].double(), dg.T @ x, du.T @ x, dy.T @ h
