"""The gated feed-forward block, its gradients and the low-rank adapters in 64 bits, each with a bound of what the kernels may be off.

Roundings: a bf16 rounding is off by at most 2^-8 of the value (half a step), every sum is f32: 2^-24 a term of the sum of the
magnitudes, whatever the order, doubled for tensor cores that truncate.  The exponential and the quotient of the activation are
within 2^-18 of the value.  What a rounded operand is off goes through the next product with the magnitudes of its weights.  An adapter's
reduced rows are one bf16 operand, or two (what the first leaves is rounded once more) where 32 of its rank exceed its input's width."""
import torch

BF = 2.0 ** -8
ACT = 2.0 ** -18


def f32_sum(a, b):
    """What sums over k of a [m, k] b [n, k]^T may be off in f32."""
    return 2 * a.shape[1] * 2.0 ** -24 * (a.abs() @ b.abs().T) + 1e-30


def project(x, w, low=None, ids=None, dx=None):
    """x w^T (+ adapters), and the bound before any rounding of the result; dx: what x is off."""
    y, e = x @ w.T, f32_sum(x, w)
    if dx is not None:
        e = e + dx @ w.abs().T
    if low is not None:
        a, b, scale = (t.double() for t in low)
        for i in range(a.shape[0]):
            rows = torch.nonzero(ids == i)[:, 0]
            if not len(rows):
                continue
            s = scale[i]
            v = s * (x[rows] @ a[i].T)
            dv = v.abs() * (BF if 32 * a.shape[1] <= x.shape[1] else BF * BF) + s.abs() * f32_sum(x[rows], a[i]) + 2.0 ** -22 * v.abs()
            if dx is not None:
                dv = dv + s.abs() * dx[rows] @ a[i].abs().T
            y[rows] += v @ b[i].T
            e[rows] += dv @ b[i].abs().T + f32_sum(v, b[i])
    return y, e


def adapter_linear(x, w, low, ids):
    y, e = project(x.double(), w.double(), low, ids)
    return y, e + (y.abs() + e) * BF


def forward(x, gate, up, down, adapters=None, ids=None, h_rounding=BF):
    """(y, bound of y), and what the backward pass needs of the way there."""
    low = adapters or {}
    x = x.double()
    g, eg = project(x, gate.double(), low.get("gate"), ids)
    u, eu = project(x, up.double(), low.get("up"), ids)
    s = torch.sigmoid(g)
    h = g * s * u
    dh = h.abs() * (h_rounding + ACT) + 1.1 * u.abs() * eg + (g * s).abs() * eu + 1.1 * eg * eu  # |silu'| <= 1.1
    y, e = project(h, down.double(), low.get("down"), ids, dx=dh)
    return (y, e + (y.abs() + e) * BF), (g, eg, u, eu, s, h, dh)


def backward(dy, x, gate, up, down):
    """[(dx, bound), (dgate, bound), (dup, bound), (ddown, bound)]"""
    _, (g, eg, u, eu, s, h, eh) = forward(x, gate, up, down)
    x, dy, gate, up, down = (t.double() for t in (x, dy, gate, up, down))
    d = dy @ down
    ed = f32_sum(dy, down.T)
    slope = s * (1 + g * (1 - s))
    dg, du = d * u * slope, d * g * s
    # |silu''| <= 0.5; the slope is a sum of s and g s (1 - s), each within ACT
    edg = dg.abs() * BF + (d * u).abs() * ACT * (s + (g * s * (1 - s)).abs() + 2 * (g * s).abs() * 2.0 ** -6)
    edg = edg + (u * slope).abs() * ed + 1.1 * d.abs() * eu + 0.5 * (d * u).abs() * eg + 2 * ed * (eu + u.abs() * eg)
    edu = du.abs() * (BF + ACT) + (g * s).abs() * ed + 1.1 * d.abs() * eg + 1.1 * ed * eg

    def rounded(v, e):
        return v, e + (v.abs() + e) * BF

    return [rounded(dg @ gate + du @ up, edg @ gate.abs() + edu @ up.abs() + f32_sum(torch.cat([dg, du], 1), torch.cat([gate, up]).T)),
            rounded(dg.T @ x, edg.T @ x.abs() + f32_sum(dg.T, x.T)),
            rounded(du.T @ x, edu.T @ x.abs() + f32_sum(du.T, x.T)),
            rounded(dy.T @ h, dy.abs().T @ eh + f32_sum(dy.T, h.T))]


def assert_within(got, ref_and_bound, what):
    ref, bound = ref_and_bound
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    over = (got.double() - ref).abs() / bound
    assert torch.isfinite(got.float()).all() and over.max() <= 1, f"{what}: {over.max().item():.3g} of the bound at {over.argmax().item()}"


def rand(seed, std, *shape):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return (torch.randn(shape, generator=gen, device="cuda") * std).to(torch.bfloat16)


def block(seed, d, F):
    return rand(seed, d ** -0.5, F, d), rand(seed + 1, d ** -0.5, F, d), rand(seed + 2, F ** -0.5, d, F)


def low_rank(seed, n, r, n_in, n_out):
    from ateniaengine_b200 import LowRankAdapters
    scale = rand(seed + 2, 1.0, n).float()
    return LowRankAdapters(rand(seed, n_in ** -0.5, n, r, n_in), rand(seed + 1, r ** -0.5, n, n_out, r), scale)


def ids_of(kind, T, n, seed=0):
    """one: one adapter; none; distinct: as many as there are; runs: requests of several tokens; odd: ids outside [0, n) too."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    t = torch.arange(T, device="cuda")
    if kind == "one":
        ids = torch.full((T,), n - 1, device="cuda")
    elif kind == "none":
        ids = torch.full((T,), -1, device="cuda")
    elif kind == "distinct":
        ids = torch.randperm(max(n, T), generator=gen, device="cuda")[:T] % n
    elif kind == "runs":
        ids = (t * 5 // max(T, 1)) * 7 % n
    else:
        choice = torch.tensor([-1, n, 0, n - 1, -(2 ** 31), 2 ** 31 - 1], device="cuda")
        ids = choice[torch.randint(0, 6, (T,), generator=gen, device="cuda")]
    return ids.to(torch.int32)
