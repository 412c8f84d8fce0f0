"""Inputs of the gated block and the adapters for which every sum and every rounded operand is exact, so that the results are known to the
last bit: a k-block, an adapter or a term that a kernel leaves out, or a partial sum in fewer bits, shows.

All values are small integers times powers of two.  Sums: the magnitudes of a product's terms, in units of the smallest of them, stay
below 2^23, so any order of f32 additions is exact.  Activation: g is 64 for every token and feature (128 or 256 with an adapter of
the gate), where 1 + exp(-g) is 1 in f32: silu(g) = g, its slope is 1.  Operands rounded to bf16 (h, dg, du, the adapters' reduced
rows) have at most eight significant bits.  So a result is the exact one, rounded once to bf16 (`check_exact` asserts these conditions on the
values themselves).

g is the same everywhere, but a sum that lacks a part of its terms is not: C columns of x are 1 and carry 64 / C of the gate each, spread over
the reduction; the others come in pairs far apart, alike in x and opposite in the gate."""
import math

import torch

BIG = 2.0 ** 23


def signs(gen, *shape):
    return torch.randint(0, 2, shape, generator=gen, device=gen.device, dtype=torch.int8).double() * 2 - 1


def sparse(gen, per_row, *shape):
    """-1, 0 or 1, about `per_row` nonzeros in the last dimension and one more among its last eight places (a short last block)."""
    keep = torch.rand(shape, generator=gen, device=gen.device) < min(1.0, per_row / shape[-1])
    row = torch.arange(shape[-2], device=gen.device)
    keep[..., row, shape[-1] - 1 - row % 8] = True
    return signs(gen, *shape) * keep


def columns(d, device):
    """The constant columns and the two sides of the pairs."""
    c = 1 << int(math.log2(min(max(d // 2, 8), 1024)))
    constant = (torch.arange(c, device=device) * d) // c
    rest = torch.ones(d, dtype=torch.bool, device=device)
    rest[constant] = False
    rest = torch.nonzero(rest)[:, 0]
    half = len(rest) // 2
    return constant, rest[:half], rest[half:2 * half]


def generator(seed, device):
    gen = torch.Generator(device=device)
    gen.manual_seed(seed)
    return gen


def make_x(T, d, seed, device):
    gen = generator(seed, device)
    x = signs(gen, T, d)
    constant, left, right = columns(d, device)
    x[:, right] = x[:, left]
    x[:, constant] = 1.0
    return x


def make_block(d, F, seed, device):
    """gate, up, down in f64: the values that bf16 holds too."""
    gen = generator(seed, device)
    constant, left, right = columns(d, device)
    gate = torch.zeros((F, d), dtype=torch.float64, device=device)
    side = signs(gen, F, len(left))
    gate[:, left], gate[:, right] = side, -side
    gate[:, constant] = 64.0 / len(constant)
    return gate, sparse(gen, 4.8, F, d), signs(gen, d, F)


def make_dy(T, d, seed, device):
    return sparse(generator(seed, device), 4.8, T, d)


def make_low(n, r, n_in, n_out, seed, device, per_row=8.0, b_per_row=None):
    """Adapters of any projection: (a, b, scale) with a sparse a, and a b that is sparse too on request."""
    gen = generator(seed, device)
    scale = torch.tensor([1.0, -1.0, 2.0, 0.5], dtype=torch.float64, device=device)[torch.randint(0, 4, (n,), generator=gen, device=device)]
    b = signs(gen, n, n_out, r) if b_per_row is None else sparse(gen, b_per_row, n, n_out, r)
    return sparse(gen, per_row, n, r, n_in), b, scale


def make_gate_low(n, r, d, F, seed, device):
    """Adapters that take g from 64 to 128 or 256: rank column 0 adds 64 or 192, the others come in pairs that add up to nothing."""
    gen = generator(seed, device)
    constant, _, _ = columns(d, device)
    a, b = sparse(gen, 8.0, n, r, d), signs(gen, n, F, r)
    half = (r - 1) // 2
    a[:, 1 + half:1 + 2 * half] = a[:, 1:1 + half]
    b[:, :, 1 + half:1 + 2 * half] = -b[:, :, 1:1 + half]
    a[:, 0] = 0.0
    a[:, 0, constant] = 64.0 / len(constant)
    b[:, :, 0] = torch.tensor([1.0, 3.0], dtype=torch.float64, device=device)[torch.randint(0, 2, (n, 1), generator=gen, device=device)]
    if r - 1 > 2 * half:
        b[:, :, r - 1] = 0.0
    return a, b, torch.ones(n, dtype=torch.float64, device=device)


def make_lows(parts, n, ranks, d, F, seed, device):
    """Adapters of the block's projections; u stays below 128 with those of up, and the reduced rows of down below 256 times g."""
    lows = {"gate": lambda r: make_gate_low(n, r, d, F, seed, device), "up": lambda r: make_low(n, r, d, F, seed + 1, device, 4.0, 4.0),
            "down": lambda r: make_low(n, r, F, d, seed + 2, device, 4.0)}
    return {p: lows[p](r) for p, r in zip(("gate", "up", "down"), ranks) if p in parts}


def make_ids(kind, T, n, seed, device):
    t = torch.arange(T, device=device)
    if kind == "runs":
        ids = (t * 5 // max(T, 1)) * 7 % n
    elif kind == "distinct":
        ids = torch.randperm(max(n, T), generator=generator(seed, device), device=device)[:T] % n
        ids = torch.where(t % 11 == 10, -1, ids)
    else:
        choice = torch.tensor([-1, n, 0, n - 1, -(2 ** 31), 2 ** 31 - 1], device=device)
        ids = choice[torch.randint(0, 6, (T,), generator=generator(seed, device), device=device)]
    return ids.to(torch.int32)


def check_sum(a, b, unit, what):
    """Products of a [m, k] and b [n, k] over k are exact in f32 in any order: multiples of `unit`, below 2^23 of them in magnitude."""
    most = (a.abs().amax(0) * b.abs().amax(0)).sum()
    if most >= BIG * unit:
        most = (a.abs() @ b.abs().T).max()
    assert most < BIG * unit, (what, most / unit)


def check_bf16(t, what):
    assert torch.equal(t.to(torch.bfloat16).to(t.dtype), t), what


def delta(x, low, ids, what, unit_x=1.0):
    """What the adapters add, and the reduced rows."""
    a, b, scale = low
    y = torch.zeros((x.shape[0], b.shape[1]), dtype=torch.float64, device=x.device)
    for i in torch.unique(ids).tolist():
        if not 0 <= i < a.shape[0]:
            continue
        rows = torch.nonzero(ids == i)[:, 0]
        check_sum(x[rows], a[i], unit_x * 2.0 ** -4, what)
        v = scale[i] * (x[rows] @ a[i].T)
        check_bf16(v, what + ": reduced rows")
        check_sum(v, b[i], unit_x / 2, what)
        y[rows] = v @ b[i].T
    return y


def linear(x, w, low=None, ids=None, unit_x=1.0, what="linear", unit_w=1.0):
    check_sum(x, w, unit_x * unit_w, what)
    y = x @ w.T
    return y if low is None else y + delta(x, low, ids, what, unit_x)


def forward(x, gate, up, down, lows=None, ids=None):
    """y, g, u, h; exact."""
    lows = lows or {}
    g = linear(x, gate, lows.get("gate"), ids, what="g", unit_w=2.0 ** -4)
    assert ((g == 64) | (g == 128) | (g == 256)).all()
    u = linear(x, up, lows.get("up"), ids, what="u")
    h = g * u
    check_bf16(h, "h")
    return linear(h, down, lows.get("down"), ids, unit_x=64.0, what="y"), g, u, h


def backward(dy, x, gate, up, down, u, h):
    """dx, dgate, dup, ddown; exact (g = 64)."""
    check_sum(dy, down.T, 1.0, "dh")
    dh = dy @ down
    dg, du = dh * u, dh * 64
    check_bf16(dg, "dg"), check_bf16(du, "du")
    check_sum(torch.cat([dg, du], 1), torch.cat([gate, up]).T, 2.0 ** -4, "dx")
    for a, b, unit, what in ((dg, x, 1.0, "dgate"), (du, x, 64.0, "dup"), (dy, h, 64.0, "ddown")):
        check_sum(a.T, b.T, unit, what)
    return dg @ gate + du @ up, dg.T @ x, du.T @ x, dy.T @ h


def low16(*ts):
    return [t.to(torch.bfloat16) for t in ts]


# Tokens, width, features: short calls; and, between them, every kernel at every cut of its reduction that the choice makes for each of the
# five products (single CTAs 128 and 256 columns wide and pairs, whole waves and a cut last one).
BLOCKS = [(1, 16, 16), (1, 512, 1408), (2, 48, 80), (4, 272, 144), (5, 512, 1408), (8, 64, 64), (9, 64, 128), (16, 1040, 48), (16, 272, 2064),
          (17, 32, 32), (17, 400, 160), (17, 656, 2160), (17, 2880, 9200), (18, 1952, 560), (64, 512, 1408), (100, 16, 2064), (127, 1040, 48),
          (128, 272, 144), (129, 272, 144), (130, 2528, 7808), (142, 1504, 9952), (148, 3968, 4928), (205, 2496, 2544), (255, 144, 272),
          (260, 3776, 1568), (278, 3056, 2016), (299, 3120, 3712), (300, 2064, 8208), (330, 2416, 6560), (363, 4032, 2544), (518, 2864, 3984),
          (526, 2688, 6528), (536, 2672, 8352), (784, 32, 6528), (1021, 2048, 5632), (1081, 848, 1840), (1757, 144, 672), (1837, 272, 672),
          (1861, 3024, 32), (1865, 528, 2480), (1967, 32, 32), (2061, 1760, 80), (2064, 2736, 2448), (2382, 1936, 32), (2396, 144, 2208),
          (2454, 1888, 1680), (2516, 2272, 1888), (2600, 2064, 4112), (2667, 1712, 912), (2883, 1584, 1184), (2895, 32, 1840)]
# Tokens, inputs, outputs, adapters, rank, ids; (rows of a few tokens with reduced rows from the tensor cores among them)
LINEARS = [(1, 16, 16, 1, 8, "odd"), (1, 512, 1408, 4, 16, "runs"), (5, 272, 144, 3, 24, "odd"), (8, 512, 400, 5, 128, "distinct"), (13, 528, 144, 20, 40, "distinct"),
           (8, 32768, 512, 3, 128, "runs"), (33, 64, 272, 40, 8, "distinct"), (64, 1040, 528, 70, 16, "distinct"), (64, 4096, 4096, 80, 16, "distinct"),
           (129, 144, 400, 150, 64, "distinct"), (130, 272, 2064, 9, 128, "odd"), (135, 3232, 2576, 12, 40, "runs"), (155, 2640, 4064, 40, 16, "distinct"),
           (300, 528, 144, 200, 16, "distinct"), (327, 3104, 3920, 40, 72, "odd"), (518, 2864, 3984, 5, 24, "runs"), (700, 1040, 1040, 600, 16, "distinct"),
           (1021, 1040, 1040, 12, 40, "runs"), (1676, 2144, 3344, 30, 8, "odd"), (2100, 512, 1552, 30, 64, "runs"), (2100, 272, 5632, 300, 16, "distinct"),
           (1500, 144, 5008, 40, 128, "odd"), (2883, 1184, 1584, 3, 96, "odd"), (5000, 5632, 2048, 9, 16, "runs")]
# Tokens, width, features, adapters, ranks of gate, up and down, ids
ADAPTED = [(1, 64, 96, 2, (8, 16, 24), "runs"), (4, 512, 1408, 3, (128, 64, 128), "distinct"), (11, 272, 144, 4, (24, 8, 128), "odd"), (24, 336, 368, 9, (8, 8, 8), "distinct"),
           (48, 512, 1408, 33, (16, 16, 16), "distinct"), (100, 1024, 14336, 6, (128, 128, 16), "distinct"), (128, 2048, 512, 5, (128, 128, 64), "runs"),
           (130, 2528, 7808, 40, (16, 16, 16), "distinct"), (142, 1504, 9952, 3, (40, 24, 64), "odd"), (200, 272, 400, 7, (8, 64, 40), "odd"),
           (330, 2416, 6560, 40, (32, 8, 16), "odd"), (397, 3104, 2512, 5, (16, 16, 48), "runs"), (700, 512, 5632, 50, (96, 40, 64), "odd"),
           (1100, 528, 1040, 16, (32, 32, 128), "runs"), (1100, 2048, 5632, 16, (24, 8, 32), "runs"), (1133, 3904, 960, 6, (64, 64, 64), "odd"),
           (1500, 272, 3600, 40, (128, 128, 16), "distinct"), (2102, 2368, 1504, 300, (8, 16, 8), "distinct")]
