"""Tree attention inputs whose scores rise, fall and peak by tens of powers of two along the context, and an emulation of the tile-by-tile softmax
that says what such inputs ask of a kernel: how often a row's state is rescaled, and what a rescale left out would do."""
import math
import random

import torch

import tree_cases as tc

D = tc.D
LOG2 = 1.0 / math.log(2.0)
SHAPES = [([3, 4, 1], [900, 31, 1500], 16, 8), ([7, 12, 0], [1333, 700, 5], 8, 2), ([25, 6], [1100, 1696], 8, 2), ([40, 33], [1300, 64], 8, 1)]


def growing_case(nodes, prefix, Hq, Hkv, seed):
    """Every key has a level along each of four directions, every query looks along one of them, 5 to 20 times its noise: levels that rise in steps of
    10 to 40 log2 units (at other places for every direction and kv head), fall in such steps, peak somewhere and fall back, or stay."""
    c = tc.attention_case(nodes, prefix, Hq, Hkv, 16, seed)
    rng = random.Random(seed)
    unit = 16.0 * c["scale"] * LOG2     # log2 units that a level of one is worth to a query that looks along it
    q, k = c["q"].clone(), c["k"].clone()
    for t in range(q.shape[0]):
        for h in range(Hq):
            q[t, h, :4] = 0
            q[t, h, (t + 3 * h) % 4] = 16.0
    for b, (n, P) in enumerate(zip(nodes, prefix)):
        if not n:
            continue
        slots = c["r2t"][int(c["rows"][b]), : P + n].long()
        for h in range(Hkv):
            steps = sorted(rng.randrange(1, P + n) for _ in range(min(7, (P + n) // 40)))
            up = [0.0]
            for _ in steps:
                up.append(up[-1] + rng.uniform(10, 40))
            at = [sum(s <= j for s in steps) for j in range(P + n)]
            late = [sum(s <= j + 50 for s in steps) for j in range(P + n)]
            top = rng.randrange(P + n)
            for j in range(P + n):
                level = (up[at[j]], up[-1] - up[late[j]], 35.0 if abs(j - top) < 20 else 0.0, 0.0)
                k[slots[j], h, :4] = torch.tensor([x / unit for x in level]).to(k.dtype)
    c["q"], c["k"] = q, k
    return c


def online_softmax(c, waves, skip=()):
    """(values, rescales) as a kernel with 32-key tiles finds them: `waves` states per row, every waves-th tile each, joined at the end; a state is
    rescaled when a tile's maximum lies 8 log2 units above its reference.  skip: what a wrong kernel leaves out ("o", "l": the rescale of the values,
    of the sum; "join": the factors of the join)."""
    q, k, v = c["q"].double(), c["k"].double(), c["v"].double()
    G = q.shape[1] // k.shape[1]
    out, count, at = torch.zeros_like(q), 0, 0
    for b, (n, P) in enumerate(zip(c["nodes"], c["prefix_list"])):
        slots = c["r2t"][int(c["rows"][b]), : P + n].long()
        see = torch.ones(n, P + n, dtype=torch.bool)
        see[:, P:] = torch.tensor([[c["masks"][at + i] >> j & 1 for j in range(n)] for i in range(n)], dtype=torch.bool).view(n, n)
        for h in range(q.shape[1]):
            s = (q[at: at + n, h] @ k[slots, h // G].T * (c["scale"] * LOG2)).masked_fill(~see, -math.inf)
            states = []
            for w in range(waves):
                m, l, o = torch.full((n,), -3e38, dtype=torch.float64), torch.zeros(n, dtype=torch.float64), torch.zeros(n, D, dtype=torch.float64)
                started = torch.zeros(n, dtype=torch.bool)
                for t0 in range(32 * w, P + n, 32 * waves):
                    x = s[:, t0: t0 + 32]
                    top = x.amax(1)
                    grown = top > m + 8
                    new = torch.where(grown, top, m)
                    f = torch.exp2(m - new)
                    count += int((grown & started).sum())
                    started |= grown
                    if "l" not in skip:
                        l = l * f
                    if "o" not in skip:
                        o = o * f[:, None]
                    m = new
                    p = torch.exp2(x - m[:, None])
                    l, o = l + p.sum(1), o + p @ v[slots[t0: t0 + 32], h // G]
                states.append((m, l, o))
            M = torch.stack([m for m, _, _ in states]).amax(0)
            f = [torch.ones_like(M) if "join" in skip else torch.exp2(m - M) for m, _, _ in states]
            L = sum(x * l for x, (_, l, _) in zip(f, states))
            O = sum(x[:, None] * o for x, (_, _, o) in zip(f, states))
            out[at: at + n, h] = torch.where((L > 0)[:, None], O / L[:, None], torch.zeros_like(O))
        at += n
    return out, count
