"""Inputs and 64-bit oracles of the speculative-decoding operators (slot maps, tree attention, log probabilities, acceptance),
written from their definitions; shared by the CPU and the GPU tests."""
import random

import torch

D = 128


def tree_parents(rng, n, chain=False):
    return [-1] + [j - 1 if chain else max(0, j - 1 - int(rng.random() ** 2 * 6)) for j in range(1, n)]


def ancestor_masks(parents):
    """Python integers: bit j of node i's mask = j is i or above it."""
    out = []
    for j, p in enumerate(parents):
        p = p if 0 <= p < j else 0
        out.append((out[p] if j else 0) | 1 << j)
    return out


def pack_masks(masks, words):
    full = 2 ** 64 - 1
    rows = [[(m >> (64 * w)) & full for w in range(words)] for m in masks]
    return torch.tensor([[v - 2 ** 64 if v >> 63 else v for v in r] for r in rows], dtype=torch.int64).view(len(masks), words)


def page_rows(lens, width, page_size, rng, spare=0):
    """(table [len(lens), width] int32, pages left over, pages in all); pages in random order, page 0 never used."""
    need = [-(-n // page_size) for n in lens]
    pages = list(range(1, sum(need) + spare + 1))
    rng.shuffle(pages)
    table, at = torch.zeros((len(lens), width), dtype=torch.int32), 0
    for b, n in enumerate(lens):
        slots = [pages[at + i // page_size] * page_size + i % page_size for i in range(n)]
        table[b, :n] = torch.tensor(slots, dtype=torch.int32)
        at += need[b]
    return table, pages[at:], len(pages)


def cumulative(lens):
    return torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32)


def attention_case(nodes, prefix, Hq, Hkv, page_size, seed, layout="interleaved", chain=False, words=None):
    rng = random.Random(seed)
    g = torch.Generator().manual_seed(seed)
    lens = [p + n for p, n in zip(prefix, nodes)]
    table, _, pages = page_rows(lens, max(lens) + 3, page_size, rng)
    rows = list(range(len(nodes)))
    rng.shuffle(rows)
    r2t = torch.zeros_like(table)
    r2t[torch.tensor(rows)] = table
    slots = (pages + 1) * page_size
    if layout == "interleaved":
        kv = torch.randn(slots, 2, Hkv, D, generator=g).to(torch.bfloat16)
        k, v = kv[:, 0], kv[:, 1]
    else:
        k, v = (torch.randn(slots, Hkv, D, generator=g).to(torch.bfloat16) for _ in range(2))
    q = (torch.randn(sum(nodes), Hq, D, generator=g) * 1.5).to(torch.bfloat16)
    masks = [m for n in nodes for m in ancestor_masks(tree_parents(rng, n, chain)[:n])]
    words = words or max(1, -(-max(nodes) // 64))
    return dict(q=q, k=k, v=v, r2t=r2t, rows=torch.tensor(rows, dtype=torch.int32), cu=cumulative(nodes), prefix=torch.tensor(prefix, dtype=torch.int32),
                mask=pack_masks(masks, words), masks=masks, nodes=list(nodes), prefix_list=list(prefix), scale=D ** -0.5)


def attention_oracle(c):
    """(exact values, sum p |v|, largest scale * sum |q k| per row) in 64 bits."""
    q, Hkv = c["q"].double(), c["k"].shape[1]
    G = q.shape[1] // Hkv
    out, absv, size = torch.zeros_like(q), torch.zeros_like(q), torch.zeros(q.shape[:2], dtype=torch.float64)
    at = 0
    for b, (n, P) in enumerate(zip(c["nodes"], c["prefix_list"])):
        slots = c["r2t"][int(c["rows"][b]), : P + n].long()
        for i in range(n):
            seen = [j for j in range(P)] + [P + j for j in range(n) if c["masks"][at + i] >> j & 1]
            if not seen:
                continue
            k, v = c["k"][slots[seen]].double(), c["v"][slots[seen]].double()  # [keys, Hkv, D]
            for h in range(q.shape[1]):
                w = torch.softmax(k[:, h // G] @ q[at + i, h] * c["scale"], 0)
                out[at + i, h] = w @ v[:, h // G]
                absv[at + i, h] = w @ v[:, h // G].abs()
                size[at + i, h] = (k[:, h // G].abs() @ q[at + i, h].abs()).max() * c["scale"]
        at += n
    return out, absv, size


def attention_tolerance(exact, absv, size):
    """Half a bf16 step (2^-8) of the result for its own rounding and of sum p |v| for the rounding of the probabilities; a score's error is
    that of 128 fp32 products and their sum, 2^-24 * 129 * size, and enters numerator and denominator; 2^-20 for the exponentials."""
    return 2.0 ** -8 * (exact.abs() + absv) * (1 + 2.0 ** -7) + absv * (2 * 129 * 2.0 ** -24 * size.unsqueeze(-1) + 2.0 ** -20)


def prepare_oracle(prefix, new, alloc, rows, free, free_range, table, page_size, capacity, parents=None, words=0, status=0):
    """Plain-Python msgl_prepare_extend on copies; parents packed request after request."""
    table = table.clone()
    bs, max_ctx = len(prefix), table.shape[1]
    head, end = free_range[0], min(free_range[1], len(free))
    bad = any(p < 0 or n < 0 or a < p or a > max_ctx or not 0 <= r < table.shape[0] for p, n, a, r in zip(prefix, new, alloc, rows))
    need = [max(0, -(-(p + n) // page_size) - -(-a // page_size)) for p, n, a in zip(prefix, new, alloc)]
    refuse = status or (3 if bad else 2 if any(p + n > max_ctx for p, n in zip(prefix, new)) else
                        4 if sum(new) > capacity or (words and any(n > 64 * words for n in new)) else 1 if sum(need) > end - head else 0)
    out = dict(positions=[0] * capacity, loc=[0] * capacity, cu=[0] * (bs + 1), seq_lens=list(prefix), alloc=list(alloc), free_range=list(free_range),
               status=refuse, table=table, pages={}, masks=[0] * capacity)
    if refuse:
        return out
    at, page = 0, head
    for b in range(bs):
        row, L, A = rows[b], prefix[b], alloc[b]
        par = parents[at: at + new[b]] if parents is not None else None
        masks = ancestor_masks(par) if par is not None else None
        for i in range(new[b]):
            pos = L + i
            if pos >= A:
                if pos % page_size:
                    slot = int(table[row, pos - 1]) + 1
                else:
                    slot = free[page] * page_size
                    out["pages"][row, pos // page_size] = free[page]
                    page += 1
                table[row, pos] = slot
            out["loc"][at + i] = int(table[row, pos])
            out["positions"][at + i] = L + (bin(masks[i]).count("1") - 1 if masks else i)
            if masks:
                out["masks"][at + i] = masks[i]
        at += new[b]
        out["cu"][b + 1] = at
        out["seq_lens"][b] = L + new[b]
        out["alloc"][b] = max(A, L + new[b])
    out["free_range"][0] = page
    return out


def accept_oracle(draft, target, parents, nodes, most):
    """Per request: (rows of the path, tokens along it)."""
    res, at = [], 0
    for n in nodes:
        par = [p if 0 <= p < j else 0 for j, p in enumerate(parents[at: at + n])]
        path = [0] if n else []
        while path and len(path) < most:
            cur = path[-1]
            kids = [j for j in range(cur + 1, n) if par[j] == cur and draft[at + j] == target[at + cur]]
            if not kids:
                break
            path.append(kids[0])
        res.append(([at + j for j in path], [target[at + j] for j in path]))
        at += n
    return res


def logprob_oracle(logits, tokens, top):
    """64-bit (logprobs, entropy, top ids, top logprobs, sum p |x - max|); NaN largest, ties to the lower index."""
    x = logits.double()
    d = x - x.amax(1, keepdim=True)
    lp = d - d.exp().sum(1, keepdim=True).log()   # (x - (max + ln Z) would lose ln Z beside a mask's -3e38)
    p = lp.exp()
    ent = -torch.where(p == 0, torch.zeros_like(p), p * lp).sum(1)
    ok = (tokens >= 0) & (tokens < x.shape[1])
    given = torch.where(ok, lp.gather(1, tokens.clamp(0, x.shape[1] - 1).long()[:, None])[:, 0], torch.full_like(lp[:, 0], float("nan")))
    rank = torch.where(torch.isnan(x), torch.full_like(x, float("inf")), x)
    order = torch.sort(rank + 0.0, dim=1, descending=True, stable=True).indices
    if bool(torch.isnan(x).any()):  # NaN before +inf
        order = torch.stack([torch.tensor(sorted(range(x.shape[1]), key=lambda j: (not bool(torch.isnan(r[j])), -float(r[j]) if not torch.isnan(r[j]) else 0, j)))
                             for r in x])
    ids = order[:, :top]
    spread = torch.where(p == 0, torch.zeros_like(p), p * d.abs()).sum(1)
    return given, ent, ids.to(torch.int32), lp.gather(1, ids), spread
