"""Cases, plain forms and exact values of the operators a step of speculative decoding with a drafted token tree adds to the
serving path: the batch's slots, positions and tree masks on the device (``prepare_extend``), attention of the tree's nodes
over the paged cache (``tree_attention``), log probabilities with entropy and top alternatives of the resulting logits
(``token_logprobs``), and the walk along the accepted nodes with the move of their cache rows (``accept_tree``).

With ``own`` false ``run`` computes each of them from elementary torch operations in 32 bits or more; with ``own`` true it
makes the calls a user of the package makes.
"""
import random

import torch

own = False

D = 128  # head dim of every model this package serves


def _ops():
    from mini_sglang_amd import ops

    return ops


# ------------------------------------------------------------------------------------------------------------- the cases
def _attention(name, bs, nodes, ctx, hq, hkv, page_size, ragged=True):
    return {"name": name, "op": "tree_attention", "bs": bs, "nodes": nodes, "ctx": ctx, "hq": hq, "hkv": hkv, "page_size": page_size,
            "ragged": ragged}


def _logprobs(name, rows, vocab, top, dtype):
    return {"name": name, "op": "token_logprobs", "rows": rows, "vocab": vocab, "top": top, "dtype": dtype}


def _prepare(name, bs, nodes, ctx, page_size, tree):
    return {"name": name, "op": "prepare_extend", "bs": bs, "nodes": nodes, "ctx": ctx, "page_size": page_size, "tree": tree}


def _accept(name, bs, nodes, layers, hkv, page_size):
    return {"name": name, "op": "accept_tree", "bs": bs, "nodes": nodes, "layers": layers, "hkv": hkv, "page_size": page_size}


def listed():
    return [
        # one chat request of the 0.6B model, a draft of four nodes: what counts is latency
        _attention("tree 1x4 ctx 500", 1, 4, 500, 16, 8, 1, False),
        # an ordinary serving batch of the 8B model, sixteen-node trees, contexts of unequal length
        _attention("tree 16x16 ctx 4000", 16, 16, 4000, 32, 8, 16),
        # a full batch with small trees: the pass over the cache is the work
        _attention("tree 64x8 ctx 8192", 64, 8, 8192, 32, 8, 16),
        # large trees over long contexts: as many products as a prefill
        _attention("tree 32x61 ctx 16000", 32, 61, 16000, 32, 8, 16),
        # one rank of eight of the 32B model, two long documents
        _attention("tree 2x32 ctx 130001 tp8", 2, 32, 130001, 8, 1, 64, False),
        # the sampled token's log probability and five alternatives, one request
        _logprobs("logprobs 1 row", 1, 151936, 5, "bfloat16"),
        # a decode batch, twenty alternatives (the most that chat interfaces ask for)
        _logprobs("logprobs 64 rows", 64, 151936, 20, "bfloat16"),
        # every node of a verified batch, in the precision a caller that post-processes its logits has them in
        _logprobs("logprobs 1000 rows fp32", 1000, 151936, 5, "float32"),
        # slots, positions and masks of a small step
        _prepare("prepare 4x8 nodes", 4, 8, 1000, 16, True),
        # slots and positions of a batch of prompts, hundreds of tokens each
        _prepare("prepare 200x900 prompt", 200, 900, 2000, 16, False),
        # acceptance in a small step of the 0.6B model: 28 layers
        _accept("accept 4x8 28 layers", 4, 8, 28, 8, 1),
        # a full batch of the 8B model: 36 layers
        _accept("accept 128x32 36 layers", 128, 32, 36, 8, 16),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["tree_attention", "tree_attention", "token_logprobs", "prepare_extend", "accept_tree"])
    if op == "tree_attention":
        hq, hkv = rng.choice([(16, 8), (32, 8), (64, 8), (8, 1), (4, 1), (16, 4), (8, 8), (2, 2), (16, 2)])
        bs, nodes, ctx = _log(rng, 1, 64), _log(rng, 1, 96), _log(rng, 1, 131072)
        # at most the cache bytes and the products of the largest listed cases
        while bs * (ctx + nodes) * hkv > 64 * 6000 * 8 or bs * (ctx + nodes) * nodes * hq > 32 * 12000 * 45 * 32:
            if ctx > 1024:
                ctx = ctx * 2 // 3
            else:
                bs = max(1, bs // 2)
        case = _attention("", bs, nodes, ctx, hq, hkv, rng.choice([1, 16, 64]), rng.random() < 0.7)
    elif op == "token_logprobs":
        vocab = _log(rng, 1000, 151936)
        rows = _log(rng, 1, 1000)
        case = _logprobs("", rows, vocab, rng.choice([0, 1, 5, 8, 20]), rng.choice(["bfloat16", "float32"]))
    elif op == "prepare_extend":
        tree = rng.random() < 0.6
        case = _prepare("", _log(rng, 1, 200), _log(rng, 1, 96 if tree else 900), _log(rng, 1, 4000), rng.choice([1, 16, 64]), tree)
    else:
        case = _accept("", _log(rng, 1, 128), _log(rng, 1, 32), rng.choice([4, 28, 36]), rng.choice([1, 2, 4, 8]), rng.choice([1, 16]))
    del case["name"]
    return case


def _shape_rng(case):
    """What the case itself fixes (lengths, trees, which drafts are right), the same for every seed."""
    return random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))


def _tree_parents(rng, n):
    """A drafter's tree in the order it grows: node 0 is the last accepted token, later nodes mostly hang off recent ones."""
    return [-1] + [max(0, j - 1 - int(rng.random() ** 2 * 6)) if rng.random() < 0.9 else rng.randrange(j) for j in range(1, n)]


def _attention_lens(case):
    rng = _shape_rng(case)
    bs, n, ctx = case["bs"], case["nodes"], case["ctx"]
    nodes = [rng.randint(max(1, n // 2), n) if case["ragged"] and b else n for b in range(bs)]
    prefix = [rng.randint(ctx // 2, ctx) if case["ragged"] and b else ctx for b in range(bs)]
    return rng, nodes, prefix


def _prepare_lens(case):
    rng = _shape_rng(case)
    bs, n, ctx, ps = case["bs"], case["nodes"], case["ctx"], case["page_size"]
    new = [rng.randint(max(1, n // 2), n) for _ in range(bs)]
    if case["tree"]:  # a step among others: earlier, partly rejected steps have left some slots with the request
        prefix = [rng.randint(max(1, ctx // 2), ctx) for _ in range(bs)]
        backed = [p + rng.choice([0, 0, 1, min(n, 5), n]) for p in prefix]
    else:  # prompts behind a page-aligned cached prefix
        prefix = [rng.randint(0, ctx) // ps * ps for _ in range(bs)]
        backed = list(prefix)
    return rng, new, prefix, backed


def _accept_shape(case):
    """Nodes, parents and, per node, the child that the model's token will confirm (-1 = none) with the accepted path."""
    rng = _shape_rng(case)
    bs, n = case["bs"], case["nodes"]
    nodes = [rng.randint(max(1, n // 2), n) for _ in range(bs)]
    parents = [_tree_parents(rng, m) for m in nodes]
    confirmed, paths = [], []
    for par in parents:
        child = []
        for i in range(len(par)):
            kids = [j for j in range(len(par)) if par[j] == i and j]
            child.append(rng.choice(kids) if kids and rng.random() < 0.75 else -1)
        path = [0]
        while child[path[-1]] >= 0:
            path.append(child[path[-1]])
        confirmed.append(child)
        paths.append(path)
    return nodes, parents, confirmed, paths


def _most_accepted(case):
    return min(case["nodes"], 16)


# ---------------------------------------------------------------------------------------------------------------- inputs
def _generator(seed, device="cuda"):
    return torch.Generator(device=device).manual_seed(int(seed) * 7919 + 17)


def _i32(values, device="cuda"):
    return torch.tensor(values, dtype=torch.int32, device=device)


def _table(lens, width, page_size, gen, spare_pages=0):
    """Random pages for `lens` positions per request: (table [bs, width], shuffled free pages, pages in all)."""
    need = [-(-length // page_size) for length in lens]
    total = sum(need) + spare_pages
    pages = torch.randperm(total, generator=gen, device="cuda").to(torch.int32) + 1  # page 0 is the dummy page
    table = torch.zeros((len(lens), width), dtype=torch.int32, device="cuda")
    at = 0
    for b, length in enumerate(lens):
        slots = (pages[at: at + need[b], None] * page_size + torch.arange(page_size, dtype=torch.int32, device="cuda")).view(-1)
        table[b, :length] = slots[:length]
        at += need[b]
    return table, pages[at:].contiguous(), total


def _masks(parents, words):
    """Bit j of a node's row: j is the node itself or one of its ancestors."""
    rows = []
    for par in parents:
        mine = []
        for j, p in enumerate(par):
            mine.append((mine[p] if j else 0) | (1 << j))
        rows += mine
    flat = [[(m >> (64 * w)) & (2 ** 64 - 1) for w in range(words)] for m in rows]
    return torch.tensor([[v - 2 ** 64 if v >= 2 ** 63 else v for v in r] for r in flat], dtype=torch.int64, device="cuda")


def _cu(lens):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return _i32(cu)


def _prepare_attention(case, seed):
    rng, nodes, prefix = _attention_lens(case)
    gen = _generator(seed)
    bs, hq, hkv, ps = case["bs"], case["hq"], case["hkv"], case["page_size"]
    lens = [p + n for p, n in zip(prefix, nodes)]
    width = -(-max(lens) // 64) * 64
    table, _, pages = _table(lens, width, ps, gen)
    order = torch.randperm(bs, generator=gen, device="cuda")
    r2t = torch.empty_like(table)
    r2t[order] = table
    slots = (pages + 1) * ps
    kv = torch.empty((slots, 2, hkv, D), dtype=torch.bfloat16, device="cuda").normal_(generator=gen)
    q = torch.empty((sum(nodes), hq, D), dtype=torch.bfloat16, device="cuda").normal_(std=1.5, generator=gen)
    words = -(-max(nodes) // 64)
    return {"op": "tree_attention", "q": q, "k": kv[:, 0], "v": kv[:, 1], "r2t": r2t, "rows": order.to(torch.int32), "cu": _cu(nodes),
            "prefix": _i32(prefix), "mask": _masks([_tree_parents(rng, n) for n in nodes], words), "scale": D ** -0.5,
            "max_q": max(nodes), "max_k": max(lens), "total_k": sum(lens)}


def _prepare_logprobs(case, seed):
    gen = _generator(seed)
    rows, vocab = case["rows"], case["vocab"]
    # a model's logits: a broad bulk and a few tokens far ahead of it
    x = torch.empty((rows, vocab), dtype=torch.float32, device="cuda").normal_(std=2.0, generator=gen)
    lead = (torch.randint(0, vocab, (rows, 1), generator=gen, device="cuda") + torch.arange(12, device="cuda") * (vocab // 12)) % vocab
    x.scatter_(1, lead, torch.empty((rows, 12), device="cuda").uniform_(4.0, 20.0, generator=gen))
    tokens = torch.where(torch.rand(rows, generator=gen, device="cuda") < 0.8, lead[:, 0],
                         torch.randint(0, vocab, (rows,), generator=gen, device="cuda")).to(torch.int32)
    return {"op": "token_logprobs", "logits": x.to(getattr(torch, case["dtype"])), "tokens": tokens, "top": case["top"]}


def _prepare_prepare(case, seed):
    rng, new, prefix, backed = _prepare_lens(case)
    gen = _generator(seed)
    bs, ps = case["bs"], case["page_size"]
    width = -(-(max(max(p + n, a) for p, n, a in zip(prefix, new, backed))) // 64) * 64
    need = [max(0, -(-(p + n) // ps) - -(-a // ps)) for p, n, a in zip(prefix, new, backed)]
    table, free, _ = _table(backed, width, ps, gen, spare_pages=sum(need) + 3)
    order = torch.randperm(bs, generator=gen, device="cuda")
    r2t = torch.empty_like(table)
    r2t[order] = table
    total, words = sum(new), -(-max(new) // 64)
    z = lambda *shape, dt=torch.int32: torch.zeros(shape, dtype=dt, device="cuda")  # noqa: E731
    return {"op": "prepare_extend", "rows": order.to(torch.int32), "prefix": _i32(prefix), "new": _i32(new), "backed": _i32(backed),
            "free": free, "free_range": _i32([0, free.numel()]), "r2t": r2t, "page_size": ps, "max_new": max(new), "total": total, "words": words,
            "parents": _i32([p for n in new for p in _tree_parents(rng, n)]) if case["tree"] else None,
            "out": {"positions": z(total), "loc": z(total), "cu": z(bs + 1), "seq_lens": z(bs), "backed": z(bs), "free_range": z(2),
                    "status": z(1), "mask": z(total, words, dt=torch.int64) if case["tree"] else None}}


def _prepare_accept(case, seed):
    nodes, parents, confirmed, _ = _accept_shape(case)
    gen = _generator(seed)
    bs, ps, total, n = case["bs"], case["page_size"], sum(nodes), case["nodes"]
    pages = bs * -(-(n + ps) // ps)
    rng = random.Random(seed)
    prefix = [rng.randint(1, 4000) for _ in range(bs)]
    table, _, _ = _table([n + ps] * bs, n + ps, ps, gen)
    loc = torch.cat([table[b, p % ps: p % ps + m] for b, (m, p) in enumerate(zip(nodes, prefix))])
    # every node drafts a token of its own; the model's token after a node is its confirmed child's, or one nobody drafted
    draft = rng.sample(range(100000), total)
    target, at = [], 0
    for child in confirmed:
        target += [draft[at + c] if c >= 0 else 100000 + rng.randrange(50000) for c in child]
        at += len(child)
    pool = torch.empty((case["layers"], (pages + 1) * ps, 2, case["hkv"], D), dtype=torch.bfloat16, device="cuda").normal_(generator=gen)
    most = _most_accepted(case)
    words = -(-max(nodes) // 64)
    z = lambda *shape: torch.zeros(shape, dtype=torch.int32, device="cuda")  # noqa: E731
    s = {"op": "accept_tree", "draft": _i32(draft), "target": _i32(target), "parents": _i32([p for par in parents for p in par]),
         "cu": _cu(nodes), "prefix": _i32(prefix), "loc": loc, "pool": pool, "most": most, "max_q": max(nodes), "mask": _masks(parents, words),
         "out": {"lens": z(bs), "rows": z(bs, most), "tokens": z(bs, most), "next": z(bs), "seq_lens": z(bs)}}
    if own:  # the caches' addresses in device memory, made once for a pool
        s["layers"] = _ops().kv_layers([x[:, 0] for x in pool], [x[:, 1] for x in pool])
    return s


def prepare(case, seed):
    return {"tree_attention": _prepare_attention, "token_logprobs": _prepare_logprobs, "prepare_extend": _prepare_prepare,
            "accept_tree": _prepare_accept}[case["op"]](case, seed)


# ------------------------------------------------------------------------------------------------------------ plain forms
def _plain_attention(s):
    cu, prefix = s["cu"].long(), s["prefix"].long()
    bs, n, length = prefix.numel(), s["max_q"], s["max_k"]
    hq, hkv = s["q"].shape[1], s["k"].shape[1]
    g = hq // hkv
    slots = s["r2t"][s["rows"].long(), :length].long()
    pos = torch.arange(length, device="cuda")
    count = cu[1:] - cu[:-1]
    slots = torch.where(pos < (prefix + count)[:, None], slots, 0)
    k = s["k"][slots].float().permute(0, 2, 3, 1).contiguous()  # [bs, hkv, D, length]
    v = s["v"][slots].float().transpose(1, 2).contiguous()      # [bs, hkv, length, D]
    node = torch.arange(n, device="cuda")
    row = (cu[:-1, None] + node).clamp(max=s["q"].shape[0] - 1)
    q = s["q"][row].float().view(bs, n, hkv, g, D).permute(0, 2, 1, 3, 4).reshape(bs, hkv, n * g, D)
    score = torch.matmul(q, k).mul_(s["scale"]).view(bs, hkv, n, g, length)
    rel = pos - prefix[:, None]                                  # [bs, length]: tree node of a position, < 0 in the prefix
    word = (rel.clamp(0, s["mask"].shape[1] * 64 - 1) >> 6)[:, None, :].expand(bs, n, length)
    bits = s["mask"][row].gather(2, word) >> (rel.clamp(min=0) & 63)[:, None, :] & 1
    seen = (rel < 0)[:, None, :] | ((bits == 1) & (rel < count[:, None])[:, None, :])
    score.masked_fill_(~seen[:, None, :, None, :], float("-inf"))
    top = score.amax(-1, keepdim=True)
    p = score.sub_(torch.where(torch.isinf(top), 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(bs, hkv, n * g, length), v).view(bs, hkv, n, g, D)
    o = torch.where(total > 0, o / total, 0.0).permute(0, 2, 1, 3, 4).reshape(bs, n, hq, D)
    return o[node < count[:, None]].to(torch.bfloat16)


def _plain_logprobs(s):
    x = s["logits"].float()
    top = x.amax(-1, keepdim=True)
    e = (x - top).exp()
    total = e.sum(-1, keepdim=True)
    lse = top + total.log()
    given = x.gather(1, s["tokens"].long()[:, None])[:, 0] - lse[:, 0]
    entropy = total.log()[:, 0] - (e * (x - top)).sum(-1) / total[:, 0]
    # order of the floats as whole numbers, ties to the lowest index: one key for both
    bits = (x + 0.0).view(torch.int32).long()
    key = torch.where(bits < 0, -1 - (bits & 0x7fffffff), bits)
    key = (key << 20) | (2 ** 20 - 1 - torch.arange(x.shape[1], device="cuda"))
    ids = 2 ** 20 - 1 - (key.topk(s["top"], dim=-1).values & (2 ** 20 - 1))
    return {"logprobs": given, "entropy": entropy, "top_ids": ids.to(torch.int32), "top_logprobs": x.gather(1, ids) - lse}


def _plain_prepare(s):
    prefix, new, backed, rows, ps = s["prefix"].long(), s["new"].long(), s["backed"].long(), s["rows"].long(), s["page_size"]
    bs, total = prefix.numel(), s["total"]
    seq = prefix + new
    have = (backed + ps - 1) // ps
    need = ((seq + ps - 1) // ps - have).clamp(min=0)
    taken = need.cumsum(0)
    ends = new.cumsum(0)
    cu = torch.cat([ends.new_zeros(1), ends])
    t = torch.arange(total, device="cuda")
    b = torch.searchsorted(ends, t, right=True)
    i = t - cu[b]
    p = prefix[b] + i
    page = (s["free_range"][0].long() + (taken - need)[b] + p // ps - have[b]).clamp(0, s["free"].numel() - 1)
    fresh = s["free"][page].long() * ps + p % ps
    last = s["r2t"][rows, (backed - 1).clamp(min=0)].long()
    run = last[b] + p - backed[b] + 1
    slot = torch.where(p < backed[b], s["r2t"][rows[b], p].long(), torch.where(p < have[b] * ps, run, fresh)).to(torch.int32)
    s["r2t"][rows[b], p] = slot
    depth, mask = i, None
    if s["parents"] is not None:
        n, words = s["max_new"], s["words"]
        node = torch.arange(n, device="cuda")
        par = s["parents"].long()[(cu[:-1, None] + node).clamp(max=total - 1)]
        a = (par[:, :, None] == node).float() * (node > 0)[:, None] + torch.eye(n, device="cuda")
        a = torch.matmul(a, a).clamp_(max=1)
        a = torch.matmul(a, a).clamp_(max=1)
        a = torch.matmul(a, a).clamp_(max=1)
        a = torch.matmul(a, a).clamp_(max=1)
        a = torch.matmul(a, a).clamp_(max=1)
        a = torch.matmul(a, a).clamp_(max=1)
        a = torch.matmul(a, a).clamp_(max=1)  # paths of up to 127 steps
        depth = (a.sum(-1).long() - 1)[b, i]
        a = torch.nn.functional.pad(a.long(), (0, words * 64 - n)).view(bs, n, words, 64)
        mask = (a << torch.arange(64, device="cuda")).sum(-1)[b, i]
    return {"positions": (prefix[b] + depth).to(torch.int32), "loc": slot, "cu": cu.to(torch.int32), "seq_lens": seq.to(torch.int32),
            "backed": torch.maximum(backed, seq).to(torch.int32), "free_range": s["free_range"] + torch.stack([taken[-1], taken[-1] * 0]).to(torch.int32),
            "status": torch.zeros_like(s["out"]["status"]), "mask": mask, "r2t": s["r2t"]}


def _plain_accept(s):
    cu = s["cu"].long()
    n, most, count = s["max_q"], s["most"], cu[1:] - cu[:-1]
    node = torch.arange(n, device="cuda")
    row = (cu[:-1, None] + node).clamp(max=s["draft"].numel() - 1)
    real = node < count[:, None]
    draft, target, par = s["draft"][row], s["target"][row], s["parents"][row].long()
    hit = real & (node > 0) & (draft == target.gather(1, par.clamp(min=0)))
    sibling = (par[:, :, None] == par[:, None, :]) & (node[None, :] < node[:, None])
    hit = (hit & ~(sibling & hit[:, None, :]).any(-1)) | (node == 0)
    above = s["mask"][row].gather(2, (node >> 6).expand(row.shape[0], n, n)) >> (node & 63) & 1 == 1
    on = real & ~(above & ~hit[:, None, :]).any(-1)
    lens = on.sum(-1).clamp(max=most)
    path = torch.where(on, node, n).sort(-1).values
    path = torch.nn.functional.pad(path, (0, max(0, most - n)))[:, :most]
    step = torch.arange(most, device="cuda")
    live = step < lens[:, None]
    path = torch.where(live, path, 0)
    rows = cu[:-1, None] + path
    tokens = torch.where(live, s["target"][rows], -1)
    nxt = tokens.gather(1, (lens - 1)[:, None])[:, 0]
    src = s["loc"][rows].long()
    dst = s["loc"][torch.where(live, cu[:-1, None] + step, cu[:-1, None])].long()
    s["pool"][:, dst] = s["pool"][:, src]
    return {"lens": lens.to(torch.int32), "rows": torch.where(live, rows, -1).to(torch.int32), "tokens": tokens, "next": nxt,
            "seq_lens": s["prefix"] + lens.to(torch.int32), "pool": list(s["pool"])}


# --------------------------------------------------------------------------------------------------------------- the calls
def _own_attention(s):
    return _ops().tree_attention(s["q"], s["k"], s["v"], s["r2t"], s["rows"], s["cu"], s["prefix"], s["mask"], s["max_q"], s["max_k"],
                                 s["scale"], total_kv=s["total_k"])


def _own_logprobs(s):
    given, entropy, ids, top = _ops().token_logprobs(s["logits"], s["tokens"], s["top"])
    return {"logprobs": given, "entropy": entropy, "top_ids": ids, "top_logprobs": top}


def _own_prepare(s):
    o = s["out"]
    _ops().prepare_extend(s["rows"], s["prefix"], s["new"], s["backed"], s["free"], s["free_range"], s["r2t"], o["positions"], o["loc"],
                          o["cu"], o["seq_lens"], o["status"], s["page_size"], parents=s["parents"], tree_mask=o["mask"],
                          alloc_out=o["backed"], free_range_out=o["free_range"])
    return dict(o, r2t=s["r2t"])


def _own_accept(s):
    o = s["out"]
    _ops().accept_tree(s["draft"], s["target"], s["parents"], s["cu"], s["prefix"], s["loc"], s["layers"], o["lens"], o["rows"], o["tokens"],
                       o["next"], o["seq_lens"])
    return dict(o, pool=list(s["pool"]))


def run(state):
    if own:
        return {"tree_attention": _own_attention, "token_logprobs": _own_logprobs, "prepare_extend": _own_prepare,
                "accept_tree": _own_accept}[state["op"]](state)
    return {"tree_attention": _plain_attention, "token_logprobs": _plain_logprobs, "prepare_extend": _plain_prepare,
            "accept_tree": _plain_accept}[state["op"]](state)


# ------------------------------------------------------------------------------------------------------------------- work
def work(case):
    if case["op"] == "tree_attention":
        _, nodes, prefix = _attention_lens(case)
        keys = sum(p + n for p, n in zip(prefix, nodes))
        words = -(-max(nodes) // 64)
        return {"bytes": keys * (case["hkv"] * 2 * D * 2 + 4) + sum(nodes) * (2 * case["hq"] * D * 2 + 8 * words) + 12 * case["bs"],
                "flops": sum(4 * case["hq"] * D * n * (p + n) for p, n in zip(prefix, nodes))}
    if case["op"] == "token_logprobs":
        size = 2 if case["dtype"] == "bfloat16" else 4
        n = case["rows"] * case["vocab"]
        return {"bytes": n * size + case["rows"] * (12 + 8 * case["top"]), "flops": 6 * n}
    if case["op"] == "prepare_extend":
        _, new, _, _ = _prepare_lens(case)
        words = -(-max(new) // 64)
        return {"bytes": sum(new) * (12 + (4 + 8 * words if case["tree"] else 0)) + case["bs"] * 24, "flops": sum(new)}
    nodes, _, _, paths = _accept_shape(case)
    most = _most_accepted(case)
    moved = sum(sum(1 for i, j in enumerate(p[:most]) if i != j) for p in paths)
    return {"bytes": sum(nodes) * 12 + case["bs"] * (16 + 8 * most) + moved * case["layers"] * case["hkv"] * 2 * D * 2 * 2, "flops": sum(nodes)}


# ------------------------------------------------------------------------------------------------------------ exact values
def exact(case, seed):
    if case["op"] == "prepare_extend":
        return None  # whole numbers throughout
    s = prepare(case, seed)
    if case["op"] == "tree_attention":
        _, nodes, prefix = _attention_lens(case)
        g, at, out = case["hq"] // case["hkv"], 0, []
        for b, (n, p) in enumerate(zip(nodes, prefix)):
            slots = s["r2t"][int(s["rows"][b])][: p + n].long()
            mask = [[m & (2 ** 64 - 1) for m in row] for row in s["mask"][at: at + n].tolist()]
            tree = torch.tensor([[row[j // 64] >> (j % 64) & 1 for j in range(n)] for row in mask], dtype=torch.float64, device="cuda")
            heads = []
            for h in range(case["hkv"]):
                k, v = s["k"][slots, h].double(), s["v"][slots, h].double()
                q = s["q"][at: at + n, h * g: h * g + g].double()
                w = torch.tensordot(q, k, dims=([2], [1])) * s["scale"]
                w[:, :, p:] += torch.log(tree)[:, None, :]
                heads.append(torch.tensordot(torch.softmax(w, dim=2), v, dims=([2], [0])))
            out.append(torch.cat(heads, dim=1))
            at += n
        return torch.cat(out)
    if case["op"] == "token_logprobs":
        logp, entropy = [], []
        for part in s["logits"].split(128):
            w = torch.log_softmax(part.double(), dim=1)
            order = torch.sort(w, dim=1, descending=True).values[:, : s["top"]]
            logp.append((w, order))
            entropy.append(-(w.exp() * w).sum(1))
        rows = torch.arange(case["rows"], device="cuda")
        given = torch.cat([w[torch.arange(w.shape[0], device="cuda"), s["tokens"][at: at + w.shape[0]].long()]
                           for (w, _), at in zip(logp, rows[::128].tolist())])
        return {"logprobs": given, "entropy": torch.cat(entropy), "top_ids": None, "top_logprobs": torch.cat([o for _, o in logp])}
    nodes, _, _, paths = _accept_shape(case)
    src, dst, at = [], [], 0
    for n, path in zip(nodes, paths):
        for i, j in enumerate(path[: s["most"]]):
            src.append(at + j)
            dst.append(at + i)
        at += n
    loc = s["loc"].long()
    pool = []
    for layer in s["pool"]:
        x = layer.double()
        x[loc[dst]] = layer.double()[loc[src]]
        pool.append(x)
    return {"lens": None, "rows": None, "tokens": None, "next": None, "seq_lens": None, "pool": pool}
