"""Speculative-decoding operators on the GPU against 64-bit oracles: slot maps and tree masks built on the device, attention of drafted
trees over the paged cache, acceptance with the move of cache rows, and token log probabilities."""
import random

import pytest
import torch

import tree_cases as tc

pytestmark = pytest.mark.gpu
DEV = "cuda"
D = 128


def _ops():
    from mini_sglang_amd import ops
    return ops


def _gpu(c):
    return {k: v.to(DEV) if isinstance(v, torch.Tensor) else v for k, v in c.items()}


def _views(c):
    """GPU copy that keeps an interleaved pool's views."""
    d = _gpu({k: v for k, v in c.items() if k not in ("k", "v")})
    if c["k"].stride(0) != c["k"].shape[1] * D:
        kv = torch.stack([c["k"], c["v"]], 1).to(DEV)
        d["k"], d["v"] = kv[:, 0], kv[:, 1]
    else:
        d["k"], d["v"] = c["k"].to(DEV), c["v"].to(DEV)
    return d


def _attend(d, **kw):
    lens = [n + p for n, p in zip(d["nodes"], d["prefix_list"])]
    args = dict(max_q=max(d["nodes"]), max_k=max(lens))
    args.update({k: kw.pop(k) for k in ("max_q", "max_k") if k in kw})
    return _ops().tree_attention(d["q"], d["k"], d["v"], d["r2t"], d["rows"], d["cu"], d["prefix"], d["mask"], args["max_q"], args["max_k"], d["scale"], **kw)


def _check(out, c):
    exact, absv, size = tc.attention_oracle(c)
    err = (out.cpu().double() - exact).abs()
    tol = tc.attention_tolerance(exact, absv, size)
    assert bool((err <= tol).all()), f"largest error {err.max():.3e}, over its tolerance by a factor {(err / tol.clamp_min(1e-30)).max():.2f}"


# ---------------------------------------------------------------------------------------------------------- attention
@pytest.mark.parametrize("Hq,Hkv", [(16, 8), (32, 8), (8, 1), (8, 8), (4, 2), (16, 2), (4, 4)])
@pytest.mark.parametrize("page_size,layout", [(1, "split"), (16, "interleaved"), (5, "interleaved")])
def test_tree_attention_heads_and_pages(Hq, Hkv, page_size, layout):
    c = tc.attention_case([3, 9, 1, 7], [40, 0, 133, 31], Hq, Hkv, page_size, 100 * Hq + Hkv + page_size, layout)
    _check(_attend(_views(c)), c)


@pytest.mark.parametrize("nodes,prefix", [([1], [0]), ([1], [1]), ([1], [700]), ([2], [0]), ([31], [32]), ([32], [31]), ([33], [33]), ([64], [63]),
                                          ([65], [64]), ([130], [500]), ([17, 1, 64, 40], [0, 1, 300, 95]), ([5] * 40, list(range(0, 80, 2)))])
def test_tree_attention_lengths(nodes, prefix):
    c = tc.attention_case(nodes, prefix, 8, 2, 16, 7 + sum(nodes))
    _check(_attend(_views(c)), c)


@pytest.mark.parametrize("Hq,Hkv,nodes", [(8, 1, 40), (4, 1, 61), (16, 8, 16), (2, 2, 3)])
def test_tree_attention_long_context_in_runs(Hq, Hkv, nodes):
    c = tc.attention_case([nodes, 2], [5003, 1700], Hq, Hkv, 64, 31 + nodes)
    d = _views(c)
    ops = _ops()
    assert ops.tree_attention_splits(2, nodes, 5003 + nodes, Hq, Hkv) > 1
    cut = _attend(d)
    _check(cut, c)
    assert torch.equal(cut, _attend(d)), "one cut always gives the same bits"
    _check(_attend(d, total_kv=5003 + 1702 + nodes), c)
    _check(_attend(d, max_k=37), c)           # a bound that is too small only leaves the last run longer
    _check(_attend(d, max_k=1 << 20), c)
    # less workspace than the cut asks for: fewer runs
    T = d["q"].shape[0]
    for runs in (0, 2, 3):
        ws = torch.full((max(16, ops.tree_attention_workspace_bytes(T, Hq, D, runs)),), 255, dtype=torch.uint8, device=DEV)
        _check(_attend(d, workspace=ws), c)


def test_tree_attention_rows_that_see_nothing_and_wide_masks():
    c = tc.attention_case([6, 4, 70], [0, 20, 0], 8, 2, 16, 5, words=3)
    for t, m in ((0, 0), (3, 0b100000), (6, 0), (9, 0b0110), (12, 0), (15, 1 << 69 | 1)):
        c["masks"][t] = m
    c["mask"] = tc.pack_masks([m | (1 << 150) for m in c["masks"]], 3)  # a bit behind the request's nodes means nothing
    out = _attend(_views(c))
    _check(out, c)
    assert bool((out[0] == 0).all()) and bool((out[12 - 2] != 0).any())


def test_tree_attention_unseen_nodes_never_reach_a_row():
    for what in (float("nan"), float("inf"), -float("inf")):
        for nodes, prefix in (([9, 40], [70, 3]), ([33], [0])):
            c = tc.attention_case(nodes, prefix, 8, 2, 16, 77 + len(nodes))
            at = 0
            k, v = c["k"].clone(), c["v"].clone()
            hidden = []
            for b, (n, P) in enumerate(zip(nodes, prefix)):
                for j in (n - 1, n // 2):   # this node's rows are poisoned; who sees it is left out of the comparison
                    slot = int(c["r2t"][int(c["rows"][b]), P + j])
                    k[slot, :, 5] = what
                    v[slot, :, 3:90:7] = what
                    hidden += [at + i for i in range(n) if c["masks"][at + i] >> j & 1]
                at += n
            clean = _attend(_views(c))
            d = _views(c)
            kv = torch.stack([k, v], 1).to(DEV)
            d["k"], d["v"] = kv[:, 0], kv[:, 1]
            out = _attend(d)
            keep = [i for i in range(sum(nodes)) if i not in hidden]
            assert keep and hidden
            assert not bool(torch.isfinite(out[hidden]).all())
            exact, absv, size = tc.attention_oracle(c)
            err = (out[keep].cpu().double() - exact[keep]).abs()
            assert bool((err <= tc.attention_tolerance(exact, absv, size)[keep]).all())
            assert bool(torch.isfinite(clean).all())


def test_tree_attention_strided_query_output_and_rows_behind_the_last():
    c = tc.attention_case([5, 12], [60, 9], 8, 2, 16, 12)
    d = _views(c)
    T = 17
    wide = torch.randn(T + 4, 12 * D, device=DEV).to(torch.bfloat16)
    wide[:T, 2 * D: 10 * D] = d["q"].view(T, -1)
    d["q"] = wide[:, 2 * D: 10 * D].unflatten(1, (8, D))
    d["mask"] = torch.cat([d["mask"], torch.full((4, 1), -1, dtype=torch.int64, device=DEV)])
    big = torch.full((T + 4, 9 * D), 7.0, dtype=torch.bfloat16, device=DEV)
    out = _attend(d, out=big[:, D:].unflatten(1, (8, D)))
    _check(out[:T], c)
    assert bool((big[:, :D] == 7).all()) and bool((big[T:] == 7).all())


def test_tree_attention_slots_beyond_32_bit_offsets():
    c = tc.attention_case([4, 9], [50, 200], 8, 8, 16, 3)
    d = _views(c)
    far = 1_200_000  # slots of 4 KiB: offsets up to 4.9 GB
    kv = torch.empty((far + c["k"].shape[0], 2, 8, D), dtype=torch.bfloat16, device=DEV)
    kv[far:, 0], kv[far:, 1] = d["k"], d["v"]
    d["k"], d["v"] = kv[:, 0], kv[:, 1]
    d["r2t"] = d["r2t"] + far
    _check(_attend(d), c)


def test_tree_attention_agrees_with_decode_and_extend():
    ops = _ops()
    c = tc.attention_case([1] * 5, [0, 15, 16, 400, 77], 16, 8, 16, 40)
    d = _views(c)
    seq = d["prefix"] + 1
    dec = ops.paged_decode(d["q"], d["k"], d["v"], d["r2t"], d["rows"], seq, d["scale"], 16)
    exact, absv, size = tc.attention_oracle(c)
    tol = tc.attention_tolerance(exact, absv, size)
    assert bool(((_attend(d).cpu().double() - dec.cpu().double()).abs() <= 2 * tol).all())
    c = tc.attention_case([30, 9], [100, 16], 16, 8, 16, 41, chain=True)
    d = _views(c)
    ext = ops.paged_extend(d["q"], d["k"], d["v"], d["r2t"], d["rows"], d["cu"], d["prefix"], 30, d["scale"], 16)
    exact, absv, size = tc.attention_oracle(c)
    tol = tc.attention_tolerance(exact, absv, size)
    assert bool(((_attend(d).cpu().double() - ext.cpu().double()).abs() <= 2 * tol).all())


def test_tree_attention_captured_and_on_another_stream():
    first = tc.attention_case([5, 12, 3], [600, 9, 2000], 8, 2, 16, 21)
    second = tc.attention_case([12, 3, 5], [1200, 1700, 4], 8, 2, 16, 22)
    slots = max(first["k"].shape[0], second["k"].shape[0])
    width = max(first["r2t"].shape[1], second["r2t"].shape[1])
    st = {"q": torch.zeros(20, 8, D, dtype=torch.bfloat16, device=DEV), "kv": torch.zeros(slots, 2, 2, D, dtype=torch.bfloat16, device=DEV),
          "r2t": torch.zeros(3, width, dtype=torch.int32, device=DEV), "rows": torch.zeros(3, dtype=torch.int32, device=DEV),
          "cu": torch.zeros(4, dtype=torch.int32, device=DEV), "prefix": torch.zeros(3, dtype=torch.int32, device=DEV),
          "mask": torch.zeros(20, 1, dtype=torch.int64, device=DEV)}
    out = torch.zeros(20, 8, D, dtype=torch.bfloat16, device=DEV)
    ops = _ops()
    ws = torch.empty(ops.tree_attention_workspace_bytes(20, 8, D, ops.tree_attention_splits(3, 12, 2048, 8, 2)), dtype=torch.uint8, device=DEV)

    def load(c):
        st["q"].copy_(c["q"]), st["rows"].copy_(c["rows"]), st["cu"].copy_(c["cu"]), st["prefix"].copy_(c["prefix"]), st["mask"].copy_(c["mask"])
        st["kv"].zero_(), st["r2t"].zero_()
        st["kv"][: c["k"].shape[0], 0], st["kv"][: c["k"].shape[0], 1] = c["k"].to(DEV), c["v"].to(DEV)
        st["r2t"][:, : c["r2t"].shape[1]] = c["r2t"].to(DEV)

    def step():
        ops.tree_attention(st["q"], st["kv"][:, 0], st["kv"][:, 1], st["r2t"], st["rows"], st["cu"], st["prefix"], st["mask"], 12, 2048, D ** -0.5,
                           out=out, workspace=ws)

    load(first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    _check(out, first)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.inference_mode(), torch.cuda.graph(graph):
        step()
    for c in (second, first, second):
        load(c)
        out.fill_(9)
        graph.replay()
        got = out.clone()
        step()
        torch.cuda.synchronize()
        assert torch.equal(got, out)
        _check(got, c)


# ---------------------------------------------------------------------------------------------------------- slot maps
def _prepare(prefix, new, alloc, page_size, seed, capacity=None, tree=True, words=None, rows=None, spare=2, cut=0, in_place=False, pages=True,
             status=0, width=None, offset=1):
    """Runs prepare_extend and the oracle on the same state and compares everything."""
    ops = _ops()
    rng = random.Random(seed)
    bs = len(prefix)
    need = sum(max(0, -(-(p + n) // page_size) - -(-a // page_size)) for p, n, a in zip(prefix, new, alloc) if n >= 0)
    width = width or max([64] + [p + max(n, 0) + 3 for p, n in zip(prefix, new)] + [a + 3 for a in alloc])
    table, free, _ = tc.page_rows([max(a, 0) for a in alloc], width, page_size, rng, spare=max(0, need + spare - cut))
    order = rows if rows is not None else rng.sample(range(bs + 3), bs)
    r2t = torch.zeros((bs + 3, width), dtype=torch.int32)
    for b, r in enumerate(order):
        if 0 <= r < bs + 3:
            r2t[r] = table[b]
    free = [9] * offset + free
    free_range = [offset, len(free)]
    capacity = sum(max(n, 0) for n in new) if capacity is None else capacity
    parents = [p for n in new for p in tc.tree_parents(rng, max(n, 0))[: max(n, 0)]] if tree else None
    words = words or max([1] + [-(-n // 64) for n in new])
    want = tc.prepare_oracle(prefix, new, alloc, order, free, free_range, r2t, page_size, capacity, parents, words if tree else 0, status)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    filled = (parents + [-1] * capacity)[:capacity] if tree else None
    got = dict(positions=i32([77] * capacity), loc=i32([77] * capacity), cu=i32([77] * (bs + 1)), seq_lens=i32([77] * bs))
    st, alloc_t, fr, tab = i32([status]), i32(alloc), i32(free_range), r2t.to(DEV)
    page_tab = torch.zeros((bs + 3, -(-width // page_size)), dtype=torch.int32, device=DEV) if pages else None
    mask = torch.full((capacity, words), 77, dtype=torch.int64, device=DEV) if tree else None
    extra = {} if in_place else dict(alloc_out=i32([77] * bs), free_range_out=i32([77, 77]))
    ops.prepare_extend(i32(order), i32(prefix), i32(new), alloc_t, i32(free), fr, tab, got["positions"], got["loc"], got["cu"], got["seq_lens"], st,
                       page_size, parents=i32(filled) if tree else None, tree_mask=mask, req_to_page=page_tab, **extra)
    for name in ("positions", "loc", "cu", "seq_lens"):
        assert got[name].tolist() == want[name], name
    assert (alloc_t if in_place else extra["alloc_out"]).tolist() == want["alloc"]
    assert (fr if in_place else extra["free_range_out"]).tolist() == want["free_range"]
    if not in_place:
        assert alloc_t.tolist() == alloc and fr.tolist() == free_range
    assert int(st) == want["status"]
    assert torch.equal(tab.cpu(), want["table"])
    if tree:
        assert torch.equal(mask.cpu(), tc.pack_masks(want["masks"], words))
    if pages:
        ref = torch.zeros_like(page_tab, device="cpu")
        if page_size > 1:
            for (r, i), page in want["pages"].items():
                ref[r, i] = page
        assert torch.equal(page_tab.cpu(), ref)
    return want["status"]


@pytest.mark.parametrize("page_size", [1, 3, 16, 64])
@pytest.mark.parametrize("tree", [True, False])
def test_prepare_extend_lengths_pages_and_backed_positions(page_size, tree):
    prefix = [0, 1, 15, 16, 17, 40, 100, 63, 5]
    new = [1, 16, 1, 33, 0, 70, 7, 2, 64]
    alloc = [0, 1, 16, 20, 17, 200, 103, 64, 30]
    assert _prepare(prefix, new, alloc, page_size, 3 + page_size, tree=tree) == 0
    assert _prepare(prefix, new, alloc, page_size, 4 + page_size, tree=tree, in_place=True, capacity=sum(new) + 37, pages=False) == 0


@pytest.mark.parametrize("bs,most,tree", [(1, 1, True), (1, 1024, True), (1030, 3, True), (2100, 5, False), (300, 90, False), (70, 130, True)])
def test_prepare_extend_sizes(bs, most, tree):
    rng = random.Random(bs)
    prefix = [rng.randint(0, 50) for _ in range(bs)]
    new = [rng.randint(0, most) for _ in range(bs)]
    new[-1] = most
    alloc = [p + rng.choice([0, 0, 2, 20]) for p in prefix]
    assert _prepare(prefix, new, alloc, 16, bs, tree=tree) == 0


def test_prepare_extend_odd_parents_and_idle_steps():
    ops = _ops()
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    parents = [5, -7, 1, 3, 2, 99] + [-1]   # anything but an earlier node is the root
    mask = torch.zeros((7, 1), dtype=torch.int64, device=DEV)
    pos, loc, cu, seq, st = i32([0] * 7), i32([0] * 7), i32([0] * 3), i32([0] * 2), i32([0])
    table = torch.zeros((2, 64), dtype=torch.int32, device=DEV)
    ops.prepare_extend(i32([0, 1]), i32([0, 0]), i32([6, 1]), i32([0, 0]), i32(list(range(1, 40))), i32([0, 39]), table, pos, loc, cu, seq, st, 16,
                       parents=i32(parents), tree_mask=mask)
    assert mask[:, 0].tolist() == [0b1, 0b11, 0b111, 0b1001, 0b10111, 0b100001, 1] and pos.tolist() == [0, 1, 2, 1, 3, 1, 0]
    assert _prepare([4, 9], [0, 0], [4, 9], 16, 2, tree=True, capacity=5) == 0
    assert _prepare([4, 9], [0, 0], [4, 9], 16, 2, tree=False, capacity=0) == 0


@pytest.mark.parametrize("tree", [True, False])
def test_prepare_extend_refusals_leave_everything_as_it_was(tree):
    ok = dict(prefix=[10, 20], new=[5, 40], alloc=[10, 25], page_size=16, seed=9, tree=tree)
    assert _prepare(**ok) == 0
    assert _prepare(**ok, cut=3, in_place=True) == 1
    assert _prepare(**ok, cut=2) == 0          # exactly enough pages
    assert _prepare(**ok, capacity=44) == 4
    assert _prepare(**ok, width=59) == 2
    assert _prepare(**dict(ok, new=[5, -1])) == 3
    assert _prepare(**dict(ok, alloc=[9, 25])) == 3
    assert _prepare(**ok, rows=[1, 5]) == 3 and _prepare(**ok, rows=[-1, 0]) == 3
    assert _prepare(**ok, status=1) == 1 and _prepare(**ok, status=7, in_place=True) == 7
    if tree:
        assert _prepare(**dict(ok, new=[5, 65]), words=1) == 4


def test_prepare_extend_chain_matches_the_host_producer():
    """The same slots, positions and table as the host-side batch producer for prompts behind page-aligned prefixes."""
    from mini_sglang_amd.mem_cache import PageAllocator, ReqToTokenPool
    from mini_sglang_amd.runtime.batch_info import BatchInfo, Req

    ops = _ops()
    for ps in (1, 16):
        pool = ReqToTokenPool(8, 512, ps, DEV)
        alloc = PageAllocator(400, ps)
        held = alloc.alloc(6 if ps > 1 else 96)
        free = alloc.free_page.clone()
        reqs = [Req(i, list(range(n))) for i, n in enumerate((37, 200, 48, 5))]
        slots = (held[:, None].int() * ps + torch.arange(ps, dtype=torch.int32)).view(-1)
        reqs[0].prefix_indices, reqs[1].prefix_indices = slots[:32], slots[32:96]
        batch = BatchInfo.init_new(reqs, pool, alloc, None)
        batch.prepare_for_extend()
        table = torch.zeros_like(pool.req_to_token)
        for r in reqs:
            table[r.req_pool_idx, : r.prefix_indices.numel()] = r.prefix_indices.to(DEV)
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
        new = [r.num_tokens - r.prefix_indices.numel() for r in reqs]
        pos, loc, cu, seq, st = i32([0] * sum(new)), i32([0] * sum(new)), i32([0] * 5), i32([0] * 4), i32([0])
        fr = i32([0, free.numel()])
        ops.prepare_extend(batch.req_pool_indices, batch.prefix_seq_lens, i32(new), batch.prefix_seq_lens.clone(), free.to(DEV), fr, table, pos, loc, cu,
                           seq, st, ps)
        assert torch.equal(pos, batch.positions) and torch.equal(loc, batch.out_cache_loc) and torch.equal(seq, batch.seq_lens)
        assert torch.equal(table, pool.req_to_token) and int(fr[0]) == free.numel() - alloc.free_count()


# ---------------------------------------------------------------------------------------------------------- acceptance
def _accept(nodes, seed, most, layers=3, Hkv=2, layout="interleaved", vocab=6, chain=False, parents=None, alias=False):
    ops = _ops()
    rng = random.Random(seed)
    T, bs = sum(nodes), len(nodes)
    parents = parents or [p for n in nodes for p in tc.tree_parents(rng, n, chain)[:n]]
    draft = [rng.randrange(vocab) for _ in range(T)]      # few tokens: siblings often draft the same one
    target = [rng.randrange(vocab) for _ in range(T)]
    prefix = [rng.randint(0, 99) for _ in nodes]
    slots = rng.sample(range(1, T + 20), T)
    pool = [torch.randn(T + 20, 2, Hkv, D, generator=torch.Generator().manual_seed(seed + l)).to(torch.bfloat16) for l in range(layers)]
    dev = [x.to(DEV) for x in pool]
    if layout == "split":
        ks, vs = [x[:, 0].contiguous() for x in dev], [x[:, 1].contiguous() for x in dev]
    else:
        ks, vs = [x[:, 0] for x in dev], [x[:, 1] for x in dev]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    pre = i32(prefix)
    seq = pre if alias else i32([77] * bs)
    out = dict(lens=i32([77] * bs), rows=torch.full((bs, most), 77, dtype=torch.int32, device=DEV), tokens=torch.full((bs, most), 77, dtype=torch.int32, device=DEV),
               next=i32([77] * bs))
    ops.accept_tree(i32(draft), i32(target), i32(parents), tc.cumulative(nodes).to(DEV), pre, i32(slots), ops.kv_layers(ks, vs) if layers else None, out["lens"],
                    out["rows"], out["tokens"], out["next"], seq)
    want = tc.accept_oracle(draft, target, parents, nodes, most)
    cu = tc.cumulative(nodes).tolist()
    for b, (path, tokens) in enumerate(want):
        assert int(out["lens"][b]) == len(path) and int(seq[b]) == prefix[b] + len(path)
        assert out["rows"][b].tolist() == path + [-1] * (most - len(path))
        assert out["tokens"][b].tolist() == tokens + [-1] * (most - len(path))
        assert int(out["next"][b]) == (tokens[-1] if path else 77)
        for x in pool:
            src = x[[slots[t] for t in path]].clone()
            for i in range(len(path)):
                x[slots[cu[b] + i]] = src[i]
    for x, k, v in zip(pool, ks, vs):
        assert torch.equal(k.cpu(), x[:, 0]) and torch.equal(v.cpu(), x[:, 1])
    return [len(p) for p, _ in want]


@pytest.mark.parametrize("nodes", [[1], [2], [7, 1, 30], [64, 63, 65], [200, 3], [5] * 300, [0, 4, 0]])
def test_accept_tree_paths_and_rows(nodes):
    deep = 0
    for seed in range(3):
        deep = max([deep] + _accept(nodes, 50 + seed, 16, vocab=2))
        _accept(nodes, 80 + seed, 3, layout="split", Hkv=1, alias=True)
    assert deep > (1 if sum(nodes) > 4 else 0)   # (of the oracle too: some path leaves its root)


def test_accept_tree_long_chains_caps_and_many_layers():
    assert max(_accept([200, 90], 1, 1024, vocab=1, chain=True)) == 200
    assert _accept([200, 90], 2, 7, vocab=1, chain=True) == [7, 7]
    assert _accept([40, 9, 12], 3, 16, layers=70, Hkv=8, vocab=2)
    assert _accept([40, 9, 12], 4, 16, layers=0, vocab=2)
    assert _accept([9], 5, 16, parents=[3, -1, -5, 99, 1, 2, 2, 2, 2], vocab=1) == [9 - 6]


# ---------------------------------------------------------------------------------------------------------- log probabilities
def _logprobs(logits, tokens, top, host=None, **kw):
    ops = _ops()
    got = ops.token_logprobs(logits, torch.tensor(tokens, dtype=torch.int32, device=DEV), top, **kw)
    x = logits.float().cpu() if host is None else host
    given, ent, ids, lps, spread = tc.logprob_oracle(x, torch.tensor(tokens), top)
    # ln Z: every exponential is off by its argument's rounding (|x - m| 2^-23) and two units of its own, and 64 terms a thread, six wave
    # steps, four waves and the segments are added in turn; the entropy's sum carries the same, times |x - m|
    segments = -(-x.shape[1] // 8192) + 1
    z = 2.0 ** -23 * (2 + spread) + 2.0 ** -24 * (64 + 6 + 4 + segments + 8)
    names = ("logprobs", "entropy", "top_logprobs")
    for name, a, e, t in zip(names, (got[0], got[1], got[3]), (given, ent, lps), (z, z * (2 + spread), z[:, None])):
        a = a.cpu().double()
        assert torch.equal(torch.isnan(a), torch.isnan(e)), name
        same = (a == e) | torch.isnan(e)   # infinities
        err = torch.where(same, torch.zeros_like(e), (a - e).abs())
        tol = t + 2.0 ** -24 * e.abs()
        assert bool((same | (err <= tol)).all()), f"{name}: error {err.max():.3e}"
    assert torch.equal(got[2].cpu(), ids)
    return got


@pytest.mark.parametrize("vocab", [1, 2, 7, 8, 255, 1000, 4099, 8191, 8192, 16383, 16384, 16385, 50001, 151936])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_token_logprobs_sizes(vocab, dtype):
    g = torch.Generator().manual_seed(vocab)
    for rows, top in ((1, min(vocab, 20)), (3, min(vocab, 5)), (5, 0), (2, min(vocab, 32))):
        x = (torch.randn(rows, vocab, generator=g) * 3).to(dtype)
        _logprobs(x.to(DEV), [int(torch.randint(0, vocab, (1,), generator=g)) for _ in range(rows)], top)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("offset,stride", [(0, 1003), (1, 1007), (3, 1001), (5, 2000), (7, 1000)])
def test_token_logprobs_rows_that_start_anywhere(dtype, offset, stride):
    g = torch.Generator().manual_seed(offset)
    flat = (torch.randn(offset + 4 * stride, generator=g) * 3).to(dtype).to(DEV)
    x = flat[offset:].as_strided((4, 1000), (stride, 1), offset)
    _logprobs(x, [0, 999, 1, 500], 9, host=x.float().cpu())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_token_logprobs_masked_tied_and_unusual_rows(dtype):
    low, inf, nan = torch.finfo(dtype).min, float("inf"), float("nan")
    V = 40000
    g = torch.Generator().manual_seed(8)
    base = (torch.randn(14, V, generator=g) * 2).to(dtype)
    base[0] = 1.5                                  # all equal
    base[1] = -inf                                 # nothing left
    base[2] = low                                  # masked with the type's lowest value, all of it
    base[3] = -inf; base[3, 39999] = 2; base[3, 17] = 2; base[3, 20000] = -4
    base[4] = low; base[4, 5] = 0; base[4, 33333] = 0
    base[5, 100] = nan
    base[6, 200] = inf
    base[7, 300] = inf; base[7, 301] = inf; base[7, 9] = nan
    base[8] = 0.0; base[8, ::2] = -0.0             # equal values of either sign
    base[9, :16384] = -inf                         # a whole segment masked
    base[10, 20000:] = low
    base[11] = -nan if dtype == torch.float32 else base[11]
    base[12] = torch.finfo(dtype).max
    base[13, 1::2] = -inf
    _logprobs(base.to(DEV), [3, 4, 5, 17, 5, 7, 8, 9, 10, 11, 12, 39999, 0, 2], 20)
    x = base[13:14].to(DEV)
    got = _ops().token_logprobs(x.expand(4, V), torch.tensor([-1, V, 2 ** 31 - 1, 1], dtype=torch.int32, device=DEV), 3)
    assert bool(torch.isnan(got[0][:3]).all()) and float(got[0][3]) == -inf
    assert torch.equal(got[2], got[2][:1].expand(4, 3))


def test_token_logprobs_many_leaders_in_few_places():
    """Alternatives that sit close together, in rising and falling runs: every choice of candidates has to cope."""
    V = 60000
    for step in (1.0, -1.0):
        x = torch.zeros(3, V) - 50
        x[0] = torch.arange(V) * step * 1e-3
        x[1, 4096:8192] = torch.arange(4096) * step * 1e-2
        x[2, ::257] = torch.arange(-(-V // 257)).float() * step
        _logprobs(x.to(DEV), [1, 5000, 257], 32)
        _logprobs(x.to(torch.bfloat16).to(DEV), [1, 5000, 257], 32)
    # 31 lanes hold hundreds of values above all but a few others
    x = torch.full((1, 16384), -9.0)
    for lane in range(31):
        for load in range(8):
            x[0, load * 2048 + lane * 8: load * 2048 + lane * 8 + 8] = 10 + lane * 0.01 + load
    x[0, 1000] = 9.0
    _logprobs(x.to(DEV), [1000], 32)
    _logprobs(x.to(torch.bfloat16).to(DEV), [1000], 32)


def test_token_logprobs_captured():
    ops = _ops()
    x = torch.zeros(4, 30001, dtype=torch.bfloat16, device=DEV)
    tok = torch.tensor([1, 2, 3, 30000], dtype=torch.int32, device=DEV)
    ws = torch.empty(ops.token_logprobs_workspace_bytes(4, 30001, x.dtype, 5), dtype=torch.uint8, device=DEV)
    ops.token_logprobs(x, tok, 5, workspace=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.inference_mode(), torch.cuda.graph(graph):
        out = ops.token_logprobs(x, tok, 5, workspace=ws)
    for seed in range(3):
        x.copy_(torch.randn(4, 30001, generator=torch.Generator().manual_seed(seed)) * 3)
        graph.replay()
        torch.cuda.synchronize()
        want = ops.token_logprobs(x, tok, 5)
        assert all(torch.equal(a, b) for a, b in zip(out, want))
