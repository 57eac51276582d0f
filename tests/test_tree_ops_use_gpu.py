"""The speculative-decoding operators in uses that share something: two captured graphs, other streams, batches padded with idle requests, the
largest trees, buffers passed on in place; and what their wrappers refuse."""
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


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _args(c):
    lens = [n + p for n, p in zip(c["nodes"], c["prefix_list"])]
    d = {k: v.to(DEV) if isinstance(v, torch.Tensor) else v for k, v in c.items()}
    return [d["q"], d["k"], d["v"], d["r2t"], d["rows"], d["cu"], d["prefix"], d["mask"], max(c["nodes"]), max(lens), c["scale"]]


def _check(out, c):
    exact, absv, size = tc.attention_oracle(c)
    assert bool(((out.cpu().double() - exact).abs() <= tc.attention_tolerance(exact, absv, size)).all())


def test_two_graphs_with_workspaces_of_their_own_making():
    """Workspaces that the wrapper allocates during capture belong to the graph: replays in turn, with eager calls between, keep their bits."""
    ops = _ops()
    cases = [tc.attention_case([6, 3], [3000, 1500], 8, 2, 16, 5), tc.attention_case([20, 17], [2500, 700], 16, 2, 16, 6)]
    args = [_args(c) for c in cases]
    logits = torch.randn(3, 40000, generator=torch.Generator().manual_seed(1)).to(DEV)
    tok = _i32([1, 2, 39999])
    eager = [(ops.tree_attention(*a), *ops.token_logprobs(logits * (i + 1), tok, 6)) for i, a in enumerate(args)]
    scaled = [logits, logits * 2]
    torch.cuda.synchronize()
    graphs, outs = [], []
    pool = torch.cuda.graph_pool_handle()
    for i, a in enumerate(args):
        g = torch.cuda.CUDAGraph()
        with torch.inference_mode(), torch.cuda.graph(g, pool=pool):
            outs.append((ops.tree_attention(*a), *ops.token_logprobs(scaled[i], tok, 6)))
        graphs.append(g)
    for order in ([0, 1], [1, 0], [0, 0, 1]):
        for i in order:
            graphs[i].replay()
            ops.tree_attention(*args[1 - i])
            torch.cuda.synchronize()
            for got, want in zip(outs[i], eager[i]):
                assert torch.equal(got, want)
    for e, c in zip(eager, cases):
        _check(e[0], c)


def test_calls_in_flight_on_two_streams():
    ops = _ops()
    cases = [tc.attention_case([9, 4], [4000, 900], 8, 2, 16, s) for s in (1, 2)]
    args = [_args(c) for c in cases]
    want = [ops.tree_attention(*a) for a in args]
    logits = [torch.randn(50, 20000, generator=torch.Generator().manual_seed(s)).to(torch.bfloat16).to(DEV) for s in (3, 4)]
    tok = _i32(list(range(50)))
    lp = [ops.token_logprobs(x, tok, 3) for x in logits]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append((ops.tree_attention(*args[i]), *ops.token_logprobs(logits[i], tok, 3)))
    torch.cuda.synchronize()
    for i in range(2):
        for g in got[i]:
            assert torch.equal(g[0], want[i]) and all(torch.equal(a, b) for a, b in zip(g[1:], lp[i]))


def test_batch_padded_with_idle_requests_and_rows():
    """Requests without nodes between and behind the others, and rows behind the last node: left as they are."""
    ops = _ops()
    c = tc.attention_case([5, 0, 2, 0], [100, 50, 9, 0], 16, 2, 16, 8)
    a = _args(c)
    out = torch.full((12, 16, D), 7.0, dtype=torch.bfloat16, device=DEV)
    a[0] = torch.cat([a[0], torch.full((5, 16, D), float("nan"), dtype=torch.bfloat16, device=DEV)])
    a[7] = torch.cat([a[7], torch.full((5, 1), -1, dtype=torch.int64, device=DEV)])
    ops.tree_attention(*a, out=out)
    _check(out[:7], c)
    assert bool((out[7:] == 7).all())


@pytest.mark.parametrize("nodes,prefix,Hq,Hkv", [([1024], [0], 8, 1), ([1023, 1], [129, 2000], 8, 8), ([1000, 1024, 3], [70, 1, 500], 4, 2)])
def test_largest_trees(nodes, prefix, Hq, Hkv):
    c = tc.attention_case(nodes, prefix, Hq, Hkv, 16, sum(nodes), words=16)
    _check(_ops().tree_attention(*_args(c)), c)


def test_bounds_that_are_too_small_or_far_too_large_change_nothing_but_the_cut():
    ops = _ops()
    c = tc.attention_case([7, 30], [900, 2000], 8, 2, 16, 11)
    a = _args(c)
    for bound, total in ((1, 0), (500, 10), (2030, 0), (2 ** 20, 0), (2 ** 30, 2 ** 40), (2030, -5)):
        a[9] = bound
        _check(ops.tree_attention(*a, total_kv=total), c)


def test_a_step_over_and_over_in_place_and_captured():
    """prepare_extend and accept_tree with every state buffer passed on in place, as a decoder uses them: a captured step and an eager one stay
    equal over many steps, and table and free list tell the same story as the page allocator's order."""
    ops, bs, most, ps = _ops(), 3, 6, 4
    rng = random.Random(2)

    def state():
        return dict(rows=_i32([2, 0, 1]), prefix=_i32([3, 8, 0]), new=_i32([0] * bs), alloc=_i32([3, 8, 0]), free=_i32(list(range(1, 201))),
                    range=_i32([4, 200]), r2t=torch.zeros(3, 256, dtype=torch.int32, device=DEV), pos=_i32([0] * bs * most), loc=_i32([0] * bs * most),
                    cu=_i32([0] * (bs + 1)), seq=_i32([0] * bs), status=_i32([0]), parents=_i32([0] * bs * most), draft=_i32([0] * bs * most),
                    target=_i32([0] * bs * most), mask=torch.zeros(bs * most, 1, dtype=torch.int64, device=DEV), lens=_i32([0] * bs),
                    arows=torch.zeros(bs, most, dtype=torch.int32, device=DEV), atok=torch.zeros(bs, most, dtype=torch.int32, device=DEV),
                    next=_i32([0] * bs), kv=torch.arange(804, device=DEV).view(804, 1, 1, 1).expand(804, 2, 1, D).to(torch.bfloat16).contiguous())

    def step(s, layers):
        ops.prepare_extend(s["rows"], s["prefix"], s["new"], s["alloc"], s["free"], s["range"], s["r2t"], s["pos"], s["loc"], s["cu"], s["seq"], s["status"],
                           ps, parents=s["parents"], tree_mask=s["mask"])
        ops.accept_tree(s["draft"], s["target"], s["parents"], s["cu"], s["prefix"], s["loc"], layers, s["lens"], s["arows"], s["atok"], s["next"],
                        s["prefix"])

    eager, captured = state(), state()
    for s in (eager, captured):   # the first rows' slots: pages 1 (request 0), 2 and 3 (request 1)
        s["r2t"][2, :4] = torch.arange(4, 8, device=DEV)
        s["r2t"][0, :8] = torch.arange(8, 16, device=DEV)
    layers = [ops.kv_layers([s["kv"][:, 0]], [s["kv"][:, 1]]) for s in (eager, captured)]
    step(captured, layers[1])     # no request has a node: nothing changes
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.inference_mode(), torch.cuda.graph(graph):
        step(captured, layers[1])
    total = 0
    for i in range(25):
        new = [rng.randint(0, most) for _ in range(bs)]
        parents = [p for n in new for p in tc.tree_parents(rng, n)[:n]]
        draft, target = ([rng.randrange(2) for _ in parents] for _ in range(2))
        for s in (eager, captured):
            s["new"].copy_(_i32(new))
            for name, v in (("parents", parents), ("draft", draft), ("target", target)):
                s[name][: len(v)].copy_(_i32(v))
        step(eager, layers[0])
        graph.replay()
        torch.cuda.synchronize()
        for name in eager:
            assert torch.equal(eager[name], captured[name]), (i, name)
        total += sum(len(p) for p, _ in tc.accept_oracle(draft, target, parents, new, most))
        assert int(eager["status"]) == 0 and int(eager["prefix"].sum()) == 11 + total
        alloc = eager["alloc"].tolist()
        assert int(eager["range"][0]) - 4 == sum(-(-a // ps) for a in alloc) - 3
        slots = torch.cat([eager["r2t"][r, :a] for r, a in zip([2, 0, 1], alloc)])
        assert slots.unique().numel() == slots.numel() and int(slots.min()) >= ps


def test_wrappers_refuse():
    ops = _ops()
    c = tc.attention_case([5, 2], [100, 9], 8, 2, 16, 8)
    a = _args(c)
    for at, bad, words in ((0, a[0].float(), "q must be"), (0, a[0][..., :64], "q must be"), (1, a[1].cpu(), "k_cache"), (2, a[2][:-1], "k_cache"),
                           (1, a[1].half(), "k_cache"), (3, a[3].long(), "req_to_token"), (3, a[3].cpu(), "req_to_token"), (4, a[4].long(), "req_pool_indices"),
                           (5, a[5][:-1], "cu_seqlens_q"), (6, a[6].cpu(), "prefix_lens"), (7, a[7][:-1], "tree_mask"), (7, a[7].int(), "tree_mask"),
                           (8, 65, "max_seqlen_q"), (8, 0, "max_seqlen_q")):
        with pytest.raises(ValueError, match=words):
            ops.tree_attention(*a[:at], bad, *a[at + 1:])
    with pytest.raises(ValueError, match="out must"):
        ops.tree_attention(*a, out=a[0].float())
    for kw in (dict(out=a[0]), dict(out=torch.empty(7, 9 * D, dtype=torch.bfloat16, device=DEV)[:1, : 8 * D].expand(7, 8 * D).view(7, 8, D))):
        with pytest.raises(Exception, match="out overwrites q|out_stride"):
            ops.tree_attention(*a, **kw)
    with pytest.raises(ValueError, match="workspace"):
        ops.tree_attention(*a, workspace=torch.empty(64, dtype=torch.uint8))
    x, tok = torch.zeros(3, 100, device=DEV), _i32([0, 1, 2])
    for args, words in (((x.half(), tok), "bf16 or fp32"), ((x, tok.long()), "token_ids"), ((x, tok[:2]), "token_ids"), ((x, tok, 33), "top_k"),
                        ((x[:, :5], tok, 6), "top_k"), ((x.t(), tok), "dense"), ((x, tok.cpu()), "token_ids")):
        with pytest.raises(ValueError, match=words):
            ops.token_logprobs(*args)
    with pytest.raises(Exception, match="workspace"):
        ops.token_logprobs(torch.zeros(3, 10000, device=DEV), tok, 2, workspace=torch.empty(16, dtype=torch.uint8, device=DEV))
    kv = torch.zeros(10, 2, 2, D, dtype=torch.bfloat16, device=DEV)
    for k, v in (([kv[:, 0]], []), ([kv[:, 0], kv[:9, 0]], [kv[:, 1], kv[:9, 1]]), ([kv[:, 0].float()], [kv[:, 1].float()])):
        with pytest.raises(ValueError):
            ops.kv_layers(k, v)
    layers = ops.kv_layers([kv[:, 0]], [kv[:, 1]])
    good = [_i32([1, 2]), _i32([1, 2]), _i32([-1, 0]), _i32([0, 2]), _i32([3]), _i32([4, 5]), layers, _i32([0]), _i32([[0, 0]]), _i32([[0, 0]]), _i32([0]), _i32([0])]
    ops.accept_tree(*good)
    for at, bad, words in ((0, good[0].long(), "draft_tokens"), (1, good[1][:1], "target_tokens"), (3, _i32([0]), "cu_seqlens_q"), (7, _i32([0, 0]), "accept_lens"),
                           (8, _i32([[0]]), "accept_rows and accept_tokens"), (9, _i32([[0, 0]]).long(), "accept_rows and accept_tokens"),
                           (10, good[10].cpu(), "next_tokens"), (5, good[5].cpu(), "out_cache_loc")):
        with pytest.raises(ValueError, match=words):
            ops.accept_tree(*good[:at], bad, *good[at + 1:])
    with pytest.raises(Exception, match="overwrites"):
        ops.accept_tree(*good[:10], good[4], good[11])
    args = [_i32([0]), _i32([1]), _i32([2]), _i32([1]), _i32([1, 2, 3]), _i32([0, 3]), torch.zeros(2, 16, dtype=torch.int32, device=DEV), _i32([0, 0]),
            _i32([0, 0]), _i32([0, 0]), _i32([0]), _i32([0])]
    for at, bad, words in ((1, args[1].long(), "prefix_lens"), (5, _i32([0]), "free_range"), (6, args[6].t(), "req_to_token"), (7, _i32([0]), "positions"),
                           (9, _i32([0]), "cu_seqlens_q"), (11, _i32([0, 0]), "status")):
        with pytest.raises(ValueError, match=words):
            ops.prepare_extend(*args[:at], bad, *args[at + 1:], 16)
    with pytest.raises(ValueError, match="go together"):
        ops.prepare_extend(*args, 16, parents=_i32([0, 0]))
    with pytest.raises(ValueError, match="tree_mask"):
        ops.prepare_extend(*args, 16, parents=_i32([0, 0]), tree_mask=torch.zeros(2, 17, dtype=torch.int64, device=DEV))
    with pytest.raises(Exception, match="overwrites"):
        ops.prepare_extend(*args[:10], args[1], args[11], 16)


@pytest.mark.parametrize("bs,longest,most,Hq,Hkv", [(70, 2500, 6, 4, 1), (130, 900, 12, 8, 1), (130, 5000, 12, 8, 1), (9, 6000, 20, 8, 4), (5, 4000, 70, 16, 2), (3, 9000, 1, 8, 8)])
def test_shares_of_unequal_requests(bs, longest, most, Hq, Hkv):
    """Requests of very different length, some without nodes: work groups that end one request and begin others, row tiles that not every request
    has, more requests than lanes; with the whole workspace, with room for a few runs per request only, and with wrong hints."""
    ops = _ops()
    rng = random.Random(bs)
    nodes = [0 if rng.random() < 0.15 else rng.randint(1, most) for _ in range(bs)]
    nodes[rng.randrange(bs)] = most
    prefix = [int(longest * rng.random() ** 3) for _ in range(bs)]
    prefix[bs // 2] = longest
    c = tc.attention_case(nodes, prefix, Hq, Hkv, 16, bs)
    a = _args(c)
    total = sum(n + p for n, p in zip(nodes, prefix))
    splits = ops.tree_attention_splits(bs, max(nodes), a[9], Hq, Hkv, total)
    assert splits > 1 or longest < 1000  # (that short, a work group per request is quicker: the other cases share)
    first = ops.tree_attention(*a, total_kv=total)
    _check(first, c)
    assert torch.equal(first, ops.tree_attention(*a, total_kv=total))
    for room in (1, 2, 3, splits + 5):
        ws = torch.empty(ops.tree_attention_workspace_bytes(sum(nodes), Hq, D, room) + 16, dtype=torch.uint8, device=DEV)
        _check(ops.tree_attention(*a, total_kv=total, workspace=ws), c)
    a[9] = longest // 3
    _check(ops.tree_attention(*a, total_kv=total // 4), c)


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("bs,most,tree", [(1024, 4, True), (1025, 4, True), (300, 90, False), (70, 130, True), (3, 5000, False), (200, 25, True), (1024, 9, False)])
def test_prepare_extend_in_place_and_apart(bs, most, tree, in_place):
    """Steps on both sides of every bound of the one-launch form, in place and not, accepted and refused."""
    from test_tree_ops_gpu import _prepare

    rng = random.Random(bs + most)
    prefix = [rng.randint(0, 50) for _ in range(bs)]
    new = [rng.randint(0, most) for _ in range(bs)]
    new[-1] = most
    alloc = [p + rng.choice([0, 0, 2, 20]) for p in prefix]
    ok = dict(prefix=prefix, new=new, alloc=alloc, page_size=16, seed=bs, tree=tree, in_place=in_place)
    assert _prepare(**ok) == 0
    assert _prepare(**ok, capacity=sum(new) + 1500) == 0
    assert _prepare(**ok, cut=3) == 1
    assert _prepare(**ok, capacity=sum(new) - 1) == 4
    assert _prepare(**ok, status=5) == 5
    assert _prepare(**dict(ok, alloc=[-1] + alloc[1:])) == 3


@pytest.mark.parametrize("form", [0, 1])
@pytest.mark.parametrize("shares", [0, 1])
def test_every_form_of_tree_attention(variants, form, shares):
    """The cases of the attention tests with every layout pinned: row tiles of 32 and the forms for more rows, a work group per request and equal
    shares of all tiles, however small the launch."""
    import test_tree_ops_gpu as t

    variants("tree_form", form)
    variants("tree_shares", shares)
    for heads in ((16, 8), (32, 8), (8, 1), (16, 2)):
        t.test_tree_attention_heads_and_pages(*heads, 5, "interleaved")
    for nodes, prefix in (([1], [0]), ([33], [33]), ([64], [63]), ([65], [64]), ([130], [500]), ([17, 1, 64, 40], [0, 1, 300, 95]), ([5] * 40, list(range(0, 80, 2))),
                          ([20, 0, 33, 7], [300, 10, 0, 64])):
        for heads in ((8, 1), (8, 2), (4, 4)):
            c = tc.attention_case(nodes, prefix, *heads, 16, 7 + sum(nodes))
            _check(_ops().tree_attention(*_args(c)), c)
    t.test_tree_attention_rows_that_see_nothing_and_wide_masks()
    t.test_tree_attention_unseen_nodes_never_reach_a_row()
    t.test_tree_attention_strided_query_output_and_rows_behind_the_last()
    t.test_tree_attention_slots_beyond_32_bit_offsets()
    t.test_tree_attention_agrees_with_decode_and_extend()
    t.test_tree_attention_captured_and_on_another_stream()
    test_batch_padded_with_idle_requests_and_rows()
    if shares:
        test_shares_of_unequal_requests(5, 4000, 70, 16, 2)


@pytest.mark.parametrize("form", [0, 1])
@pytest.mark.parametrize("nodes,prefix,Hq,Hkv", [([61, 40, 33], [3000, 700, 5000], 32, 8), ([30, 20], [2500, 2600], 32, 8), ([14, 9, 16], [4000, 100, 900], 16, 4),
                                                 ([100], [3000], 16, 2), ([1023, 1], [129, 2000], 8, 8)])
def test_every_form_over_long_prefixes(variants, form, nodes, prefix, Hq, Hkv):
    variants("tree_form", form)
    c = tc.attention_case(nodes, prefix, Hq, Hkv, 16, sum(nodes))
    a = _args(c)
    _check(_ops().tree_attention(*a), c)
    _check(_ops().tree_attention(*a, workspace=torch.empty(16, dtype=torch.uint8, device=DEV)), c)


@pytest.mark.parametrize("in_place", [True, False])
def test_prepare_extend_with_an_empty_free_list(in_place):
    """No page left at all: a step that needs none goes through, one that needs one is refused."""
    ops = _ops()
    for new, status in (([3, 0], 0), ([4, 0], 1)):
        alloc, rng = _i32([8, 5]), _i32([0, 0])
        r2t = torch.zeros(2, 32, dtype=torch.int32, device=DEV)
        r2t[0, :8], r2t[1, :5] = torch.arange(8, 16), torch.arange(24, 29)
        pos, loc, cu, seq, st = _i32([9] * 4), _i32([9] * 4), _i32([9] * 3), _i32([9] * 2), _i32([0])
        extra = {} if in_place else dict(alloc_out=_i32([0, 0]), free_range_out=_i32([7, 7]))
        ops.prepare_extend(_i32([0, 1]), _i32([5, 5]), _i32(new), alloc, _i32([]), rng, r2t, pos, loc, cu, seq, st, 8, **extra)
        assert int(st) == status and cu.tolist() == ([0, 3, 3] if status == 0 else [0, 0, 0])
        assert loc.tolist() == ([13, 14, 15, 0] if status == 0 else [0] * 4)
        assert (rng if in_place else extra["free_range_out"]).tolist() == [0, 0]


def test_accept_tree_without_any_node():
    ops = _ops()
    none, lens, nxt, seq = _i32([]), _i32([9, 9]), _i32([9, 9]), _i32([0, 0])
    rows, tokens = _i32([[9], [9]]), _i32([[9], [9]])
    ops.accept_tree(none, none, none, _i32([0, 0, 0]), _i32([5, 7]), none, None, lens, rows, tokens, nxt, seq)
    assert lens.tolist() == [0, 0] and seq.tolist() == [5, 7] and nxt.tolist() == [9, 9] and rows.tolist() == tokens.tolist() == [[-1], [-1]]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [700, 4675, 30001])
def test_token_logprobs_far_from_zero(dtype, vocab):
    """Log probabilities do not depend on where the logits lie: no rounding may grow with them."""
    from test_tree_ops_gpu import _logprobs

    g = torch.Generator().manual_seed(vocab)
    for offset in (418.0, -700.0, 9000.0, -80000.0, 99999.0, 200000.0):
        x = torch.randn(3, vocab, generator=g) * 3
        x[1] *= 20
        x[2, vocab // 2] += 200
        x = (x + offset).to(dtype)
        _logprobs(x.to(DEV), [0, vocab - 1, vocab // 2], 11, host=x.float())
