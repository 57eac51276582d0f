"""Edges of the speculative-decoding operators and of the decoder that runs them."""
import random

import pytest
import torch

import tree_cases as tc
import tree_growth_cases as growth

pytestmark = pytest.mark.gpu
DEV = "cuda"
D = 128


def _ops():
    from mini_sglang_amd import ops
    return ops


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _attend(c, **kw):
    d = {k: v.to(DEV) if isinstance(v, torch.Tensor) else v for k, v in c.items()}
    return _ops().tree_attention(d["q"], d["k"], d["v"], d["r2t"], d["rows"], d["cu"], d["prefix"], d["mask"], max(c["nodes"]),
                                 max(n + p for n, p in zip(c["nodes"], c["prefix_list"])), c["scale"], **kw)


FORMS = [(form, shares) for form in (0, 1) for shares in (0, 1)]
# rows per kv head: up to 32, 64, 128, 256 and beyond; prefixes that end inside a tile, at its end and that are empty
SHAPES = [([3, 1, 4], [40, 0, 64], 16, 8), ([7, 12, 0], [333, 31, 5], 8, 2), ([25, 6], [500, 96], 8, 2), ([40, 33], [1300, 0], 8, 1)]


@pytest.mark.parametrize("form,shares", FORMS)
@pytest.mark.parametrize("nodes,prefix,Hq,Hkv", SHAPES)
def test_scale_zero_is_the_mean_of_the_visible_values(variants, form, shares, nodes, prefix, Hq, Hkv):
    variants("tree_form", form), variants("tree_shares", shares)
    c = tc.attention_case(nodes, prefix, Hq, Hkv, 16, 3 + sum(nodes))
    c["scale"] = 0.0
    c["masks"][1] = 0   # sees its prefix alone
    if 0 in prefix:
        c["masks"][sum(nodes[: prefix.index(0)])] = 0   # sees nothing
    c["mask"] = tc.pack_masks(c["masks"], c["mask"].shape[1])
    exact, absv, size = tc.attention_oracle(c)
    err = (_attend(c).cpu().double() - exact).abs()
    assert bool((err <= tc.attention_tolerance(exact, absv, size)).all())


@pytest.mark.parametrize("form,shares", FORMS)
@pytest.mark.parametrize("nodes,prefix,Hq,Hkv", SHAPES)
def test_scores_far_below_zero_are_ordinary_scores(variants, form, shares, nodes, prefix, Hq, Hkv):
    """Scores -scale and -2 scale (or with the other sign), exact in 32 bits: the softmax is the mean over the keys with the larger one, whatever
    the scale."""
    variants("tree_form", form), variants("tree_shares", shares)
    c = tc.attention_case(nodes, prefix, Hq, Hkv, 16, 5 + sum(nodes))
    k = torch.zeros_like(c["k"])
    k[:, :, 0] = -1.0 - torch.randint(0, 2, k.shape[:2], generator=torch.Generator().manual_seed(1)).to(k.dtype)
    c["k"] = k
    for sign in (1.0, -1.0):
        c["q"] = torch.zeros_like(c["q"])
        c["q"][:, :, 0] = sign
        c["scale"] = 64.0                 # e^-64 is nothing beside 1: the limit that every larger scale has
        exact, absv, _ = tc.attention_oracle(c)
        tol = tc.attention_tolerance(exact, absv, torch.zeros(exact.shape[:2], dtype=torch.float64)) + absv * 2.0 ** -64
        for scale in (64.0, 1e20, 1e31, 1e36, 1e38):
            c["scale"] = scale
            err = (_attend(c).cpu().double() - exact).abs()
            assert bool((err <= tol).all()), (sign, scale)


@pytest.mark.parametrize("form,shares", FORMS)
@pytest.mark.parametrize("nodes,prefix,Hq,Hkv", SHAPES)
def test_large_scores_leave_the_largest_and_its_ties(variants, form, shares, nodes, prefix, Hq, Hkv):
    """Whole-number queries and keys, so that products and ties are exact: from a scale of a few hundred on the softmax is the mean over the keys with
    the largest product, however far the scores lie apart."""
    variants("tree_form", form), variants("tree_shares", shares)
    c = tc.attention_case(nodes, prefix, Hq, Hkv, 16, 9 + sum(nodes))
    g = torch.Generator().manual_seed(2)
    c["q"], c["k"] = (torch.randint(-2, 3, x.shape, generator=g).to(torch.bfloat16) for x in (c["q"], c["k"]))
    c["scale"] = 300.0     # e^-300 is nothing beside 1
    exact, absv, _ = tc.attention_oracle(c)
    tol = tc.attention_tolerance(exact, absv, torch.zeros(exact.shape[:2], dtype=torch.float64))
    for scale in (300.0, 1.7e5, 3.3e7, 1e10, 1e20, 1e35):   # (products up to 512: the largest scores are 5e37)
        c["scale"] = scale
        err = (_attend(c).cpu().double() - exact).abs()
        assert bool((err <= tol).all()), scale


@pytest.mark.parametrize("nodes,prefix,Hq,Hkv", [([3, 1, 4], [400, 0, 64], 16, 8), ([7, 8, 0], [1333, 31, 5], 8, 2), ([4, 1, 3], [40, 700, 3], 8, 1),
                                                 ([32, 20], [2000, 0], 4, 4)])
@pytest.mark.parametrize("shares", [0, 1])
def test_up_to_32_rows_per_kv_head_the_result_is_rounded_once(variants, shares, nodes, prefix, Hq, Hkv):
    """As in the decode kernel that such a step stands in for: 2^-8 of the result, for its own rounding, beside errors of 32-bit arithmetic and 2^-16 of
    sum p |v| for the probabilities in two bf16 parts (each half a step: 2^-8 of what the first leaves)."""
    variants("tree_shares", shares)
    c = tc.attention_case(nodes, prefix, Hq, Hkv, 16, 40 + sum(nodes))
    exact, absv, size = tc.attention_oracle(c)
    rest = absv * (2 * 129 * 2.0 ** -24 * size.unsqueeze(-1) + 2.0 ** -20 + 2.0 ** -16)
    err = (_attend(c).cpu().double() - exact).abs()
    assert bool((err <= 2.0 ** -8 * (exact.abs() + rest) + rest).all()), float((err / (2.0 ** -8 * (exact.abs() + rest) + rest)).max())


@pytest.mark.parametrize("form,shares", FORMS)
@pytest.mark.parametrize("shape", growth.SHAPES)
def test_scores_that_grow_along_the_context(variants, form, shares, shape):
    """Maxima that rise by 10 to 40 log2 units several times, fall and peak, at other places for every direction a query looks in: every rescale of a
    state, and factors of the joins between waves and runs from 1 to nothing."""
    variants("tree_form", form), variants("tree_shares", shares)
    for seed in (5, 6):
        c = growth.growing_case(*shape, seed)
        exact, absv, size = tc.attention_oracle(c)
        tol = tc.attention_tolerance(exact, absv, size)
        err = (_attend(c).cpu().double() - exact).abs()
        assert bool((err <= tol).all()), seed
        ws = torch.empty(_ops().tree_attention_workspace_bytes(sum(shape[0]), shape[2], D, 3), dtype=torch.uint8, device=DEV)
        err = (_attend(c, workspace=ws).cpu().double() - exact).abs()   # room for three runs per request
        assert bool((err <= tol).all()), seed


def _build(ps, lens, budget=120, use_graph=True):
    from test_tree_decode_gpu import _build as build
    return build(ps, lens, budget, use_graph)


@pytest.mark.parametrize("ps,use_graph", [(1, True), (16, True), (16, False)])
def test_tree_steps_go_on_after_plain_decoding(ps, use_graph):
    """Tree steps, plain decoding, tree steps, chained decoding, tree steps: one greedy stream, and no page lost on the way."""
    from mini_sglang_amd.runtime import decode_loop
    from mini_sglang_amd.runtime.device_decode import DeviceDecodeLoop
    from mini_sglang_amd.runtime.tree_decode import TreeDecoder

    lens, steps = [15, 16, 33, 300], 70
    mr, batch = _build(ps, lens, use_graph=use_graph)
    start = [len(r.token_ids) for r in batch.reqs]
    decode_loop.decode_steps(mr, batch, steps)
    truth = [r.token_ids[n:] for r, n in zip(batch.reqs, start)]

    mr, batch = _build(ps, lens, use_graph=use_graph)
    pages = mr.page_allocator.free_count()
    dec = TreeDecoder(mr, batch, 6, max_new_tokens=16, use_graph=use_graph)
    rng = random.Random(ps)

    def done():
        return [len(r.token_ids) - n for r, n in zip(batch.reqs, start)]

    def tree_steps(n):
        for _ in range(n):
            drafts = []
            for t, d in zip(truth, done()):
                right = rng.randint(0, 3)   # that many of the chain's five tokens are the true ones
                drafts.append((t[d: d + right] + [rng.randrange(2048) for _ in range(5 - right)], [0, 1, 2, 3, 4]))
            dec.step(drafts)
        dec.sync_host()

    def check():
        for r, n, t, d, length in zip(batch.reqs, start, truth, done(), lens):
            assert r.token_ids[n:] == t[:d]
        assert batch.seq_lens_cpu.tolist() == [n + d for n, d in zip(lens, done())]
        assert mr.page_allocator.free_count() == pages - sum(-(-(n + d) // ps) - -(-n // ps) for n, d in zip(lens, done()))

    tree_steps(3)
    check()
    decode_loop.decode_steps(mr, batch, 5)
    check()
    tree_steps(3)
    check()
    decode_loop.decode_steps(mr, batch, 18)   # beyond what the captured bounds were made for
    tree_steps(2)
    check()
    if use_graph:
        loop = DeviceDecodeLoop(mr, batch, max_steps=4)
        loop.run(4)
        loop.sync_host()
        tree_steps(1)
        check()
    assert max(done()) <= steps


def test_decoder_refuses_requests_that_moved_on_without_it():
    from mini_sglang_amd.runtime import decode_loop
    from mini_sglang_amd.runtime.tree_decode import TreeDecoder

    mr, batch = _build(64, [10, 70])     # (a page has room for all that follows: the page allocator does not change)
    dec = TreeDecoder(mr, batch, 4)
    none = [([], [])] * 2
    dec.step(none)
    decode_loop.decode_steps(mr, batch, 1)   # without sync_host
    with pytest.raises(RuntimeError, match="sync_host"):
        dec.step(none)
    mr, batch = _build(64, [10, 70])
    dec = TreeDecoder(mr, batch, 4)
    batch.reqs[0].token_ids.append(5)        # a token that no cache row stands behind
    with pytest.raises(RuntimeError, match="token"):
        dec.step(none)
    batch.reqs[0].token_ids.pop()
    dec.step(none)
    batch.filter_reqs([1])
    with pytest.raises(RuntimeError, match="requests"):
        dec.step(none)
    with pytest.raises(RuntimeError, match="requests"):
        dec.sync_host()


@pytest.mark.parametrize("bs,capacity,tree", [(3, 40, True), (3, 5000, True), (3, 5000, False), (1500, 3000, False)])
@pytest.mark.parametrize("named", [(True, True), (True, False), (False, True)])
def test_prepare_extend_in_place_by_name(bs, capacity, tree, named):
    """alloc_out = alloc_lens and free_range_out = free_range by name are the in-place call, and one of them may be."""
    ops = _ops()
    rng = random.Random(bs)
    prefix = [rng.randint(0, 30) for _ in range(bs)]
    new = [rng.randint(0, 2) for _ in range(bs)]
    results = []
    for by_name in (False, True):
        alloc, fr = _i32(prefix), _i32([0, 4 * bs])
        r2t = torch.arange(bs * 64, dtype=torch.int32, device=DEV).view(bs, 64) + 16 * (4 * bs + 1)
        out = [_i32([9] * capacity), _i32([9] * capacity), _i32([9] * (bs + 1)), _i32([9] * bs), _i32([0])]
        mask = torch.zeros(capacity, 1, dtype=torch.int64, device=DEV) if tree else None
        extra = dict(alloc_out=alloc if named[0] else _i32([9] * bs), free_range_out=fr if named[1] else _i32([9, 9])) if by_name else {}
        ops.prepare_extend(_i32(list(range(bs))), _i32(prefix), _i32(new), alloc, _i32(list(range(1, 4 * bs + 1))), fr, r2t, *out, 16,
                           parents=_i32([-1] * capacity) if tree else None, tree_mask=mask, **extra)
        results.append([r2t, *out, *([mask] if tree else []), extra.get("alloc_out", alloc), extra.get("free_range_out", fr)])
    assert int(results[0][5]) == 0
    for a, b in zip(*results):
        assert torch.equal(a, b)


@pytest.mark.parametrize("tree", [True, False])
def test_prepare_extend_of_an_empty_batch_clears_every_row(tree):
    """Rows behind the last token are the dummy slot's, also where there is no request at all: a model run over them writes nothing that is somebody's."""
    ops = _ops()
    none = _i32([])
    for apart in (False, True):
        pos, loc, cu, fr, st = _i32([7] * 9), _i32([7] * 9), _i32([7]), _i32([3, 8]), _i32([0])
        mask = torch.full((9, 2), 7, dtype=torch.int64, device=DEV) if tree else None
        fro = _i32([9, 9]) if apart else None
        r2t = torch.full((2, 32), 5, dtype=torch.int32, device=DEV)
        ops.prepare_extend(none, none, none, none, _i32([1] * 8), fr, r2t, pos, loc, cu, none, st, 16, parents=_i32([0] * 9) if tree else None,
                           tree_mask=mask, free_range_out=fro)
        assert pos.tolist() == loc.tolist() == [0] * 9 and cu.tolist() == [0] and int(st) == 0
        assert fr.tolist() == [3, 8] and (fro is None or fro.tolist() == [3, 8]) and bool((r2t == 5).all())
        assert mask is None or not bool(mask.any())


@pytest.mark.parametrize("bs", [3, 1500])
def test_prepare_extend_with_arrays_side_by_side(bs):
    """Cut out of one buffer, next to one another and in the gaps between the table's rows, arrays share no memory; page_size 1 has one table for both."""
    ops = _ops()
    prefix, new = [i % 7 for i in range(bs)], [1 + i % 3 for i in range(bs)]
    total = sum(new)
    results = []
    for side_by_side in (False, True):
        if side_by_side:
            flat = torch.full((8 * bs + 2 * total + 200,), 9, dtype=torch.int32, device=DEV)
            wide = torch.zeros(bs, 16 + 8, dtype=torch.int32, device=DEV)
            at = [0]

            def make(values):
                at[0] += len(values)
                flat[at[0] - len(values): at[0]] = _i32(values)
                return flat[at[0] - len(values): at[0]]

            table, fr = wide[:, :16], wide[bs - 2, 16:18]
            fr.copy_(_i32([0, 3 * bs]))
        else:
            make, table, fr = _i32, torch.zeros(bs, 16, dtype=torch.int32, device=DEV), _i32([0, 3 * bs])
        args = [make(list(range(bs))), make(prefix), make(new), make(prefix), _i32(list(range(1, 3 * bs + 1))), fr, table]
        out = [make([9] * total), make([9] * total), make([9] * (bs + 1)), make([9] * bs), make([0])]
        ops.prepare_extend(*args, *out, 1, req_to_page=table)
        results.append([args[3], args[5], table, *out])
    assert int(results[0][-1]) == 0
    for a, b in zip(*results):
        assert torch.equal(a, b)


def test_accept_tree_refuses_outputs_among_its_nodes():
    ops = _ops()
    flat = _i32([0] * 40)
    good = dict(draft=flat[:6], target=flat[6: 12], parents=flat[12: 18], cu=_i32([0, 3, 6]), prefix=_i32([1, 2]), loc=flat[18: 24], lens=flat[24: 26],
                rows=flat[26: 30].view(2, 2), tokens=flat[30: 34].view(2, 2), next=flat[34: 36], seq=flat[36: 38])

    def call(**change):
        a = dict(good, **change)
        ops.accept_tree(a["draft"], a["target"], a["parents"], a["cu"], a["prefix"], a["loc"], None, a["lens"], a["rows"], a["tokens"], a["next"], a["seq"])

    call()   # side by side is apart
    for change in (dict(lens=flat[4: 6]), dict(next=flat[5: 7]), dict(seq=flat[10: 12]), dict(rows=flat[20: 24].view(2, 2)), dict(tokens=flat[15: 19].view(2, 2)),
                   dict(loc=flat[23: 29])):
        with pytest.raises(Exception, match="overwrites"):
            call(**change)


def test_tree_attention_with_queries_and_outputs_in_one_buffer():
    """Columns of one wide buffer and rows taken in turn are apart, whatever their strides; the query's own place is not."""
    c = tc.attention_case([5, 12, 1], [60, 9, 100], 8, 2, 16, 12)
    exact, absv, size = tc.attention_oracle(c)
    tol = tc.attention_tolerance(exact, absv, size)
    for make in (lambda n: torch.zeros(n, 20 * D, dtype=torch.bfloat16, device=DEV).split([2 * D, 8 * D, 2 * D, 8 * D], 1)[1::2],
                 lambda n: torch.zeros(n, 2, 8 * D, dtype=torch.bfloat16, device=DEV).unbind(1),
                 lambda n: torch.zeros(2, n, 8 * D, dtype=torch.bfloat16, device=DEV).unbind(0)):
        q, out = (x.unflatten(1, (8, D)) for x in make(18))
        q.copy_(c["q"])
        d = dict(c, q=q)
        assert _attend(d, out=out) is out
        assert bool(((out.cpu().double() - exact).abs() <= tol).all())
        with pytest.raises(Exception, match="overwrites"):
            _attend(d, out=q)
    flat = torch.zeros(20 * 8 * D, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(Exception, match="overwrites"):   # half a head further on
        _attend(dict(c, q=flat[: 18 * 8 * D].view(18, 8, D)), out=flat[64: 64 + 18 * 8 * D].view(18, 8, D))
