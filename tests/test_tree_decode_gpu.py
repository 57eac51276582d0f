"""The speculative step as it is used: slots and masks, the model over all nodes with tree attention, greedy tokens, log probabilities, acceptance and
the move of cache rows, captured in one graph, on a small stack; its tokens are those of plain greedy decoding whatever was drafted."""
import gc
import random

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_decoder_outlives_its_test():
    """torch's captured graphs share the generator's two seed tensors, made by the first of them that is alive: made inside inference mode, where this
    package captures its steps, they would refuse a capture outside it.  (A test that expects exceptions leaves its decoder to the collector.)"""
    yield
    gc.collect()


def _build(ps, lens, budget=96, use_graph=False):
    from mini_sglang_amd.runtime import decode_loop
    from mini_sglang_amd.runtime.qwen3 import Qwen3Config

    torch.manual_seed(1234)  # the harness fills the K/V pools from torch's generator: same contexts in every run
    cfg = Qwen3Config(hidden_size=256, num_hidden_layers=3, num_attention_heads=8, num_key_value_heads=2, intermediate_size=512, vocab_size=2048,
                      max_position_embeddings=4096, tie_word_embeddings=False)
    return decode_loop.build_decode_state(cfg, len(lens), 0, ps, budget, use_graph=use_graph, seed=3, seq_lens=list(lens))


def _draft(rng, truth, at, nodes, kind):
    """A tree below the token `truth[at - 1]`: the true continuation with probability, and wrong branches around it."""
    tokens, parents, path = [], [], 0  # path: the node whose continuation is still true (-1: lost)
    depth = {0: 0}
    for i in range(1, nodes):
        p = 0 if kind == "flat" else i - 1 if kind == "chain" else rng.randrange(max(0, i - 4), i)
        true_here = p == path and at + depth[p] < len(truth)
        if true_here and rng.random() < 0.8:
            tokens.append(truth[at + depth[p]])
            path = i
        else:
            tokens.append(rng.randrange(2048))
        depth[i] = depth[p] + 1
        parents.append(p)
    return tokens, parents


@pytest.mark.parametrize("ps,kind,use_graph", [(1, "tree", True), (16, "tree", True), (16, "chain", False), (16, "flat", True), (64, "tree", False)])
def test_tree_decoding_gives_the_greedy_tokens(ps, kind, use_graph):
    from mini_sglang_amd.runtime import decode_loop
    from mini_sglang_amd.runtime.tree_decode import TreeDecoder

    lens, steps = [15, 16, 33, 700, 1], 40
    mr_a, batch_a = _build(ps, lens)
    start = [len(r.token_ids) for r in batch_a.reqs]
    decode_loop.decode_steps(mr_a, batch_a, steps)
    truth = [r.token_ids[n:] for r, n in zip(batch_a.reqs, start)]

    mr, batch = _build(ps, lens, budget=steps + 40)
    pages = mr.page_allocator.free_count()
    dec = TreeDecoder(mr, batch, 12, max_new_tokens=24, use_graph=use_graph, logprobs=4)
    rng = random.Random(ps)
    done, forwards = [0] * len(lens), 0
    while min(done) < steps - 12:
        drafts = [([], []) if forwards % 5 == 4 else _draft(rng, t, d, rng.randint(1, 12), kind) for t, d in zip(truth, done)]
        got = dec.step(drafts)
        for b, new in enumerate(got):
            assert 1 <= len(new) <= 12
            assert new == truth[b][done[b]: done[b] + len(new)][: len(new)] or done[b] + len(new) > steps
            done[b] += len(new)
            assert len(dec.last_logprobs[b]) == len(new)
            for tok, (lp, ent, ids, tops) in zip(new, dec.last_logprobs[b]):
                assert ids[0] == tok and tops[0] == lp and tops == sorted(tops, reverse=True) and ent > 0 and lp < 0
        forwards += 1
        if max(done) > steps - 12:
            break
        if forwards == 6:
            dec.sync_host()   # spare pages go back and the step goes on
            assert mr.page_allocator.free_count() == pages - sum(-(-(n + d) // ps) - -(-n // ps) for n, d in zip(lens, done))
    assert sum(done) > 1.3 * forwards * len(lens) or kind == "flat", "drafts were accepted"
    dec.sync_host()
    for r, n, d in zip(batch.reqs, lens, done):
        assert r.last_slot == int(mr.req_to_token_pool.req_to_token[r.req_pool_idx, n + d - 1])
    assert batch.seq_lens_cpu.tolist() == [n + d for n, d in zip(lens, done)]
    assert mr.page_allocator.free_count() == pages - sum(-(-(n + d) // ps) - -(-n // ps) for n, d in zip(lens, done))
    # plain decoding goes on from there: the accepted nodes' cache rows are where it looks for them
    left = steps - max(done)
    if left > 0:
        decode_loop.decode_steps(mr, batch, left)
        for r, n, t, d in zip(batch.reqs, start, truth, done):
            assert r.token_ids[n:] == t[: d + left]


def test_tree_step_refusal_changes_nothing():
    from mini_sglang_amd.runtime.tree_decode import TreeDecoder

    mr, batch = _build(1, [10, 20])
    dec = TreeDecoder(mr, batch, 6)
    want = _build(1, [10, 20])
    other = TreeDecoder(*want, 6)
    drafts = [([1, 2, 3], [0, 1, 1]), ([5], [0])]
    dec.free_range[1] = 5   # six slots are needed
    with pytest.raises(RuntimeError, match="free list exhausted"):
        dec.step(drafts)
    dec.free_range[1] = mr.page_allocator.free_count()
    assert dec.prefix_lens.tolist() == [10, 20] and dec.alloc_lens.tolist() == [10, 20]
    for _ in range(3):
        assert dec.step(drafts) == other.step(drafts)
    with pytest.raises(ValueError, match="parent"):
        dec.step([([1], [1]), ([], [])])
    for token in (-1, 2048):
        with pytest.raises(ValueError, match="vocabulary"):
            dec.step([([token], [0]), ([], [])])
    with pytest.raises(ValueError, match="announced"):
        dec.step([([1] * 6, [0] * 6), ([], [])])
    with pytest.raises(ValueError, match="drafts for"):
        dec.step([([], [])])
    with pytest.raises(ValueError, match="max_nodes"):
        TreeDecoder(mr, batch, 2000)


def test_two_decoders_captured_on_one_runner():
    """Two batches with a captured step each, on one model runner: neither's static buffers are the other's."""
    from mini_sglang_amd.runtime.batch_info import BatchInfo
    from mini_sglang_amd.runtime.tree_decode import TreeDecoder

    def halves(batch):
        out = []
        for part in (slice(0, 2), slice(2, 4)):
            b = BatchInfo.init_new(batch.reqs[part], batch.req_to_token_pool, batch.page_allocator, batch.kv_cache_pool)
            b.forward_mode, b.seq_lens, b.seq_lens_cpu = batch.forward_mode, batch.seq_lens[part], batch.seq_lens_cpu[part]
            b.req_pool_indices = batch.req_pool_indices[part]
            out.append(b)
        return out

    lens = [30, 200, 17, 64]
    mr, batch = _build(16, lens)
    want = [[], [], [], []]
    dec = TreeDecoder(mr, batch, 4)
    for _ in range(6):
        for w, new in zip(want, dec.step([([7], [0])] * 4)):
            w += new
    mr, batch = _build(16, lens)
    first, second = (TreeDecoder(mr, b, 4) for b in halves(batch))
    got = [[], [], [], []]
    for _ in range(6):
        for dec, at in ((first, 0), (second, 2)):
            for w, new in zip(got[at: at + 2], dec.step([([7], [0])] * 2)):
                w += new
            with pytest.raises(RuntimeError, match="page allocator changed"):   # two pages back to the pool without the decoder's knowledge
                mr.page_allocator.free(mr.page_allocator.alloc(2))
                dec.sync_host()
            mr.page_allocator.free_page = dec._uploaded
            dec.sync_host()
    assert [g[:6] for g in got] == [w[:6] for w in want]
