"""The speculative-decoding operators as far as no GPU is needed: what their C entry points refuse before any launch, workspace sizes, and the
64-bit oracles of the GPU tests against torch's own functions and the host-side producers."""
import random

import pytest
import torch

import tree_cases as tc

A = [0x100000 + 4096 * i for i in range(16)]  # aligned addresses that nothing reads: every call below is refused, or has nothing to do


def _lib():
    from mini_sglang_amd import _capi
    return _capi.lib, _capi.last_error


def _call(name, order, defaults, change):
    lib, error = _lib()
    assert set(change) <= set(order)
    rc = getattr(lib, name)(*[change.get(k, defaults[k]) for k in order])
    return rc, error()


PREPARE = ("req prefix new alloc free free_capacity range r2t r2t_stride table_rows max_ctx r2p r2p_stride parents mask words positions loc capacity cu "
           "seq alloc_out range_out status bs page_size ws ws_bytes stream").split()
PREPARE_OK = dict(req=A[0], prefix=A[1], new=A[2], alloc=A[3], free=A[4], free_capacity=10, range=A[5], r2t=A[6], r2t_stride=64, table_rows=4, max_ctx=64,
                  r2p=None, r2p_stride=0, parents=A[7], mask=A[8], words=1, positions=A[9], loc=A[10], capacity=8, cu=A[11], seq=A[12], alloc_out=A[3],
                  range_out=A[5], status=A[13], bs=2, page_size=16, ws=None, ws_bytes=0, stream=None)


@pytest.mark.parametrize("change,words", [
    (dict(bs=-1), "bs=-1"), (dict(page_size=0), "page_size=0"), (dict(capacity=-1), "capacity=-1"), (dict(max_ctx=0), "max_ctx=0"),
    (dict(table_rows=0), "table_rows=0"), (dict(free_capacity=-2), "free_capacity=-2"), (dict(max_ctx=2 ** 31 - 5, r2t_stride=2 ** 40), "32 bits"),
    (dict(capacity=2 ** 30 + 1), "32 bits"),
    *[({k: None}, "null pointer") for k in "req prefix new alloc free range r2t positions loc cu seq alloc_out range_out status".split()],
    (dict(parents=None), "go together"), (dict(mask=None), "go together"), (dict(words=0), "mask_words"), (dict(words=17), "mask_words"),
    (dict(r2t_stride=63), "r2t_stride"), (dict(r2p=A[14], r2p_stride=3), "r2p_stride"),
    (dict(seq=A[1]), "overwrites"), (dict(alloc_out=A[1]), "overwrites"), (dict(positions=A[7]), "overwrites"), (dict(cu=A[2]), "overwrites"),
    (dict(range_out=A[3]), "overwrites"), (dict(bs=2000), "workspace"), (dict(bs=2000, ws=A[15], ws_bytes=2000 * 16 - 1), "workspace"),
    (dict(capacity=5000), "workspace"), (dict(bs=2000, ws=A[15] + 4, ws_bytes=1 << 20), "aligned")])
def test_prepare_extend_refuses(change, words):
    rc, error = _call("msgl_prepare_extend", PREPARE, PREPARE_OK, change)
    assert rc < 0 and words in error, error


ATTEND = ("q q_stride k v cache_stride r2t r2t_stride req cu prefix mask words out out_stride tokens bs max_q max_k total Hq Hkv D scale ws ws_bytes "
          "stream").split()
ATTEND_OK = dict(q=A[0], q_stride=1024, k=A[1], v=A[2], cache_stride=512, r2t=A[3], r2t_stride=64, req=A[4], cu=A[5], prefix=A[6], mask=A[7], words=1,
                 out=A[8], out_stride=1024, tokens=8, bs=2, max_q=8, max_k=64, total=0, Hq=8, Hkv=2, D=128, scale=0.1, ws=None, ws_bytes=0, stream=None)


@pytest.mark.parametrize("change,words", [
    (dict(D=64), "head dim"), (dict(Hkv=3), "heads"), (dict(Hkv=0), "heads"), (dict(Hq=6), "heads"), (dict(Hq=32), "heads"), (dict(Hkv=16, Hq=16), "heads"),
    (dict(bs=-1), "bs=-1"), (dict(tokens=-1), "total_tokens=-1"), (dict(max_q=-1), "max_seqlen_q=-1"), (dict(max_q=65), "mask words"),
    (dict(words=0), "mask words"), (dict(words=17), "mask words"), (dict(max_k=0), "max_seqlen_k"), (dict(max_k=2 ** 30 + 1), "max_seqlen_k"),
    *[({k: None}, "null pointer") for k in "q k v r2t req cu prefix mask out".split()],
    (dict(scale=-0.1), "scale"), (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(out=A[0]), "overwrites"),
    (dict(out_stride=1016), "out_stride"), (dict(q_stride=-1024), "q_stride"), (dict(q=A[0] + 2), "aligned"), (dict(k=A[1] + 8), "aligned"),
    (dict(out_stride=1028), "aligned"), (dict(cache_stride=260), "aligned"), (dict(cache_stride=248), "cache_stride")])
def test_tree_attention_refuses(change, words):
    rc, error = _call("msgl_tree_attention", ATTEND, ATTEND_OK, change)
    assert rc < 0 and words in error, error


ACCEPT = "draft target parents cu prefix loc layers num_layers stride Hkv D lens rows tokens next seq bs most stream".split()
ACCEPT_OK = dict(draft=A[0], target=A[1], parents=A[2], cu=A[3], prefix=A[4], loc=A[5], layers=A[6], num_layers=2, stride=512, Hkv=2, D=128, lens=A[7],
                 rows=A[8], tokens=A[9], next=A[10], seq=A[4], bs=2, most=8, stream=None)


@pytest.mark.parametrize("change,words", [
    (dict(bs=-1), "bs=-1"), (dict(bs=2 ** 21), "bs="), (dict(num_layers=-1), "num_layers=-1"), (dict(most=0), "max_accept=0"), (dict(most=1025), "max_accept"),
    *[({k: None}, "null pointer") for k in "draft target parents cu prefix loc layers lens rows tokens next seq".split()],
    (dict(next=A[0]), "overwrites"), (dict(tokens=A[1]), "overwrites"), (dict(lens=A[4]), "overwrites"), (dict(seq=A[3]), "overwrites"),
    (dict(D=6, Hkv=1), "16-byte"), (dict(stride=248), "cache_stride"), (dict(stride=516), "cache_stride"), (dict(Hkv=0), "Hkv=0")])
def test_accept_tree_refuses(change, words):
    rc, error = _call("msgl_accept_tree", ACCEPT, ACCEPT_OK, change)
    assert rc < 0 and words in error, error


LOGPROBS = "logits stride elem ids logprobs entropy top_ids top_lp rows vocab top ws ws_bytes stream".split()
LOGPROBS_OK = dict(logits=A[0], stride=20000, elem=2, ids=A[1], logprobs=A[2], entropy=A[3], top_ids=A[4], top_lp=A[5], rows=3, vocab=20000, top=4, ws=A[6],
                   ws_bytes=1 << 20, stream=None)


@pytest.mark.parametrize("change,words", [
    (dict(rows=-1), "rows=-1"), (dict(vocab=0), "vocab=0"), (dict(vocab=2 ** 30 + 1), "vocab"), (dict(elem=8), "elem_bytes=8"), (dict(top=-1), "top=-1"),
    (dict(top=33), "top=33"), (dict(vocab=3), "top=4"), *[({k: None}, "null pointer") for k in "logits ids logprobs entropy top_ids top_lp".split()],
    (dict(logits=A[0] + 1), "misaligned"), (dict(stride=-1), "row_stride"), (dict(rows=2 ** 24), "segments"), (dict(ws=None), "workspace"),
    (dict(ws_bytes=16), "workspace"), (dict(ws=A[6] + 8), "aligned")])
def test_token_logprobs_refuses(change, words):
    rc, error = _call("msgl_token_logprobs", LOGPROBS, LOGPROBS_OK, change)
    assert rc < 0 and words in error, error


def test_nothing_to_do_is_no_error_and_needs_no_workspace():
    assert _call("msgl_prepare_extend", PREPARE, PREPARE_OK, dict(bs=0))[0] == 0
    for change in (dict(bs=0), dict(tokens=0), dict(max_q=0)):
        assert _call("msgl_tree_attention", ATTEND, ATTEND_OK, change)[0] == 0
    assert _call("msgl_accept_tree", ACCEPT, ACCEPT_OK, dict(bs=0))[0] == 0
    assert _call("msgl_token_logprobs", LOGPROBS, LOGPROBS_OK, dict(rows=0))[0] == 0
    lib, _ = _lib()
    assert lib.msgl_prepare_extend_workspace_bytes(1024, 4096, 1 << 20, 1) == 0 and lib.msgl_prepare_extend_workspace_bytes(1025, 1, 64, 0) == 1025 * 16
    assert lib.msgl_prepare_extend_workspace_bytes(10, 4097, 64, 1) == 160 and lib.msgl_prepare_extend_workspace_bytes(10, 1 << 20, 64, 0) == 0
    assert lib.msgl_tree_attention_workspace_bytes(10, 8, 128, 1) == 0 and lib.msgl_tree_attention_workspace_bytes(10, 8, 128, 3) == 10 * 8 * (3 * 130 + 1) * 4
    assert lib.msgl_token_logprobs_workspace_bytes(0, 100, 2, 0) == 0 and lib.msgl_token_logprobs_workspace_bytes(5, 8185, 2, 9) == 0  # one segment
    assert lib.msgl_token_logprobs_workspace_bytes(5, 8186, 2, 9) > 0 and lib.msgl_token_logprobs_workspace_bytes(5, 8189, 4, 9) == 0


def test_splits_follow_the_bounds():
    from mini_sglang_amd import ops

    assert ops.tree_attention_splits(64, 8, 8192, 16, 8) == 1                # enough requests for every unit
    assert ops.tree_attention_splits(1, 4, 100, 16, 8) == 1                  # nothing worth cutting
    assert ops.tree_attention_splits(0, 4, 100, 16, 8) == ops.tree_attention_splits(2 ** 31 - 1, 4, 2 ** 30, 16, 8, 2 ** 62) == 1
    assert 1 < ops.tree_attention_splits(1, 4, 2 ** 30, 16, 8) <= 256
    assert ops.tree_attention_splits(2, 32, 130001, 4, 1) > 64
    assert ops.tree_attention_splits(16, 16, 16000, 16, 8, 16 * 4000) >= ops.tree_attention_splits(16, 16, 16000, 16, 8) >= 1  # short ones beside a long one


def test_wrappers_refuse_tensors_that_are_not_on_a_gpu():
    from mini_sglang_amd import ops

    i = torch.zeros(2, dtype=torch.int32)
    bf = torch.zeros(2, 4, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="GPU"):
        ops.prepare_extend(i, i, i, i, i, i, i.view(1, 2), i, i, i, i, i, 16)
    with pytest.raises(ValueError, match="GPU"):
        ops.tree_attention(bf, bf, bf, i.view(1, 2), i, i, i, i.view(2, 1).long(), 1, 1, 1.0)
    with pytest.raises(ValueError, match="GPU"):
        ops.accept_tree(i, i, i, i, i, i, None, i, i.view(2, 1), i.view(2, 1), i, i)
    with pytest.raises(ValueError, match="GPU"):
        ops.token_logprobs(bf[0], i)


def test_attention_base_class_has_no_verify_form():
    from mini_sglang_amd.attn.backend_api import AttentionBackend
    from mini_sglang_amd.runtime.batch_info import ForwardMode

    class Nothing(AttentionBackend):
        def init_forward_metadata(self, batch):
            pass

    batch = type("Batch", (), dict(forward_mode=ForwardMode.VERIFY))()
    with pytest.raises(NotImplementedError, match="forward_verify"):
        Nothing().forward(None, None, None, None, batch)
    assert not ForwardMode.VERIFY.is_extend() and not ForwardMode.VERIFY.is_decode() and ForwardMode.VERIFY.is_verify()


# ---------------------------------------------------------------------------------------------------------- the oracles themselves
@pytest.mark.parametrize("Hq,Hkv,nodes,prefix", [(4, 2, [5, 1], [7, 0]), (8, 1, [70], [33])])
def test_attention_oracle_of_a_chain_is_causal_attention(Hq, Hkv, nodes, prefix):
    c = tc.attention_case(nodes, prefix, Hq, Hkv, 4, 3, chain=True)
    exact, _, _ = tc.attention_oracle(c)
    at = 0
    for b, (n, p) in enumerate(zip(nodes, prefix)):
        slots = c["r2t"][c["rows"][b], : p + n].long()
        k, v = (c[x][slots].double().transpose(0, 1).repeat_interleave(Hq // Hkv, 0) for x in "kv")
        seen = torch.ones(n, p + n, dtype=torch.bool).tril(p)
        want = torch.nn.functional.scaled_dot_product_attention(c["q"][at: at + n].double().transpose(0, 1)[None], k[None], v[None], attn_mask=seen,
                                                                scale=c["scale"])[0].transpose(0, 1)
        assert torch.allclose(exact[at: at + n], want, rtol=1e-12, atol=1e-13)
        at += n


def test_logprob_oracle_is_torch_log_softmax():
    x = torch.randn(5, 333, generator=torch.Generator().manual_seed(1)) * 4
    tok = torch.tensor([0, 5, 332, -1, 333], dtype=torch.int32)
    lp, ent, ids, top, _ = tc.logprob_oracle(x, tok, 7)
    want = torch.log_softmax(x.double(), 1)
    assert torch.allclose(lp[:3], want[torch.arange(3), tok[:3].long()], rtol=1e-12) and torch.isnan(lp[3:]).all()
    assert torch.allclose(ent, torch.distributions.Categorical(logits=x.double()).entropy(), rtol=1e-12)
    vals, best = want.topk(7, 1)
    assert torch.equal(ids.long(), best) and torch.allclose(top, vals, rtol=1e-12)


def test_accept_oracle_follows_the_greedy_sequence():
    """Trees that hold the true continuation accept exactly that much of it."""
    rng = random.Random(4)
    for _ in range(50):
        n = rng.randint(1, 40)
        parents = tc.tree_parents(rng, n)
        draft, target = [rng.randrange(3) for _ in range(n)], [rng.randrange(3) for _ in range(n)]
        (path, tokens), = tc.accept_oracle(draft, target, parents, [n], 1024)
        assert path[0] == 0 and all(parents[b] == a or (a == 0 and parents[b] < 0) for a, b in zip(path, path[1:]))
        assert all(draft[b] == target[a] for a, b in zip(path, path[1:])) and tokens == [target[a] for a in path]
        assert not any(max(0, parents[j]) == path[-1] and draft[j] == target[path[-1]] for j in range(path[-1] + 1, n))
