"""What the speculative-decoding operators refuse because memory is shared that must not be: several work groups read while others write (every call
here is refused before any launch); and what the GPU tests' inputs of growing scores ask of a kernel."""
import pytest

import tree_cases as tc
import tree_growth_cases as growth
from test_tree_ops_cpu import (A, ACCEPT, ACCEPT_OK, ATTEND, ATTEND_OK, LOGPROBS, LOGPROBS_OK, PREPARE, PREPARE_OK,
                               _call)

I32 = 4


@pytest.mark.parametrize("change", [
    dict(seq=A[1] + I32), dict(cu=A[2] - I32), dict(status=A[2] + I32),           # an output that begins inside an input, or ends in one
    dict(positions=A[7] + 7 * I32), dict(loc=A[7] - 7 * I32), dict(alloc_out=A[3] + I32), dict(range_out=A[5] - I32), dict(mask=A[4] + 9 * I32),
    dict(r2t=A[0] - 3 * 64 * I32 - 63 * I32),                                     # the last entry of the table's last row
    dict(r2p=A[1] - 3 * 8 * I32 - 3 * I32, r2p_stride=8),
    dict(loc=A[9] + 7 * I32), dict(status=A[11] + 2 * I32), dict(seq=A[3]), dict(positions=A[6] + 64 * I32), dict(mask=A[10] - 7 * 8)])  # two outputs
def test_prepare_extend_refuses_memory_that_is_shared(change):
    rc, error = _call("msgl_prepare_extend", PREPARE, PREPARE_OK, change)
    assert rc < 0 and "overwrites" in error, error


def test_prepare_extend_refuses_a_workspace_on_its_arrays():
    big = dict(req=1 << 30, prefix=2 << 30, new=3 << 30, alloc=4 << 30, alloc_out=4 << 30, seq=5 << 30, cu=6 << 30, bs=2000, ws_bytes=1 << 20)
    for ws in ((1 << 30) - 16, (5 << 30) + 7984):
        rc, error = _call("msgl_prepare_extend", PREPARE, PREPARE_OK, dict(big, ws=ws))
        assert rc < 0 and "overwrites" in error, error


@pytest.mark.parametrize("change", [
    dict(lens=A[3] + 2 * I32), dict(next=A[4] - I32), dict(seq=A[4] + I32), dict(rows=A[5] - 15 * I32), dict(tokens=A[6] - 8 * I32), dict(rows=A[6] + 7 * I32),
    dict(lens=A[8] + 15 * I32), dict(next=A[9] + 3 * I32), dict(seq=A[10] - I32)])
def test_accept_tree_refuses_memory_that_is_shared(change):
    rc, error = _call("msgl_accept_tree", ACCEPT, ACCEPT_OK, change)
    assert rc < 0 and "overwrites" in error, error


# (8 rows of 8 heads x 128: q and out are 16 KiB each, rows of 2 KiB)
@pytest.mark.parametrize("change", [
    dict(out=A[0] + 2048), dict(out=A[0] - 16), dict(out=A[0] + 8 * 2048 - 16), dict(q_stride=4096, out=A[0] + 2 * 4096 + 2032, out_stride=4096),
    dict(q_stride=0, out=A[0] + 2032), dict(out=A[0] - 2048 * 5 + 16, out_stride=2048, q_stride=1024),
    dict(cu=A[8] - 8), dict(prefix=A[8] + 8 * 2048 - 4), dict(req=A[8] + 48), dict(mask=A[8] - 7 * 8), dict(ws=A[8] + 1024, ws_bytes=1 << 20, max_k=1 << 20),
    dict(ws=A[0] - 4096, ws_bytes=1 << 20, max_k=1 << 20)])
def test_tree_attention_refuses_memory_that_is_shared(change):
    rc, error = _call("msgl_tree_attention", ATTEND, ATTEND_OK, change)
    assert rc < 0 and "overwrites" in error, error


@pytest.mark.parametrize("change", [
    dict(logprobs=(1 << 30) + 2 * 200 + 196), dict(entropy=(1 << 30) + 402), dict(top_lp=A[1] + 8), dict(top_ids=A[1] - 4 * 12 + 4), dict(entropy=A[2] + 8),
    dict(top_lp=A[4]), dict(ws=(1 << 30) - 16, vocab=20000, stride=20000)])
def test_token_logprobs_refuses_memory_that_is_shared(change):
    ok = dict(LOGPROBS_OK, logits=1 << 30, stride=200, vocab=100)
    rc, error = _call("msgl_token_logprobs", LOGPROBS, ok, change)
    assert rc < 0 and "overwrites" in error, error


@pytest.mark.parametrize("shape", growth.SHAPES)
@pytest.mark.parametrize("waves", [1, 4])
def test_growing_scores_ask_for_every_rescale(shape, waves):
    """The inputs of the GPU test of growing scores: rows are rescaled again and again, and a kernel that left one kind of rescale out would be wrong by
    many times the test's tolerance in a tenth of its rows or more."""
    c = growth.growing_case(*shape, 5)
    exact, absv, size = tc.attention_oracle(c)
    tol = tc.attention_tolerance(exact, absv, size)
    got, count = growth.online_softmax(c, waves)
    assert bool(((got - exact).abs() <= 1e-9 * (1 + absv)).all())
    assert 2 * count > sum(shape[0]) * shape[2]   # one for every other (node, head) pair: a quarter of them look along rising levels, several steps each
    for left_out in ("o", "l") if waves == 1 else ("o", "l", "join"):
        wrong, _ = growth.online_softmax(c, waves, skip=(left_out,))
        rows = ((wrong - exact).abs() > 10 * tol).any(-1)
        assert float(rows.double().mean()) > 0.1, left_out
