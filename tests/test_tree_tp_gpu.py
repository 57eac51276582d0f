"""Tree decoding with the model split over two ranks: heads, cache and vocabulary sharded, the trees' layout and acceptance the same on both."""
import json
import os
import socket
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
HERE = os.path.dirname(os.path.abspath(__file__))


def test_two_ranks_decode_trees_to_the_reference_stream():
    import golden_cases as gc

    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    env = dict(os.environ, MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), WORLD_SIZE="2", HSA_ENABLE_IPC_MODE_LEGACY="0", OMP_NUM_THREADS="2")
    procs = [subprocess.Popen([sys.executable, "-u", os.path.join(HERE, "tree_tp_worker.py")], env=dict(env, RANK=str(r)), stdout=subprocess.PIPE,
                              stderr=subprocess.STDOUT, text=True) for r in range(2)]
    outs = []
    for p in procs:
        try:
            out, _ = p.communicate(timeout=110)
        except subprocess.TimeoutExpired:
            for q in procs:
                if q.poll() is None:
                    q.kill()  # exactly the processes started above
            out, _ = p.communicate()
        outs.append(out)
    report = "\n".join(o[-2000:] for o in outs)
    assert all(p.returncode == 0 for p in procs), report
    want = gc.load("e2e_tiny_ps16.pt")["tokens"][:, :24].tolist()
    for out in outs:
        assert json.loads([ln for ln in out.splitlines() if ln.startswith("TOKENS ")][-1][7:]) == want, report
        assert int([ln for ln in out.splitlines() if ln.startswith("STEPS ")][-1][6:]) < 20, report   # drafts were accepted
