"""Drawn tokens under tensor parallelism: two gloo ranks serve requests of which some draw (``serve_draws_worker.py``)."""
import json
import os
import sys

import pytest

from ml_framework_b200.dist.launcher import ProcessLauncher

HERE = os.path.dirname(os.path.abspath(__file__))


def _free_port() -> int:
    import socket
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        return s.getsockname()[1]


@pytest.mark.timeout(360)
def test_two_ranks_draw_alike(tmp_path):
    """Each rank's draws are those of the statement over all ranks' logits (checked in the worker). A greedy request, and one with top_k 1, gets the
    tokens beside drawing ones that it gets alone among greedy ones."""
    log, ok = "", False
    for attempt in range(2):              # a second rendezvous on a fresh port if the first one could not be set up
        d = tmp_path / f"try{attempt}"
        launcher = ProcessLauncher(master_port=_free_port(), log_dir=str(d))
        launcher.launch([sys.executable, os.path.join(HERE, "serve_draws_worker.py")], 2)
        ok = launcher.wait_for_all(timeout_s=150)
        log = (d / "rank_0.log").read_text()
        if ok:
            break
        log += (d / "rank_1.log").read_text()
        if "rendezvous" not in log.lower() and "address" not in log.lower() and "connect" not in log.lower():
            break
    assert ok, log[-4000:]
    tokens = json.loads([ln for ln in log.splitlines() if ln.startswith("{")][-1])["tokens"]
    assert len(tokens) == 4 and all(len(t) == 8 and all(0 <= x < 300 for x in t) for run in tokens for t in run)
    for drawn, greedy in (tokens[:2], tokens[2:]):
        assert drawn[1] == greedy[1] and drawn[4] == greedy[4]
        assert drawn[0] != greedy[0] and drawn[2] != greedy[2] and drawn[3] != greedy[3]
