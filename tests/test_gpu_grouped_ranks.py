"""GPU: a sharded run whose Adam phase is GroupedAdamW with a clipped gradient, in float32 and in 8 bits.  What is clipped is the gradient of
the whole closure (it has been all-reduced before the step), so the replicas stay the same bits.  Two ranks share cuda:0 over gloo;
on RCCL one rank runs eagerly and from a captured graph."""
import json
import os
import socket
import subprocess
import sys

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

HERE = os.path.dirname(os.path.abspath(__file__))
STEPS = 40


def ranks(backend, bits, world, tmp_path):
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    procs, outs = [], []
    for r in range(world):
        env = dict(os.environ, RANK=str(r), WORLD_SIZE=str(world), LOCAL_RANK="0", MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port),
                   HSA_ENABLE_IPC_MODE_LEGACY="0")
        outs.append(str(tmp_path / ("rank%d.json" % r)))
        log = open(str(tmp_path / ("rank%d.log" % r)), "w")
        procs.append((subprocess.Popen([sys.executable, "-u", os.path.join(HERE, "grouped_ranks_worker.py"), backend, str(bits), outs[-1]],
                                       env=env, stdout=log, stderr=subprocess.STDOUT), log))
    codes = []
    try:
        for p, log in procs:
            codes.append(p.wait(timeout=100))
            log.close()
    finally:
        for p, _ in procs:
            if p.poll() is None:
                p.kill()                       # exactly the children started here
    assert codes == [0] * world, [open(str(tmp_path / ("rank%d.log" % r))).read()[-3000:] for r in range(world)]
    return [json.load(open(o))["runs"] for o in outs]


def theta(run):
    return np.frombuffer(bytes.fromhex(run["theta"]), dtype=np.float32).astype(np.float64)


def check(run):
    assert run["steps"] == [float(STEPS)] * 10 and np.isfinite(theta(run)).all()
    assert run["step_norm"] == run["full_norm"] > 1e-2                         # the same kernel's sum; it clips


@pytest.mark.parametrize("bits", [32, 8])
def test_two_ranks_keep_the_same_bits(bits, tmp_path):
    a, b = ranks("gloo", bits, 2, tmp_path)
    for key in ("theta", "state", "norm", "full_norm", "step_norm"):
        assert a["eager"][key] == b["eager"][key], key
    check(a["eager"])
    if bits == 32:      # sums over ranks in another order: within 1e-4 after such a run, as for FusedAdam (8-bit codes may fall on another side)
        one, two = theta(a["single"]), theta(a["eager"])
        assert np.linalg.norm(one - two) / np.linalg.norm(one) < 1e-4


@pytest.mark.parametrize("bits", [32, 8])
def test_one_rank_on_rccl_eagerly_and_from_a_graph(bits, tmp_path):
    run, = ranks("nccl", bits, 1, tmp_path)
    for name in ("eager", "graph"):
        check(run[name])
        if bits == 32:
            one, two = theta(run["single"]), theta(run[name])
            assert np.linalg.norm(one - two) / np.linalg.norm(one) < 1e-4
    assert run["graph"]["replays"] == STEPS - 3 and run["eager"]["replays"] == 0
