"""gradient_sync.sync_expert_bias over several ranks: processes over gloo on the
CPU with stand-ins for the kernels, and one GPU for each rank where there are two."""

import os
import subprocess
import sys

import pytest
import torch

from tests.test_multiprocess_cpu import ROOT, free_port


def run_ranks(where, world):
    port, env = free_port(), dict(os.environ, DGN_NVLS="0")  # workers may leave early: keep them off the multicast object
    procs = [subprocess.Popen([sys.executable, os.path.join(ROOT, "tests", "mp_bias_worker.py"), where, str(r), str(world),
                               port], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, env=env)
             for r in range(world)]
    # On GPUs every wait of a worker is bounded, and it leaves on its own.
    limit, outs = (180 if where == "cpu" else None), []
    for p in procs:
        try:
            outs.append(p.communicate(timeout=limit)[0])
        except subprocess.TimeoutExpired:
            for q in procs:
                q.kill()
            raise
    for r, (p, out) in enumerate(zip(procs, outs)):
        assert p.returncode == 0 and "WORKER_OK {}".format(r) in out, out[-2000:]


@pytest.mark.parametrize("world", [2, 3])
def test_ranks_step_the_bias_together(world):
    run_ranks("cpu", world)


@pytest.mark.gpu
@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs at least two GPUs")
def test_ranks_step_the_bias_together_on_gpus(dgn_lib):
    run_ranks("gpu", 2)
