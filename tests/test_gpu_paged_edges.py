"""Calls of the paged-cache operators next to a limit."""
import os
import subprocess
import sys

import numpy as np
import pytest

from oracle import paged as ref
from test_gpu_paged import plan_case, run_plan, same_plan

pytestmark = pytest.mark.gpu

HERE = os.path.dirname(os.path.abspath(__file__))
REPO = os.path.dirname(HERE)


def plans_ascending(torch, glc):
    """Every request count around the one where static and dynamic shared memory
    together pass 48 KB, ascending, so that no larger call came before."""
    for B in range(2440, 2461):
        ctx, new, table, pool, free = plan_case(np.random.default_rng(B), B, 16, 90, 3)
        want = ref.plan(ctx, new, 16, table, pool, free, 6000)
        same_plan(run_plan(torch, glc, ctx, new, 16, table, pool, free, 6000), want)


def test_plan_of_every_size_in_a_fresh_process(cuda):
    code = ("import torch\nfrom glacier.inference import distributed_b200 as glc\n"
            "from test_gpu_paged_edges import plans_ascending\nplans_ascending(torch, glc)\n")
    env = dict(os.environ, PYTHONPATH=os.pathsep.join([REPO, HERE, os.environ.get("PYTHONPATH", "")]))
    out = subprocess.run([sys.executable, "-c", code], env=env, capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stdout[-2000:] + out.stderr[-2000:]
