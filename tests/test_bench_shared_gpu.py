"""bench.py with more ranks than GPUs: what a rank takes for itself leaves room for the others."""
import ast
import os
import subprocess
import sys

import pytest

from __graft_entry__ import ROOT


def _env_of(world, devices):
    """bench.shared_gpu_env in a process of its own (importing bench.py alters the environment)."""
    r = subprocess.run([sys.executable, "-c", f"import bench; print(bench.shared_gpu_env({world}, {devices}))"], cwd=ROOT,
                       capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr[-2000:]
    return ast.literal_eval(r.stdout.splitlines()[-1])


@pytest.mark.parametrize("world,devices", [(2, 1), (8, 1), (16, 1), (4, 2), (5, 2), (8, 0)])
def test_the_extents_of_all_ranks_fit_the_device(world, devices):
    per_device = -(-world // max(1, devices))
    e = _env_of(world, devices)
    f = float(e["PA_ARENA_FRACTION"])
    # the library takes no fraction below 0.05 (csrc/pa_arena.hip): what it makes of the value, times the ranks of a device
    assert 0 < f and per_device * max(f, 0.05) <= 0.80
    if per_device <= 8:
        assert per_device * f <= 0.701
        # 256^3 rows per rank: one 16 GiB extent for the matrix streams and one 4 GiB step for the vectors of 288 GB
        assert f * 288e9 >= 20 * 2 ** 30
    assert int(e["PA_FUSED_TAIL_BLOCKS"]) == 32


@pytest.mark.parametrize("world,devices", [(1, 0), (1, 1), (8, 8), (4, 8)])
def test_a_rank_with_a_gpu_of_its_own_keeps_the_defaults(world, devices):
    assert _env_of(world, devices) == {}
