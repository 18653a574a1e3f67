"""bench.py with several ranks: a kernel that waits for a lost neighbour gives up before the section's timer ends the process."""
import os
import re
import subprocess
import sys

import pytest

from __graft_entry__ import ROOT


def _wait(section):
    """What bench.py makes of a section time-out, in a process of its own (importing it alters the environment)."""
    env = {k: v for k, v in os.environ.items() if k not in ("PA_IPC_TIMEOUT_S", "PA_BENCH_SECTION_TIMEOUT_S")}
    if section is not None:
        env["PA_BENCH_SECTION_TIMEOUT_S"] = section
    r = subprocess.run([sys.executable, "-c", "import bench; print(bench.in_launch_wait_s())"], cwd=ROOT, env=env,
                       capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr[-2000:]
    return float(r.stdout.split()[-1])


@pytest.mark.parametrize("section", ["0.5", "10", "49.5", "300"])
def test_the_wait_ends_before_the_section(section):
    """One launch waits at most twice in a row (the neighbour's acknowledgement, then its arrival); half the section is left for
    what the rank does before the launch and behind it."""
    assert 0 < 2 * _wait(section) < float(section) / 2


def test_the_wait_ends_before_every_section_without_the_switch():
    w = _wait(None)
    txt = open(os.path.join(ROOT, "bench.py")).read()
    # (the smallest a section can get: a sum's constant alone)
    sections = re.findall(r'with optional_section\("[^"]+", ([^,]+), N, rank\)', txt)
    assert len(sections) >= 5
    for s in sections:
        assert 0 < 2 * w < int(re.findall(r"\d+", s)[-1]) / 2, s


def test_the_run_uses_that_wait():
    """The limit is read when a link is made: it is set before the package is loaded, once, and a user's own value stands."""
    txt = open(os.path.join(ROOT, "bench.py")).read()
    code = txt[txt.index("\ndef main("):]
    uses = [m.start() for m in re.finditer("PA_IPC_TIMEOUT_S", code)]
    assert len(uses) == 1
    assert code[uses[0]:].startswith('PA_IPC_TIMEOUT_S", str(in_launch_wait_s()))') and uses[0] < code.index("pa = load_package()")


@pytest.mark.parametrize("transport,switch,wanted", [("ipc", None, True), ("ipc", "1", True), ("rccl", None, False), ("rccl", "0", False),
                                                     ("rccl", "1", True), ("host", None, True)])
def test_the_wait_inside_the_launch_is_not_timed_over_rccl_unless_asked_for(transport, switch, wanted):
    env = {} if switch is None else {"PA_MUL_FUSED_RCCL": switch}
    r = subprocess.run([sys.executable, "-c", f"import bench; print(bench.one_launch_section({transport!r}, {env!r}))"], cwd=ROOT,
                       capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr[-2000:]
    assert r.stdout.split()[-1] == str(wanted)
    txt = open(os.path.join(ROOT, "bench.py")).read()
    assert "if N > 1 and want_fused and one_launch_section(transport):" in txt and 'environ["PA_MUL_FUSED_RCCL"]' not in txt
