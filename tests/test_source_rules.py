"""Rules that every source, script and build file of the tree keeps, read from the text: no GPU is needed and nothing is run."""
import os
import re

from __graft_entry__ import ROOT

CODE = (".hip", ".h", ".cpp", ".c", ".py", ".sh", ".jl")
FOLDERS = ("bench", "examples", "include", "oracle", "partitionedarrays.jl_amd", "tests", "tools")


def _sources():
    """(path, text) of every source, script and Makefile at the top and in the source folders, this file left out."""
    paths = [os.path.join(ROOT, f) for f in sorted(os.listdir(ROOT))]
    for top in FOLDERS:
        for d, dirs, files in os.walk(os.path.join(ROOT, top)):
            dirs[:] = sorted(x for x in dirs if x not in ("__pycache__", "obj", "build"))
            paths += [os.path.join(d, f) for f in sorted(files)]
    for p in paths:
        if os.path.isfile(p) and (p.endswith(CODE) or os.path.basename(p) == "Makefile") and not os.path.samefile(p, __file__):
            yield os.path.relpath(p, ROOT), open(p, errors="replace").read()


def _places(pattern):
    rx = re.compile(pattern)
    return [f"{p}:{i}: {l.strip()}" for p, txt in _sources() for i, l in enumerate(txt.splitlines(), 1) if rx.search(l)]


def test_the_walk_sees_the_device_code():
    seen = {p for p, _ in _sources()}
    assert {"partitionedarrays.jl_amd/csrc/pa_csr.hip", "partitionedarrays.jl_amd/csrc/Makefile", "tools/probe/spmv_probe.hip", "bench.py"} <= seen


def test_no_write_through_the_scalar_data_cache():
    """The scalar data cache is read-only here: no scalar store or atomic, no write-back or discard of it, comments included."""
    assert _places(r"\bs_(?:(?:buffer|scratch)_)?(?:store|atomic)_|\bs_dcache_(?:wb|discard)") == []


def test_every_stream_has_the_default_priority():
    """Work on streams of different priorities has hung this GPU for good: nothing asks for another one."""
    assert _places(r"StreamCreateWithPriority|Stream\([^)]*priority *=|is_high_priority_stream *= *True") == []


def test_what_a_graph_may_hold_is_cleared_by_a_kernel():
    """A memset recorded into a graph has given wrong results on replays after the first.  pa_scatter_add is the entry point that
    clears memory and may be recorded; the library's other memsets stand in calls that create, allocate or synchronise."""
    txt = dict(_sources())["partitionedarrays.jl_amd/csrc/pa_csr.hip"]
    body = txt[txt.index('extern "C" int pa_scatter_add('):]
    body = body[:body.index("\n}")]
    assert "zero_first" in body and "hipMemset" not in body


def test_device_code_is_compiled_without_packed_float32_instructions():
    """Some packed Float32 instructions have given wrong results on this GPU now and then, and the optimiser makes them from ordinary
    float code: every line that compiles device code switches them off, and no source writes one."""
    assert _places(r"\bv_pk_(add|mul|fma)_f32") == []
    compiles = [(p, l) for p, txt in _sources() for l in txt.replace("\\\n", " ").splitlines()
                if "-O3" in l and re.search(r"--offload-arch=(gfx950|\$\(ARCH\))", l)]
    assert len(compiles) >= 5
    assert [f"{p}: {l}" for p, l in compiles if "-Xclang -target-feature -Xclang -packed-fp32-ops" not in l] == []
